// What follows a product of the feed-forward operators where the fp32 sums of a tile lie in
// shared memory, in parts of its depth over the CTAs of a cluster: each CTA sends the others
// their shares (rows) of its part, adds up its own in the order of the parts, applies
// the epilogue and writes it. The shares travel as bulk copies: read by loads from the other
// CTAs' memory, 64 KB took 5 us.
#pragma once
#include <cstdint>

#include "activation.cuh"
#include "ffn_internal.h"
#include "sm100_ptx.cuh"

namespace felix_ffn {

// Outputs and inputs of an epilogue (see Product). extra: bits 1 and 2 for outputs that are
// wanted besides the first. vec: all rows are whole 16-byte vectors.
struct Finish {
  void* out[kMaxProblems];
  int64_t out_ld[kMaxProblems];
  const void* in[2];
  int64_t in_ld[2];
  const void* bias;
  int act;
  uint32_t extra, vec;
};

template <class T>
__device__ __forceinline__ void unpack8(const uint4& w, float (&v)[8]) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Pair<T>::unpack(x[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <class T, int V>
__device__ __forceinline__ void load_values(const uint16_t* p, float (&v)[V]) {
  if constexpr (V == 8)
    unpack8<T>(*reinterpret_cast<const uint4*>(p), v);
  else
    v[0] = Pair<T>::to_float(*p);
}
template <class T, int V>
__device__ __forceinline__ void store_values(uint16_t* p, const float (&v)[V]) {
  if constexpr (V == 8) {
    uint4 w;
    w.x = Pair<T>::pack(v[0], v[1]);
    w.y = Pair<T>::pack(v[2], v[3]);
    w.z = Pair<T>::pack(v[4], v[5]);
    w.w = Pair<T>::pack(v[6], v[7]);
    *reinterpret_cast<uint4*>(p) = w;
  } else {
    *p = Pair<T>::of_float(v[0]);
  }
}

// V features (from f on) of a token, summed over P parts in their order.
template <uint32_t W, int P, int V>
__device__ __forceinline__ void sum_parts(const float4* const (&part)[P], uint32_t row,
                                          uint32_t token, uint32_t f, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = 0.f;
#pragma unroll
  for (int s = 0; s < P; ++s) {
    if constexpr (V == 8) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 x = part[s][row * (W / 4) + ((f / 4 + j) ^ (token & 7))];
        v[4 * j] += x.x;
        v[4 * j + 1] += x.y;
        v[4 * j + 2] += x.z;
        v[4 * j + 3] += x.w;
      }
    } else {
      v[0] += reinterpret_cast<const float*>(part[s])[(row * (W / 4) + ((f / 4) ^ (token & 7))) * 4 +
                                                      f % 4];
    }
  }
}

// The epilogue of V features of a token: v the sums (kGated: of the gate, `up` of the up
// projection), row and f where they stand in the outputs and inputs.
template <class T, int EPI, int V>
__device__ __forceinline__ void finish_values(const Finish& p, uint32_t prob, int64_t row,
                                              uint32_t f, float (&v)[V], const float (&up)[V]) {
  auto out = [&](uint32_t which) {
    return static_cast<uint16_t*>(p.out[which]) + row * p.out_ld[which] + f;
  };
  auto in = [&](uint32_t which) {
    return static_cast<const uint16_t*>(p.in[which]) + row * p.in_ld[which] + f;
  };
  if constexpr (EPI == kLinear) {
    float x[V];
    if (p.in[0]) load_values<T, V>(in(0), x);
    if (p.bias) {
      float b[V];
      load_values<T, V>(static_cast<const uint16_t*>(p.bias) + f, b);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += b[j];
    }
    if (p.extra >> 1 & 1) store_values<T, V>(out(1), v);
    with_activation(p.act, [&]<int ACT>() {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = activate<ACT>(v[j]);
    });
    if (p.in[0]) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += x[j];
    }
    store_values<T, V>(out(prob), v);
  } else if constexpr (EPI == kGated) {
    if (p.extra >> 1 & 1) store_values<T, V>(out(1), v);
    if (p.extra >> 2 & 1) store_values<T, V>(out(2), up);
    with_activation(p.act, [&]<int ACT>() {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = activate<ACT>(v[j]) * up[j];
    });
    store_values<T, V>(out(0), v);
  } else {
    float g[V], u[V], du[V], h[V];
    load_values<T, V>(in(0), g);
    load_values<T, V>(in(1), u);
    with_activation(p.act, [&]<int ACT>() {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float a, d;
        activate_both<ACT>(g[j], a, d);
        du[j] = v[j] * a;
        h[j] = a * u[j];
        v[j] *= u[j] * d;
      }
    });
    store_values<T, V>(out(0), v);
    store_values<T, V>(out(1), du);
    if (p.extra >> 2 & 1) store_values<T, V>(out(2), h);
  }
}

// Where a tile's values go: `tokens` x `features` from (t0, f0) on, of problem `prob`.
struct TilePlace {
  uint32_t prob, t0, f0, tokens, features;
};

// A part is [token][W features] in float4 of 4 features, the q-th of a token at q ^ (token & 7):
// neither 8 tokens' same features nor 32 features of a token conflict.
//
// Rows [me, me + 1) R / P of a tile of R rows (tokens) of W features (kGated: the gate's, then
// from W / 2 on the up projection's). own: this CTA's part, followed by what the others sent,
// in their order.
template <class T, int EPI, uint32_t W, uint32_t R, int P, int V>
__device__ __forceinline__ void finish_share(const Finish& p, const TilePlace& at,
                                             const uint8_t* own, uint32_t me, uint32_t threads) {
  constexpr uint32_t kShare = R / P, kBytes = kShare * W * 4;
  const float4* part[P];
#pragma unroll
  for (uint32_t s = 0; s < P; ++s)
    part[s] = reinterpret_cast<const float4*>(
        s == me ? own + me * kBytes : own + R * W * 4 + (s < me ? s : s - 1) * kBytes);
  const uint32_t first = me * kShare;
  const uint32_t tokens = at.tokens > first ? min(kShare, at.tokens - first) : 0u;
  constexpr uint32_t kPieces = (EPI == kGated ? W / 2 : W) / V;
#pragma unroll 2
  for (uint32_t i = threadIdx.x; i < tokens * kPieces; i += threads) {
    const uint32_t row = i / kPieces, f = i % kPieces * V, token = first + row;
    if (f >= at.features) continue;
    float v[V], up[V];
    sum_parts<W, P, V>(part, row, token, f, v);
    if constexpr (EPI == kGated) sum_parts<W, P, V>(part, row, token, W / 2 + f, up);
    finish_values<T, EPI, V>(p, at.prob, int64_t(at.t0) + token, at.f0 + f, v, up);
  }
}

// Exchanges the shares of a tile whose parts lie at `own` in CTAs first + j * step of the
// cluster (this one: j = me), and finishes this one's. Every thread of the cluster comes here,
// after the parts have been written and fence_proxy_async_smem() by whoever wrote. received:
// a barrier with count 1, in its first phase. Behind `own`, R * W * 4 bytes, there is room for
// (MAXP - 1) / MAXP as much; parts: 1, 2, 4 or 8, MAXP at most.
template <class T, int EPI, uint32_t W, uint32_t R, uint32_t MAXP>
__device__ __forceinline__ void finish_tile(const Finish& p, const TilePlace& at, uint8_t* own,
                                            uint32_t parts, uint32_t me, uint32_t first,
                                            uint32_t step, uint32_t threads, uint64_t* received,
                                            unsigned* status) {
  using namespace felix_sm100;
  if (parts > 1) {
    const uint32_t bytes = R / parts * W * 4;
    cluster_sync();  // every part is there, and nobody's memory is in other use
    if (threadIdx.x < 32 && elect_one()) {
      mbar_arrive_expect_tx(received, (parts - 1) * bytes);
      for (uint32_t j = 1; j < parts; ++j) {
        const uint32_t to = (me + j) % parts;
        bulk_copy_to_cta(smem_u32(own + to * bytes),
                         smem_u32(own + R * W * 4 + (me < to ? me : me - 1) * bytes), bytes,
                         smem_u32(received), first + to * step);
      }
    }
    __syncwarp();
    // Whoever gave up before comes here too, and the others send to it all the same: their
    // copies land before it leaves.
    int none = 0;
    const bool ok = __all_sync(~0u, mbar_sleep_wait(received, 0, &none, status,
                                                    kWdEpilogueTmemFull)) != 0;
    cluster_arrive();
    if (!ok) return cluster_wait();
  } else {
    __syncthreads();
  }
  auto go = [&]<int P>() {
    if (p.vec)
      finish_share<T, EPI, W, R, P, 8>(p, at, own, me, threads);
    else
      finish_share<T, EPI, W, R, P, 1>(p, at, own, me, threads);
  };
  if (parts == 1)
    go.template operator()<1>();
  else if (parts == 2)
    go.template operator()<2>();
  else if constexpr (MAXP >= 4) {
    if (parts == 4)
      go.template operator()<4>();
    else
      go.template operator()<8>();
  }
  if (parts > 1) cluster_wait();  // what this CTA sent has arrived
}

// Host: the epilogue's arguments.
inline Finish finish_of(const Product& x) {
  Finish f{};
  bool vec = true;
  auto check = [&](const void* p, int64_t ld, uint32_t rows) {
    if (p && ((reinterpret_cast<uintptr_t>(p) & 15) || (rows > 1 && ld % 8))) vec = false;
  };
  for (uint32_t i = 0; i < kMaxProblems; ++i) {
    const uint32_t prob = i < x.problems ? i : x.problems - 1;
    f.out[i] = x.out[i].p;
    f.out_ld[i] = x.out[i].ld;
    check(f.out[i], f.out_ld[i], x.m[prob]);
    if (x.n[prob] % 8) vec = false;
    if (f.out[i] && i && x.problems == 1) f.extra |= 1u << i;
  }
  for (uint32_t i = 0; i < 2; ++i) {
    f.in[i] = x.in[i].p;
    f.in_ld[i] = x.in[i].ld;
    check(f.in[i], f.in_ld[i], x.m[0]);
  }
  f.bias = x.bias;
  check(f.bias, 0, 1);
  f.act = x.act;
  f.vec = vec;
  return f;
}

}  // namespace felix_ffn

// Sampling of one token per row of logits from a given uniform number, with
// temperature, top-k, top-p and min-p, for sm_100a.
//
// Definition (x the row, NaN counting as -inf; m its maximum, T > 0):
//   w_i = exp((x_i - m) / T),  mass_i = round(w_i * 2^31), an integer
//   order: larger x first, ties by lower index
//   top-k keeps the first k; top-p those with less than p of the mass of the
//   kept ones before them; min-p those with w_i >= min_p; the first one always
//   stays. The token is the first, by index, at which the running sum of the
//   kept masses exceeds floor(u * their total).
// T <= 0 takes the first of the largest. A row with nothing above -inf gives -1.
//
// Probabilities are summed as integers: the sums, and so every comparison, do
// not depend on the order or on how the row is split, and the same row and
// number give the same token in every batch. 2^-31 of the largest probability
// is the resolution (a running sum in fp32 would have 2^-24 of the total).
// All three filters keep a prefix of the order, so together they are a threshold
// on (value, index), held as one 64-bit number that is larger for what comes first.
//
// A cluster of CTAs shares a row, and each keeps its part in shared memory (or, where
// that is too large, reads it again through the L2): the logits come from HBM once.
// Thresholds come from a histogram over the distance from the maximum (2048 bins up to
// where masses round to 0; even in value, so that few tokens share a bin), merged over
// the cluster by slices. Where a bin holds too many (equal values, a flat row) it is
// split again into 2048 by (value, index) until it does not.
//   top-k of up to 1024 (with or without the others): tokens are counted only, no
//   exponentials; those down to the bin in which the k-th falls go to the first CTA
//   of the cluster, which sorts them and finishes alone. 1 x 32000 fp16: 16 us (21 by
//   one CTA); 256 x 131072 fp32: 152 to 165 us for 134 MB, 13 % of the card's copy rate: three
//   passes of 64 values a thread, barriers, and 15 us of the first CTA alone.
//   else: the bins' masses are summed too; the tokens of the bin in which top-p (or a
//   large top-k) cuts, a few dozen as a rule, are gathered and sorted by every CTA, and
//   a last pass sums what stays. 33 x 50021 bf16: 41 to 42 us, whatever the cluster's size.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "felix_internal.h"
#include "sm100_ptx.cuh"

namespace felix_impl {
namespace smp {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxCtas = 8;
constexpr int kMost = 1024;  // tokens of a bin that are sorted: two per thread
// Tokens of a CTA at most: the low halves of as many masses fit 32 bits. A vocabulary
// of kMaxCtas * kMaxPart, the largest that is taken, has parts of just that.
constexpr uint32_t kMaxPart = 65536;
static_assert(uint64_t(kMaxPart) * 0xffff <= 0xffffffffu);
// Tokens of a CTA where C share a row of V; the last ones may have fewer.
__host__ __device__ constexpr uint32_t part_of(uint32_t V, uint32_t C) {
  return ((V + C - 1) / C + 7) & ~7u;
}
static_assert(part_of(524288, kMaxCtas) == kMaxPart);

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

// NaN as -inf, -0 as +0.
__device__ __forceinline__ float plain(float x) { return x != x ? -INFINITY : x + 0.f; }
// Unsigned key in the order of the values.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ u64 place_of(float x, uint32_t i) {
  return u64(key_of(plain(x))) << 32 | ~i;
}
// (x - top) / T, correctly rounded. With r = RN(1 / T), q = RN(d r) is within a unit
// in the last place, d - q T is exact in one fused operation and q + r (d - q T)
// rounds to the quotient (Markstein, "Computation of elementary functions on the IBM
// RISC System/6000 processor", 1990); quotients near the ends of the range, where
// the remainder is not exact, are divided.
struct Scale {
  float top, temp, rcp;
  bool quick;  // T where no quotient that matters leaves the range
  __device__ __forceinline__ float operator()(float x) const {
    if (x == top) return 0.f;
    const float d = x - top;
    const float q = d * rcp;
    if (quick && q < -1e-20f && q > -1e20f) return fmaf(rcp, fmaf(-q, temp, d), q);
    return __fdiv_rn(d, temp);
  }
};
// expf, not an approximation: the masses are part of the definition.
__device__ __forceinline__ uint32_t mass_of(float x, const Scale& z) {
  return __float2uint_rn(expf(z(x)) * 2147483648.f);
}

struct Cut {  // a bin in which a threshold falls
  int bin;    // kBins: what is past the bins
  uint32_t count, before;  // tokens in it, and in the bins before it
  u64 mass_before;
};

constexpr uint32_t kFew = 1024;  // the largest top-k that one CTA finishes
constexpr int kList = 1024;      // tokens that it sorts

struct Shared {
  // Tokens of a bin, and their masses as sums of the low 16 and of the high bits: 32
  // bits hold those of kMaxPart tokens.
  alignas(16) uint32_t count[kBins];
  union {
    struct {
      uint32_t lo[kBins], hi[kBins];
    };
    u64 list[kList];  // in the first CTA: tokens of a small top-k
  };
  u64 mine[kMost], all[kMost];
  u64 red[kWarps];
  uint32_t red2[kWarps];
  Cut cut;
  u64 found, found_mass;  // of a ranking
  // for the other CTAs of the cluster
  float top;
  u64 kept, first, range[2], slice_mass[2][kMaxCtas];
  uint32_t gathered, listed, slice_count[2][kMaxCtas];  // [0] of the bins, [1] of a bin split again
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int d = 16; d; d /= 2) v += __shfl_xor_sync(~0u, v, d);
  return v;
}
__device__ __forceinline__ u64 warp_max(u64 v) {
#pragma unroll
  for (int d = 16; d; d /= 2) {
    const u64 o = __shfl_xor_sync(~0u, v, d);
    v = o > v ? o : v;
  }
  return v;
}

// Sorts a[0 .. n - 1], n <= 2 * kThreads, in shared memory: bitonic, one or two items
// a thread in registers (tid and tid + kThreads), exchanged by shuffles inside a warp
// and through `a` between warps. Not inlined, as other code that runs once: what a
// row waits for here is, more than anything, instructions that are not yet in the
// SM's cache.
__device__ __noinline__ void sort(u64* a, uint32_t n, bool descending) {
  const uint32_t tid = threadIdx.x;
  uint32_t size = 32;
  while (size < n) size *= 2;
  const u64 flip = descending ? ~0ull : 0;  // sorts a ^ flip upwards
  u64 x[2];
#pragma unroll
  for (int e = 0; e < 2; ++e)
    x[e] = tid + e * kThreads < n ? a[tid + e * kThreads] ^ flip : ~0ull;
  const bool two = size > kThreads;
  if (tid < size || two) {  // whole warps
    for (uint32_t k = 2; k <= 32; k *= 2)
      for (uint32_t j = k / 2; j; j /= 2)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (e && !two) break;
          const u64 y = __shfl_xor_sync(~0u, x[e], j);
          const bool low = ((tid & j) == 0) == (((tid + e * kThreads) & k) == 0);
          x[e] = (x[e] < y) == low ? x[e] : y;
        }
  }
  for (uint32_t k = 64; k <= size; k *= 2) {
    uint32_t j = k / 2;
    if (j == kThreads) {
      const u64 lo = min(x[0], x[1]);
      x[1] = max(x[0], x[1]);
      x[0] = lo;
      j /= 2;
    }
    for (; j >= 32; j /= 2) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (tid + e * kThreads < size) a[tid + e * kThreads] = x[e];
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t i = tid + e * kThreads;
        if (i < size) {
          const u64 y = a[i ^ j];
          const bool low = ((i & j) == 0) == ((i & k) == 0);
          x[e] = (x[e] < y) == low ? x[e] : y;
        }
      }
    }
    if (tid < size || two) {
      for (j = 16; j; j /= 2)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (e && !two) break;
          const u64 y = __shfl_xor_sync(~0u, x[e], j);
          const bool low = ((tid & j) == 0) == (((tid + e * kThreads) & k) == 0);
          x[e] = (x[e] < y) == low ? x[e] : y;
        }
    }
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (tid + e * kThreads < size) a[tid + e * kThreads] = x[e] ^ flip;
  __syncthreads();
}

// Exclusive prefix of the masses of items 2 tid and 2 tid + 1, and their sum.
struct Prefix {
  u64 upto[2], total;
};
__device__ __noinline__ Prefix scan2(uint32_t m0, uint32_t m1, u64* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 v = u64(m0) + m1;
  const u64 own = v;
  for (int d = 1; d < 32; d *= 2) {
    const u64 y = __shfl_up_sync(~0u, v, d);
    if (lane >= d) v += y;
  }
  __syncthreads();
  if (lane == 31) red[warp] = v;
  __syncthreads();
  Prefix r;
  r.total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) v += red[w];
    r.total += red[w];
  }
  r.upto[0] = v - own;
  r.upto[1] = r.upto[0] + m0;
  return r;
}

// A row's part in one CTA: tokens lo .. lo + n - 1. Staged: in shared memory, else
// read from global memory in each pass.
template <typename T, bool kStaged>
struct Row {
  const T* g;     // the row
  const T* s;     // token lo in shared memory
  uint32_t lo, n;
  uint32_t pad;   // the part starts this many elements past a 16-byte boundary
  __device__ __forceinline__ float at(uint32_t j) const {
    return plain(to_f<T>(kStaged ? s[j] : g[lo + j]));
  }
  // f(value, j) for the CTA's tokens, spread over its threads: 16 bytes at a time,
  // kBatch loads under way in a thread, the ends one by one. Values come as they are:
  // NaN and -0 among them.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    constexpr uint32_t kPer = 16 / sizeof(T), kBatch = kStaged ? 1 : 4;
    const T* src = kStaged ? s : g + lo;
    const uint32_t head = min((kPer - pad) % kPer, n), vecs = (n - head) / kPer;
    const uint32_t ends = n - vecs * kPer;
    const uint4* from = reinterpret_cast<const uint4*>(src + head);
    for (uint32_t v0 = threadIdx.x; v0 < vecs; v0 += kBatch * kThreads) {
      uint4 w[kBatch];
#pragma unroll
      for (uint32_t k = 0; k < kBatch; ++k)
        if (v0 + k * kThreads < vecs) w[k] = from[v0 + k * kThreads];
#pragma unroll
      for (uint32_t k = 0; k < kBatch; ++k) {
        const uint32_t v = v0 + k * kThreads;
        if (v >= vecs) break;
        const T* e = reinterpret_cast<const T*>(&w[k]);
#pragma unroll
        for (uint32_t i = 0; i < kPer; ++i) f(to_f<T>(e[i]), head + v * kPer + i);
      }
    }
    for (uint32_t i = threadIdx.x; i < ends; i += kThreads) {
      const uint32_t j = i < head ? i : n - ends + i;
      f(to_f<T>(src[j]), j);
    }
  }
};

template <typename T, bool kStaged>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs A) {
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t C = cluster.num_blocks(), rank = cluster.block_rank();
  const uint32_t row = blockIdx.x / C, V = A.vocab;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float temp = A.temperature ? A.temperature[row] : 1.f;
  const int k = A.top_k ? A.top_k[row] : 0;
  const float p = A.top_p ? A.top_p[row] : 1.f, mp = A.min_p ? A.min_p[row] : 0.f;
  auto of = [&](auto* x, uint32_t r) { return cluster.map_shared_rank(x, r); };

  Row<T, kStaged> x;
  x.g = static_cast<const T*>(A.logits) + int64_t(row) * A.stride;
  const uint32_t run = part_of(V, C);
  x.lo = min(rank * run, V);
  x.n = min(run, V - x.lo);

  // ---- the maximum, and the part into shared memory: 16 bytes at a time, at the
  // same offset from a 16-byte boundary in both memories
  float top = -INFINITY;
  x.pad = uint32_t(reinterpret_cast<uintptr_t>(x.g + x.lo) & 15) / sizeof(T);
  if (kStaged) {
    constexpr uint32_t kPer = 16 / sizeof(T);
    const T* src = x.g + x.lo;
    const uint32_t pad = x.pad;
    T* dst = reinterpret_cast<T*>(raw + ((sizeof(Shared) + 15) & ~size_t(15)));
    x.s = dst + pad;
    const uint32_t vecs = (pad + x.n + kPer - 1) / kPer;
    const uint4* from = reinterpret_cast<const uint4*>(src - pad);
#pragma unroll 4
    for (uint32_t v = tid; v < vecs; v += kThreads) {
      if (v * kPer >= pad && (v + 1) * kPer <= pad + x.n) {
        const uint4 w = __ldg(from + v);
        reinterpret_cast<uint4*>(dst)[v] = w;
        const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (uint32_t i = 0; i < kPer; ++i) top = fmaxf(top, to_f<T>(e[i]));  // not NaN's
      } else {
        for (uint32_t i = v * kPer; i < (v + 1) * kPer; ++i)
          if (i >= pad && i < pad + x.n) {
            const T e = src[i - pad];
            dst[i] = e;
            top = fmaxf(top, to_f<T>(e));
          }
      }
    }
  } else {
    x.each([&](float v, uint32_t) { top = fmaxf(top, v); });
  }
  for (int b = tid; b < kBins; b += kThreads) sh.count[b] = sh.lo[b] = sh.hi[b] = 0;
#pragma unroll
  for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
  if (lane == 0) sh.red2[warp] = __float_as_uint(top);
  __syncthreads();
  top = __uint_as_float(sh.red2[lane % kWarps]);
#pragma unroll
  for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
  if (tid == 0) sh.top = top, sh.listed = 0;
  cluster.sync();
  for (uint32_t r = 0; r < C; ++r) top = fmaxf(top, *of(&sh.top, r));
  top += 0.f;

  if (top == -INFINITY || !(temp > 0.f)) {  // the first of the largest, or none
    u64 best = 0;
    x.each([&](float v, uint32_t j) { best = max(best, place_of(v, x.lo + j)); });
    best = warp_max(best);
    if (lane == 0) sh.red[warp] = best;
    __syncthreads();
    best = warp_max(sh.red[lane % kWarps]);
    if (tid == 0) sh.first = best;
    cluster.sync();
    for (uint32_t r = 0; r < C; ++r) best = max(best, *of(&sh.first, r));
    if (rank == 0 && tid == 0) {
      A.tokens[row] = top == -INFINITY ? -1 : int32_t(~uint32_t(best));
      A.logprobs[row] = top == -INFINITY ? -INFINITY : 0.f;
    }
    cluster.sync();
    return;
  }

  // ---- the histogram
  const Scale z = {top, temp, __frcp_rn(temp), temp > 1e-10f && temp < 1e10f};
  const float to_bin = kBins / (22.5f * temp);  // exp(-22.5) 2^31 < 1/2: mass 0 from there
  auto bin_of = [&](float v) {
    if (v == top) return 0;
    const float d = (top - v) * to_bin;
    return d < float(kBins) ? int(d) : kBins;  // even where d is NaN
  };
  auto tally = [&](int bin, uint32_t mass) {
    atomicAdd(&sh.count[bin], 1u);
    atomicAdd(&sh.lo[bin], mass & 0xffffu);
    atomicAdd(&sh.hi[bin], mass >> 16);
  };
  // The merged histogram, a slice of kBins / C neighbouring bins in each CTA, kEach
  // in each of its first threads, and what is before them in the slice. (Reading all
  // bins of all CTAs in each took longer than the two barriers of the slices: 17
  // against 6 us with masses.) Masses are left out where none were summed.
  constexpr int kEach = kBins / kThreads;
  static_assert(kEach == 4, "bins are read as vectors of four");
  const uint32_t slice = kBins / C;
  uint32_t bc[kEach], pc = 0;
  u64 bm[kEach], pm = 0;
  auto merge = [&](bool with_mass, int which) {
    cluster.sync();
    uint32_t c = 0;
    u64 m = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) bc[e] = 0, bm[e] = 0;
    if (uint32_t(tid) * kEach < slice) {
      const uint32_t at = (rank * slice) / kEach + tid;
#pragma unroll
      for (uint32_t r0 = 0; r0 < uint32_t(kMaxCtas); r0 += 4) {
        uint4 v[4], l[4], h[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
          const uint32_t r = r0 + i;
          v[i] = l[i] = h[i] = make_uint4(0, 0, 0, 0);
          if (r < C) {
            v[i] = reinterpret_cast<const uint4*>(of(sh.count, r))[at];
            if (with_mass) {
              l[i] = reinterpret_cast<const uint4*>(of(sh.lo, r))[at];
              h[i] = reinterpret_cast<const uint4*>(of(sh.hi, r))[at];
            }
          }
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
          bc[0] += v[i].x, bc[1] += v[i].y, bc[2] += v[i].z, bc[3] += v[i].w;
          bm[0] += l[i].x + (u64(h[i].x) << 16), bm[1] += l[i].y + (u64(h[i].y) << 16);
          bm[2] += l[i].z + (u64(h[i].z) << 16), bm[3] += l[i].w + (u64(h[i].w) << 16);
        }
        if (r0 + 4 >= C) break;
      }
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) c += bc[e], m += bm[e];
    uint32_t ic = c;
    u64 im = m;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const uint32_t yc = __shfl_up_sync(~0u, ic, d);
      const u64 ym = __shfl_up_sync(~0u, im, d);
      if (lane >= d) ic += yc, im += ym;
    }
    __syncthreads();
    if (lane == 31) sh.red2[warp] = ic, sh.red[warp] = im;
    __syncthreads();
    pc = ic - c, pm = im - m;
    uint32_t tokens = 0;
    u64 masses = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) pc += sh.red2[w], pm += sh.red[w];
      tokens += sh.red2[w], masses += sh.red[w];
    }
    if (tid < int(C)) {
      *of(&sh.slice_count[which][rank], tid) = tokens;
      *of(&sh.slice_mass[which][rank], tid) = masses;
    }
    cluster.sync();
  };
  // The last bin with tokens before which there is less than `want` (tokens or mass),
  // of the merged ones, with base_* before the first; of `members` tokens those past
  // the bins count as one more bin. One CTA finds it and tells the others.
  auto pick = [&](int which, bool by_mass, double want, uint32_t base_count, u64 base_mass,
                  uint32_t members) -> Cut {
    uint32_t c = base_count + pc, inside = base_count;
    u64 m = base_mass + pm, masses = base_mass;
    for (uint32_t r = 0; r < C; ++r) {
      const uint32_t tokens = sh.slice_count[which][r];
      const u64 mass = sh.slice_mass[which][r];
      if (r < rank) c += tokens, m += mass;
      inside += tokens, masses += mass;
    }
    const bool beyond = inside < members && (by_mass ? double(masses) : double(inside)) < want;
    if (tid == 0 && rank == 0 && beyond)
      for (uint32_t r = 0; r < C; ++r) *of(&sh.cut, r) = {kBins, members - inside, inside, masses};
    if (!beyond) {
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const uint32_t ac = c + bc[e];
        const u64 am = m + bm[e];
        // it qualifies, and what comes after it does not or is nothing
        if (bc[e] && (by_mass ? double(m) : double(c)) < want &&
            (!((by_mass ? double(am) : double(ac)) < want) || ac == inside))
          for (uint32_t r = 0; r < C; ++r)
            *of(&sh.cut, r) = {int(rank * slice) + tid * kEach + e, bc[e], c, m};
        c = ac, m = am;
      }
    }
    if (tid == 0) sh.gathered = 0;
    cluster.sync();
    return sh.cut;
  };
  // The threshold: the last token, in the order, before which there is less than
  // `want`, among those of a cut of the bins. *mass: of all up to and with it.
  auto resolve = [&](bool by_mass, double want, Cut cut, u64* mass) -> u64 {
    u64 low = 0, high = ~0ull;  // once the cut has been split: its range of places
    bool split = false;
    const int bin = cut.bin;
    auto in = [&](float v, u64 c) { return split ? c >= low && c <= high : bin_of(v) == bin; };
    while (cut.count > uint32_t(kMost)) {
      if (!split) {  // the range of the cut
        u64 least = 0, most = 0;  // as maxima of ~c and c
        x.each([&](float v, uint32_t j) {
          const u64 c = place_of(v, x.lo + j);
          if (in(v, c)) least = max(least, ~c), most = max(most, c);
        });
        least = warp_max(least), most = warp_max(most);
        __syncthreads();
        if (lane == 0) sh.mine[warp] = least, sh.mine[kWarps + warp] = most;
        __syncthreads();
        least = warp_max(sh.mine[lane % kWarps]), most = warp_max(sh.mine[kWarps + lane % kWarps]);
        if (tid == 0) sh.range[0] = least, sh.range[1] = most;
        cluster.sync();
        for (uint32_t r = 0; r < C; ++r)
          least = max(least, of(sh.range, r)[0]), most = max(most, of(sh.range, r)[1]);
        low = ~least, high = most;
        split = true;
      }
      int shift = 0;
      while ((high - low) >> shift >= u64(kBins)) ++shift;
      cluster.sync();  // the histograms have been read
      for (int b = tid; b < kBins; b += kThreads) sh.count[b] = sh.lo[b] = sh.hi[b] = 0;
      __syncthreads();
      x.each([&](float v, uint32_t j) {
        const u64 c = place_of(v, x.lo + j);
        if (c >= low && c <= high) tally(int((high - c) >> shift), mass_of(v, z));
      });
      merge(true, 1);
      cut = pick(1, by_mass, want, cut.before, cut.mass_before, 0);
      const u64 up = high - (u64(cut.bin) << shift);
      const u64 down = (u64(1) << shift) - 1;
      low = up - low < down ? low : up - down;
      high = up;
    }
    x.each([&](float v, uint32_t j) {
      const u64 c = place_of(v, x.lo + j);
      if (in(v, c)) sh.mine[atomicAdd(&sh.gathered, 1u)] = c;
    });
    cluster.sync();  // histograms have been read too
    uint32_t n = 0;
    for (uint32_t r = 0; r < C; ++r) {
      const uint32_t m = *of(&sh.gathered, r);
      const u64* from = of(sh.mine, r);
      for (uint32_t j = tid; j < m; j += kThreads) {
        const u64 c = from[j];
        sh.all[n + j] = c;
      }
      n += m;
    }
    __syncthreads();
    sort(sh.all, n, true);
    uint32_t m[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
      m[e] = 2 * tid + e < n ? mass_of(value_of(uint32_t(sh.all[2 * tid + e] >> 32)), z) : 0u;
    const Prefix at = scan2(m[0], m[1], sh.red);
    // the last one that stays is the one whose successor, in the order, does not
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t i = 2 * tid + e;
      const u64 m0 = cut.mass_before + at.upto[e], m1 = m0 + m[e];
      const uint32_t c0 = cut.before + i;
      const bool stays = (by_mass ? double(m0) : double(c0)) < want;
      const bool next = i + 1 < n && (by_mass ? double(m1) : double(c0 + 1)) < want;
      if (i < n && stays && !next) sh.found = sh.all[i], sh.found_mass = m1;
    }
    __syncthreads();
    *mass = sh.found_mass;
    return sh.found;
  };

  u64 least = 0;  // what stays: places from here up
  const bool only_first = (A.top_p && !(p > 0.f)) || (A.min_p && !(mp <= 1.f));
  const bool by_count = k > 0 && uint32_t(k) < V, by_mass = A.top_p && p < 1.f;

  // ---- a small top-k: the first CTA finishes
  bool few = by_count && uint32_t(k) <= kFew;
  if (few) {
    x.each([&](float v, uint32_t) {
      const int b = bin_of(v);
      if (b < kBins) atomicAdd(&sh.count[b], 1u);
    });
    merge(false, 0);
    const Cut cut = pick(0, false, double(k), 0, 0, V);
    few = cut.before + cut.count <= uint32_t(kList);
    if (few) {
      // The smallest value in the bin: bins go up as values go down. It is a few
      // roundings from top - (bin + 1) / to_bin; where that does not bracket it, the
      // whole range of values does.
      uint32_t low = key_of(-INFINITY), high = key_of(top);
      const float guess = top - float(cut.bin + 1) / to_bin;
      if (guess < top && guess > -INFINITY) {
        const uint32_t l = max(key_of(guess - 1e-5f * (fabsf(top) + fabsf(guess))), low);
        const uint32_t h = min(key_of(guess + 1e-5f * (fabsf(top) + fabsf(guess))), high);
        if (bin_of(value_of(l)) > cut.bin) low = l;
        if (bin_of(value_of(h)) <= cut.bin) high = h;
      }
      while (cut.bin < kBins && low < high) {
        const uint32_t mid = low + (high - low) / 2;
        if (bin_of(value_of(mid)) <= cut.bin) high = mid;
        else low = mid + 1;
      }
      const float from = cut.bin < kBins ? value_of(high) : -INFINITY;
      x.each([&](float v, uint32_t j) {
        if (plain(v) >= from) sh.mine[atomicAdd(&sh.gathered, 1u)] = place_of(v, x.lo + j);
      });
      __syncthreads();
      // its place in the first CTA's list, then the copy
      const uint32_t n = sh.gathered;
      if (tid == 0) sh.red2[0] = atomicAdd(of(&sh.listed, 0), n);
      __syncthreads();
      u64* list = of(sh.list, 0) + sh.red2[0];
      for (uint32_t i = tid; i < n; i += kThreads) list[i] = sh.mine[i];
    } else {  // many near the k-th: the other way, with the bins' masses
      for (int b = tid; b < kBins; b += kThreads) sh.count[b] = 0;
    }
    cluster.sync();
  }
  if (few) {
    if (rank != 0) return;
    const uint32_t n = sh.listed;
    sort(sh.list, n, true);
    // masses in the order, what stays of them, and those in the order of indexes
    const uint32_t first_k = min(n, uint32_t(k));
    uint32_t m[2], stay = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t i = 2 * tid + e;
      m[e] = i < first_k ? mass_of(value_of(uint32_t(sh.list[i] >> 32)), z) : 0u;
    }
    Prefix at = scan2(m[0], m[1], sh.red);
    const double want = double(p) * double(at.total);
    u64 item[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t i = 2 * tid + e;
      bool on = i < first_k && (!by_mass || double(at.upto[e]) < want);
      if (on && A.min_p) on = !(expf(z(value_of(uint32_t(sh.list[i] >> 32)))) < mp);
      if (only_first) on = false;
      on |= i == 0;
      item[e] = on ? u64(~uint32_t(sh.list[i])) << 32 | m[e] : ~0ull;
      stay += on;
    }
    __syncthreads();
    stay = uint32_t(__syncthreads_count(stay > 0)) + uint32_t(__syncthreads_count(stay > 1));
#pragma unroll
    for (int e = 0; e < 2; ++e) sh.list[2 * tid + e] = item[e];
    __syncthreads();
    sort(sh.list, stay, false);  // what stays is a prefix: the first `stay`, by index
#pragma unroll
    for (int e = 0; e < 2; ++e)
      m[e] = 2 * tid + e < stay ? uint32_t(sh.list[2 * tid + e]) : 0u;
    at = scan2(m[0], m[1], sh.red);
    const u64 total = at.total;
    const double u = double(A.uniform[row]) * double(total);
    u64 target = u > 0. ? u64(u) : 0;
    if (target >= total) target = total - 1;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (target >= at.upto[e] && target < at.upto[e] + m[e]) {
        const uint32_t i = uint32_t(sh.list[2 * tid + e] >> 32);
        const T* g = x.g;
        A.tokens[row] = int32_t(i);
        A.logprobs[row] =
            z(plain(to_f<T>(g[i]))) - logf(__ull2float_rn(total) * 4.656612873077393e-10f);
      }
    return;
  }

  if (only_first) {
    least = ~0ull;
  } else if (by_count || by_mass) {
    x.each([&](float v, uint32_t) {
      const int b = bin_of(v);
      if (b < kBins) tally(b, mass_of(v, z));
    });
    merge(true, 0);
    u64 total = 0;
    for (uint32_t r = 0; r < C; ++r) total += sh.slice_mass[0][r];
    // top-k, then top-p of what it leaves; `resolve` may use the bins again
    const uint32_t opc = pc, oc[kEach] = {bc[0], bc[1], bc[2], bc[3]};
    const u64 opm = pm, om[kEach] = {bm[0], bm[1], bm[2], bm[3]};
#pragma unroll 1
    for (int pass = by_count ? 0 : 1; pass < (by_mass ? 2 : 1); ++pass) {
      const double want = pass ? double(p) * double(total) : double(k);
      const Cut cut = pick(0, pass, want, 0, 0, pass ? 0 : V);
      least = max(least, resolve(pass, want, cut, &total));
      if (pass || !by_mass) break;
#pragma unroll
      for (int e = 0; e < kEach; ++e) bc[e] = oc[e], bm[e] = om[e];
      pc = opc, pm = opm;
      cluster.sync();  // lists have been read
    }
  }

  // ---- the kept mass: each warp a run of neighbouring tokens
  const u64 top_place = key_of(top);
  auto kept = [&](uint32_t j) -> uint32_t {
    const float v = x.at(j);
    const u64 c = place_of(v, x.lo + j);
    if (only_first ? (c >> 32) != top_place : c < least) return 0u;
    const float w = expf(z(v));
    if (v != top && w < mp) return 0u;
    return __float2uint_rn(w * 2147483648.f);
  };
  const uint32_t part = ((x.n + kWarps - 1) / kWarps + 31) & ~31u;
  const uint32_t j0 = min(warp * part, x.n), j1 = min(j0 + part, x.n);
  u64 sum = 0;
  for (uint32_t j = j0 + lane; j < j1; j += 32) sum += kept(j);
  sum = warp_sum(sum);
  if (lane == 0) sh.red[warp] = sum;
  __syncthreads();
  u64 here = 0, before_warp = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before_warp += sh.red[w];
    here += sh.red[w];
  }
  if (tid == 0) sh.kept = here;
  cluster.sync();
  u64 total = 0, before = 0;
  for (uint32_t r = 0; r < C; ++r) {
    const u64 v = *of(&sh.kept, r);
    if (r < rank) before += v;
    total += v;
  }
  // only_first: of the largest ones the first, whatever u
  const double u = only_first ? 0. : double(A.uniform[row]) * double(total);
  u64 target = u > 0. ? u64(u) : 0;
  if (target >= total) target = total - 1;
  before += before_warp;
  if (target >= before && target < before + sum) {  // in this warp's run
    for (uint32_t b = j0; b < j1; b += 32) {
      const uint32_t j = b + lane;
      const uint32_t m = j < j1 ? kept(j) : 0u;
      u64 upto = m;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const u64 y = __shfl_up_sync(~0u, upto, d);
        if (lane >= d) upto += y;
      }
      const uint32_t over = __ballot_sync(~0u, before + upto > target);
      if (over) {
        if (lane == __ffs(over) - 1) {
          A.tokens[row] = int32_t(x.lo + j);
          const u64 all = only_first ? u64(1) << 31 : total;
          A.logprobs[row] = z(x.at(j)) -
                            logf(__ull2float_rn(all) * 4.656612873077393e-10f);
        }
        break;
      }
      before += __shfl_sync(~0u, upto, 31);
    }
  }
  cluster.sync();  // no CTA leaves while another reads from it
}

template <typename T>
FelixCode launch(const SampleArgs& a, DeviceInfo* dev, cudaStream_t stream) {
  const size_t fixed = (sizeof(Shared) + 15) & ~size_t(15);
  // Enough CTAs that every SM has one, as long as each has 2048 tokens or more; at most
  // kMaxPart tokens in each (the histogram's sums) and 208 KB. Parts of which two fit
  // an SM's shared memory are staged there; larger ones (many rows of a large
  // vocabulary) are read again through the L2: two CTAs an SM of 208 KB are half of it,
  // what one die's half holds. With 256 rows of fp32, top-k 1000, in clusters of 2, 4
  // and 8: 100000 tokens 128, 154 and 207 us; 131072 tokens 131 to 200, depending on
  // where the rows lie, 155 and 220; 151936 tokens 176 and 229 by 4 and 8; 200003 tokens
  // 205 and 256.
  uint32_t C = 1;
  auto bytes = [&](uint32_t c) {
    return fixed + (size_t(part_of(a.vocab, c)) + 16) * sizeof(T);
  };
  while (C < kMaxCtas && ((a.rows * uint64_t(C) < uint32_t(dev->num_sms) && a.vocab / C > 4096) ||
                          part_of(a.vocab, C) > kMaxPart ||
                          a.vocab / C * sizeof(T) > 208 * 1024))
    C *= 2;
  const bool staged = bytes(C) <= 110 * 1024;
  static PerDeviceOnce once;
  const int rc = once.run(dev->ordinal, [&] {
    return cudaFuncSetAttribute(sample_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                dev->max_smem_optin) == cudaSuccess &&
                   cudaFuncSetAttribute(sample_kernel<T, false>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        int(fixed)) == cudaSuccess
               ? 0 : -1;
  });
  if (rc != 0) return launch_error(cudaGetLastError(), "sample: attributes");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.rows * C);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = staged ? bytes(C) : fixed;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = C;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = staged ? cudaLaunchKernelEx(&cfg, sample_kernel<T, true>, a)
                               : cudaLaunchKernelEx(&cfg, sample_kernel<T, false>, a);
  if (e != cudaSuccess) return launch_error(e, "sample");
  return FelixCode{FELIX_SUCCESS, cudaSuccess};
}

}  // namespace smp

FelixCode sample_launch(const SampleArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return FelixCode{FELIX_SUCCESS, cudaSuccess};
  DeviceInfo* dev = current_device_info();
  if (!dev) return launch_error(cudaGetLastError(), "sample: no device");
  switch (a.dtype) {
    case FELIX_F16: return smp::launch<__half>(a, dev, stream);
    case FELIX_BF16: return smp::launch<__nv_bfloat16>(a, dev, stream);
    default: return smp::launch<float>(a, dev, stream);
  }
}

}  // namespace felix_impl

// Attention over the 4-bit paged cache for sm_100a: the new tokens of every
// slot (one in a decode step, a few when drafts are verified) against all that
// the slot's cache holds.
//
//   O = softmax(scale * q K^T) V,  K = base_k + scale_k (c_k - 8), V likewise,
//   row i of a slot's n new tokens sees the tokens 0 .. len - n + i.
//
// Mathematics. Nothing is dequantised. With one (scale, base) per token,
//   q . K_t = scale_k (q . c_t) + (base_k - 8 scale_k) sum(q),
//   sum_t p_t V_t = sum_t (p_t scale_v) (c_t - 8) + sum_t p_t base_v,
// so the matrix instructions multiply the raw codes, which the cache's layout
// gives as fp16 subnormals (exact), and the scales meet fp32 scores and
// probabilities. Both products run transposed (codes are the 16-row operand,
// 8 query rows the n side): a group of query heads of one key/value head fills
// the instruction, and the scores' registers become the other operand of the
// second product by an 8 x 8 transpose in the warp. p_t scale_v is rounded to
// fp16 for that product; its exponent is taken out first (the running maximum is
// that of score + exponent of scale_v), so that neither tiny nor huge values
// lose bits, and the -8 is applied to the sum of the same rounded numbers, so
// that the offset cancels exactly. Sums and statistics are fp32.
#include "felix_internal.h"
#include "kv4_layout.cuh"
#include "sm100_ptx.cuh"

namespace felix_impl {
namespace kv4 {

using namespace felix_kv4;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kCentre = 8;  // blocks of a warp between two centrings of the sums
constexpr int kTile = kBlock * kWarps;  // tokens of a tile: one block per warp

struct AttnParams {
  CacheView c;
  const void* q;
  int64_t qs_slot, qs_head, qs_row;  // element strides of q
  void* out;                         // [slots, heads, rows, D] contiguous
  float* lse;                        // [slots, heads, rows] or nullptr
  const int32_t* counts;             // new tokens of each slot, or nullptr: rows
  uint32_t heads, rows, group;       // group = heads / kv_heads
  uint32_t row_tiles;                // tiles of 8 * NT (row, head) pairs
  float scale_log2;                  // softmax scale * log2(e)
  uint32_t* counters;                // one per CTA, zero between launches
  float* partials;                   // [CTA][2][8 NT][D + 2]
};

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int W>
struct Words;  // W 32-bit words loaded as one vector
template <>
struct Words<4> {
  uint32_t w[4];
  __device__ __forceinline__ void load(const unsigned char* p) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  }
};
template <>
struct Words<2> {
  uint32_t w[2];
  __device__ __forceinline__ void load(const unsigned char* p) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = v.x, w[1] = v.y;
  }
};

// A lane's share of one block: D/32 words of K for tokens g and g + 8, of V for
// the token pairs of both halves, and the parameters of tokens g and g + 8.
template <int D>
struct BlockRegs {
  Words<D / 32> k0, k1, v0, v1;
  uint32_t kp0, kp1, vp0, vp1;
  bool there;
  __device__ __forceinline__ void load(const unsigned char* p, int lane) {
    there = p != nullptr;
    if (!there) return;
    constexpr int kLane = D / 8;  // bytes of a lane's vector
    const int g = lane >> 2;
    k0.load(p + lane * kLane);
    k1.load(p + 4 * D + lane * kLane);
    v0.load(p + v_codes_at(D) + lane * kLane);
    v1.load(p + v_codes_at(D) + 4 * D + lane * kLane);
    const uint32_t* kp = reinterpret_cast<const uint32_t*>(p + k_params_at(D));
    const uint32_t* vp = reinterpret_cast<const uint32_t*>(p + v_params_at(D));
    kp0 = __ldg(kp + g), kp1 = __ldg(kp + g + 8);
    vp0 = __ldg(vp + g), vp1 = __ldg(vp + g + 8);
  }
};

// (scale, base) of a K token -> scale and base - 8 scale.
__device__ __forceinline__ float2 k_params(uint32_t p) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
  return make_float2(f.x, fmaf(-8.f, f.x, f.y));
}
// (scale, base) of a V token: the scale's exponent E (of the smallest normal
// where it is subnormal), 2^-E, scale * 2^-E, base * 2^-E.
struct VParams {
  float e, inv, mant, base;
};
__device__ __forceinline__ VParams v_params(uint32_t p) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
  const int e = max(int((p >> 10) & 31u), 1) - 15;
  VParams r;
  r.e = float(e);
  r.inv = __int_as_float((127 - e) << 23);
  r.mant = f.x * r.inv;
  r.base = f.y * r.inv;
  return r;
}

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

// One segment (slot, kv head, tile of rows) or a part of it: tokens
// [tile_lo, tile_hi) * kTile. Registers of a warp after its blocks.
template <typename T, int D, int NT>
struct Attn {
  static constexpr int kRows = 8 * NT;
  static constexpr int kW = D / 32;       // words of a lane's vector
  uint32_t q[NT][2 * kW][2];              // operand registers of 8 query rows each
  // score = (raw * scale_k + qs * (base_k - 8 scale_k)) * f: raw sums are in units
  // of 2^-24 and of the row's power of two, and so is qs = sum(q), so that the
  // terms cancel before anything is rounded to a scale
  float f[NT][2], qs[NT][2];
  int lim[NT][2];                         // tokens that this thread's two rows see
  float o[NT][D / 16][4], o8[NT][4];      // sums of p scale_v c, of 8 p scale_v since centre()
  float m[NT][2], l[NT][2], b[NT][2];     // running maximum, sum of p, sum of p base_v
  int low;                                // the smallest of lim

  __device__ __forceinline__ void load_q(const AttnParams& P, uint32_t slot, uint32_t kvh,
                                         uint32_t rt, int len, int count, int lane) {
    const int g = lane >> 2, t = lane & 3;
    low = len;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint32_t r = rt * kRows + 8 * n + g;
      const uint32_t row = r / P.group, head = kvh * P.group + r % P.group;
      const bool live = row < P.rows && int(row) < count;
      float v[D / 4];
      float top = 0.f, sum = 0.f;
      const T* src = static_cast<const T*>(P.q) + int64_t(slot) * P.qs_slot +
                     int64_t(head) * P.qs_head + int64_t(row) * P.qs_row + t * (D / 4);
#pragma unroll
      for (int i = 0; i < D / 4; ++i) {
        v[i] = live ? to_f<T>(src[i]) : 0.f;
        top = fmaxf(top, fabsf(v[i]));
      }
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
      // scale the row by a power of two so that its largest value is in
      // [2^12, 2^13): fp16 then holds bf16 and tiny rows too
      const int e = int(__float_as_uint(top) >> 23) - 127;
      const int up = (top > 0.f && e < 128) ? min(12 - e, 100) : 0;
      const float mul = __int_as_float((127 + up) << 23);
#pragma unroll
      for (int i = 0; i < D / 4; ++i) {
        v[i] *= mul;
        sum += v[i];
      }
      sum += __shfl_xor_sync(~0u, sum, 1);
      sum += __shfl_xor_sync(~0u, sum, 2);
#pragma unroll
      for (int w = 0; w < kW; ++w) {
        const float* x = v + 8 * w;
        constexpr float s = 0.0625f;
        q[n][2 * w][0] = felix_sm100::pack_half2(x[0], x[4]);
        q[n][2 * w][1] = felix_sm100::pack_half2(x[1] * s, x[5] * s);
        q[n][2 * w + 1][0] = felix_sm100::pack_half2(x[2], x[6]);
        q[n][2 * w + 1][1] = felix_sm100::pack_half2(x[3] * s, x[7] * s);
      }
      // statistics of rows 2t and 2t + 1, which lanes 4 * (2t) and 4 * (2t + 1) hold
      const float down = __int_as_float((127 - up) << 23);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int from = 4 * (2 * t + c);
        const float dn = __shfl_sync(~0u, down, from), sm = __shfl_sync(~0u, sum, from);
        f[n][c] = P.scale_log2 * dn * 16777216.f;  // raw sums are of code * 2^-24
        qs[n][c] = sm * (1.f / 16777216.f);
        const uint32_t rr = rt * kRows + 8 * n + 2 * t + c;
        const int rw = int(rr / P.group);
        lim[n][c] = (rw < int(P.rows) && rw < count) ? max(len - count + rw + 1, 0) : 0;
        m[n][c] = -INFINITY;
        l[n][c] = b[n][c] = 0.f;
      }
      // rows past the last do not narrow the unmasked range
      const bool past = rt * kRows + 8 * n + 2 * t >= P.rows * P.group;
      if (!past) low = min(low, min(lim[n][0], rt * kRows + 8 * n + 2 * t + 1 < P.rows * P.group
                                                   ? lim[n][1] : lim[n][0]));
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[n][j][c] = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) o8[n][c] = 0.f;
    }
    low = min(low, __shfl_xor_sync(~0u, low, 1));
    low = min(low, __shfl_xor_sync(~0u, low, 2));
  }

  __device__ __forceinline__ void block(const BlockRegs<D>& x, int token0, int lane) {
    const int g = lane >> 2;
    const float2 ka = k_params(x.kp0), kb = k_params(x.kp1);
    const VParams va = v_params(x.vp0), vb = v_params(x.vp1);
    uint32_t pt[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kW; ++w) {
        const uint32_t lo = 0x000f000fu, hi = 0x00f000f0u;
        const uint32_t a = x.k0.w[w], c = x.k1.w[w], a8 = a >> 8, c8 = c >> 8;
        mma16816(s, a & lo, c & lo, a & hi, c & hi, q[n][2 * w][0], q[n][2 * w][1]);
        mma16816(s, a8 & lo, c8 & lo, a8 & hi, c8 & hi, q[n][2 * w + 1][0], q[n][2 * w + 1][1]);
      }
      // s[0], s[1]: token g of rows 2t, 2t + 1; s[2], s[3]: token g + 8.
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        s[c] = fmaf(fmaf(s[c], ka.x, qs[n][c] * ka.y), f[n][c], va.e);
        s[2 + c] = fmaf(fmaf(s[2 + c], kb.x, qs[n][c] * kb.y), f[n][c], vb.e);
      }
      bool on[4] = {true, true, true, true};
      if (token0 + int(kBlock) > low) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          on[c] = token0 + g < lim[n][c];
          on[2 + c] = token0 + g + 8 < lim[n][c];
          if (!on[c]) s[c] = -INFINITY;
          if (!on[2 + c]) s[2 + c] = -INFINITY;
        }
      }
      // The sums are kept relative to a maximum that is only moved when a score
      // passes it by 2^8: probabilities stay below 2^9 and fp16 holds them.
      const bool over = s[0] > m[n][0] + 8.f || s[2] > m[n][0] + 8.f || s[1] > m[n][1] + 8.f ||
                        s[3] > m[n][1] + 8.f;
      if (__any_sync(~0u, over)) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float top = fmaxf(m[n][c], fmaxf(s[c], s[2 + c]));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
          const float keep = top == -INFINITY ? 1.f : ex2(m[n][c] - top);
          m[n][c] = top;
          l[n][c] *= keep;
          b[n][c] *= keep;
          o8[n][c] *= keep;
          o8[n][2 + c] *= keep;
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            o[n][j][c] *= keep;
            o[n][j][2 + c] *= keep;
          }
        }
      }
      float p[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float e = on[c] ? ex2(s[c] - m[n][c & 1]) : 0.f;
        const VParams& v = c < 2 ? va : vb;
        // a masked token's parameters may be anything, NaN among it
        p[c] = on[c] ? e * v.mant : 0.f;
        l[n][c & 1] = on[c] ? fmaf(e, v.inv, l[n][c & 1]) : l[n][c & 1];
        b[n][c & 1] = on[c] ? fmaf(e, v.base, b[n][c & 1]) : b[n][c & 1];
      }
      pt[n][0] = transpose8x8(felix_sm100::pack_half2(p[0], p[1]));
      pt[n][1] = transpose8x8(felix_sm100::pack_half2(p[2], p[3]));
      constexpr uint32_t eight = 0x00080008u;  // 8 * 2^-24, the codes' unit
      mma16816(o8[n], eight, eight, eight, eight, pt[n][0], pt[n][1]);
    }
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      const uint32_t lo = 0x000f000fu, hi = 0x00f000f0u;
      const uint32_t a = x.v0.w[w], c = x.v1.w[w], a8 = a >> 8, c8 = c >> 8;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma16816(o[n][2 * w], a & lo, a & hi, c & lo, c & hi, pt[n][0], pt[n][1]);
        mma16816(o[n][2 * w + 1], a8 & lo, a8 & hi, c8 & lo, c8 & hi, pt[n][0], pt[n][1]);
      }
    }
  }

  // Takes the codes' offset out of the sums: o (the odd registers are of 16 code)
  // would otherwise grow with the number of tokens, and its last bits with it,
  // while the result is a mean. Once every kCentre blocks.
  __device__ __forceinline__ void centre() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          o[n][j][c] -= o8[n][c];
          o[n][j][2 + c] = fmaf(-16.f, o8[n][c], o[n][j][2 + c]);
        }
#pragma unroll
      for (int c = 0; c < 4; ++c) o8[n][c] = 0.f;
    }
  }

  // Writes the warp's sums to shared memory: O [kRows][D] (base term included)
  // and (m, l) of each row.
  __device__ __forceinline__ void park(float* so, float* sml, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int x = 4; x < 32; x *= 2) {
          l[n][c] += __shfl_xor_sync(~0u, l[n][c], x);
          b[n][c] += __shfl_xor_sync(~0u, b[n][c], x);
        }
        const int r = 8 * n + 2 * t + c;
        if (g == 0) sml[2 * r] = m[n][c], sml[2 * r + 1] = l[n][c];
        constexpr float u = 16777216.f;
        const float off = b[n][c];
        float4* dst = reinterpret_cast<float4*>(so + r * D + g * (D / 8));
#pragma unroll
        for (int w = 0; w < kW; ++w)
          dst[w] = make_float4(fmaf(o[n][2 * w][c], u, off), fmaf(o[n][2 * w][2 + c], u / 16, off),
                               fmaf(o[n][2 * w + 1][c], u, off),
                               fmaf(o[n][2 * w + 1][2 + c], u / 16, off));
      }
    }
  }
};

// Persistent grid. The work is a line of units (a segment's tiles of kTile
// tokens, segment after segment; an empty slot counts as one unit), cut into
// equal shares, one per CTA, whatever the slots' lengths. A segment that lies in
// several shares is finished by the CTA that comes last to it, which joins the
// parts in the order of the shares: the result does not depend on who is last.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads) kv4_attn_kernel(const AttnParams P) {
  constexpr int kRows = 8 * NT;
  __shared__ __align__(16) float so[kWarps][kRows * D];
  __shared__ float sml[kWarps][2 * kRows];
  __shared__ uint32_t s_scan[kWarps];
  __shared__ uint32_t s_at[2];
  __shared__ uint32_t s_ticket;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const CacheView& c = P.c;
  const uint32_t per_tile = c.kv_heads * P.row_tiles;

  // ---- this CTA's share: units before each thread's run of slots, then the slot
  const uint32_t run = (c.slots + kThreads - 1) / kThreads;
  const uint32_t s0 = min(tid * run, c.slots), s1 = min(s0 + run, c.slots);
  uint32_t mine = 0;
  for (uint32_t s = s0; s < s1; ++s)
    mine += max((slot_reach(c, s) + kTile - 1) / kTile, 1) * per_tile;
  uint32_t upto = mine;
#pragma unroll
  for (int x = 1; x < 32; x *= 2) {
    const uint32_t v = __shfl_up_sync(~0u, upto, x);
    if (lane >= x) upto += v;
  }
  if (lane == 31) s_scan[warp] = upto;
  __syncthreads();
  uint32_t total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) upto += s_scan[w];
    total += s_scan[w];
  }
  const uint32_t quota = (total + gridDim.x - 1) / gridDim.x;
  const uint32_t first = blockIdx.x * quota, last = min(first + quota, total);
  if (first >= last) return;
  if (first >= upto - mine && first < upto) {
    uint32_t at = upto - mine;
    for (uint32_t s = s0; s < s1; ++s) {
      const uint32_t n = max((slot_reach(c, s) + kTile - 1) / kTile, 1) * per_tile;
      if (first < at + n) {
        s_at[0] = s, s_at[1] = at;
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  uint32_t slot = s_at[0], slot_at = s_at[1];

  for (uint32_t u = first; u < last;) {
    const int len = slot_length(c, slot), reach = slot_reach(c, slot);
    const uint32_t tiles = max((reach + kTile - 1) / kTile, 1);
    if (u >= slot_at + tiles * per_tile) {
      slot_at += tiles * per_tile;
      ++slot;
      continue;
    }
    const uint32_t seg = (u - slot_at) / tiles, tile_lo = (u - slot_at) % tiles;
    const uint32_t kvh = seg / P.row_tiles, rt = seg % P.row_tiles;
    const uint32_t tile_hi = min(tiles, tile_lo + (last - u));
    const int count = P.counts ? min(max(P.counts[slot], 0), int(P.rows)) : int(P.rows);

    Attn<T, D, NT> A;
    A.load_q(P, slot, kvh, rt, len, count, lane);
    BlockRegs<D> cur, next;
    int token = int(tile_lo) * kTile + warp * int(kBlock);
    const int end = min(reach, int(tile_hi) * kTile);
    cur.load(token < end ? block_of(c, slot, token, kvh, D) : nullptr, lane);
    for (int k = 1; token < end; token += kTile, ++k) {
      const int then = token + kTile;
      next.load(then < end ? block_of(c, slot, then, kvh, D) : nullptr, lane);
      if (cur.there) A.block(cur, token, lane);
      if (k % kCentre == 0) A.centre();
      cur = next;
    }
    A.centre();
    A.park(so[warp], sml[warp], lane);
    __syncthreads();

    // ---- join the warps; write the result, or this share's part of it
    const bool whole = tile_lo == 0 && tile_hi == tiles;
    const uint32_t seg_lo = slot_at + seg * tiles, seg_hi = seg_lo + tiles;
    const uint32_t c0 = seg_lo / quota, c1 = (seg_hi - 1) / quota;
    const size_t part = size_t(kRows) * (D + 2);
    float* mypart = P.partials + (size_t(blockIdx.x) * 2 + (tile_lo == 0 ? 1 : 0)) * part;
    auto put = [&](int r, int d, float val, float top, float sum) {
      const uint32_t rr = rt * kRows + r;
      const uint32_t row = rr / P.group, head = kvh * P.group + rr % P.group;
      if (row >= P.rows) return;
      const size_t at = (size_t(slot) * P.heads + head) * P.rows + row;
      static_cast<T*>(P.out)[at * D + d] = from_f<T>(sum == 0.f ? 0.f : val / sum);
      if (P.lse && d == 0)
        P.lse[at] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
    };
    for (int i = tid; i < kRows * D; i += kThreads) {
      const int r = i / D, d = i % D;
      float top = sml[0][2 * r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sml[w][2 * r]);
      float val = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        // a warp that saw nothing of the row has m = -inf, l = 0 and O = 0
        const float k = sml[w][2 * r] == -INFINITY ? 0.f : ex2(sml[w][2 * r] - top);
        if (k != 0.f) {
          val = fmaf(so[w][i], k, val);
          sum = fmaf(sml[w][2 * r + 1], k, sum);
        } else if (sml[w][2 * r + 1] != sml[w][2 * r + 1]) {
          val = sum = sml[w][2 * r + 1];  // NaN
        }
      }
      if (whole) {
        put(r, d, val, top, sum);
      } else {
        mypart[r * D + d] = val;
        if (d == 0) mypart[kRows * D + 2 * r] = top, mypart[kRows * D + 2 * r + 1] = sum;
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      if (tid == 0) s_ticket = atomicAdd(P.counters + c0, 1u);
      __syncthreads();
      if (s_ticket == c1 - c0) {
        __threadfence();
        for (int i = tid; i < kRows * D; i += kThreads) {
          const int r = i / D, d = i % D;
          float top = -INFINITY, val = 0.f, sum = 0.f;
          for (uint32_t k = c0; k <= c1; ++k) {
            const float* pp = P.partials + (size_t(k) * 2 + (k == c0 ? 1 : 0)) * part;
            const float pm = __ldcg(pp + kRows * D + 2 * r), pl = __ldcg(pp + kRows * D + 2 * r + 1);
            const float pv = __ldcg(pp + r * D + d);
            if (pl == 0.f) continue;  // saw nothing of the row
            const float to = fmaxf(top, pm);
            const float ka = top == -INFINITY ? 0.f : ex2(top - to);
            const float kb = pm == -INFINITY ? 1.f : ex2(pm - to);
            val = val * ka + pv * kb;
            sum = sum * ka + pl * kb;
            top = to;
          }
          put(r, d, val, top, sum);
        }
        if (tid == 0) P.counters[c0] = 0;
      }
    }
    __syncthreads();
    u += tile_hi - tile_lo;
  }
}

template <typename T, int D, int NT>
FelixCode launch(AttnParams& P, DeviceInfo* dev, void* workspace, size_t ws_bytes,
                 cudaStream_t stream) {
  static int per_sm[64];
  static PerDeviceOnce once;
  const int rc = once.run(dev->ordinal, [&] {
    return cudaOccupancyMaxActiveBlocksPerMultiprocessor(
               &per_sm[dev->ordinal], kv4_attn_kernel<T, D, NT>, kThreads, 0) == cudaSuccess ? 0 : -1;
  });
  if (rc != 0) return launch_error(cudaGetLastError(), "kv4_attention: occupancy");
  const uint32_t grid = uint32_t(dev->num_sms) * uint32_t(min(per_sm[dev->ordinal], 8));
  const size_t need = kWsCounterBytes + size_t(grid) * 2 * 8 * NT * (D + 2) * sizeof(float);
  if (workspace && ws_bytes < need)
    return api_error("kv4_attention: workspace smaller than felix_kv4_attention_workspace_size");
  void* ws = workspace ? workspace : library_workspace(dev, stream, need);
  if (!ws) return launch_error(cudaErrorMemoryAllocation, "kv4_attention: workspace");
  P.counters = static_cast<uint32_t*>(ws);
  P.partials = reinterpret_cast<float*>(static_cast<char*>(ws) + kWsCounterBytes);
  P.row_tiles = (P.rows * P.group + 8 * NT - 1) / (8 * NT);
  kv4_attn_kernel<T, D, NT><<<grid, kThreads, 0, stream>>>(P);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return launch_error(e, "kv4_attention");
  return FelixCode{FELIX_SUCCESS, cudaSuccess};
}

}  // namespace kv4

// At most 8 CTAs per SM: what a caller's workspace must hold on any device.
size_t kv4_attention_workspace_bytes(uint32_t head_dim, int num_sms) {
  return kWsCounterBytes + size_t(num_sms) * 8 * 2 * 8 * 2 * (head_dim + 2) * sizeof(float);
}

FelixCode kv4_attention_launch(const felix_kv4::CacheView& c, uint32_t head_dim, const void* q,
                               bool bf16, uint32_t heads, uint32_t rows, const int64_t* strides,
                               const int32_t* counts, float scale, void* out, float* lse,
                               void* workspace, size_t ws_bytes, cudaStream_t stream) {
  DeviceInfo* dev = current_device_info();
  if (!dev) return launch_error(cudaGetLastError(), "kv4_attention: no device");
  kv4::AttnParams P;
  P.c = c;
  P.q = q;
  P.qs_slot = strides[0], P.qs_head = strides[1], P.qs_row = strides[2];
  P.out = out;
  P.lse = lse;
  P.counts = counts;
  P.heads = heads;
  P.rows = rows;
  P.group = heads / c.kv_heads;
  P.scale_log2 = (scale > 0.f ? scale : 1.0f / sqrtf(float(head_dim))) * 1.4426950408889634f;
  const bool two = rows * P.group > 8;
#define KV4_GO(T, D)                                                              \
  return two ? kv4::launch<T, D, 2>(P, dev, workspace, ws_bytes, stream)          \
             : kv4::launch<T, D, 1>(P, dev, workspace, ws_bytes, stream)
  if (bf16) {
    if (head_dim == 128) KV4_GO(__nv_bfloat16, 128);
    KV4_GO(__nv_bfloat16, 64);
  }
  if (head_dim == 128) KV4_GO(__half, 128);
  KV4_GO(__half, 64);
#undef KV4_GO
}

}  // namespace felix_impl

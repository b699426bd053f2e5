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
// second product by an 8 x 8 transpose in the warp.
//
// Rounding. p_t scale_v is rounded to fp16's 11 bits, P_t, for the second product.
// Its exponent is taken out first (the running maximum is that of score + exponent
// of scale_v). The result is
//   (sum P (c - 8) + sum P base_v / scale_v) / sum P / scale_v,
// the mean of the held values under the weights P / scale_v: rounded weights in
// the numerator and the denominator, so that a row that one token rules has no
// error from them. P is rounded with fp32's exponents, so that a weight keeps its 11
// bits however far it is below the others. Only its copy for the product with (c - 8) goes
// through fp16, where what is 2^-20 of the largest P (2^6 or more) is subnormal and
// loses at most 2^-25: 2^-31 of the largest token's share, for each such token. (With
// the weights taken from that copy too, a token whose scale is 2^-30 of another's
// left the denominator, as if it were masked.) The log-sum-exp has its own sum of
// unrounded p. Sums and statistics are fp32.
//
// Measured: 96 slots of up to 12288 tokens, 8 heads of 128: 135 to 139 us for 585 MB
// (64 to 66 % of the card's copy rate; its loads alone take 100 us), 517 instructions a
// warp's step of 4352 bytes, 160 of them the masks and shifts of codes. Four slots of
// 131071 tokens, 40 rows a group, heads of 64: 317 us, 586 instructions a step and 24
// rows. One slot of 1037 tokens: 8.8 us in the kernel, 14.4 us a call.
//
// The mma.sync form is used, not tcgen05: the product has 8 useful columns (one
// group of heads), the codes reach the instruction from registers after one
// logic operation per pair, and the kernel waits for its own latencies (half of the
// issue slots, half of the ALU and a third of the matrix unit are used at three warps a
// scheduler), not for the matrix unit; tcgen05 would need the codes
// expanded to fp16 in shared or tensor memory, four times the bytes of the cache.
#include <algorithm>

#include "felix_internal.h"
#include "kv4_layout.cuh"
#include "sm100_ptx.cuh"

namespace felix_impl {
namespace kv4 {

using namespace felix_kv4;

constexpr int kStep = 2;                     // blocks that a warp takes at once
constexpr int kStepTokens = kStep * kBlock;  // 32: one per lane

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
  float* partials;                   // [CTA][2][8 NT][D + 3]
  unsigned* status;                  // watchdog word
  bool q_vec;                        // rows of q are 16-byte aligned
};

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d = a * b + c, c left as it is
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1,
                                         const float (&c)[4]) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]),
        "f"(c[3]));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 numbers in a register pair, one instruction for both: here always the
// two query rows 2t, 2t + 1 that a thread holds of a matrix instruction's result.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 un(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 add(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
// Rounded to 11 bits, whatever the exponent: TF32 has fp16's significand and fp32's
// exponents. (96 slots 137 us, 131071 x 40 rows 328; by Veltkamp's splitting 138 and
// 332. Weights from the fp16 copy, wrong below 2^-14, saved 5 % of the latter.)
__device__ __forceinline__ F2 round11(F2 a) {
  const float2 x = un(a);
  uint32_t r0, r1;
  asm("cvt.rn.tf32.f32 %0, %1;" : "=r"(r0) : "f"(x.x));
  asm("cvt.rn.tf32.f32 %0, %1;" : "=r"(r1) : "f"(x.y));
  return f2(__uint_as_float(r0), __uint_as_float(r1));
}

template <int W>
struct Words;  // W 32-bit words loaded as one vector from shared memory
template <>
struct Words<4> {
  uint32_t w[4];
  __device__ __forceinline__ void load(const unsigned char* p) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  }
};
template <>
struct Words<2> {
  uint32_t w[2];
  __device__ __forceinline__ void load(const unsigned char* p) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  }
};

// What a step's tokens bring to scores and sums, decoded once by one lane each.
// Each number stands twice, as the pair that F2 operations take.
struct alignas(16) Pair2 {
  F2 a, b;
};
struct alignas(16) TokenParams {
  Pair2 k[kStepTokens];  // scale_k; base_k - 8 scale_k
  Pair2 e[kStepTokens];  // exponent E of scale_v; 2^-E
  Pair2 v[kStepTokens];  // scale_v 2^-E; 1 / scale_v
  F2 b[kStepTokens];     // base_v / scale_v
};
__device__ __forceinline__ float2 k_params(uint32_t p) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
  return make_float2(f.x, fmaf(-8.f, f.x, f.y));
}
struct VParams {
  float e, inv, mant, rcp, base;
};
// A vector of scale 0 is its base, whatever its codes (8 where it was appended, 0 in
// a page that nobody has written). 2^-60 stands in for the scale: codes then add
// nothing that shows, and the exponent leaves the maximum to the others, whose P a
// likely token of zeros would otherwise push out of fp16's range.
__device__ __forceinline__ VParams v_params(uint32_t p) {
  float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
  if (f.x == 0.f) f.x = 0x1p-60f;
  // a NaN counts as fp16's largest exponent
  const int e = min(int(__float_as_uint(f.x) >> 23 & 255) - 127, 16);
  VParams r;
  r.e = float(e);
  r.inv = __int_as_float((127 - e) << 23);
  r.mant = f.x * r.inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.rcp) : "f"(f.x));
  r.base = f.y * r.rcp;
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

// The sums of one warp over its steps of a segment (slot, kv head, tile of rows).
template <typename T, int D, int NT>
struct Attn {
  static constexpr int kRows = 8 * NT;
  static constexpr int kW = D / 32;       // words of a lane's vector
  static constexpr int kLane = D / 8;     // its bytes
  uint32_t q[NT][2 * kW][2];              // operand registers of 8 query rows each
  // score = (raw * scale_k + qs * (base_k - 8 scale_k)) * f: raw sums are in units
  // of 2^-24 and of the row's power of two, and so is qs = sum(q), so that the
  // terms cancel before anything is rounded to a scale
  F2 f[NT], qs[NT];
  int lim[NT][2];                         // tokens that this thread's two rows see
  F2 o[NT][D / 16][2];                    // sums of p scale_v (c - 8); odd rows 16 times that
  float m[NT][2];                         // what exponents are relative to
  // sums of p, of P / scale_v and of P base_v / scale_v
  F2 l[NT], w[NT], b[NT];
  int low;                                // the smallest of lim

  // r0: the warp's first (row, head) pair of the segment's P.rows * P.group
  __device__ __forceinline__ void load_q(const AttnParams& P, uint32_t slot, uint32_t kvh,
                                         uint32_t r0, int len, int count, int lane) {
    const int g = lane >> 2, t = lane & 3;
    low = len;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint32_t r = r0 + 8 * n + g;
      const uint32_t row = r / P.group, head = kvh * P.group + r % P.group;
      const bool live = row < P.rows && int(row) < count;
      float v[D / 4];
      float top = 0.f, sum = 0.f;
      const T* src = static_cast<const T*>(P.q) + int64_t(slot) * P.qs_slot +
                     int64_t(head) * P.qs_head + int64_t(row) * P.qs_row + t * (D / 4);
      if (live && P.q_vec) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const uint4 w = reinterpret_cast<const uint4*>(src)[i];
          const T* x = reinterpret_cast<const T*>(&w);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[8 * i + j] = to_f<T>(x[j]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < D / 4; ++i) v[i] = live ? to_f<T>(src[i]) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < D / 4; ++i) top = fmaxf(top, fabsf(v[i]));
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
      float fc[2], qc[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int from = 4 * (2 * t + c);
        const float dn = __shfl_sync(~0u, down, from), sm = __shfl_sync(~0u, sum, from);
        fc[c] = P.scale_log2 * dn * 16777216.f;  // raw sums are of code * 2^-24
        qc[c] = sm * (1.f / 16777216.f);
        const uint32_t rr = r0 + 8 * n + 2 * t + c;
        const int rw = int(rr / P.group);
        lim[n][c] = (rw < int(P.rows) && rw < count) ? max(len - count + rw + 1, 0) : 0;
        m[n][c] = -INFINITY;
      }
      f[n] = f2(fc[0], fc[1]);
      qs[n] = f2(qc[0], qc[1]);
      l[n] = w[n] = b[n] = f2(0.f, 0.f);
      // rows past the last do not narrow the unmasked range
      const bool past = r0 + 8 * n + 2 * t >= P.rows * P.group;
      if (!past) low = min(low, min(lim[n][0], r0 + 8 * n + 2 * t + 1 < P.rows * P.group
                                                   ? lim[n][1] : lim[n][0]));
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) o[n][j][h] = f2(0.f, 0.f);
    }
    low = min(low, __shfl_xor_sync(~0u, low, 1));
    low = min(low, __shfl_xor_sync(~0u, low, 2));
  }

  // Scores of a step -> probabilities as operand registers `pt`, and the sums.
  // s[n][b][h]: token 8h + g of block b, rows 2t and 2t + 1. kMask: some of the
  // tokens are not there or not seen by every row.
  template <bool kMask>
  __device__ __forceinline__ void softmax(float (&s)[NT][kStep][4], const TokenParams& tp,
                                          uint32_t there, int token0, int g,
                                          uint32_t (&pt)[NT][kStep][2]) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float2 x[kStep][2];
      bool on[kStep][2][2];
      float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
      for (int k = 0; k < kStep; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = k * 16 + h * 8 + g;
          const Pair2 kp = tp.k[i];
          const F2 raw = f2(s[n][k][2 * h], s[n][k][2 * h + 1]);
          x[k][h] = un(fma(fma(raw, kp.a, mul(qs[n], kp.b)), f[n], tp.e[i].a));
          if (kMask) {
            const bool in = there >> k & 1;
            on[k][h][0] = in && token0 + i < lim[n][0];
            on[k][h][1] = in && token0 + i < lim[n][1];
            if (!on[k][h][0]) x[k][h].x = -INFINITY;
            if (!on[k][h][1]) x[k][h].y = -INFINITY;
          }
          t0 = fmaxf(t0, x[k][h].x);
          t1 = fmaxf(t1, x[k][h].y);
        }
      // Probabilities with the m at hand, while a vote says whether it holds (it mostly
      // does). 131071 x 40 rows 317 us against 329 by voting first, 96 slots 138 against
      // 139.
      float2 e[kStep][2];
      auto exponents = [&]() {
        const F2 minus = f2(-m[n][0], -m[n][1]);
#pragma unroll
        for (int k = 0; k < kStep; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 d = un(add(f2(x[k][h].x, x[k][h].y), minus));
            e[k][h] = make_float2(ex2(d.x), ex2(d.y));
          }
      };
      exponents();
      // Exponents are relative to m, 2^6 below a maximum that is only moved when a
      // score passes it by 2^8: P stays below 2^15.
      if (__any_sync(~0u, t0 > m[n][0] + 14.f || t1 > m[n][1] + 14.f)) {
        float keep[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float top = c ? t1 : t0;
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
          top = fmaxf(m[n][c], top - 6.f);
          keep[c] = top == -INFINITY ? 1.f : ex2(m[n][c] - top);
          m[n][c] = top;
        }
        const F2 kk = f2(keep[0], keep[1]);
        l[n] = mul(l[n], kk);
        w[n] = mul(w[n], kk);
        b[n] = mul(b[n], kk);
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) o[n][j][h] = mul(o[n][j][h], kk);
        exponents();
      }
#pragma unroll
      for (int k = 0; k < kStep; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = k * 16 + h * 8 + g;
          Pair2 v = tp.v[i];
          F2 inv = tp.e[i].b, base = tp.b[i];
          if (kMask) {  // a masked token's parameters may be anything
            auto seen = [&](F2 a) {
              const float2 y = un(a);
              return f2(on[k][h][0] ? y.x : 0.f, on[k][h][1] ? y.y : 0.f);
            };
            if (!on[k][h][0]) e[k][h].x = 0.f;
            if (!on[k][h][1]) e[k][h].y = 0.f;
            inv = seen(inv), base = seen(base), v.a = seen(v.a), v.b = seen(v.b);
          }
          const F2 ee = f2(e[k][h].x, e[k][h].y);
          l[n] = fma(ee, inv, l[n]);
          const F2 P = round11(mul(ee, v.a));
          const float2 pr = un(P);
          const __half2 ph = __floats2half2_rn(pr.x, pr.y);  // exact but below 2^-14
          w[n] = fma(P, v.b, w[n]);
          b[n] = fma(P, base, b[n]);
          pt[n][k][h] = transpose8x8(*reinterpret_cast<const uint32_t*>(&ph));
        }
    }
  }

  // One step: kStep blocks at `x`, of which those in `there` exist.
  __device__ __forceinline__ void step(const unsigned char* x, TokenParams& tp, uint32_t there,
                                       int token0, int lane) {
    constexpr uint32_t lo = 0x000f000fu, hi = 0x00f000f0u;
    constexpr int kB = int(block_bytes(D));
    const int g = lane >> 2;
#pragma unroll
    for (int i = lane; i < kStepTokens; i += 32) {
      const unsigned char* p = x + (i / 16) * kB;
      const float2 k = k_params(reinterpret_cast<const uint32_t*>(p + k_params_at(D))[i & 15]);
      const VParams v = v_params(reinterpret_cast<const uint32_t*>(p + v_params_at(D))[i & 15]);
      tp.k[i] = {f2(k.x, k.x), f2(k.y, k.y)};
      tp.e[i] = {f2(v.e, v.e), f2(v.inv, v.inv)};
      tp.v[i] = {f2(v.mant, v.mant), f2(v.rcp, v.rcp)};
      tp.b[i] = f2(v.base, v.base);
    }
    float s[NT][kStep][4];
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < kStep; ++b) {
      Words<kW> k0, k1;
      k0.load(x + b * kB + lane * kLane);
      k1.load(x + b * kB + 4 * D + lane * kLane);
      float s2[4];  // two chains where few others run beside them
#pragma unroll
      for (int w = 0; w < kW; ++w) {
        const uint32_t a = k0.w[w], c = k1.w[w], a8 = a >> 8, c8 = c >> 8;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (w == 0)
            mma16816(s[n][b], a & lo, c & lo, a & hi, c & hi, q[n][0][0], q[n][0][1], zero);
          else
            mma16816(s[n][b], a & lo, c & lo, a & hi, c & hi, q[n][2 * w][0], q[n][2 * w][1]);
          if (NT > 1)
            mma16816(s[n][b], a8 & lo, c8 & lo, a8 & hi, c8 & hi, q[n][2 * w + 1][0],
                     q[n][2 * w + 1][1]);
          else if (w == 0)
            mma16816(s2, a8 & lo, c8 & lo, a8 & hi, c8 & hi, q[n][1][0], q[n][1][1], zero);
          else
            mma16816(s2, a8 & lo, c8 & lo, a8 & hi, c8 & hi, q[n][2 * w + 1][0],
                     q[n][2 * w + 1][1]);
        }
      }
      if (NT == 1)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[0][b][c] += s2[c];
    }
    __syncwarp();  // tp is written
    uint32_t pt[NT][kStep][2];
    if (there == (1u << kStep) - 1 && token0 <= low - kStepTokens)
      softmax<false>(s, tp, there, token0, g, pt);
    else
      softmax<true>(s, tp, there, token0, g, pt);
    // -8 sum(p scale_v) of the step in the codes' unit, 16 times that for the odd
    // rows: where the second product starts, so that it sums to what is small.
    float start[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      constexpr uint32_t m8 = 0x80088008u, m128 = 0x80808080u;
      mma16816(start[n], m8, m128, m8, m128, pt[n][0][0], pt[n][0][1], zero);
#pragma unroll
      for (int b = 1; b < kStep; ++b)
        mma16816(start[n], m8, m128, m8, m128, pt[n][b][0], pt[n][b][1]);
    }
    Words<kW> v0[kStep], v1[kStep];
#pragma unroll
    for (int b = 0; b < kStep; ++b) {
      v0[b].load(x + b * kB + v_codes_at(D) + lane * kLane);
      v1[b].load(x + b * kB + v_codes_at(D) + 4 * D + lane * kLane);
    }
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      float r[NT][2][4];
#pragma unroll
      for (int b = 0; b < kStep; ++b) {
        const uint32_t a = v0[b].w[w], c = v1[b].w[w], a8 = a >> 8, c8 = c >> 8;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (b == 0) {
            mma16816(r[n][0], a & lo, a & hi, c & lo, c & hi, pt[n][b][0], pt[n][b][1], start[n]);
            mma16816(r[n][1], a8 & lo, a8 & hi, c8 & lo, c8 & hi, pt[n][b][0], pt[n][b][1],
                     start[n]);
          } else {
            mma16816(r[n][0], a & lo, a & hi, c & lo, c & hi, pt[n][b][0], pt[n][b][1]);
            mma16816(r[n][1], a8 & lo, a8 & hi, c8 & lo, c8 & hi, pt[n][b][0], pt[n][b][1]);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            o[n][2 * w + i][h] = add(o[n][2 * w + i][h], f2(r[n][i][2 * h], r[n][i][2 * h + 1]));
    }
    __syncwarp();  // the stage and tp are free
  }

  // Writes the warp's sums to shared memory: O [kRows][D] (base term included)
  // and (m, l, w) of each row.
  __device__ __forceinline__ void park(float* so, float* sml, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float2 ls = un(l[n]), ws = un(w[n]), bs = un(b[n]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float lc = c ? ls.y : ls.x, wc = c ? ws.y : ws.x, off = c ? bs.y : bs.x;
#pragma unroll
        for (int x = 4; x < 32; x *= 2) {
          lc += __shfl_xor_sync(~0u, lc, x);
          wc += __shfl_xor_sync(~0u, wc, x);
          off += __shfl_xor_sync(~0u, off, x);
        }
        const int r = 8 * n + 2 * t + c;
        if (g == 0) sml[3 * r] = m[n][c], sml[3 * r + 1] = lc, sml[3 * r + 2] = wc;
        constexpr float u = 16777216.f;
        float4* dst = reinterpret_cast<float4*>(so + r * D + g * (D / 8));
        auto at = [&](int j, int h) {
          const float2 v = un(o[n][j][h]);
          return c ? v.y : v.x;
        };
#pragma unroll
        for (int j = 0; j < kW; ++j)
          dst[j] = make_float4(fmaf(at(2 * j, 0), u, off), fmaf(at(2 * j, 1), u / 16, off),
                               fmaf(at(2 * j + 1, 0), u, off), fmaf(at(2 * j + 1, 1), u / 16, off));
      }
    }
  }
};

// A CTA: kCW consumer warps and one that fetches. The consumers are kRW groups
// of rows times kTW = kCW / kRW that share a group's tokens; a stage of the ring
// holds a step of each of the kTW.
template <int D, int NT, int kRW, int kCW>
struct Shape {
  static constexpr int kTW = kCW / kRW;
  static constexpr int kJoin = 32 * kCW;  // threads of the consumers
  // Eight consumers are two warpgroups, the warp that fetches is in a third, which
  // gives most of its registers to them.
  static constexpr int kThreads = kCW == 8 ? 384 : 160;
  static constexpr int kRows = 8 * NT;        // rows of a warp
  static constexpr int kTileRows = kRW * kRows;
  static constexpr int kBlocks = kTW * kStep;  // of a stage
  static constexpr int kStageBytes = kBlocks * int(block_bytes(D));
  // 50 KB of stages for a CTA of 4 consumers (three to an SM), 100 KB for one of 8
  // (one to an SM)
  static constexpr int kStages = (kCW == 4 ? 53000 : 100000) / kStageBytes;
};
// Registers of a CTA of 8 consumers: launched with 168 a thread (65536 / 384),
// then 40 for the fetching warpgroup and 232 for the others: 40 * 128 + 232 * 256 =
// 168 * 384. The host checks the launch count before the first launch.
constexpr int kRegsLaunch = 168, kRegsFetch = 40, kRegsSums = 232;
static_assert(kRegsFetch * 128 + kRegsSums * 256 <= kRegsLaunch * 384);

template <int D, int NT, int kRW, int kCW>
struct Smem {
  using H = Shape<D, NT, kRW, kCW>;
  alignas(128) unsigned char ring[H::kStages][H::kStageBytes];
  alignas(16) float o[kCW][H::kRows * D];
  TokenParams tp[kCW];
  uint64_t full[H::kStages], empty[H::kStages];
  uint32_t there[H::kStages];
  float ml[kCW][3 * H::kRows];  // (m, l, w) of each row
  uint32_t scan[H::kThreads / 32], at[2], ticket;
  int abort;
};

// A bounded wait of a whole warp. Lanes may give up at different times; what follows
// has warp-wide operations, so that all go on or none.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* abort_flag,
                                          unsigned* status) {
  return __all_sync(~0u, felix_sm100::mbar_wait(bar, parity, abort_flag, status,
                                                felix_sm100::kWdKv4Load));
}
// After a wait that gave up, copies may still be under way into this CTA's shared
// memory: they get time to land before it goes to another. (Any warp may be the last to
// leave: the one that fetches is mostly done by then.)
__device__ __forceinline__ void let_copies_land() {
  const uint64_t t0 = felix_sm100::globaltimer_ns();
  while (felix_sm100::globaltimer_ns() - t0 < 1000000ull) {
  }
}

// Units of a segment beyond its steps (`open` below): what opening and closing it
// costs (q, the join of the warps), about 12 steps. Without them a share of many
// short segments takes longest. Where there are few steps per CTA, the shares are
// kept even in steps instead; at least 1, so that an empty slot is in a share too.
constexpr uint32_t kMaxOpen = 12;

// A place in a CTA's share of the work: the part [lo, hi) of a segment's units,
// whose first `open` units hold no steps.
struct Place {
  uint32_t open_units;
  uint32_t slot, slot_at;  // slot, and the units before it
  uint32_t size;           // units of each of the slot's segments
  int len, reach;
  uint32_t kvh, rt, seg_at, lo, hi;
  __device__ __forceinline__ void read(const AttnParams& P) {
    len = slot_length(P.c, slot);
    reach = slot_reach(P.c, slot);
    size = open_units + (uint32_t(reach) + kStepTokens - 1) / kStepTokens;
  }
  // unit u, at or after the current slot's first
  __device__ __forceinline__ void open(const AttnParams& P, uint32_t u, uint32_t last) {
    const uint32_t per = P.c.kv_heads * P.row_tiles;
    while (u >= slot_at + size * per) {
      slot_at += size * per;
      ++slot;
      read(P);
    }
    const uint32_t seg = (u - slot_at) / size;
    kvh = seg / P.row_tiles;
    rt = seg - kvh * P.row_tiles;
    seg_at = slot_at + seg * size;
    lo = u - seg_at;
    hi = min(size, lo + (last - u));
  }
  __device__ __forceinline__ uint32_t end() const { return seg_at + hi; }
  __device__ __forceinline__ uint32_t first_step() const {
    return lo > open_units ? lo - open_units : 0;
  }
  __device__ __forceinline__ uint32_t end_step() const {
    return hi > open_units ? hi - open_units : 0;
  }
};

// Persistent grid. The work is a line of units (a segment's steps of 32 tokens and
// `open` for the segment itself, one after another), cut into equal shares, one
// per CTA, whatever the slots' lengths. The last warp looks pages up and fills the
// ring of stages with bulk copies, across segments; the others take their steps
// of each stage, and their registers hold sums only. A segment that lies in
// several shares is finished by the CTA that comes last to it, which joins the
// parts in a fixed order: the result does not depend on who is last.
template <typename T, int D, int NT, int kRW, int kCW>
__global__ void __launch_bounds__(kCW == 8 ? 384 : 160, kCW == 8 ? 1 : 3)
    kv4_attn_kernel(const AttnParams P) {
  using H = Shape<D, NT, kRW, kCW>;
  using S = Smem<D, NT, kRW, kCW>;
  constexpr int kRows = H::kRows, kTW = H::kTW, kThreads = H::kThreads;
  constexpr int kB = int(block_bytes(D));
  constexpr int kVec = H::kTileRows * D / 4, kWarpVec = kRows * D / 4;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  S& sm = *reinterpret_cast<S*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const CacheView& c = P.c;
  const uint32_t per_seg = c.kv_heads * P.row_tiles;

  // ---- this CTA's share: units before each thread's run of slots, then the slot
  const uint32_t run = (c.slots + kThreads - 1) / kThreads;
  const uint32_t s0 = min(tid * run, c.slots), s1 = min(s0 + run, c.slots);
  auto steps = [&](uint32_t s) {
    return (uint32_t(slot_reach(c, s)) + kStepTokens - 1) / kStepTokens * per_seg;
  };
  uint32_t mine = 0;
  for (uint32_t s = s0; s < s1; ++s) mine += steps(s);
  uint32_t upto = mine;
#pragma unroll
  for (int x = 1; x < 32; x *= 2) {
    const uint32_t v = __shfl_up_sync(~0u, upto, x);
    if (lane >= x) upto += v;
  }
  if (lane == 31) sm.scan[warp] = upto;
  if (tid == 0) {
    sm.abort = 0;
    for (int s = 0; s < H::kStages; ++s) {
      felix_sm100::mbar_init(&sm.full[s], 1);
      felix_sm100::mbar_init(&sm.empty[s], kCW);
    }
    felix_sm100::fence_mbar_init();
    felix_sm100::fence_proxy_async_smem();
  }
  __syncthreads();
  uint32_t total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) upto += sm.scan[w];
    total += sm.scan[w];
  }
  const uint32_t open = min(max(total / (4 * gridDim.x), 1u), kMaxOpen);
  mine += open * (s1 - s0) * per_seg;
  upto += open * s1 * per_seg;
  total += open * c.slots * per_seg;
  // at least a step for each warp: smaller parts cost more to join than they save
  // (the host keeps the total below 2^32; shares past it may lie beyond)
  const uint32_t quota = max(total / gridDim.x + (total % gridDim.x != 0), uint32_t(kTW));
  const uint32_t first = uint32_t(min(uint64_t(blockIdx.x) * quota, uint64_t(total)));
  const uint32_t last = first + min(quota, total - first);
  if (first >= last) return;
  if (first >= upto - mine && first < upto) {
    uint32_t at = upto - mine;
    for (uint32_t s = s0; s < s1; ++s) {
      const uint32_t n = steps(s) + open * per_seg;
      if (first < at + n) {
        sm.at[0] = s, sm.at[1] = at;
        break;
      }
      at += n;
    }
  }
  __syncthreads();

  Place use;
  use.open_units = open;
  use.slot = sm.at[0], use.slot_at = sm.at[1];
  use.read(P);
  use.open(P, first, last);
  int stage = 0;
  uint32_t parity = 0;
  auto advance = [&]() {
    if (++stage == H::kStages) stage = 0, parity ^= 1;
  };

  if (warp >= kCW) {  // ---- the warp that fetches: lane b has block b of a stage
    if constexpr (kCW == 8) felix_sm100::setmaxnreg_dec<kRegsFetch>();
    if (warp > kCW) return;
    const uint32_t blocks = 1u << (c.page_shift - 4);  // of a page and head
    uint32_t t = use.first_step(), end = use.end_step();
    bool more = true;
    int page = -1;
    uint32_t in_page = 0;
    auto look = [&]() {  // the next round's pages
      while (more && t >= end) {
        const uint32_t u = use.end();
        more = u < last;
        if (more) {
          use.open(P, u, last);
          t = use.first_step();
          end = use.end_step();
        }
      }
      if (!more) return;
      const uint32_t token = t * kStepTokens + lane * kBlock;
      page = -1;
      if (lane < H::kBlocks && t + lane / kStep < end && int(token) < use.reach) {
        page = c.table[size_t(use.slot) * c.width + (token >> c.page_shift)];
        in_page = use.kvh * blocks + ((token >> 4) & (blocks - 1));
      }
      t += kTW;
    };
    look();
    while (more) {
      const bool ok = page >= 0 && uint64_t(page) < c.num_pages;
      const unsigned char* src =
          c.pages + size_t(ok ? page : 0) * c.page_bytes + size_t(in_page) * kB;
      const uint32_t there = __ballot_sync(~0u, ok);
      look();  // the table is read while the stage is waited for
      if (!warp_wait(&sm.empty[stage], parity ^ 1, &sm.abort, P.status)) break;
      if (lane == 0) {
        sm.there[stage] = there;
        felix_sm100::mbar_arrive_expect_tx(&sm.full[stage], __popc(there) * kB);
      }
      __syncwarp();
      if (ok) felix_sm100::bulk_load_1d(&sm.ring[stage][lane * kB], src, kB, &sm.full[stage]);
      advance();
    }
    if (sm.abort) let_copies_land();
    return;
  }
  if constexpr (kCW == 8) felix_sm100::setmaxnreg_inc<kRegsSums>();

  const int rw = warp / kTW, tw = warp - rw * kTW;  // group of rows, place among its tokens
  bool gone = false;  // a wait gave up: the rest is passed over
  for (;;) {
    const uint32_t kvh = use.kvh, rt = use.rt;
    const int count = P.counts ? min(max(P.counts[use.slot], 0), int(P.rows)) : int(P.rows);
    Attn<T, D, NT> A;
    A.load_q(P, use.slot, kvh, rt * H::kTileRows + rw * kRows, use.len, count, lane);
    const uint32_t end = use.end_step();
    for (uint32_t t = use.first_step(); t < end && !gone; t += kTW) {
      if (!warp_wait(&sm.full[stage], parity, &sm.abort, P.status)) {
        gone = true;
        break;
      }
      const uint32_t there = sm.there[stage] >> (tw * kStep) & ((1u << kStep) - 1);
      if (there)
        A.step(sm.ring[stage] + tw * kStep * kB, sm.tp[warp], there, int(t + tw) * kStepTokens,
               lane);
      __syncwarp();
      if (lane == 0) felix_sm100::mbar_arrive(&sm.empty[stage]);
      advance();
    }
    A.park(sm.o[warp], sm.ml[warp], lane);
    felix_sm100::named_barrier_sync(1, H::kJoin);

    // ---- join the warps; write the result, or this share's part of it
    const bool whole = use.lo == 0 && use.hi == use.size;
    const uint32_t c0 = use.seg_at / quota, c1 = (use.seg_at + use.size - 1) / quota;
    constexpr size_t kPart = size_t(H::kTileRows) * (D + 3);
    float* mypart = P.partials + (size_t(blockIdx.x) * 2 + (use.lo == 0 ? 1 : 0)) * kPart;
    // Sums of a row: O is relative to `top`, as l and w are.
    struct Row {
      float top, l, w;
    };
    auto put = [&](int i, float4 v, Row s) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      const uint32_t rr = rt * H::kTileRows + r;
      const uint32_t row = rr / P.group, head = kvh * P.group + rr % P.group;
      if (row >= P.rows) return;
      const size_t at = (size_t(use.slot) * P.heads + head) * P.rows + row;
      const float k = s.l == 0.f ? 0.f : 1.f / s.w;  // l = 0: the row saw nothing, O is 0
      const T x[4] = {from_f<T>(v.x * k), from_f<T>(v.y * k), from_f<T>(v.z * k),
                      from_f<T>(v.w * k)};
      *reinterpret_cast<uint2*>(static_cast<T*>(P.out) + at * D + d) =
          *reinterpret_cast<const uint2*>(x);
      if (P.lse && d == 0)
        P.lse[at] = s.l == 0.f ? -INFINITY : (s.top + log2f(s.l)) * 0.6931471805599453f;
    };
    // O vector and statistics of a row from `n` sources as one: source(k, &m, &l, &w)
    // gives its vector. A source that saw nothing of the row has l = 0 and O = 0;
    // m = -inf with l not 0 is one that saw NaN only.
    auto joined = [&](int n, auto&& stats, auto&& vec, Row* s) {
      s->top = -INFINITY;
#pragma unroll
      for (int k = 0; k < n; ++k) s->top = fmaxf(s->top, stats(k)[0]);
      s->l = s->w = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < n; ++k) {
        const float m = stats(k)[0], l = stats(k)[1];
        if (l == 0.f) continue;
        const float to = m == -INFINITY ? 1.f : ex2(m - s->top);
        const float4 x = vec(k);
        v.x = fmaf(x.x, to, v.x), v.y = fmaf(x.y, to, v.y);
        v.z = fmaf(x.z, to, v.z), v.w = fmaf(x.w, to, v.w);
        s->l = fmaf(l, to, s->l);
        s->w = fmaf(stats(k)[2], to, s->w);
      }
      return v;
    };
    for (int i = tid; i < kVec; i += H::kJoin) {
      const int group = i / kWarpVec, j = i % kWarpVec;  // the rows' warps, place in them
      Row s;
      const float4 v = joined(
          kTW, [&](int k) { return sm.ml[group * kTW + k] + 3 * (j / (D / 4)); },
          [&](int k) { return reinterpret_cast<const float4*>(sm.o[group * kTW + k])[j]; }, &s);
      if (whole) {
        put(i, v, s);
      } else {
        reinterpret_cast<float4*>(mypart)[i] = v;
        if (i % (D / 4) == 0) {
          float* x = mypart + H::kTileRows * D + 3 * (i / (D / 4));
          x[0] = s.top, x[1] = s.l, x[2] = s.w;
        }
      }
    }
    if (!whole) {
      felix_sm100::named_barrier_sync(1, H::kJoin);
      if (tid == 0) {
        __threadfence();  // the barrier has ordered the CTA's stores before it
        sm.ticket = atomicAdd(P.counters + c0, 1u);
        __threadfence();
      }
      felix_sm100::named_barrier_sync(1, H::kJoin);
      if (sm.ticket == c1 - c0) {
        auto part_at = [&](uint32_t k) {
          return P.partials + (size_t(k) * 2 + (k == c0 ? 1 : 0)) * kPart;
        };
        // a thread joins two vectors of O over all parts, kParts parts' loads at a time
        constexpr int kTwo = kVec / 2, kParts = NT == 1 ? 6 : 4;
        for (int i = tid; i < kTwo; i += H::kJoin) {
          Row s[2] = {{-INFINITY, 0.f, 0.f}, {-INFINITY, 0.f, 0.f}};
          float4 v[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
          for (uint32_t k0 = c0; k0 <= c1; k0 += kParts) {
            float m[2][kParts], l[2][kParts], w[2][kParts];
            float4 x[2][kParts];
#pragma unroll
            for (int j = 0; j < kParts; ++j) {
              const float* p = part_at(min(k0 + j, c1));
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const float* q = p + H::kTileRows * D + 3 * ((i + y * kTwo) / (D / 4));
                m[y][j] = __ldcg(q), l[y][j] = __ldcg(q + 1), w[y][j] = __ldcg(q + 2);
                x[y][j] = __ldcg(reinterpret_cast<const float4*>(p) + i + y * kTwo);
                if (k0 + j > c1) l[y][j] = 0.f, m[y][j] = -INFINITY;
              }
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              float top = s[y].top;
#pragma unroll
              for (int j = 0; j < kParts; ++j) top = fmaxf(top, m[y][j]);
              const float keep = s[y].top == -INFINITY ? 1.f : ex2(s[y].top - top);
              v[y].x *= keep, v[y].y *= keep, v[y].z *= keep, v[y].w *= keep;
              s[y] = {top, s[y].l * keep, s[y].w * keep};
#pragma unroll
              for (int j = 0; j < kParts; ++j) {
                if (l[y][j] == 0.f) continue;
                const float to = m[y][j] == -INFINITY ? 1.f : ex2(m[y][j] - top);
                v[y].x = fmaf(x[y][j].x, to, v[y].x), v[y].y = fmaf(x[y][j].y, to, v[y].y);
                v[y].z = fmaf(x[y][j].z, to, v[y].z), v[y].w = fmaf(x[y][j].w, to, v[y].w);
                s[y].l = fmaf(l[y][j], to, s[y].l);
                s[y].w = fmaf(w[y][j], to, s[y].w);
              }
            }
          }
          put(i, v[0], s[0]);
          put(i + kTwo, v[1], s[1]);
        }
        if (tid == 0) P.counters[c0] = 0;
      }
    }
    felix_sm100::named_barrier_sync(1, H::kJoin);
    const uint32_t u = use.end();
    if (u >= last) break;
    use.open(P, u, last);
  }
  if (gone) let_copies_land();
}

// Scratch: counters, then two parts per CTA. A grid has at most three CTAs of 8
// rows per SM, or one of up to max_rows(D).
constexpr size_t part_bytes(uint32_t ctas, int rows, int D) {
  return size_t(ctas) * 2 * rows * (D + 3) * sizeof(float);
}
// Tiles of 8 query rows that a warp keeps in registers.
constexpr int max_nt(int D) { return D == 64 ? 3 : 2; }
constexpr int max_rows(int D) { return 4 * 8 * max_nt(D); }

template <typename T, int D, int NT, int kRW, int kCW>
FelixCode launch(AttnParams& P, DeviceInfo* dev, void* workspace, size_t ws_bytes,
                 cudaStream_t stream) {
  using H = Shape<D, NT, kRW, kCW>;
  static int per_sm[64];
  static PerDeviceOnce once;
  constexpr int smem = int(sizeof(Smem<D, NT, kRW, kCW>));
  auto* kernel = kv4_attn_kernel<T, D, NT, kRW, kCW>;
  const int rc = once.run(dev->ordinal, [&] {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) !=
        cudaSuccess)
      return -1;
    cudaFuncAttributes attr;
    if (cudaFuncGetAttributes(&attr, kernel) != cudaSuccess) return -1;
    if (kCW == 8 && attr.numRegs != kRegsLaunch) return -2;  // the split would wait for ever
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, H::kThreads, smem) !=
            cudaSuccess || n < 1)
      return -1;
    per_sm[dev->ordinal] = kCW == 4 ? (n < 3 ? n : 3) : 1;
    return 0;
  });
  if (rc == -2) return api_error("kv4_attention: built with another register count than 168");
  if (rc != 0) return launch_error(cudaGetLastError(), "kv4_attention: occupancy");
  const uint32_t grid = uint32_t(dev->num_sms) * uint32_t(per_sm[dev->ordinal]);
  const size_t need = kWsCounterBytes + part_bytes(grid, H::kTileRows, D);
  if (workspace && ws_bytes < need)
    return api_error("kv4_attention: workspace smaller than felix_kv4_attention_workspace_size");
  // the library's own is asked for at its largest: growing waits for the stream
  const size_t most = kv4_attention_workspace_bytes(128, dev->num_sms);
  Workspace scratch;  // until the launch
  if (!workspace) scratch = library_workspace(dev, stream, most);
  void* ws = workspace ? workspace : scratch.ptr;
  if (!ws) return launch_error(cudaErrorMemoryAllocation, "kv4_attention: workspace");
  P.counters = static_cast<uint32_t*>(ws);
  P.partials = reinterpret_cast<float*>(static_cast<char*>(ws) + kWsCounterBytes);
  P.row_tiles = (P.rows * P.group + H::kTileRows - 1) / H::kTileRows;
  const uint64_t steps = (uint64_t(P.c.width) << P.c.page_shift) / kStepTokens + 1 + kMaxOpen;
  if (double(P.c.slots) * P.c.kv_heads * P.row_tiles * double(steps) >= 4294967296.0)
    return api_error("kv4_attention: slots x heads x rows x tokens past 2^32 steps in one call");
  kernel<<<grid, H::kThreads, smem, stream>>>(P);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return launch_error(e, "kv4_attention");
  return FelixCode{FELIX_SUCCESS, cudaSuccess};
}

// Up to 8 rows: four consumers that share all tokens, three CTAs to an SM. More:
// eight, in as many groups of rows as registers ask for, so that the cache is read
// once for up to max_rows(D) rows; beyond that each further tile reads it again.
template <typename T, int D>
FelixCode launch_rows(AttnParams& P, DeviceInfo* dev, void* ws, size_t n, cudaStream_t stream) {
  const uint32_t eights = (P.rows * P.group + 7) / 8, most = max_nt(D);
  if (eights == 1) return launch<T, D, 1, 1, 4>(P, dev, ws, n, stream);
  const uint32_t tiles = (eights + 4 * most - 1) / (4 * most);
  const uint32_t per_tile = (eights + tiles - 1) / tiles;
  const uint32_t rw = per_tile <= most ? 1 : per_tile <= 2 * most ? 2 : 4;
  const bool three = D == 64 && per_tile > 2 * rw;
  if constexpr (D == 64) {
    if (three) {
      if (rw == 1) return launch<T, D, 3, 1, 8>(P, dev, ws, n, stream);
      if (rw == 2) return launch<T, D, 3, 2, 8>(P, dev, ws, n, stream);
      return launch<T, D, 3, 4, 8>(P, dev, ws, n, stream);
    }
  }
  if (rw == 1) return launch<T, D, 2, 1, 8>(P, dev, ws, n, stream);
  if (rw == 2) return launch<T, D, 2, 2, 8>(P, dev, ws, n, stream);
  return launch<T, D, 2, 4, 8>(P, dev, ws, n, stream);
}

}  // namespace kv4

size_t kv4_attention_workspace_bytes(uint32_t head_dim, int num_sms) {
  const uint32_t sms = uint32_t(num_sms);
  const int D = int(head_dim);
  return kWsCounterBytes + std::max(kv4::part_bytes(3 * sms, 8, D),
                                    kv4::part_bytes(sms, kv4::max_rows(D), D));
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
  P.status = dev->status_word;
  P.q_vec = ((reinterpret_cast<uintptr_t>(q) | uintptr_t(strides[0] * 2) |
              uintptr_t(strides[1] * 2) | uintptr_t(strides[2] * 2)) & 15) == 0;
  if (bf16) {
    if (head_dim == 128)
      return kv4::launch_rows<__nv_bfloat16, 128>(P, dev, workspace, ws_bytes, stream);
    return kv4::launch_rows<__nv_bfloat16, 64>(P, dev, workspace, ws_bytes, stream);
  }
  if (head_dim == 128) return kv4::launch_rows<__half, 128>(P, dev, workspace, ws_bytes, stream);
  return kv4::launch_rows<__half, 64>(P, dev, workspace, ws_bytes, stream);
}

}  // namespace felix_impl

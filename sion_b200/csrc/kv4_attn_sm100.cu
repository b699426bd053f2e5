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
//
// The mma.sync form is used, not tcgen05: the product has 8 useful columns (one
// group of heads), the codes reach the instruction from registers after one
// logic operation per pair, and the kernel is bound by reading the cache and by
// those logic operations, not by the matrix unit; tcgen05 would need the codes
// expanded to fp16 in shared or tensor memory, four times the bytes of the cache.
#include "felix_internal.h"
#include "kv4_layout.cuh"
#include "sm100_ptx.cuh"

namespace felix_impl {
namespace kv4 {

using namespace felix_kv4;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
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
  float* partials;                   // [CTA][2][8 NT][D + 2]
  unsigned* status;                  // watchdog word
  bool q_vec;                        // rows of q are 16-byte aligned
};

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d = a * b + c, c left as it is
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1,
                                         const float (&c)[4]) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]),
        "f"(c[3]));
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
  Pair2 v[kStepTokens];  // scale_v 2^-E; base_v 2^-E
};
__device__ __forceinline__ float2 k_params(uint32_t p) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
  return make_float2(f.x, fmaf(-8.f, f.x, f.y));
}
// E is the exponent of the smallest normal where scale_v is subnormal or zero.
__device__ __forceinline__ float4 v_params(uint32_t p) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
  const int e = max(int((p >> 10) & 31u), 1) - 15;
  const float inv = __int_as_float((127 - e) << 23);
  return make_float4(float(e), inv, f.x * inv, f.y * inv);
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
  float m[NT][2];                         // running maximum
  F2 l[NT], b_[NT];                       // sum of p, sum of p base_v
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
        const uint32_t rr = rt * kRows + 8 * n + 2 * t + c;
        const int rw = int(rr / P.group);
        lim[n][c] = (rw < int(P.rows) && rw < count) ? max(len - count + rw + 1, 0) : 0;
        m[n][c] = -INFINITY;
      }
      f[n] = f2(fc[0], fc[1]);
      qs[n] = f2(qc[0], qc[1]);
      l[n] = b_[n] = f2(0.f, 0.f);
      // rows past the last do not narrow the unmasked range
      const bool past = rt * kRows + 8 * n + 2 * t >= P.rows * P.group;
      if (!past) low = min(low, min(lim[n][0], rt * kRows + 8 * n + 2 * t + 1 < P.rows * P.group
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
      for (int b = 0; b < kStep; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = b * 16 + h * 8 + g;
          const Pair2 k = tp.k[i];
          const F2 raw = f2(s[n][b][2 * h], s[n][b][2 * h + 1]);
          x[b][h] = un(fma(fma(raw, k.a, mul(qs[n], k.b)), f[n], tp.e[i].a));
          if (kMask) {
            const bool in = there >> b & 1;
            on[b][h][0] = in && token0 + i < lim[n][0];
            on[b][h][1] = in && token0 + i < lim[n][1];
            if (!on[b][h][0]) x[b][h].x = -INFINITY;
            if (!on[b][h][1]) x[b][h].y = -INFINITY;
          }
          t0 = fmaxf(t0, x[b][h].x);
          t1 = fmaxf(t1, x[b][h].y);
        }
      // The sums are kept relative to a maximum that is only moved when a score
      // passes it by 2^8: probabilities stay below 2^9 and fp16 holds them.
      if (__any_sync(~0u, t0 > m[n][0] + 8.f || t1 > m[n][1] + 8.f)) {
        float keep[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float top = fmaxf(m[n][c], c ? t1 : t0);
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
          keep[c] = top == -INFINITY ? 1.f : ex2(m[n][c] - top);
          m[n][c] = top;
        }
        const F2 kk = f2(keep[0], keep[1]);
        l[n] = mul(l[n], kk);
        b_[n] = mul(b_[n], kk);
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) o[n][j][h] = mul(o[n][j][h], kk);
      }
      const F2 minus = f2(-m[n][0], -m[n][1]);
#pragma unroll
      for (int b = 0; b < kStep; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = b * 16 + h * 8 + g;
          const float2 d = un(add(f2(x[b][h].x, x[b][h].y), minus));
          float2 e = make_float2(ex2(d.x), ex2(d.y));
          Pair2 v = tp.v[i];
          F2 inv = tp.e[i].b;
          if (kMask) {  // a masked token's parameters may be anything
            if (!on[b][h][0]) e.x = 0.f;
            if (!on[b][h][1]) e.y = 0.f;
            const float2 a = un(v.a), w = un(v.b), u = un(inv);
            v.a = f2(on[b][h][0] ? a.x : 0.f, on[b][h][1] ? a.y : 0.f);
            v.b = f2(on[b][h][0] ? w.x : 0.f, on[b][h][1] ? w.y : 0.f);
            inv = f2(on[b][h][0] ? u.x : 0.f, on[b][h][1] ? u.y : 0.f);
          }
          const F2 ee = f2(e.x, e.y);
          l[n] = fma(ee, inv, l[n]);
          b_[n] = fma(ee, v.b, b_[n]);
          const float2 p = un(mul(ee, v.a));
          pt[n][b][h] = transpose8x8(felix_sm100::pack_half2(p.x, p.y));
        }
    }
  }

  // One step: kStep blocks at `x`, of which those in `there` exist.
  __device__ __forceinline__ void step(const unsigned char* x, TokenParams& tp, uint32_t there,
                                       int token0, int lane) {
    constexpr uint32_t lo = 0x000f000fu, hi = 0x00f000f0u;
    constexpr int kB = int(block_bytes(D));
    const int g = lane >> 2;
    {
      const unsigned char* p = x + (lane / 16) * kB;
      const float2 k = k_params(reinterpret_cast<const uint32_t*>(p + k_params_at(D))[lane & 15]);
      const float4 v = v_params(reinterpret_cast<const uint32_t*>(p + v_params_at(D))[lane & 15]);
      tp.k[lane] = {f2(k.x, k.x), f2(k.y, k.y)};
      tp.e[lane] = {f2(v.x, v.x), f2(v.y, v.y)};
      tp.v[lane] = {f2(v.z, v.z), f2(v.w, v.w)};
    }
    __syncwarp();
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
    uint32_t pt[NT][kStep][2];
    if (there == (1u << kStep) - 1 && token0 + kStepTokens <= low)
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
  // and (m, l) of each row.
  __device__ __forceinline__ void park(float* so, float* sml, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float2 ls = un(l[n]), bs = un(b_[n]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float lc = c ? ls.y : ls.x, off = c ? bs.y : bs.x;
#pragma unroll
        for (int x = 4; x < 32; x *= 2) {
          lc += __shfl_xor_sync(~0u, lc, x);
          off += __shfl_xor_sync(~0u, off, x);
        }
        const int r = 8 * n + 2 * t + c;
        if (g == 0) sml[2 * r] = m[n][c], sml[2 * r + 1] = lc;
        constexpr float u = 16777216.f;
        float4* dst = reinterpret_cast<float4*>(so + r * D + g * (D / 8));
        auto at = [&](int j, int h) {
          const float2 v = un(o[n][j][h]);
          return c ? v.y : v.x;
        };
#pragma unroll
        for (int w = 0; w < kW; ++w)
          dst[w] = make_float4(fmaf(at(2 * w, 0), u, off), fmaf(at(2 * w, 1), u / 16, off),
                               fmaf(at(2 * w + 1, 0), u, off), fmaf(at(2 * w + 1, 1), u / 16, off));
      }
    }
  }
};

template <int D, int NT>
struct Smem {
  // stages of kStep blocks per warp: 37 to 52 KB of cache are under way per CTA, about
  // 150 KB per SM
  static constexpr int kStages = D == 128 ? 3 : 4;
  static constexpr int kRows = 8 * NT;
  alignas(128) unsigned char ring[kWarps][kStages][kStep * block_bytes(D)];
  alignas(16) float o[kWarps][kRows * D];
  TokenParams tp[kWarps];
  uint64_t full[kWarps][kStages];
  uint32_t there[kWarps][kStages];
  float ml[kWarps][2 * kRows];
  uint32_t scan[kWarps], at[2], ticket;
  int abort;
};

// Units of a segment beyond its steps: what opening and closing it costs (q, the
// join of the warps). Without them a share of many short segments takes longest.
constexpr uint32_t kOpen = 12;

// A place in a CTA's share of the work: the part [lo, hi) of a segment's units,
// whose first kOpen units hold no steps.
struct Place {
  uint32_t slot, slot_at;  // slot, and the units before it
  uint32_t size;           // units of each of the slot's segments
  int len, reach;
  uint32_t kvh, rt, seg_at, lo, hi;
  __device__ __forceinline__ void read(const AttnParams& P) {
    len = slot_length(P.c, slot);
    reach = slot_reach(P.c, slot);
    size = kOpen + (reach + kStepTokens - 1) / kStepTokens;
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
  __device__ __forceinline__ uint32_t first_step() const { return lo > kOpen ? lo - kOpen : 0; }
  __device__ __forceinline__ uint32_t end_step() const { return hi > kOpen ? hi - kOpen : 0; }
};

// Persistent grid. The work is a line of units (a segment's steps of 32 tokens and
// kOpen for the segment itself, one after another), cut into equal shares, one
// per CTA, whatever the slots' lengths; the warps of a CTA take its steps in turn.
// Each warp has a ring of stages of its own in shared memory, filled by bulk
// copies that it issues itself a few steps ahead, across segments: no barrier in
// the loop, and the registers hold sums only. A segment that lies in several
// shares is finished by the CTA that comes last to it, which joins the parts in a
// fixed order: the result does not depend on who is last.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads) kv4_attn_kernel(const AttnParams P) {
  constexpr int kRows = 8 * NT, kB = int(block_bytes(D)), kVec = kRows * D / 4;
  using S = Smem<D, NT>;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  S& sm = *reinterpret_cast<S*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const CacheView& c = P.c;
  const uint32_t per_seg = c.kv_heads * P.row_tiles;

  // ---- this CTA's share: units before each thread's run of slots, then the slot
  const uint32_t run = (c.slots + kThreads - 1) / kThreads;
  const uint32_t s0 = min(tid * run, c.slots), s1 = min(s0 + run, c.slots);
  auto units = [&](uint32_t s) {
    return (kOpen + uint32_t(slot_reach(c, s) + kStepTokens - 1) / kStepTokens) * per_seg;
  };
  uint32_t mine = 0;
  for (uint32_t s = s0; s < s1; ++s) mine += units(s);
  uint32_t upto = mine;
#pragma unroll
  for (int x = 1; x < 32; x *= 2) {
    const uint32_t v = __shfl_up_sync(~0u, upto, x);
    if (lane >= x) upto += v;
  }
  if (lane == 31) sm.scan[warp] = upto;
  if (tid == 0) sm.abort = 0;
  if (lane < S::kStages) felix_sm100::mbar_init(&sm.full[warp][lane], 1);
  felix_sm100::fence_mbar_init();
  felix_sm100::fence_proxy_async_smem();
  __syncthreads();
  uint32_t total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) upto += sm.scan[w];
    total += sm.scan[w];
  }
  // at least a segment's opening and one step for each warp: smaller parts cost
  // more to join than they save
  const uint32_t quota = max((total + gridDim.x - 1) / gridDim.x, kOpen + kWarps);
  const uint32_t first = min(blockIdx.x * quota, total), last = min(first + quota, total);
  if (first >= last) return;
  if (first >= upto - mine && first < upto) {
    uint32_t at = upto - mine;
    for (uint32_t s = s0; s < s1; ++s) {
      const uint32_t n = units(s);
      if (first < at + n) {
        sm.at[0] = s, sm.at[1] = at;
        break;
      }
      at += n;
    }
  }
  __syncthreads();

  Place use, get;  // the part being summed, and the one whose steps are being fetched
  use.slot = sm.at[0], use.slot_at = sm.at[1];
  use.read(P);
  use.open(P, first, last);
  get = use;
  uint32_t get_t = get.first_step() + warp, get_end = get.end_step();
  bool more = true;
  const uint32_t blocks = 1u << (c.page_shift - 4);  // of a page and head
  // the next step to fetch: lane b looks up the page of its block b
  int page = -1;
  uint32_t in_page = 0;
  auto look = [&]() {
    while (more && get_t >= get_end) {
      const uint32_t u = get.end();
      more = u < last;
      if (more) {
        get.open(P, u, last);
        get_t = get.first_step() + warp;
        get_end = get.end_step();
      }
    }
    if (!more) return;
    const uint32_t token = get_t * kStepTokens + lane * kBlock;
    page = -1;
    if (lane < kStep && int(token) < get.reach) {
      page = c.table[size_t(get.slot) * c.width + (token >> c.page_shift)];
      in_page = get.kvh * blocks + ((token >> 4) & (blocks - 1));
    }
    get_t += kWarps;
  };
  auto fetch = [&](int stage) {  // issues the step that look() found
    if (!more) return;
    const bool ok = page >= 0 && uint64_t(page) < c.num_pages;
    const uint32_t there = __ballot_sync(~0u, ok);
    if (lane == 0) {
      sm.there[warp][stage] = there;
      felix_sm100::mbar_arrive_expect_tx(&sm.full[warp][stage], __popc(there) * kB);
    }
    __syncwarp();
    if (ok)
      felix_sm100::bulk_load_1d(&sm.ring[warp][stage][lane * kB],
                                c.pages + size_t(page) * c.page_bytes + size_t(in_page) * kB, kB,
                                &sm.full[warp][stage]);
  };
  for (int s = 0; s < S::kStages; ++s) {
    look();
    fetch(s);
  }
  look();

  int stage = 0;
  uint32_t parity = 0;
  for (;;) {
    const uint32_t kvh = use.kvh, rt = use.rt;
    const int count =
        P.counts ? min(max(P.counts[use.slot], 0), int(P.rows)) : int(P.rows);
    Attn<T, D, NT> A;
    A.load_q(P, use.slot, kvh, rt, use.len, count, lane);
    for (uint32_t t = use.first_step() + warp; t < use.end_step(); t += kWarps) {
      if (felix_sm100::mbar_wait(&sm.full[warp][stage], parity, &sm.abort, P.status,
                                 felix_sm100::kWdKv4Load)) {
        const uint32_t there = sm.there[warp][stage];
        if (there) A.step(sm.ring[warp][stage], sm.tp[warp], there, int(t) * kStepTokens, lane);
      }
      __syncwarp();
      fetch(stage);
      look();
      if (++stage == S::kStages) stage = 0, parity ^= 1;
    }
    A.park(sm.o[warp], sm.ml[warp], lane);
    __syncthreads();

    // ---- join the warps; write the result, or this share's part of it
    const bool whole = use.lo == 0 && use.hi == use.size;
    const uint32_t c0 = use.seg_at / quota, c1 = (use.seg_at + use.size - 1) / quota;
    constexpr size_t kPart = size_t(kRows) * (D + 2);
    float* mypart = P.partials + (size_t(blockIdx.x) * 2 + (use.lo == 0 ? 1 : 0)) * kPart;
    auto put = [&](int r, int d, float4 v, float top, float sum) {
      const uint32_t rr = rt * kRows + r;
      const uint32_t row = rr / P.group, head = kvh * P.group + rr % P.group;
      if (row >= P.rows) return;
      const size_t at = (size_t(use.slot) * P.heads + head) * P.rows + row;
      const float k = sum == 0.f ? 0.f : 1.f / sum;
      T x[4] = {from_f<T>(sum == 0.f ? 0.f : v.x * k), from_f<T>(sum == 0.f ? 0.f : v.y * k),
                from_f<T>(sum == 0.f ? 0.f : v.z * k), from_f<T>(sum == 0.f ? 0.f : v.w * k)};
      *reinterpret_cast<uint2*>(static_cast<T*>(P.out) + at * D + d) =
          *reinterpret_cast<const uint2*>(x);
      if (P.lse && d == 0)
        P.lse[at] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
    };
    for (int i = tid; i < kVec; i += kThreads) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      float top = sm.ml[0][2 * r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sm.ml[w][2 * r]);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        // a warp that saw nothing of the row has l = 0 and O = 0; m = -inf with l
        // not 0 is a warp that saw NaN only
        const float wl = sm.ml[w][2 * r + 1], wm = sm.ml[w][2 * r];
        if (wl == 0.f) continue;
        const float k = wm == -INFINITY ? 1.f : ex2(wm - top);
        const float4 x = reinterpret_cast<const float4*>(sm.o[w])[i];
        v.x = fmaf(x.x, k, v.x), v.y = fmaf(x.y, k, v.y);
        v.z = fmaf(x.z, k, v.z), v.w = fmaf(x.w, k, v.w);
        sum = fmaf(wl, k, sum);
      }
      if (whole) {
        put(r, d, v, top, sum);
      } else {
        reinterpret_cast<float4*>(mypart)[i] = v;
        if (d == 0) mypart[kRows * D + 2 * r] = top, mypart[kRows * D + 2 * r + 1] = sum;
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      if (tid == 0) sm.ticket = atomicAdd(P.counters + c0, 1u);
      __syncthreads();
      if (sm.ticket == c1 - c0) {
        __threadfence();
        // each warp joins every kWarps-th part, then the warps are joined: all
        // loads of a warp are independent of one another
        auto part_at = [&](uint32_t k) {
          return P.partials + (size_t(k) * 2 + (k == c0 ? 1 : 0)) * kPart;
        };
        for (int r = lane; r < kRows; r += 32) {
          float top = -INFINITY, sum = 0.f;
          for (uint32_t k = c0 + warp; k <= c1; k += kWarps)
            top = fmaxf(top, __ldcg(part_at(k) + kRows * D + 2 * r));
          for (uint32_t k = c0 + warp; k <= c1; k += kWarps) {
            const float pm = __ldcg(part_at(k) + kRows * D + 2 * r);
            const float pl = __ldcg(part_at(k) + kRows * D + 2 * r + 1);
            if (pl != 0.f) sum = fmaf(pl, pm == -INFINITY ? 1.f : ex2(pm - top), sum);
          }
          sm.ml[warp][2 * r] = top;
          sm.ml[warp][2 * r + 1] = sum;
        }
        __syncwarp();
        constexpr int kPer = kVec / 32;  // vectors of a lane
        for (int j0 = 0; j0 < kPer; j0 += 8) {
          float4 v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
          for (uint32_t k = c0 + warp; k <= c1; k += kWarps) {
            const float* pp = part_at(k);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (j0 + j >= kPer) break;
              const int i = (j0 + j) * 32 + lane, r = i / (D / 4);
              const float pm = __ldcg(pp + kRows * D + 2 * r), pl = __ldcg(pp + kRows * D + 2 * r + 1);
              const float4 x = __ldcg(reinterpret_cast<const float4*>(pp) + i);
              const float w = pl == 0.f ? 0.f : pm == -INFINITY ? 1.f : ex2(pm - sm.ml[warp][2 * r]);
              v[j].x = fmaf(x.x, w, v[j].x), v[j].y = fmaf(x.y, w, v[j].y);
              v[j].z = fmaf(x.z, w, v[j].z), v[j].w = fmaf(x.w, w, v[j].w);
            }
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j0 + j < kPer)
              reinterpret_cast<float4*>(sm.o[warp])[(j0 + j) * 32 + lane] = v[j];
        }
        __syncthreads();
        for (int i = tid; i < kVec; i += kThreads) {
          const int r = i / (D / 4), d = i % (D / 4) * 4;
          float top = -INFINITY, sum = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm.ml[w][2 * r]);
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float wl = sm.ml[w][2 * r + 1], wm = sm.ml[w][2 * r];
            if (wl == 0.f) continue;
            const float k = wm == -INFINITY ? 1.f : ex2(wm - top);
            const float4 x = reinterpret_cast<const float4*>(sm.o[w])[i];
            v.x = fmaf(x.x, k, v.x), v.y = fmaf(x.y, k, v.y);
            v.z = fmaf(x.z, k, v.z), v.w = fmaf(x.w, k, v.w);
            sum = fmaf(wl, k, sum);
          }
          put(r, d, v, top, sum);
        }
        if (tid == 0) P.counters[c0] = 0;
      }
    }
    __syncthreads();
    const uint32_t u = use.end();
    if (u >= last) break;
    use.open(P, u, last);
  }
  // after a wait that gave up, copies may still be under way into this CTA's
  // shared memory: give them time to land (with a limit) before it goes to another
  if (sm.abort)
    for (int s = 0; s < S::kStages; ++s) {
      const uint64_t t0 = felix_sm100::globaltimer_ns();
      while (!felix_sm100::mbar_try_wait(felix_sm100::smem_u32(&sm.full[warp][s]), parity) &&
             felix_sm100::globaltimer_ns() - t0 < 1000000ull) {
      }
    }
}

// CTAs per SM that a caller's workspace has room for.
constexpr int kMaxPerSm = 4;
constexpr size_t ws_bytes_for(uint32_t grid, int rows, int D) {
  return kWsCounterBytes + size_t(grid) * 2 * rows * (D + 2) * sizeof(float);
}
// Tiles of 8 query rows that a warp keeps in registers: 5 of D = 64, 3 of D = 128.
constexpr int max_nt(int D) { return D == 64 ? 5 : 3; }

template <typename T, int D, int NT>
FelixCode launch(AttnParams& P, DeviceInfo* dev, void* workspace, size_t ws_bytes,
                 cudaStream_t stream) {
  static int per_sm[64];
  static PerDeviceOnce once;
  constexpr int smem = int(sizeof(Smem<D, NT>));
  const int rc = once.run(dev->ordinal, [&] {
    if (cudaFuncSetAttribute(kv4_attn_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             smem) != cudaSuccess)
      return -1;
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kv4_attn_kernel<T, D, NT>, kThreads,
                                                      smem) != cudaSuccess || n < 1)
      return -1;
    per_sm[dev->ordinal] = n < kMaxPerSm ? n : kMaxPerSm;
    return 0;
  });
  if (rc != 0) return launch_error(cudaGetLastError(), "kv4_attention: occupancy");
  const uint32_t grid = uint32_t(dev->num_sms) * uint32_t(per_sm[dev->ordinal]);
  const size_t need = ws_bytes_for(grid, 8 * NT, D);
  if (workspace && ws_bytes < need)
    return api_error("kv4_attention: workspace smaller than felix_kv4_attention_workspace_size");
  void* ws = workspace ? workspace : library_workspace(dev, stream, need);
  if (!ws) return launch_error(cudaErrorMemoryAllocation, "kv4_attention: workspace");
  P.counters = static_cast<uint32_t*>(ws);
  P.partials = reinterpret_cast<float*>(static_cast<char*>(ws) + kWsCounterBytes);
  P.row_tiles = (P.rows * P.group + 8 * NT - 1) / (8 * NT);
  kv4_attn_kernel<T, D, NT><<<grid, kThreads, smem, stream>>>(P);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return launch_error(e, "kv4_attention");
  return FelixCode{FELIX_SUCCESS, cudaSuccess};
}

// The fewest row tiles that registers allow, then as even as possible: each tile
// of rows reads the cache again.
template <typename T, int D>
FelixCode launch_rows(AttnParams& P, DeviceInfo* dev, void* workspace, size_t ws_bytes,
                      cudaStream_t stream) {
  const uint32_t eights = (P.rows * P.group + 7) / 8;
  const uint32_t tiles = (eights + max_nt(D) - 1) / max_nt(D);
  switch ((eights + tiles - 1) / tiles) {
    case 1: return launch<T, D, 1>(P, dev, workspace, ws_bytes, stream);
    case 2: return launch<T, D, 2>(P, dev, workspace, ws_bytes, stream);
    case 3: return launch<T, D, 3>(P, dev, workspace, ws_bytes, stream);
    default: break;
  }
  if constexpr (D == 64) {
    if ((eights + tiles - 1) / tiles == 4) return launch<T, D, 4>(P, dev, workspace, ws_bytes, stream);
    return launch<T, D, 5>(P, dev, workspace, ws_bytes, stream);
  }
  return api_error("kv4_attention: rows");
}

}  // namespace kv4

size_t kv4_attention_workspace_bytes(uint32_t head_dim, int num_sms) {
  return kv4::ws_bytes_for(uint32_t(num_sms) * kv4::kMaxPerSm, 8 * kv4::max_nt(int(head_dim)),
                           int(head_dim));
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

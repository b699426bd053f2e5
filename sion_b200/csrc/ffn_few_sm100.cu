// Products of a few tokens (up to 8) with a layer's weights: y = x W^T with the same
// epilogues as ffn_product_sm100.cu. Bound by reading W once.
//
// A CTA owns 16 rows of W (gated: 16 of the gate's and the same 16 of the up
// projection's), its 8 warps take every 8th block of 64 k, so that a row
// is read 1 KB at a time, and their sums meet in shared memory: no second pass, no
// atomics, and the result does not depend on the grid. W goes from memory straight into
// the operands of m16n8k16 (rows of W x 8 tokens): a product does not care for the order of
// k, so lane t of a quad takes k 8 t .. 8 t + 7 of 32 as one 16-byte load for two
// instructions, and x is read the same way. Not tcgen05: its smallest tile is 128 rows,
// which would leave 32 CTAs for 4096 rows, and W would pass through shared memory.
//
// Measured, one token: 4096 x 4096 7.9 us (4.25 TB/s; launch, start and tail of the stream),
// two projections of 4096 x 11264 29.9 to 31.3 us (6 TB/s).
#include <cuda_runtime.h>

#include <algorithm>

#include "activation.cuh"
#include "ffn_internal.h"
#include "sm100_ptx.cuh"

namespace felix_ffn {
namespace few {

constexpr uint32_t kWarps = 8, kBlock = 64;  // warps of a CTA, k of a warp's step

struct Params {
  const uint16_t *x, *w[2], *bias, *residual;
  int64_t x_ld, w_ld[2], residual_ld;
  uint16_t* out[3];
  int64_t out_ld[3];
  uint32_t tokens, n, k;
  int act;
};

// 8 elements of a row from k on; what lies behind the row's end is 0. Not by read-only loads:
// the launch before may still write while this kernel lives, and the compiler may move those
// in front of the wait for it.
template <bool VEC, bool STREAM>
__device__ __forceinline__ uint4 load8(const uint16_t* row, uint32_t k, uint32_t K, bool there) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if constexpr (VEC) {
    if (there && k < K) {
      const uint4* p = reinterpret_cast<const uint4*>(row + k);
      if constexpr (STREAM)
        asm volatile("ld.global.L1::no_allocate.L2::128B.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "l"(p));
      else
        v = *p;
    }
  } else if (there) {
    uint32_t e[8];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) e[i] = k + i < K ? row[k + i] : 0u;
    v = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
  }
  return v;
}

template <class T>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                    uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (Pair<T>::kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// VEC: rows of whole 16-byte vectors. Steps under way (D) and CTAs per SM, one token, us: one
// matrix 4096 x 16384 25.0 with 4 and 2, 25.7 with 2 and 3; two of 4096 x 11264 31.7 with 1 and
// 3 (5.8 TB/s), 34.4 with 2 and 2.
template <class T, bool GATED, bool VEC>
__global__ void __launch_bounds__(32 * kWarps, GATED ? 3 : 2) few_kernel(const Params p) {
  constexpr uint32_t kRows = 16;         // output features of a CTA
  constexpr int MT = GATED ? 2 : 1;      // tiles of 16 rows of weights
  constexpr int D = VEC && !GATED ? 4 : 1;  // steps of a warp under way
  __shared__ float part[kWarps][MT * 16][9];
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const uint32_t n0 = blockIdx.x * kRows;

  const uint16_t* wrow[MT][2];
  bool wthere[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t row = n0 + h * 8 + g;
      wthere[m][h] = row < p.n;
      wrow[m][h] = p.w[m] + int64_t(row) * p.w_ld[m];
    }
  const bool xthere = g < p.tokens;
  const uint16_t* xrow = p.x + int64_t(g) * p.x_ld;

  float c[MT][4] = {};
  uint4 wv[D][MT][2][2], xv[D][2];
  auto fetch = [&](int d, uint32_t step) {
    const uint32_t k = (step * kWarps + warp) * kBlock + t * 8;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r)
          wv[d][m][r][h] = load8<VEC, true>(wrow[m][r], k + 32 * h, p.k, wthere[m][r]);
      xv[d][h] = load8<VEC, false>(xrow, k + 32 * h, p.k, xthere);
    }
  };
  felix_sm100::launch_dependents();
  felix_sm100::wait_for_earlier_launches();
  const uint32_t steps = (p.k + kBlock * kWarps - 1) / (kBlock * kWarps);
#pragma unroll
  for (int d = 0; d < D; ++d) fetch(d, d);
  for (uint32_t s = 0; s < steps; s += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint4 a = wv[d][m][0][h], b = wv[d][m][1][h], x = xv[d][h];
          mma<T>(c[m], a.x, b.x, a.y, b.y, x.x, x.y);
          mma<T>(c[m], a.z, b.z, a.w, b.w, x.z, x.w);
        }
      fetch(d, s + D + d);
    }
  }

#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][m * 16 + (i >> 1) * 8 + g][2 * t + (i & 1)] = c[m][i];
  __syncthreads();

  // consecutive threads take consecutive features of a token
  for (uint32_t i = threadIdx.x; i < kRows * p.tokens; i += 32 * kWarps) {
    const uint32_t r = i % kRows, token = i / kRows, col = n0 + r;
    if (col >= p.n) continue;
    float v = 0.f;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) v += part[w][r][token];
    if constexpr (GATED) {
      float up = 0.f;
#pragma unroll
      for (uint32_t w = 0; w < kWarps; ++w) up += part[w][kRows + r][token];
      if (p.out[1]) p.out[1][token * p.out_ld[1] + col] = Pair<T>::of_float(v);
      if (p.out[2]) p.out[2][token * p.out_ld[2] + col] = Pair<T>::of_float(up);
      with_activation(p.act, [&]<int ACT>() { v = activate<ACT>(v) * up; });
    } else {
      if (p.bias) v += Pair<T>::to_float(p.bias[col]);
      if (p.out[1]) p.out[1][token * p.out_ld[1] + col] = Pair<T>::of_float(v);
      with_activation(p.act, [&]<int ACT>() { v = activate<ACT>(v); });
      if (p.residual) v += Pair<T>::to_float(p.residual[token * p.residual_ld + col]);
    }
    p.out[0][token * p.out_ld[0] + col] = Pair<T>::of_float(v);
  }
}

template <class T, bool GATED>
cudaError_t launch(const Params& p, bool vec, cudaStream_t stream) {
  const uint32_t grid = (p.n + 15) / 16;
  return vec ? launch_behind(few_kernel<T, GATED, true>, grid, 1, 32 * kWarps, 0, 1, stream, p)
             : launch_behind(few_kernel<T, GATED, false>, grid, 1, 32 * kWarps, 0, 1, stream, p);
}

}  // namespace few

FelixCode few_launch(const Product& x, cudaStream_t stream) {
  few::Params p{};
  const bool gated = x.epilogue == kGated;
  auto vec = [&](const Mat& m, uint32_t rows) {
    return (reinterpret_cast<uintptr_t>(m.p) & 15) == 0 && (rows <= 1 || m.ld % 8 == 0);
  };
  p.x = static_cast<const uint16_t*>(x.a[0].p);
  p.x_ld = x.a[0].ld;
  bool all = x.k[0] % 8 == 0 && vec(x.a[0], x.m[0]);
  for (int i = 0; i < (gated ? 2 : 1); ++i) {
    p.w[i] = static_cast<const uint16_t*>(x.b[i].p);
    p.w_ld[i] = x.b[i].ld;
    all = all && vec(x.b[i], x.n[0]);
  }
  p.bias = static_cast<const uint16_t*>(x.bias);
  p.residual = static_cast<const uint16_t*>(x.in[0].p);
  p.residual_ld = x.in[0].ld;
  for (int i = 0; i < 3; ++i) {
    p.out[i] = static_cast<uint16_t*>(x.out[i].p);
    p.out_ld[i] = x.out[i].ld;
  }
  p.tokens = x.m[0];
  p.n = x.n[0];
  p.k = x.k[0];
  p.act = x.act;
  const cudaError_t e =
      gated ? x.bf16 ? few::launch<__nv_bfloat16, true>(p, all, stream)
                     : few::launch<__half, true>(p, all, stream)
            : x.bf16 ? few::launch<__nv_bfloat16, false>(p, all, stream)
                     : few::launch<__half, false>(p, all, stream);
  if (e != cudaSuccess) return felix_impl::launch_error(e, "feed-forward: few tokens");
  return FelixCode{FELIX_SUCCESS, cudaSuccess};
}

}  // namespace felix_ffn

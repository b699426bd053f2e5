// Feed-forward operators: the linear layer and the gated block, forward and backward, as
// runs of products (ffn_product_sm100.cu) with the element-wise passes between them, and
// the extern "C" entry points declared in include/felix_c.h.
#include <cuda_runtime.h>

#include <algorithm>
#include <exception>
#include <initializer_list>

#include "activation.cuh"
#include "ffn_finish.cuh"
#include "ffn_internal.h"
#include "sm100_ptx.cuh"

namespace felix_ffn {
namespace {

using felix_impl::api_error;
using felix_impl::launch_error;

constexpr FelixCode kDone{FELIX_SUCCESS, cudaSuccess};

// ------------------------------------------------------------ element-wise passes
// Rows that TMA cannot address (odd sizes, addresses or strides, repeated rows) are
// copied to rows of a multiple of 16 bytes; what lies beside a row is never used. A thread
// writes one vector from the 4 or 5 aligned words that hold it, each with an element of the
// row (10 MB: 13 -> 6 us against one
// element at a time).
__global__ void __launch_bounds__(256)
    pack_kernel(const uint16_t* src, int64_t src_ld, uint16_t* dst, int64_t dst_ld, uint32_t rows,
                uint32_t cols) {
  felix_sm100::launch_dependents();
  felix_sm100::wait_for_earlier_launches();
  const uint32_t vectors = (cols + 7) / 8;
  const uint64_t all = uint64_t(rows) * vectors, stride = uint64_t(gridDim.x) * 256;
#pragma unroll 2
  for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < all; i += stride) {
    const uint32_t r = uint32_t(i / vectors), c = uint32_t(i - uint64_t(r) * vectors) * 8;
    const uint16_t* s = src + int64_t(r) * src_ld + c;
    uint32_t v[4];
    if (c + 8 <= cols) {
      const uint32_t odd = uint32_t(reinterpret_cast<uintptr_t>(s) >> 1) & 1;
      const uint32_t* w = reinterpret_cast<const uint32_t*>(s - odd);
      uint32_t x[5];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = w[j];
      x[4] = odd ? w[4] : 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __funnelshift_r(x[j], x[j + 1], 16 * odd);
    } else {
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        const uint32_t lo = c + 2 * j < cols ? s[2 * j] : 0u, hi = c + 2 * j + 1 < cols ? s[2 * j + 1] : 0u;
        v[j] = lo | hi << 16;
      }
    }
    *reinterpret_cast<uint4*>(dst + int64_t(r) * dst_ld + c) = make_uint4(v[0], v[1], v[2], v[3]);
  }
}

struct Elementwise {
  const uint16_t *grad, *z, *up;  // z: in front of the activation; up: gated only
  int64_t grad_ld, z_ld, up_ld;
  uint16_t *out, *out_up;  // dz, or dg and du
  int64_t out_ld;
  float* sums;  // [row blocks][cols], may be null
  uint16_t* bias;      // the bias' gradient
  unsigned* counters;  // one per block of columns, zero before and after
  uint32_t rows, cols, rows_per_block;
  int act;
};

// dz = grad act'(z) (z null: grad), or gated dg = grad up act'(z), du = grad act(z), and the
// columns' sums of dz for the bias' gradient. One pass: a warp reads 32 V columns of a row,
// the block's 8 warps take every 8th row; the last block of a range of columns adds up all
// blocks' sums in their order. Bound by memory: 8192 x 16384 with sums 147 us (5.5 TB/s).
template <class T, int V, bool GATED>
__global__ void __launch_bounds__(256) elementwise_kernel(const Elementwise p) {
  felix_sm100::launch_dependents();
  felix_sm100::wait_for_earlier_launches();
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const uint32_t col = (blockIdx.x * 32 + lane) * V;
  const uint32_t r0 = blockIdx.y * p.rows_per_block;
  const uint32_t r1 = min(p.rows, r0 + p.rows_per_block);
  float sum[V] = {};
  if (col < p.cols) {
    with_activation(p.act, [&]<int ACT>() {
#pragma unroll 4
      for (uint32_t r = r0 + warp; r < r1; r += 8) {
        float g[V], z[V], a, d;
        load_values<T, V>(p.grad + int64_t(r) * p.grad_ld + col, g);
        if constexpr (GATED) {
          float up[V], du[V];
          load_values<T, V>(p.z + int64_t(r) * p.z_ld + col, z);
          load_values<T, V>(p.up + int64_t(r) * p.up_ld + col, up);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            activate_both<ACT>(z[i], a, d);
            du[i] = g[i] * a;
            g[i] *= up[i] * d;
          }
          store_values<T, V>(p.out_up + int64_t(r) * p.out_ld + col, du);
        } else if constexpr (ACT != FELIX_ACT_NONE) {
          load_values<T, V>(p.z + int64_t(r) * p.z_ld + col, z);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            activate_both<ACT>(z[i], a, d);
            g[i] *= d;
          }
        }
        if (GATED || p.out) store_values<T, V>(p.out + int64_t(r) * p.out_ld + col, g);
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] += g[i];
      }
    });
  }
  if constexpr (!GATED) {
    if (!p.sums) return;
    __shared__ float part[8][32 * V];
    __shared__ bool last;
#pragma unroll
    for (int i = 0; i < V; ++i) part[warp][i * 32 + lane] = sum[i];
    __syncthreads();
    const uint32_t i = threadIdx.x, c = (blockIdx.x * 32 + i % 32) * V + i / 32;
    const bool mine = i < 32 * V && c < p.cols;
    if (mine) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) s += part[w][i];
      __stcg(p.sums + size_t(blockIdx.y) * p.cols + c, s);
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
      last = atomicAdd(&p.counters[blockIdx.x], 1u) == gridDim.y - 1;
      if (last) p.counters[blockIdx.x] = 0;
    }
    __syncthreads();
    if (!last || !mine) return;
    __threadfence();
    float s = 0.f;
#pragma unroll 16
    for (uint32_t b = 0; b < gridDim.y; ++b) s += __ldcg(p.sums + size_t(b) * p.cols + c);
    p.bias[c] = Pair<T>::of_float(s);
  }
}

// ------------------------------------------------------------------------ a call
// One call: first without memory, which only counts what it needs, then with it.
struct Call {
  DeviceInfo* dev;
  cudaStream_t stream;
  bool bf16;
  enum { kCount, kLaunch } pass = kCount;
  uint8_t* base = nullptr;
  // The products' counters come first. In the library's scratch other calls rely on them
  // even where this one has no product that uses them.
  static constexpr size_t kFront = felix_impl::kWsCounterBytes;
  bool tiled = false;  // a product uses them
  size_t used = 0;     // bytes behind them
  FelixCode code = kDone;

  bool ok() const { return code.type == FELIX_SUCCESS; }
  bool counting() const { return pass == kCount; }
  size_t total() const { return tiled || used ? kFront + used : 0; }

  void* take(size_t bytes) {
    void* p = counting() ? nullptr : base + kFront + used;
    used += (bytes + 255) / 256 * 256;
    return p;
  }
  // A matrix of rows that TMA can address.
  MutMat matrix(uint32_t rows, uint32_t cols) {
    const int64_t ld = (int64_t(cols) + 7) / 8 * 8;
    return {take(size_t(rows) * ld * 2), ld};
  }
  void check(cudaError_t e, const char* what) {
    if (ok() && e != cudaSuccess) code = launch_error(e, what);
  }
  // m itself, or a copy where TMA cannot address it.
  Mat addressable(const felix_matrix& m, uint32_t rows, uint32_t cols) {
    if (tma_ok(m.data, m.stride, rows, cols)) return {m.data, m.stride};
    const MutMat c = matrix(rows, cols);
    if (!counting() && ok()) {
      const uint64_t vectors = uint64_t(rows) * ((cols + 7) / 8);
      const uint32_t grid = uint32_t(std::min<uint64_t>((vectors + 255) / 256, 16u * dev->num_sms));
      check(launch_behind(pack_kernel, grid, 1, 256, 0, 1, stream,
                          static_cast<const uint16_t*>(m.data), m.stride,
                          static_cast<uint16_t*>(c.p), c.ld, rows, cols),
            "feed-forward: copy");
    }
    return {c.p, c.ld};
  }
  // An operand of a product: as it is for few tokens, else addressable by TMA.
  Mat operand(const Product& p, const felix_matrix& m, uint32_t rows, uint32_t cols) {
    return few_tokens(p) ? Mat{m.data, m.stride} : addressable(m, rows, cols);
  }
  void run(const Product& p) {
    if (few_tokens(p)) {
      if (!counting() && ok()) code = few_launch(p, stream);
    } else if (narrow_tokens(p)) {
      if (!counting() && ok()) code = narrow_launch(dev, p, stream);
    } else if (counting()) {
      tiled = true;
    } else if (ok()) {
      code = product_launch(dev, p, base, stream);
    }
  }
  void zero_bytes(void* p, size_t bytes) {
    if (counting() || !ok()) return;
    const cudaError_t e = cudaMemsetAsync(p, 0, bytes, stream);
    if (e != cudaSuccess) code = launch_error(e, "feed-forward: zero");
  }
  void zero(const felix_matrix& m, uint32_t rows, uint32_t cols) {
    if (counting() || !ok() || !m.data) return;
    const size_t width = size_t(cols) * 2, pitch = rows > 1 ? size_t(m.stride) * 2 : width;
    const cudaError_t e = cudaMemset2DAsync(m.data, pitch, 0, width, rows, stream);
    if (e != cudaSuccess) code = launch_error(e, "feed-forward: zero");
  }
};

bool vectors(std::initializer_list<Mat> list, uint32_t rows, uint32_t cols) {
  if (cols % 8) return false;
  for (const Mat& m : list)
    if (m.p && ((reinterpret_cast<uintptr_t>(m.p) & 15) || (rows > 1 && m.ld % 8))) return false;
  return true;
}

template <class T, bool GATED>
void elementwise(Call& c, Elementwise& e, uint32_t blocks, bool vec) {
  const auto kernel = vec ? elementwise_kernel<T, 8, GATED> : elementwise_kernel<T, 1, GATED>;
  c.check(launch_behind(kernel, (e.cols + (vec ? 255 : 31)) / (vec ? 256 : 32), blocks, 256, 0, 1,
                        c.stream, e),
          "feed-forward: element-wise pass");
}

Mat as_mat(const felix_matrix& m) { return {m.data, m.stride}; }
MutMat as_mut(const felix_matrix& m) { return {m.data, m.stride}; }
Mat as_mat(const MutMat& m) { return {m.p, m.ld}; }

// The products of a backward pass, in one launch or two, deepest first: B always lies with n
// contiguous, A with k (dx) or m (the weights' gradients).
struct Backward {
  struct One {
    uint32_t m, n, k, segments;
    bool a_mn;
    Mat a[2], b[2];
    MutMat out;
  };
  One list[kMaxProblems];
  uint32_t count = 0;
  void add(const One& one) { list[count++] = one; }
  void run(Call& c) {
    if (!count) return;
    std::stable_sort(list, list + count, [](const One& x, const One& y) {
      return uint64_t(x.k) * x.segments > uint64_t(y.k) * y.segments;
    });
    Product p;
    p.bf16 = c.bf16;
    p.problems = count;
    uint32_t operand = 0;
    for (uint32_t i = 0; i < count; ++i) {
      const One& one = list[i];
      p.m[i] = one.m;
      p.n[i] = one.n;
      p.k[i] = one.k;
      p.segments[i] = one.segments;
      p.a_mn[i] = one.a_mn;
      p.b_mn[i] = true;
      p.out[i] = one.out;
      for (uint32_t s = 0; s < one.segments; ++s, ++operand) {
        p.a[operand] = one.a[s];
        p.b[operand] = one.b[s];
      }
    }
    c.run(p);
  }
};

// dz and the bias' gradient; returns dz as the products read it. It is rounded to 16 bits, as
// the tensor cores' operands are (a product in more bits would take several), which together
// with the results' own rounding makes their error 1.4 times that of the latter alone; the
// bias' gradient is summed from the values before it.
Mat linear_gradient(Call& c, const felix_linear_args& a) {
  const uint32_t T = a.tokens, N = a.out_features;
  const bool acts = a.activation != FELIX_ACT_NONE;
  const bool copy = (a.dx.data || a.dweight.data) &&
                    (acts || !tma_ok(a.grad.data, a.grad.stride, T, N));
  MutMat dz;
  if (copy) dz = c.matrix(T, N);
  const bool vec = vectors({as_mat(a.grad), {acts ? a.pre.data : nullptr, a.pre.stride}}, T, N);
  // blocks of rows for some 16 CTAs per SM, of 32 rows at least: the last one adds up all
  // blocks' sums, 16 at a time
  const uint32_t columns = (N + (vec ? 255 : 31)) / (vec ? 256 : 32), sms = uint32_t(c.dev->num_sms);
  const uint32_t want = std::max(1u, 16 * sms / columns);
  const uint32_t per = std::max(32u, ((T + want - 1) / want + 7) / 8 * 8);
  const uint32_t blocks = (T + per - 1) / per;
  float* sums = nullptr;
  unsigned* counters = nullptr;
  if (a.dbias) {
    sums = static_cast<float*>(c.take(size_t(blocks) * N * 4));
    // in front of the scratch, or of their own where there are very many columns
    c.tiled = true;
    counters = static_cast<unsigned*>(columns <= felix_impl::kWsMaxCounters - 2
                                          ? c.base
                                          : c.take(size_t(columns) * 4));
    if (columns > felix_impl::kWsMaxCounters - 2) c.zero_bytes(counters, size_t(columns) * 4);
  }
  if (!c.counting() && c.ok() && (copy || a.dbias)) {
    Elementwise e{};
    e.grad = static_cast<const uint16_t*>(a.grad.data);
    e.grad_ld = a.grad.stride;
    e.z = static_cast<const uint16_t*>(a.pre.data);
    e.z_ld = a.pre.stride;
    e.out = static_cast<uint16_t*>(dz.p);
    e.out_ld = dz.ld;
    e.sums = sums;
    e.bias = static_cast<uint16_t*>(a.dbias);
    e.counters = counters;
    e.rows = T;
    e.cols = N;
    e.rows_per_block = per;
    e.act = a.activation;
    c.bf16 ? elementwise<__nv_bfloat16, false>(c, e, blocks, vec)
           : elementwise<__half, false>(c, e, blocks, vec);
  }
  return copy ? Mat{dz.p, dz.ld} : Mat{a.grad.data, a.grad.stride};
}

void linear(Call& c, const felix_linear_args& a) {
  if (!a.tokens) return;
  Product p;
  p.bf16 = c.bf16;
  p.k[0] = a.in_features;
  p.m[0] = a.tokens;
  p.n[0] = a.out_features;
  p.a[0] = c.operand(p, a.x, a.tokens, a.in_features);
  p.b[0] = c.operand(p, a.weight, a.out_features, a.in_features);
  p.out[0] = as_mut(a.out);
  p.out[1] = as_mut(a.pre);
  p.in[0] = as_mat(a.residual);
  p.bias = a.bias;
  p.act = a.activation;
  c.run(p);
}

void linear_bwd(Call& c, const felix_linear_args& a) {
  const uint32_t T = a.tokens, K = a.in_features, N = a.out_features;
  if (!T) {
    c.zero(a.dweight, N, K);
    c.zero({a.dbias, 0}, 1, N);
    return;
  }
  const Mat dz = linear_gradient(c, a);
  Backward all;
  if (a.dx.data)
    all.add({T, K, N, 1, false, {dz}, {c.addressable(a.weight, N, K)}, as_mut(a.dx)});
  if (a.dweight.data)
    all.add({N, K, T, 1, true, {dz}, {c.addressable(a.x, T, K)}, as_mut(a.dweight)});
  all.run(c);
}

// h = act(x Wg^T) (x Wu^T), and g, u where they are wanted.
void gated_product(Call& c, const felix_gated_args& a, const MutMat& h) {
  Product p;
  p.epilogue = kGated;
  p.bf16 = c.bf16;
  p.k[0] = a.features;
  p.m[0] = a.tokens;
  p.n[0] = a.hidden;
  p.a[0] = c.operand(p, a.x, a.tokens, a.features);
  p.b[0] = c.operand(p, a.w_gate, a.hidden, a.features);
  p.b[1] = c.operand(p, a.w_up, a.hidden, a.features);
  p.out[0] = h;
  p.out[1] = as_mut(a.gate);
  p.out[2] = as_mut(a.up);
  p.act = a.activation;
  c.run(p);
}

void gated_linear(Call& c, const felix_gated_args& a) {
  if (a.tokens) gated_product(c, a, as_mut(a.out));
}

// h, the second product's operand, is rounded to 16 bits: 1.2 times the error of y's rounding.
void gated_ffn(Call& c, const felix_gated_args& a) {
  if (!a.tokens) return;
  const MutMat h = c.matrix(a.tokens, a.hidden);
  gated_product(c, a, h);
  Product p;
  p.bf16 = c.bf16;
  p.k[0] = a.hidden;
  p.m[0] = a.tokens;
  p.n[0] = a.features;
  p.a[0] = as_mat(h);
  p.b[0] = c.operand(p, a.w_down, a.features, a.hidden);
  p.out[0] = as_mut(a.out);
  p.in[0] = as_mat(a.residual);
  c.run(p);
}

// The gradients of x and of the weights from dg, du (and h), operands of 16 bits as dz is.
void gated_products(Call& c, const felix_gated_args& a, const MutMat& dg, const MutMat& du,
                    const Mat& grad, const MutMat& h) {
  const uint32_t T = a.tokens, K = a.features, F = a.hidden;
  Backward all;
  if (a.dx.data)
    all.add({T, K, F, 2, false, {as_mat(dg), as_mat(du)},
             {c.addressable(a.w_gate, F, K), c.addressable(a.w_up, F, K)}, as_mut(a.dx)});
  if (a.dw_gate.data || a.dw_up.data) {
    const Mat x = c.addressable(a.x, T, K);
    if (a.dw_gate.data) all.add({F, K, T, 1, true, {as_mat(dg)}, {x}, as_mut(a.dw_gate)});
    if (a.dw_up.data) all.add({F, K, T, 1, true, {as_mat(du)}, {x}, as_mut(a.dw_up)});
  }
  if (a.dw_down.data) all.add({K, F, T, 1, true, {grad}, {as_mat(h)}, as_mut(a.dw_down)});
  all.run(c);
}

void no_tokens(Call& c, const felix_gated_args& a) {
  c.zero(a.dw_gate, a.hidden, a.features);
  c.zero(a.dw_up, a.hidden, a.features);
  c.zero(a.dw_down, a.features, a.hidden);
}

bool no_gradient(const felix_gated_args& a) {
  return !a.dx.data && !a.dw_gate.data && !a.dw_up.data && !a.dw_down.data;
}

void gated_linear_bwd(Call& c, const felix_gated_args& a) {
  if (!a.tokens) return no_tokens(c, a);
  if (no_gradient(a)) return;
  const uint32_t T = a.tokens, F = a.hidden;
  const MutMat dg = c.matrix(T, F), du = c.matrix(T, F);
  if (!c.counting() && c.ok()) {
    Elementwise e{};
    e.grad = static_cast<const uint16_t*>(a.grad.data);
    e.grad_ld = a.grad.stride;
    e.z = static_cast<const uint16_t*>(a.gate.data);
    e.z_ld = a.gate.stride;
    e.up = static_cast<const uint16_t*>(a.up.data);
    e.up_ld = a.up.stride;
    e.out = static_cast<uint16_t*>(dg.p);
    e.out_up = static_cast<uint16_t*>(du.p);
    e.out_ld = dg.ld;
    e.rows = T;
    e.cols = F;
    e.rows_per_block = std::max(32u, (T + 65534) / 65535);
    e.act = a.activation;
    const uint32_t blocks = (T + e.rows_per_block - 1) / e.rows_per_block;
    const bool vec = vectors({as_mat(a.grad), as_mat(a.gate), as_mat(a.up)}, T, F);
    c.bf16 ? elementwise<__nv_bfloat16, true>(c, e, blocks, vec)
           : elementwise<__half, true>(c, e, blocks, vec);
  }
  gated_products(c, a, dg, du, Mat{}, MutMat{});
}

void gated_ffn_bwd(Call& c, const felix_gated_args& a) {
  if (!a.tokens) return no_tokens(c, a);
  if (no_gradient(a)) return;
  const uint32_t T = a.tokens, K = a.features, F = a.hidden;
  const Mat grad = c.addressable(a.grad, T, K);
  const MutMat dg = c.matrix(T, F), du = c.matrix(T, F);
  const MutMat h = a.dw_down.data ? c.matrix(T, F) : MutMat{};  // nothing else reads it
  Product p;
  p.epilogue = kDGated;
  p.bf16 = c.bf16;
  p.k[0] = K;
  p.m[0] = T;
  p.n[0] = F;
  p.a[0] = grad;
  p.b[0] = c.addressable(a.w_down, K, F);
  p.b_mn[0] = true;
  p.in[0] = as_mat(a.gate);
  p.in[1] = as_mat(a.up);
  p.out[0] = dg;
  p.out[1] = du;
  p.out[2] = h;
  p.act = a.activation;
  c.run(p);
  gated_products(c, a, dg, du, grad, h);
}

// ------------------------------------------------------------------------- checks
constexpr uint32_t kMostSize = 1u << 30;

FelixCode check_common(uint32_t tokens, uint32_t in, uint32_t out, int dtype, int act) {
  if (dtype != FELIX_F16 && dtype != FELIX_BF16)
    return api_error("feed-forward: elements must be fp16 or bf16");
  if (act < FELIX_ACT_NONE || act > FELIX_ACT_SIGMOID)
    return api_error("feed-forward: unknown activation");
  if (in == 0 || out == 0 || in > kMostSize || out > kMostSize || tokens > kMostSize)
    return api_error("feed-forward: features must be 1..2^30, tokens at most 2^30");
  return kDone;
}

// An input that the call reads: null only where it is optional or there are no tokens; rows
// may repeat. (What a call does not read is not checked.)
FelixCode check_in(const felix_matrix& m, const char* null_text, bool optional) {
  if (!m.data) return optional ? kDone : api_error(null_text);
  if (reinterpret_cast<uintptr_t>(m.data) & 1)
    return api_error("feed-forward: matrices must be 2-byte aligned");
  if (m.stride < 0) return api_error("feed-forward: strides must not be negative");
  return kDone;
}
FelixCode check_out(const felix_matrix& m, uint32_t rows, uint32_t cols, const char* null_text,
                    bool optional) {
  const FelixCode rc = check_in(m, null_text, optional);
  if (rc.type != FELIX_SUCCESS || !m.data) return rc;
  if (rows > 1 && m.stride < int64_t(cols))
    return api_error("feed-forward: rows of an output overlap (stride below its columns)");
  return kDone;
}

#define FELIX_CHECK(x)                                   \
  do {                                                   \
    const FelixCode rc_ = (x);                           \
    if (rc_.type != FELIX_SUCCESS) return rc_;           \
  } while (0)

constexpr char kNull[] = "feed-forward: null pointer";

FelixCode check_linear(const felix_linear_args* a, bool backward) {
  if (!a) return api_error(kNull);
  const uint32_t T = a->tokens, K = a->in_features, N = a->out_features;
  FELIX_CHECK(check_common(T, K, N, a->dtype, a->activation));
  const bool none = T == 0;
  if (!backward) {
    FELIX_CHECK(check_in(a->x, kNull, none));
    FELIX_CHECK(check_in(a->weight, kNull, none));
    FELIX_CHECK(check_in(a->residual, kNull, true));
    FELIX_CHECK(check_out(a->out, T, N, kNull, none));
    FELIX_CHECK(check_out(a->pre, T, N, kNull, true));
    FELIX_CHECK(check_in({const_cast<void*>(a->bias), 0}, kNull, true));
    return kDone;
  }
  FELIX_CHECK(check_in(a->grad, kNull, none));
  if (a->dweight.data) FELIX_CHECK(check_in(a->x, kNull, none));
  if (a->dx.data) FELIX_CHECK(check_in(a->weight, kNull, none));
  if (a->activation != FELIX_ACT_NONE)
    FELIX_CHECK(check_in(a->pre, "feed-forward: the backward pass of an activation needs pre", none));
  FELIX_CHECK(check_out(a->dx, T, K, kNull, true));
  FELIX_CHECK(check_out(a->dweight, N, K, kNull, true));
  FELIX_CHECK(check_in({a->dbias, 0}, kNull, true));
  return kDone;
}

FelixCode check_gated(const felix_gated_args* a, bool ffn, bool backward) {
  if (!a) return api_error(kNull);
  const uint32_t T = a->tokens, K = a->features, F = a->hidden;
  FELIX_CHECK(check_common(T, K, F, a->dtype, a->activation));
  const bool none = T == 0;
  if (!backward) {
    FELIX_CHECK(check_in(a->x, kNull, none));
    FELIX_CHECK(check_in(a->w_gate, kNull, none));
    FELIX_CHECK(check_in(a->w_up, kNull, none));
    if (ffn) FELIX_CHECK(check_in(a->w_down, kNull, none));
    FELIX_CHECK(check_in(a->residual, kNull, true));
    if (!ffn && a->residual.data)
      return api_error("feed-forward: a gated projection alone has no residual");
    FELIX_CHECK(check_out(a->out, T, ffn ? K : F, kNull, none));
    FELIX_CHECK(check_out(a->gate, T, F, kNull, true));
    FELIX_CHECK(check_out(a->up, T, F, kNull, true));
    return kDone;
  }
  FELIX_CHECK(check_in(a->grad, kNull, none));
  FELIX_CHECK(check_in(a->gate, kNull, none));
  FELIX_CHECK(check_in(a->up, kNull, none));
  if (a->dw_gate.data || a->dw_up.data) FELIX_CHECK(check_in(a->x, kNull, none));
  if (a->dx.data) FELIX_CHECK(check_in(a->w_gate, kNull, none));
  if (a->dx.data) FELIX_CHECK(check_in(a->w_up, kNull, none));
  if (ffn) FELIX_CHECK(check_in(a->w_down, kNull, none));
  FELIX_CHECK(check_out(a->dx, T, K, kNull, true));
  FELIX_CHECK(check_out(a->dw_gate, F, K, kNull, true));
  FELIX_CHECK(check_out(a->dw_up, F, K, kNull, true));
  FELIX_CHECK(check_out(a->dw_down, K, F, kNull, true));
  if (!ffn && a->dw_down.data)
    return api_error("feed-forward: a gated projection alone has no down projection");
  return kDone;
}

// Counts a call's memory, finds it, and makes the call.
template <class Args>
FelixCode perform(void (*op)(Call&, const Args&), const Args& a, void* workspace, size_t bytes,
                  size_t* need, void* stream_) {
  DeviceInfo* dev = felix_impl::current_device_info();
  if (!dev) return launch_error(cudaGetLastError(), "feed-forward: no CUDA device");
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  Call count{dev, stream, a.dtype == FELIX_BF16};
  op(count, a);
  if (need) {
    *need = count.total();
    return kDone;
  }
  Call call = count;
  call.used = 0;
  felix_impl::Workspace scratch;  // until the last launch
  if (!workspace && count.total()) {
    scratch = felix_impl::library_workspace(dev, stream, count.total());
    workspace = scratch.ptr;
    if (!workspace) return launch_error(cudaErrorMemoryAllocation, "feed-forward: workspace");
  } else if (workspace) {
    if (bytes < count.total()) return api_error("feed-forward: workspace too small");
    // a caller's memory may hold anything: the products' counters start from zero
    if (count.tiled) {
      const cudaError_t e =
          cudaMemsetAsync(workspace, 0, felix_impl::kWsCounterBytes, stream);
      if (e != cudaSuccess) return launch_error(e, "feed-forward: workspace");
    }
  }
  call.pass = Call::kLaunch;
  call.base = static_cast<uint8_t*>(workspace);
  op(call, a);
  return call.code;
}

template <class F>
int guarded(F&& f) {
  try {
    return felix_impl::finish(f());
  } catch (const std::exception& e) {
    return api_error(e.what(), cudaErrorMemoryAllocation).type;
  } catch (...) {
    return api_error("unknown C++ exception", cudaErrorUnknown).type;
  }
}

template <class Args>
int entry(const FelixCode& checked, void (*op)(Call&, const Args&), const Args* a, void* workspace,
          size_t bytes, size_t* need, void* stream) {
  return guarded([&]() -> FelixCode {
    FELIX_CHECK(checked);
    if (reinterpret_cast<uintptr_t>(workspace) & 255)
      return api_error("feed-forward: workspace must be 256-byte aligned");
    return perform(op, *a, workspace, bytes, need, stream);
  });
}

}  // namespace
}  // namespace felix_ffn

using namespace felix_ffn;

extern "C" {

int felix_linear(const felix_linear_args* a, void* ws, size_t bytes, void* stream) {
  return entry(check_linear(a, false), &linear, a, ws, bytes, nullptr, stream);
}
int felix_linear_bwd(const felix_linear_args* a, void* ws, size_t bytes, void* stream) {
  return entry(check_linear(a, true), &linear_bwd, a, ws, bytes, nullptr, stream);
}
int felix_gated_linear(const felix_gated_args* a, void* ws, size_t bytes, void* stream) {
  return entry(check_gated(a, false, false), &gated_linear, a, ws, bytes, nullptr, stream);
}
int felix_gated_linear_bwd(const felix_gated_args* a, void* ws, size_t bytes, void* stream) {
  return entry(check_gated(a, false, true), &gated_linear_bwd, a, ws, bytes, nullptr, stream);
}
int felix_gated_ffn(const felix_gated_args* a, void* ws, size_t bytes, void* stream) {
  return entry(check_gated(a, true, false), &gated_ffn, a, ws, bytes, nullptr, stream);
}
int felix_gated_ffn_bwd(const felix_gated_args* a, void* ws, size_t bytes, void* stream) {
  return entry(check_gated(a, true, true), &gated_ffn_bwd, a, ws, bytes, nullptr, stream);
}

int felix_linear_workspace_size(const felix_linear_args* a, int backward, size_t* bytes) {
  size_t need = 0;
  const int rc = entry(check_linear(a, backward != 0), backward ? &linear_bwd : &linear, a, nullptr,
                       0, &need, nullptr);
  if (rc == FELIX_SUCCESS && bytes) *bytes = need;
  return rc;
}
int felix_gated_workspace_size(const felix_gated_args* a, int ffn, int backward, size_t* bytes) {
  size_t need = 0;
  const auto op = ffn ? (backward ? &gated_ffn_bwd : &gated_ffn)
                      : (backward ? &gated_linear_bwd : &gated_linear);
  const int rc = entry(check_gated(a, ffn != 0, backward != 0), op, a, nullptr, 0, &need, nullptr);
  if (rc == FELIX_SUCCESS && bytes) *bytes = need;
  return rc;
}

}  // extern "C"

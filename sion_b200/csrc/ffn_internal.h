// Host-side interfaces of the feed-forward operators' translation units.
#pragma once
#include <utility>

#include "felix_internal.h"

namespace felix_ffn {

using felix_impl::DeviceInfo;
using felix_impl::FelixCode;

// A matrix of 16-bit elements whose rows are `ld` elements apart.
struct Mat {
  const void* p = nullptr;
  int64_t ld = 0;
};
struct MutMat {
  void* p = nullptr;
  int64_t ld = 0;
};

// What a product's epilogue makes of the fp32 accumulators.
enum Epilogue {
  kLinear = 0,  // out0 = act(v + bias) + in0, out1 = v + bias
  kGated = 1,   // v = g | u: out0 = act(g) u, out1 = g, out2 = u
  kDGated = 2   // v = dh, in0 = g, in1 = u: out0 = dh u act'(g), out1 = dh act(g), and, where it
                // is wanted, out2 = act(g) u
};

constexpr uint32_t kMaxProblems = 4, kMaxOperands = 5;

// D[m][n] = sum over segments and k of A[m][k] B[n][k], for one or (kLinear without anything
// behind the product) several independent problems, deepest first. An operand is stored
// either with k contiguous (A [m][k], B [n][k]) or, "mn", with m or n contiguous (A [k][m],
// B [k][n]).
struct Product {
  Epilogue epilogue = kLinear;
  bool bf16 = false;
  uint32_t problems = 1;
  uint32_t m[kMaxProblems] = {}, n[kMaxProblems] = {};
  uint32_t k[kMaxProblems] = {};                    // depth of one segment
  uint32_t segments[kMaxProblems] = {1, 1, 1, 1};   // kLinear only
  bool a_mn[kMaxProblems] = {}, b_mn[kMaxProblems] = {};
  Mat a[kMaxOperands], b[kMaxOperands];  // problem after problem; kGated: b[0] gate, b[1] up
  MutMat out[kMaxProblems];  // of the problems, or one problem's (null: not wanted)
  Mat in[2];
  const void* bias = nullptr;
  int act = FELIX_ACT_NONE;
};

// A launch that may be set up while the one before it runs or drains (the kernel waits for
// that one itself, wait_for_earlier_launches): 2.3 us less for one token x 4096 x 4096, 3.5
// us for a gated block. The kernels of a few tokens and the element-wise ones let the next
// launch in from their start; those that fill an SM's shared memory do not (the next
// launch's CTAs would scatter their clusters: 1031 x 768 x 2312 backward 31 instead of 25 us).
template <class... K, class... A>
cudaError_t launch_behind(void (*kernel)(K...), uint32_t grid_x, uint32_t grid_y, uint32_t threads,
                          uint32_t smem, uint32_t cluster, cudaStream_t stream, A&&... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid_x, grid_y);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}

// Whether TMA can address a matrix of these rows.
inline bool tma_ok(const void* p, int64_t ld, uint32_t rows, uint64_t cols) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 &&
         (rows <= 1 || (ld % 8 == 0 && ld >= int64_t(cols) && ld < (int64_t(1) << 38)));
}

// A product of any size: a and b must be addressable by TMA; workspace: kWsCounterBytes of
// counters that are zero before and after.
FelixCode product_launch(DeviceInfo* dev, const Product& p, void* workspace, cudaStream_t stream);

// Products of few tokens, for which reading the weights is all: up to 8 (operands of any
// address and stride) and up to 64 (addressable by TMA). Neither needs scratch.
inline bool forward_product(const Product& p) {
  return p.epilogue != kDGated && p.problems == 1 && p.segments[0] == 1 && !p.a_mn[0] && !p.b_mn[0];
}
inline bool few_tokens(const Product& p) { return p.m[0] <= 8 && forward_product(p); }
FelixCode few_launch(const Product& p, cudaStream_t stream);
inline bool narrow_tokens(const Product& p) { return p.m[0] <= 64 && forward_product(p); }
FelixCode narrow_launch(DeviceInfo* dev, const Product& p, cudaStream_t stream);

}  // namespace felix_ffn

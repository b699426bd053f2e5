// sion:: LibTorch wrappers and the Python module `sion_b200._sion`.
//
// Same validation, output allocation, stream pickup and error conversion as the
// reference wrappers (src/sion/gemm/sgemm/sgemm.cpp:5-32,
// src/sion/gemm/hgemm/hgemm.cpp:4-83, src/sion/gemm/gemm.cpp:10-31,
// src/sion/flash_attention/flash_attn.cpp:7-66), calling the felix:: API with
// the reference's kernel names. Differences, all additive:
//   * C is zero-filled when beta != 0 (the reference reads uninitialised
//     torch::empty memory there, sgemm.cpp:19,27);
//   * flash_attention accepts any seqlen (the reference requires seqlen % 64);
//   * flash_attention_lse also returns the fp32 log-sum-exp; both take an
//     optional causal mask;
//   * the Python functions take named arguments (python/binding.cpp:6-11 has none).
#include <sion/sion.hpp>

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <felix/felix.hpp>
#include <torch/extension.h>

#include <array>

namespace sion {

namespace {
torch::Tensor make_output(int64_t M, int64_t N, const torch::TensorOptions& opt, float beta) {
  return beta != 0.f ? torch::zeros({M, N}, opt) : torch::empty({M, N}, opt);
}
}  // namespace

torch::Tensor sgemm(const torch::Tensor& A, const torch::Tensor& B, float alpha, float beta) {
  TORCH_CHECK(A.is_cuda(), "A must be CUDA tensor");
  TORCH_CHECK(B.is_cuda(), "B must be CUDA tensor");
  TORCH_CHECK(A.dtype() == torch::kFloat32, "A must be float32");
  TORCH_CHECK(B.dtype() == torch::kFloat32, "B must be float32");
  TORCH_CHECK(A.dim() == 2 && B.dim() == 2, "A and B must be 2D");
  const c10::cuda::CUDAGuard guard(A.device());
  auto Ac = A.contiguous();
  auto Bc = B.contiguous();
  const int64_t M = Ac.size(0), K = Ac.size(1), N = Bc.size(1);
  TORCH_CHECK(Bc.size(0) == K, "B.size(0) must match A.size(1)");
  auto C = make_output(M, N, Ac.options(), beta);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  auto status = felix::ampere_sgemm_launch(uint32_t(M), uint32_t(N), uint32_t(K), alpha,
                                           Ac.data_ptr<float>(), Bc.data_ptr<float>(), beta,
                                           C.data_ptr<float>(), stream);
  TORCH_CHECK(status.ok(), "SGEMM launch failed: ", status.str());
  return C;
}

namespace {
torch::Tensor hgemm_impl(const torch::Tensor& A, const torch::Tensor& B, float alpha, float beta,
                         bool nt) {
  TORCH_CHECK(A.is_cuda(), "A must be CUDA tensor");
  TORCH_CHECK(B.is_cuda(), "B must be CUDA tensor");
  TORCH_CHECK(A.dtype() == torch::kFloat16, "A must be float16");
  TORCH_CHECK(B.dtype() == torch::kFloat16, "B must be float16");
  TORCH_CHECK(A.dim() == 2, "A must be 2D");
  TORCH_CHECK(B.dim() == 2, "B must be 2D");
  TORCH_CHECK(A.is_contiguous(), "A must be contiguous");
  TORCH_CHECK(B.is_contiguous(), "B must be contiguous");
  const c10::cuda::CUDAGuard guard(A.device());
  const int64_t M = A.size(0), K = A.size(1);
  const int64_t N = nt ? B.size(0) : B.size(1);
  if (nt) {
    TORCH_CHECK(B.size(1) == K, "B.size(1) must match A.size(1) for NT GEMM");
  } else {
    TORCH_CHECK(B.size(0) == K, "B.size(0) must match A.size(1)");
  }
  auto C = make_output(M, N, A.options(), beta);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  auto status = felix::ampere_hgemm_launch(
      uint32_t(M), uint32_t(N), uint32_t(K), alpha,
      reinterpret_cast<const half*>(A.data_ptr<at::Half>()),
      reinterpret_cast<const half*>(B.data_ptr<at::Half>()), beta,
      reinterpret_cast<half*>(C.data_ptr<at::Half>()), stream,
      nt ? "cute_hgemm_128x128_nt" : "cute_hgemm_128x128_nn");
  TORCH_CHECK(status.ok(), nt ? "HGEMM NT launch failed: " : "HGEMM launch failed: ",
              status.str());
  return C;
}
}  // namespace

torch::Tensor hgemm(const torch::Tensor& A, const torch::Tensor& B, float alpha, float beta) {
  return hgemm_impl(A, B, alpha, beta, false);
}

torch::Tensor hgemm_nt(const torch::Tensor& A, const torch::Tensor& B, float alpha, float beta) {
  return hgemm_impl(A, B, alpha, beta, true);
}

torch::Tensor gemm(const torch::Tensor& A, const torch::Tensor& B, float alpha, float beta) {
  TORCH_CHECK(A.is_cuda(), "A must be CUDA tensor");
  TORCH_CHECK(B.is_cuda(), "B must be CUDA tensor");
  TORCH_CHECK(A.dtype() == B.dtype(), "A and B must have the same dtype");
  switch (A.scalar_type()) {
    case torch::kFloat32: return sgemm(A, B, alpha, beta);
    case torch::kFloat16: return hgemm(A, B, alpha, beta);
    default: TORCH_CHECK(false, "Unsupported dtype for gemm: ", A.dtype());
  }
}

namespace {
void check_attn_inputs(const torch::Tensor& Q, const torch::Tensor& K, const torch::Tensor& V) {
  TORCH_CHECK(Q.is_cuda() && K.is_cuda() && V.is_cuda(), "All tensors must be CUDA tensors");
  TORCH_CHECK(Q.dtype() == torch::kHalf && K.dtype() == torch::kHalf && V.dtype() == torch::kHalf,
              "All tensors must be half");
  TORCH_CHECK(Q.dim() == 4 && K.dim() == 4 && V.dim() == 4, "All tensors must be 4D");
  TORCH_CHECK(Q.sizes() == K.sizes() && Q.sizes() == V.sizes(),
              "query, key and value must have the same shape [B, H, S, D]");
}

std::tuple<torch::Tensor, torch::Tensor> attn_impl(const torch::Tensor& query,
                                                   const torch::Tensor& key,
                                                   const torch::Tensor& value, bool want_lse,
                                                   bool causal) {
  check_attn_inputs(query, key, value);
  const c10::cuda::CUDAGuard guard(query.device());
  auto Q = query.contiguous(), K = key.contiguous(), V = value.contiguous();
  const int64_t B = Q.size(0), H = Q.size(1), S = Q.size(2), D = Q.size(3);
  auto O = torch::empty({B, H, S, D}, Q.options());
  torch::Tensor L;
  if (want_lse) L = torch::empty({B, H, S}, Q.options().dtype(torch::kFloat32));
  half* q = reinterpret_cast<half*>(Q.data_ptr<at::Half>());
  half* k = reinterpret_cast<half*>(K.data_ptr<at::Half>());
  half* v = reinterpret_cast<half*>(V.data_ptr<at::Half>());
  half* o = reinterpret_cast<half*>(O.data_ptr<at::Half>());
  float* l = want_lse ? L.data_ptr<float>() : nullptr;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  felix::FelixStatus status;
  switch (D) {
    case 64:
      status = (want_lse || causal)
                   ? felix::flash_attn_fwd_lse_launch<64, 64>(q, k, v, o, l, uint32_t(H),
                                                              uint32_t(B), uint32_t(S), stream,
                                                              causal)
                        : felix::ampere_flash_attn_launch<64, 64>(q, k, v, o, uint32_t(H),
                                                                  uint32_t(B), uint32_t(S), stream);
      break;
    case 128:
      status = (want_lse || causal)
                   ? felix::flash_attn_fwd_lse_launch<128, 64>(q, k, v, o, l, uint32_t(H),
                                                               uint32_t(B), uint32_t(S), stream,
                                                               causal)
                   : felix::ampere_flash_attn_launch<128, 64>(q, k, v, o, uint32_t(H),
                                                              uint32_t(B), uint32_t(S), stream);
      break;
    default: TORCH_CHECK(false, "flash_attention: unsupported head dimension ", D);
  }
  TORCH_CHECK(status.ok(), "flash_attention: kernel launch failed: ", status.str());
  return {O, L};
}
}  // namespace

torch::Tensor flash_attention(const torch::Tensor& query, const torch::Tensor& key,
                              const torch::Tensor& value) {
  return std::get<0>(attn_impl(query, key, value, false, false));
}

torch::Tensor flash_attention(const torch::Tensor& query, const torch::Tensor& key,
                              const torch::Tensor& value, bool causal) {
  return std::get<0>(attn_impl(query, key, value, false, causal));
}

std::tuple<torch::Tensor, torch::Tensor> flash_attention_lse(const torch::Tensor& query,
                                                             const torch::Tensor& key,
                                                             const torch::Tensor& value,
                                                             bool causal) {
  return attn_impl(query, key, value, true, causal);
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> flash_attention_backward(
    const torch::Tensor& query, const torch::Tensor& key, const torch::Tensor& value,
    const torch::Tensor& out, const torch::Tensor& lse, const torch::Tensor& grad_out,
    bool causal) {
  check_attn_inputs(query, key, value);
  TORCH_CHECK(out.sizes() == query.sizes() && grad_out.sizes() == query.sizes(),
              "out and grad_out must have the shape of query");
  TORCH_CHECK(out.dtype() == torch::kHalf && grad_out.dtype() == torch::kHalf,
              "out and grad_out must be half");
  TORCH_CHECK(out.is_cuda() && grad_out.is_cuda() && lse.is_cuda(), "All tensors must be CUDA tensors");
  const int64_t B = query.size(0), H = query.size(1), S = query.size(2), D = query.size(3);
  TORCH_CHECK(lse.dtype() == torch::kFloat32 && lse.dim() == 3 && lse.size(0) == B &&
                  lse.size(1) == H && lse.size(2) == S,
              "lse must be float32 [B, H, S]");
  const c10::cuda::CUDAGuard guard(query.device());
  auto Q = query.contiguous(), K = key.contiguous(), V = value.contiguous();
  auto O = out.contiguous(), G = grad_out.contiguous(), L = lse.contiguous();
  auto dQ = torch::empty_like(Q), dK = torch::empty_like(Q), dV = torch::empty_like(Q);
  auto hp = [](const torch::Tensor& t) { return reinterpret_cast<half*>(t.data_ptr<at::Half>()); };
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  felix::FelixStatus status;
  switch (D) {
    case 64:
      status = felix::flash_attn_bwd_launch<64>(hp(Q), hp(K), hp(V), hp(O), hp(G),
                                                L.data_ptr<float>(), hp(dQ), hp(dK), hp(dV),
                                                uint32_t(H), uint32_t(B), uint32_t(S), stream,
                                                causal);
      break;
    case 128:
      status = felix::flash_attn_bwd_launch<128>(hp(Q), hp(K), hp(V), hp(O), hp(G),
                                                 L.data_ptr<float>(), hp(dQ), hp(dK), hp(dV),
                                                 uint32_t(H), uint32_t(B), uint32_t(S), stream,
                                                 causal);
      break;
    default: TORCH_CHECK(false, "flash_attention_backward: unsupported head dimension ", D);
  }
  TORCH_CHECK(status.ok(), "flash_attention_backward: kernel launch failed: ", status.str());
  return {dQ, dK, dV};
}

// ------------------------------------------------- decoding: cache and sampling
namespace {
using OptTensor = std::optional<torch::Tensor>;

void check_i32(const torch::Tensor& t, const torch::Device& dev, int64_t dim, const char* name) {
  TORCH_CHECK(t.device() == dev, name, " must be on ", dev);
  TORCH_CHECK(t.dtype() == torch::kInt32, name, " must be int32");
  TORCH_CHECK(t.dim() == dim, name, " must be ", dim, "D");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}
const int32_t* i32(const torch::Tensor& t) { return t.data_ptr<int32_t>(); }
// A size as the C ABI takes it: what does not fit is refused, not cut off.
constexpr int64_t kMostSlots = 1 << 24, kMostInt = 0x7fffffff, kMostHeads = 65535;
uint32_t u32(int64_t n, int64_t most, const char* what) {
  TORCH_CHECK(n <= most, what, " must be at most ", most);
  return uint32_t(n);
}
const int32_t* counts_of(const OptTensor& counts, const torch::Tensor& lens) {
  if (!counts) return nullptr;
  check_i32(*counts, lens.device(), 1, "counts");
  TORCH_CHECK(counts->size(0) == lens.size(0), "counts must have one entry per slot");
  return i32(*counts);
}

felix::Kv4Cache cache_of(const torch::Tensor& pages, const torch::Tensor& table,
                         const torch::Tensor& lens, int64_t kv_heads, int64_t head_dim) {
  TORCH_CHECK(pages.is_cuda(), "pages must be CUDA tensor");
  TORCH_CHECK(pages.dtype() == torch::kUInt8 && pages.dim() == 2 && pages.is_contiguous(),
              "pages must be contiguous uint8 [pages, page bytes]");
  check_i32(table, pages.device(), 2, "table");
  check_i32(lens, pages.device(), 1, "lens");
  TORCH_CHECK(table.size(0) == lens.size(0), "table and lens must have the same slots");
  TORCH_CHECK(kv_heads > 0, "kv_heads must be positive");
  const uint32_t heads = u32(kv_heads, kMostHeads, "kv_heads");
  TORCH_CHECK(head_dim == 64 || head_dim == 128, "unsupported head dimension ", head_dim);
  const int64_t token = kv_heads * (head_dim + 8);
  TORCH_CHECK(pages.size(1) > 0 && pages.size(1) % token == 0,
              "a page's bytes must be page_size * kv_heads * (head_dim + 8)");
  return {pages.data_ptr(),
          uint64_t(pages.size(0)),
          u32(pages.size(1) / token, kMostInt, "page_size"),
          heads,
          uint32_t(head_dim),
          i32(table),
          i32(lens),
          u32(table.size(0), kMostSlots, "slots"),
          u32(table.size(1), kMostInt, "table's width")};
}

felix::ElementType half_type(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(t.dtype() == torch::kHalf || t.dtype() == torch::kBFloat16, name,
              " must be float16 or bfloat16");
  return t.dtype() == torch::kHalf ? felix::ElementType::F16 : felix::ElementType::BF16;
}

// Strides are passed on; only the innermost dimension has to be contiguous.
torch::Tensor inner_contiguous(const torch::Tensor& t) {
  return t.size(3) == 1 || t.stride(3) == 1 ? t : t.contiguous();
}

std::tuple<torch::Tensor, torch::Tensor> kv4_attention_impl(
    const torch::Tensor& query, const torch::Tensor& pages, const torch::Tensor& table,
    const torch::Tensor& lens, int64_t kv_heads, const OptTensor& counts, double scale,
    bool want_lse) {
  TORCH_CHECK(query.is_cuda(), "query must be CUDA tensor");
  TORCH_CHECK(query.dim() == 4, "query must be 4D [slots, heads, rows, D]");
  const auto type = half_type(query, "query");
  const auto cache = cache_of(pages, table, lens, kv_heads, query.size(3));
  TORCH_CHECK(query.device() == pages.device(), "query must be on ", pages.device());
  TORCH_CHECK(query.size(0) == table.size(0), "query must have one entry per slot");
  TORCH_CHECK(query.size(1) > 0 && query.size(1) % kv_heads == 0,
              "query's heads must be a multiple of kv_heads");
  const uint32_t heads = u32(query.size(1), kMostHeads, "heads");
  const uint32_t rows = u32(query.size(2), kMostHeads, "rows");
  const int32_t* n = counts_of(counts, lens);
  const c10::cuda::CUDAGuard guard(query.device());
  const auto Q = inner_contiguous(query);
  auto O = torch::empty(Q.sizes(), Q.options());
  torch::Tensor L;
  if (want_lse) L = torch::empty(Q.sizes().slice(0, 3), Q.options().dtype(torch::kFloat32));
  const auto status = felix::kv4_attention_launch(
      cache, Q.data_ptr(), type, heads, rows, Q.strides().data(), n,
      float(scale), O.data_ptr(), want_lse ? L.data_ptr<float>() : nullptr,
      at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(status.ok(), "kv4_attention: kernel launch failed: ", status.str());
  return {O, L};
}

// Straight from the allocator: a page operation returns four small tensors, and the
// dispatcher would take longer over them than the GPU over the operation.
torch::Tensor empty_i32(at::IntArrayRef sizes, const torch::Device& dev) {
  return at::Tensor(at::detail::empty_cuda(sizes, torch::kInt32, dev, std::nullopt));
}

// Outputs of a page operation: `out`, or new tensors of the inputs' shapes.
template <size_t N>
std::array<torch::Tensor, N> page_outputs(const std::array<const torch::Tensor*, N>& in,
                                          const Kv4Out& out) {
  std::array<torch::Tensor, N> r;
  if (out) TORCH_CHECK(out->size() == N, "out must have ", N, " tensors");
  for (size_t i = 0; i < N; ++i) {
    if (!out) {
      r[i] = empty_i32(in[i]->sizes(), in[i]->device());
      continue;
    }
    const auto& t = (*out)[i];
    check_i32(t, in[i]->device(), in[i]->dim(), "out");
    TORCH_CHECK(t.sizes() == in[i]->sizes(), "out must have the inputs' shapes");
    r[i] = t;
  }
  return r;
}

void check_state(const torch::Tensor& table, const torch::Tensor* lens, const torch::Tensor& refs) {
  TORCH_CHECK(table.is_cuda(), "table must be CUDA tensor");
  check_i32(table, table.device(), 2, "table");
  check_i32(refs, table.device(), 1, "refs");
  u32(table.size(0), kMostSlots, "slots");
  u32(table.size(1), kMostInt, "table's width");
  u32(refs.size(0), kMostInt, "pages");
  if (!lens) return;
  check_i32(*lens, table.device(), 1, "lens");
  TORCH_CHECK(table.size(0) == lens->size(0), "table and lens must have the same slots");
}
felix::Kv4Pages pages_of(const torch::Tensor& table, const torch::Tensor* lens,
                         const torch::Tensor& refs) {
  return {table.data_ptr<int32_t>(), lens ? lens->data_ptr<int32_t>() : nullptr,
          refs.data_ptr<int32_t>()};
}
void check_pool(const torch::Tensor& pages, const torch::Tensor& refs) {
  TORCH_CHECK(pages.device() == refs.device() && pages.dtype() == torch::kUInt8 &&
                  pages.dim() == 2 && pages.is_contiguous(),
              "pages must be contiguous uint8 [pages, page bytes]");
  TORCH_CHECK(pages.size(0) == refs.size(0), "refs must have one entry per page");
}
uint32_t page_size_of(int64_t page_size) {
  TORCH_CHECK(page_size >= 16 && page_size <= 4096 && (page_size & (page_size - 1)) == 0,
              "page_size must be a power of two, 16..4096");
  return uint32_t(page_size);
}
}  // namespace

int64_t kv4_page_bytes(int64_t kv_heads, int64_t head_dim, int64_t page_size) {
  TORCH_CHECK(kv_heads > 0, "kv_heads must be positive");
  TORCH_CHECK(head_dim == 64 || head_dim == 128, "unsupported head dimension ", head_dim);
  return int64_t(felix::kv4_page_bytes(u32(kv_heads, kMostHeads, "kv_heads"), uint32_t(head_dim),
                                       page_size_of(page_size)));
}

void kv4_append(const torch::Tensor& pages, const torch::Tensor& table, const torch::Tensor& lens,
                const torch::Tensor& key, const torch::Tensor& value, const OptTensor& counts) {
  TORCH_CHECK(key.dim() == 4 && key.sizes() == value.sizes(),
              "key and value must have the same shape [slots, kv_heads, rows, D]");
  const auto type = half_type(key, "key");
  TORCH_CHECK(value.dtype() == key.dtype(), "key and value must have the same dtype");
  const auto cache = cache_of(pages, table, lens, key.size(1), key.size(3));
  TORCH_CHECK(key.device() == pages.device() && value.device() == pages.device(),
              "key and value must be on ", pages.device());
  TORCH_CHECK(key.size(0) == table.size(0), "key must have one entry per slot");
  const uint32_t rows = u32(key.size(2), kMostInt, "rows");
  const int32_t* n = counts_of(counts, lens);
  const c10::cuda::CUDAGuard guard(pages.device());
  const auto K = inner_contiguous(key), V = inner_contiguous(value);
  const auto status = felix::kv4_append_launch(
      cache, K.data_ptr(), V.data_ptr(), type, rows, K.strides().data(),
      V.strides().data(), n, at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(status.ok(), "kv4_append: kernel launch failed: ", status.str());
}

std::tuple<torch::Tensor, torch::Tensor> kv4_read(const torch::Tensor& pages,
                                                  const torch::Tensor& table,
                                                  const torch::Tensor& lens, int64_t rows,
                                                  int64_t kv_heads, int64_t head_dim,
                                                  const OptTensor& counts) {
  TORCH_CHECK(rows >= 0 && rows <= 0x7fffffff, "rows must be 0..2^31-1");
  const auto cache = cache_of(pages, table, lens, kv_heads, head_dim);
  const int32_t* n = counts_of(counts, lens);
  const c10::cuda::CUDAGuard guard(pages.device());
  const auto opt = pages.options().dtype(torch::kHalf);
  auto K = torch::empty({table.size(0), kv_heads, rows, head_dim}, opt);
  auto V = torch::empty_like(K);
  if (K.numel() == 0) return {K, V};
  const auto status = felix::kv4_read_launch(
      cache, uint32_t(rows), n, reinterpret_cast<half*>(K.data_ptr<at::Half>()),
      reinterpret_cast<half*>(V.data_ptr<at::Half>()), at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(status.ok(), "kv4_read: kernel launch failed: ", status.str());
  return {K, V};
}

torch::Tensor kv4_attention(const torch::Tensor& query, const torch::Tensor& pages,
                            const torch::Tensor& table, const torch::Tensor& lens, int64_t kv_heads,
                            const OptTensor& counts, double scale) {
  return std::get<0>(
      kv4_attention_impl(query, pages, table, lens, kv_heads, counts, scale, false));
}

std::tuple<torch::Tensor, torch::Tensor> kv4_attention_lse(
    const torch::Tensor& query, const torch::Tensor& pages, const torch::Tensor& table,
    const torch::Tensor& lens, int64_t kv_heads, const OptTensor& counts, double scale) {
  return kv4_attention_impl(query, pages, table, lens, kv_heads, counts, scale, true);
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> kv4_reserve(
    const torch::Tensor& table, const torch::Tensor& lens, const torch::Tensor& refs,
    const torch::Tensor& counts, int64_t page_size, const Kv4Out& out) {
  check_state(table, &lens, refs);
  const int32_t* n = counts_of(counts, lens);
  const uint32_t size = page_size_of(page_size);
  const c10::cuda::CUDAGuard guard(table.device());
  const auto o = page_outputs<3>({&table, &lens, &refs}, out);
  auto report = empty_i32({2}, lens.device());
  const auto status = felix::kv4_reserve_launch(
      pages_of(table, &lens, refs), n, uint32_t(table.size(0)), uint32_t(table.size(1)),
      uint32_t(refs.size(0)), size, pages_of(o[0], &o[1], o[2]), report.data_ptr<int32_t>(),
      at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(status.ok(), "kv4_reserve: kernel launch failed: ", status.str());
  return {o[0], o[1], o[2], report};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> kv4_fork(
    const torch::Tensor& pages, const torch::Tensor& table, const torch::Tensor& lens,
    const torch::Tensor& refs, const torch::Tensor& parents, const torch::Tensor& children,
    int64_t page_size, const Kv4Out& out) {
  check_state(table, &lens, refs);
  check_pool(pages, refs);
  check_i32(parents, table.device(), 1, "parents");
  check_i32(children, table.device(), 1, "children");
  TORCH_CHECK(parents.size(0) == children.size(0), "parents and children must have the same length");
  const uint32_t size = page_size_of(page_size);
  const c10::cuda::CUDAGuard guard(table.device());
  const auto o = page_outputs<3>({&table, &lens, &refs}, out);
  auto report = empty_i32({2}, lens.device());
  const auto status = felix::kv4_fork_launch(
      pages.data_ptr(), size_t(pages.size(1)), pages_of(table, &lens, refs), i32(parents),
      i32(children), u32(parents.size(0), kMostSlots, "pairs"), uint32_t(table.size(0)),
      uint32_t(table.size(1)),
      uint32_t(refs.size(0)), size, pages_of(o[0], &o[1], o[2]), report.data_ptr<int32_t>(),
      at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(status.ok(), "kv4_fork: kernel launch failed: ", status.str());
  return {o[0], o[1], o[2], report};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> kv4_free(
    const torch::Tensor& table, const torch::Tensor& lens, const torch::Tensor& refs,
    const torch::Tensor& slots, int64_t page_size, const Kv4Out& out) {
  check_state(table, &lens, refs);
  check_i32(slots, table.device(), 1, "slots");
  const uint32_t size = page_size_of(page_size);
  const c10::cuda::CUDAGuard guard(table.device());
  const auto o = page_outputs<3>({&table, &lens, &refs}, out);
  const auto status = felix::kv4_free_launch(
      pages_of(table, &lens, refs), i32(slots), u32(slots.size(0), kMostSlots, "slots to free"),
      uint32_t(table.size(0)), uint32_t(table.size(1)), uint32_t(refs.size(0)), size, pages_of(o[0], &o[1], o[2]),
      at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(status.ok(), "kv4_free: kernel launch failed: ", status.str());
  return {o[0], o[1], o[2]};
}

std::tuple<torch::Tensor, torch::Tensor> kv4_compact(const torch::Tensor& pages,
                                                     const torch::Tensor& table,
                                                     const torch::Tensor& refs,
                                                     const Kv4Out& out) {
  check_state(table, nullptr, refs);
  check_pool(pages, refs);
  const c10::cuda::CUDAGuard guard(table.device());
  const auto o = page_outputs<2>({&table, &refs}, out);
  const auto status = felix::kv4_compact_launch(
      pages.data_ptr(), size_t(pages.size(1)), pages_of(table, nullptr, refs),
      uint32_t(table.size(0)), uint32_t(table.size(1)), uint32_t(refs.size(0)),
      pages_of(o[0], nullptr, o[1]), at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(status.ok(), "kv4_compact: kernel launch failed: ", status.str());
  return {o[0], o[1]};
}

void kv4_copy_pages(const torch::Tensor& src_pages, const torch::Tensor& dst_pages,
                    const torch::Tensor& src, const torch::Tensor& dst) {
  for (const auto* p : {&src_pages, &dst_pages})
    TORCH_CHECK(p->is_cuda() && p->dtype() == torch::kUInt8 && p->dim() == 2 && p->is_contiguous(),
                "pages must be contiguous uint8 [pages, page bytes] on a CUDA device");
  TORCH_CHECK(src_pages.device() == dst_pages.device() && src_pages.size(1) == dst_pages.size(1),
              "both pools must be on one device and have pages of the same bytes");
  check_i32(src, dst_pages.device(), 1, "src");
  check_i32(dst, dst_pages.device(), 1, "dst");
  TORCH_CHECK(src.size(0) == dst.size(0), "src and dst must have the same length");
  const c10::cuda::CUDAGuard guard(dst_pages.device());
  const auto status = felix::kv4_copy_pages_launch(
      src_pages.data_ptr(), uint64_t(src_pages.size(0)), dst_pages.data_ptr(),
      uint64_t(dst_pages.size(0)), size_t(dst_pages.size(1)), i32(src), i32(dst),
      u32(src.size(0), kMostInt, "pages to copy"), at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(status.ok(), "kv4_copy_pages: kernel launch failed: ", status.str());
}

std::tuple<torch::Tensor, torch::Tensor> sample(const torch::Tensor& logits,
                                                const torch::Tensor& uniform,
                                                const OptTensor& temperature,
                                                const OptTensor& top_k, const OptTensor& top_p,
                                                const OptTensor& min_p) {
  TORCH_CHECK(logits.is_cuda(), "logits must be CUDA tensor");
  TORCH_CHECK(logits.dim() == 2, "logits must be 2D [rows, vocab]");
  TORCH_CHECK(logits.dtype() == torch::kFloat32 || logits.dtype() == torch::kHalf ||
                  logits.dtype() == torch::kBFloat16,
              "logits must be float32, float16 or bfloat16");
  TORCH_CHECK(logits.size(1) > 0, "vocab must not be empty");
  TORCH_CHECK(logits.size(1) <= 524288, "vocab must be 1..524288");
  const int64_t rows = logits.size(0);
  u32(rows, 1 << 27, "rows");
  auto per_row = [&](const torch::Tensor& t, torch::ScalarType type, const char* name) {
    TORCH_CHECK(t.device() == logits.device(), name, " must be on ", logits.device());
    TORCH_CHECK(t.scalar_type() == type, name, " must be ", type);
    TORCH_CHECK(t.dim() == 1 && t.size(0) == rows && t.is_contiguous(), name,
                " must be contiguous with one entry per row");
  };
  auto f32 = [&](const OptTensor& t, const char* name) -> const float* {
    if (!t) return nullptr;
    per_row(*t, torch::kFloat32, name);
    return t->data_ptr<float>();
  };
  per_row(uniform, torch::kFloat32, "uniform");
  if (top_k) per_row(*top_k, torch::kInt32, "top_k");
  const float *t = f32(temperature, "temperature"), *p = f32(top_p, "top_p"),
              *m = f32(min_p, "min_p");
  const c10::cuda::CUDAGuard guard(logits.device());
  const auto X = logits.stride(1) == 1 || logits.size(1) == 1 ? logits : logits.contiguous();
  auto tokens = empty_i32({rows}, X.device());
  auto logprobs =
      at::Tensor(at::detail::empty_cuda({rows}, torch::kFloat32, X.device(), std::nullopt));
  const auto type = X.dtype() == torch::kFloat32 ? felix::ElementType::F32 : half_type(X, "logits");
  const auto status = felix::sample_launch(
      X.data_ptr(), type, uint32_t(rows), uint32_t(X.size(1)), X.stride(0),
      uniform.data_ptr<float>(), t, top_k ? i32(*top_k) : nullptr, p, m, tokens.data_ptr<int32_t>(),
      logprobs.data_ptr<float>(), at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(status.ok(), "sample: kernel launch failed: ", status.str());
  return {tokens, logprobs};
}

// ---------------------------------------------------------- feed-forward operators
namespace {
constexpr int64_t kMostFeatures = 1 << 30;

felix::Activation activation_of(const std::string& name) {
  constexpr const char* names[] = {"none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid"};
  for (int i = 0; i < 6; ++i)
    if (name == names[i]) return static_cast<felix::Activation>(i);
  TORCH_CHECK(false, "unknown activation \"", name,
              "\" (none, relu, gelu, gelu_tanh, silu, sigmoid)");
}

// A tensor as rows of contiguous elements; any leading dimensions, a copy only where the
// last one is not contiguous or the rows are not evenly spaced.
struct Rows {
  torch::Tensor t;
  int64_t rows = 0, cols = 0;
  felix::Matrix m() const { return {t.data_ptr(), t.stride(0)}; }
};
Rows rows_of(const torch::Tensor& t, const torch::Tensor& like, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be CUDA tensor");
  TORCH_CHECK(t.device() == like.device(), name, " must be on ", like.device());
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " must be ", like.scalar_type());
  TORCH_CHECK(t.dim() >= 1 && t.size(-1) > 0, name, " must have a last dimension that is not empty");
  Rows r;
  r.cols = t.size(-1);
  r.rows = t.numel() / r.cols;
  r.t = t.dim() == 2 ? t : t.reshape({r.rows, r.cols});
  if (r.cols > 1 && r.t.stride(1) != 1) r.t = r.t.contiguous();
  return r;
}
Rows weight_of(const torch::Tensor& w, const torch::Tensor& like, const char* name, int64_t rows,
               int64_t cols) {
  TORCH_CHECK(w.dim() == 2, name, " must be 2D");
  TORCH_CHECK((rows < 0 || w.size(0) == rows) && w.size(1) == cols, name, " must be [",
              rows < 0 ? std::string("out") : std::to_string(rows), ", ", cols, "]");
  TORCH_CHECK(w.size(0) > 0, name, " must not be empty");
  return rows_of(w, like, name);
}
std::vector<int64_t> with_last(const torch::Tensor& t, int64_t n) {
  auto s = t.sizes().vec();
  s.back() = n;
  return s;
}
void check_sizes(const torch::Tensor& t, const std::vector<int64_t>& s, const char* name) {
  TORCH_CHECK(t.sizes().vec() == s, name, " must have the shape ", at::IntArrayRef(s));
}
felix::Matrix out_of(const torch::Tensor& t) { return {t.data_ptr(), t.size(-1)}; }

// Scratch past this size comes from torch's allocator and goes back to it; below it the
// library keeps one per stream.
constexpr size_t kOwnScratch = size_t(32) << 20;
struct Scratch {
  torch::Tensor t;
  size_t bytes = 0;
  void* ptr() const { return bytes ? t.data_ptr() : nullptr; }
};
Scratch scratch_of(size_t need, const torch::Tensor& like) {
  if (need <= kOwnScratch) return {};
  return {torch::empty({int64_t(need)}, like.options().dtype(torch::kUInt8)), need};
}

struct LinearCall {
  felix::LinearArgs a;
  std::vector<torch::Tensor> held;  // what the arguments point into
  void hold(const Rows& r, felix::Matrix* to) {
    held.push_back(r.t);
    *to = r.m();
  }
};
LinearCall linear_call(const torch::Tensor& x, const torch::Tensor& weight,
                       const std::string& activation) {
  LinearCall c;
  TORCH_CHECK(x.is_cuda(), "x must be CUDA tensor");
  c.a.type = half_type(x, "x");
  c.a.activation = activation_of(activation);
  const Rows X = rows_of(x, x, "x");
  const Rows W = weight_of(weight, x, "weight", -1, X.cols);
  c.a.tokens = u32(X.rows, kMostFeatures, "tokens");
  c.a.in_features = u32(X.cols, kMostFeatures, "in_features");
  c.a.out_features = u32(W.rows, kMostFeatures, "out_features");
  c.hold(X, &c.a.x);
  c.hold(W, &c.a.weight);
  return c;
}

std::tuple<torch::Tensor, torch::Tensor> linear_impl(const torch::Tensor& x,
                                                     const torch::Tensor& weight,
                                                     const OptTensor& bias,
                                                     const OptTensor& residual,
                                                     const std::string& activation, bool save) {
  TORCH_CHECK(x.is_cuda(), "x must be CUDA tensor");
  const c10::cuda::CUDAGuard guard(x.device());
  LinearCall c = linear_call(x, weight, activation);
  const auto shape = with_last(x, c.a.out_features);
  if (bias) {
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == weight.size(0),
                "bias must have one entry per output feature");
    const Rows b = rows_of(*bias, x, "bias");
    c.held.push_back(b.t);
    c.a.bias = b.t.data_ptr();
  }
  if (residual) {
    check_sizes(*residual, shape, "residual");
    c.hold(rows_of(*residual, x, "residual"), &c.a.residual);
  }
  auto y = torch::empty(shape, x.options());
  torch::Tensor pre;
  c.a.out = out_of(y);
  if (save) {
    pre = torch::empty(shape, x.options());
    c.a.pre = out_of(pre);
  }
  size_t need = 0;
  auto status = felix::linear_workspace_size(c.a, false, &need);
  TORCH_CHECK(status.ok(), "linear: ", status.str());
  const Scratch s = scratch_of(need, x);
  status = felix::linear_launch(c.a, at::cuda::getCurrentCUDAStream(), s.ptr(), s.bytes);
  TORCH_CHECK(status.ok(), "linear: kernel launch failed: ", status.str());
  return {y, pre};
}

struct GatedCall {
  felix::GatedArgs a;
  std::vector<torch::Tensor> held;
  void hold(const Rows& r, felix::Matrix* to) {
    held.push_back(r.t);
    *to = r.m();
  }
};
GatedCall gated_call(const torch::Tensor& x, const torch::Tensor& w_gate, const torch::Tensor& w_up,
                     const torch::Tensor* w_down, const std::string& activation) {
  GatedCall c;
  TORCH_CHECK(x.is_cuda(), "x must be CUDA tensor");
  c.a.type = half_type(x, "x");
  c.a.activation = activation_of(activation);
  const Rows X = rows_of(x, x, "x");
  const Rows G = weight_of(w_gate, x, "w_gate", -1, X.cols);
  const Rows U = weight_of(w_up, x, "w_up", G.rows, X.cols);
  c.a.tokens = u32(X.rows, kMostFeatures, "tokens");
  c.a.features = u32(X.cols, kMostFeatures, "features");
  c.a.hidden = u32(G.rows, kMostFeatures, "hidden");
  c.hold(X, &c.a.x);
  c.hold(G, &c.a.w_gate);
  c.hold(U, &c.a.w_up);
  if (w_down) c.hold(weight_of(*w_down, x, "w_down", X.cols, G.rows), &c.a.w_down);
  return c;
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> gated_impl(
    const torch::Tensor& x, const torch::Tensor& w_gate, const torch::Tensor& w_up,
    const torch::Tensor* w_down, const OptTensor& residual, const std::string& activation,
    bool save) {
  TORCH_CHECK(x.is_cuda(), "x must be CUDA tensor");
  const c10::cuda::CUDAGuard guard(x.device());
  GatedCall c = gated_call(x, w_gate, w_up, w_down, activation);
  const auto wide = with_last(x, c.a.hidden);
  const auto shape = w_down ? x.sizes().vec() : wide;
  if (residual) {
    check_sizes(*residual, shape, "residual");
    c.hold(rows_of(*residual, x, "residual"), &c.a.residual);
  }
  auto y = torch::empty(shape, x.options());
  c.a.out = out_of(y);
  torch::Tensor gate, up;
  if (save) {
    gate = torch::empty(wide, x.options());
    up = torch::empty(wide, x.options());
    c.a.gate = out_of(gate);
    c.a.up = out_of(up);
  }
  size_t need = 0;
  auto status = felix::gated_workspace_size(c.a, w_down != nullptr, false, &need);
  TORCH_CHECK(status.ok(), "gated feed-forward: ", status.str());
  const Scratch s = scratch_of(need, x);
  const auto stream = at::cuda::getCurrentCUDAStream();
  status = w_down ? felix::gated_ffn_launch(c.a, stream, s.ptr(), s.bytes)
                  : felix::gated_linear_launch(c.a, stream, s.ptr(), s.bytes);
  TORCH_CHECK(status.ok(), "gated feed-forward: kernel launch failed: ", status.str());
  return {y, gate, up};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> gated_backward_impl(
    const torch::Tensor& grad, const torch::Tensor& x, const torch::Tensor& w_gate,
    const torch::Tensor& w_up, const torch::Tensor* w_down, const torch::Tensor& gate,
    const torch::Tensor& up, const std::string& activation, bool need_x, bool need_weights) {
  TORCH_CHECK(x.is_cuda(), "x must be CUDA tensor");
  const c10::cuda::CUDAGuard guard(x.device());
  GatedCall c = gated_call(x, w_gate, w_up, w_down, activation);
  const auto wide = with_last(x, c.a.hidden);
  check_sizes(grad, w_down ? x.sizes().vec() : wide, "grad");
  check_sizes(gate, wide, "gate");
  check_sizes(up, wide, "up");
  c.hold(rows_of(grad, x, "grad"), &c.a.grad);
  c.hold(rows_of(gate, x, "gate"), &c.a.gate);
  c.hold(rows_of(up, x, "up"), &c.a.up);
  torch::Tensor dx, dg, du, dd;
  const auto opt = x.options();
  if (need_x) {
    dx = torch::empty(x.sizes(), opt);
    c.a.dx = out_of(dx);
  }
  if (need_weights) {
    dg = torch::empty(w_gate.sizes(), opt);
    du = torch::empty(w_up.sizes(), opt);
    c.a.dw_gate = out_of(dg);
    c.a.dw_up = out_of(du);
    if (w_down) {
      dd = torch::empty(w_down->sizes(), opt);
      c.a.dw_down = out_of(dd);
    }
  }
  size_t need = 0;
  auto status = felix::gated_workspace_size(c.a, w_down != nullptr, true, &need);
  TORCH_CHECK(status.ok(), "gated feed-forward backward: ", status.str());
  const Scratch s = scratch_of(need, x);
  const auto stream = at::cuda::getCurrentCUDAStream();
  status = w_down ? felix::gated_ffn_bwd_launch(c.a, stream, s.ptr(), s.bytes)
                  : felix::gated_linear_bwd_launch(c.a, stream, s.ptr(), s.bytes);
  TORCH_CHECK(status.ok(), "gated feed-forward backward: kernel launch failed: ", status.str());
  return {dx, dg, du, dd};
}
}  // namespace

torch::Tensor linear(const torch::Tensor& x, const torch::Tensor& weight, const OptTensor& bias,
                     const OptTensor& residual, const std::string& activation) {
  return std::get<0>(linear_impl(x, weight, bias, residual, activation, false));
}
std::tuple<torch::Tensor, torch::Tensor> linear_save(const torch::Tensor& x,
                                                     const torch::Tensor& weight,
                                                     const OptTensor& bias,
                                                     const OptTensor& residual,
                                                     const std::string& activation) {
  return linear_impl(x, weight, bias, residual, activation, true);
}
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> linear_backward(
    const torch::Tensor& grad, const torch::Tensor& x, const torch::Tensor& weight,
    const OptTensor& pre, const std::string& activation, bool bias, bool need_x,
    bool need_weight) {
  TORCH_CHECK(x.is_cuda(), "x must be CUDA tensor");
  const c10::cuda::CUDAGuard guard(x.device());
  LinearCall c = linear_call(x, weight, activation);
  const auto shape = with_last(x, c.a.out_features);
  check_sizes(grad, shape, "grad");
  c.hold(rows_of(grad, x, "grad"), &c.a.grad);
  if (c.a.activation != felix::Activation::None) {
    TORCH_CHECK(pre, "pre (from linear_save) is needed for the backward pass of ", activation);
    check_sizes(*pre, shape, "pre");
    c.hold(rows_of(*pre, x, "pre"), &c.a.pre);
  }
  torch::Tensor dx, dw, db;
  const auto opt = x.options();
  if (need_x) {
    dx = torch::empty(x.sizes(), opt);
    c.a.dx = out_of(dx);
  }
  if (need_weight) {
    dw = torch::empty(weight.sizes(), opt);
    c.a.dweight = out_of(dw);
  }
  if (bias) {
    db = torch::empty({weight.size(0)}, opt);
    c.a.dbias = db.data_ptr();
  }
  size_t need = 0;
  auto status = felix::linear_workspace_size(c.a, true, &need);
  TORCH_CHECK(status.ok(), "linear_backward: ", status.str());
  const Scratch s = scratch_of(need, x);
  status = felix::linear_bwd_launch(c.a, at::cuda::getCurrentCUDAStream(), s.ptr(), s.bytes);
  TORCH_CHECK(status.ok(), "linear_backward: kernel launch failed: ", status.str());
  return {dx, dw, db};
}

torch::Tensor gated_linear(const torch::Tensor& x, const torch::Tensor& w_gate,
                           const torch::Tensor& w_up, const std::string& activation) {
  return std::get<0>(gated_impl(x, w_gate, w_up, nullptr, std::nullopt, activation, false));
}
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> gated_linear_save(
    const torch::Tensor& x, const torch::Tensor& w_gate, const torch::Tensor& w_up,
    const std::string& activation) {
  return gated_impl(x, w_gate, w_up, nullptr, std::nullopt, activation, true);
}
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> gated_linear_backward(
    const torch::Tensor& grad, const torch::Tensor& x, const torch::Tensor& w_gate,
    const torch::Tensor& w_up, const torch::Tensor& gate, const torch::Tensor& up,
    const std::string& activation, bool need_x, bool need_weights) {
  auto r = gated_backward_impl(grad, x, w_gate, w_up, nullptr, gate, up, activation, need_x,
                               need_weights);
  return {std::get<0>(r), std::get<1>(r), std::get<2>(r)};
}
torch::Tensor gated_ffn(const torch::Tensor& x, const torch::Tensor& w_gate,
                        const torch::Tensor& w_up, const torch::Tensor& w_down,
                        const OptTensor& residual, const std::string& activation) {
  return std::get<0>(gated_impl(x, w_gate, w_up, &w_down, residual, activation, false));
}
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> gated_ffn_save(
    const torch::Tensor& x, const torch::Tensor& w_gate, const torch::Tensor& w_up,
    const torch::Tensor& w_down, const OptTensor& residual, const std::string& activation) {
  return gated_impl(x, w_gate, w_up, &w_down, residual, activation, true);
}
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> gated_ffn_backward(
    const torch::Tensor& grad, const torch::Tensor& x, const torch::Tensor& w_gate,
    const torch::Tensor& w_up, const torch::Tensor& w_down, const torch::Tensor& gate,
    const torch::Tensor& up, const std::string& activation, bool need_x, bool need_weights) {
  return gated_backward_impl(grad, x, w_gate, w_up, &w_down, gate, up, activation, need_x,
                             need_weights);
}

}  // namespace sion

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  namespace py = pybind11;
  m.doc() = "Sion operators on sm_100a (tcgen05 HGEMM / flash attention, FFMA SGEMM)";
  m.def("sgemm", &sion::sgemm, "fp32 GEMM: alpha * A @ B + beta * C", py::arg("A"), py::arg("B"),
        py::arg("alpha") = 1.0f, py::arg("beta") = 0.0f);
  m.def("hgemm", &sion::hgemm, "fp16 GEMM, B stored K x N", py::arg("A"), py::arg("B"),
        py::arg("alpha") = 1.0f, py::arg("beta") = 0.0f);
  m.def("hgemm_nt", &sion::hgemm_nt, "fp16 GEMM, B stored N x K", py::arg("A"), py::arg("B"),
        py::arg("alpha") = 1.0f, py::arg("beta") = 0.0f);
  m.def("gemm", &sion::gemm, "GEMM dispatching on dtype (fp32 -> sgemm, fp16 -> hgemm)",
        py::arg("A"), py::arg("B"), py::arg("alpha") = 1.0f, py::arg("beta") = 0.0f);
  m.def("flash_attention",
        py::overload_cast<const torch::Tensor&, const torch::Tensor&, const torch::Tensor&, bool>(
            &sion::flash_attention),
        "flash attention forward (causal=True: query i sees keys 0..i)", py::arg("query"),
        py::arg("key"), py::arg("value"), py::arg("causal") = false);
  m.def("flash_attention_lse", &sion::flash_attention_lse,
        "flash attention forward returning (O, fp32 LSE)", py::arg("query"), py::arg("key"),
        py::arg("value"), py::arg("causal") = false);
  m.def("flash_attention_backward", &sion::flash_attention_backward,
        "flash attention backward returning (dQ, dK, dV)", py::arg("query"), py::arg("key"),
        py::arg("value"), py::arg("out"), py::arg("lse"), py::arg("grad_out"),
        py::arg("causal") = false);
  const auto none = py::none();
  m.def("kv4_page_bytes", &sion::kv4_page_bytes, "bytes of a page of the 4-bit cache",
        py::arg("kv_heads"), py::arg("head_dim"), py::arg("page_size"));
  m.def("kv4_append", &sion::kv4_append, "write new tokens into the 4-bit cache", py::arg("pages"),
        py::arg("table"), py::arg("lens"), py::arg("key"), py::arg("value"),
        py::arg("counts") = none);
  m.def("kv4_read", &sion::kv4_read, "the last tokens of each slot as fp16 (K, V)",
        py::arg("pages"), py::arg("table"), py::arg("lens"), py::arg("rows"), py::arg("kv_heads"),
        py::arg("head_dim"), py::arg("counts") = none);
  m.def("kv4_attention", &sion::kv4_attention, "attention of new tokens over the 4-bit cache",
        py::arg("query"), py::arg("pages"), py::arg("table"), py::arg("lens"), py::arg("kv_heads"),
        py::arg("counts") = none, py::arg("scale") = 0.0);
  m.def("kv4_attention_lse", &sion::kv4_attention_lse, "kv4_attention returning (O, fp32 LSE)",
        py::arg("query"), py::arg("pages"), py::arg("table"), py::arg("lens"), py::arg("kv_heads"),
        py::arg("counts") = none, py::arg("scale") = 0.0);
  m.def("kv4_reserve", &sion::kv4_reserve, "pages for each slot's next tokens", py::arg("table"),
        py::arg("lens"), py::arg("refs"), py::arg("counts"), py::arg("page_size"),
        py::arg("out") = none);
  m.def("kv4_fork", &sion::kv4_fork, "slots that share a parent's pages", py::arg("pages"),
        py::arg("table"), py::arg("lens"), py::arg("refs"), py::arg("parents"),
        py::arg("children"), py::arg("page_size"), py::arg("out") = none);
  m.def("kv4_free", &sion::kv4_free, "empty slots", py::arg("table"), py::arg("lens"),
        py::arg("refs"), py::arg("slots"), py::arg("page_size"), py::arg("out") = none);
  m.def("kv4_compact", &sion::kv4_compact, "move the pages in use to the lowest numbers",
        py::arg("pages"), py::arg("table"), py::arg("refs"), py::arg("out") = none);
  m.def("kv4_copy_pages", &sion::kv4_copy_pages, "copy pages between pools", py::arg("src_pages"),
        py::arg("dst_pages"), py::arg("src"), py::arg("dst"));
  m.def("sample", &sion::sample, "one token per row of logits (tokens, log-probabilities)",
        py::arg("logits"), py::arg("uniform"), py::arg("temperature") = none,
        py::arg("top_k") = none, py::arg("top_p") = none, py::arg("min_p") = none);
  m.def("linear", &sion::linear, "act(x weight^T + bias) + residual", py::arg("x"),
        py::arg("weight"), py::arg("bias") = none, py::arg("residual") = none,
        py::arg("activation") = "none");
  m.def("linear_save", &sion::linear_save, "linear returning (y, what the activation was given)",
        py::arg("x"), py::arg("weight"), py::arg("bias") = none, py::arg("residual") = none,
        py::arg("activation") = "none");
  m.def("linear_backward", &sion::linear_backward, "gradients of linear (dx, dweight, dbias)",
        py::arg("grad"), py::arg("x"), py::arg("weight"), py::arg("pre") = none,
        py::arg("activation") = "none", py::arg("bias") = false, py::arg("need_x") = true,
        py::arg("need_weight") = true);
  m.def("gated_linear", &sion::gated_linear, "act(x w_gate^T) * (x w_up^T)", py::arg("x"),
        py::arg("w_gate"), py::arg("w_up"), py::arg("activation") = "silu");
  m.def("gated_linear_save", &sion::gated_linear_save, "gated_linear returning (h, gate, up)",
        py::arg("x"), py::arg("w_gate"), py::arg("w_up"), py::arg("activation") = "silu");
  m.def("gated_linear_backward", &sion::gated_linear_backward,
        "gradients of gated_linear (dx, dw_gate, dw_up)", py::arg("grad"), py::arg("x"),
        py::arg("w_gate"), py::arg("w_up"), py::arg("gate"), py::arg("up"),
        py::arg("activation") = "silu", py::arg("need_x") = true, py::arg("need_weights") = true);
  m.def("gated_ffn", &sion::gated_ffn, "gated_linear, the down projection and a residual",
        py::arg("x"), py::arg("w_gate"), py::arg("w_up"), py::arg("w_down"),
        py::arg("residual") = none, py::arg("activation") = "silu");
  m.def("gated_ffn_save", &sion::gated_ffn_save, "gated_ffn returning (y, gate, up)", py::arg("x"),
        py::arg("w_gate"), py::arg("w_up"), py::arg("w_down"), py::arg("residual") = none,
        py::arg("activation") = "silu");
  m.def("gated_ffn_backward", &sion::gated_ffn_backward,
        "gradients of gated_ffn (dx, dw_gate, dw_up, dw_down)", py::arg("grad"), py::arg("x"),
        py::arg("w_gate"), py::arg("w_up"), py::arg("w_down"), py::arg("gate"), py::arg("up"),
        py::arg("activation") = "silu", py::arg("need_x") = true, py::arg("need_weights") = true);
}

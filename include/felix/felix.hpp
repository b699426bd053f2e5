// felix operator API (libfelix_b200.so). The four entry points keep the
// reference's exact signatures and default kernel names
// (include/felix/felix.hpp:7-28 of the reference); the named kernels are served
// by the sm_100a kernels of this library. Additions are marked "new".
#pragma once
#include <cstdint>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <felix/status.hpp>
#include <string>

namespace felix {

FelixStatus ampere_sgemm_launch(uint32_t M, uint32_t N, uint32_t K, float alpha, float const* A,
                                float const* B, float beta, float* C, cudaStream_t stream,
                                const std::string& kernel_name = "cute_sgemm_64x64_nn");

FelixStatus ampere_hgemm_launch(uint32_t M, uint32_t N, uint32_t K, float alpha, half const* A,
                                half const* B, float beta, half* C, cudaStream_t stream,
                                const std::string& kernel_name = "cute_hgemm_128x128_nn");

// k-th largest / smallest value per slice ("sorting_radix_select" and
// "sm100_topk" both select the sm_100a radix-select kernels).
FelixStatus sorting_radix_select_launch(float const* data, float* out, uint32_t num_slices,
                                        uint32_t slice_size, uint32_t k, bool largest,
                                        cudaStream_t stream,
                                        const std::string& kernel_name = "sorting_radix_select");

template <int HEAD_DIM, int Bc = 64>
FelixStatus ampere_flash_attn_launch(half* Q, half* K, half* V, half* O, uint32_t heads,
                                     uint32_t batch_size, uint32_t QKV_seqlen,
                                     cudaStream_t stream,
                                     const std::string& kernel_name =
                                         "ampere_flash_attn_mma16168_64_1D_warp_tiling");

// new: same operator with the fp32 natural-log LSE of every query row
// ([batch, heads, seqlen]; lse may be nullptr) and an optional causal mask
// (query i attends to keys 0..i).
template <int HEAD_DIM, int Bc = 64>
FelixStatus flash_attn_fwd_lse_launch(half* Q, half* K, half* V, half* O, float* lse,
                                      uint32_t heads, uint32_t batch_size, uint32_t QKV_seqlen,
                                      cudaStream_t stream, bool causal = false);

// new: attention backward. Given Q, K, V, the forward output O and its LSE
// (from flash_attn_fwd_lse_launch) and dO, writes dQ, dK, dV (all fp16
// [batch, heads, seqlen, HEAD_DIM]). Library-owned fp32 scratch (dQ
// accumulator, per-row dO.O) is allocated on first use per device and stream.
// No reference counterpart: the reference has a forward operator only.
template <int HEAD_DIM>
FelixStatus flash_attn_bwd_launch(const half* Q, const half* K, const half* V, const half* O,
                                  const half* dO, const float* lse, half* dQ, half* dK, half* dV,
                                  uint32_t heads, uint32_t batch_size, uint32_t QKV_seqlen,
                                  cudaStream_t stream, bool causal = false);

// new: the 4-bit paged cache of keys and values, its attention and its pages,
// and token sampling (felix_c.h describes the arguments). No reference
// counterpart: the reference has no cache and no sampling.
enum class ElementType : int { F16 = 0, BF16 = 1, F32 = 2 };

struct Kv4Cache {
  void* pages;
  uint64_t num_pages;
  uint32_t page_size, kv_heads, head_dim;
  const int32_t* table;  // [slots, width]
  const int32_t* lens;   // [slots]
  uint32_t slots, width;
};

// Bytes of a page; 0 where the sizes are not supported.
size_t kv4_page_bytes(uint32_t kv_heads, uint32_t head_dim, uint32_t page_size);

FelixStatus kv4_append_launch(const Kv4Cache& cache, const void* key, const void* value,
                              ElementType type, uint32_t rows, const int64_t key_strides[3],
                              const int64_t value_strides[3], const int32_t* counts,
                              cudaStream_t stream);
FelixStatus kv4_read_launch(const Kv4Cache& cache, uint32_t rows, const int32_t* counts, half* key,
                            half* value, cudaStream_t stream);
FelixStatus kv4_attention_launch(const Kv4Cache& cache, const void* q, ElementType type,
                                 uint32_t heads, uint32_t rows, const int64_t q_strides[3],
                                 const int32_t* counts, float scale, void* out, float* lse,
                                 cudaStream_t stream);

// State of a pool's pages: table [slots, width], lens [slots], refs [num_pages].
struct Kv4Pages {
  int32_t *table, *lens, *refs;
};
FelixStatus kv4_reserve_launch(const Kv4Pages& in, const int32_t* counts, uint32_t slots,
                               uint32_t width, uint32_t num_pages, uint32_t page_size,
                               const Kv4Pages& out, int32_t* status, cudaStream_t stream);
FelixStatus kv4_fork_launch(void* pages, size_t page_bytes, const Kv4Pages& in,
                            const int32_t* parents, const int32_t* children, uint32_t n,
                            uint32_t slots, uint32_t width, uint32_t num_pages, uint32_t page_size,
                            const Kv4Pages& out, int32_t* status, cudaStream_t stream);
FelixStatus kv4_free_launch(const Kv4Pages& in, const int32_t* list, uint32_t n, uint32_t slots,
                            uint32_t width, uint32_t num_pages, uint32_t page_size,
                            const Kv4Pages& out, cudaStream_t stream);
FelixStatus kv4_compact_launch(void* pages, size_t page_bytes, const Kv4Pages& in, uint32_t slots,
                               uint32_t width, uint32_t num_pages, const Kv4Pages& out,
                               cudaStream_t stream);
FelixStatus kv4_copy_pages_launch(const void* from, uint64_t from_pages, void* to,
                                  uint64_t to_pages, size_t page_bytes, const int32_t* src,
                                  const int32_t* dst, uint32_t n, cudaStream_t stream);

FelixStatus sample_launch(const void* logits, ElementType type, uint32_t rows, uint32_t vocab,
                          int64_t stride, const float* uniform, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p,
                          int32_t* tokens, float* logprobs, cudaStream_t stream);

// new: feed-forward operators, fp16 or bf16 (felix_c.h describes the arguments and the
// formulas): a linear layer with bias, activation and residual in the product's
// epilogue, and a gated block, each with its backward pass. No reference counterpart.
enum class Activation : int { None = 0, Relu = 1, Gelu = 2, GeluTanh = 3, Silu = 4, Sigmoid = 5 };

struct Matrix {
  void* data = nullptr;
  int64_t stride = 0;  // elements from a row to the next
};

struct LinearArgs {
  uint32_t tokens = 0, in_features = 0, out_features = 0;
  ElementType type = ElementType::F16;
  Activation activation = Activation::None;
  Matrix x, weight, residual;
  const void* bias = nullptr;
  Matrix out, pre;
  Matrix grad, dx, dweight;  // backward
  void* dbias = nullptr;
};

struct GatedArgs {
  uint32_t tokens = 0, features = 0, hidden = 0;
  ElementType type = ElementType::F16;
  Activation activation = Activation::Silu;
  Matrix x, w_gate, w_up, w_down, residual;
  Matrix out, gate, up;
  Matrix grad, dx, dw_gate, dw_up, dw_down;  // backward
};

// workspace: nullptr = library-owned, else *_workspace_size bytes for these arguments.
FelixStatus linear_launch(const LinearArgs& a, cudaStream_t stream, void* workspace = nullptr,
                          size_t workspace_bytes = 0);
FelixStatus linear_bwd_launch(const LinearArgs& a, cudaStream_t stream, void* workspace = nullptr,
                              size_t workspace_bytes = 0);
FelixStatus linear_workspace_size(const LinearArgs& a, bool backward, size_t* bytes);
FelixStatus gated_linear_launch(const GatedArgs& a, cudaStream_t stream, void* workspace = nullptr,
                                size_t workspace_bytes = 0);
FelixStatus gated_linear_bwd_launch(const GatedArgs& a, cudaStream_t stream,
                                    void* workspace = nullptr, size_t workspace_bytes = 0);
FelixStatus gated_ffn_launch(const GatedArgs& a, cudaStream_t stream, void* workspace = nullptr,
                             size_t workspace_bytes = 0);
FelixStatus gated_ffn_bwd_launch(const GatedArgs& a, cudaStream_t stream, void* workspace = nullptr,
                                 size_t workspace_bytes = 0);
FelixStatus gated_workspace_size(const GatedArgs& a, bool ffn, bool backward, size_t* bytes);

// new: reads (and clears) the device watchdog word; KERNEL_RUNTIME_ERROR when a
// bounded wait inside a kernel gave up. Synchronises the device.
FelixStatus check_watchdog();

}  // namespace felix

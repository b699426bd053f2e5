// sion:: LibTorch wrappers over the felix operators. Same signatures as the
// reference (include/sion/sion.hpp:4-14); flash_attention_lse is new.
#pragma once
#include <optional>
#include <string>
#include <torch/torch.h>
#include <tuple>
#include <vector>

namespace sion {

torch::Tensor flash_attention(const torch::Tensor& query, const torch::Tensor& key,
                              const torch::Tensor& value);
torch::Tensor sgemm(const torch::Tensor& A, const torch::Tensor& B, float alpha, float beta);
torch::Tensor hgemm(const torch::Tensor& A, const torch::Tensor& B, float alpha, float beta);
torch::Tensor hgemm_nt(const torch::Tensor& A, const torch::Tensor& B, float alpha, float beta);
torch::Tensor gemm(const torch::Tensor& A, const torch::Tensor& B, float alpha, float beta);

// new: causal-mask variant (query i attends to keys 0..i)
torch::Tensor flash_attention(const torch::Tensor& query, const torch::Tensor& key,
                              const torch::Tensor& value, bool causal);
// new: (O, LSE) with LSE fp32 [B, H, S]
std::tuple<torch::Tensor, torch::Tensor> flash_attention_lse(const torch::Tensor& query,
                                                             const torch::Tensor& key,
                                                             const torch::Tensor& value,
                                                             bool causal = false);
// new: gradients (dQ, dK, dV) of flash_attention given its inputs, the forward
// output O and LSE (from flash_attention_lse) and the output gradient dO
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> flash_attention_backward(
    const torch::Tensor& query, const torch::Tensor& key, const torch::Tensor& value,
    const torch::Tensor& out, const torch::Tensor& lse, const torch::Tensor& grad_out,
    bool causal = false);

// new: decoding with a 4-bit paged cache of keys and values. pages: uint8
// [pages, page bytes] (kv4_page_bytes); table: int32 [slots, pages of a slot];
// lens: int32 [slots], new tokens included; refs: int32 [pages], how many slots
// hold a page. query / key / value: fp16 or bf16 [slots, heads, rows, D], D 64
// or 128; counts (int32 [slots]): how many of the rows are tokens, all if absent.
int64_t kv4_page_bytes(int64_t kv_heads, int64_t head_dim, int64_t page_size);
void kv4_append(const torch::Tensor& pages, const torch::Tensor& table, const torch::Tensor& lens,
                const torch::Tensor& key, const torch::Tensor& value,
                const std::optional<torch::Tensor>& counts = std::nullopt);
std::tuple<torch::Tensor, torch::Tensor> kv4_read(
    const torch::Tensor& pages, const torch::Tensor& table, const torch::Tensor& lens, int64_t rows,
    int64_t kv_heads, int64_t head_dim, const std::optional<torch::Tensor>& counts = std::nullopt);
torch::Tensor kv4_attention(const torch::Tensor& query, const torch::Tensor& pages,
                            const torch::Tensor& table, const torch::Tensor& lens, int64_t kv_heads,
                            const std::optional<torch::Tensor>& counts = std::nullopt,
                            double scale = 0.0);
std::tuple<torch::Tensor, torch::Tensor> kv4_attention_lse(
    const torch::Tensor& query, const torch::Tensor& pages, const torch::Tensor& table,
    const torch::Tensor& lens, int64_t kv_heads,
    const std::optional<torch::Tensor>& counts = std::nullopt, double scale = 0.0);

// Page operations: the results are new tensors, or `out` (table, lens, refs;
// compact: table, refs), which may be the inputs themselves. status: int32
// [pages missing, list entries skipped]; where pages are missing nothing changed.
using Kv4Out = std::optional<std::vector<torch::Tensor>>;
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> kv4_reserve(
    const torch::Tensor& table, const torch::Tensor& lens, const torch::Tensor& refs,
    const torch::Tensor& counts, int64_t page_size, const Kv4Out& out = std::nullopt);
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> kv4_fork(
    const torch::Tensor& pages, const torch::Tensor& table, const torch::Tensor& lens,
    const torch::Tensor& refs, const torch::Tensor& parents, const torch::Tensor& children,
    int64_t page_size, const Kv4Out& out = std::nullopt);
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> kv4_free(
    const torch::Tensor& table, const torch::Tensor& lens, const torch::Tensor& refs,
    const torch::Tensor& slots, int64_t page_size, const Kv4Out& out = std::nullopt);
std::tuple<torch::Tensor, torch::Tensor> kv4_compact(const torch::Tensor& pages,
                                                     const torch::Tensor& table,
                                                     const torch::Tensor& refs,
                                                     const Kv4Out& out = std::nullopt);
void kv4_copy_pages(const torch::Tensor& src_pages, const torch::Tensor& dst_pages,
                    const torch::Tensor& src, const torch::Tensor& dst);

// new: one token per row of logits [rows, vocab] (fp16, bf16 or fp32) from
// uniform [rows] in [0, 1); temperature, top_p, min_p fp32 [rows], top_k int32
// [rows], each optional. Returns (tokens int32, log-probabilities fp32).
std::tuple<torch::Tensor, torch::Tensor> sample(
    const torch::Tensor& logits, const torch::Tensor& uniform,
    const std::optional<torch::Tensor>& temperature = std::nullopt,
    const std::optional<torch::Tensor>& top_k = std::nullopt,
    const std::optional<torch::Tensor>& top_p = std::nullopt,
    const std::optional<torch::Tensor>& min_p = std::nullopt);

// new: feed-forward operators in fp16 or bf16. x [..., in], weights as torch.nn.Linear
// holds them ([out, in]), activation "none", "relu", "gelu", "gelu_tanh", "silu" or
// "sigmoid". linear: act(x weight^T + bias) + residual; linear_save also returns what
// stands in front of the activation, which linear_backward takes ((dx, dweight, dbias),
// undefined where not wanted).
torch::Tensor linear(const torch::Tensor& x, const torch::Tensor& weight,
                     const std::optional<torch::Tensor>& bias = std::nullopt,
                     const std::optional<torch::Tensor>& residual = std::nullopt,
                     const std::string& activation = "none");
std::tuple<torch::Tensor, torch::Tensor> linear_save(
    const torch::Tensor& x, const torch::Tensor& weight,
    const std::optional<torch::Tensor>& bias = std::nullopt,
    const std::optional<torch::Tensor>& residual = std::nullopt,
    const std::string& activation = "none");
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> linear_backward(
    const torch::Tensor& grad, const torch::Tensor& x, const torch::Tensor& weight,
    const std::optional<torch::Tensor>& pre, const std::string& activation = "none",
    bool bias = false, bool need_x = true, bool need_weight = true);

// new: act(x w_gate^T) * (x w_up^T); *_save also return both projections; gated_ffn
// continues with w_down [in, hidden] and an optional residual.
torch::Tensor gated_linear(const torch::Tensor& x, const torch::Tensor& w_gate,
                           const torch::Tensor& w_up, const std::string& activation = "silu");
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> gated_linear_save(
    const torch::Tensor& x, const torch::Tensor& w_gate, const torch::Tensor& w_up,
    const std::string& activation = "silu");
// (dx, dw_gate, dw_up)
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> gated_linear_backward(
    const torch::Tensor& grad, const torch::Tensor& x, const torch::Tensor& w_gate,
    const torch::Tensor& w_up, const torch::Tensor& gate, const torch::Tensor& up,
    const std::string& activation = "silu", bool need_x = true, bool need_weights = true);
torch::Tensor gated_ffn(const torch::Tensor& x, const torch::Tensor& w_gate,
                        const torch::Tensor& w_up, const torch::Tensor& w_down,
                        const std::optional<torch::Tensor>& residual = std::nullopt,
                        const std::string& activation = "silu");
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> gated_ffn_save(
    const torch::Tensor& x, const torch::Tensor& w_gate, const torch::Tensor& w_up,
    const torch::Tensor& w_down, const std::optional<torch::Tensor>& residual = std::nullopt,
    const std::string& activation = "silu");
// (dx, dw_gate, dw_up, dw_down)
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> gated_ffn_backward(
    const torch::Tensor& grad, const torch::Tensor& x, const torch::Tensor& w_gate,
    const torch::Tensor& w_up, const torch::Tensor& w_down, const torch::Tensor& gate,
    const torch::Tensor& up, const std::string& activation = "silu", bool need_x = true,
    bool need_weights = true);

}  // namespace sion

/*
 * felix_c.h — C ABI of the sm_100a operator library (libfelix_b200.so).
 *
 * Plain pointers, sizes and an opaque stream handle (a cudaStream_t passed as
 * void*; NULL = legacy default stream). No C++ or torch types cross this
 * boundary. All device pointers are caller-owned; launches are asynchronous on
 * the given stream and never synchronise. Every function returns a status
 * type code that maps 1:1 onto felix::FelixStatus::Type
 * (reference: include/felix/status.hpp:10-15); the CUDA error behind a failure
 * and a readable message are kept per calling thread.
 *
 * fp16 data is passed as `const void*` / `void*` holding IEEE binary16 values.
 */
#ifndef FELIX_C_H
#define FELIX_C_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status type codes (== felix::FelixStatus::Type, include/felix/status.hpp:10-15). */
#define FELIX_SUCCESS 0
#define FELIX_KERNEL_LAUNCH_FAILED 1
#define FELIX_KERNEL_RUNTIME_ERROR 2
#define FELIX_API_ERROR 3

/* B operand storage for HGEMM. */
#define FELIX_B_KN 0 /* "nn": B stored K x N row-major (cute_hgemm_128x128_nn)        */
#define FELIX_B_NK 1 /* "nt": B stored N x K row-major, i.e. column-major K x N (_nt) */

/* CUDA error code behind the last non-success status on this thread (0 if none). */
int felix_last_cuda_error(void);
/* Human-readable message for the last non-success status on this thread. */
const char* felix_last_error_message(void);
/* Library version string. */
const char* felix_version(void);

/*
 * SGEMM, fp32 SIMT: C = alpha * A * B + beta * C.
 * A [M x K], B [K x N], C [M x N], all row-major fp32.
 * Replaces felix::ampere_sgemm_launch (reference include/felix/felix.hpp:7-10,
 * src/felix/base/felix_api.cpp:22-28; default kernel cute_sgemm_64x64_nn,
 * src/felix/gemm/sgemm/cute_sgemm_64x64_nn_kernel_launch.cu:7-63).
 * Any M, N, K (no alignment requirement). beta == 0 never reads C.
 */
int felix_sgemm(uint32_t M, uint32_t N, uint32_t K, float alpha, const float* A,
                const float* B, float beta, float* C, void* stream);

/*
 * SGEMM with explicit split-K and caller-owned workspace.
 * split_k: 0 = auto, 1 = none, n = n-way. workspace may be NULL (library-owned
 * per-stream scratch); otherwise it must hold felix_sgemm_workspace_size()
 * bytes and be zero-filled before its first use (the kernel leaves its
 * counters at zero). No reference counterpart: the reference has no split-K.
 */
int felix_sgemm_ex(uint32_t M, uint32_t N, uint32_t K, float alpha, const float* A,
                   const float* B, float beta, float* C, int split_k, void* workspace,
                   size_t workspace_bytes, void* stream);
int felix_sgemm_workspace_size(uint32_t M, uint32_t N, uint32_t K, int split_k,
                               size_t* bytes);

/*
 * SGEMM that allocates nothing. No counterpart in the reference.
 *
 * For callers that cannot call cudaMalloc from inside an operator call: hosts
 * that own all device memory through their own pool or a fixed memory budget,
 * plugin runtimes that forbid allocation in a kernel launch path, and
 * latency-critical code that cannot accept cudaMalloc's implicit device-wide
 * synchronisation. Same arithmetic and arguments as felix_sgemm_ex; the
 * split-K scratch (tile counters + fp32 partial tiles) lives in a static
 * array inside the library's device image instead of being allocated:
 *   - size: 16 MiB of partial tiles + 16 KiB of counters, held by every GPU
 *     that loads the library until the process exits;
 *   - split_k = 0 picks the largest automatic split whose partials fit;
 *     an explicit split_k > 1 with tiles x split_k > 256 (tiles =
 *     ceil(M/128) * ceil(N/128); checked on the requested split_k, before
 *     it is clamped to ceil(K/16)) is rejected with FELIX_API_ERROR;
 *   - it never falls back to an allocated workspace: a scratch that does not
 *     fit is an FELIX_API_ERROR, not a cudaMalloc;
 *   - the first call on a device looks up the scratch's device address
 *     (cudaGetSymbolAddress) for that device; make that first call before any
 *     stream capture;
 *   - each call clears the counters on `stream` before its kernel;
 *   - all calls share the one array: calls whose execution overlaps on the GPU
 *     (different streams without ordering) race and give wrong results.
 * The caller still owns A, B and C.
 */
int felix_sgemm_noalloc(uint32_t M, uint32_t N, uint32_t K, float alpha, const float* A,
                        const float* B, float beta, float* C, int split_k, void* stream);

/*
 * HGEMM, fp16 tensor cores (tcgen05, fp32 accumulate in TMEM, fp16 output):
 * C = alpha * A * op(B) + beta * C. A [M x K] row-major; B per b_layout
 * (FELIX_B_KN or FELIX_B_NK); C [M x N] row-major.
 * Replaces felix::ampere_hgemm_launch with kernel names "cute_hgemm_128x128_nn"
 * / "cute_hgemm_128x128_nt" (reference include/felix/felix.hpp:12-15,
 * src/felix/base/felix_api.cpp:30-36,
 * src/felix/gemm/hgemm/cute_hgemm_128x128_{nn,nt}_kernel_launch.cu).
 * The reference accumulates in fp16; this accumulates in fp32.
 * Requirements: K % 8 == 0; for FELIX_B_KN also N % 8 == 0; A, B 16-byte
 * aligned (C too when N % 8 == 0). M, N, K need not be tile multiples
 * (the reference requires M, N % 128 and K % 64).
 */
int felix_hgemm(uint32_t M, uint32_t N, uint32_t K, float alpha, const void* A, const void* B,
                float beta, void* C, int b_layout, void* stream);

/*
 * HGEMM with explicit schedule and caller-owned workspace (no reference
 * counterpart; the reference has no split-K / stream-K).
 * block_n: 0 auto, 64, 128 or 256. stream_k: 0 auto, 1 off, 2 on whenever the last
 * wave of tiles is incomplete. max_ctas: 0 = one persistent CTA per SM.
 * workspace: NULL = library-owned per-(device, stream) scratch; otherwise at
 * least felix_hgemm_workspace_size() bytes, zero-filled before first use. Its
 * first 16 KiB are counters (stream-K tickets; for shapes of four or more
 * waves of tiles, the counter that hands whole tiles out at run time) that
 * every launch leaves at zero, so launches that share a workspace must not
 * overlap on the GPU.
 */
int felix_hgemm_ex(uint32_t M, uint32_t N, uint32_t K, float alpha, const void* A,
                   const void* B, float beta, void* C, int b_layout, int block_n, int stream_k,
                   int max_ctas, void* workspace, size_t workspace_bytes, void* stream);
int felix_hgemm_workspace_size(uint32_t M, uint32_t N, uint32_t K, int block_n, int stream_k,
                               int max_ctas, size_t* bytes);
/*
 * felix_hgemm_ex plus cta_pair (no reference counterpart): 0 auto (pairs when
 * M, N >= 256, K >= 512 with K (and N for FELIX_B_KN) a multiple of 64, and at
 * least one wave of 256 x 256 tiles, with block_n, stream_k, max_ctas all 0),
 * 1 off, 2 = 256 x 256 tiles computed by 2-CTA clusters with cta_group::2 MMAs
 * (each CTA loads its 128 rows of A and half of the tile's B, the leader
 * issues M = 256 MMAs; block_n must be 0 or 256; K, and N for FELIX_B_KN,
 * multiples of 64). felix_hgemm and felix_hgemm_ex use the same automatic
 * choice. Workspace size from felix_hgemm_workspace_size2 with the same
 * options.
 */
int felix_hgemm_ex2(uint32_t M, uint32_t N, uint32_t K, float alpha, const void* A,
                    const void* B, float beta, void* C, int b_layout, int block_n, int stream_k,
                    int max_ctas, int cta_pair, void* workspace, size_t workspace_bytes,
                    void* stream);
int felix_hgemm_workspace_size2(uint32_t M, uint32_t N, uint32_t K, int block_n, int stream_k,
                                int max_ctas, int cta_pair, size_t* bytes);

/*
 * Flash-attention forward, fp16, no mask: O = softmax(Q K^T * scale) V per
 * (batch, head). Q, K, V, O are [batch, heads, seqlen, head_dim] contiguous
 * fp16. lse (optional, may be NULL) receives the fp32 natural-log
 * log-sum-exp of each query row, [batch, heads, seqlen].
 * scale <= 0 selects the reference's fixed 1/sqrt(head_dim).
 * Replaces felix::ampere_flash_attn_launch<HEAD_DIM, 64> (reference
 * include/felix/felix.hpp:22-28, src/felix/base/felix_api.cpp:47-68,
 * src/felix/flash_attention/ampere_flash_attn_mma16168_64_1D_warp_tiling_kernel_launch.cu:8-55),
 * which supports head_dim 64/128 and seqlen % 64 == 0 and has no LSE output.
 * Here: head_dim in {64, 128}, any seqlen >= 1.
 */
int felix_flash_attn_fwd(const void* Q, const void* K, const void* V, void* O, float* lse,
                         uint32_t heads, uint32_t batch, uint32_t seqlen, uint32_t head_dim,
                         float scale, void* stream);

/*
 * Flash-attention forward with an optional causal mask (causal != 0: query i
 * attends to keys 0..i, queries and keys aligned at position 0, as
 * scaled_dot_product_attention(is_causal=True) with equal lengths). Otherwise
 * identical to felix_flash_attn_fwd. No reference counterpart: the reference
 * kernel supports no mask (reference README.md:23).
 */
int felix_flash_attn_fwd_ex(const void* Q, const void* K, const void* V, void* O, float* lse,
                            uint32_t heads, uint32_t batch, uint32_t seqlen, uint32_t head_dim,
                            float scale, int causal, void* stream);

/*
 * Flash-attention backward (no reference counterpart; the reference has a
 * forward kernel only): given Q, K, V, the forward output O, its gradient dO
 * (all fp16 [batch, heads, seqlen, head_dim]) and the forward's fp32
 * natural-log LSE [batch, heads, seqlen], writes dQ, dK, dV (fp16, same
 * shape). scale <= 0 selects 1/sqrt(head_dim); causal as in
 * felix_flash_attn_fwd_ex. workspace: NULL = library-owned scratch, else at
 * least felix_flash_attn_bwd_workspace_size() bytes (fp32 dQ accumulator and
 * the per-row dO.O sums; its contents need no initialisation).
 */
int felix_flash_attn_bwd(const void* Q, const void* K, const void* V, const void* O,
                         const void* dO, const float* lse, void* dQ, void* dK, void* dV,
                         uint32_t heads, uint32_t batch, uint32_t seqlen, uint32_t head_dim,
                         float scale, int causal, void* workspace, size_t workspace_bytes,
                         void* stream);
int felix_flash_attn_bwd_workspace_size(uint32_t heads, uint32_t batch, uint32_t seqlen,
                                        uint32_t head_dim, size_t* bytes);

/*
 * k-th value per slice (radix select): out[s] = the k-th largest (largest != 0)
 * or k-th smallest value of data[s * slice_size, (s + 1) * slice_size), fp32,
 * returned bit-exactly (order: NaN above +inf, -0.0 below +0.0).
 * Replaces felix::sorting_radix_select_launch / "sorting_radix_select"
 * (reference include/felix/felix.hpp:17-20,
 * src/felix/topk/sorting_radix_select_kernel_launch.cu:7-38); same argument
 * rules: num_slices == 0 is a no-op, null pointers or k outside
 * [1, slice_size] are FELIX_API_ERROR.
 */
int felix_topk_select(const float* data, float* out, uint32_t num_slices, uint32_t slice_size,
                      uint32_t k, int largest, void* stream);

/*
 * 4-bit paged cache of keys and values (no reference counterpart: the
 * reference has no cache). A pool is num_pages pages of
 * felix_kv4_page_bytes() bytes; a page holds page_size tokens (a power of two,
 * 16..4096) of every key/value head. Each head vector (head_dim 64 or 128) is
 * held as x ~ base + scale * (code - 8): a code of 0..15 per value and an fp16
 * (scale, base) per token and head, (head_dim + 8) bytes for K and V together
 * (byte order: csrc/kv4_layout.cuh). `table` [slots][width] names the pages of
 * each slot in order, `lens` [slots] the tokens in it, new ones included.
 * Entries of `table` that name no page of the pool are not an error: tokens
 * there are not written, read as zero, and attention does not see them. All
 * arrays are on the device; pages is 16-byte aligned. Limits: 65535 heads, 2^24
 * slots, width * page_size and rows below 2^31 (attention: 65535 rows).
 */
typedef struct felix_kv4_cache {
  void* pages;
  uint64_t num_pages;
  uint32_t page_size, kv_heads, head_dim;
  const int32_t* table;
  const int32_t* lens;
  uint32_t slots, width;
} felix_kv4_cache;

/* Element types of the new operators' inputs. */
#define FELIX_F16 0
#define FELIX_BF16 1
#define FELIX_F32 2

int felix_kv4_page_bytes(uint32_t kv_heads, uint32_t head_dim, uint32_t page_size, size_t* bytes);

/*
 * Writes new tokens into the cache: row i (0..rows-1) of slot s is token
 * lens[s] - counts[s] + i where i < counts[s] (counts NULL: rows), other rows
 * are left out. key, value: fp16 or bf16 [slot][head][row][head_dim] with the
 * given element strides of slot, head and row (head_dim is contiguous). Per
 * vector scale = fp16((max - min) / 15), base = fp16(min + 8 scale), code =
 * clamp(rint((x - base) / scale) + 8, 0, 15). bf16 values past fp16's range are
 * held as its largest value; a vector with an infinity or a NaN reads as NaN.
 */
int felix_kv4_append(const felix_kv4_cache* cache, const void* key, const void* value, int dtype,
                     uint32_t rows, const int64_t* key_strides, const int64_t* value_strides,
                     const int32_t* counts, void* stream);
/*
 * Reads the last tokens of each slot back as fp16, [slots][kv_heads][rows]
 * [head_dim] contiguous, rows as in felix_kv4_append; rows that are no token
 * are zero.
 */
int felix_kv4_read(const felix_kv4_cache* cache, uint32_t rows, const int32_t* counts, void* key,
                   void* value, void* stream);
/*
 * Attention of new tokens over the cache (append them first): q, fp16 or bf16,
 * [slot][head][row][head_dim] with the given strides; row i of slot s, with
 * n = counts[s] (NULL: rows), sees the tokens 0 .. lens[s] - n + i. heads is a
 * multiple of the cache's kv_heads; head h reads key/value head
 * h / (heads / kv_heads). out [slots][heads][rows][head_dim] contiguous in q's
 * type; lse (may be NULL) fp32 [slots][heads][rows], natural log. Rows that see
 * nothing (i >= n, an empty slot) give zeros and lse = -inf. scale <= 0 selects
 * 1/sqrt(head_dim). workspace: NULL = library-owned per (device, stream), else
 * felix_kv4_attention_workspace_size() bytes, 16-byte aligned and zero-filled before
 * its first use. out is 8-byte aligned.
 */
int felix_kv4_attention(const felix_kv4_cache* cache, const void* q, int dtype, uint32_t heads,
                        uint32_t rows, const int64_t* q_strides, const int32_t* counts,
                        float scale, void* out, float* lse, void* workspace,
                        size_t workspace_bytes, void* stream);
int felix_kv4_attention_workspace_size(uint32_t head_dim, size_t* bytes);

/*
 * Page operations. table [slots][width], lens [slots], refs [num_pages] (how
 * many slots hold a page; <= 0: free); the *_out arrays are written whole and
 * each may be its input. Free pages are given out from the lowest number up.
 * status (reserve, fork): [0] pages that were missing (0: done; otherwise
 * nothing was changed), [1] entries of the lists that were skipped.
 *   reserve: lens grows by counts and each slot gets the pages for that (pages
 *            past a slot's width count as missing).
 *   fork:    slot children[i] becomes a copy of slot parents[i]: whole pages are
 *            shared, a last page that is not full is copied to a fresh one (where
 *            the table names no page for it, the child has none there either).
 *            Skipped: numbers out of range, a child that holds tokens, is its
 *            parent or was named before.
 *   free:    the listed slots become empty; pages that no slot holds any more
 *            are free. Numbers out of range are ignored, repeated ones count once.
 *   compact: pages in use move to the lowest numbers (the used pages past the
 *            number in use fill the free ones below it, both in ascending
 *            order), bytes included; table and refs follow.
 */
int felix_kv4_reserve(const int32_t* table, const int32_t* lens, const int32_t* refs,
                      const int32_t* counts, uint32_t slots, uint32_t width, uint32_t num_pages,
                      uint32_t page_size, int32_t* table_out, int32_t* lens_out,
                      int32_t* refs_out, int32_t* status, void* stream);
int felix_kv4_fork(void* pages, size_t page_bytes, const int32_t* table, const int32_t* lens,
                   const int32_t* refs, const int32_t* parents, const int32_t* children,
                   uint32_t n, uint32_t slots, uint32_t width, uint32_t num_pages,
                   uint32_t page_size, int32_t* table_out, int32_t* lens_out, int32_t* refs_out,
                   int32_t* status, void* stream);
int felix_kv4_free(const int32_t* table, const int32_t* lens, const int32_t* refs,
                   const int32_t* list, uint32_t n, uint32_t slots, uint32_t width,
                   uint32_t num_pages, uint32_t page_size, int32_t* table_out, int32_t* lens_out,
                   int32_t* refs_out, void* stream);
int felix_kv4_compact(void* pages, size_t page_bytes, const int32_t* table, const int32_t* refs,
                      uint32_t slots, uint32_t width, uint32_t num_pages, int32_t* table_out,
                      int32_t* refs_out, void* stream);
/*
 * Copies page src[i] of one pool to page dst[i] of another (or of the same,
 * where no page is both source and destination; dst without repeats). Numbers
 * outside their pool are left out.
 */
int felix_kv4_copy_pages(const void* from, uint64_t from_pages, void* to, uint64_t to_pages,
                         size_t page_bytes, const int32_t* src, const int32_t* dst, uint32_t n,
                         void* stream);

/*
 * Samples a token per row of logits (FELIX_F16, FELIX_BF16 or FELIX_F32,
 * [rows][vocab], `stride` elements between rows) from uniform[row] in [0, 1).
 * Per-row parameters, each may be NULL: temperature (NULL: 1; <= 0: the first
 * of the largest), top_k (NULL or <= 0: all), top_p (NULL or >= 1: all), min_p
 * (NULL or <= 0: all). With w = exp((x - max) / T) as 31-bit fixed point and
 * the order larger first, ties by lower index: top-k keeps the first k, top-p
 * those with less than p of the kept mass before them, min-p those with
 * w >= min_p, and the first always stays; the token is the first by index at
 * which the running sum of kept mass exceeds floor(uniform * total). NaN counts
 * as -inf. vocab is at most 524288. logprobs: log of the probability with which the token was drawn (0
 * where temperature <= 0). A row with nothing above -inf: -1 and -inf.
 */
int felix_sample(const void* logits, int dtype, uint32_t rows, uint32_t vocab, int64_t stride,
                 const float* uniform, const float* temperature, const int32_t* top_k,
                 const float* top_p, const float* min_p, int32_t* tokens, float* logprobs,
                 void* stream);

/*
 * Feed-forward operators (no reference counterpart: the reference has plain products
 * only). fp16 or bf16 (`dtype`) in and out, sums in fp32, everything that follows a
 * product done before its only rounding. Matrices are rows of contiguous elements,
 * `stride` elements apart (rows of an input may repeat or overlap, stride 0 included).
 * Any sizes from 1 up and any 2-byte alignment; rows that are no multiples of 16 bytes
 * (or lie at other addresses) cost a copy of that input. Optional matrices have data
 * NULL. Outputs may not overlap inputs or each other, but for `out`, which may be
 * `residual` itself. tokens == 0 leaves outputs empty and sets the weights' gradients to zero.
 *
 * Activations: relu z < 0 ? 0 : z (derivative 0 at 0), gelu z Phi(z), gelu_tanh its
 * form with tanh, silu z sigma(z), sigmoid sigma(z).
 */
#define FELIX_ACT_NONE 0
#define FELIX_ACT_RELU 1
#define FELIX_ACT_GELU 2
#define FELIX_ACT_GELU_TANH 3
#define FELIX_ACT_SILU 4
#define FELIX_ACT_SIGMOID 5

typedef struct felix_matrix {
  void* data;
  int64_t stride; /* elements from a row to the next; not used where there is one row */
} felix_matrix;

/*
 * Linear layer. Forward, felix_linear: with z = x weight^T + bias,
 *   out [tokens][out_features] = act(z) + residual, pre (optional) = z.
 * x [tokens][in_features], weight [out_features][in_features], bias (optional)
 * [out_features], residual (optional) as out.
 * Backward, felix_linear_bwd: with dz = grad act'(pre) (pre is not read without an
 * activation), each where wanted (not NULL): dx = dz weight, dweight = dz^T x, dbias =
 * the sum of dz's rows. dz is rounded to 16 bits once, as the products read it; dbias
 * sums it in fp32 before that. (The residual's gradient is grad itself.)
 * Fields that a direction does not name are not read, nor what only a gradient needs that
 * is not wanted.
 */
typedef struct felix_linear_args {
  uint32_t tokens, in_features, out_features;
  int dtype, activation;
  felix_matrix x, weight, residual;
  const void* bias;
  felix_matrix out, pre;
  felix_matrix grad, dx, dweight;
  void* dbias;
} felix_linear_args;

/*
 * Gated feed-forward block. g = x w_gate^T, u = x w_up^T [tokens][hidden],
 * h = act(g) u in one kernel; gate and up (optional) receive g and u.
 *   felix_gated_linear: out [tokens][hidden] = h.
 *   felix_gated_ffn:    out [tokens][features] = h w_down^T + residual (optional); h is
 *                       rounded to 16 bits in between.
 * w_gate, w_up [hidden][features], w_down [features][hidden].
 * Backward from gate and up: dh = grad (felix_gated_linear_bwd, grad [tokens][hidden])
 * or grad w_down (felix_gated_ffn_bwd, grad [tokens][features]; dh is never rounded),
 *   dg = dh u act'(g), du = dh act(g), each rounded once;
 * and where wanted dx = dg w_gate + du w_up, dw_gate = dg^T x, dw_up = du^T x,
 * dw_down = grad^T (act(g) u). (The residual's gradient is grad itself.)
 * Fields are read as in felix_linear_args; felix_gated_linear wants residual, and
 * felix_gated_linear_bwd dw_down, NULL. What is rounded in between (h, dg, du, and dz of the
 * linear layer) is an operand of the next product and has the range of its type: past 65504
 * it is infinite in fp16.
 */
typedef struct felix_gated_args {
  uint32_t tokens, features, hidden;
  int dtype, activation;
  felix_matrix x, w_gate, w_up, w_down, residual;
  felix_matrix out, gate, up;
  felix_matrix grad, dx, dw_gate, dw_up, dw_down;
} felix_gated_args;

/*
 * workspace: NULL = library-owned per (device, stream), which stays as large as the
 * largest call on the stream needed (the backward passes keep matrices of [tokens]
 * [hidden] there); otherwise felix_*_workspace_size() bytes for these very arguments,
 * 256-byte aligned, with any contents.
 */
int felix_linear(const felix_linear_args* args, void* workspace, size_t workspace_bytes,
                 void* stream);
int felix_linear_bwd(const felix_linear_args* args, void* workspace, size_t workspace_bytes,
                     void* stream);
int felix_linear_workspace_size(const felix_linear_args* args, int backward, size_t* bytes);
int felix_gated_linear(const felix_gated_args* args, void* workspace, size_t workspace_bytes,
                       void* stream);
int felix_gated_linear_bwd(const felix_gated_args* args, void* workspace, size_t workspace_bytes,
                           void* stream);
int felix_gated_ffn(const felix_gated_args* args, void* workspace, size_t workspace_bytes,
                    void* stream);
int felix_gated_ffn_bwd(const felix_gated_args* args, void* workspace, size_t workspace_bytes,
                        void* stream);
int felix_gated_workspace_size(const felix_gated_args* args, int ffn, int backward, size_t* bytes);

/*
 * Device watchdog. Every bounded wait inside the kernels records a nonzero
 * site code in a per-device status word when it gives up. Reads (and, when
 * clear != 0, resets) the word of the current device; synchronises the device.
 * Returns FELIX_KERNEL_RUNTIME_ERROR when the word was nonzero.
 */
int felix_watchdog_status(unsigned* code, int clear);

/*
 * Test hook for the watchdog: launches one CTA that waits on an mbarrier no
 * one arrives on, with a limit of limit_us microseconds (1..1000000). The wait
 * gives up, records its site code and the kernel returns normally.
 */
int felix_watchdog_probe(uint32_t limit_us, void* stream);

/* Number of SMs of the current device (persistent grid size). */
int felix_num_sms(int* count);

#ifdef __cplusplus
}
#endif

#endif /* FELIX_C_H */

"""sion_b200 — Sion's operator hot path (SGEMM, HGEMM, flash-attention forward)
as sm_100a kernels behind the reference's felix:: / sion:: interfaces.

Python surface (mirrors the reference module ``sion``, python/binding.cpp:6-11):

    sgemm(A, B, alpha=1, beta=0)        fp32, A [M,K] @ B [K,N]
    hgemm(A, B, alpha=1, beta=0)        fp16, B stored [K,N]   ("nn")
    hgemm_nt(A, B, alpha=1, beta=0)     fp16, B stored [N,K]   ("nt")
    gemm(A, B, alpha=1, beta=0)         dispatch on dtype
    flash_attention(Q, K, V)            fp16 [B,H,S,D], D in {64,128}
    flash_attention_lse(Q, K, V)        -> (O, fp32 LSE [B,H,S])
    flash_attention_backward(Q, K, V, O, LSE, dO) -> (dQ, dK, dV)
    flash_attention_autograd(Q, K, V)   differentiable forward (torch.autograd)

Decoding (no counterpart in the reference): a paged cache of keys and values in
4 bits, attention of new tokens over it, its pages, and sampling:

    kv4_append(pages, table, lens, K, V)       new tokens into the cache
    kv4_read(pages, table, lens, rows, Hkv, D) the last tokens back as fp16
    kv4_attention(Q, pages, table, lens, Hkv)  Q fp16/bf16 [slots,H,rows,D]
    kv4_attention_lse(...)                     -> (O, fp32 LSE)
    kv4_reserve / kv4_fork / kv4_free / kv4_compact / kv4_copy_pages
    sample(logits, uniform, temperature, top_k, top_p, min_p)

Feed-forward (no counterpart in the reference), fp16 or bf16, weights [out, in]:

    linear(x, W, bias, residual, activation)   act(x W^T + b) + r
    gated_linear(x, Wg, Wu, activation)        act(x Wg^T) * (x Wu^T)
    gated_ffn(x, Wg, Wu, Wd, residual, ...)    the whole block
    *_save(...)                                also what the backward pass needs
    *_backward(...), *_autograd(...)           gradients, torch.autograd

These come from the native module ``_sion`` (LibTorch C++), which calls the
felix:: C++ API in ``libfelix_b200.so``. The C ABI of that library
(include/felix_c.h) is reachable through :mod:`sion_b200.abi`. There is no
fallback: if the native libraries are missing, every call raises.
"""
from __future__ import annotations

import os

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, "libfelix_b200.so")

_ext = None


def _load_ext():
    global _ext
    if _ext is None:
        import importlib

        import torch  # noqa: F401  (loads libc10/libtorch for the extension)

        if not os.path.exists(LIB_PATH):
            raise ImportError(
                f"{LIB_PATH} is missing: build it with `python -m sion_b200.build`")
        try:
            _ext = importlib.import_module("sion_b200._sion")
        except ImportError as e:
            raise ImportError(
                "sion_b200._sion native module is missing or failed to load "
                f"({e}); build it with `python -m sion_b200.build`") from e
    return _ext


def sgemm(A, B, alpha: float = 1.0, beta: float = 0.0):
    return _load_ext().sgemm(A, B, alpha, beta)


def hgemm(A, B, alpha: float = 1.0, beta: float = 0.0):
    return _load_ext().hgemm(A, B, alpha, beta)


def hgemm_nt(A, B, alpha: float = 1.0, beta: float = 0.0):
    return _load_ext().hgemm_nt(A, B, alpha, beta)


def gemm(A, B, alpha: float = 1.0, beta: float = 0.0):
    return _load_ext().gemm(A, B, alpha, beta)


def flash_attention(query, key, value, causal: bool = False):
    return _load_ext().flash_attention(query, key, value, causal)


def flash_attention_lse(query, key, value, causal: bool = False):
    return _load_ext().flash_attention_lse(query, key, value, causal)


def flash_attention_backward(query, key, value, out, lse, grad_out, causal: bool = False):
    """(dQ, dK, dV) of flash_attention given the forward's O and LSE."""
    return _load_ext().flash_attention_backward(query, key, value, out, lse, grad_out, causal)


def _autograd_function():
    import torch

    class FlashAttentionFunction(torch.autograd.Function):
        @staticmethod
        def forward(ctx, query, key, value, causal):
            out, lse = flash_attention_lse(query, key, value, causal)
            ctx.save_for_backward(query, key, value, out, lse)
            ctx.causal = causal
            return out

        @staticmethod
        def backward(ctx, grad_out):
            q, k, v, out, lse = ctx.saved_tensors
            dq, dk, dv = flash_attention_backward(q, k, v, out, lse, grad_out.contiguous(),
                                                  ctx.causal)
            return dq, dk, dv, None

    return FlashAttentionFunction


_FA_FN = None


def flash_attention_autograd(query, key, value, causal: bool = False):
    """flash_attention that torch.autograd can differentiate (the backward runs
    the sm_100a backward kernel)."""
    global _FA_FN
    if _FA_FN is None:
        _FA_FN = _autograd_function()
    return _FA_FN.apply(query, key, value, causal)


def kv4_page_bytes(kv_heads: int, head_dim: int, page_size: int) -> int:
    """Bytes of a page: page_size * kv_heads * (head_dim + 8). A pool of the
    4-bit cache is a uint8 tensor [pages, kv4_page_bytes(...)]."""
    return _load_ext().kv4_page_bytes(kv_heads, head_dim, page_size)


def kv4_append(pages, table, lens, key, value, counts=None):
    """Writes new tokens into the cache: row i of key / value [slots, kv_heads,
    rows, D] is token lens - counts + i of its slot (`lens` includes the new
    tokens; `counts`, int32 [slots], says how many of the rows are tokens)."""
    _load_ext().kv4_append(pages, table, lens, key, value, counts)


def kv4_read(pages, table, lens, rows: int, kv_heads: int, head_dim: int, counts=None):
    """(K, V), fp16 [slots, kv_heads, rows, D]: the last tokens of each slot as
    the cache holds them; rows that are no token are zero."""
    return _load_ext().kv4_read(pages, table, lens, rows, kv_heads, head_dim, counts)


def kv4_attention(query, pages, table, lens, kv_heads: int, counts=None, scale: float = 0.0):
    """Attention of the new tokens query [slots, heads, rows, D] (fp16 or bf16)
    over the cache: row i of n sees the tokens 0 .. len - n + i. Rows that see
    nothing give zeros. scale <= 0: 1 / sqrt(D)."""
    return _load_ext().kv4_attention(query, pages, table, lens, kv_heads, counts, scale)


def kv4_attention_lse(query, pages, table, lens, kv_heads: int, counts=None, scale: float = 0.0):
    """kv4_attention returning (O, LSE), LSE fp32 [slots, heads, rows] (-inf
    where a row sees nothing)."""
    return _load_ext().kv4_attention_lse(query, pages, table, lens, kv_heads, counts, scale)


def kv4_reserve(table, lens, refs, counts, page_size: int, out=None):
    """(table, lens, refs, status) after each slot has grown by counts tokens and
    has the pages for them, the lowest free ones first. status[0]: pages that
    were missing; nothing changes unless it is 0. `out`: tensors to write, which
    may be (table, lens, refs) themselves."""
    return _load_ext().kv4_reserve(table, lens, refs, counts, page_size, out)


def kv4_fork(pages, table, lens, refs, parents, children, page_size: int, out=None):
    """(table, lens, refs, status) after slot children[i] (empty before) has
    become a copy of slot parents[i]: whole pages are shared, a last page that is
    not full is copied. status: [pages missing, pairs skipped]."""
    return _load_ext().kv4_fork(pages, table, lens, refs, parents, children, page_size, out)


def kv4_free(table, lens, refs, slots, page_size: int, out=None):
    """(table, lens, refs) after the listed slots were emptied."""
    return _load_ext().kv4_free(table, lens, refs, slots, page_size, out)


def kv4_compact(pages, table, refs, out=None):
    """(table, refs) after the pages in use have moved to the lowest numbers."""
    return _load_ext().kv4_compact(pages, table, refs, out)


def kv4_copy_pages(src_pages, dst_pages, src, dst):
    """Copies page src[i] of one pool to page dst[i] of another."""
    _load_ext().kv4_copy_pages(src_pages, dst_pages, src, dst)


def sample(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
    """One token per row of logits [rows, vocab] from uniform [rows] in [0, 1):
    (tokens int32 [rows], log-probability of each under the kept tokens).
    temperature, top_p, min_p (fp32 [rows]) and top_k (int32 [rows]) may be
    numbers, for all rows, or None. A number is written into a tensor by a small
    kernel first (about 5 us each): a loop that keeps its tensors saves that."""
    import torch

    def rows(v, dtype):
        if v is None or isinstance(v, torch.Tensor):
            return v
        return torch.full((logits.shape[0],), v, dtype=dtype, device=logits.device)

    return _load_ext().sample(logits, uniform, rows(temperature, torch.float32),
                              rows(top_k, torch.int32), rows(top_p, torch.float32),
                              rows(min_p, torch.float32))


def linear(x, weight, bias=None, residual=None, activation: str = "none"):
    """act(x weight^T + bias) + residual in one kernel, rounded once. x [..., in] fp16 or
    bf16, weight [out, in], bias [out], residual [..., out]. activation: "none", "relu",
    "gelu", "gelu_tanh", "silu" or "sigmoid"."""
    return _load_ext().linear(x, weight, bias, residual, activation)


def linear_save(x, weight, bias=None, residual=None, activation: str = "none"):
    """linear returning (y, pre), pre = x weight^T + bias for linear_backward."""
    return _load_ext().linear_save(x, weight, bias, residual, activation)


def linear_backward(grad, x, weight, pre=None, activation: str = "none", bias: bool = False,
                    need_x: bool = True, need_weight: bool = True):
    """(dx, dweight, dbias) of linear from grad [..., out] and, with an activation, pre;
    None where not wanted. The residual's gradient is grad."""
    return _load_ext().linear_backward(grad, x, weight, pre, activation, bias, need_x, need_weight)


def gated_linear(x, w_gate, w_up, activation: str = "silu"):
    """act(x w_gate^T) * (x w_up^T) in one kernel. x [..., in], both weights [hidden, in]."""
    return _load_ext().gated_linear(x, w_gate, w_up, activation)


def gated_linear_save(x, w_gate, w_up, activation: str = "silu"):
    """gated_linear returning (h, gate, up), the projections for gated_linear_backward."""
    return _load_ext().gated_linear_save(x, w_gate, w_up, activation)


def gated_linear_backward(grad, x, w_gate, w_up, gate, up, activation: str = "silu",
                          need_x: bool = True, need_weights: bool = True):
    """(dx, dw_gate, dw_up) of gated_linear; None where not wanted."""
    return _load_ext().gated_linear_backward(grad, x, w_gate, w_up, gate, up, activation, need_x,
                                             need_weights)


def gated_ffn(x, w_gate, w_up, w_down, residual=None, activation: str = "silu"):
    """gated_linear(x, w_gate, w_up) w_down^T + residual; w_down [in, hidden]."""
    return _load_ext().gated_ffn(x, w_gate, w_up, w_down, residual, activation)


def gated_ffn_save(x, w_gate, w_up, w_down, residual=None, activation: str = "silu"):
    """gated_ffn returning (y, gate, up), the projections for gated_ffn_backward."""
    return _load_ext().gated_ffn_save(x, w_gate, w_up, w_down, residual, activation)


def gated_ffn_backward(grad, x, w_gate, w_up, w_down, gate, up, activation: str = "silu",
                       need_x: bool = True, need_weights: bool = True):
    """(dx, dw_gate, dw_up, dw_down) of gated_ffn; None where not wanted. The residual's
    gradient is grad."""
    return _load_ext().gated_ffn_backward(grad, x, w_gate, w_up, w_down, gate, up, activation,
                                          need_x, need_weights)


def _ffn_functions():
    import torch
    from torch.autograd.function import once_differentiable

    # What a backward pass does not read is not kept: x where no weight needs a gradient,
    # weights where x needs none. Of these it takes the shape alone.
    def stand_in(grad, shape):
        return grad.new_empty(shape[-1]).expand(shape)

    class Linear(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, bias, residual, activation):
            need, pre = ctx.needs_input_grad, None
            if activation == "none" or not any(need[:3]):
                y = linear(x, weight, bias, residual, activation)
            else:
                y, pre = linear_save(x, weight, bias, residual, activation)
            ctx.save_for_backward(x if need[1] else None, weight if need[0] else None, pre)
            ctx.shapes = x.shape, weight.shape
            ctx.activation = activation
            return y

        @staticmethod
        @once_differentiable
        def backward(ctx, grad):
            x, weight, pre = ctx.saved_tensors
            need = ctx.needs_input_grad
            dx = dw = db = None
            if any(need[:3]):
                dx, dw, db = linear_backward(
                    grad, stand_in(grad, ctx.shapes[0]) if x is None else x,
                    stand_in(grad, ctx.shapes[1]) if weight is None else weight, pre,
                    ctx.activation, need[2], need[0], need[1])
            return dx, dw, db, grad if need[3] else None, None

    class GatedLinear(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w_gate, w_up, activation):
            need = ctx.needs_input_grad
            h, gate, up = gated_linear_save(x, w_gate, w_up, activation)
            ctx.save_for_backward(x if any(need[1:3]) else None,
                                  *((w_gate, w_up) if need[0] else (None, None)), gate, up)
            ctx.shapes = x.shape, w_gate.shape
            ctx.activation = activation
            return h

        @staticmethod
        @once_differentiable
        def backward(ctx, grad):
            x, w_gate, w_up, gate, up = ctx.saved_tensors
            need = ctx.needs_input_grad
            if x is None:
                x = stand_in(grad, ctx.shapes[0])
            if w_gate is None:
                w_gate = w_up = stand_in(grad, ctx.shapes[1])
            return *gated_linear_backward(grad, x, w_gate, w_up, gate, up, ctx.activation, need[0],
                                          any(need[1:3])), None

    class GatedFfn(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w_gate, w_up, w_down, residual, activation):
            need = ctx.needs_input_grad
            ctx.activation = activation
            if not any(need[:4]):
                return gated_ffn(x, w_gate, w_up, w_down, residual, activation)
            y, gate, up = gated_ffn_save(x, w_gate, w_up, w_down, residual, activation)
            ctx.save_for_backward(x if any(need[1:4]) else None,
                                  *((w_gate, w_up) if need[0] else (None, None)), w_down, gate, up)
            ctx.shapes = x.shape, w_gate.shape
            return y

        @staticmethod
        @once_differentiable
        def backward(ctx, grad):
            need = ctx.needs_input_grad
            d = (None,) * 4
            if any(need[:4]):
                x, w_gate, w_up, w_down, gate, up = ctx.saved_tensors
                if x is None:
                    x = stand_in(grad, ctx.shapes[0])
                if w_gate is None:
                    w_gate = w_up = stand_in(grad, ctx.shapes[1])
                d = gated_ffn_backward(grad, x, w_gate, w_up, w_down, gate, up, ctx.activation,
                                       need[0], any(need[1:4]))
            return *d, grad if need[4] else None, None

    return Linear, GatedLinear, GatedFfn


_FFN_FNS = None


def _ffn_function(i):
    global _FFN_FNS
    if _FFN_FNS is None:
        _FFN_FNS = _ffn_functions()
    return _FFN_FNS[i]


def _needs_gradient(*tensors):
    import torch
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def linear_autograd(x, weight, bias=None, residual=None, activation: str = "none"):
    """linear that torch.autograd can differentiate (first derivatives); linear itself
    where no input needs a gradient."""
    if not _needs_gradient(x, weight, bias, residual):
        return linear(x, weight, bias, residual, activation)
    return _ffn_function(0).apply(x, weight, bias, residual, activation)


def gated_linear_autograd(x, w_gate, w_up, activation: str = "silu"):
    """gated_linear that torch.autograd can differentiate (first derivatives); gated_linear
    itself where no input needs a gradient."""
    if not _needs_gradient(x, w_gate, w_up):
        return gated_linear(x, w_gate, w_up, activation)
    return _ffn_function(1).apply(x, w_gate, w_up, activation)


def gated_ffn_autograd(x, w_gate, w_up, w_down, residual=None, activation: str = "silu"):
    """gated_ffn that torch.autograd can differentiate (first derivatives); gated_ffn
    itself where no input needs a gradient."""
    if not _needs_gradient(x, w_gate, w_up, w_down, residual):
        return gated_ffn(x, w_gate, w_up, w_down, residual, activation)
    return _ffn_function(2).apply(x, w_gate, w_up, w_down, residual, activation)


__all__ = ["sgemm", "hgemm", "hgemm_nt", "gemm", "flash_attention", "flash_attention_lse",
           "flash_attention_backward", "flash_attention_autograd", "kv4_page_bytes", "kv4_append",
           "kv4_read", "kv4_attention", "kv4_attention_lse", "kv4_reserve", "kv4_fork", "kv4_free",
           "kv4_compact", "kv4_copy_pages", "sample", "linear", "linear_save", "linear_backward",
           "linear_autograd", "gated_linear", "gated_linear_save", "gated_linear_backward",
           "gated_linear_autograd", "gated_ffn", "gated_ffn_save", "gated_ffn_backward",
           "gated_ffn_autograd", "LIB_PATH"]

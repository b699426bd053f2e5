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


__all__ = ["sgemm", "hgemm", "hgemm_nt", "gemm", "flash_attention", "flash_attention_lse",
           "flash_attention_backward", "flash_attention_autograd", "kv4_page_bytes", "kv4_append",
           "kv4_read", "kv4_attention", "kv4_attention_lse", "kv4_reserve", "kv4_fork", "kv4_free",
           "kv4_compact", "kv4_copy_pages", "sample", "LIB_PATH"]

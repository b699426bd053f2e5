"""``import sion`` for existing callers of the reference's Python module.

The reference builds its operators as a module named ``sion``
(python/binding.cpp:6-11: ``sgemm``, ``flash_attention``), imported by its
python/sgemm_test.py and python/flash_attn_test.py. This package re-exports
the sm_100a implementation in :mod:`sion_b200` under that name, so those
callers run unchanged; the extra operators (hgemm, hgemm_nt, gemm,
flash_attention_lse, the backward, the 4-bit cache and sampling) come along.
"""
from sion_b200 import (  # noqa: F401
    LIB_PATH,
    flash_attention,
    flash_attention_autograd,
    flash_attention_backward,
    flash_attention_lse,
    gated_ffn,
    gated_ffn_autograd,
    gated_ffn_backward,
    gated_ffn_save,
    gated_linear,
    gated_linear_autograd,
    gated_linear_backward,
    gated_linear_save,
    gemm,
    hgemm,
    hgemm_nt,
    kv4_append,
    kv4_attention,
    kv4_attention_lse,
    kv4_compact,
    kv4_copy_pages,
    kv4_fork,
    kv4_free,
    kv4_page_bytes,
    kv4_read,
    kv4_reserve,
    linear,
    linear_autograd,
    linear_backward,
    linear_save,
    sample,
    sgemm,
)

__all__ = ["sgemm", "hgemm", "hgemm_nt", "gemm", "flash_attention", "flash_attention_lse",
           "flash_attention_backward", "flash_attention_autograd", "kv4_page_bytes", "kv4_append",
           "kv4_read", "kv4_attention", "kv4_attention_lse", "kv4_reserve", "kv4_fork", "kv4_free",
           "kv4_compact", "kv4_copy_pages", "sample", "linear", "linear_save", "linear_backward",
           "linear_autograd", "gated_linear", "gated_linear_save", "gated_linear_backward",
           "gated_linear_autograd", "gated_ffn", "gated_ffn_save", "gated_ffn_backward",
           "gated_ffn_autograd", "LIB_PATH"]

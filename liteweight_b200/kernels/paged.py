"""Attention over a paged key-value cache, and the pass that fills it.

The reference keeps one contiguous block per layer (KVCache,
liteweight/generate.py:7-46); here a cache is a pool of pages that sequences
of any lengths share:

    k_pages, v_pages   fp16 or bf16 [pages, kv heads, page_size, head_dim], any
                       strides with the last dimension contiguous (a transposed
                       [pages, page_size, kv heads, head_dim] pool, or halves of
                       one pool, are fine); page_size 16, 32, 64, 128 or 256,
                       head_dim 64 or 128
    page_table         int32 [batch, width]: token t of sequence b is in slot
                       t % page_size of page page_table[b, t // page_size];
                       entries that no visible token needs are not read
    kv_lens            int32 [batch]: tokens of each sequence, the newest included
    q_offsets          int32 [batch + 1]: rows q_offsets[b] .. q_offsets[b+1] - 1
                       are the newest tokens of sequence b; None: row b is the
                       one new token of sequence b

A page id outside the pool, a length past the table or a position past the
rotation table makes the kernels skip that access (the key is hidden, the token
is not stored) and record LW_ERR_BAD_INDEX, which check_device_error() raises.

Every call runs on torch's current stream of its tensors' device, allocates its
output and scratch from torch, and can be captured in a CUDA graph.
"""

from __future__ import annotations

import ctypes

import torch

from liteweight_b200 import _native as nat

c_int, c_void_p, c_float, c_size_t, c_ll = (ctypes.c_int, ctypes.c_void_p, ctypes.c_float, ctypes.c_size_t,
                                            ctypes.c_longlong)


class PagedCacheArgs(ctypes.Structure):
    """Mirror of lw_paged_cache (include/liteweight_b200.h)."""
    _fields_ = [("k_pages", c_void_p), ("v_pages", c_void_p), ("k_strides", c_ll * 3), ("v_strides", c_ll * 3),
                ("n_pages", c_int), ("page_size", c_int), ("n_kv_heads", c_int), ("head_dim", c_int),
                ("dtype", c_int), ("batch", c_int), ("page_table", c_void_p), ("table_stride", c_ll),
                ("table_width", c_int), ("kv_lens", c_void_p)]


class QkNormRopeArgs(ctypes.Structure):
    """Mirror of lw_qk_norm_rope_args (include/liteweight_b200.h)."""
    _fields_ = [("cache", PagedCacheArgs), ("q", c_void_p), ("k", c_void_p), ("v", c_void_p),
                ("q_strides", c_ll * 2), ("k_strides", c_ll * 2), ("v_strides", c_ll * 2), ("q_out", c_void_p),
                ("out_strides", c_ll * 2), ("tokens", c_int), ("n_q_heads", c_int), ("q_offsets", c_void_p),
                ("rope_cos", c_void_p), ("rope_sin", c_void_p), ("rope_stride", c_ll), ("rope_dtype", c_int),
                ("rope_rows", c_int), ("q_weight", c_void_p), ("k_weight", c_void_p), ("eps", c_float),
                ("zero_tail", c_int), ("pdl", c_int)]


class PagedAttentionArgs(ctypes.Structure):
    """Mirror of lw_paged_attention_args (include/liteweight_b200.h)."""
    _fields_ = [("cache", PagedCacheArgs), ("q", c_void_p), ("q_strides", c_ll * 2), ("out", c_void_p),
                ("out_strides", c_ll * 2), ("tokens", c_int), ("n_q_heads", c_int), ("q_offsets", c_void_p),
                ("window", c_int), ("sinks", c_int), ("scale", c_float), ("zero_tail", c_int), ("pdl", c_int),
                ("workspace", c_void_p), ("workspace_bytes", c_size_t)]


nat.register("lw_qk_norm_rope", [ctypes.POINTER(QkNormRopeArgs), c_void_p])
nat.register("lw_paged_attention", [ctypes.POINTER(PagedAttentionArgs), c_void_p])
nat.register("lw_paged_attention_workspace_size", [ctypes.POINTER(PagedAttentionArgs)], c_size_t)


def check_device_error() -> None:
    """Raise LiteweightError if a kernel of the library recorded an error on the
    current device since the last check (an index out of range, a wait that gave
    up). Synchronises the device."""
    nat.check("lw_take_device_error", nat.lib().lw_take_device_error())


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                 k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
                 q_offsets: torch.Tensor | None = None, *, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Per-head RMS norm of q and k, rotation by position, append of k and v to the cache.

        y = x * rsqrt(mean(x^2) + eps) * weight        (no weights: y = x)
        o = y * cos[p] + rotate_half(y) * sin[p]

    in fp32 with one rounding at the end; p is the row's position, kv_lens[b] -
    (new tokens of b) + (its place among them), kv_lens counting the new tokens.

    Args:
        q:          [tokens, q heads, head_dim]; k, v: [tokens, kv heads, head_dim],
                    in the cache's dtype, e.g. slices of one q|k|v tensor
        cos, sin:   [positions, head_dim] fp32 or the cache's dtype (both halves,
                    as HF's rotary embedding gives them)
        q_weight, k_weight: [head_dim] norm weights, or both None
        out:        [tokens, q heads, head_dim] for the rotated queries (may be q)

    Returns the rotated queries. Rows of no sequence (kv_lens[b] = 0, or from
    q_offsets[-1] on) are zero, or left as they were in a given `out`. New tokens
    must not share a slot.
    """
    got = nat.bind().qk_norm_rope(q, k, v, cos, sin, k_pages, v_pages, page_table, kv_lens, q_offsets, q_weight,
                                  k_weight, eps, out)
    if type(got) is int:
        nat.check("lw_qk_norm_rope", got)
    return got


def _attention(q, k_pages, v_pages, page_table, kv_lens, q_offsets, window, sinks, scale, out):
    got = nat.bind().attention(q, k_pages, v_pages, page_table, kv_lens, q_offsets, window, sinks, scale, out)
    if type(got) is int:
        nat.check("lw_paged_attention", got)
    return got


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    kv_lens: torch.Tensor, *, window: int | None = None, sinks: int = 0, scale: float | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over the paged cache.

        out[b, h] = sum_j softmax_j(scale * q[b, h] . k_j) v_j

    over the keys j that position p = kv_lens[b] - 1 sees: all of 0 .. p, or with
    a window those with p - j < window or j < sinks. Query head h reads kv head
    h // (q heads / kv heads). A sequence of length 0 gives zeros; one whose scores are
    all minus infinity gives NaN. The softmax weights are rounded to q's type for the
    product with v; scores, maxima and sums are fp32.

    Args:
        q:      [batch, q heads, head_dim], in the cache's dtype
        scale:  of the scores, above 0; head_dim ** -0.5 by default
        out:    [batch, q heads, head_dim] (may not overlap q)
    """
    return _attention(q, k_pages, v_pages, page_table, kv_lens, None, window, sinks, scale, out)


def prompt_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                     kv_lens: torch.Tensor, q_offsets: torch.Tensor, *, window: int | None = None, sinks: int = 0,
                     scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of prompt chunks over the paged cache.

    Rows q_offsets[b] .. q_offsets[b+1] - 1 are the newest tokens of sequence b;
    each attends as paged_attention's one row does, from its own position, over
    the tokens the cache keeps (the chunk's own among them, stored before).

    Args:
        q:      [tokens, q heads, head_dim], in the cache's dtype
        out:    [tokens, q heads, head_dim] (may not overlap q)

    Rows from q_offsets[-1] on, and those of a sequence whose offsets run past q (which
    is recorded), are zero, or left as they were in a given `out`.
    """
    assert q_offsets is not None, "q_offsets: int32 [batch + 1]"
    return _attention(q, k_pages, v_pages, page_table, kv_lens, q_offsets, window, sinks, scale, out)

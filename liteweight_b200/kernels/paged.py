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
import struct

import torch

from liteweight_b200 import _native as nat

c_int, c_void_p, c_float, c_size_t, c_ll = (ctypes.c_int, ctypes.c_void_p, ctypes.c_float, ctypes.c_size_t,
                                            ctypes.c_longlong)
_INT_MAX = 2**31 - 1
_WORKSPACE = 7   # LW_ERR_WORKSPACE
# what torch.cuda.current_device() and current_stream().cuda_stream come to
_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
_F16, _BF16, _F32, _I32 = torch.float16, torch.bfloat16, torch.float32, torch.int32


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


# The calls below write the same structs with struct.pack (one call instead of a
# ctypes object per field: a decode step makes two of them per layer). Native
# alignment, so the layouts are the C compiler's.
_CACHE_FMT = "PP6q6iPqi0qP"
_ROPE = struct.Struct("@" + _CACHE_FMT + "PPP6qP2qii0qPPPqiiPPfii0q")
_ATTN = struct.Struct("@" + _CACHE_FMT + "P2qP2qii0qPiifii0qPN")
assert _ROPE.size == ctypes.sizeof(QkNormRopeArgs) and _ATTN.size == ctypes.sizeof(PagedAttentionArgs)

nat.register("lw_qk_norm_rope", [c_void_p, c_void_p])
nat.register("lw_paged_attention", [c_void_p, c_void_p])
nat.register("lw_paged_attention_workspace_size", [c_void_p], c_size_t)


def _rows(name: str, t: torch.Tensor, dtype: torch.dtype, hd: int) -> tuple[int, int]:
    """(token, head) strides of a [tokens, heads, head_dim] tensor."""
    assert t.dtype is dtype, f"{name} is {t.dtype}, the cache {dtype}"
    strides = t.stride()
    assert len(strides) == 3 and t.shape[2] == hd, f"{name} must be [tokens, heads, {hd}], got {tuple(t.shape)}"
    assert strides[2] == 1 or t.numel() == 0, f"{name}'s last dimension must be contiguous"
    return strides[:2]


def _cache_fields(k_pages, v_pages, page_table, kv_lens) -> tuple:
    dt = k_pages.dtype
    assert (dt is _F16 or dt is _BF16) and v_pages.dtype is dt, "k_pages / v_pages: both float16 or both bfloat16"
    shape = k_pages.shape
    assert len(shape) == 4 and shape == v_pages.shape, "k_pages / v_pages: [pages, kv heads, page, head_dim]"
    assert page_table.dtype is _I32 and kv_lens.dtype is _I32, "page_table and kv_lens are int32"
    ks, vs, ts = k_pages.stride(), v_pages.stride(), page_table.stride()
    assert len(ts) == 2 and kv_lens.dim() == 1, "page_table: [batch, width], kv_lens: [batch]"
    batch, width = page_table.shape
    assert len(kv_lens) == batch, "page_table: [batch, width], kv_lens: [batch]"
    assert (ks[3] == 1 and vs[3] == 1) or k_pages.numel() == 0, "the pools' last dimension must be contiguous"
    assert ts[1] == 1 or width <= 1, "page_table's rows must be contiguous"
    assert batch <= 1 or kv_lens.stride(0) == 1, "kv_lens must be contiguous"
    return (k_pages.data_ptr(), v_pages.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], shape[0], shape[2],
            shape[1], shape[3], 0 if dt is _F16 else 1, batch, page_table.data_ptr(), ts[0], width, kv_lens.data_ptr())


def _offsets(q_offsets, batch: int, tokens: int) -> int:
    if q_offsets is None:
        assert tokens == batch, f"one new token per sequence: {tokens} rows for {batch} sequences"
        return 0
    assert q_offsets.dtype is _I32 and q_offsets.shape == (batch + 1,), f"q_offsets: int32 [{batch + 1}]"
    assert q_offsets.stride(0) == 1, "q_offsets must be contiguous"
    return q_offsets.data_ptr()


def _refuse_devices(*ts) -> None:
    nat.require_cuda(*ts)
    raise AssertionError("all tensors must be on one device")


def _run(fn: str, args: bytes, dev: int) -> None:
    status = _status(getattr(nat.lib(), fn), args, dev)
    if status:
        nat.check(fn, status)


def _status(call, args: bytes, dev: int) -> int:
    """One C call on the current stream of device `dev`, as the current device."""
    if _current_device() == dev:
        return call(args, _raw_stream(dev))
    with torch.cuda.device(dev):
        return call(args, _raw_stream(dev))


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
    cache = _cache_fields(k_pages, v_pages, page_table, kv_lens)
    dt, nkv, hd, batch = k_pages.dtype, cache[10], cache[11], cache[13]
    qs, ks, vs = _rows("q", q, dt, hd), _rows("k", k, dt, hd), _rows("v", v, dt, hd)
    T, nq, _ = q.shape
    assert k.shape == (T, nkv, hd) and v.shape == k.shape, f"k and v: [{T}, {nkv}, {hd}]"
    tt, tshape, ts = cos.dtype, cos.shape, cos.stride()
    assert len(tshape) == 2 and tshape[1] == hd and tshape == sin.shape, f"cos / sin: [positions, {hd}]"
    assert (tt is dt or tt is _F32) and sin.dtype is tt, f"cos / sin: {dt} or float32"
    assert ts == sin.stride() and (ts[1] == 1 or cos.numel() == 0), "cos / sin: rows contiguous, strides alike"
    assert (q_weight is None) == (k_weight is None), "norm weights for both queries and keys, or for neither"
    if q_weight is not None:
        for w in (q_weight, k_weight):
            assert w.dtype is dt and w.shape == (hd,) and w.stride(0) == 1, f"norm weights: {dt} [{hd}]"
    off = _offsets(q_offsets, batch, T)
    assert out is None or out.shape == q.shape, "out must have q's shape"
    dev = q.get_device()
    if not (0 <= dev == k.get_device() == v.get_device() == cos.get_device() == sin.get_device() == k_pages.get_device()
            == v_pages.get_device() == page_table.get_device() == kv_lens.get_device()
            and all(t is None or t.get_device() == dev for t in (q_offsets, q_weight, k_weight, out))):
        _refuse_devices(q, k, v, cos, sin, k_pages, v_pages, page_table, kv_lens, q_offsets, q_weight, k_weight, out)
    fresh = out is None
    if fresh:
        out = torch.empty_like(q)
    os_ = _rows("out", out, dt, hd)
    _run("lw_qk_norm_rope", _ROPE.pack(
        *cache, q.data_ptr(), k.data_ptr(), v.data_ptr(), *qs, *ks, *vs, out.data_ptr(), *os_, T, nq, off,
        cos.data_ptr(), sin.data_ptr(), ts[0], 2 if tt is _F32 else cache[12], tshape[0],
        0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr(), eps, fresh, 1),
        dev)
    return out


def _attention(q, k_pages, v_pages, page_table, kv_lens, q_offsets, window, sinks, scale, out):
    cache = _cache_fields(k_pages, v_pages, page_table, kv_lens)
    dt, hd, batch = k_pages.dtype, cache[11], cache[13]
    qs = _rows("q", q, dt, hd)
    T, nq, _ = q.shape
    assert nq % cache[10] == 0, f"{nq} query heads over {cache[10]} kv heads"
    assert window is None or window >= 1, "window: at least 1, or None"
    assert sinks >= 0, "sinks: at least 0"
    off = _offsets(q_offsets, batch, T)
    assert out is None or (out.shape == q.shape and out.dtype is dt), "out must have q's shape and type"
    dev = q.get_device()
    if not (0 <= dev == k_pages.get_device() == v_pages.get_device() == page_table.get_device() == kv_lens.get_device()
            and (q_offsets is None or q_offsets.get_device() == dev) and (out is None or out.get_device() == dev)):
        _refuse_devices(q, k_pages, v_pages, page_table, kv_lens, q_offsets, out)
    fresh = out is None
    if fresh:
        out = torch.empty_like(q)
    fields = (*cache, q.data_ptr(), *qs, out.data_ptr(), *_rows("out", out, dt, hd), T, nq, off,
              min(window or 0, _INT_MAX), min(sinks, _INT_MAX), hd ** -0.5 if scale is None else scale, fresh, 1)
    lib, args = nat.lib(), _ATTN.pack(*fields, 0, 0)
    status = _status(lib.lw_paged_attention, args, dev)
    if status == _WORKSPACE:   # not a short one: with scratch of this call alone, which no other stream or graph shares
        with torch.cuda.device(dev):
            need = lib.lw_paged_attention_workspace_size(args)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        status = _status(lib.lw_paged_attention, _ATTN.pack(*fields, ws.data_ptr(), ws.numel()), dev)
    if status:
        nat.check("lw_paged_attention", status)
    return out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    kv_lens: torch.Tensor, *, window: int | None = None, sinks: int = 0, scale: float | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over the paged cache.

        out[b, h] = sum_j softmax_j(scale * q[b, h] . k_j) v_j

    over the keys j that position p = kv_lens[b] - 1 sees: all of 0 .. p, or with
    a window those with p - j < window or j < sinks. Query head h reads kv head
    h // (q heads / kv heads). A sequence of length 0 gives zeros.

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

    Rows from q_offsets[-1] on are zero, or left as they were in a given `out`.
    """
    assert q_offsets is not None, "q_offsets: int32 [batch + 1]"
    return _attention(q, k_pages, v_pages, page_table, kv_lens, q_offsets, window, sinks, scale, out)

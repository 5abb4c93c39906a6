"""The paged-cache operators against their definitions in 64 bits.

Tolerances, fixed before the first run. With h = finfo(dtype).eps / 2 (the largest
relative error of one rounding), w_j the softmax weights and A = sum_j w_j |v_j|:
  * the output's own rounding                                    h |out|
  * every weight rounded to dtype for the second product         h A
    (fp16 weights below 2^-14 are rounded by at most 2^-25 each, against a sum
    of weights >= 1: 2^-25 sum_j |v_j|)
  * a score is hd products summed in fp32, off by at most hd 2^-23 sum_d |q_d k_d|;
    it moves a weight and the sum of weights by that much each   2 hd 2^-23 S A,
    S = max_j scale sum_d |q_d k_jd|
  * sums over n keys in fp32 and the exponentials                (n + 64) 2^-23 A
  * fp16 outputs below the normal range                          2^-25
"""

import math

import pytest
import torch

from liteweight_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
DTYPES = [torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


class Batch:
    """A paged cache filled with random tokens, its unused slots poisoned."""

    def __init__(self, lens, nkv, hd, page, dtype, seed=0, order="phsd", table_garbage=-7, spare=2):
        g = gen(seed)
        self.lens, self.page, self.hd, self.nkv, self.dtype = lens, page, hd, nkv, dtype
        need = [-(-n // page) for n in lens]
        n_pages = sum(need) + spare
        shape = (n_pages, nkv, page, hd)
        if order == "phsd":
            pools = [torch.full(shape, float("nan"), dtype=dtype, device=DEV) for _ in range(2)]
        elif order == "pshd":   # [page, slot, head, dim]
            pools = [torch.full((n_pages, page, nkv, hd), float("nan"), dtype=dtype, device=DEV).transpose(1, 2)
                     for _ in range(2)]
        else:                   # one pool for both, head by head
            both = torch.full((nkv, n_pages, 2, page, hd), float("nan"), dtype=dtype, device=DEV)
            pools = [both[:, :, i].transpose(0, 1) for i in range(2)]
        self.k_pages, self.v_pages = pools
        perm = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
        width = max(need, default=0) + 1
        # rows of the table lie further apart than they are long
        self.table = torch.full((len(lens), width + 3), table_garbage, dtype=torch.int32, device=DEV)[:, :width]
        at = 0
        self.k, self.v = [], []
        for b, n in enumerate(lens):
            self.table[b, :need[b]] = perm[at:at + need[b]]
            at += need[b]
            self.k.append(torch.randn(n, nkv, hd, generator=g, device=DEV).to(dtype))
            self.v.append(torch.randn(n, nkv, hd, generator=g, device=DEV).to(dtype))
            self.put(b, 0, self.k[b], self.v[b])
        self.kv_lens = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def where(self, b, first, n):
        t = torch.arange(first, first + n, device=DEV)
        return self.table[b].long()[t // self.page], t % self.page

    def put(self, b, first, k, v):
        p, s = self.where(b, first, k.shape[0])
        self.k_pages[p, :, s] = k
        self.v_pages[p, :, s] = v

    def cache(self):
        return self.k_pages, self.v_pages, self.table, self.kv_lens


def attend(q, k, v, first, window, sinks, scale, dtype):
    """(out, tolerance) in fp64 for rows at positions first.. over k, v [n, nkv, hd]."""
    T, nq, hd = q.shape
    n, nkv = k.shape[0], k.shape[1]
    h = torch.finfo(dtype).eps / 2
    p = torch.arange(first, first + T, device=DEV)[:, None]
    j = torch.arange(n, device=DEV)[None]
    seen = j <= p
    if window:
        seen &= (p - j < window) | (j < sinks)
    out = torch.zeros(T, nq, hd, dtype=torch.float64, device=DEV)
    tol = torch.full_like(out, 2.0 ** -25)
    for a in range(nq):
        kk, vv = k[:, a * nkv // nq].double(), v[:, a * nkv // nq].double()
        qq = q[:, a].double()
        x = (qq @ kk.T * scale).masked_fill(~seen, -math.inf)
        w = torch.softmax(x, -1)
        w = torch.where(seen.any(-1, keepdim=True), w, torch.zeros_like(w))
        o = w @ vv
        A = w @ vv.abs()
        S = ((qq.abs() @ kk.abs().T) * scale).masked_fill(~seen, 0).amax(-1, keepdim=True) if n else 0
        U = seen.double() @ vv.abs() * (2.0 ** -25 if dtype == torch.float16 else 0.0)
        out[:, a] = o
        tol[:, a] += h * o.abs() + (h + 2 * hd * 2.0 ** -23 * S + (n + 64) * 2.0 ** -23) * A + U
    return out, tol


def check(got, want, tol):
    if got.numel() == 0:
        return
    assert torch.isfinite(got.float()).all(), "a hidden value reached the result"
    bad = (got.double() - want).abs() > tol
    worst = ((got.double() - want).abs() / tol).max().item()
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {worst:.2f} of the tolerance"


LENS = {
    "one": [1], "tile-edges": [15, 16, 17, 0, 33, 128, 1], "long": [5003], "ragged": [700, 3, 0, 2047, 64, 1290, 31],
    "many": [(i * 37) % 150 for i in range(301)],
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nkv,group", [(2, 4), (3, 1), (1, 8), (2, 12), (1, 20)])
@pytest.mark.parametrize("lens,page,window,sinks", [
    ("one", 16, None, 0), ("tile-edges", 16, None, 0), ("tile-edges", 64, 5, 2), ("long", 32, None, 0),
    ("long", 256, 1000, 37), ("ragged", 128, None, 0), ("ragged", 16, 100, 0), ("ragged", 16, 33, 4),
    ("ragged", 32, 1, 0), ("ragged", 32, 5000, 4), ("many", 16, 64, 1)])
def test_decode(dtype, hd, nkv, group, lens, page, window, sinks):
    c = Batch(LENS[lens], nkv, hd, page, dtype, seed=hd + group + page)
    q = (torch.randn(len(c.lens), nkv * group, hd, generator=gen(7), device=DEV) * 1.7).to(dtype)
    got = kernels.paged_attention(q, *c.cache(), window=window, sinks=sinks)
    kernels.check_device_error()
    for b, n in enumerate(c.lens):
        want, tol = attend(q[b:b + 1], c.k[b], c.v[b], n - 1, window, sinks, hd ** -0.5, dtype)
        check(got[b:b + 1], want, tol)


@pytest.mark.parametrize("order", ["phsd", "pshd", "both"])
def test_decode_orders_scale_and_strided_rows(order):
    c = Batch([77, 500, 0, 16], 2, 128, 16, torch.float16, order=order)
    wide = torch.randn(4, 3, 8, 128, generator=gen(1), device=DEV).half()
    q = wide[:, 1]
    out = torch.full((4, 16, 128), 5.0, device=DEV).half()[:, ::2]
    got = kernels.paged_attention(q, *c.cache(), scale=0.3, out=out)
    assert got is out
    for b, n in enumerate(c.lens):
        check(out[b:b + 1], *attend(q[b:b + 1], c.k[b], c.v[b], n - 1, None, 0, 0.3, torch.float16))


def test_decode_reads_only_pages_that_are_seen():
    """Under a window, pages that no visible key needs may be gone: their table
    entries hold ids far outside the pool and nothing is recorded."""
    c = Batch([1000, 2000], 2, 64, 16, torch.float16)
    q = torch.randn(2, 4, 64, generator=gen(2), device=DEV).half()
    want = kernels.paged_attention(q, *c.cache(), window=100, sinks=20)
    good = c.table.clone()
    for b, n in enumerate(c.lens):
        first = (n - 100) // 16
        c.table[b, 2:first] = 2 ** 30
    got = kernels.paged_attention(q, *c.cache(), window=100, sinks=20)
    kernels.check_device_error()
    assert torch.equal(got, want) and torch.isfinite(got.float()).all()
    off = torch.tensor([0, 40, 90], dtype=torch.int32, device=DEV)
    q = torch.randn(90, 4, 64, generator=gen(2), device=DEV).half()
    c.table[:] = good
    for b, n in enumerate(c.lens):   # the rows reach 40 / 50 positions further back
        c.table[b, 2:(n - 150) // 16] = 2 ** 30
    got = kernels.prompt_attention(q, *c.cache(), off, window=100, sinks=20)
    kernels.check_device_error()
    for b, n in enumerate(c.lens):
        rows = slice(int(off[b]), int(off[b + 1]))
        check(got[rows], *attend(q[rows], c.k[b], c.v[b], n - int(off[b + 1] - off[b]), 100, 20, 0.125, torch.float16))


def test_bad_indexes_are_skipped_and_recorded():
    """A page id outside the pool hides its keys; a length past the table is cut."""
    from liteweight_b200._native import LiteweightError
    page = 16
    for bad in (-1, 10 ** 6):
        c = Batch([100, 64], 2, 64, page, torch.float16)
        c.table[0, 2] = bad
        q = torch.randn(2, 4, 64, generator=gen(2), device=DEV).half()
        got = kernels.paged_attention(q, *c.cache())
        with pytest.raises(LiteweightError, match="out of range"):
            kernels.check_device_error()
        kernels.check_device_error()   # reported once
        kept = torch.cat([torch.arange(32), torch.arange(48, 100)])
        k, v = c.k[0][kept], c.v[0][kept]
        check(got[:1], *attend(q[:1], k, v, 83, None, 0, 0.125, torch.float16))
        check(got[1:], *attend(q[1:], c.k[1], c.v[1], 63, None, 0, 0.125, torch.float16))
        off = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
        got = kernels.prompt_attention(q, *c.cache(), off)
        with pytest.raises(LiteweightError, match="out of range"):
            kernels.check_device_error()
        check(got[:1], *attend(q[:1], k, v, 83, None, 0, 0.125, torch.float16))
    c = Batch([48], 1, 64, page, torch.float16)
    c.kv_lens[0] = 10 ** 9
    c.table = c.table[:, :3]
    q = torch.randn(1, 2, 64, generator=gen(2), device=DEV).half()
    check(kernels.paged_attention(q, *c.cache()), *attend(q, c.k[0], c.v[0], 47, None, 0, 0.125, torch.float16))
    with pytest.raises(LiteweightError, match="out of range"):
        kernels.check_device_error()


@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 0), (20, 5)])
def test_lengths_past_the_table_are_cut(window, sinks):
    """The chunk's rows are then the last the table addresses."""
    from liteweight_b200._native import LiteweightError
    c = Batch([64], 1, 64, 16, torch.float16)
    c.table = c.table[:, :4].contiguous()
    q = torch.randn(30, 2, 64, generator=gen(2), device=DEV).half()
    off = torch.tensor([0, 30], dtype=torch.int32, device=DEV)
    for length in (90, 10 ** 9, 2 ** 31 - 1):
        c.kv_lens[0] = length
        got = kernels.prompt_attention(q, *c.cache(), off, window=window, sinks=sinks)
        with pytest.raises(LiteweightError, match="out of range"):
            kernels.check_device_error()
        check(got, *attend(q, c.k[0], c.v[0], 34, window, sinks, 0.125, torch.float16))
        got = kernels.paged_attention(q[:1], *c.cache(), window=window, sinks=sinks)
        with pytest.raises(LiteweightError, match="out of range"):
            kernels.check_device_error()
        check(got, *attend(q[:1], c.k[0], c.v[0], 63, window, sinks, 0.125, torch.float16))


def test_offsets_past_the_rows_are_refused_on_the_device():
    from liteweight_b200._native import LiteweightError
    c = Batch([40, 30], 1, 64, 16, torch.float16)
    q = torch.randn(20, 2, 64, generator=gen(2), device=DEV).half()
    off = torch.tensor([0, 12, 25], dtype=torch.int32, device=DEV)   # rows 20 .. 24 are not there
    got = kernels.prompt_attention(q, *c.cache(), off)
    with pytest.raises(LiteweightError, match="out of range"):
        kernels.check_device_error()
    check(got[:12], *attend(q[:12], c.k[0], c.v[0], 28, None, 0, 0.125, torch.float16))
    off = torch.tensor([3, 12, 18], dtype=torch.int32, device=DEV)   # rows before the first and behind the last
    got = kernels.prompt_attention(q, *c.cache(), off)
    kernels.check_device_error()
    assert (got[:3] == 0).all() and (got[18:] == 0).all()
    check(got[3:12], *attend(q[3:12], c.k[0], c.v[0], 31, None, 0, 0.125, torch.float16))


def test_largest_windows_and_sinks():
    c = Batch([300, 20], 2, 64, 16, torch.float16)
    q = torch.randn(2, 4, 64, generator=gen(2), device=DEV).half()
    off = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    want, cut = kernels.paged_attention(q, *c.cache()), kernels.paged_attention(q, *c.cache(), window=7, sinks=2)
    for window, sinks, x in ((2 ** 40, 0, want), (2 ** 31 - 1, 2 ** 40, want), (1, 2 ** 31 - 1, want), (7, 2, cut)):
        for got in (kernels.paged_attention(q, *c.cache(), window=window, sinks=sinks),
                    kernels.prompt_attention(q, *c.cache(), off, window=window, sinks=sinks)):
            assert (got.float() - x.float()).abs().max() < 4e-3
    kernels.check_device_error()


def test_far_pages():
    """Offsets past 2^31 elements: a pool of 5 GB of which the last pages are used."""
    nkv, page, hd = 8, 256, 128
    n_pages = (5 << 30) // (2 * nkv * page * hd)
    pools = [torch.empty(n_pages, nkv, page, hd, dtype=torch.float16, device=DEV) for _ in range(2)]
    k, v = (torch.randn(300, nkv, hd, generator=gen(i), device=DEV).half() for i in range(2))
    table = torch.tensor([[n_pages - 1, n_pages - 3]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([300], dtype=torch.int32, device=DEV)
    cos, sin = torch.ones(300, hd, device=DEV), torch.zeros(300, hd, device=DEV)
    off = torch.tensor([0, 300], dtype=torch.int32, device=DEV)
    q = torch.randn(300, nkv, hd, generator=gen(5), device=DEV).half()
    turned = kernels.qk_norm_rope(q, k, v, cos, sin, *pools, table, lens, off)
    assert torch.equal(turned, q)
    got = kernels.prompt_attention(q, *pools, table, lens, off)
    check(got, *attend(q, k, v, 0, None, 0, hd ** -0.5, torch.float16))
    got = kernels.paged_attention(q[299:], *pools, table, lens)
    check(got, *attend(q[299:], k, v, 299, None, 0, hd ** -0.5, torch.float16))
    kernels.check_device_error()


PROMPTS = {
    "one": ([1], [1]), "odd": ([257], [257]), "chunk": ([900], [130]), "ragged": ([130, 64, 700, 5, 1, 333],
                                                                                  [130, 1, 77, 0, 1, 300]),
    "empty": ([40, 0, 3, 0], [17, 0, 3, 0]), "deep": ([4100], [70]),
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nkv,group", [(2, 4), (3, 1), (1, 5), (2, 8), (1, 48)])
@pytest.mark.parametrize("name,page,window,sinks", [
    ("one", 16, None, 0), ("odd", 16, None, 0), ("odd", 64, 33, 4), ("chunk", 32, None, 0), ("chunk", 128, 70, 0),
    ("ragged", 16, None, 0), ("ragged", 256, 1, 0), ("ragged", 64, 100, 70), ("empty", 16, None, 0),
    ("deep", 32, None, 0), ("deep", 16, 1500, 130)])
def test_prompt(dtype, hd, nkv, group, name, page, window, sinks):
    lens, new = PROMPTS[name]
    c = Batch(lens, nkv, hd, page, dtype, seed=hd + group + page)
    off = [0]
    for n in new:
        off.append(off[-1] + n)
    q = (torch.randn(off[-1] + 9, nkv * group, hd, generator=gen(3), device=DEV) * 1.7).to(dtype)
    q[off[-1]:] = float("nan")   # rows behind the last sequence
    offs = torch.tensor(off, dtype=torch.int32, device=DEV)
    got = kernels.prompt_attention(q, *c.cache(), offs, window=window, sinks=sinks)
    kernels.check_device_error()
    assert (got[off[-1]:] == 0).all()
    for b, n in enumerate(lens):
        rows = slice(off[b], off[b + 1])
        if new[b]:
            check(got[rows], *attend(q[rows], c.k[b], c.v[b], n - new[b], window, sinks, hd ** -0.5, dtype))
    out = torch.full_like(got, 3.0)
    kernels.prompt_attention(q, *c.cache(), offs, window=window, sinks=sinks, out=out)
    assert torch.equal(out[:off[-1]], got[:off[-1]]) and (out[off[-1]:] == 3).all()   # left as they were


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window,sinks", [(None, 0), (2000, 150)])
def test_few_rows_of_short_and_long_contexts(hd, window, sinks):
    """A table that can hold far more than the sequences do: the launch provides for
    slices of the keys that only the long ones take; and the same for single tokens."""
    lens, new = [300, 0, 40, 6000, 1], [20, 0, 5, 33, 1]
    c = Batch(lens, 1, hd, 16, torch.bfloat16)
    wide = torch.full((5, 5000), -7, dtype=torch.int32, device=DEV)
    wide[:, :c.table.shape[1]] = c.table
    off = [0, 20, 20, 25, 58, 59]
    q = torch.randn(62, 4, hd, generator=gen(4), device=DEV).bfloat16()
    offs = torch.tensor(off, dtype=torch.int32, device=DEV)
    got = kernels.prompt_attention(q, c.k_pages, c.v_pages, wide, c.kv_lens, offs, window=window, sinks=sinks)
    one = kernels.paged_attention(q[:5], c.k_pages, c.v_pages, wide, c.kv_lens, window=window, sinks=sinks)
    kernels.check_device_error()
    assert (got[59:] == 0).all() and (one[1] == 0).all()
    for b, n in enumerate(lens):
        if n:
            rows = slice(off[b], off[b + 1])
            check(got[rows], *attend(q[rows], c.k[b], c.v[b], n - new[b], window, sinks, hd ** -0.5, torch.bfloat16))
            check(one[b:b + 1], *attend(q[b:b + 1], c.k[b], c.v[b], n - 1, window, sinks, hd ** -0.5, torch.bfloat16))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3)])
def test_prompt_rows_are_not_reached_by_what_they_do_not_see(value, hd, window, sinks):
    """A key and value that hold infinities or NaN: rows that do not see the key
    are what they are without it, rows that see it are not finite."""
    c = Batch([300], 2, hd, 16, torch.bfloat16)
    q = torch.randn(300, 4, hd, generator=gen(3), device=DEV).bfloat16()
    off = torch.tensor([0, 300], dtype=torch.int32, device=DEV)
    for key in (0, 2, 77, 128, 250, 299):
        k, v = c.k[0].clone(), c.v[0].clone()
        v[key, :, 5] = value
        c.put(0, 0, k, v)
        got = kernels.prompt_attention(q, *c.cache(), off, window=window, sinks=sinks)
        p = torch.arange(300, device=DEV)
        seen = (p >= key) & ((p - key < window) | (key < sinks) if window else True)
        clean = c.v[0].clone()
        clean[key] = 0
        want, tol = attend(q, k, clean, 0, window, sinks, hd ** -0.5, torch.bfloat16)
        check(got[~seen], want[~seen], tol[~seen])
        x = got[seen][:, :, 5].float()
        assert (x.isnan().all() if math.isnan(value) else (x == value).all()), "a visible value was lost"
        other = torch.arange(hd, device=DEV) != 5
        check(got[seen][:, :, other], *(y[seen][:, :, other] for y in attend(q, k, c.v[0], 0, window, sinks, hd ** -0.5,
                                                                            torch.bfloat16)))
        k[key] = float("nan")
        c.put(0, 0, k, v)
        got = kernels.prompt_attention(q, *c.cache(), off, window=window, sinks=sinks)
        check(got[~seen], want[~seen], tol[~seen])
        assert got[seen].isnan().all()


def rope_want(q, k, cos, sin, pos, qw, kw, eps):
    outs = []
    hd = q.shape[-1]
    for x, w in ((q, qw), (k, kw)):
        x = x.double()
        if w is not None:
            x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
        r = torch.cat([-x[..., hd // 2:], x[..., :hd // 2]], -1)
        a, b = x * cos.double()[pos][:, None], r * sin.double()[pos][:, None]
        outs.append((a + b, a.abs() + b.abs()))
    return outs


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("f32_table", [True, False])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("nq,nkv,lens,new,page,order", [
    (8, 2, [1], None, 16, "phsd"), (5, 5, [17, 0, 900, 1, 33], None, 32, "pshd"),
    (32, 8, [300, 0, 41, 5], [300, 0, 17, 1], 16, "both"), (12, 1, [2000, 1500], [1999, 1001], 64, "phsd")])
def test_rope(dtype, hd, f32_table, norm, nq, nkv, lens, new, page, order):
    """Against fp64. One rounding of the result (half a step), and fp32 arithmetic:
    the mean, the reciprocal root, two products and a sum, under 32 steps of 2^-24
    of the terms' magnitude (hd terms of one sign in the mean: at most hd 2^-24,
    halved by the root)."""
    c = Batch(lens, nkv, hd, page, dtype, order=order)
    g = gen(hd + nq)
    counts = new or [1] * len(lens)
    off = [0]
    for n in counts:
        off.append(off[-1] + n)
    T = off[-1] + (3 if new else 0)
    packed = torch.randn(T, nq + 2 * nkv, hd, generator=g, device=DEV).to(dtype)
    q, k, v = packed[:, :nq], packed[:, nq:nq + nkv], packed[:, nq + nkv:]
    cos, sin = (torch.randn(max(lens), hd, generator=g, device=DEV).to(torch.float32 if f32_table else dtype)
                for _ in range(2))
    qw, kw = ((1 + 0.2 * torch.randn(hd, generator=g, device=DEV)).to(dtype) if norm else None for _ in range(2))
    offs = torch.tensor(off, dtype=torch.int32, device=DEV) if new else None
    before = c.k_pages.clone(), c.v_pages.clone()
    got = kernels.qk_norm_rope(q, k, v, cos, sin, *c.cache(), offs, q_weight=qw, k_weight=kw, eps=1e-5)
    kernels.check_device_error()
    h = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    kp, vp = before
    for b, n in enumerate(lens):
        rows = slice(off[b], off[b + 1])
        if n == 0 or counts[b] == 0:
            assert (got[rows] == 0).all()
            continue
        pos = torch.arange(n - counts[b], n, device=DEV)
        (qo, qm), (ko, km) = rope_want(q[rows], k[rows], cos, sin, pos, qw, kw, 1e-5)
        room = (hd / 2 + 32) * 2.0 ** -24
        assert ((got[rows].double() - qo).abs() <= h * qo.abs() + room * qm + tiny).all()
        pages, slots = c.where(b, n - counts[b], counts[b])
        at = c.k_pages[pages, :, slots]
        assert ((at.double() - ko).abs() <= h * ko.abs() + room * km + tiny).all()
        assert torch.equal(c.v_pages[pages, :, slots], v[rows])
        kp[pages, :, slots], vp[pages, :, slots] = at, v[rows]
    assert (got[off[-1]:] == 0).all()
    for now, then in ((c.k_pages, kp), (c.v_pages, vp)):   # every other slot as it was, NaN for NaN
        assert torch.equal(now.contiguous().view(torch.int16), then.contiguous().view(torch.int16))
    # in place, and rows of no sequence left as they were
    out = torch.full_like(got, 3.0)
    kernels.qk_norm_rope(q, k, v, cos, sin, *c.cache(), offs, q_weight=qw, k_weight=kw, eps=1e-5, out=out)
    mine = torch.zeros(T, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        mine[off[b]:off[b + 1]] = n > 0
    assert torch.equal(out[mine], got[mine]) and (out[~mine] == 3).all()
    kernels.qk_norm_rope(q, k, v, cos, sin, *c.cache(), offs, q_weight=qw, k_weight=kw, eps=1e-5, out=q)
    assert torch.equal(q[mine], got[mine])


def test_rope_skips_what_is_out_of_range():
    from liteweight_b200._native import LiteweightError
    c = Batch([20, 40], 2, 64, 16, torch.float16)
    q = torch.randn(2, 4, 64, generator=gen(1), device=DEV).half()
    k, v = q[:, :2].contiguous(), q[:, 2:].contiguous()
    cos, sin = torch.ones(40, 64, device=DEV), torch.zeros(40, 64, device=DEV)
    kept = c.k_pages.clone(), c.v_pages.clone()

    def unchanged():
        return all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip((c.k_pages, c.v_pages), kept))

    good = c.table.clone()
    c.table[:] = 10 ** 6
    got = kernels.qk_norm_rope(q, k, v, cos, sin, *c.cache())
    with pytest.raises(LiteweightError, match="out of range"):
        kernels.check_device_error()
    assert unchanged() and torch.equal(got, q)
    c.table[:] = good
    for lens in ([10 ** 9, 10 ** 9], [60, 60]):   # past the rotation table, past the page table
        c.kv_lens[:] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        got = kernels.qk_norm_rope(q, k, v, cos, sin, *c.cache())
        with pytest.raises(LiteweightError, match="out of range"):
            kernels.check_device_error()
        assert unchanged() and (got == 0).all()
    c.kv_lens[:] = 1
    off = torch.tensor([0, 2, 2], dtype=torch.int32, device=DEV)   # two new tokens of a sequence of one
    kernels.qk_norm_rope(q, k, v, cos, sin, *c.cache(), off)
    with pytest.raises(LiteweightError, match="out of range"):
        kernels.check_device_error()


def test_a_run_of_them():
    """Prompts in two chunks, then new tokens one by one, as a layer of a served
    model runs them, against attention over everything in fp64."""
    nq, nkv, hd, page, dtype = 8, 2, 64, 16, torch.float16
    total, first = [150, 40, 260], [100, 40, 30]
    steps = 5
    g = gen(11)
    c = Batch([n + steps for n in total], nkv, hd, page, dtype)
    qkv = [torch.randn(n + steps, nq + 2 * nkv, hd, generator=g, device=DEV).half() for n in total]
    ang = torch.arange(300, device=DEV)[:, None] * 1e4 ** (-torch.arange(0, hd, 2, device=DEV) / hd)
    cos, sin = torch.cat([ang, ang], -1).cos(), torch.cat([ang, ang], -1).sin()
    qw, kw = ((1 + 0.1 * torch.randn(hd, generator=g, device=DEV)).half() for _ in range(2))
    c.k_pages.fill_(float("nan"))
    c.v_pages.fill_(float("nan"))
    outs = [[] for _ in total]
    queries = [[] for _ in total]

    def forward(counts, done):
        rows = torch.cat([qkv[b][done[b]:done[b] + n] for b, n in enumerate(counts)])
        q, k, v = rows[:, :nq], rows[:, nq:nq + nkv], rows[:, nq + nkv:]
        c.kv_lens[:] = torch.tensor([d + n for d, n in zip(done, counts)], dtype=torch.int32, device=DEV)
        off = [0]
        for n in counts:
            off.append(off[-1] + n)
        single = all(n == 1 for n in counts)
        offs = None if single else torch.tensor(off, dtype=torch.int32, device=DEV)
        q = kernels.qk_norm_rope(q, k, v, cos, sin, *c.cache(), offs, q_weight=qw, k_weight=kw)
        o = kernels.paged_attention(q, *c.cache()) if single else kernels.prompt_attention(q, *c.cache(), offs)
        for b in range(len(counts)):
            outs[b].append(o[off[b]:off[b + 1]])
            queries[b].append(q[off[b]:off[b + 1]])
        return [d + n for d, n in zip(done, counts)]

    done = forward(first, [0, 0, 0])
    done = forward([t - d for t, d in zip(total, done)], done)
    for _ in range(steps):
        done = forward([1, 1, 1], done)
    kernels.check_device_error()
    for b, n in enumerate(total):
        pages, slots = c.where(b, 0, n + steps)
        k, v = c.k_pages[pages, :, slots], c.v_pages[pages, :, slots]
        q = torch.cat(queries[b])
        (qo, qm), (ko, km) = rope_want(qkv[b][:, :nq], qkv[b][:, nq:nq + nkv], cos, sin,
                                       torch.arange(n + steps, device=DEV), qw, kw, 1e-6)
        for x, want, mag in ((q, qo, qm), (k, ko, km)):
            assert ((x.double() - want).abs() <= 2.0 ** -11 * want.abs() + 64 * 2.0 ** -24 * mag + 2.0 ** -25).all()
        check(torch.cat(outs[b]), *attend(q, k, v, 0, None, 0, hd ** -0.5, dtype))


def test_same_bits_every_time_and_on_other_streams():
    c = Batch([4000, 31, 0, 900], 2, 128, 32, torch.bfloat16)
    q = torch.randn(4, 16, 128, generator=gen(2), device=DEV).bfloat16()
    off = torch.tensor([0, 1, 2, 2, 4], dtype=torch.int32, device=DEV)
    one = kernels.paged_attention(q, *c.cache()), kernels.prompt_attention(q, *c.cache(), off)
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for s in streams:   # two calls at once
            with torch.cuda.stream(s):
                got.append((kernels.paged_attention(q, *c.cache()), kernels.prompt_attention(q, *c.cache(), off)))
        torch.cuda.synchronize()
        for pair in got:
            assert torch.equal(pair[0], one[0]) and torch.equal(pair[1], one[1])


def test_graphs():
    """Captured calls read lengths, table and inputs anew on every replay; two
    graphs replayed at once on two streams do not share scratch."""
    lens = [700, 90]
    c = Batch(lens, 2, 128, 16, torch.float16)
    d = Batch([3, 2000], 2, 128, 16, torch.float16, seed=9)
    q = torch.randn(2, 8, 128, generator=gen(2), device=DEV).half()
    off = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    k, v = (torch.randn(2, 2, 128, generator=gen(i), device=DEV).half() for i in (3, 4))
    cos, sin = torch.ones(4000, 128, device=DEV), torch.zeros(4000, 128, device=DEV)

    def step(x):
        r = kernels.qk_norm_rope(q.clone(), k, v, cos, sin, *x.cache())
        return kernels.paged_attention(r, *x.cache()), kernels.prompt_attention(r, *x.cache(), off)

    graphs, outs = [], []
    for x in (c, d):
        step(x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(x))
        graphs.append(g)
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    for i in range(8):
        c.kv_lens[0], d.kv_lens[1] = 700 - 50 * i, 2000 - 120 * i
        q.copy_(torch.randn(2, 8, 128, generator=gen(50 + i), device=DEV).half())
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for x, o in zip((c, d), outs):
            want = step(x)
            torch.cuda.synchronize()
            assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
    kernels.check_device_error()


def test_two_threads():
    """Calls of several host threads at once, each on its own stream."""
    import threading
    c = Batch([900, 40], 2, 128, 16, torch.float16)
    q = torch.randn(2, 8, 128, generator=gen(2), device=DEV).half()
    off = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    want = kernels.paged_attention(q, *c.cache()), kernels.prompt_attention(q, *c.cache(), off)
    torch.cuda.synchronize()
    wrong = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream(DEV)):
            for _ in range(50):
                got = kernels.paged_attention(q, *c.cache()), kernels.prompt_attention(q, *c.cache(), off)
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want)):
                wrong.append(1)

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_first_calls_of_a_process_may_be_captured():
    import subprocess
    import sys
    code = """
import torch
from liteweight_b200 import kernels
k = torch.randn(8, 2, 16, 64, device="cuda").half()
table = torch.arange(8, device="cuda", dtype=torch.int32).view(2, 4)
lens = torch.tensor([40, 64], device="cuda", dtype=torch.int32)
off = torch.tensor([0, 1, 2], device="cuda", dtype=torch.int32)
q = torch.randn(2, 4, 64, device="cuda").half()
cos, sin = torch.ones(64, 64, device="cuda"), torch.zeros(64, 64, device="cuda")
new = torch.zeros(2, 2, 64, device="cuda").half()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    r = kernels.qk_norm_rope(q, new, new, cos, sin, k, k.clone(), table, lens)
    a, b = kernels.paged_attention(r, k, k, table, lens), kernels.prompt_attention(r, k, k, table, lens, off)
g.replay()
torch.cuda.synchronize()
assert torch.equal(r, q) and (a.float() - b.float()).abs().max() < 4e-3
kernels.check_device_error()
"""
    from pathlib import Path
    subprocess.run([sys.executable, "-c", code], check=True, timeout=120, cwd=Path(__file__).resolve().parent.parent)


def test_empty_batches():
    c = Batch([5], 2, 64, 16, torch.float16)
    none = torch.empty(0, 4, 64, dtype=torch.float16, device=DEV)
    assert kernels.paged_attention(none, c.k_pages, c.v_pages, c.table[:0], c.kv_lens[:0]).shape == (0, 4, 64)
    off = torch.zeros(2, dtype=torch.int32, device=DEV)
    assert kernels.prompt_attention(none, *c.cache(), off).shape == (0, 4, 64)
    rows = torch.ones(3, 4, 64, dtype=torch.float16, device=DEV)
    assert (kernels.prompt_attention(rows, *c.cache(), off) == 0).all()
    assert (kernels.paged_attention(rows, c.k_pages[:0], c.v_pages[:0], torch.empty(3, 0, dtype=torch.int32, device=DEV),
                                    torch.zeros(3, dtype=torch.int32, device=DEV)) == 0).all()
    assert (kernels.prompt_attention(rows, c.k_pages[:0], c.v_pages[:0], torch.empty(1, 0, dtype=torch.int32, device=DEV),
                                     torch.zeros(1, dtype=torch.int32, device=DEV), off) == 0).all()
    kernels.check_device_error()

"""The paged-cache operators where values, lengths and launches are extreme.

Tolerances as in test_paged_gpu.py (derived there), unless a test states its own.
"""

import math

import pytest
import torch

from liteweight_b200 import kernels
from test_paged_gpu import DEV, DTYPES, Batch, attend, check, gen

pytestmark = pytest.mark.gpu


def offsets(*counts):
    off = [0]
    for n in counts:
        off.append(off[-1] + n)
    return torch.tensor(off, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ weights and scores

def spread_context(n, hd, gap, dtype):
    """One key whose score is `gap` above the others', which are all alike; its
    value is 0, the others' are between 0.5 and 1.5."""
    c = Batch([n], 1, hd, 64, dtype)
    k = torch.zeros_like(c.k[0])
    k[0, 0, 0] = gap
    v = (0.5 + torch.rand(n, 1, hd, generator=gen(4), device=DEV)).to(dtype)
    v[0] = 0
    c.put(0, 0, k, v)
    return c, k, v


def check_spread(got, q, k, v, first, hd, dtype, floor):
    """`floor`: the largest error that the rounding of one weight leaves in the
    result, relative to the sum of the weights. The other terms as in attend():
    every rounding of a weight within its type's normal range is relative."""
    want, _ = attend(q, k, v, first, None, 0, hd ** -0.5, dtype)
    h = torch.finfo(dtype).eps / 2
    n = k.shape[0]
    score = float(k[0, 0, 0])
    rel = 2 * h + (n + 64) * 2.0 ** -23 + 2 * hd * 2.0 ** -23 * score
    tol = rel * want.abs() + floor * v.double().sum(0)[None] + 2.0 ** -25   # values are positive: A = |out|
    check(got, want, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("gap", [16.8, 18.0, 21.0])
@pytest.mark.parametrize("n", [4000, 131071])
def test_many_small_weights_beside_a_large_one(dtype, hd, gap, n):
    """Weights far below the largest add up over a long context. 4000 keys run in
    clusters, 131071 in runs and a join. A fp16 weight is off by at most 2^-25 below
    the normal range; decode keeps its weights up to 2^15 (2^-40 of the largest),
    prompts theirs up to 2^7 of the base they were taken from (2^-32)."""
    c, k, v = spread_context(n, hd, gap, dtype)
    q = torch.zeros(3, 2, hd, device=DEV, dtype=dtype)
    q[:, :, 0] = hd ** 0.5
    got = kernels.paged_attention(q[:1], *c.cache())
    check_spread(got, q[:1], k, v, n - 1, hd, dtype, 2.0 ** -40 if dtype == torch.float16 else 0.0)
    got = kernels.prompt_attention(q, *c.cache(), offsets(3))
    check_spread(got, q, k, v, n - 3, hd, dtype, 2.0 ** -32 if dtype == torch.float16 else 0.0)
    kernels.check_device_error()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size", [300.0, 1000.0, 3000.0])
def test_huge_scores(dtype, hd, size):
    """Scores of 2^19 to 2^26 (times log2 e), where fp32 holds them to whole numbers
    or worse: one key is far above the others, and the result is its value."""
    n = 700
    for seed in range(6):
        c = Batch([n], 1, hd, 16, dtype, seed=seed)
        top = (size * torch.randn(hd, generator=gen(seed), device=DEV)).to(dtype)
        k = c.k[0].clone()
        at = (97 * seed + 5) % (n - 2)
        k[at, 0] = top
        c.put(0, 0, k, c.v[0])
        q = top.expand(2, 1, hd).contiguous()
        want = c.v[0][at].double().expand(2, 1, hd)
        tol = torch.finfo(dtype).eps * want.abs() + 2.0 ** -23   # a weight that is one, up to a rounding; the result's
        check(kernels.paged_attention(q[:1], *c.cache()), want[:1], tol[:1])
        check(kernels.prompt_attention(q, *c.cache(), offsets(2)), want, tol)
    kernels.check_device_error()


# ------------------------------------------------------------------ infinities and NaN that are seen

# a cluster per item; runs whose items lie within one; a long item cut by CTAs; both with a wide group
DECODE_FORMS = {"cluster": ([300, 77], 4), "cluster-wide": ([900], 12), "runs": ([200 + i % 9 for i in range(700)], 4),
                "join": ([20000, 77], 4), "join-wide": ([9000], 12)}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("form", DECODE_FORMS)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_decode_shows_the_infinities_and_nans_that_it_sees(dtype, hd, form, value):
    """A value's infinity or NaN reaches its own dim of the rows that see it and
    nothing else; a key's NaN the whole row of its kv head."""
    lens, group = DECODE_FORMS[form]
    c = Batch(lens, 2, hd, 16, dtype)
    q = torch.randn(len(lens), 2 * group, hd, generator=gen(3), device=DEV).to(dtype)
    dims = torch.arange(hd, device=DEV) != 5
    n = lens[0]
    want, tol = attend(q[:1], c.k[0], c.v[0], n - 1, None, 0, hd ** -0.5, dtype)
    others = kernels.paged_attention(q, *c.cache())[1:]
    for key in (0, 17, n // 2, n - 1):
        k, v = c.k[0].clone(), c.v[0].clone()
        v[key, 1, 5] = value
        c.put(0, 0, k, v)
        got = kernels.paged_attention(q, *c.cache())
        x = got[0, group:, 5].float()
        assert (x.isnan() if math.isnan(value) else x == value).all(), "a visible value was lost"
        check(got[:1, :, dims], want[:, :, dims], tol[:, :, dims])
        check(got[:1, :group], want[:, :group], tol[:, :group])
        assert torch.equal(got[1:], others)
        k[key, 1, 7] = float("nan")
        c.put(0, 0, k, c.v[0])
        got = kernels.paged_attention(q, *c.cache())
        assert got[0, group:].isnan().all()
        check(got[:1, :group], want[:, :group], tol[:, :group])
        assert torch.equal(got[1:], others)
    kernels.check_device_error()


def all_below(c, b, keys):
    """Keys whose score is minus infinity for queries with q[..., 0] > 0."""
    k = c.k[b].clone()
    k[keys, :, 0] = -float("inf")
    c.put(b, 0, k, c.v[b])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("form", DECODE_FORMS)
def test_scores_of_minus_infinity(dtype, hd, form):
    """Such a key has no weight beside others; a row that sees only such keys is
    NaN, as a softmax of them is, where one that sees no key is zero."""
    lens, group = DECODE_FORMS[form]
    c = Batch(lens, 1, hd, 16, dtype)
    q = torch.randn(len(lens), group, hd, generator=gen(3), device=DEV).to(dtype)
    q[..., 0] = q[..., 0].abs() + 0.1
    n = lens[0]
    others = kernels.paged_attention(q, *c.cache())[1:]
    kept = torch.tensor([2, n // 2, n - 2], device=DEV)
    gone = torch.ones(n, dtype=torch.bool, device=DEV)
    gone[kept] = False
    all_below(c, 0, gone)
    want, tol = attend(q[:1], c.k[0][kept], c.v[0][kept], 2, None, 0, hd ** -0.5, dtype)
    got = kernels.paged_attention(q, *c.cache())
    check(got[:1], want, tol)
    assert torch.equal(got[1:], others)
    all_below(c, 0, slice(None))
    got = kernels.paged_attention(q, *c.cache())
    assert got[0].isnan().all() and torch.equal(got[1:], others)
    kernels.check_device_error()
    c.table[0] = -1   # nothing is visible then
    got = kernels.paged_attention(q, *c.cache())
    assert (got[0] == 0).all()
    with pytest.raises(Exception, match="out of range"):
        kernels.check_device_error()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3)])
@pytest.mark.parametrize("width", [40, 2000])
def test_scores_of_minus_infinity_in_prompts(dtype, hd, window, sinks, width):
    """With the wide table the rows' keys are cut into slices."""
    n, rows = 600, 90
    c = Batch([n], 1, hd, 16, dtype)
    wide = torch.full((1, width), -5, dtype=torch.int32, device=DEV)
    wide[:, :-(-n // 16)] = c.table[:, :-(-n // 16)]
    cache = (c.k_pages, c.v_pages, wide, c.kv_lens)
    q = torch.randn(rows, 3, hd, generator=gen(3), device=DEV).to(dtype)
    q[..., 0] = q[..., 0].abs() + 0.1
    p = torch.arange(n - rows, n, device=DEV)
    for kept in ([550], [1, 530, 599], []):
        gone = torch.ones(n, dtype=torch.bool, device=DEV)
        gone[kept] = False
        all_below(c, 0, gone)
        got = kernels.prompt_attention(q, *cache, offsets(rows), window=window, sinks=sinks)
        j = torch.tensor(kept, device=DEV, dtype=torch.int64)[None]
        seen = (j <= p[:, None]) & ((p[:, None] - j < window) | (j < sinks) if window else True)
        some = seen.any(-1)
        for i in range(rows):
            if not some[i]:
                assert got[i].isnan().all(), i
        for mask in seen[some].unique(dim=0) if kept else ():
            at = (seen == mask).all(-1)
            use = torch.tensor(kept, device=DEV)[mask]
            # every row of the group sees all of `use`
            first = [attend(q[i:i + 1], c.k[0][use], c.v[0][use], len(use) - 1, None, 0, hd ** -0.5, dtype)
                     for i in at.nonzero()[:, 0].tolist()]
            check(got[at], torch.cat([x[0] for x in first]), torch.cat([x[1] for x in first]))
    kernels.check_device_error()
    c.table[0] = -1
    got = kernels.prompt_attention(q, *c.cache(), offsets(rows), window=window, sinks=sinks)
    assert (got == 0).all()
    with pytest.raises(Exception, match="out of range"):
        kernels.check_device_error()


# ------------------------------------------------------------------ rows that are refused

@pytest.mark.parametrize("width", [3, 5000])
def test_rows_of_a_refused_sequence(width):
    """A sequence whose rows run past q's is not computed; its rows in q are zero, or
    as they were in a given `out`, with key slices (the wide table) and without.
    What the allocator hands out is NaN and large numbers before the call."""
    c = Batch([40, 30], 1, 64, 16, torch.float16)
    wide = torch.full((2, width), -5, dtype=torch.int32, device=DEV)
    wide[:, :3] = c.table[:, :3]
    cache = (c.k_pages, c.v_pages, wide, c.kv_lens)
    q = torch.randn(320, 2, 64, generator=gen(2), device=DEV).half()
    for off, mine in (([0, 12, 400], slice(0, 12)), ([0, 12, 2 ** 31 - 1], slice(0, 12)),
                      ([-5, 290, 320], slice(290, 320)), ([-300, 290, 320], slice(290, 320))):
        counts = [b - a for a, b in zip(off, off[1:])]
        b = 0 if mine.start == 0 else 1
        want, tol = attend(q[mine], c.k[b], c.v[b], c.lens[b] - counts[b], None, 0, 0.125, torch.float16)
        offs = torch.tensor(off, dtype=torch.int32, device=DEV)
        theirs = torch.ones(320, dtype=torch.bool, device=DEV)
        theirs[mine] = False
        for given in (False, True):
            for shape, dtype, value in (((320, 2, 64), torch.float16, float("nan")), ((1 << 24,), torch.int32, 7)):
                left = [torch.full(shape, value, dtype=dtype, device=DEV) for _ in range(3)]
                del left
            out = torch.full_like(q, 3.0) if given else None
            got = kernels.prompt_attention(q, *cache, offs, out=out)
            with pytest.raises(Exception, match="out of range"):
                kernels.check_device_error()
            check(got[mine], want, tol)
            assert (got[theirs] == (3 if given else 0)).all()


# ------------------------------------------------------------------ the error word

def test_a_wait_that_gave_up_is_reported_before_an_index(tmp_path):
    """A launch that records both has invalid results, whatever came first. The word
    is the one every .cu file of the library has, here in a small library of its own."""
    import ctypes
    import subprocess

    from liteweight_b200 import build
    src = tmp_path / "word.cu"
    src.write_text('#include "lw_common.cuh"\n'
                   "__global__ void record(int a, int b) { if (a) lw::lw_record_error(a); if (b) lw::lw_record_error(b); }\n"
                   'extern "C" int both(int a, int b) { record<<<1, 1>>>(a, b); return lw_tu_take_error(); }\n')
    out = tmp_path / "libword.so"
    subprocess.run([build.nvcc(), *build.ARCH, *build.FLAGS, "-shared", "-I", str(build.CSRC), str(src), "-o", str(out)],
                   check=True, timeout=300)
    lib = ctypes.CDLL(str(out))
    timeout, index = 8, 9
    for a, b, want in ((0, 0, 0), (index, 0, index), (timeout, 0, timeout), (timeout, index, timeout),
                       (index, timeout, timeout), (index, index, index)):
        assert lib.both(a, b) == want
        assert lib.both(0, 0) == 0


def test_errors_of_calls_still_running_on_other_streams():
    """check_device_error waits for them."""
    c = Batch([100], 2, 64, 16, torch.float16)
    q = torch.randn(1, 4, 64, generator=gen(2), device=DEV).half()
    kernels.paged_attention(q, *c.cache())
    c.table[0, 2] = 10 ** 6
    torch.cuda.synchronize()
    kernels.check_device_error()
    with torch.cuda.stream(torch.cuda.Stream(DEV)):
        torch.cuda._sleep(200_000_000)   # cycles: about 0.1 s
        kernels.paged_attention(q, *c.cache())
    with pytest.raises(Exception, match="out of range"):
        kernels.check_device_error()
    kernels.check_device_error()


# ------------------------------------------------------------------ many first keys beside a window

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("sinks", [128, 130, 512, 1000, 1900])
@pytest.mark.parametrize("new", [77, 2000])
def test_sinks_that_fill_tiles(dtype, hd, sinks, new):
    """First keys that every row sees, those that part of the rows' windows reach,
    and what an infinity in the one or the other gives."""
    n, window, group = 2000, 90, 5
    c = Batch([n], 1, hd, 32, dtype)
    q = torch.randn(new, group, hd, generator=gen(6), device=DEV).to(dtype)
    first = n - new
    want, tol = attend(q, c.k[0], c.v[0], first, window, sinks, hd ** -0.5, dtype)
    check(kernels.prompt_attention(q, *c.cache(), offsets(new), window=window, sinks=sinks), want, tol)
    p = torch.arange(first, n, device=DEV)
    dims = torch.arange(hd, device=DEV) != 5
    for key in (0, 127, sinks - 1, sinks, n - 60, n - 1):
        v = c.v[0].clone()
        v[key, 0, 5] = float("inf")
        c.put(0, 0, c.k[0], v)
        got = kernels.prompt_attention(q, *c.cache(), offsets(new), window=window, sinks=sinks)
        seen = (p >= key) & ((p - key < window) | (key < sinks))
        assert (got[seen][:, :, 5] == float("inf")).all()
        check(got[~seen], want[~seen], tol[~seen])
        check(got[:, :, dims], want[:, :, dims], tol[:, :, dims])
        c.put(0, 0, c.k[0], c.v[0])
    kernels.check_device_error()


def test_an_infinity_beside_many_sinks_costs_what_it_costs_beside_few():
    """Only tiles that part of the rows see are searched for it: walking all first
    keys took 46 times as long for 16384 of them as for 256, and past some 340000 a row
    tile's walk would outlast the other warps' bounded waits."""
    hd, new, batch, window = 128, 128, 10, 100
    took = []
    for sinks in (256, 16384):
        n = sinks + 512
        c = Batch([n], 8, hd, 64, torch.float16)
        v = c.v[0].clone()
        v[n - 5, :, 3] = float("inf")
        c.put(0, 0, c.k[0], v)
        table = c.table[:, :-(-n // 64)].expand(batch, -1).contiguous()   # the same pages for all
        lens = c.kv_lens.expand(batch).contiguous()
        q = torch.randn(new * batch, 16, hd, generator=gen(1), device=DEV).half()
        call = lambda: kernels.prompt_attention(q, c.k_pages, c.v_pages, table, lens, offsets(*[new] * batch),  # noqa: E731
                                                window=window, sinks=sinks)
        got = call()
        want, tol = attend(q[:new], c.k[0], c.v[0], n - new, window, sinks, hd ** -0.5, torch.float16)
        dims = torch.arange(hd, device=DEV) != 3
        check(got[:new, :, dims], want[:, :, dims], tol[:, :, dims])
        seen = torch.arange(n - new, n, device=DEV) >= n - 5
        assert (got[:new][seen][:, :, 3] == float("inf")).all()
        check(got[:new][~seen], want[~seen], tol[~seen])
        times = []
        for _ in range(3):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            call()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        took.append(min(times))
    kernels.check_device_error()
    assert took[1] < 5 * took[0], took


# ------------------------------------------------------------------ layouts

def test_strides_of_dimensions_of_one_element():
    """They address nothing, so any will do: one token, one kv head, one page, one position."""
    hd = 64

    def odd(x, *dims):   # the same tensor, with strides of 3 for these dimensions of one element
        assert all(x.shape[d] == 1 for d in dims)
        return x.as_strided(x.shape, [3 if d in dims else s for d, s in enumerate(x.stride())])

    pools = [torch.randn(1, 1, 16, hd, generator=gen(i), device=DEV).half() for i in range(2)]
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    lens = torch.ones(1, dtype=torch.int32, device=DEV)
    off = offsets(1)
    q, k, v = (torch.randn(1, n, hd, generator=gen(9), device=DEV).half() for n in (4, 1, 1))
    cos, sin = (torch.randn(1, hd, generator=gen(i), device=DEV) for i in range(2))
    results = []
    for make in (lambda x, *dims: x.clone(), odd):
        kp, vp = (make(x.clone(), 0, 1) for x in pools)
        out = make(torch.zeros(1, 4, hd, device=DEV).half(), 0)
        got = kernels.qk_norm_rope(make(q, 0), make(k, 0, 1), make(v, 0, 1), make(cos, 0), make(sin, 0), kp, vp, table,
                                   lens, out=out)
        lens += 5
        one = kernels.paged_attention(make(got, 0), kp, vp, table, lens)
        all_of_it = kernels.prompt_attention(make(got, 0), kp, vp, table, lens, off, out=make(torch.zeros_like(q), 0))
        lens -= 5
        results.append([got, kp, vp, one, all_of_it])
    # cos a row of a wide tensor, sin one of a narrow one
    wide = torch.cat([cos, cos], dim=1)[:, :hd]
    kp, vp = (x.clone() for x in pools)
    results.append([kernels.qk_norm_rope(q, k, v, wide, sin, kp, vp, table, lens), kp, vp])
    kernels.check_device_error()
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ launches of more work than the GPU takes at once

def prompt_blocks(rows, group, nkv, batch):
    """Blocks of a prompt_attention launch without key slices: 2 * (128 // group) positions each."""
    return (rows // (2 * (128 // group)) + batch) * nkv


# ragged, with sequences of no and of one new token, cached prefixes, and a last row tile that is not full
MANY = ([1, 700, 0, 333, 64, 0, 1, 415, 37], [0, 150, 9, 1000, 64, 40, 700, 0, 3])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nkv,group", [(2, 48), (2, 64), (3, 33)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (130, 0), (70, 5)])
def test_blocks_take_over_the_work_of_others(dtype, hd, nkv, group, window, sinks):
    """Several pieces per CTA: rows of one and of two row tiles, of few and of many key
    tiles follow one another in the same barriers, ring slots and tensor memory."""
    new, before = MANY
    lens = [a + b for a, b in zip(new, before)]
    assert prompt_blocks(sum(new), group, nkv, len(new)) > 2 * torch.cuda.get_device_properties(0).multi_processor_count
    c = Batch(lens, nkv, hd, 16, dtype, seed=group)
    off = offsets(*new)
    q = (torch.randn(sum(new), nkv * group, hd, generator=gen(3), device=DEV) * 1.7).to(dtype)
    got = kernels.prompt_attention(q, *c.cache(), off, window=window, sinks=sinks)
    kernels.check_device_error()
    at = 0
    for b, n in enumerate(new):
        rows = slice(at, at + n)
        at += n
        if n:
            check(got[rows], *attend(q[rows], c.k[b], c.v[b], before[b], window, sinks, hd ** -0.5, dtype))
    for _ in range(3):
        assert torch.equal(kernels.prompt_attention(q, *c.cache(), off, window=window, sinks=sinks), got)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 3)])
def test_an_infinity_of_one_piece_stays_out_of_the_next(hd, window, sinks):
    """A CTA's piece whose values were searched and mended, then pieces that do not see the infinity."""
    n, nkv, group, dtype = 900, 2, 48, torch.bfloat16
    lens = [n, 200, 300]
    assert prompt_blocks(sum(lens), group, nkv, 3) > 2 * torch.cuda.get_device_properties(0).multi_processor_count
    c = Batch(lens, nkv, hd, 32, dtype)
    q = torch.randn(sum(lens), nkv * group, hd, generator=gen(3), device=DEV).to(dtype)
    off = offsets(*lens)
    clean = kernels.prompt_attention(q, *c.cache(), off, window=window, sinks=sinks)
    p = torch.arange(n, device=DEV)
    for key in (0, 450, 801):
        v = c.v[0].clone()
        v[key, 1, 5] = float("inf")
        c.put(0, 0, c.k[0], v)
        got = kernels.prompt_attention(q, *c.cache(), off, window=window, sinks=sinks)
        seen = (p >= key) & ((p - key < window) | (key < sinks) if window else True)
        assert (got[:n][seen][:, group:, 5] == float("inf")).all()
        want, tol = attend(q[:n], c.k[0], c.v[0], 0, window, sinks, hd ** -0.5, dtype)
        check(got[:n][~seen], want[~seen], tol[~seen])
        check(got[:n, :group], want[:, :group], tol[:, :group])
        dims = torch.arange(hd, device=DEV) != 5
        check(got[:n][:, :, dims], want[:, :, dims], tol[:, :, dims])
        assert torch.equal(got[n:], clean[n:])   # sequences that do not hold the key
        c.put(0, 0, c.k[0], c.v[0])
    kernels.check_device_error()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,nkv,group", [(64, 2, 4), (128, 1, 8), (128, 2, 12)])
@pytest.mark.parametrize("lens,window,sinks", [
    ([131071], None, 0), ([40001, 3, 90000, 0], None, 0), ([131071, 70000], 60000, 5000)])
def test_decode_over_long_contexts(dtype, hd, nkv, group, lens, window, sinks):
    """One item spans dozens of CTAs, whose pieces the second kernel joins."""
    c = Batch(lens, nkv, hd, 64, dtype, seed=hd)
    q = (torch.randn(len(lens), nkv * group, hd, generator=gen(7), device=DEV) * 1.7).to(dtype)
    got = kernels.paged_attention(q, *c.cache(), window=window, sinks=sinks)
    kernels.check_device_error()
    for b, n in enumerate(lens):
        check(got[b:b + 1], *attend(q[b:b + 1], c.k[b], c.v[b], n - 1, window, sinks, hd ** -0.5, dtype))
    assert torch.equal(kernels.paged_attention(q, *c.cache(), window=window, sinks=sinks), got)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_over_long_contexts(dtype):
    """A chunk far into its context, with key slices (few rows) and without (a batch of them)."""
    lens, new = [70001, 5, 66000], [20, 5, 40]
    c = Batch(lens, 2, 64, 64, dtype)
    for copies in (1, 9):
        table, kv = c.table.repeat(copies, 1), c.kv_lens.repeat(copies)
        off = offsets(*(new * copies))
        q = torch.randn(sum(new) * copies, 64, 64, generator=gen(3), device=DEV).to(dtype)
        got = kernels.prompt_attention(q, c.k_pages, c.v_pages, table, kv, off)
        kernels.check_device_error()
        for i in {0, len(new) * copies - 1, 1}:
            b, rows = i % len(new), slice(int(off[i]), int(off[i + 1]))
            check(got[rows], *attend(q[rows], c.k[b], c.v[b], lens[b] - new[b], None, 0, 0.125, dtype))


# ------------------------------------------------------------------ rope in runs of heads

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("f32_table", [True, False])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("nq,nkv", [(32, 8), (20, 10), (9, 9)])
@pytest.mark.parametrize("order", ["phsd", "pshd", "both"])
def test_rope_in_runs_of_heads(dtype, hd, f32_table, norm, nq, nkv, order):
    """Enough tokens for runs of 8 heads, full ones and remainders; tolerances as in test_rope."""
    lens, new = [3001, 17, 0, 2500], [2990, 17, 0, 2201]
    T = sum(new) + 5
    runs = -(-nq // 8) + 2 * -(-nkv // 8)
    assert T * runs * (hd // 16) >= 256 * 2 * torch.cuda.get_device_properties(0).multi_processor_count
    from test_paged_gpu import rope_want
    c = Batch(lens, nkv, hd, 64, dtype, order=order)
    g = gen(hd + nq)
    packed = torch.randn(T, nq + 2 * nkv, hd, generator=g, device=DEV).to(dtype)
    q, k, v = packed[:, :nq], packed[:, nq:nq + nkv], packed[:, nq + nkv:]
    cos, sin = (torch.randn(max(lens), hd, generator=g, device=DEV).to(torch.float32 if f32_table else dtype)
                for _ in range(2))
    qw, kw = ((1 + 0.2 * torch.randn(hd, generator=g, device=DEV)).to(dtype) if norm else None for _ in range(2))
    kp, vp = c.k_pages.clone(), c.v_pages.clone()
    got = kernels.qk_norm_rope(q, k, v, cos, sin, *c.cache(), offsets(*new), q_weight=qw, k_weight=kw, eps=1e-5)
    kernels.check_device_error()
    h = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    room = (hd / 2 + 32) * 2.0 ** -24
    at = 0
    for b, n in enumerate(new):
        rows = slice(at, at + n)
        at += n
        if not n:
            continue
        pos = torch.arange(lens[b] - n, lens[b], device=DEV)
        (qo, qm), (ko, km) = rope_want(q[rows], k[rows], cos, sin, pos, qw, kw, 1e-5)
        assert ((got[rows].double() - qo).abs() <= h * qo.abs() + room * qm + tiny).all()
        pages, slots = c.where(b, lens[b] - n, n)
        kept = c.k_pages[pages, :, slots]
        assert ((kept.double() - ko).abs() <= h * ko.abs() + room * km + tiny).all()
        kp[pages, :, slots], vp[pages, :, slots] = kept, v[rows]
    assert (got[at:] == 0).all()
    for now, then in ((c.k_pages, kp), (c.v_pages, vp)):   # v as it was given, every other slot as it was
        assert torch.equal(now.contiguous().view(torch.int16), then.contiguous().view(torch.int16))


# ------------------------------------------------------------------ several host threads

def test_every_result_of_several_threads():
    """Each thread on its own stream, every one of its results compared."""
    import threading
    c = Batch([900, 40, 9000], 2, 128, 16, torch.float16)
    q = torch.randn(3, 8, 128, generator=gen(2), device=DEV).half()
    off = offsets(1, 1, 1)
    k, v = (torch.randn(3, 2, 128, generator=gen(i), device=DEV).half() for i in (3, 4))
    cos, sin = (torch.randn(9000, 128, generator=gen(i), device=DEV) for i in (5, 6))
    spare = [torch.empty_like(x) for x in (c.k_pages, c.v_pages)]   # not what the attention reads

    def calls(pools):
        return (kernels.paged_attention(q, *c.cache()), kernels.prompt_attention(q, *c.cache(), off),
                kernels.qk_norm_rope(q, k, v, cos, sin, *pools, c.table, c.kv_lens))

    want = calls(spare)
    torch.cuda.synchronize()
    done, wrong = [], []

    def work():
        try:
            pools = [torch.empty_like(x) for x in spare]
            with torch.cuda.stream(torch.cuda.Stream(DEV)):
                got = [calls(pools) for _ in range(50)]
                torch.cuda.current_stream().synchronize()
            done.append(sum(all(torch.equal(a, b) for a, b in zip(x, want)) for x in got))
        except BaseException as e:   # noqa: BLE001  (an exception in a thread is a failure here)
            wrong.append(e)

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and done == [50] * 3
    kernels.check_device_error()


# ------------------------------------------------------------------ lengths and batches

@pytest.mark.parametrize("window,sinks", [(None, 0), (3, 0), (3, 1), (2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("hd,group", [(64, 4), (128, 1)])
def test_more_rows_than_the_length_counts(window, sinks, hd, group):
    """Rows before the first token see nothing; the others are right; recorded."""
    for rows, length in ((12, 5), (300, 5), (300, 290), (9, 0)):
        c = Batch([length, 50], 1, hd, 16, torch.float16)
        q = torch.randn(rows + 20, group, hd, generator=gen(2), device=DEV).half()
        got = kernels.prompt_attention(q, *c.cache(), offsets(rows, 20), window=window, sinks=sinks)
        with pytest.raises(Exception, match="out of range"):
            kernels.check_device_error()
        early = rows - length
        assert (got[:early] == 0).all()
        if length:
            check(got[early:rows], *attend(q[early:rows], c.k[0], c.v[0], 0, window, sinks, hd ** -0.5, torch.float16))
        check(got[rows:], *attend(q[rows:], c.k[1], c.v[1], 30, window, sinks, hd ** -0.5, torch.float16))


@pytest.mark.parametrize("batch", [33, 70, 1025, 4000])
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 2)])
def test_prompts_and_steps_of_many_sequences(batch, window, sinks):
    """A row tile finds its sequence among thousands, many of them without a new token."""
    g = torch.Generator().manual_seed(batch)
    new = [int(x) if y > 0 else 0 for x, y in zip(torch.randint(1, 6, (batch,), generator=g),
                                                 torch.randint(0, 3, (batch,), generator=g))]
    new[batch // 2], new[batch - 1] = 150, 77
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 40, (batch,), generator=g))]
    hd, dtype = 64, torch.bfloat16
    width = -(-max(lens) // 16)
    # sequences of a batch share a few pages: enough of them to tell one from another
    n_pages = 500
    pools = [torch.randn(n_pages, 1, 16, hd, generator=gen(i), device=DEV).to(dtype) for i in range(2)]
    table = torch.randint(0, n_pages, (batch, width), generator=gen(5), device=DEV, dtype=torch.int32)
    kv = torch.tensor(lens, dtype=torch.int32, device=DEV)
    off = offsets(*new)
    q = torch.randn(sum(new) + 3, 3, hd, generator=gen(7), device=DEV).to(dtype)
    got = kernels.prompt_attention(q, *pools, table, kv, off, window=window, sinks=sinks)
    step = torch.randn(batch, 3, hd, generator=gen(8), device=DEV).to(dtype)
    one = kernels.paged_attention(step, *pools, table, kv, window=window, sinks=sinks)
    kernels.check_device_error()
    assert (got[sum(new):] == 0).all()
    at = 0
    for b, n in enumerate(new):
        if batch <= 70 or b % 41 == 0 or n > 5 or b > batch - 20:
            k, v = (x[table[b].long()].transpose(1, 2).reshape(-1, 1, hd)[:lens[b]] for x in pools)
            if n:
                check(got[at:at + n], *attend(q[at:at + n], k, v, lens[b] - n, window, sinks, 0.125, dtype))
            if lens[b]:
                check(one[b:b + 1], *attend(step[b:b + 1], k, v, lens[b] - 1, window, sinks, 0.125, dtype))
            else:
                assert (one[b] == 0).all()
        at += n


def test_a_captured_padded_batch():
    """One graph, replayed for batches of other lengths, offsets and pages: rows behind the last
    sequence are zero and nothing of the replay before is left."""
    hd, rows, batch = 128, 200, 4
    c = Batch([400, 300, 200, 100], 2, hd, 16, torch.float16)
    wide = torch.full((batch, 2000), -9, dtype=torch.int32, device=DEV)   # a server's: far wider than needed
    wide[:, :c.table.shape[1]] = c.table
    packed = torch.randn(rows, 12, hd, generator=gen(2), device=DEV).half()
    cos, sin = torch.ones(500, hd, device=DEV), torch.zeros(500, hd, device=DEV)
    off, lens = offsets(50, 50, 50, 50), c.kv_lens.clone()

    def step():
        q, k, v = packed[:, :8], packed[:, 8:10], packed[:, 10:]
        r = kernels.qk_norm_rope(q, k, v, cos, sin, c.k_pages, c.v_pages, wide, lens, off)
        return r, kernels.prompt_attention(r, c.k_pages, c.v_pages, wide, lens, off, window=250, sinks=3)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rotated, out = step()
    for new, total in (([50, 50, 50, 50], [400, 300, 200, 100]), ([1, 0, 130, 7], [390, 0, 150, 99]),
                       ([0, 0, 0, 0], [0, 0, 0, 0]), ([200, 0, 0, 0], [400, 12, 0, 3]), ([0, 0, 0, 1], [0, 0, 0, 1])):
        off.copy_(offsets(*new))
        lens.copy_(torch.tensor(total, dtype=torch.int32))
        packed.copy_(torch.randn(rows, 12, hd, generator=gen(sum(total)), device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        kernels.check_device_error()
        at = 0
        for b, n in enumerate(new):
            if n:
                pages, slots = c.where(b, 0, total[b])
                k, v = c.k_pages[pages, :, slots], c.v_pages[pages, :, slots]
                assert torch.equal(k[total[b] - n:], packed[at:at + n, 8:10]) and torch.equal(rotated[at:at + n],
                                                                                             packed[at:at + n, :8])
                check(out[at:at + n], *attend(packed[at:at + n, :8], k, v, total[b] - n, 250, 3, hd ** -0.5,
                                              torch.float16))
            at += n
        assert (out[at:] == 0).all() and (rotated[at:] == 0).all()

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

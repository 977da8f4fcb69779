"""GPU tests of the bounds that include/verbo_cache.h states for values of very different
scales in one row (attend), and for kept tokens beside rejected ones (append and free)."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import verbo_b200 as vb  # noqa: E402
from tests.test_gpu_cache import BF16, F16, F32, filled, gathered, i32, queries, widened  # noqa: E402


@pytest.fixture(autouse=True)
def _needs(cuda_lib):
    if not torch.cuda.is_available():
        pytest.fail("gpu tests need a CUDA device")


def check(c, q):
    """Tolerance: a weight is off by 2^-22 of itself and by 2^-39 of a weight of 1 (the largest, so the weights' sum is at
    least that) times the quotient of the scales, which its value's scale cancels: 2^-39 of the largest scale times
    the codes.  Scores as in test_gpu_cache.check_attend: all off by d, they move a weighted mean by less than 4 d of
    its absolute terms; sums' roundings are below 2^-18 of those."""
    got = c.attend(0, q, dtype=F32)
    vb.check()
    group = q.shape[1] // c.heads
    for r, n in enumerate(c.lens.tolist()):
        k, _ = gathered(c, 0, r, n, c.k, c.k_scale)
        v, _ = gathered(c, 0, r, n, c.v, c.v_scale)
        codes, _ = gathered(c, 0, r, n, c.v, torch.ones_like(c.v_scale))
        x = q[r].double().view(c.heads, group, c.dim)
        s = x @ k.transpose(1, 2) / math.sqrt(c.dim)
        w = torch.softmax(s, 2)
        want = w @ v
        sums = (x.abs() @ k.abs().transpose(1, 2)).amax(2) / math.sqrt(c.dim)
        large = x.abs().amax(2) * k.abs().sum(2).amax(1)[:, None] / math.sqrt(c.dim)
        d = 2.0**-22 * (large + 16 * sums + 3 * (s.abs().amax(2) + 1))
        tol = (4 * d + 2.0**-18)[..., None] * (w @ v.abs()) + 2.0**-39 * float(c.v_scale.max()) * codes.abs().sum(1)[:, None]
        off = (got[r].double().view(c.heads, group, c.dim) - want).abs()
        assert bool((off <= tol + 2.0**-24 * want.abs()).all()), (r, float((off / tol).max()))


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("power", [0, 10, 20, 26, 40])
@pytest.mark.parametrize("dim,group,dtype", [(64, 7, F32), (80, 4, BF16), (128, 12, F16)])
def test_one_block_of_large_values(dim, group, dtype, power, wide):
    """A block whose keys are opposite to the queries, so that its weights are nearly 0, with values up to 2^40 times the
    others'."""
    c = filled([800, 33], 2, dim, 16)
    if wide:
        c = widened(c)
    q = queries(2, 2 * group, dim, dtype, size=0.5).abs()
    for r, at in ((0, 7), (1, 0)):
        p = int(c.table[r, at])
        c.k.view(torch.uint8)[0, p] = 0xFE  # -448
        c.k_scale[0, p] = 2.0**-3
        c.v_scale[0, p] *= 2.0**power
    check(c, q)


def test_tokens_beside_a_rejected_one():
    """Kept tokens are off by half a step of the raised scale, 2^-10 where that is below the smallest normal code, no
    more, once the token that raised it is gone."""
    c = vb.PagedCache.new(1, 4, 1, 64, 1, 4, 16)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(8, 1, 64, generator=g, device="cuda")
    start, _ = c.reserve(i32([7]))
    c.append(0, x[:7], x[:7], start)
    before = gathered(c, 0, 0, 7, c.v, c.v_scale)[0]
    start, _ = c.reserve(i32([1]))
    c.append(0, x[7:], 1e4 * x[7:], start)
    c.free(i32([7]))
    scale = float(c.v_scale[0, int(c.table[0, 0]), 0, 0])
    after = gathered(c, 0, 0, 7, c.v, c.v_scale)[0]
    assert scale > 1 and bool(((after - before).abs() <= torch.maximum(before.abs() * 2.0**-4, torch.tensor(scale * 2.0**-10))).all())
    assert not torch.equal(after, before)
    vb.check()

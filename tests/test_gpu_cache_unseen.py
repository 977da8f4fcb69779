"""GPU tests of attention of several tokens a row (verbo_cache_attend) where values are
NaN at places that only the later of them see: the earlier ones' results are those
without that place, to the last bit, and the later ones' NaN in its dims alone."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import verbo_b200 as vb  # noqa: E402
from tests.test_gpu_cache import BF16, F16, F32, check_attend, filled, i32, queries, tokens, widened  # noqa: E402

NAN = 0x7F


@pytest.fixture(autouse=True)
def _needs(cuda_lib):
    if not torch.cuda.is_available():
        pytest.fail("gpu tests need a CUDA device")


def place(c, row, i):
    return int(c.table[row, i // c.page]), i % c.page


def seen_nans(c, lens, steps, heads, nan):
    """Which results see one of `nan`: (row, place, head, dim)s; dim None: the scale
    of the place's block."""
    out = torch.zeros(len(lens), steps, heads, c.dim, dtype=torch.bool)
    group = heads // c.heads
    for row, i, head, dim in nan:
        for s in range(steps):
            if (i if dim is not None else i // 16 * 16) < lens[row] - (steps - 1 - s):
                out[row, s, head * group:(head + 1) * group, slice(None) if dim is None else dim] = True
    return out.view(-1, heads, c.dim)


def both(c, q, lens, steps, nan):
    """Against the same cache with zeros in the NaNs' places."""
    want = check_attend(c, q)  # 64 bits
    for row, i, head, dim in nan:
        p, at = place(c, row, i)
        if dim is None:
            c.v_scale[0, p, head, at // 16] = 0.0
        else:
            c.v.view(torch.uint8)[0, p, head, at, dim] = 0
    zero = c.attend(0, q)
    for row, i, head, dim in nan:
        p, at = place(c, row, i)
        if dim is None:
            c.v_scale[0, p, head, at // 16] = float("nan") if i % 2 else float("inf")
        else:
            c.v.view(torch.uint8)[0, p, head, at, dim] = NAN | (i % 2) << 7
    got = c.attend(0, q)
    vb.check()
    mask = seen_nans(c, lens, steps, q.shape[1], nan).cuda()
    assert torch.equal(torch.isnan(got), mask)
    assert torch.equal(got[~mask], zero[~mask])
    untouched = sorted(set(range(len(lens))) - {n[0] for n in nan})
    for r in untouched:
        assert torch.equal(got[r * steps:(r + 1) * steps], want[r * steps:(r + 1) * steps])


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("heads,group,steps", [(2, 2, 4), (1, 7, 5), (2, 1, 32), (1, 4, 2)])
def test_nan_values_of_later_tokens(dim, dtype, heads, group, steps, wide):
    """A row's last tokens, in its last block, over a block's and a page's border, in a row shorter than the steps."""
    lens = [300, 33, 49, 64, 3, 100]
    c = filled(lens, heads, dim, 16)
    if wide:
        c = widened(c)
    q = queries(len(lens) * steps, heads * group, dim, dtype)
    h = heads - 1
    nan = [(0, 299, 0, 3), (0, 298, h, dim - 1), (1, 32, h, 0), (2, 48, 0, 5), (2, 47, 0, 15), (2, 46, 0, 5),
           (3, 63, h, dim // 2), (4, 2, 0, 9), (4, 0, h, 8), (5, 20, 0, 1)]
    both(c, q, lens, steps, nan)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dim,group,dtype", [(64, 3, F32), (96, 2, BF16), (128, 4, F16), (128, 1, F32)])
def test_a_later_blocks_scale_that_is_no_number(dim, group, dtype, wide):
    """A block that the first of four tokens do not see, with a scale of NaN or infinity."""
    lens = [49, 50, 18, 160]
    c = filled(lens, 2, dim, 32)
    if wide:
        c = widened(c)
    q = queries(len(lens) * 4, 2 * group, dim, dtype)
    both(c, q, lens, 4, [(0, 48, 1, None), (1, 48, 0, None), (1, 49, 0, 4), (2, 17, 1, None)])


def test_appended_nan():
    """As a speculation brings it: the last of three new tokens has a NaN among its values."""
    c = filled([20, 45], 2, 64, 16, spare=8, width=8)
    q = queries(6, 4, 64, BF16)
    k, v = tokens(6, 2, 64, BF16, 3), tokens(6, 2, 64, BF16, 4)
    v[5, 1, 7] = 0.0
    start, _ = c.reserve(i32([3, 3]))
    c.append(0, k, v, start)
    want = c.attend(0, q)
    v[5, 1, 7] = float("nan")
    c.append(0, k, v, start)
    got = c.attend(0, q)
    mask = torch.zeros_like(got, dtype=torch.bool)
    mask[5, 2:, 7] = True
    assert torch.equal(torch.isnan(got), mask) and torch.equal(got[~mask], want[~mask])

"""GPU tests of how near a row's sum (verbo_beam_select's lse) comes to 64 bits.

A beam's score is chosen as minus its first token's log-probability, so that the value
that comes back is the error of lse and what rounding the score left.

Tolerance.  A term e^(x - ref) with its reference at most 1 below it and at most the row's
maximum M above: d = x - ref is rounded once and its product with log2(e) once, 2^-24 |d| of the
term each; the exponential is off by 2^-22 of it, and nine fp32 additions at most by 2^-24 each:
less than 2^-23 (|d| + 6.5) with |d| <= max(1, M - x).  A column that stands out by more than 1 is
counted in 64 bits: it has no error.  What is done in 64 bits stays below 1e-12."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import verbo_b200 as vb  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def _needs(cuda_lib):
    if not torch.cuda.is_available():
        pytest.fail("gpu tests need a CUDA device")


def exact(x):
    """(log-probability of the first token, tolerance of lse) of each row, in 64 bits."""
    x = x.double()
    two = x.topk(2, 1).values
    m = two[:, :1]
    w = torch.exp(x - m)
    total = w.sum(1)
    e = 2.0**-23 * ((m - x).clamp(min=1.0) + 6.5)
    e = torch.where((x == m) & (two[:, 1:] < m - 1), 0.0, e)
    return -total.log(), (torch.where(w > 0, w * e, 0.0).sum(1) / total) + 1e-12


def check(x):
    lp, tol = exact(x)
    s = (-lp).float()
    v, p, t = vb.beam_select(x, s, 1, 1)
    vb.check()
    want = s.double() + lp
    off = (v[:, 0].double() - want).abs()
    worst = int((off / tol).argmax())
    assert bool((off <= tol + 2.0**-24 * want.abs()).all()), (worst, float(off[worst]), float(tol[worst]))
    return float(off.max())


def flat(rows, vocab, seed, size=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(rows, vocab, generator=g, device="cuda") * size, g


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab", [(9, 7), (16, 1000), (8, 50257), (8, 151936), (300, 20011)])
def test_one_column_above_the_rest(dtype, rows, vocab):
    """By 1.5 to 45, in the first batch, in the last, in every CTA's part: it makes up the row's sum."""
    x, g = flat(rows, vocab, vocab)
    at = torch.arange(rows, device="cuda") * (vocab - 1) // max(1, rows - 1)
    for above in (1.5, 5.3, 11.7, 20.1, 30.9, 45.3):
        y = x.clone()
        y[torch.arange(rows, device="cuda"), at] = x.amax(1) + above + torch.rand(rows, generator=g, device="cuda")
        off = check(y.to(dtype))
        if above > 11:  # the rest is less than one part in 200
            assert off < 1e-7


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("size", [0.1, 2.0, 4.0, 6.0, 12.0])
def test_rows_of_any_width(dtype, size):
    for rows, vocab in ((5, 151936), (160, 32000), (7, 50257)):
        check(flat(rows, vocab, rows, size)[0].to(dtype))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_a_few_columns_share_the_row(dtype):
    for gap in (0.0, 0.3, 0.9, 1.1, 3.0):
        x, g = flat(40, 60000, int(10 * gap))
        at = torch.rand(40, 60000, generator=g, device="cuda").topk(6, 1).indices
        x.scatter_(1, at, 25.0 - gap * torch.arange(6, device="cuda").float().expand(40, 6))
        check(x.to(dtype))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("low,high", [(-60.0, 30.0), (30.0, -60.0), (-8.0, 8.0)])
def test_rows_that_rise_and_fall(dtype, low, high):
    """Each batch's largest column is above all before it, or below."""
    for rows, vocab in ((3, 100003), (200, 40000)):
        ramp = torch.linspace(low, high, vocab, device="cuda", dtype=torch.float64).expand(rows, vocab)
        check(ramp.to(dtype).contiguous())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_candidates_that_lie_close(dtype):
    """The first of two beams whose best continuations differ by 1e-8 to 1e-6."""
    n, vocab = 200, 33000
    x, g = flat(2 * n, vocab, 3)
    at = torch.randint(0, vocab, (2 * n, 1), generator=g, device="cuda")
    x.scatter_(1, at, x.amax(1, keepdim=True) + 14 + 25 * torch.rand(2 * n, 1, generator=g, device="cuda"))
    x = x.to(dtype)
    lp, tol = exact(x)
    apart = 10.0 ** (-8 + 2 * torch.rand(n, generator=g, device="cuda", dtype=torch.float64))
    apart = torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, apart, -apart)
    s = -lp.view(n, 2)
    s = torch.stack((s[:, 0] + apart, s[:, 1]), 1).float()
    value = s.double() + lp.view(n, 2)
    clear = (value[:, 0] - value[:, 1]).abs() > tol.view(n, 2).sum(1)
    assert int(clear.sum()) > 0.95 * n
    v, p, t = vb.beam_select(x, s.view(-1), 2, 1)
    first = (value[:, 1] > value[:, 0]).int()
    assert torch.equal(p[clear, 0], first[clear])
    assert torch.equal(t[clear, 0], at.view(n, 2).gather(1, first.long()[:, None])[clear, 0].int())

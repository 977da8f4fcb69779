"""GPU tests of the operators around the sampler at the ends of their ranges,
against plain computations in 64 bits.

Tolerances.  u = 2^-24 is half a step of fp32.  A log-probability (v - m) / T -
log s has three roundings of the result's size (the difference, the quotient, the
last subtraction), and log s: one of its own size (CUDA's logf: 1 step, 2u) and the
relative error of s.  A term of s has two exponentials (ex2: 2^-22 each) and its
argument's rounding, weighted by the terms at most log2(vocab) <= 22 bits times 2u;
a term goes through 16 additions in its batch of 32 columns at most, one for each
batch of its thread, and 12 on the way to the row's sum.
"""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NEG = float("-inf")


@pytest.fixture(scope="module")
def vb(cuda_lib):
    if not torch.cuda.is_available():
        pytest.fail("gpu tests need a CUDA device")
    import verbo_b200

    return verbo_b200


# ============================================================== logprobs ==
def in_64_bits(x, ids, top, temp):
    """(logprob, rank, top_ids, top_logprobs), by the definition."""
    t = float(np.float32(temp))
    v = torch.where(torch.isnan(x), torch.full((), NEG, device=x.device, dtype=x.dtype), x).double() + 0.0
    rows, vocab = v.shape
    m = v.max(1, keepdim=True).values
    d = torch.where(v == m, 0.0, (v - m) / t)
    lp = torch.where(v == NEG, NEG, d - d.exp().sum(1, keepdim=True).log())
    mine = v.gather(1, ids[:, None])
    before = (v > mine) | ((v == mine) & (torch.arange(vocab, device="cuda") < ids[:, None]))
    # the first columns: by value, ties by the lower column
    order = torch.sort(v, dim=1, descending=True, stable=True).indices[:, :top] if top else ids[:, None][:, :0]
    best = v.gather(1, order) > NEG
    return (lp.gather(1, ids[:, None])[:, 0], before.sum(1), torch.where(best, order, -1),
            torch.where(best, lp.gather(1, order), NEG))


def check_logprobs(vb, x, ids, top, temp, batches):
    lp, rank, tid, tlp = vb.token_logprobs(x, ids.int(), top=top, temp=temp)
    wlp, wrank, wtid, wtlp = in_64_bits(x, ids, top, temp)
    assert torch.equal(rank.long(), wrank), (temp, rank, wrank)
    assert torch.equal(tid.long(), wtid), (temp, tid, wtid)
    rel = 2.0 ** -21 + 22 * 2 * U + (16 + batches + 12) * U
    logs = np.log(x.shape[1])
    for got, want in ((lp.double(), wlp), (tlp.double(), wtlp)):
        want = torch.where(want < -torch.finfo(F32).max, NEG, want)  # (-3e38 - m) / 1e-4: -inf in fp32
        fin = torch.isfinite(want)
        assert torch.equal(got[~fin], want[~fin]), (temp, got, want)
        tol = 3 * U * (1 + 2.0 ** -20) * (want[fin].abs() + logs) + 2 * U * logs + rel
        off = (got[fin] - want[fin]).abs()
        assert bool((off <= tol).all()), (temp, float((off - tol).max()), got, want)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("fill", [-1e9, -2e9, -5e9, -1e10, 2.5e9, -3e30, -3e38])
def test_logprobs_of_masked_rows(vb, fill, dtype):
    """Rows masked with a large finite value: whole batches of it, where c v (c =
    log2(e) / temp) is so large that its rounding alone is up to 128 and more."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    vocab = 20000
    real = torch.randn(7, vocab, generator=g, device="cuda") * 3
    x = torch.full((7, vocab), fill, device="cuda")
    x[1, [0, 7001, vocab - 1]] = real[1, :3]
    x[2, 3 * vocab // 4:] = real[2, 3 * vocab // 4:]
    x[3, ::2] = NEG
    few = torch.rand(vocab, generator=g, device="cuda") < 0.01
    x[4, few] = real[4, few]
    x[5, ::3] = float("nan")
    x[6] = real[6]
    x = x.to(dtype)
    ids = torch.tensor([11, 7001, vocab - 2, 1, 0, 4, 17], device="cuda")
    temps = {round(0.3 + 0.05 * i, 2) for i in range(55)} | {0.31, 0.575, 0.625, 0.635, 0.715, 0.745, 0.89, 1.075, 1.135,
                                                             1.27, 1.515, 1.585, 1.78, 2.31, 2.455, 1e-4, 0.01, 1e4}
    for temp in sorted(temps):
        check_logprobs(vb, x, ids, 4, temp, 3)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_logprobs_of_large_values_at_low_temperatures(vb, dtype):
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    rows, vocab = 400, 3001
    size = (1.5e5 + 4.5e5 * torch.rand(rows, 1, generator=g, device="cuda")).to(dtype).float()
    size[::2] *= -1
    x = size.expand(rows, vocab).clone()
    x[:, 1::2] -= 4 * torch.rand(rows, vocab // 2, generator=g, device="cuda")
    x = x.to(dtype)
    for temp in (1e-4, 2.5e-4, 1e-3):
        check_logprobs(vb, x, torch.arange(rows, device="cuda") * 7, 5, temp, 3)


# ==================================================================== q4 ==
def make_q4(g, outs, ins, group, zeros):
    """(q, s, zeros, the matrix in 64 bits)."""
    q = g.integers(0, 256, (outs, ins // 2), dtype=np.uint8)
    cells = (outs, -(-ins // group))
    s = (np.abs(g.standard_normal(cells)) * 0.01 + 1e-4).astype(np.float16)
    z = g.integers(0, 16, cells, dtype=np.uint8) if zeros else None
    b = q.reshape(outs, ins // 32, 16)
    w = np.concatenate([b & 15, b >> 4], axis=2).reshape(outs, ins).astype(np.float64)
    at = np.arange(ins) // group
    return q, s, z, (w - (8 if z is None else z[:, at])) * s.astype(np.float64)[:, at]


@pytest.mark.parametrize("group", [64, 96, 4096, 2**31 - 32, 2**31 - 64, 2**31 - 128])
def test_q4_groups_longer_than_a_row(vb, group):
    """One scale per row, whatever the group's length.  One-hot rows read the matrix
    back, exactly."""
    g = np.random.default_rng(5)
    for ins in (64, 32):
        q, s, z, w = make_q4(g, 50, ins, group, True)
        assert s.shape == (50, 1)
        layer = vb.Q4Linear(q, s, zeros=z, group=group)
        y = layer.matvec(torch.eye(ins, device="cuda"))
        np.testing.assert_array_equal(y.double().cpu().numpy().T, w)

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

from tests.test_gpu_ops import check_q4  # noqa: E402

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


def in_order(x, ids, top):
    """(rank, first columns) of rows without NaN: by one whole number per column,
    value first, then the lower column."""
    vocab = x.shape[1]
    bits = (x.float() + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * 2**23 + (2**23 - 1 - torch.arange(vocab, device="cuda"))
    rank = (key > key.gather(1, ids[:, None])).sum(1)
    return rank, torch.topk(key, top, 1).indices if top else ids[:, None][:, :0]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,tops", [(160, 151936, (0, 1, 20, 32)), (37, 4194304, (32,)), (149, 4194303, (5,))])
def test_logprobs_of_many_batches(vb, rows, vocab, tops, dtype):
    """Rows that a CTA passes in more batches than it keeps maxima of (8), 512 at the
    most, with the largest columns anywhere."""
    g = torch.Generator(device="cuda")
    g.manual_seed(vocab)
    x = torch.randn(rows, vocab, generator=g, device="cuda")
    x[1, -70:] += 9  # the last batch holds the first columns
    x[2, ::vocab // 40] += 9  # all of them do
    x[3] = x[3].sort().values
    x[4] = x[4].sort(descending=True).values
    x[5] = 0  # ties alone: the lists overflow
    x[6] = torch.randint(-2, 3, (vocab,), generator=g, device="cuda").float()
    x[7, :-3], x[7, -3:] = NEG, torch.tensor([1.0, 3.0, 2.0], device="cuda")
    x[8] = -1e9
    x[9, vocab // 2:] = x[9, vocab // 2:].sort().values + 5
    x = x.to(dtype)
    ids = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    ids[:10] = torch.tensor([0, vocab - 1, vocab // 40, vocab - 5, 3, vocab - 1, vocab // 2, vocab - 2, vocab - 1, vocab - 9],
                            device="cuda")
    v = x.double()
    m = v.max(1, keepdim=True).values
    logs = (v - m).exp().sum(1, keepdim=True).log()
    for top in tops:
        lp, rank, tid, tlp = vb.token_logprobs(x, ids.int(), top=top)
        wrank, order = in_order(x, ids, top)
        assert torch.equal(rank.long(), wrank)
        best = v.gather(1, order)
        assert torch.equal(tid.long(), torch.where(best > NEG, order, -1))
        batches = -(-vocab * x.element_size() // (16 * 4 * 512))
        rel = 2.0 ** -21 + 22 * 2 * U + (16 + batches + 12) * U
        for got, want in ((lp, v.gather(1, ids[:, None])[:, 0]), (tlp, best)):
            # (a column at -inf, in a row of -inf alone too: -inf)
            want = torch.where(want > NEG, want - (m + logs if want.dim() == 2 else (m + logs)[:, 0]), NEG)
            fin = torch.isfinite(want)
            assert torch.equal(got.double()[~fin], want[~fin])
            tol = 3 * U * (1 + 2.0 ** -20) * (want[fin].abs() + 16) + 2 * U * 16 + rel
            assert bool(((got.double()[fin] - want[fin]).abs() <= tol).all())


# =============================================================== process ==
def listed(g, rows, most, vocab):
    """CSR lists of up to `most` ids: frequent ones, ids at the same place of one slice
    of 4096 columns after the other, and ids outside the row."""
    lens = g.integers(0, most + 1, rows)
    lens[0], lens[-1] = 0, most
    off = np.zeros(rows + 1, np.int64)
    off[1:] = np.cumsum(lens)
    ids = (vocab ** g.random(off[-1])).astype(np.int64) - 1
    some = g.random(off[-1])
    ids = np.where(some < 0.4, (4096 * g.integers(0, 1 + vocab // 4096, off[-1]) + g.integers(0, 6, off[-1])) % vocab, ids)
    ids = np.where(some > 0.97, g.choice(np.array([-1, vocab, vocab + 7, 2**31 - 1, -2**31]), off[-1]), ids)
    return torch.from_numpy(ids).cuda(), torch.from_numpy(off).cuda()


def process_64(x, rates, hist, off, last, bias_ids, bias, bias_off, allowed):
    """(values, error bound): five roundings of at most u times the value rounded."""
    rows, vocab = x.shape

    def place(ids, off):
        row = torch.repeat_interleave(torch.arange(rows, device="cuda"), off[1:] - off[:-1])
        good = (ids >= 0) & (ids < vocab)
        return row, good, torch.where(good, row * vocab + ids, 0)

    v = x.double()
    mag = torch.zeros_like(v)
    row, good, at = place(hist, off)
    if last > 0:
        good &= torch.arange(len(hist), device="cuda") >= (off[1:] - last)[row]
    c = torch.zeros(rows * vocab, dtype=torch.float64, device="cuda").scatter_add_(0, at, good.double()).view(rows, vocab)
    seen = c > 0
    rep, freq, pres = (rates[:, i:i + 1].double() for i in range(3))
    p = torch.where(v > 0, v / rep, v * rep)
    s = p - freq * c - pres
    mag = torch.where(seen, p.abs() + (freq * c).abs() + (p - freq * c).abs() + s.abs(), mag)
    v = torch.where(seen, s, v)
    row, good, at = place(bias_ids, bias_off)
    i = torch.where(good, torch.arange(len(bias), device="cuda"), -1)
    last_at = torch.full((rows * vocab,), -1, device="cuda").scatter_reduce_(0, at, i, "amax").view(rows, vocab)
    v = torch.where(last_at >= 0, v + bias.double()[last_at], v)
    mag = torch.where(last_at >= 0, mag + v.abs(), mag)
    return torch.where(allowed, v, NEG), torch.where(allowed, U * (1 + 2.0 ** -20) * mag, 0.0)


@pytest.mark.parametrize("rows,vocab,ld,dtype,in_place", [
    (300, 70001, 70001, F32, False), (700, 70001, 70004, F32, True), (256, 151936, 151936, BF16, False),
    (130, 151936, 151939, F16, False), (520, 151936, 151936, F32, True), (520, 151935, 151937, F32, False)])
def test_process_of_many_slices(vb, rows, vocab, ld, dtype, in_place):
    """Rows that a CTA walks in several slices (2 to 8): each slice's counters start
    at 0, whatever the one before counted."""
    assert rows * -(-vocab // 4096) >= 2 * 148 * 16
    g = np.random.default_rng([rows, vocab])
    x = torch.from_numpy(g.standard_normal((rows, ld)).astype(np.float32) * 3).cuda().to(dtype)
    beside = x[:, vocab:].clone()
    x = x[:, :vocab]
    hist, off = listed(g, rows, 1500, vocab)
    bias_ids, bias_off = listed(g, rows, 400, vocab)
    bias = torch.from_numpy(g.standard_normal(len(bias_ids)).astype(np.float32)).cuda() * 4
    words = torch.from_numpy(g.integers(-2**31, 2**31, (rows, -(-vocab // 32)), dtype=np.int64).astype(np.int32)).cuda()
    words[0], words[-1] = -1, 0
    allowed = ((words[:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).view(rows, -1)[:, :vocab] != 0
    rates = torch.from_numpy(1 + 0.4 * g.random((rows, 3)).astype(np.float32)).cuda()
    for last in (0, 700):
        want, tol = process_64(x, rates, hist, off, last, bias_ids, bias, bias_off, allowed)
        given = x.clone() if not in_place else torch.cat([x, beside], 1)[:, :vocab]
        kw = dict(hist=hist.int(), hist_off=off, row_penalties=rates, bias_ids=bias_ids.int(), bias=bias, bias_off=bias_off,
                  mask=words)
        got = vb.process_logits(given if in_place else x, vb.Penalties(last=last), out=given if in_place else None, **kw)
        got = got.double()
        assert torch.equal(torch.isneginf(got), ~allowed)
        assert bool(((got - want).abs()[allowed] <= tol[allowed]).all())
        if in_place:
            assert torch.equal(given.as_strided((rows, ld - vocab), (ld, 1), vocab), beside)


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


@pytest.mark.parametrize("n", [129, 4097, 65535])
@pytest.mark.parametrize("outs,ins", [(33, 64), (200, 160)])
def test_q4_of_prompts(vb, n, outs, ins):
    """As many rows as a call takes."""
    g = np.random.default_rng([n, outs])
    q, s, z, w = make_q4(g, outs, ins, 64, True)
    layer = vb.Q4Linear(q, s, zeros=z, group=64)
    for dtype in (F32, BF16):
        x = torch.from_numpy(g.standard_normal((n, ins)).astype(np.float32)).cuda().to(dtype)
        check_q4(layer.matvec(x), x, w, None)


def test_the_sampler_right_behind_a_layer(vb):
    """A layer's grid lets the next one start early; each of the sampler's paths and
    the tail has to wait for the layer's rows, without a kernel between them."""
    g = np.random.default_rng(27)
    vocab = 40000
    q, s, z, w = make_q4(g, vocab, 256, 32, False)
    layer = vb.Q4Linear(q, s)
    rows = 6
    xs = [torch.randn(rows, 256, device="cuda") for _ in range(12)]
    lg = torch.empty(rows, vocab, device="cuda")
    hist = torch.randint(0, vocab, (rows * 32,), device="cuda", dtype=torch.int32)
    off = torch.arange(rows + 1, device="cuda") * 32
    for o in (vb.Sampling(temp=0.0), vb.Sampling(temp=0.0, repeat=1.3, repeat_last=32), vb.Sampling(temp=0.9, top_k=40),
              vb.Sampling(temp=0.9, top_k=40, repeat=1.3, repeat_last=32), vb.Sampling(temp=0.8, top_k=300),
              vb.Sampling(temp=1.0, top_k=0, top_p=0.9)):
        kw = dict(hist=hist, hist_off=off) if o.repeat != 1 else {}

        def step(x, rng):
            layer.matvec(x, out=lg)
            return vb.sample(lg, o, rng=rng, **kw).clone()

        first = torch.from_numpy(np.array(vb.seed_states(range(1, rows + 1)), np.uint64).view(np.int64)).cuda()
        rng = first.clone()
        want = []
        for x in xs:
            want.append(step(x, rng))
            torch.cuda.synchronize()
        for _ in range(5):
            rng = first.clone()
            got = [step(x, rng) for x in xs]
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), o
    vb.check()

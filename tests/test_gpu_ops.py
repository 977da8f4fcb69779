"""GPU tests of the operators around the sampler (include/verbo_ops.h), each
against a plain computation in 64 bits, and a run of them together against the
sampler's oracle.

Tolerances.  u = 2^-24 is half a step of fp32 (a rounding to nearest), h(t) =
eps(t) / 2 that of an output type t.
  * process: five roundings (the penalty, f * c, two subtractions, the bias),
    each of at most u times the value it rounds: u times the sum of the five
    magnitudes.
  * q4: x is met to within 2u of each value, the products are exact; K additions
    and one multiplication by a scale,
    in fp32 in the tensor core's order, whose additions may truncate: at most
    2u each, of partial sums no larger than A = sum |w x| (+ |b|); then the
    output's rounding.  Norm-wise, K/16 + K/32 + 16 roundings (an instruction
    sums 16 products) of partial sums no larger in the mean than the result.
  * logprobs: (v - m)/T has two roundings, 2u of itself; log s one of its own
    size (CUDA's logf: 1 step) plus the relative error of s: ex2 2^-22, the
    argument's rounding weighted by the terms, at most log2(vocab) <= 22 bits
    times 2u, and fewer than 64 additions on any term's way: 2^-22 + 22 * 2u +
    64 u < 2^-17.
"""
from __future__ import annotations

import numpy as np
import pytest

from oracle import pyoracle as po
from tests.gpu_util import compare, to_dev_rng

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


def dev(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda().to(dtype) if dtype else torch.from_numpy(
        np.ascontiguousarray(a)).cuda()


def csr(rng, rows, lens, vocab, wild=False):
    off = np.zeros(rows + 1, np.int64)
    off[1:] = np.cumsum(lens)
    ids = rng.integers(0, max(1, min(vocab, 1 + vocab // 3)), off[-1]).astype(np.int32)  # ids repeat
    if wild and len(ids) > 8:
        ids[::7] = np.resize(np.array([-1, vocab, 2**31 - 1, -2**31, vocab + 5], np.int32), len(ids[::7]))
    return ids, off


# =============================================================== process ==
def plain_process(x, pen=None, hist=None, off=None, rows_pen=None, bias_ids=None, bias=None, bias_off=None, allowed=None):
    """(values, error bound) in 64 bits."""
    v = x.astype(np.float64)
    mag = np.zeros_like(v)
    rows, vocab = v.shape
    for r in range(rows):
        if pen is not None and hist is not None:
            w = hist[off[r]:off[r + 1]]
            w = w[-pen.last:] if pen.last > 0 else w
            w = w[(w >= 0) & (w < vocab)]
            ids, c = np.unique(w, return_counts=True)
            rep, freq, pres = np.float64(np.float32([pen.repeat, pen.frequency, pen.presence])) if rows_pen is None \
                else rows_pen[r].astype(np.float64)
            a = v[r, ids]
            p = np.where(a > 0, a / rep, a * rep)
            q = p - freq * c
            s = q - pres
            v[r, ids] = s
            for t in (p, freq * c, q, s):
                mag[r, ids] += np.abs(t)
        if bias is not None:
            last = dict(zip(bias_ids[bias_off[r]:bias_off[r + 1]].tolist(), bias[bias_off[r]:bias_off[r + 1]].tolist()))
            for i, b in last.items():
                if 0 <= i < vocab:
                    v[r, i] += b
                    mag[r, i] += abs(v[r, i])
        if allowed is not None:
            v[r, ~allowed[r]] = NEG
            mag[r, ~allowed[r]] = 0
    return v, U * (1 + 2.0 ** -20) * mag


def words(allowed):
    rows, vocab = allowed.shape
    bits = np.zeros((rows, -(-vocab // 32) * 32), np.uint8)
    bits[:, :vocab] = allowed
    return np.packbits(bits, axis=1, bitorder="little").view(np.int32).copy()


def check_process(got, want, tol):
    got = got.astype(np.float64)
    fin = np.isfinite(want)
    np.testing.assert_array_equal(got[~fin], want[~fin])
    assert np.all(np.abs(got[fin] - want[fin]) <= tol[fin]), np.max(np.abs(got[fin] - want[fin]) - tol[fin])


SHAPES = [(1, 1), (1, 31), (2, 33), (3, 2047), (2, 8193), (1, 49152), (2, 151936), (301, 4099), (20, 70001)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_process_everything(vb, rows, vocab, dtype):
    g = np.random.default_rng([rows, vocab])
    x = dev(g.standard_normal((rows, vocab)).astype(np.float32) * 3, dtype)
    lens = g.integers(0, 200, rows)
    lens[0] = 0 if rows > 1 else 150
    hist, off = csr(g, rows, lens, vocab, wild=True)
    bias_ids, boff = csr(g, rows, lens[::-1] // 4, vocab, wild=True)
    bias = g.standard_normal(len(bias_ids)).astype(np.float32) * 4
    allowed = g.random((rows, vocab)) < 0.7
    if rows > 1:
        allowed[-1] = False
        allowed[0] = True
    pen = vb.Penalties(1.3, 0.37, 0.21, last=100)
    out = vb.process_logits(x, pen, hist=dev(hist), hist_off=dev(off), bias_ids=dev(bias_ids), bias=dev(bias),
                            bias_off=dev(boff), mask=dev(words(allowed)))
    assert out.dtype == F32 and out.shape == (rows, vocab)
    want, tol = plain_process(x.float().cpu().numpy(), pen, hist, off, None, bias_ids, bias, boff, allowed)
    check_process(out.cpu().numpy(), want, tol)


@pytest.mark.parametrize("rows,vocab,last", [(1, 700, 0), (4, 9000, 0), (4, 9000, 1), (3, 20000, 64), (200, 8200, 33)])
def test_process_history_alone(vb, rows, vocab, last):
    g = np.random.default_rng([rows, vocab, last])
    x = g.standard_normal((rows, vocab)).astype(np.float32)
    x[0, :5] = [0.0, -0.0, np.inf, -np.inf, 3.4e38]
    hist, off = csr(g, rows, g.integers(0, 400, rows), vocab)
    hist[:5] = [0, 1, 2, 3, 4][:len(hist[:5])]
    pen = vb.Penalties(1.1, -0.5, 0.25, last=last)
    per = (1.0 + g.random((rows, 3))).astype(np.float32)
    for rp in (None, per):
        out = vb.process_logits(dev(x), pen, hist=dev(hist), hist_off=dev(off),
                                row_penalties=None if rp is None else dev(rp)).cpu().numpy()
        want, tol = plain_process(x, pen, hist, off, rp)
        check_process(out, want, tol)
    # without penalties the history is not looked at, and row_penalties alone take all of it
    assert np.array_equal(vb.process_logits(dev(x), None, hist=dev(hist), hist_off=dev(off)).cpu().numpy(), x)
    out = vb.process_logits(dev(x), hist=dev(hist), hist_off=dev(off), row_penalties=dev(per)).cpu().numpy()
    want, tol = plain_process(x, vb.Penalties(), hist, off, per)
    check_process(out, want, tol)


def test_process_long_history(vb):
    """One id 70000 times, and a window of it: counts above 16 bits."""
    vocab = 5000
    x = np.linspace(-3, 3, 2 * vocab, dtype=np.float32).reshape(2, vocab)
    hist = np.concatenate([np.full(70000, 4321), np.arange(3000), np.full(10, 7)]).astype(np.int32)
    off = np.array([0, 73000, 73010], np.int64)
    for last in (0, 72000, 5):
        pen = vb.Penalties(1.0, 0.001, 0.0, last=last)
        out = vb.process_logits(dev(x), pen, hist=dev(hist), hist_off=dev(off)).cpu().numpy()
        want, tol = plain_process(x, pen, hist, off)
        check_process(out, want, tol)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,first,ld,ld_out", [(3, 1000, 1, 1003, 1001), (5, 8191, 3, 8200, 8193),
                                                        (180, 9001, 5, 9010, 9004), (2, 30, 7, 41, 33)])
def test_process_strides(vb, rows, vocab, first, ld, ld_out, dtype):
    """Rows that start anywhere; what lies beside them stays."""
    g = np.random.default_rng([rows, vocab, first])
    buf = dev(g.standard_normal((rows, ld)).astype(np.float32), dtype)
    x = buf[:, first:first + vocab] if first + vocab <= ld else buf[:, :vocab]
    obuf = torch.full((rows, ld_out + 6), 77.0, device="cuda")
    out = obuf[:, 2:2 + vocab]
    allowed = g.random((1, vocab)) < 0.5
    mask = torch.zeros(1, -(-vocab // 32) + 3, dtype=torch.int32, device="cuda")
    mask[:, :-3] = dev(words(allowed))
    hist, off = csr(g, rows, np.full(rows, 40), vocab)
    pen = vb.Penalties(1.5, 0.1, 0.1)
    assert vb.process_logits(x, pen, hist=dev(hist), hist_off=dev(off), mask=mask, out=out) is out
    want, tol = plain_process(x.float().cpu().numpy(), pen, hist, off, allowed=np.repeat(allowed, rows, 0))
    got = obuf.cpu().numpy()
    check_process(got[:, 2:2 + vocab], want, tol)
    assert np.all(got[:, :2] == 77.0) and np.all(got[:, 2 + vocab:] == 77.0)


@pytest.mark.parametrize("rows,vocab,ld", [(1, 40, 40), (3, 8193, 8193), (2, 49152, 49156), (200, 8211, 8213)])
def test_process_in_place(vb, rows, vocab, ld):
    g = np.random.default_rng([rows, vocab, 1])
    buf = g.standard_normal((rows, ld)).astype(np.float32)
    buf[0, 3] = np.nan  # untouched columns keep their bits, a masked NaN does not
    allowed = g.random((rows, vocab)) < np.resize([0.001, 0.5, 0.999], (rows, 1))
    allowed[0, 3] = True
    if rows > 2:
        allowed[2] = False
        buf[2, :9] = [np.nan, np.inf, -np.inf, np.finfo(np.float32).min, 0, -0.0, 1, 2, 3]
    hist, off = csr(g, rows, np.full(rows, 30), vocab)
    hist = hist[hist != 3] if rows == 1 else np.where(hist == 3, 4, hist).astype(np.int32)
    off = np.minimum(off, len(hist))
    bias_ids, boff = csr(g, rows, np.full(rows, 9), vocab)
    bias_ids[bias_ids == 3] = 4
    bias = g.standard_normal(len(bias_ids)).astype(np.float32)
    pen = vb.Penalties(1.2, 0.3, 0.1)
    d = dev(buf)
    x = d[:, :vocab]
    assert vb.process_logits(x, pen, hist=dev(hist), hist_off=dev(off), bias_ids=dev(bias_ids), bias=dev(bias),
                             bias_off=dev(boff), mask=dev(words(allowed)), out=x) is x
    want, tol = plain_process(buf[:, :vocab], pen, hist, off, None, bias_ids, bias, boff, allowed)
    got = d.cpu().numpy()
    nan = np.isnan(want)
    assert nan.sum() == 1 and np.isnan(got[:, :vocab][nan]).all()
    check_process(np.where(nan, 0, got[:, :vocab]), np.where(nan, 0, want), tol)
    np.testing.assert_array_equal(got[:, vocab:], buf[:, vocab:])
    # in place equals out of place, bit for bit
    other = vb.process_logits(dev(buf)[:, :vocab], pen, hist=dev(hist), hist_off=dev(off), bias_ids=dev(bias_ids),
                              bias=dev(bias), bias_off=dev(boff), mask=dev(words(allowed))).cpu().numpy()
    np.testing.assert_array_equal(other, got[:, :vocab])


def test_process_bias_listed_twice(vb):
    x = torch.zeros(1, 50, device="cuda")
    ids = np.array([7, 9, 7, 7, 9], np.int32)
    b = np.array([1, 2, 3, 4, 5], np.float32)
    out = vb.process_logits(x, bias_ids=dev(ids), bias=dev(b), bias_off=dev(np.array([0, 5]))).cpu().numpy()[0]
    assert out[7] == 4 and out[9] == 5 and np.count_nonzero(out) == 2


def test_process_refusals_on_device(vb):
    x = torch.zeros(2, 64, device="cuda")
    h, o = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    bad = [dict(hist=h), dict(hist=h.long(), hist_off=o, penalties=vb.Penalties()), dict(hist=h, hist_off=o[:2], penalties=vb.Penalties()),
           dict(hist=h.cpu(), hist_off=o), dict(mask=torch.zeros(2, 1, dtype=torch.int32, device="cuda")),
           dict(mask=torch.zeros(3, 2, dtype=torch.int32, device="cuda")), dict(mask=torch.zeros(2, 2, device="cuda")),
           dict(out=torch.zeros(1, 64, device="cuda")), dict(out=x.half()), dict(out=x[:, 1:], vocab=63), dict(vocab=65),
           dict(row_penalties=torch.ones(2, 2, device="cuda")), dict(row_penalties=torch.ones(3, 2, device="cuda")),
           dict(bias=torch.zeros(1, device="cuda"))]
    for kw in bad:
        with pytest.raises(vb.VerboCudaError):
            vb.process_logits(x, **kw)
    with pytest.raises(vb.VerboCudaError):
        vb.process_logits(x.t())
    with pytest.raises(vb.VerboCudaError):
        vb.process_logits(x.double())
    assert vb.process_logits(x[:0]).shape == (0, 64)
    # two halves of one buffer lie beside each other
    both = torch.randn(3, 128, device="cuda")
    vb.process_logits(both[:, :64], out=both[:, 64:])
    assert torch.equal(both[:, :64], both[:, 64:])


# ============================================================== logprobs ==
def plain_logprobs(x, ids, top, temp):
    """In 64 bits: (logprob, rank, top_ids, top_logprobs, tolerance of a log-probability)."""
    t = float(np.float32(temp))
    v = x.astype(np.float64) + 0.0
    v[np.isnan(v)] = NEG
    rows, vocab = v.shape
    lp = np.full(rows, NEG)
    rank = np.full(rows, -1)
    tid = np.full((rows, top), -1)
    tlp = np.full((rows, top), NEG)
    for r in range(rows):
        m = v[r].max()
        with np.errstate(invalid="ignore"):
            d = np.where(v[r] == m, 0.0, (v[r] - m) / t)
        logs = np.log(np.exp(d).sum())
        l = np.where(v[r] == NEG, NEG, d - logs)
        order = np.lexsort((np.arange(vocab), -v[r]))
        good = order[v[r][order] > NEG][:top]
        tid[r, :len(good)] = good
        tlp[r, :len(good)] = l[good]
        if ids is not None and 0 <= ids[r] < vocab:
            lp[r] = l[ids[r]]
            rank[r] = np.flatnonzero(order == ids[r])[0]
    return lp, rank, tid, tlp


def check_lp(got, want):
    got = got.astype(np.float64)
    fin = np.isfinite(want)
    np.testing.assert_array_equal(got[~fin], want[~fin])
    # |d| + |log s| <= |lp| + 2 |log s|, and log s <= log(vocab) < 16
    tol = 2 * U * (np.abs(want[fin]) + 2 * 16) + 2.0 ** -17
    assert np.all(np.abs(got[fin] - want[fin]) <= tol), np.max(np.abs(got[fin] - want[fin]))


def check_logprobs(vb, x, ids, top, temp, **kw):
    lp, rank, tid, tlp = vb.token_logprobs(x, None if ids is None else dev(ids.astype(np.int32)), top=top, temp=temp, **kw)
    vocab = kw.get("vocab", x.shape[1])
    wlp, wrank, wtid, wtlp = plain_logprobs(x[:, :vocab].float().cpu().numpy(), ids, top, temp)
    if ids is None:
        assert lp is None and rank is None
    else:
        np.testing.assert_array_equal(rank.cpu().numpy(), wrank)
        check_lp(lp.cpu().numpy(), wlp)
    np.testing.assert_array_equal(tid.cpu().numpy(), wtid)
    check_lp(tlp.cpu().numpy(), wtlp)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,top,temp", [(1, 1, 1, 1.0), (1, 7, 32, 0.5), (3, 31, 5, 1.7), (2, 2049, 32, 1.0),
                                                 (5, 8193, 17, 0.8), (1, 49152, 5, 0.7), (2, 151936, 16, 1.0),
                                                 (150, 9001, 3, 1.3), (600, 5003, 20, 1.0), (3, 327681, 32, 1.0),
                                                 (4, 151936, 0, 1.0)])
def test_logprobs(vb, rows, vocab, top, temp, dtype):
    g = np.random.default_rng([rows, vocab, top])
    x = dev((g.standard_normal((rows, vocab)) * 3).astype(np.float32), dtype)
    ids = g.integers(0, vocab, rows)
    ids[0] = int(x[0].float().argmax())
    check_logprobs(vb, x, ids, top, temp)


@pytest.mark.parametrize("vocab", [100, 5000, 60001])
def test_logprobs_hard_rows(vb, vocab):
    """Ties, masks, infinities, NaN, sorted rows: what makes a bound useless."""
    g = np.random.default_rng(vocab)
    low = np.finfo(np.float32).min
    x = np.zeros((16, vocab), np.float32)
    x[1] = np.arange(vocab)
    x[2] = -np.arange(vocab)
    x[3] = NEG
    x[4] = low
    x[5], x[5, vocab // 2:vocab // 2 + 3] = NEG, [1, 3, 2]
    x[6], x[6, -1] = low, 5.0
    x[7] = g.standard_normal(vocab)
    x[7, ::3], x[7, 1::3] = np.nan, NEG
    x[8] = g.integers(-2, 3, vocab)
    x[9] = g.standard_normal(vocab)
    x[9, [3, vocab - 2]] = np.inf
    x[10] = np.inf
    x[11] = np.nan
    x[12, ::2] = -0.0
    x[13] = 3e38 * (g.random(vocab) - 0.5)
    x[14], x[14, vocab // 3:] = NEG, g.standard_normal(vocab - vocab // 3)
    x[15] = np.where(g.random(vocab) < 0.01, g.standard_normal(vocab) * 5, NEG)
    for dtype in (F32, BF16):
        t = dev(x, dtype)
        for ids in (np.full(16, vocab // 2), np.zeros(16, int), np.full(16, vocab - 1)):
            for top in (0, 1, 20, 32):
                check_logprobs(vb, t, ids, top, 1.0)


def test_logprobs_differences_beyond_fp32(vb):
    """Values whose difference fp32 does not hold, and a temperature that makes a
    number of it again.  Three roundings of the result's own size: 3u."""
    x = np.array([[3e38, -3e38, 1.0, -1e38], [-3.4e38, 3.4e38, NEG, 1e30]], np.float32)
    for temp in (2.0, 10.0, 1e4):
        _, _, tid, tlp = vb.token_logprobs(dev(x), top=4, temp=temp)
        _, _, wtid, wtlp = plain_logprobs(x, None, 4, temp)
        np.testing.assert_array_equal(tid.cpu().numpy(), wtid)
        np.testing.assert_allclose(tlp.double().cpu().numpy(), wtlp, rtol=3 * U * (1 + 2.0 ** -20), atol=0)


def test_logprobs_ids_outside_and_none(vb):
    x = torch.randn(4, 300, device="cuda")
    check_logprobs(vb, x, np.array([-1, 300, 2**31 - 1, 299]), 4, 1.0)
    check_logprobs(vb, x, None, 4, 1.0)


@pytest.mark.parametrize("temp", [1e-4, 0.05, 30.0, 1e4])
def test_logprobs_temperatures(vb, temp):
    x = torch.randn(3, 20000, device="cuda") * 4
    v = x.cpu().numpy()
    check_logprobs(vb, x, v.argmax(1), 8, temp)


@pytest.mark.parametrize("dtype", [F32, F16], ids=["f32", "f16"])
def test_logprobs_strides(vb, dtype):
    buf = torch.randn(7, 10007, device="cuda").to(dtype)
    for first, n in ((0, 10000), (1, 9999), (3, 8193), (5, 17)):
        check_logprobs(vb, buf[:, first:first + n], np.arange(7) % n, 9, 1.0)
    check_logprobs(vb, buf, np.arange(7), 9, 1.0, vocab=5001)


# ==================================================================== q4 ==
def unpack(q):
    outs, half = q.shape
    b = q.reshape(outs, half // 16, 16)
    return np.concatenate([b & 15, b >> 4], axis=2).reshape(outs, 2 * half)


def make_q4(g, outs, ins, group, zeros, bias):
    q = g.integers(0, 256, (outs, ins // 2), dtype=np.uint8)
    groups = -(-ins // group)
    s = (np.abs(g.standard_normal((outs, groups))) * 0.01 + 1e-4).astype(np.float16)
    z = g.integers(0, 16, (outs, groups), dtype=np.uint8) if zeros else None
    b = g.standard_normal(outs).astype(np.float32) if bias else None
    at = np.arange(ins) // group
    w = (unpack(q).astype(np.float64) - (8.0 if z is None else z.astype(np.float64)[:, at])) * s.astype(np.float64)[:, at]
    return q, s, z, b, w


def check_q4(y, x, w, b):
    got = y.double().cpu()
    xd, wd = x.double().cpu(), torch.from_numpy(w)
    want = xd @ wd.t()
    size = xd.abs() @ wd.abs().t()
    ins = w.shape[1]
    if b is not None:
        want += torch.from_numpy(b).double()
        size += torch.from_numpy(b).double().abs()
    h = torch.finfo(y.dtype).eps / 2
    tol = (ins + 2) * 2 * U * size + h * want.abs() * (1 + 2.0 ** -8) + (2.0 ** -25 if y.dtype == F16 else 0)
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() - tol).max())
    norm = float(want.norm())
    if norm and want.numel() >= 64:
        rel = float((got - want).norm()) / norm
        assert rel <= (ins / 16 + ins / 32 + 16) * 2 * U + h, rel


Q4_SHAPES = [(1, 32, 32), (7, 64, 32), (16, 128, 64), (17, 96, 64), (33, 160, 128), (100, 896, 32), (896, 4832, 128),
             (300, 1024, 96), (2500, 256, 256), (5000, 128, 128), (64, 8192, 128), (48, 16384, 64), (16, 32768, 32)]


@pytest.mark.parametrize("zeros,bias", [(False, False), (True, True)], ids=["plain", "zeros-bias"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("outs,ins,group", Q4_SHAPES)
def test_q4(vb, outs, ins, group, dtype, zeros, bias):
    g = np.random.default_rng([outs, ins, group, zeros])
    q, s, z, b, w = make_q4(g, outs, ins, group, zeros, bias)
    layer = vb.Q4Linear(q, s, zeros=z, bias=b, group=group)
    for n in (1, 2, 3, 8, 9, 17, 40):
        x = dev(g.standard_normal((n, ins)).astype(np.float32), dtype)
        y = layer.matvec(x)
        assert y.dtype == dtype and y.shape == (n, outs)
        check_q4(y, x, w, b)
        if n == 3 and dtype != F32:
            check_q4(layer.matvec(x, dtype=F32), x, w, b)
    layer.close()


@pytest.mark.parametrize("n", [1, 2, 5, 13, 33, 64, 65, 130])
def test_q4_many_rows(vb, n):
    g = np.random.default_rng(n)
    q, s, z, b, w = make_q4(g, 1111, 1184, 32, True, True)
    layer = vb.Q4Linear(q, s, zeros=z, bias=b, group=32)
    for dtype in (F32, F16, BF16):
        x = dev(g.standard_normal((n, 1184)).astype(np.float32), dtype)
        for out in (F32, F16, BF16):
            check_q4(layer.matvec(x, dtype=out), x, w, b)


def test_q4_each_weight_lands_in_its_place(vb):
    """One-hot x reads the matrix back, exactly."""
    g = np.random.default_rng(3)
    for outs, ins, group, zeros in ((50, 416, 32, True), (37, 256, 128, False), (18, 320, 64, True)):
        q, s, z, b, w = make_q4(g, outs, ins, group, zeros, False)
        layer = vb.Q4Linear(q, s, zeros=z, group=group)
        for dtype in (F32, F16, BF16):
            y = layer.matvec(torch.eye(ins, device="cuda").to(dtype), dtype=F32)
            np.testing.assert_array_equal(y.double().cpu().numpy().T, w)


def test_q4_inputs_of_all_sizes(vb):
    """x of widely spread sizes, last places of fp32, and what is not a number."""
    g = np.random.default_rng(4)
    q, s, _, _, w = make_q4(g, 40, 64, 32, False, False)
    layer = vb.Q4Linear(q, s)
    x = (g.standard_normal((4, 64)) * 10.0 ** g.integers(-12, 12, (4, 64))).astype(np.float32)
    one = np.zeros((2, 64), np.float32)
    one[0, 5], one[1, 9] = 1 + 2.0 ** -23, -(2.0 - 2.0 ** -23) * 2.0 ** 20
    check_q4(layer.matvec(dev(x)), dev(x), w, None)
    np.testing.assert_array_equal(layer.matvec(dev(one)).double().cpu().numpy(), (one.astype(np.float64) @ w.T).astype(np.float32))
    bad = np.ones((3, 64), np.float32)
    bad[0, 7], bad[1, 7], bad[2, 7] = np.inf, np.nan, -np.inf
    for dtype in (F32, F16, BF16):
        y = layer.matvec(dev(bad, dtype), dtype=F32).cpu().numpy()
        np.testing.assert_array_equal(np.isnan(y[1]), True)
        with np.errstate(invalid="ignore"):
            hit = w[:, 7] != 0
        np.testing.assert_array_equal(y[0][hit], np.where(w[hit, 7] > 0, np.inf, -np.inf))
        np.testing.assert_array_equal(y[2], -y[0])


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_q4_strides(vb, dtype):
    g = np.random.default_rng(8)
    q, s, z, b, w = make_q4(g, 77, 224, 32, False, True)
    layer = vb.Q4Linear(q, s, bias=b)
    buf = dev(g.standard_normal((11, 235)).astype(np.float32), dtype)
    for first in (0, 1, 8):
        x = buf[:, first:first + 224]
        obuf = torch.full((11, 90), 5.0, device="cuda", dtype=dtype)
        out = obuf[:, 3:80]
        assert layer.matvec(x, out=out) is out
        check_q4(out, x, w, b)
        assert bool((obuf[:, :3] == 5).all()) and bool((obuf[:, 80:] == 5).all())
    layer.matvec(buf[:0, :224])


def test_q4_device_arrays_and_determinism(vb):
    g = np.random.default_rng(9)
    q, s, z, b, w = make_q4(g, 3000, 896, 32, True, True)
    host = vb.Q4Linear(q, s, zeros=z, bias=b)
    onto = vb.Q4Linear(dev(q), dev(s), zeros=dev(z), bias=dev(b))
    x = torch.randn(5, 896, device="cuda")
    first = host.matvec(x)
    for _ in range(3):
        assert torch.equal(onto.matvec(x), first)
    # the order of the sums goes by n: another batch has the same row within its rounding
    check_q4(host.matvec(x[2:3]), x[2:3], w, b)
    check_q4(first, x, w, b)


def test_q4_refusals_on_device(vb):
    g = np.random.default_rng(1)
    q, s, *_ = make_q4(g, 8, 64, 32, False, False)
    layer = vb.Q4Linear(q, s)
    x = torch.zeros(2, 64, device="cuda")
    for bad in (x[:, :32], x.double(), x.cpu(), x[0], torch.zeros(64, 2, device="cuda").t(), x[:1].expand(2, 64)):
        with pytest.raises(vb.VerboCudaError):
            layer.matvec(bad)
    for kw in (dict(dtype=torch.int32), dict(out=torch.zeros(2, 9, device="cuda")), dict(out=torch.zeros(1, 8, device="cuda")),
               dict(out=x[:, :8]), dict(out=torch.zeros(2, 8, device="cuda"), dtype=F16)):
        with pytest.raises(vb.VerboCudaError):
            layer.matvec(x, **kw)
    # a workspace that is missing, too small or in the way
    lib, many = layer._lib, torch.zeros(40, 64, device="cuda")
    y = torch.zeros(40, 8, device="cuda")
    need = lib.verbo_ops_q4_workspace(layer._h, 0, 40)
    assert need > 0 and lib.verbo_ops_q4_workspace(layer._h, 0, 1) == 0
    assert lib.verbo_ops_q4_workspace(layer._h, 0, 65536) == -1 and lib.verbo_ops_q4_workspace(layer._h, 7, 1) == -1
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    for at, size in ((None, need), (ws.data_ptr(), need - 1), (ws.data_ptr() + 4, need), (y.data_ptr(), need)):
        assert lib.verbo_ops_q4_matvec(layer._h, many.data_ptr(), 0, 40, 64, y.data_ptr(), 0, 8, at, size, None) == -1
        assert "workspace" in lib.verbo_cuda_last_error().decode()
    layer.close()
    with pytest.raises(vb.VerboCudaError):
        layer.matvec(x)


# ============================================================== together ==
def decode_inputs(g, rows, vocab, ins):
    q, s, z, b, w = make_q4(g, vocab, ins, 32, False, False)
    hidden = g.standard_normal((rows, ins)).astype(np.float32)
    hist, off = csr(g, rows, g.integers(0, 100, rows), vocab)
    bias_ids, boff = csr(g, rows, g.integers(0, 20, rows), vocab)
    bias = g.standard_normal(len(bias_ids)).astype(np.float32)
    allowed = g.random((rows, vocab)) < 0.4
    allowed[:, 17] = True
    return q, s, hidden, hist, off, bias_ids, boff, bias, allowed


@pytest.mark.parametrize("opts", [dict(temp=0.0), dict(temp=0.8, top_k=40, top_p=0.9), dict(temp=1.0, top_k=0, top_p=0.95)],
                         ids=["greedy", "top-k", "nucleus"])
def test_decode_step_with_a_grammar(vb, opts):
    """Hidden rows -> 4-bit head -> penalties, biases, mask in place -> the sampler's
    pick -> its log-probability; the picks against the oracle's on the same rows."""
    rows, vocab, ins = 12, 49152, 256
    g = np.random.default_rng(21)
    q, s, hidden, hist, off, bias_ids, boff, bias, allowed = decode_inputs(g, rows, vocab, ins)
    head = vb.Q4Linear(q, s)
    lg = head.matvec(dev(hidden))
    before = lg.cpu().numpy()
    pen = vb.Penalties(1.2, 0.2, 0.1, last=64)
    vb.process_logits(lg, pen, hist=dev(hist), hist_off=dev(off), bias_ids=dev(bias_ids), bias=dev(bias),
                      bias_off=dev(boff), mask=dev(words(allowed)), out=lg)
    want, tol = plain_process(before, pen, hist, off, None, bias_ids, bias, boff, allowed)
    x = lg.cpu().numpy()
    check_process(x, want, tol)
    seeds = np.arange(1, rows + 1, dtype=np.uint64)
    ids = vb.sample(lg, vb.Sampling(repeat=1.0, **opts), rng=to_dev_rng(po.seed_states(seeds)))
    vb.check()
    got = ids.cpu().numpy()
    ref, st = po.sample_rows(x, po.sampling(repeat=1.0, **opts), po.seed_states(seeds), None, None)
    compare(got[:, None], ref[:, None], st[:, None])
    assert allowed[np.arange(rows), got].all()
    lp, rank, tid, tlp = vb.token_logprobs(lg, ids, top=10)
    wlp, wrank, wtid, wtlp = plain_logprobs(x, got, 10, 1.0)
    np.testing.assert_array_equal(rank.cpu().numpy(), wrank)
    np.testing.assert_array_equal(tid.cpu().numpy(), wtid)
    check_lp(lp.cpu().numpy(), wlp)
    check_lp(tlp.cpu().numpy(), wtlp)
    assert allowed[np.repeat(np.arange(rows), 10), tid.cpu().numpy().ravel()].all()


def test_captured_step_replays_on_new_inputs(vb):
    rows, vocab, ins = 6, 20011, 128
    g = np.random.default_rng(22)
    q, s, hidden, hist, off, bias_ids, boff, bias, allowed = decode_inputs(g, rows, vocab, ins)
    head = vb.Q4Linear(q, s)
    x, h, o = dev(hidden), dev(hist), dev(off)
    bi, bo, bv, mk = dev(bias_ids), dev(boff), dev(bias), dev(words(allowed))
    ids = torch.zeros(rows, dtype=torch.int32, device="cuda")
    pen = vb.Penalties(1.2, 0.2, 0.1)

    def step():
        lg = head.matvec(x)
        lg = vb.process_logits(lg, pen, hist=h, hist_off=o, bias_ids=bi, bias=bv, bias_off=bo, mask=mk, out=lg)
        return (lg, *vb.token_logprobs(lg, ids, top=7))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = step()
    with torch.cuda.graph(second):
        b = step()
    for seed in range(3):
        x.copy_(torch.randn(rows, ins, device="cuda"))
        ids.copy_(torch.randint(0, vocab, (rows,), device="cuda", dtype=torch.int32))
        mk.copy_(torch.randint(-2**31, 2**31 - 1, mk.shape, device="cuda").int())
        want = [t.clone() for t in step()]
        graph.replay()
        second.replay()
        for got in (a, b):
            for u, v in zip(got, want):
                assert torch.equal(u, v)


def test_calls_on_several_streams(vb):
    """Calls on streams of their own, at once, give what they give alone."""
    g = np.random.default_rng(23)
    q, s, _, _, w = make_q4(g, 9000, 512, 64, False, False)
    layer = vb.Q4Linear(q, s, group=64)
    x = [torch.randn(3, 512, device="cuda") for _ in range(4)]
    want = [(layer.matvec(t), *vb.token_logprobs(layer.matvec(t), top=5)[2:]) for t in x]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in x]
    got = []
    for _ in range(5):
        for t, st in zip(x, streams):
            y = layer.matvec(t, stream=st)
            got.append((y, *vb.token_logprobs(y, top=5, stream=st)[2:]))
    torch.cuda.synchronize()
    for i, t in enumerate(got):
        for u, v in zip(t, want[i % 4]):
            assert torch.equal(u, v)


def test_calls_from_several_threads(vb):
    """Threads of their own streams, calls of other sizes at once."""
    import threading

    g = np.random.default_rng(24)
    q, s, _, _, w = make_q4(g, 3000, 2048, 64, False, False)
    layer = vb.Q4Linear(q, s, group=64)
    sizes = (1, 3, 8, 12, 40)
    x = [torch.randn(n, 2048, device="cuda").half() for n in sizes]
    want = [(layer.matvec(t), *vb.token_logprobs(layer.matvec(t), top=3)[2:]) for t in x]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        st = torch.cuda.Stream()
        for _ in range(30):
            y = layer.matvec(x[i], stream=st)
            got = (y, *vb.token_logprobs(y, top=3, stream=st)[2:])
            st.synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sizes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_layer_freed_during_a_capture(vb):
    """Garbage collection frees a layer whenever it likes: not into a capture."""
    g = np.random.default_rng(25)
    q, s, _, _, w = make_q4(g, 64, 64, 32, False, False)
    layer, other = vb.Q4Linear(q, s), vb.Q4Linear(q, s)
    x = torch.randn(2, 64, device="cuda")
    want = layer.matvec(x).clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer.matvec(x)
        other.close()
    graph.replay()
    assert torch.equal(y, want)


def test_sampler_after_a_layer_on_one_stream(vb):
    """The layers and the sampler's kernels start early on one another's heels; each
    step has to see what the one before wrote."""
    g = np.random.default_rng(26)
    q, s, _, _, w = make_q4(g, 20000, 256, 32, False, False)
    layer = vb.Q4Linear(q, s)
    xs = [torch.randn(4, 256, device="cuda") for _ in range(20)]
    lg = torch.empty(4, 20000, device="cuda")
    hist = torch.randint(0, 20000, (4 * 32,), device="cuda", dtype=torch.int32)
    off = torch.arange(5, device="cuda") * 32
    o = vb.Sampling(temp=0.0, repeat=1.2, repeat_last=32)
    mask = torch.randint(-2**31, 2**31 - 1, (4, 625), device="cuda").int()

    def step(x):
        layer.matvec(x, out=lg)
        vb.process_logits(lg, mask=mask, out=lg)
        ids = vb.sample(lg, o, hist=hist, hist_off=off)
        return ids, *vb.token_logprobs(lg, ids, top=2)

    want = []
    for x in xs:
        want.append([t.clone() for t in step(x)])
        torch.cuda.synchronize()
    for _ in range(5):
        got = [step(x) for x in xs]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_rows_beyond_32_bits(vb):
    """Rows more than 2^31 elements apart."""
    ld, vocab = 2**31 + 9, 4000
    buf = torch.zeros(ld + vocab, dtype=BF16, device="cuda")
    x = buf.as_strided((2, vocab), (ld, 1))
    x.copy_(torch.randn(2, vocab, device="cuda"))
    near = x.contiguous()
    assert torch.equal(vb.process_logits(x), near.float())
    ids = np.array([17, 3999])
    check_logprobs(vb, x, ids, 5, 1.0)
    g = np.random.default_rng(30)
    q, s, _, _, w = make_q4(g, 48, 3200, 128, False, False)
    layer = vb.Q4Linear(q, s, group=128)
    assert torch.equal(layer.matvec(x[:, :3200]), layer.matvec(near[:, :3200].contiguous()))
    far = torch.zeros(2**31 // 2 + 9 + 64, device="cuda").as_strided((2, 48), (2**31 // 2 + 9, 1))
    layer.matvec(near[:, :3200].contiguous(), out=far, dtype=F32)
    check_q4(far.contiguous(), near[:, :3200], w, None)


def test_many_short_rows(vb):
    rows, vocab = 70001, 37
    g = np.random.default_rng(31)
    x = g.standard_normal((rows, vocab)).astype(np.float32)
    allowed = g.random((rows, vocab)) < 0.6
    out = vb.process_logits(dev(x), mask=dev(words(allowed))).cpu().numpy()
    np.testing.assert_array_equal(out, np.where(allowed, x, NEG))
    ids = g.integers(0, vocab, rows)
    lp, rank, tid, tlp = vb.token_logprobs(dev(out), dev(ids.astype(np.int32)), top=2)
    v = out.astype(np.float64)
    with np.errstate(divide="ignore"):
        want = v - np.log(np.exp(v).sum(1, keepdims=True))
    check_lp(lp.cpu().numpy()[allowed.any(1)], want[np.arange(rows), ids][allowed.any(1)])
    mine = v[np.arange(rows), ids][:, None]
    before = (v > mine) | ((v == mine) & (np.arange(vocab) < ids[:, None]))
    np.testing.assert_array_equal(rank.cpu().numpy(), before.sum(1))
    first = v.argmax(1)
    np.testing.assert_array_equal(tid.cpu().numpy()[:, 0], np.where(allowed.any(1), first, -1))


def test_the_rings_wait_gives_up(vb, tmp_path):
    """The wait of the 4-bit products' ring on a barrier that nothing arrives on ends
    after its limit, and the context goes on."""
    import ctypes
    import subprocess
    from pathlib import Path

    from verbo_b200 import build

    root = Path(__file__).resolve().parent.parent
    so = tmp_path / "libops_wait.so"
    subprocess.run([build.nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-O2", "-std=c++17", "-shared",
                    "-Xcompiler", "-fPIC", f"-I{root / 'verbo_b200' / 'csrc'}", "-o", str(so),
                    str(root / "tests" / "cpp" / "ops_wait_timeout.cu")], check=True, capture_output=True)
    lib = ctypes.CDLL(str(so))
    gave_up, waited, limit = ctypes.c_uint(7), ctypes.c_ulonglong(0), ctypes.c_ulonglong(0)
    assert lib.run_ops_wait_timeout(ctypes.byref(gave_up), ctypes.byref(waited), ctypes.byref(limit)) == 0
    assert gave_up.value == 1
    assert limit.value <= waited.value < 20 * limit.value
    x = torch.randn(2, 64, device="cuda")
    assert torch.equal(vb.process_logits(x), x)
    vb.check()

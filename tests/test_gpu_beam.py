"""GPU tests of beam search's operators (verbo_b200/beam.py) against the formula in
64 bits.

A score's tolerance: a term of a row's sum is off by the roundings of x - m and of
its product with log2(e), 2^-24 |t| each, by the exponential's 2^-22, and by up to
fifteen fp32 additions, 2^-24 each; the terms that make up a sum have |t| below 17 +
log2 of the columns, so the sum, and with it lse, is off by less than 2^-24 (2 * 40
+ 4 + 15) < 6e-6.  The score is rounded to fp32 once: 2^-24 of it."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import verbo_b200 as vb  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF = float("inf")


@pytest.fixture(autouse=True)
def _needs(cuda_lib):
    if not torch.cuda.is_available():
        pytest.fail("gpu tests need a CUDA device")


def oracle(x, scores, beams, take):
    """The definition, on the CPU, in 64 bits: (values, parents, tokens) as lists per request."""
    x = x.double().cpu().numpy()
    x = np.where(np.isnan(x), -INF, x)
    scores = scores.double().cpu().numpy().reshape(-1)
    out = []
    for r in range(x.shape[0] // beams):
        cand = []
        for b in range(beams):
            row, s = x[r * beams + b], scores[r * beams + b]
            if not s > -INF:
                continue
            m = row.max()
            if m == -INF:
                continue
            if m == INF:
                at = np.flatnonzero(row == INF)
                lp = np.full(at.size, -np.log(at.size))
            else:
                at = np.argsort(-row, kind="stable")[:take]
                at = at[row[at] > -INF]
                lp = row[at] - (m + np.log(np.exp(row - m).sum()))
            for i, l in list(zip(at, lp))[:take]:
                cand.append((s + l, b, int(i)))
        order = sorted(range(len(cand)), key=lambda i: -cand[i][0])[:take]  # stable: the beam, then the beam's own order
        got = [cand[i] for i in order]
        out.append(got + [(-INF, -1, -1)] * (take - len(got)))
    return out


def check(x, scores, beams, take, vocab=None):
    got = vb.beam_select(x, scores, beams, take, vocab=vocab)
    vb.check()
    want = oracle(x if vocab is None else x[:, :vocab], scores, beams, take)
    v, p, t = (g.cpu().numpy() for g in got)
    assert v.dtype == np.float32 and p.dtype == np.int32 and t.dtype == np.int32
    assert p.tolist() == [[c[1] for c in r] for r in want]
    assert t.tolist() == [[c[2] for c in r] for r in want]
    w = np.array([[c[0] for c in r] for r in want]).reshape(v.shape)
    live = np.isfinite(w)
    assert np.array_equal(v[~live], w[~live].astype(np.float32))
    assert (np.abs(v[live] - w[live]) <= 6e-6 + 2.0**-24 * np.abs(w[live])).all()
    return got


def make(rows, vocab, dtype, seed, ld=None, shift=0):
    """Rows of a row stride `ld`, the first `shift` elements off a 16-byte boundary."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    ld = ld or vocab
    flat = torch.full((rows * ld + shift,), 1e4, dtype=dtype, device="cuda")  # between the rows: what nobody may read
    x = flat[shift:].view(rows, ld)[:, :vocab]
    x.copy_(torch.randn(rows, vocab, generator=g, device="cuda") * 2)
    return x, -5 * torch.rand(rows, generator=g, device="cuda")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("requests,beams,vocab,take", [
    (1, 1, 1, 1), (1, 1, 1, 3), (3, 2, 2, 64), (2, 3, 7, 5), (2, 2, 8, 16), (1, 4, 9, 64), (5, 5, 17, 10),
    (4, 32, 1000, 64), (3, 7, 4097, 14), (1, 4, 49152, 8), (2, 5, 50257, 10), (1, 32, 16384, 32), (2, 8, 151936, 16),
    (40, 8, 2049, 9),
])
def test_sizes(dtype, requests, beams, vocab, take):
    check(*make(requests * beams, vocab, dtype, vocab + take), beams, take)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [5, 31, 1001, 20011])
@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (3, 2), (8, 3), (8, 7)])
def test_rows_anywhere(dtype, vocab, pad, shift):
    x, s = make(6, vocab, dtype, 5, vocab + pad, shift)
    check(x, s, 3, 7)
    check(x, s, 3, 7, vocab=vocab - 2)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab,ld", [(1003, 1003), (1003, 1008), (40009, 40009)])
def test_equal_rows_are_equal(dtype, vocab, ld):
    """Beams with the same row and the same score: the lower beam comes first, token by token, wherever the rows lie."""
    x, s = make(8, vocab, dtype, 6, ld)
    x[1:] = x[0]
    s[:] = s[0]
    v, p, t = check(x, s, 8, 24)
    assert p[0].tolist() == list(range(8)) * 3
    assert torch.equal(v[0].view(3, 8), v[0].view(3, 8)[:, :1].expand(3, 8))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [600, 30000])
def test_ties_within_a_row(dtype, vocab):
    x, s = make(4, vocab, dtype, 7)
    x[0] = 1.5
    x[1, ::2] = 3.0
    x[2] = 0.0
    x[2, 1::3] = -0.0
    x[3] = torch.where(x[3] > 0, 2.0, x[3].float()).to(dtype)
    check(x, s, 4, 64)
    check(x, s, 1, 40)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_nothing_and_infinities(dtype):
    x, s = make(12, 3001, dtype, 8)
    x[0] = -INF  # nothing allowed
    x[1, 5:] = -INF  # a few
    x[2, ::3] = float("nan")
    x[3, 17] = INF
    x[4, 100:104] = INF
    x[4, 0] = float("nan")
    x[5] = float("nan")
    x[6, 1:] = -INF  # one token alone: its logarithm is 0
    s[7] = -INF
    s[8] = float("nan")
    x[9] = -6e4  # masked by large finite values, all
    x[10, 3:] = -6e4
    x[11] = INF
    for beams in (1, 2, 3, 4, 12):
        check(x, s, beams, 6)
    s[:] = -INF
    v, p, t = check(x, s, 12, 6)
    assert (p == -1).all() and (t == -1).all() and (v == -INF).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("low", [-1e10, -3.38e38])
def test_large_finite_masks(low, dtype):
    x, s = make(6, 5000, dtype, 9)
    x[0] = low
    x[1, 7:] = low
    x[2, :4999] = low
    x[3] = low / 2
    x[3, 9] = low
    x[4, 0] = -low
    # at this size a step of fp32 is far above 1, so a row's columns at its maximum share the probability
    check(x, s, 3, 4)


def test_first_step():
    """All beams hold the prompt: one has a score."""
    x, _ = make(8, 9001, F32, 10)
    x[1:4], x[5:] = x[0], x[4]
    s = torch.tensor([[0.0, -INF, -INF, -INF]] * 2, device="cuda")
    v, p, t = check(x, s, 4, 8)
    assert (p == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16])
def test_more_batches_than_maxima_are_kept_of(dtype):
    """A row of 4194304 columns, the first ones at its end and in its middle."""
    x = torch.full((2, 4194304), -1.0, dtype=dtype, device="cuda")
    x[0, -5:] = torch.tensor([3.0, 4.0, 2.0, 4.0, 1.0])
    x[0, 2097152] = 5.0
    x[1, ::65536] = 2.0
    s = torch.zeros(2, device="cuda")
    check(x, s, 2, 40)
    check(x, s, 1, 40)


def test_many_requests():
    """More rows than CTAs fit, of a few columns each; and one beam each."""
    x, s = make(24000, 37, F16, 12)
    v, p, t = vb.beam_select(x, s, 3, 4)
    pick = [0, 1, 4000, 7999]
    rows = [3 * r + b for r in pick for b in range(3)]
    w = check(x[rows].contiguous(), s[rows].contiguous(), 3, 4)
    for a, b in zip((v, p, t), w):
        assert torch.equal(a[pick], b)
    x, s = make(70000, 5, F32, 13)
    v, p, t = vb.beam_select(x, s, 1, 2)
    assert torch.equal(t.long(), x.topk(2, 1).indices) and bool((p == 0).all())
    state = torch.arange(70000, device="cuda").view(-1, 1).repeat(1, 3)
    vb.beam_reorder(state, torch.zeros(35000, 2, dtype=torch.int32, device="cuda"), 2)
    assert torch.equal(state[1::2], state[::2]) and torch.equal(state[::2, 0], torch.arange(0, 70000, 2, device="cuda"))


def test_scores_in_place():
    """out_scores may be the scores where as many are taken."""
    x, s = make(4, 700, F32, 11)
    want = vb.beam_select(x, s, 2, 2)
    lib = vb.beam._beam()[0]
    p, t = torch.empty(2, 2, dtype=torch.int32, device="cuda"), torch.empty(2, 2, dtype=torch.int32, device="cuda")
    ws = torch.empty(lib.verbo_beam_workspace(2, 2, 2), dtype=torch.uint8, device="cuda")
    rc = lib.verbo_beam_select(x.data_ptr(), 0, 2, 2, 700, 700, s.data_ptr(), 2, s.data_ptr(), p.data_ptr(),
                               t.data_ptr(), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert torch.equal(s.view(2, 2), want[0]) and torch.equal(p, want[1]) and torch.equal(t, want[2])


# ---------------------------------------------------------------- reorder --
def reordered(t, parents, beams):
    rows = t.shape[0]
    p = parents[:, :beams].long().cpu()
    own = torch.arange(beams).expand_as(p)
    p = torch.where((p < 0) | (p >= beams), own, p)
    at = (torch.arange(rows // beams)[:, None] * beams + p).view(-1)
    return t.cpu()[at]


@pytest.mark.parametrize("beams", [1, 2, 3, 4, 5, 8, 9, 16, 17, 32])
def test_reorder(beams):
    requests = 3
    rows = requests * beams
    g = torch.Generator(device="cuda")
    g.manual_seed(beams)

    def rand(*shape):
        return torch.randint(-128, 128, shape, generator=g, device="cuda")

    wide = rand(rows, 96).to(torch.int8)
    states = [rand(rows, 7).to(torch.int8), rand(rows, 5).int(), rand(rows, 4, 3, 8).half(), rand(rows, 3000).float(),
              rand(rows).to(torch.int64), rand(rows, 1).to(torch.int8), rand(rows, 4, 64).bfloat16(), rand(rows, 0).int(),
              rand(rows, 33).int()[:, 1:], wide[:, :48], wide[:, 48:], rand(rows, 2) > 0]
    parents = torch.randint(-1, beams + 1, (requests, beams + 2), generator=g, device="cuda", dtype=torch.int32)
    parents[0, :beams] = torch.arange(beams - 1, -1, -1)
    want = [reordered(t, parents, beams) for t in states]
    vb.beam_reorder(states, parents, beams)
    for t, w in zip(states, want):
        assert torch.equal(t.cpu(), w)
    one = rand(rows, 20).int()
    want = reordered(one, parents, beams)
    vb.beam_reorder(one, parents, beams)
    assert torch.equal(one.cpu(), want)


def test_reorder_many_states():
    parents = torch.tensor([[1, 0], [1, 1]], dtype=torch.int32, device="cuda")
    states = [torch.arange(4 * n, device="cuda").view(4, n) for n in range(1, 80)]
    want = [reordered(t, parents, 2) for t in states]
    vb.beam_reorder(states, parents, 2)
    assert all(torch.equal(t.cpu(), w) for t, w in zip(states, want))


def test_reorder_beyond_32_bits():
    """Rows 2.2 GB apart."""
    big = torch.zeros(2, 2_200_000_016, dtype=torch.uint8, device="cuda")
    big[0, -20:], big[1, -20:] = 1, 2
    big[0, :3], big[1, :3] = 3, 4
    vb.beam_reorder(big, torch.tensor([[1, 0]], dtype=torch.int32, device="cuda"), 2)
    assert big[0, -20:].tolist() == [2] * 20 and big[1, -20:].tolist() == [1] * 20
    assert big[0, :3].tolist() == [4] * 3 and big[1, :3].tolist() == [3] * 3 and int(big[0, 3:-20].max()) == 0


# ------------------------------------------------------- streams, captures --
def test_captured_and_replayed():
    x, s = make(12, 50001, BF16, 20)
    state = torch.arange(12 * 40, device="cuda").view(12, 40)
    vb.beam_select(x, s, 4, 8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        v, p, t = vb.beam_select(x, s, 4, 8)
        vb.beam_reorder(state, p, 4)
    for seed in (21, 22):
        y, z = make(12, 50001, BF16, seed)
        x.copy_(y)
        s.copy_(z)
        state.copy_(torch.arange(12 * 40, device="cuda").view(12, 40))
        graph.replay()
        want = vb.beam_select(y, z, 4, 8)
        for a, b in zip((v, p, t), want):
            assert torch.equal(a, b)
        assert torch.equal(state.cpu(), reordered(torch.arange(12 * 40, device="cuda").view(12, 40), want[1], 4))


def test_streams():
    """Calls on several streams at once, each with its own results."""
    streams = [torch.cuda.Stream() for _ in range(4)]
    data = [make(8, 30000 + i, F32, 30 + i) for i in range(4)]
    torch.cuda.synchronize()
    got = [[] for _ in streams]
    for _ in range(5):
        for i, st in enumerate(streams):
            got[i].append(vb.beam_select(*data[i], 4, 6, stream=st))
    torch.cuda.synchronize()
    for i, st in enumerate(streams):
        want = vb.beam_select(*data[i], 4, 6)
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want))

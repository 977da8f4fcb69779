"""GPU tests of the paged cache (verbo_b200/cache.py): bookkeeping and codes against
the definition (tests/cache_model.py), which they equal exactly, and attention
against 64 bits."""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import verbo_b200 as vb  # noqa: E402
from tests.cache_model import Model, same  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF = float("inf")
E4M3 = torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _needs(cuda_lib):
    if not torch.cuda.is_available():
        pytest.fail("gpu tests need a CUDA device")


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def new(layers=2, pages=40, heads=2, dim=32, rows=4, width=8, page=16, seed=0):
    """A cache with random codes (no NaN) and scales in every page, and no rows yet."""
    c = vb.PagedCache.new(layers, pages, heads, dim, rows, width, page)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    for t in (c.k, c.v):
        t.copy_((torch.randn(t.shape, generator=g, device="cuda") * 64).clamp(-448, 448).to(E4M3))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.exp2(torch.randint(-8, -3, t.shape, generator=g, device="cuda").float()))
    return c


def model(c):
    def np_(t):
        return t.view(torch.uint8).cpu().numpy() if t.dtype == E4M3 else t.cpu().numpy()

    return Model(*(np_(t) for t in (c.k, c.v, c.k_scale, c.v_scale, c.table, c.lens, c.refs)))


def check(c, m):
    vb.check()
    got = model(c)
    assert got.lens.tolist() == m.lens.tolist()
    assert got.table.tolist() == m.table.tolist()
    assert got.refs.tolist() == m.refs.tolist()
    counted = np.bincount(got.table[got.table >= 0], minlength=got.refs.size)
    assert got.refs.tolist() == counted.tolist()
    assert same(got.k, m.k) and same(got.v, m.v)
    assert np.array_equal(got.ks, m.ks) and np.array_equal(got.vs, m.vs)


def reserve(c, m, add):
    start, status = c.reserve(i32(add))
    want, code = m.reserve(np.asarray(add))
    check(c, m)
    assert status.tolist() == [code]
    assert start.tolist() == want.tolist()
    return start, code


# ------------------------------------------------------------------ pages --
def test_reserve_boundaries():
    c = new()
    m = model(c)
    for add in ([1, 0, 16, 17], [15, -3, 16, 15], [1, 1, 0, 0], [0, 0, 0, 0], [16, 33, 1, 2]):
        assert reserve(c, m, add)[1] == 0


def test_reserve_fills_the_pool_to_the_last_page():
    c = new(pages=6, rows=3, width=8)
    m = model(c)
    assert reserve(c, m, [33, 16, 0])[1] == 0
    assert reserve(c, m, [16, 17, 16])[1] == 2  # four pages wanted, two left
    assert reserve(c, m, [0, 16, 16])[1] == 0
    assert reserve(c, m, [0, 1, 0])[1] == 1
    assert reserve(c, m, [15, 0, 0])[1] == 0  # inside a page: needs none


def test_reserve_refuses_what_the_table_does_not_hold():
    c = new(pages=40, rows=3, width=3)
    m = model(c)
    assert reserve(c, m, [48, 0, 0])[1] == 0
    assert reserve(c, m, [0, 49, 49])[1] == -2
    assert reserve(c, m, [1, 1, 1])[1] == -1
    assert reserve(c, m, [0, 0, 2**31 - 1])[1] == -3
    assert reserve(c, m, [-2**31, 48, 48])[1] == 0


def test_shared_pages_are_copied_on_write():
    c = new(rows=4, pages=60)
    m = model(c)
    reserve(c, m, [20, 0, 0, 0])
    parents = np.zeros((1, 4), dtype=np.int32)
    c.fork(i32(parents), 4)
    m.fork(parents, 4)
    check(c, m)
    reserve(c, m, [0, 1, 0, 1])  # two of four write: both copy
    reserve(c, m, [1, 0, 1, 0])  # the last two: one copies, one keeps
    reserve(c, m, [3, 14, 2, 40])


def test_fork_and_free_of_single_rows():
    c = new(rows=6, pages=60, width=5)
    m = model(c)
    reserve(c, m, [16, 17, 0, 80, 1, 33])
    for parents, beams in (([[1, 1, -1], [2, 0, 7]], 3), ([[0]] * 6, 1), ([[5, 4, 3, 2, 1, 0]], 6), ([[0, 0]] * 3, 2)):
        c.fork(i32(parents), beams)
        m.fork(np.asarray(parents), beams)
        check(c, m)
    for keep in ([-1, 100, 5, 0, 16, 17], [0, 15, 16, 17, 1, 2], [0] * 6):
        c.free(i32(keep))
        m.free(np.asarray(keep))
        check(c, m)


@pytest.mark.parametrize("pages,live", [(40, 0), (40, 1), (40, 20), (40, 39), (40, 40), (16384, 9000), (16385, 3),
                                        (16385, 16385), (33000, 12345)])
def test_compact(pages, live):
    """Pools that one CTA looks through, and larger ones."""
    width = -(-pages // 5)
    c = new(pages=pages, rows=5, width=width, layers=2 if pages < 100 else 1, heads=1, dim=16)
    order = np.random.default_rng(live).permutation(pages)[:live]
    t = np.full((5, width), -1, dtype=np.int32)
    t.reshape(-1)[:live] = order
    c.table.copy_(i32(t))
    c.lens.copy_(i32((t >= 0).sum(1) * 16))
    c.refs.copy_(i32(np.bincount(order, minlength=pages)))
    m = model(c)
    info = c.compact()
    want = m.compact()
    check(c, m)
    assert info.tolist() == list(want)
    assert c.compact().tolist() == [live, 0]
    check(c, m)


@pytest.mark.parametrize("seed,rows,beams,pages,page,dim,heads", [
    (0, 8, 4, 300, 16, 16, 1), (1, 12, 3, 90, 32, 48, 2), (2, 5, 5, 60, 256, 128, 1), (3, 64, 32, 5000, 16, 16, 1),
    (4, 12, 4, 17000, 16, 16, 1),
])
def test_any_sequence(seed, rows, beams, pages, page, dim, heads):
    rng = np.random.default_rng(seed)
    c = new(pages=pages, rows=rows, width=7, page=page, dim=dim, heads=heads, layers=1, seed=seed)
    m = model(c)
    for _ in range(40):
        op = rng.integers(0, 8)
        if op < 4:
            reserve(c, m, rng.integers(-1, rng.choice([2, page, 3 * page]), rows))
        elif op < 6:
            parents = rng.integers(-1 if rng.random() < 0.2 else 0, beams, (rows // beams, beams))
            c.fork(i32(parents), beams)
            m.fork(parents, beams)
        elif op == 6:
            keep = np.where(rng.random(rows) < 0.3, rng.integers(0, 4 * page, rows), -1)
            c.free(i32(keep))
            m.free(keep)
        else:
            assert c.compact().tolist() == list(m.compact())
        check(c, m)


def test_no_rows():
    c = new(rows=0, pages=5)
    start, status = c.reserve(i32([]))
    assert start.numel() == 0 and status.tolist() == [0]
    c.fork(i32([]).view(0, 2), 2)
    c.free(i32([]))
    c.append(0, torch.empty(0, 2, 32, device="cuda"), torch.empty(0, 2, 32, device="cuda"), i32([]))
    assert c.attend(0, torch.empty(0, 4, 32, device="cuda")).shape == (0, 4, 32)
    assert c.compact().tolist() == [0, 0]
    vb.check()


def test_the_largest_tables():
    """4096 rows, pages of several chunks, one page shared by all."""
    c = new(layers=1, pages=20000, heads=1, dim=16, rows=4096, width=4)
    m = model(c)
    reserve(c, m, np.where(np.arange(4096) == 4095, 10, 0))
    c.table.copy_(c.table[4095].expand(4096, 4).contiguous())
    c.lens.fill_(10)
    c.refs[c.table[0, 0]] = 4096
    m = model(c)
    reserve(c, m, np.arange(4096) % 3)
    reserve(c, m, 1 + np.arange(4096) % 40)
    assert c.compact().tolist() == list(m.compact())
    check(c, m)


def test_the_largest_pool():
    """4194304 pages: the lowest free ones first, and the highest live ones moved first."""
    pages = 4194304
    c = vb.PagedCache.new(1, pages, 1, 16, 2, 8, 16)
    far = [4194303, 3, 2048, 4192256]
    c.table[0, :4] = i32(far)
    c.refs[torch.tensor(far, device="cuda")] = 1
    c.lens[0] = 60
    for n, p in enumerate(far):
        c.k.view(torch.uint8)[0, p] = n + 1
        c.v_scale[0, p] = n + 1
    start, status = c.reserve(i32([5, 33]))
    assert status.tolist() == [0] and start.tolist() == [60, 0]
    assert c.table.tolist() == [far + [0, -1, -1, -1], [1, 2, 4, -1, -1, -1, -1, -1]]
    c.free(i32([-1, 17]))
    assert c.table[1].tolist() == [1, 2] + [-1] * 6
    assert c.compact().tolist() == [7, 3]  # live: 0, 1, 2, 3, 2048, 4192256, 4194303
    assert c.table.tolist() == [[4, 3, 6, 5, 0, -1, -1, -1], [1, 2, -1, -1, -1, -1, -1, -1]]
    assert c.refs[:8].tolist() == [1] * 7 + [0] and int(c.refs.sum()) == 7
    assert [int(c.k.view(torch.uint8)[0, p].max()) for p in (4, 3, 6, 5)] == [1, 2, 3, 4]
    assert [float(c.v_scale[0, p].max()) for p in (4, 3, 6, 5)] == [1, 2, 3, 4]
    vb.check()


# ----------------------------------------------------------------- append --
def tokens(n, heads, dim, dtype, seed, spread=3.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(n, heads, dim, generator=g, device="cuda")
    return (x * torch.exp2((torch.rand(n, 1, 1, generator=g, device="cuda") * 2 - 1) * spread)).to(dtype)


def append(c, m, layer, k, v, start, off=None):
    given = None if off is None else torch.tensor(off, dtype=torch.int64, device="cuda")
    if off is None:
        off = np.arange(c.rows + 1) * (k.shape[0] // c.rows)
    c.append(layer, k, v, i32(start), off=given)
    m.append(layer, k.float().cpu().numpy(), v.float().cpu().numpy(), start, off)
    check(c, m)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim,heads,page", [(16, 1, 16), (48, 3, 32), (64, 2, 16), (80, 2, 48), (128, 1, 256)])
def test_append_steps(dtype, dim, heads, page):
    """Token by token over a block's end, with a prompt before it."""
    c = new(rows=3, width=6, pages=20, dim=dim, heads=heads, page=page)
    m = model(c)
    seed = 0
    for add in ([5, 14, 0], [1, 1, 1], [1, 1, 1], [1, 1, 1], [20, 3, 31], [1, 0, 1]):
        start, code = reserve(c, m, add)
        assert code == 0
        off = np.concatenate([[0], np.cumsum(add)])
        k, v = (tokens(int(off[-1]), heads, dim, dtype, seed + i) for i in (0, 1))
        append(c, m, seed // 2 % 2, k, v, start.cpu().numpy(), off)
        seed += 2


@pytest.mark.parametrize("n", [1, 2, 17])
def test_append_equal_numbers(n):
    c = new(rows=4, width=6, pages=30)
    m = model(c)
    reserve(c, m, [3, 16, 0, 31])
    start, _ = reserve(c, m, [n] * 4)
    append(c, m, 1, tokens(4 * n, 2, 32, BF16, 1), tokens(4 * n, 2, 32, BF16, 2), start.cpu().numpy())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_values(dtype):
    """Zeros, infinities, NaNs, tiny and huge values, ties between codes, amax at a scale's border."""
    c = new(rows=1, width=8, pages=8, heads=1, layers=1)
    m = model(c)
    for i, fill in enumerate([0.0, -0.0, INF, -INF, float("nan"), 1e-45, 1e-30, 2.0**-64, 3e38, 448.0, 449.0, 464.0,
                              448.0 * 2**-3, 2.0**-9, 2.0**-10, 3 * 2.0**-10, -1.0625, 1.1875, 7.0, 896.0, 1792.0]):
        start, _ = reserve(c, m, [1])
        k = torch.full((1, 1, 32), fill, dtype=F32, device="cuda")
        k[0, 0, ::2] = 0.5 if i % 2 else fill
        k[0, 0, 1] = -1.5 if i % 3 == 0 else fill
        v = torch.full((1, 1, 32), fill, dtype=F32, device="cuda")
        append(c, m, 0, k.to(dtype), v.to(dtype), start.cpu().numpy())


def test_append_rows_left_out():
    c = new(rows=4, width=2, pages=6, layers=1)
    m = model(c)
    start, code = reserve(c, m, [40, 0, 0, 0])
    assert code == -1 and start.tolist() == [-1] * 4
    append(c, m, 0, tokens(8, 2, 32, F16, 0), tokens(8, 2, 32, F16, 1), start.cpu().numpy())
    reserve(c, m, [5, 0, 32, 1])
    c.table[3, 0] = 77  # no page: its tokens are not written
    m = model(c)
    off = torch.tensor([0, 5, 5, 37, 38], device="cuda")
    k, v = tokens(38, 2, 32, F16, 2), tokens(38, 2, 32, F16, 3)
    c.append(0, k, v, i32([0, -1, 0, 0]), off=off)
    m.append(0, k.float().cpu().numpy(), v.float().cpu().numpy(), [0, -1, 0, 0], off.tolist())
    vb.check()
    got = model(c)
    assert same(got.k, m.k) and same(got.v, m.v) and np.array_equal(got.ks, m.ks)
    # behind the table's width: what lies there is not written
    before = got
    c.append(0, tokens(4, 2, 32, F16, 4), tokens(4, 2, 32, F16, 5), i32([32, 32, 2**31 - 1, 40]))
    after = model(c)
    assert same(before.k, after.k) and np.array_equal(before.vs, after.vs)


def test_append_strides():
    """Keys and values out of one fused projection, and heads before tokens; odd addresses."""
    c = new(rows=2, width=4, pages=8, heads=3, dim=48, layers=1)
    m = model(c)
    start, _ = reserve(c, m, [9, 9])
    fused = tokens(18, 8, 48, BF16, 0)
    append(c, m, 0, fused[:, 2:5], fused[:, 5:], start.cpu().numpy())
    start, _ = reserve(c, m, [4, 4])
    turned = tokens(3, 8, 48, F32, 1).transpose(0, 1)
    append(c, m, 0, turned, turned.flip(0).contiguous(), start.cpu().numpy())
    start, _ = reserve(c, m, [2, 2])
    flat = tokens(1, 1, 4 * 3 * 48 + 1, F16, 2).view(-1)[1:].view(4, 3, 48)
    append(c, m, 0, flat, flat, start.cpu().numpy())


# ----------------------------------------------------------------- attend --
def filled(lens, heads, dim, page, seed=0, layers=1, spare=0, scales=(-8, -5), width=None):
    """A cache whose rows have these lengths, in scattered pages, with unit keys and values."""
    used = [-(-n // page) for n in lens]
    pages = max(1, sum(used)) + spare
    c = new(layers=layers, pages=pages, heads=heads, dim=dim, rows=len(lens), width=width or max(1, max(used)), page=page,
            seed=seed)
    order = np.random.default_rng(seed).permutation(pages)
    t = np.full((len(lens), c.width), -1, dtype=np.int32)
    at = 0
    for r, n in enumerate(used):
        t[r, :n] = order[at:at + n]
        at += n
    c.table.copy_(i32(t))
    c.lens.copy_(i32(lens))
    c.refs.copy_(i32(np.bincount(t[t >= 0], minlength=pages)))
    for s in (c.k_scale, c.v_scale):
        s.copy_(torch.exp2(torch.randint(*scales, s.shape, device="cuda",
                                         generator=torch.Generator("cuda").manual_seed(seed)).float()))
    return c


def gathered(c, layer, r, n, what, scale):
    pid = c.table[r, :-(-n // c.page)].long()
    ok = (pid >= 0) & (pid < c.pages)
    at = torch.where(ok, pid, 0)
    x = what[layer].view(torch.uint8)[at].view(E4M3).double() * scale[layer][at].double().repeat_interleave(16, 2)[..., None]
    x = x.transpose(0, 1).reshape(c.heads, -1, c.dim)[:, :n]
    return x, ok.repeat_interleave(c.page)[:n]


def check_attend(c, q, layer=0, scale=None, dtype=None, out=None):
    """Against 64 bits.  Tolerance: a score is off by its products, 2^-22 of the row's
    largest |q| times the sum of |k|, by sixteen cut additions on the tensor cores,
    2^-22 of the sum of |q k| each at most, and by three roundings and the exponential,
    2^-22 of (|s| + 1); scores that are all off by d move a mean of values by less than 4 d of the
    largest.  The weights' and sums' own roundings are below 2^-18 of the largest."""
    got = c.attend(layer, q, scale=scale, dtype=dtype, out=out)
    vb.check()
    sc = 1.0 / math.sqrt(c.dim) if scale is None else scale
    steps = q.shape[0] // c.rows
    group = q.shape[1] // c.heads
    eps = torch.finfo(got.dtype).eps / 2
    lens = c.lens.tolist()
    for r in range(c.rows):
        n = max(0, min(lens[r], c.width * c.page))
        k, ok = gathered(c, layer, r, n, c.k, c.k_scale)
        v, _ = gathered(c, layer, r, n, c.v, c.v_scale)
        for i in range(steps):
            end = n - (steps - 1 - i)
            y = got[r * steps + i].double().view(c.heads, group, c.dim)
            if end <= 0 or not bool(ok[:end].any()):
                assert bool((y == 0).all())
                continue
            x = q[r * steps + i].double().view(c.heads, group, c.dim)
            kk, vv = k[:, :end][:, ok[:end]], v[:, :end][:, ok[:end]]
            s = x @ kk.transpose(1, 2) * sc
            want = torch.softmax(s, 2) @ vv
            sums = (x.abs() @ kk.abs().transpose(1, 2)).amax(2) * abs(sc)
            large = x.abs().amax(2) * kk.abs().sum(2).amax(1)[:, None] * abs(sc)
            d = 2.0**-22 * (large + 16 * sums + 3 * (s.abs().amax(2) + 1))
            tol = (4 * d + 2.0**-18)[..., None] * vv.abs().amax((1, 2))[:, None, None] + eps * want.abs()
            if got.dtype == F16:
                tol = tol + 2.0**-25  # subnormal results
            worst = ((y - want).abs() / tol).max()
            assert bool(((y - want).abs() <= tol).all()), (r, i, float(worst))
    return got


def widened(c, tokens=100000):
    """The same cache with room for longer rows: its attention is split over the card, not over a cluster."""
    table = torch.full((c.rows, -(-tokens // c.page)), -1, dtype=torch.int32, device="cuda")
    table[:, :c.width] = c.table
    return vb.PagedCache(c.k, c.v, c.k_scale, c.v_scale, table, c.lens, c.refs)


def queries(n, heads, dim, dtype, seed=1, size=2.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(n, heads, dim, generator=g, device="cuda") * size).to(dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 7), (3, 8), (1, 12)])
def test_attend_shapes(dtype, dim, heads, group):
    c = filled([0, 1, 15, 16, 17, 100, 1, 333], heads, dim, 16)
    q = queries(8, heads * group, dim, dtype)
    check_attend(c, q)
    check_attend(widened(c), q)


@pytest.mark.parametrize("page", [16, 48, 256])
@pytest.mark.parametrize("steps", [1, 2, 5, 32])
@pytest.mark.parametrize("dim,group,dtype", [(64, 4, BF16), (128, 3, BF16), (80, 5, F16), (128, 2, F32)])
def test_attend_steps(page, steps, dim, group, dtype):
    """Several last tokens, each sees up to its own; rows shorter than them."""
    c = filled([40, 0, 1, 5, 31, 32, 33, 700], 2, dim, page, layers=2)
    q = queries(8 * steps, 2 * group, dim, dtype)
    check_attend(c, q, layer=1, dtype=F32)
    check_attend(widened(c), q, layer=1, dtype=F32)


@pytest.mark.parametrize("dim,heads,group,lens", [
    (128, 8, 4, [5000, 1, 0, 9000, 333, 64]), (64, 2, 7, [20011]), (128, 1, 64, [3001]), (128, 8, 1, [40000]),
    (64, 1, 1, [100003]), (80, 4, 8, [777] * 40), (128, 2, 16, [130] * 100), (64, 4, 4, [16] * 500),
])
def test_attend_lengths(dim, heads, group, lens):
    c = filled(lens, heads, dim, 64)
    check_attend(c, queries(len(lens), heads * group, dim, F32))
    check_attend(c, queries(len(lens), heads * group, dim, BF16, size=20.0))


def test_attend_4096_rows():
    lens = [(i * 37) % 50 for i in range(4096)]
    c = filled(lens, 1, 32, 16)
    q = queries(4096, 2, 32, F16)
    got = c.attend(0, q)
    short = filled(lens, 1, 32, 16)
    # the same rows, some of them alone, against 64 bits
    pick = [0, 1, 2, 4095, 4094, 2048, 777]
    sub = vb.PagedCache(short.k, short.v, short.k_scale, short.v_scale, short.table[pick].contiguous(),
                        short.lens[pick].contiguous(), short.refs)
    want = check_attend(sub, q[pick].contiguous())
    # the parts are cut elsewhere: equal but for the last bits of fp16
    assert torch.allclose(got[pick].float(), want.float(), rtol=2.0**-10, atol=2.0**-12)


@pytest.mark.parametrize("dim", [64, 128])
def test_attend_scales(dim):
    """Blocks whose scales lie far apart, zero among them; large and small queries; a negative and a zero scale."""
    c = filled([500, 33], 2, dim, 32, scales=(-12, 6))
    c.v_scale[0, ::5] = 0.0
    c.k_scale[0, ::7] = 0.0
    c.v_scale.view(-1)[3] = 2.0**-40
    for size, scale in ((1e-3, None), (1e-6, 30.0), (0.02, -0.5), (5.0, 0.0)):
        check_attend(c, queries(2, 6, dim, F32, size=size), scale=scale)
    check_attend(c, queries(2, 6, dim, F32, size=1e-30), scale=1e28)
    zero = torch.zeros(2, 6, dim, device="cuda")
    check_attend(c, zero)


def test_attend_scales_of_the_caller():
    """Scales that are no powers of two."""
    c = filled([700, 31], 2, 64, 16)
    c.k_scale.mul_(1.37)
    c.v_scale.mul_(0.61)
    check_attend(c, queries(2, 4, 64, BF16), dtype=F32)


@pytest.mark.parametrize("dim", [64, 96, 128])
def test_what_lies_behind_a_row_is_not_seen(dim):
    """NaN codes, infinite scales: in the rest of a block, of a page, and in other pages."""
    c = filled([21, 0, 64, 1], 2, dim, 32, spare=3)
    q = queries(4, 4, dim, BF16)
    want = check_attend(c, q)
    live = torch.zeros(c.pages, c.page, dtype=torch.bool, device="cuda")
    for r, n in enumerate(c.lens.tolist()):
        for i in range(n):
            live[int(c.table[r, i // c.page]), i % c.page] = True
    for t in (c.k, c.v):
        t.view(torch.uint8).masked_fill_(~live[None, :, None, :, None], 0x7F)
    block = live.view(c.pages, -1, 16).any(2)
    for t in (c.k_scale, c.v_scale):
        t.masked_fill_(~block[None, :, None, :], float("nan"))
    c.table.masked_fill_(c.table < 0, 2**31 - 1)
    assert torch.equal(c.attend(0, q), want)


def test_bad_pages_and_lengths_are_bounded():
    """Entries that are no pages are left out; lengths beyond the table end with it."""
    c = filled([100, 100, 100, 64], 2, 64, 16, width=8)
    c.table[0, 2] = -1
    c.table[1, :] = 2**31 - 1
    c.table[2, 6] = c.pages
    c.table[3, 4:] = c.table[0, 0]
    c.lens.copy_(i32([100, 100, -5, 2**31 - 1]))
    check_attend(c, queries(4, 2, 64, F32))


def test_nan_and_infinite_tokens():
    """A NaN in a row's own tokens is the result's; other rows and heads are untouched."""
    c = filled([50, 50], 2, 64, 16)
    q = queries(2, 4, 64, F32)
    want = c.attend(0, q)
    c.v.view(torch.uint8)[0, int(c.table[0, 1]), 0, 3, 5] = 0x7F
    got = c.attend(0, q)
    assert bool(torch.isnan(got[0, :2, 5]).all())
    assert torch.equal(got[1], want[1]) and torch.equal(got[0, 2:], want[0, 2:])
    keep = [i for i in range(64) if i != 5]
    assert torch.equal(got[0, :2, keep], want[0, :2, keep])
    q[1, 0, 0] = float("nan")
    assert bool(torch.isnan(c.attend(0, q)[1, 0]).all())


def test_attend_strides():
    """Queries out of a fused projection, heads before tokens, odd addresses; an output of the caller's."""
    c = filled([90, 7], 2, 48, 16)
    fused = queries(4, 10, 48, BF16)
    want = check_attend(c, fused[:, :6].contiguous())
    assert torch.equal(check_attend(c, fused[:, :6]), want)
    turned = fused[:, :6].transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.zeros(6, 4, 48, dtype=BF16, device="cuda").transpose(0, 1)
    assert torch.equal(check_attend(c, turned, out=out), want) and torch.equal(out, want)
    flat = torch.zeros(4 * 6 * 48 + 1, dtype=BF16, device="cuda")[1:].view(4, 6, 48)
    flat.copy_(fused[:, :6])
    wide = torch.full((4, 6, 52), 9.0, dtype=F32, device="cuda")
    got = c.attend(0, flat, out=wide[:, :, 1:49])
    assert torch.equal(got.bfloat16(), want) and bool((wide[:, :, 49:] == 9).all()) and bool((wide[:, :, 0] == 9).all())


def test_pools_beyond_32_bits():
    """Pages more than 4 GB into the pools."""
    c = vb.PagedCache.new(2, 20000, 8, 128, 1, 4, 128)  # 2.6 GB a layer
    c.table.copy_(i32([[19999, 0, 19998, -1]]))
    c.lens.fill_(0)
    c.refs[[0, 19998, 19999]] = 1
    k, v = tokens(300, 8, 128, BF16, 0, 0.0), tokens(300, 8, 128, BF16, 1, 0.0)
    c.lens.fill_(300)
    c.append(1, k, v, i32([0]))
    got = c.attend(1, queries(1, 32, 128, F32))
    small = vb.PagedCache.new(1, 3, 8, 128, 1, 4, 128)
    small.table.copy_(i32([[2, 0, 1, -1]]))
    small.refs.fill_(1)
    small.lens.fill_(300)
    small.append(0, k, v, i32([0]))
    assert torch.equal(got, check_attend(small, queries(1, 32, 128, F32)))
    assert c.compact().tolist() == [3, 2]
    assert c.table.tolist() == [[1, 0, 2, -1]]
    assert torch.equal(got, c.attend(1, queries(1, 32, 128, F32)))


# ------------------------------------------------------- streams, captures --
def test_a_step_captured_and_replayed():
    """Reserve, append, attend and fork of a step in one graph, replayed over page borders; the eager cache beside it."""
    def start():
        return filled([30, 14, 31, 1], 2, 64, 16, seed=3, spare=30, width=8)

    a, b = start(), start()
    q, k, v = queries(4, 4, 64, BF16), tokens(4, 2, 64, BF16, 1), tokens(4, 2, 64, BF16, 2)
    add, parents = i32([1, 1, 1, 1]), i32([[1, 1], [0, 1]])

    def step(c):
        first, status = c.reserve(add)
        c.append(0, k, v, first)
        y = c.attend(0, q)
        c.fork(parents, 2)
        return first, status, y

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(start())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(a)
    for i in range(20):
        for t, s in ((q, 10 + i), (k, 40 + i), (v, 70 + i)):
            t.copy_(queries(4, t.shape[1], 64, BF16, s))
        graph.replay()
        want = step(b)
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        m = model(b)
        check(a, m)


def test_streams():
    """Attention of several caches on several streams at once."""
    streams = [torch.cuda.Stream() for _ in range(4)]
    caches = [filled([1000 * i + 5, 77, 300], 2, 128, 16, seed=i) for i in range(4)]
    qs = [queries(3, 8, 128, F16, seed=i) for i in range(4)]
    torch.cuda.synchronize()
    got = [[] for _ in streams]
    for _ in range(5):
        for i, st in enumerate(streams):
            got[i].append(caches[i].attend(0, qs[i], stream=st))
    torch.cuda.synchronize()
    for i in range(4):
        want = caches[i].attend(0, qs[i])
        assert all(torch.equal(g, want) for g in got[i])


def test_free_and_compact_captured():
    c = filled([40, 33, 16, 1], 2, 64, 16, spare=20, width=4)
    keep = i32([-1, 10, 0, 1])
    c.free(i32([-1] * 4))
    c.compact()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.free(keep)
        info = c.compact()
    for kept in ([-1, 10, 0, 1], [20, 20, 20, 0], [0, 3, 1, 1]):
        keep.copy_(i32(kept))
        m = model(c)
        graph.replay()
        m.free(np.asarray(kept))
        want = m.compact()
        assert info.tolist() == list(want)
        check(c, m)


def test_threads():
    """Host threads, each with its own cache and stream, one step after the other."""
    import threading

    def work(i, out):
        with torch.cuda.stream(torch.cuda.Stream()):
            c = filled([50 + i, 7, 333], 2, 64, 16, seed=i, spare=20, width=30)
            add = i32([1, 0, 2])
            for n in range(20):
                start, status = c.reserve(add)
                c.append(0, tokens(6, 2, 64, F16, n), tokens(6, 2, 64, F16, n + 1), start,
                         off=torch.tensor([0, 1, 1, 3], device="cuda"))
                y = c.attend(0, queries(3, 4, 64, BF16, seed=n))
                s = vb.beam_select(y.view(3, -1), torch.zeros(3, device="cuda"), 3, 5)
            torch.cuda.current_stream().synchronize()
            out[i] = (y, *s, c.table, c.lens, status)

    alone, together = {}, {}
    for i in range(4):
        work(i, alone)
    threads = [threading.Thread(target=work, args=(i, together)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    vb.check()
    for i in range(4):
        assert all(torch.equal(a, b) for a, b in zip(alone[i], together[i]))


def test_python_refusals():
    c = filled([10, 20], 2, 64, 16)
    q = queries(2, 4, 64, BF16)
    for fn in (lambda: c.attend(1, q), lambda: c.attend(0, q[:1]), lambda: c.attend(0, q[:, :, :32]),
               lambda: c.attend(0, q.cpu()), lambda: c.attend(0, q.double()), lambda: c.attend(0, queries(2, 3, 64, F32)),
               lambda: c.attend(0, queries(66, 4, 64, F32)), lambda: c.attend(0, q.transpose(1, 2)),
               lambda: c.attend(0, q, out=q), lambda: c.attend(0, q, dtype=torch.float64),
               lambda: c.attend(0, q, out=torch.empty(2, 4, 64, device="cuda"), dtype=F16),
               lambda: c.attend(0, q, scale=INF), lambda: c.append(0, q, q, i32([0, 0])),
               lambda: c.append(0, q[:, :2], q[:1, :2], i32([0, 0])), lambda: c.append(0, q[:, :2], q[:, :2], i32([0])),
               lambda: c.append(0, q[:, :2], q[:, :2], i32([0, 0]).long()),
               lambda: c.append(0, q[:1, :2], q[:1, :2], i32([0, 0])), lambda: c.append(2, q[:, :2], q[:, :2], i32([0, 0])),
               lambda: c.reserve(i32([1])), lambda: c.reserve(i32([1, 1]).float()), lambda: c.fork(i32([[0, 0]]), 3),
               lambda: c.fork(i32([[0, 0, 0]]), 0), lambda: c.fork(i32([[0], [0]]), 2), lambda: c.free(i32([1, 2, 3]))):
        with pytest.raises(vb.VerboCudaError):
            fn()

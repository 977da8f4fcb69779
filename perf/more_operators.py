"""Beam search and the cache that its beams share, as they are measured.

``select``   a step of beam search over the model's logits: the best continuations of each request's beams by their
             summed log-probabilities, and the beams' states put in the order of the chosen parents
``append``   new keys and values written into a paged cache of 8-bit floats (e4m3) with a power-of-two scale for each
             block of 16 tokens and head
``attend``   attention of a row's last tokens over its pages of that cache
``branch``   the cache after a step of the search: rows fork from their parents and share their pages, and the pages
             that the next token would write are made their own
``compact``  the cache's live pages moved to the front of the pool

``run`` computes them in plain torch, or calls the library where ``own`` is true.
"""
import math

import torch

own = False

VOCAB = 151936  # the vocabulary of the library's own workloads; 49152 is that of its single-row one
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 16  # tokens that share a scale
LOWEST = -64  # the smallest exponent of a scale


# ------------------------------------------------------------------ cases --
def _select(name, requests, beams, vocab, dtype, take, hist, extra=0, first=False, masked="none"):
    return {"name": name, "op": "select", "requests": requests, "beams": beams, "vocab": vocab, "dtype": dtype,
            "take": take, "hist": hist, "extra": extra, "first": first, "masked": masked}


def _append(name, rows, tokens, ragged, kv, dim, page, longest, dtype):
    return {"name": name, "op": "append", "rows": rows, "tokens": tokens, "ragged": ragged, "kv": kv, "dim": dim,
            "page": page, "longest": longest, "dtype": dtype}


def _attend(name, rows, steps, heads, kv, dim, page, shortest, longest, dtype, out_dtype):
    return {"name": name, "op": "attend", "rows": rows, "steps": steps, "heads": heads, "kv": kv, "dim": dim,
            "page": page, "shortest": shortest, "longest": longest, "dtype": dtype, "out_dtype": out_dtype}


def _branch(name, requests, beams, add, kv, dim, page, layers, shortest, longest):
    return {"name": name, "op": "branch", "requests": requests, "beams": beams, "add": add, "kv": kv, "dim": dim,
            "page": page, "layers": layers, "shortest": shortest, "longest": longest}


def _compact(name, rows, pages, live, kv, dim, page, layers):
    return {"name": name, "op": "compact", "rows": rows, "pages": pages, "live": live, "kv": kv, "dim": dim,
            "page": page, "layers": layers}


def listed():
    return [
        # one request's first step: all beams hold the prompt, so one of them alone has a score
        _select("select-1x4", 1, 4, 49152, "f32", 8, 64, first=True),
        # a batch with a vocabulary of odd size, under a grammar's mask, whose decoder carries a recurrent state
        _select("select-16x5-odd", 16, 5, 50257, "f32", 10, 300, extra=65536, masked="mixed"),
        # the largest batch, bf16 logits
        _select("select-64x8-bf16", 64, 8, VOCAB, "bf16", 16, 1024),
        # one decode step of a serving batch
        _append("append-64", 64, 1, False, 8, 128, 64, 1024, "bf16"),
        # four prompts of different lengths
        _append("append-prompts", 4, 2000, True, 8, 128, 64, 4096, "f16"),
        # one generation of a small model (14 heads over 2, 64 wide)
        _attend("attend-1", 1, 1, 14, 2, 64, 16, 1500, 1500, "f32", "f32"),
        # a serving batch of mixed lengths, one of the rows empty
        _attend("attend-64", 64, 1, 32, 8, 128, 64, 0, 8192, "bf16", "bf16"),
        # two long documents, four speculated tokens each
        _attend("attend-2-long", 2, 4, 32, 8, 128, 64, 100003, 131072, "f16", "f16"),
        # a step of one request with four beams
        _branch("branch-1x4", 1, 4, 1, 2, 64, 16, 2, 700, 700),
        # a step of thirty-two requests with eight beams
        _branch("branch-32x8", 32, 8, 1, 8, 128, 64, 2, 300, 2500),
        # a small pool in which half of the pages are left after requests have ended
        _compact("compact-600", 8, 600, 0.5, 2, 64, 16, 2),
        # the same for a serving pool
        _compact("compact-5000", 64, 5000, 0.6, 8, 128, 64, 2),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(["select", "append", "attend", "branch", "compact"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    kv, dim, page = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 96, 128]), rng.choice([16, 32, 64, 128])
    if op == "select":
        beams = _spread(rng, 1, 32)
        vocab = _spread(rng, 1000, VOCAB)
        most = 64 * 8 * VOCAB * 2 // (vocab * SIZE[dtype] * beams)
        requests = _spread(rng, 1, max(1, min(512 // beams, most)))
        c = _select("", requests, beams, vocab, dtype, min(64, beams * rng.choice([1, 2, 2])), _spread(rng, 1, 2048),
                    extra=rng.choice([0, 0, _spread(rng, 1, 65536)]), first=rng.random() < 0.2,
                    masked=rng.choice(["none", "none", "mixed"]))
    elif op == "append":
        ragged = rng.random() < 0.5
        tokens = _spread(rng, 1, 2000) if ragged else rng.choice([1, 1, 2, 5])
        rows = _spread(rng, 1, max(1, min(128, 8000 // tokens)))
        c = _append("", rows, tokens, ragged, kv, dim, page, max(1, min(4096, 66000 // rows)), dtype)
    elif op == "attend":
        steps, group = rng.choice([1, 1, 1, 2, 4, 8]), rng.choice([1, 2, 4, 7, 8, 16])
        rows = _spread(rng, 1, 128)
        longest = _spread(rng, 1, max(1, min(131072, 64 * 4096 * 1024 // (rows * kv * dim * max(1, steps * group // 8)))))
        c = _attend("", rows, steps, kv * group, kv, dim, page, rng.choice([0, longest // 2, longest]), longest, dtype,
                    rng.choice(["f32", dtype]))
    elif op == "branch":
        requests, beams = _spread(rng, 1, 32), _spread(rng, 2, 8)
        longest = max(1, min(2500, _spread(rng, 20, 4000)))
        c = _branch("", requests, beams, rng.choice([1, 1, 1, 3, 16]), kv, dim, page, 2,
                    rng.choice([1, longest // 2 + 1, longest]), longest)
    else:
        pages = _spread(rng, 20, 5000)
        page = min(page, 64)
        c = _compact("", _spread(rng, 1, min(64, pages // 4)), pages, rng.choice([0.1, 0.4, 0.6, 0.9, 1.0]), kv, dim,
                     page, 2)
    del c["name"]
    return c


# ----------------------------------------------------------------- inputs --
def _lens(case):
    """The rows' lengths, spread evenly over the case's range: what a pass has to move goes by the case alone."""
    n, a, b = case["rows"], case["shortest"], case["longest"]
    return [b if n == 1 else a + (b - a) * i // (n - 1) for i in range(n)]


def _counts(case):
    """New tokens of each row: the same for all, or from a half of the most up to it."""
    n, most = case["rows"], case["tokens"]
    return [most if n == 1 or not case["ragged"] else most - (most - most // 2) * i // (n - 1) for i in range(n)]


def _pool(gen, layers, pages, kv, page, dim):
    """Keys or values as they are held: codes of about unit values, and the blocks' scales, powers of two."""
    codes = (torch.randn(layers, pages, kv, page, dim, generator=gen, device="cuda", dtype=torch.bfloat16) * 64)
    q = torch.randint(-7, -4, (layers, pages, kv, page // BLOCK), generator=gen, device="cuda")
    return codes.clamp_(-448, 448).to(torch.float8_e4m3fn), torch.exp2(q.float())


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    cpu = torch.Generator()
    cpu.manual_seed(seed)
    s = {"case": case}
    op = case["op"]
    if op == "select":
        rows, vocab, beams = case["requests"] * case["beams"], case["vocab"], case["beams"]
        x = torch.randn(rows, vocab, generator=gen, device="cuda") * 2
        if case["masked"] != "none":
            # a third of the rows in free text, a third where nearly all is allowed, a third where a few tokens are
            kind = torch.randint(0, 3, (rows, 1), generator=gen, device="cuda")
            share = torch.tensor([2.0, 0.97, 0.002], device="cuda")[kind]
            x.masked_fill_(torch.rand(rows, vocab, generator=gen, device="cuda") >= share, float("-inf"))
        s["logits"] = x.to(TYPES[case["dtype"]])
        s["scores"] = -10.0 - 5.0 * torch.rand(case["requests"], beams, generator=gen, device="cuda")
        if case["first"]:
            s["scores"][:, 1:] = float("-inf")
            s["scores"][:, 0] = 0.0
        # what a beam carries: its tokens, and in some models a state
        s["states"] = [torch.randint(0, vocab, (rows, case["hist"]), generator=gen, device="cuda", dtype=torch.int32)]
        if case["extra"]:
            s["states"].append(torch.randn(rows, case["extra"], generator=gen, device="cuda").half())
        return s
    kv, dim, page = case["kv"], case["dim"], case["page"]
    if op == "append":
        rows, most, longest = case["rows"], case["tokens"], case["longest"]
        count = torch.tensor(_counts(case))
        off = torch.zeros(rows + 1, dtype=torch.int64)
        off[1:] = count.cumsum(0)
        start = torch.randint(0, longest + 1, (rows,), generator=cpu)
        width = -(-(longest + most) // page)
        pages = rows * width
        s["table"] = torch.randperm(pages, generator=cpu).view(rows, width).int().cuda()
        s["k"], s["k_scale"] = _pool(gen, 1, pages, kv, page, dim)
        s["v"], s["v_scale"] = _pool(gen, 1, pages, kv, page, dim)
        total = int(off[-1])
        # a few channels are much larger than the others, as keys' are
        wide = 1 + 7 * (torch.rand(kv, dim, generator=gen, device="cuda") < 0.03)
        s["new_k"] = (torch.randn(total, kv, dim, generator=gen, device="cuda") * wide).to(TYPES[case["dtype"]])
        s["new_v"] = torch.randn(total, kv, dim, generator=gen, device="cuda").to(TYPES[case["dtype"]])
        s["start"], s["off"] = start.int().cuda(), off.cuda()
        s["lens"] = (start + count).int().cuda()
        s["blocks"] = (most + 2 * BLOCK - 2) // BLOCK  # of a row, at most
    elif op == "attend":
        lens = _lens(case)
        rows, width = case["rows"], max(1, -(-case["longest"] // page))
        used = [-(-n // page) for n in lens]
        pages = max(1, sum(used))
        order = torch.randperm(pages, generator=cpu).int()
        table = torch.full((rows, width), -1, dtype=torch.int32)
        at = 0
        for r, n in enumerate(used):
            table[r, :n] = order[at:at + n]
            at += n
        s["table"], s["lens"] = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
        s["k"], s["k_scale"] = _pool(gen, 1, pages, kv, page, dim)
        s["v"], s["v_scale"] = _pool(gen, 1, pages, kv, page, dim)
        s["q"] = (torch.randn(rows * case["steps"], case["heads"], dim, generator=gen, device="cuda") * 2).to(
            TYPES[case["dtype"]])
    elif op == "branch":
        groups, beams, add = case["requests"], case["beams"], case["add"]
        rows = groups * beams
        n = torch.tensor(_lens({**case, "rows": groups}))
        width = -(-(case["longest"] + add) // page)
        used = -(-n // page)
        # the last two pages of a beam are its own (one of three shares them with the beam before it), the others
        # the request's; a third of the pool is free
        mine = torch.clamp(used, max=2)
        pages = int((used + beams * mine).sum()) * 3 // 2 + rows * 3
        order = torch.randperm(pages, generator=cpu).int()
        table = torch.full((rows, width), -1, dtype=torch.int32)
        at = 0
        like = torch.rand(rows, generator=cpu) < 1 / 3
        for g in range(groups):
            u, m = int(used[g]), int(mine[g])
            table[g * beams:(g + 1) * beams, :u - m] = order[at:at + u - m]
            at += u - m
            for r in range(g * beams, (g + 1) * beams):
                if r > g * beams and like[r]:
                    table[r, u - m:u] = table[r - 1, u - m:u]
                else:
                    table[r, u - m:u] = order[at:at + m]
                    at += m
        s["table"], s["lens"] = table.cuda(), n.repeat_interleave(beams).int().cuda()
        s["refs"] = torch.bincount(table[table >= 0].long(), minlength=pages).int().cuda()
        s["parents"] = torch.randint(0, beams, (groups, beams), generator=cpu).int().cuda()
        s["add"] = torch.full((rows,), add, dtype=torch.int32).cuda()
        s["k"], s["k_scale"] = _pool(gen, case["layers"], pages, kv, page, dim)
        s["v"], s["v_scale"] = _pool(gen, case["layers"], pages, kv, page, dim)
    else:
        rows, pages = case["rows"], case["pages"]
        live = max(1, int(pages * case["live"]))
        width = -(-live // rows)
        table = torch.full((rows * width,), -1, dtype=torch.int32)
        table[:live] = torch.randperm(pages, generator=cpu)[:live].int()
        table = table.view(rows, width)
        s["table"], s["lens"] = table.cuda(), ((table >= 0).sum(1) * page).int().cuda()
        s["refs"] = torch.bincount(table[table >= 0].long(), minlength=pages).int().cuda()
        s["k"], s["k_scale"] = _pool(gen, case["layers"], pages, kv, page, dim)
        s["v"], s["v_scale"] = _pool(gen, case["layers"], pages, kv, page, dim)
    if "refs" not in s:
        s["refs"] = torch.zeros(s["k"].shape[1], dtype=torch.int32, device="cuda")
        s["refs"][s["table"][s["table"] >= 0].long()] = 1
    if op in ("branch", "compact"):  # the state before the step
        s["before"] = {n: s[n].clone() for n in ("table", "lens", "refs")}
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["op"] != "select":
        import verbo_b200

        s["cache"] = verbo_b200.PagedCache(s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], s["lens"], s["refs"])
    return s


# -------------------------------------------------------------- one pass --
def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _restore(s):
    """A step changes the tables: each pass starts from the same ones."""
    for name, v in s["before"].items():
        s[name].copy_(v)


def _held(s):
    return s["k"], s["v"], s["k_scale"], s["v_scale"]


def _own_select(s):
    import verbo_b200

    c = s["case"]
    scores, parents, tokens = verbo_b200.beam_select(s["logits"], s["scores"], c["beams"], c["take"])
    verbo_b200.beam_reorder(s["states"], parents, c["beams"])
    return scores, parents, tokens, s["states"]


def _own_append(s):
    s["cache"].append(0, s["new_k"], s["new_v"], s["start"], off=s["off"] if s["case"]["ragged"] else None)
    return _held(s)


def _own_attend(s):
    return s["cache"].attend(0, s["q"], dtype=TYPES[s["case"]["out_dtype"]])


def _own_branch(s):
    _restore(s)
    s["cache"].fork(s["parents"], s["case"]["beams"])
    start, status = s["cache"].reserve(s["add"])
    return s["table"], s["lens"], s["refs"], start, status, _held(s)


def _own_compact(s):
    _restore(s)
    return s["cache"].compact(), s["table"], s["refs"], _held(s)


_own = {"select": _own_select, "append": _own_append, "attend": _own_attend, "branch": _own_branch,
        "compact": _own_compact}


def _plain_select(s):
    c = s["case"]
    n, beams, take, vocab = c["requests"], c["beams"], c["take"], c["vocab"]
    x = s["logits"].float()
    top = min(take, vocab)
    value, token = torch.sort(x, dim=1, descending=True, stable=True)
    value, token = value[:, :top].double(), token[:, :top]
    best = value[:, :1]
    # sums in 64 bits: the order of two beams' candidates goes by them
    lse = best + (x.double() - best).exp().sum(1, keepdim=True).log()
    score = s["scores"].double().view(-1, 1)
    total = torch.where(value > float("-inf"), score + (value - lse), float("-inf")).view(n, beams * top)
    total, at = torch.sort(total, dim=1, descending=True, stable=True)
    missing = max(0, take - beams * top)
    total = torch.nn.functional.pad(total[:, :take], (0, missing), value=float("-inf"))
    at = torch.nn.functional.pad(at[:, :take], (0, missing))
    none = total == float("-inf")
    parents = torch.where(none, -1, at // top).int()
    tokens = torch.where(none, -1, token.reshape(n, beams * top).gather(1, at)).int()
    row = torch.arange(n * beams, device="cuda").view(n, beams)
    if take >= beams:
        p = parents[:, :beams]
        row = torch.where(p < 0, row, row[:, :1] + p)
    for state in s["states"]:
        state.copy_(state[row.view(-1)])
    return total.float(), parents, tokens, s["states"]


def _plain_append(s):
    c = s["case"]
    page, rows = c["page"], c["rows"]
    start, off = s["start"].long(), s["off"]
    count = off[1:] - off[:-1]
    pos = (start // BLOCK * BLOCK)[:, None] + torch.arange(s["blocks"] * BLOCK, device="cuda")
    new = (pos >= start[:, None]) & (pos < (start + count)[:, None])
    old = (pos < start[:, None])
    block = new.view(rows, -1, BLOCK).any(2)  # blocks that get a token
    r, j = block.nonzero(as_tuple=True)
    pos, new, old = (t.view(rows, -1, BLOCK)[r, j] for t in (pos, new, old))  # [blocks, 16]
    at = s["table"][r, pos[:, 0] // page].long()  # the block's page
    inside = pos % page
    which = inside[:, 0] // BLOCK
    token = (off[:-1][r, None] + pos - start[r, None]).clamp(0, s["new_k"].shape[0] - 1)
    for x, held, scale in ((s["new_k"], s["k"][0], s["k_scale"][0]), (s["new_v"], s["v"][0], s["v_scale"][0])):
        x = x[token].float().transpose(1, 2)  # [blocks, heads, 16, dim]
        live = new[:, None, :, None]
        most = torch.where(live, x.abs(), 0.0).amax((2, 3))
        half, e = torch.frexp(most)
        need = torch.where(half > 0.875, e - 8, e - 9)
        need = torch.where(most > 0, need, LOWEST).clamp(min=LOWEST)
        need = torch.ldexp(torch.ones_like(most), need)
        had = scale[at, :, which]
        after = torch.where(old.any(1)[:, None], torch.maximum(had, need), need)
        bytes_ = held.view(torch.uint8)
        codes = bytes_[at[:, None], :, inside].transpose(1, 2)
        before = codes.contiguous().view(torch.float8_e4m3fn).float() * had[:, :, None, None]
        x = torch.where(live, x, before) / after[:, :, None, None]
        x = x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        x = torch.where((new | old)[:, None, :, None], x, codes)
        bytes_[at[:, None], :, inside] = x.transpose(1, 2)
        scale[at, :, which] = after
    return _held(s)


def _gathered(s, held, scale):
    """A layer's keys or values of all rows: [rows, heads, width * page, dim]."""
    t = s["table"].clamp(min=0).long()
    x = held.view(torch.uint8)[0][t].view(torch.float8_e4m3fn).float()
    x = x * scale[0][t].repeat_interleave(BLOCK, 3)[..., None]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attend(s):
    c = s["case"]
    rows, steps, kv, dim = c["rows"], c["steps"], c["kv"], c["dim"]
    group = c["heads"] // kv
    k, v = _gathered(s, s["k"], s["k_scale"]), _gathered(s, s["v"], s["v_scale"])
    q = s["q"].float().view(rows, steps, kv, group, dim).transpose(1, 2).reshape(rows, kv, steps * group, dim)
    x = q @ k.transpose(2, 3) * (1.0 / math.sqrt(dim))
    end = s["lens"].long()[:, None] - (steps - 1) + torch.arange(steps, device="cuda")  # [rows, steps]
    seen = torch.arange(x.shape[3], device="cuda") < end.repeat_interleave(group, 1)[:, None, :, None]
    x = torch.where(seen, x, float("-inf"))
    p = (x - x.amax(3, keepdim=True).clamp(min=-3e38)).exp()
    total = p.sum(3, keepdim=True)
    # pages behind a row's end hold what they hold
    v = torch.where(torch.arange(x.shape[3], device="cuda")[:, None] < s["lens"][:, None, None, None], v, 0.0)
    y = torch.where(total > 0, (p @ v) / total, 0.0)
    y = y.view(rows, kv, steps, group, dim).transpose(1, 2).reshape(rows * steps, kv * group, dim)
    return y.to(TYPES[c["out_dtype"]])


def _plain_branch(s):
    _restore(s)
    c = s["case"]
    page, groups, beams = c["page"], c["requests"], c["beams"]
    table, lens, refs, rows = s["table"], s["lens"], s["refs"], groups * beams
    width, pages = table.shape[1], refs.shape[0]
    # fork
    row = (torch.arange(groups, device="cuda")[:, None] * beams + s["parents"]).view(-1)
    forked = table[row]
    one = torch.ones(rows * width, dtype=torch.int32, device="cuda")
    for t, by in ((table, -1), (forked, 1)):
        refs.scatter_add_(0, t.view(-1).clamp(min=0).long(), by * one * (t.view(-1) >= 0))
    table.copy_(forked)
    lens.copy_(lens[row])
    # reserve
    n, add = lens.long(), s["add"].long()
    used = (n + page - 1) // page
    last = table.gather(1, (n // page).clamp(max=width - 1)[:, None])[:, 0].long()
    part = (add > 0) & (n % page > 0)
    same = (last[:, None] == last[None, :]) & part[:, None] & part[None, :]
    before = same.tril(-1).sum(1)  # rows before this one that write into the same page
    copy = part & (refs[last.clamp(min=0)] - before > 1)
    fresh = torch.where(add > 0, (n + add + page - 1) // page - used, 0)
    need = copy.long() + fresh
    upto = need.cumsum(0)
    free = refs == 0
    status = (upto[-1] - free.sum()).clamp(min=0)
    ok = status == 0
    ids = torch.argsort(free.int(), descending=True, stable=True)  # the lowest free page first
    first = upto - need
    copy = copy & ok
    src, dst = last[copy], ids[first[copy]]
    refs.scatter_add_(0, src, -torch.ones_like(src, dtype=torch.int32))
    table[copy, (n // page)[copy]] = dst.int()
    refs[dst] = 1
    for i in range(-(-c["add"] // page) + 1):
        r = ((fresh > i) & ok).nonzero()[:, 0]
        page_id = ids[first[r] + copy[r].long() + i]
        table[r, used[r] + i] = page_id.int()
        refs[page_id] = 1
    start = torch.where(ok & (add > 0), n, -1).int()
    lens.copy_(torch.where(ok, n + add, n))
    for held in _held(s):
        held = held.view(torch.uint8) if held.dtype == torch.float8_e4m3fn else held
        held[:, dst] = held[:, src]
    return table, lens, refs, start, status.int().view(1), _held(s)


def _plain_compact(s):
    _restore(s)
    table, refs = s["table"], s["refs"]
    pages = refs.shape[0]
    live = refs > 0
    n = live.sum()
    ids = torch.arange(pages, device="cuda")
    holes = (~live & (ids < n)).nonzero()[:, 0]
    moved = (live & (ids >= n)).nonzero()[:, 0].flip(0)  # the last live page goes into the first hole
    to = ids.clone()
    to[moved] = holes
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], -1))
    refs[holes] = refs[moved]
    refs[moved] = 0
    for held in _held(s):
        held = held.view(torch.uint8) if held.dtype == torch.float8_e4m3fn else held
        held[:, holes] = held[:, moved]
    info = torch.stack((n, torch.full_like(n, holes.shape[0]))).int()
    return info, table, refs, _held(s)


_plain = {"select": _plain_select, "append": _plain_append, "attend": _plain_attend, "branch": _plain_branch,
          "compact": _plain_compact}


# ------------------------------------------------------------------- work --
def work(case):
    op = case["op"]
    if op == "select":
        rows = case["requests"] * case["beams"]
        size = rows * case["vocab"] * SIZE[case["dtype"]] + 12 * case["requests"] * case["take"] + 4 * rows
        if case["take"] >= case["beams"]:
            size += 2 * rows * (4 * case["hist"] + 2 * case["extra"])
        return {"bytes": size, "flops": 4 * rows * case["vocab"]}
    token = 2 * case["kv"] * case["dim"]  # bytes of a token's keys and values
    if op == "append":
        total = sum(_counts(case))
        return {"bytes": total * token * (1 + SIZE[case["dtype"]]), "flops": 4 * total * token}
    if op == "attend":
        n = sum(_lens(case))
        rows = case["rows"] * case["steps"] * case["heads"] * case["dim"]
        size = n * token + n // BLOCK * case["kv"] * 8 + 4 * n // case["page"]
        return {"bytes": size + rows * (SIZE[case["dtype"]] + SIZE[case["out_dtype"]]),
                "flops": 4 * n * case["steps"] * case["heads"] * case["dim"]}
    held = case["layers"] * case["page"] * token + case["layers"] * case["kv"] * case["page"] // BLOCK * 8
    if op == "branch":
        beams = case["beams"]
        rows = case["requests"] * beams
        copies = case["requests"] * beams * (1 - 1 / beams) ** beams  # parents that two rows share, in the mean
        used = -(-(case["shortest"] + case["longest"]) // 2 // case["page"])
        return {"bytes": int(2 * copies * held + 8 * rows * used), "flops": rows * used}
    live = int(case["pages"] * case["live"])
    moved = live * (case["pages"] - live) // case["pages"]
    return {"bytes": 2 * moved * held + 8 * case["pages"] + 8 * live, "flops": case["pages"]}


# --------------------------------------------------------- in 64 bits -----
def exact(case, seed):
    if case["op"] in ("branch", "compact"):
        return None  # nothing is computed but whole numbers
    s = _inputs(case, seed)
    if case["op"] == "select":
        n, beams, take, vocab = case["requests"], case["beams"], case["take"], case["vocab"]
        total = torch.full((n, take), float("-inf"), dtype=torch.float64, device="cuda")
        parents = torch.full((n, take), -1, dtype=torch.int32, device="cuda")
        tokens = parents.clone()
        states = [t.clone() for t in s["states"]]
        for g in range(n):
            x = s["logits"][g * beams:(g + 1) * beams].double()
            y = (torch.log_softmax(x, 1) + s["scores"][g].double()[:, None]).view(-1)
            y = torch.where(x.view(-1) == float("-inf"), float("-inf"), y)
            limit = torch.topk(y, min(take, y.numel())).values[-1]
            at = (y >= limit).nonzero()[:, 0]
            at = at[torch.sort(y[at], descending=True, stable=True).indices][:take]
            at = at[y[at] > float("-inf")]
            m = at.numel()
            total[g, :m], parents[g, :m], tokens[g, :m] = y[at], (at // vocab).int(), (at % vocab).int()
            if take >= beams:
                for b, p in enumerate(parents[g, :beams].tolist()):
                    for new, old in zip(states, s["states"]):
                        if p >= 0:
                            new[g * beams + b] = old[g * beams + p]
        return total, parents, tokens, [t.double() if t.is_floating_point() else t for t in states]
    page = case["page"]
    if case["op"] == "append":
        grid = torch.arange(256, device="cuda").to(torch.uint8).view(torch.float8_e4m3fn).double()
        grid = grid[:127]  # 0, 2^-9, ... 448 in order
        out = [t[0].double() for t in _held(s)]
        start, off = s["start"].tolist(), s["off"].tolist()
        for r in range(case["rows"]):
            a, e = start[r], start[r] + off[r + 1] - off[r]
            if e == a:
                continue
            first = a // BLOCK * BLOCK
            pos = torch.arange(first, -(-e // BLOCK) * BLOCK, device="cuda").view(-1, BLOCK)
            pid = s["table"][r].long()[pos // page]
            inside = pos % page
            block, which = pid[:, 0], inside[:, 0] // BLOCK
            for new, held, scale in ((s["new_k"], out[0], out[2]), (s["new_v"], out[1], out[3])):
                had = scale[block, :, which]
                value = held[pid, :, inside] * had[:, None, :, None]  # [blocks, 16, heads, dim]
                if a > first:
                    value[0, a - first:] = 0
                else:
                    value[0] = 0
                value[1:] = 0
                fresh = torch.zeros_like(value).flatten(0, 1)
                fresh[a - first:e - first] = new[off[r]:off[r + 1]].double()
                fresh = fresh.view_as(value)
                most = fresh.abs().amax((1, 3))
                q = torch.ceil(torch.log2((most / 448).clamp(min=2.0 ** LOWEST)))
                q = torch.where(torch.exp2(q - 1) * 448 >= most, q - 1, q).clamp(min=LOWEST)
                now = torch.exp2(q)
                if a > first:
                    now[0] = torch.maximum(now[0], had[0])
                y = (value + fresh) / now[:, None, :, None]
                size = y.abs().clamp(max=448).contiguous()
                hi = torch.searchsorted(grid, size).clamp(max=126)
                lo = (hi - 1).clamp(min=0)
                near = size - grid[lo] < grid[hi] - size
                tie = size - grid[lo] == grid[hi] - size
                code = torch.where(near | (tie & (lo % 2 == 0)), lo, hi)
                y = torch.copysign(grid[code], y)
                inner = ((pos >= first) & (pos < e))[:, :, None, None]
                held[pid, :, inside] = torch.where(inner, y, held[pid, :, inside])
                scale[block, :, which] = now
        return [t[None] for t in out]
    # attend: one row and head of the cache after the other
    steps, kv, dim = case["steps"], case["kv"], case["dim"]
    group = case["heads"] // kv
    out = torch.zeros(case["rows"] * steps, case["heads"], dim, dtype=torch.float64, device="cuda")
    for r, n in enumerate(_lens(case)):
        if n == 0:
            continue
        pid = s["table"][r, :-(-n // page)].long()
        for h in range(kv):
            k, v = ((held[0].view(torch.uint8)[pid, h].view(torch.float8_e4m3fn).double().view(-1, BLOCK, dim)
                     * scale[0][pid, h].double().view(-1, 1, 1)).view(-1, dim)[:n]
                    for held, scale in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
            for i in range(steps):
                end = n - (steps - 1 - i)
                if end > 0:
                    q = s["q"][r * steps + i, h * group:(h + 1) * group].double()
                    w = torch.softmax(q @ k[:end].t() / math.sqrt(dim), 1)
                    out[r * steps + i, h * group:(h + 1) * group] = w @ v[:end]
    return out

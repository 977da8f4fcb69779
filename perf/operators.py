"""The operators that stand around the token sampler, as they are measured.

Three of them, in the order in which a decode step of a server runs them:

``q4``        products of a few hidden rows with 4-bit weights and group scales (the layers of a quantised model
              and its LM head): y = x W^T + b,  W[o, i] = s[o, g] (q[o, i] - z[o, g]),  g = i // group
``process``   what a request may do to its logits before the pick: penalties for repeated tokens, biases on
              single tokens, and a grammar's mask of allowed tokens
``logprobs``  what a server reports of a pick: the log-probability and the rank of the chosen token, and the most
              likely tokens with theirs

``run`` computes them in plain torch, or calls the library where ``own`` is true.
"""
import torch

own = False

VOCAB = 151936  # the vocabulary of the library's own workloads; 49152 is that of its single-row one
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------ cases --
def _process(name, rows, vocab, dtype, hist, last, bias, mask, penalties=True, per_row=False, inplace=False):
    return {"name": name, "op": "process", "rows": rows, "vocab": vocab, "dtype": dtype, "hist": hist, "last": last,
            "bias": bias, "mask": mask, "penalties": penalties, "per_row": per_row, "inplace": inplace}


def _q4(name, n, outs, ins, group, dtype, out_dtype, zeros, bias):
    return {"name": name, "op": "q4", "n": n, "outs": outs, "ins": ins, "group": group, "dtype": dtype,
            "out_dtype": out_dtype, "zeros": zeros, "bias": bias}


def _logprobs(name, rows, vocab, dtype, top, temp):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top, "temp": temp}


def listed():
    return [
        # one generation: a chat's window of 64 ids, a handful of biased tokens, a grammar
        _process("process-1", 1, 49152, "f32", 64, 64, 8, "mixed"),
        # a serving batch of bf16 logits, every request with its own history, biases and grammar
        _process("process-256-bf16", 256, VOCAB, "bf16", 200, 128, 24, "mixed"),
        # structured output alone: the grammar's mask written into the rows that the sampler reads
        _process("process-mask-64", 64, VOCAB, "f32", 0, 0, 0, "mixed", penalties=False, inplace=True),
        # the largest batch, each request with penalties of its own over long histories, no grammar
        _process("process-512-long", 512, VOCAB, "f32", 1024, 0, 0, "none", per_row=True),
        # one token through the LM head of the library's tail workload, hidden state and logits in fp32
        _q4("q4-head-1", 1, VOCAB, 896, 32, "f32", "f32", False, False),
        # one token through a square projection of a larger model, zero points of its own for each group
        _q4("q4-square-1", 1, 4096, 4096, 128, "bf16", "bf16", True, False),
        # three speculated tokens through a narrow down projection with a short last group
        _q4("q4-narrow-3", 3, 896, 4832, 128, "f16", "f16", False, True),
        # sixteen generations through a gate projection
        _q4("q4-gate-16", 16, 14336, 4096, 64, "bf16", "bf16", False, False),
        # sixty-four generations through the LM head
        _q4("q4-head-64", 64, VOCAB, 896, 32, "bf16", "f32", False, False),
        # one generation that reports its five most likely tokens
        _logprobs("logprobs-1", 1, 49152, "f32", 5, 0.7),
        # a serving batch that reports twenty each, from bf16 logits
        _logprobs("logprobs-256-bf16", 256, VOCAB, "bf16", 20, 1.0),
        # the largest batch, scored tokens only
        _logprobs("logprobs-512", 512, VOCAB, "f32", 0, 1.0),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(["process", "q4", "logprobs"])
    if op == "q4":
        group = rng.choice([32, 64, 128])
        while True:
            outs, ins = _spread(rng, 64, VOCAB), 32 * _spread(rng, 2, 512)
            if outs * ins <= VOCAB * 896:
                break
        dtype = rng.choice(["f32", "f16", "bf16"])
        out_dtype = rng.choice(["f32", dtype])
        c = _q4("", _spread(rng, 1, 64), outs, ins, group, dtype, out_dtype, rng.random() < 0.4, rng.random() < 0.4)
    else:
        vocab = _spread(rng, 1000, VOCAB)
        rows = _spread(rng, 1, min(512, 512 * VOCAB // vocab))
        dtype = rng.choice(["f32", "f16", "bf16"])
        if op == "process":
            inplace = rng.random() < 0.25
            hist = 0 if inplace or rng.random() < 0.2 else _spread(rng, 1, 1024)
            c = _process("", rows, vocab, "f32" if inplace else dtype, hist, rng.choice([0, 16, 64, 256]),
                         0 if inplace or rng.random() < 0.3 else _spread(rng, 1, 300),
                         "mixed" if inplace else rng.choice(["none", "mixed", "shared"]), penalties=hist > 0,
                         per_row=rng.random() < 0.5, inplace=inplace)
        else:
            c = _logprobs("", rows, vocab, dtype, rng.choice([0, 1, 5, 10, 20, 32]), round(0.4 + 1.2 * rng.random(), 2))
    del c["name"]
    return c


# ----------------------------------------------------------------- inputs --
def _lists(gen, rows, most, vocab):
    """Ragged lists of ids, about `most` a row and the first row's empty where there are several: frequent tokens are
    frequent, as in text."""
    lens = torch.randint(most // 2, most + 1, (rows,), generator=gen, device="cuda")
    lens[0] = 0 if rows > 1 else most
    lens[-1] = most
    off = torch.zeros(rows + 1, dtype=torch.int64, device="cuda")
    off[1:] = lens.cumsum(0)
    total = int(off[-1])
    ids = (float(vocab) ** torch.rand(total, generator=gen, device="cuda", dtype=torch.float64)).long() - 1
    return (ids * 7919 % vocab).int(), off


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "q4":
        outs, ins, group = case["outs"], case["ins"], case["group"]
        groups = -(-ins // group)
        s["x"] = torch.randn(case["n"], ins, generator=gen, device="cuda").to(TYPES[case["dtype"]])
        s["q"] = torch.randint(0, 256, (outs, ins // 2), generator=gen, device="cuda", dtype=torch.uint8)
        s["s"] = (torch.randn(outs, groups, generator=gen, device="cuda").abs() * 0.004 + 1e-4).half()
        s["zeros"] = s["b"] = None
        if case["zeros"]:
            s["zeros"] = torch.randint(5, 11, (outs, groups), generator=gen, device="cuda", dtype=torch.uint8)
        if case["bias"]:
            s["b"] = torch.randn(outs, generator=gen, device="cuda")
        return s
    rows, vocab = case["rows"], case["vocab"]
    s["logits"] = (torch.randn(rows, vocab, generator=gen, device="cuda") * 2).to(TYPES[case["dtype"]])
    if case["op"] == "logprobs":
        # half of the chosen tokens are among the likely ones, as a sampler's are
        some = torch.randint(0, vocab, (rows, 64), generator=gen, device="cuda")
        best = some.gather(1, s["logits"].gather(1, some).float().argmax(1, keepdim=True))[:, 0]
        s["ids"] = torch.where(torch.arange(rows, device="cuda") % 2 == 0, best, some[:, 0]).int()
        return s
    s["hist"] = s["hist_off"] = s["row"] = s["bias_ids"] = s["bias"] = s["bias_off"] = s["mask"] = None
    if case["hist"]:
        s["hist"], s["hist_off"] = _lists(gen, rows, case["hist"], vocab)
    one = torch.tensor([[1.1, 0.3, 0.2]], device="cuda")
    s["rates"] = one.expand(rows, 3).contiguous()
    if case["per_row"]:
        s["rates"] = s["row"] = one + torch.rand(rows, 3, generator=gen, device="cuda") * 0.4
    if case["bias"]:
        s["bias_ids"], s["bias_off"] = _lists(gen, rows, case["bias"], vocab)
        s["bias"] = torch.randn(s["bias_ids"].numel(), generator=gen, device="cuda") * 5
    if case["mask"] != "none":
        # a third of the rows in free text (all allowed), a third inside a string (nearly all), a third at a point
        # of the grammar that a few tokens alone can continue
        n = 1 if case["mask"] == "shared" else rows
        kind = torch.randint(0, 3, (n, 1), generator=gen, device="cuda")
        share = torch.tensor([2.0, 0.97, 0.002], device="cuda")[kind]
        bits = torch.rand(n, -(-vocab // 32) * 32, generator=gen, device="cuda") < share
        weight = torch.ones(32, dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")
        s["mask"] = (bits.view(n, -1, 32) * weight).sum(2).to(torch.int32)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["op"] == "q4":
        import verbo_b200

        s["layer"] = verbo_b200.Q4Linear(s["q"], s["s"], zeros=s["zeros"], bias=s["b"], group=case["group"])
    return s


# -------------------------------------------------------------- one pass --
def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _own_process(s):
    import verbo_b200

    c = s["case"]
    last = verbo_b200.Penalties(1.1, 0.3, 0.2, last=c["last"]) if c["penalties"] else None
    return verbo_b200.process_logits(s["logits"], last, hist=s["hist"], hist_off=s["hist_off"], row_penalties=s["row"],
                                     bias_ids=s["bias_ids"], bias=s["bias"], bias_off=s["bias_off"], mask=s["mask"],
                                     out=s["logits"] if c["inplace"] else None)


def _own_q4(s):
    return s["layer"].matvec(s["x"], dtype=TYPES[s["case"]["out_dtype"]])


def _own_logprobs(s):
    import verbo_b200

    return verbo_b200.token_logprobs(s["logits"], s["ids"], top=s["case"]["top"], temp=s["case"]["temp"])


_own = {"process": _own_process, "q4": _own_q4, "logprobs": _own_logprobs}


def _plain_process(s):
    c = s["case"]
    rows, vocab = s["logits"].shape
    x = s["logits"].float()
    if c["hist"]:
        off = s["hist_off"]
        row = torch.repeat_interleave(torch.arange(rows, device="cuda"), off[1:] - off[:-1], output_size=s["hist"].numel())
        first = off[:-1] if c["last"] <= 0 else torch.maximum(off[:-1], off[1:] - c["last"])
        inside = torch.arange(s["hist"].numel(), device="cuda") >= first[row]
        count = torch.zeros(rows * vocab, dtype=torch.int32, device="cuda")
        count = count.scatter_add(0, row * vocab + s["hist"], inside.int()).view(rows, vocab)
        repeat, frequency, presence = (s["rates"][:, i:i + 1] for i in range(3))
        seen = count > 0
        x = torch.where(seen, torch.where(x > 0, x / repeat, x * repeat), x)
        x = x - frequency * count
        x = x - presence * seen
    if c["bias"]:
        off = s["bias_off"]
        n = s["bias"].numel()
        row = torch.repeat_interleave(torch.arange(rows, device="cuda"), off[1:] - off[:-1], output_size=n)
        # an id listed twice in a row has the bias that is listed last
        at = torch.full((rows * vocab,), -1, device="cuda")
        at = at.scatter_reduce(0, row * vocab + s["bias_ids"], torch.arange(n, device="cuda"), "amax")
        x = x + torch.where(at >= 0, s["bias"][at], 0.0).view(rows, vocab)
    if c["mask"] != "none":
        bits = (s["mask"].unsqueeze(2) >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        allowed = bits.view(bits.shape[0], -1)[:, :vocab] != 0
        x = torch.where(allowed, x, float("-inf"))
    return s["logits"].copy_(x) if c["inplace"] else x


def _plain_q4(s):
    c = s["case"]
    outs, ins = c["outs"], c["ins"]
    # a block of 32 weights is 16 bytes: the first 16 weights in their low halves, the others in the high ones
    q = s["q"].view(outs, ins // 32, 1, 16)
    w = torch.cat((q & 15, q >> 4), 2).view(outs, ins).float()
    group = torch.arange(ins, device="cuda") // c["group"]
    w = w - (8.0 if s["zeros"] is None else s["zeros"].float()[:, group])
    w = w * s["s"].float()[:, group]
    y = s["x"].float() @ w.t()
    if s["b"] is not None:
        y = y + s["b"]
    return y.to(TYPES[c["out_dtype"]])


def _plain_logprobs(s):
    top, temp = s["case"]["top"], s["case"]["temp"]
    x = s["logits"].float() + 0.0
    best = x.max(1, keepdim=True).values
    d = (x - best) / torch.full_like(best, temp)
    lp = d - d.exp().sum(1, keepdim=True).log()
    id = s["ids"].long()[:, None]
    mine = x.gather(1, id)
    column = torch.arange(x.shape[1], device="cuda")
    rank = ((x > mine) | ((x == mine) & (column < id))).sum(1).int()
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top] if top else id[:, :0]
    return lp.gather(1, id)[:, 0], rank, order.int(), lp.gather(1, order)


_plain = {"process": _plain_process, "q4": _plain_q4, "logprobs": _plain_logprobs}


# ------------------------------------------------------------------- work --
def work(case):
    if case["op"] == "q4":
        n, outs, ins = case["n"], case["outs"], case["ins"]
        groups = -(-ins // case["group"])
        size = outs * ins // 2 + outs * groups * (3 if case["zeros"] else 2) + (4 * outs if case["bias"] else 0)
        return {"bytes": size + n * ins * SIZE[case["dtype"]] + n * outs * SIZE[case["out_dtype"]],
                "flops": 2 * n * outs * ins}
    rows, vocab = case["rows"], case["vocab"]
    row = vocab * SIZE[case["dtype"]]
    if case["op"] == "logprobs":
        return {"bytes": rows * (row + 12 + 8 * case["top"]), "flops": 4 * rows * vocab}
    size = 0 if case["mask"] == "none" else (1 if case["mask"] == "shared" else rows) * 4 * -(-vocab // 32)
    size += rows * (4 * case["hist"] * 3 // 4 + 8 * case["bias"] * 3 // 4)
    if case["inplace"]:  # the mask is read, and a third of the rows' columns (and 3 in a hundred of another) written
        return {"bytes": size + rows * vocab * 4 * 343 // 1000, "flops": rows * vocab}
    return {"bytes": size + rows * (row + 4 * vocab), "flops": rows * vocab}


# --------------------------------------------------------- in 64 bits -----
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "q4":
        x, outs = s["x"].double(), case["outs"]
        y = torch.zeros(case["n"], outs, dtype=torch.float64, device="cuda")
        for g in range(s["s"].shape[1]):
            first, last = g * case["group"], min(case["ins"], (g + 1) * case["group"])
            z = 8.0 if s["zeros"] is None else s["zeros"][:, g:g + 1].double()
            part = torch.zeros_like(y)
            for b in range(first // 32, last // 32):
                byte = s["q"][:, 16 * b:16 * b + 16]
                part += x[:, 32 * b:32 * b + 16] @ (byte % 16 - z).double().t()
                part += x[:, 32 * b + 16:32 * b + 32] @ (byte // 16 - z).double().t()
            y += part * s["s"][:, g].double()
        return y if s["b"] is None else y + s["b"].double()
    rows, vocab = case["rows"], case["vocab"]
    x = s["logits"].double()
    if case["op"] == "logprobs":
        t = float(torch.tensor(case["temp"], dtype=torch.float32))
        z = x / t
        lse = torch.logsumexp(z, 1, keepdim=True)
        id = s["ids"].long()[:, None]
        # order by value, then by the lower index: sorted ascending by both at once, from the end
        bits = s["logits"].float().add(0.0).view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * 262144 + (262143 - torch.arange(vocab, device="cuda"))
        rank = (key > key.gather(1, id)).sum(1).int()
        order = torch.topk(key, case["top"], 1).indices if case["top"] else id[:, :0]
        return (z.gather(1, id) - lse)[:, 0], rank, order.int(), z.gather(1, order) - lse
    flat = x.view(-1)
    if case["hist"]:
        h, off = s["hist"].cpu(), s["hist_off"].cpu().tolist()
        for r in range(rows):
            ids = h[off[r]:off[r + 1]]
            ids = ids[-case["last"]:] if case["last"] > 0 else ids
            ids, count = (v.cuda() for v in torch.unique(ids.long(), return_counts=True))
            rep, freq, pres = s["rates"][r].double()
            v = x[r, ids]
            x[r, ids] = torch.where(v > 0, v / rep, v * rep) - freq * count - pres
    if case["bias"]:
        off = s["bias_off"].cpu().tolist()
        place, value = [], []
        ids, bias = s["bias_ids"].cpu().tolist(), s["bias"].cpu().tolist()
        for r in range(rows):
            last = dict(zip(ids[off[r]:off[r + 1]], bias[off[r]:off[r + 1]]))
            place += [r * vocab + i for i in last]
            value += last.values()
        flat[torch.tensor(place, dtype=torch.int64, device="cuda")] += torch.tensor(value, dtype=torch.float64, device="cuda")
    if case["mask"] != "none":
        column = torch.arange(vocab, device="cuda")
        word = s["mask"].long()[:, column // 32] % 4294967296
        x.masked_fill_((word // (1 << (column % 32))) % 2 == 0, float("-inf"))
    return x

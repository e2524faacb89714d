"""Rotary positions, a paged cache of keys and values, and the attention that reads it: what is measured of them.

  rotary  ``nn.RotaryEmbedding``: queries and keys turned by their positions, forward or forward and backward
  append  ``nn.KVCache.Append``: new keys (turned) and values written to their sequences' pages, the queries turned on the way
  attend  ``nn.KVCache.Attend``: new tokens over the keys and values of their sequences
  shared  the same for sequences whose first pages are the same ones

Rotation of a pair (a, b) of a head at position p: (a cos - b sin, a sin + b cos) * amplitude with the angle p w_i.  Pairs are
(i, i + dim / 2) or, interleaved, (2 i, 2 i + 1), i < dim / 2; columns from dim on are left alone.  w_i = base^(-2 i / dim), for longer
contexts than a model was trained on
  linear  w_i / factor
  base    base replaced by base * factor^(dim / (dim - 2))
  bands   w_i (g + (1 - g) / factor), g = (original w_i / 2 pi - low) / (high - low), kept within 0 and 1

A cache is two tensors (pages, heads, page size, head size).  Position p of sequence b lies in row p % page size of page
table[b, p // page size].  lengths[b] positions are there before a call; its token t < counts[b] takes position lengths[b] + t, whose
query sees the positions up to its own.  Results of the tokens from counts[b] on are zeros; nothing of them is written to a cache.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
PLAIN = {"interleaved": False, "base": 10000.0, "scaling": "none", "factor": 1.0, "original": 0, "low": 1.0, "high": 32.0, "amplitude": 1.0}


def listed():
    return [
        # one new token of the 1.3 B model: queries and keys of 16 heads each
        {"name": "rotary, one token", "op": "rotary", "dtype": "bf16", "batch": 1, "tokens": 1, "heads": 32, "width": 128, "dim": 128,
         "start": 1531, "grad": False, **PLAIN},
        # the training batch of the 12-layer model, queries and keys of 12 heads each, forward and backward
        {"name": "rotary, 16 x 1024 tokens", "op": "rotary", "dtype": "bf16", "batch": 16, "tokens": 1024, "heads": 24, "width": 64, "dim": 64,
         "start": 0, "grad": True, **PLAIN},
        # fp32, pairs side by side, part of each head, far positions of a context that was made longer
        {"name": "rotary, ragged fp32", "op": "rotary", "dtype": "f32", "batch": 3, "tokens": 1531, "heads": 7, "width": 80, "dim": 52,
         "start": 100003, "grad": True, **PLAIN, "interleaved": True, "scaling": "bands", "factor": 8.0, "original": 4096, "amplitude": 1.2},
        # one new token of the 1.3 B model behind 1000 others
        {"name": "append, one token", "op": "append", "dtype": "bf16", "batch": 1, "tokens": 1, "heads": 16, "kv": 16, "width": 128, "dim": 128,
         "length": 1000, "page": 64, "padded": False, **PLAIN},
        # four prompts of the 1.3 B model's full length
        {"name": "append, 4 x 2048 tokens", "op": "append", "dtype": "bf16", "batch": 4, "tokens": 2048, "heads": 16, "kv": 16, "width": 128,
         "dim": 128, "length": 0, "page": 64, "padded": False, **PLAIN},
        # a padded batch of short pieces, four heads to a key, odd pages
        {"name": "append, ragged fp16", "op": "append", "dtype": "f16", "batch": 37, "tokens": 13, "heads": 12, "kv": 3, "width": 72, "dim": 40,
         "length": 1531, "page": 24, "padded": True, **PLAIN, "interleaved": True, "scaling": "linear", "factor": 4.0},
        # one sequence of the 1.3 B model's full length, one new token
        {"name": "attend, one token", "op": "attend", "dtype": "bf16", "batch": 1, "tokens": 1, "heads": 16, "kv": 16, "width": 128,
         "length": 2047, "page": 64, "padded": False},
        # a server's batch of long sequences, four heads to a key: the cache's bytes are what counts
        {"name": "attend, 64 sequences", "op": "attend", "dtype": "bf16", "batch": 64, "tokens": 1, "heads": 32, "kv": 8, "width": 128,
         "length": 32768, "page": 64, "padded": False},
        # several proposed tokens at once for a padded batch, odd pages
        {"name": "attend, 5 tokens ragged fp16", "op": "attend", "dtype": "f16", "batch": 13, "tokens": 5, "heads": 12, "kv": 4, "width": 64,
         "length": 5003, "page": 24, "padded": True},
        # the second half of four long prompts, behind the first one: the products count
        {"name": "attend, 4 x 2048 tokens", "op": "attend", "dtype": "bf16", "batch": 4, "tokens": 2048, "heads": 16, "kv": 16, "width": 128,
         "length": 2048, "page": 64, "padded": False},
        # 16 answers of the 1.3 B model to one prompt
        {"name": "shared, 16 answers", "op": "shared", "dtype": "bf16", "batch": 16, "tokens": 1, "heads": 16, "kv": 16, "width": 128,
         "prefix": 1920, "length": 128, "page": 64, "padded": False},
        # 256 sequences behind one long document, four heads to a key
        {"name": "shared, 256 sequences", "op": "shared", "dtype": "bf16", "batch": 256, "tokens": 1, "heads": 32, "kv": 8, "width": 128,
         "prefix": 16384, "length": 512, "page": 64, "padded": False},
    ]


def draw(rng):
    def size(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    op = rng.choice(["rotary", "append", "attend", "shared"])
    case = {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"] if op != "shared" else ["bf16", "f16"])}
    if op in ("rotary", "append"):
        case["width"] = 8 * rng.randint(2, 16)
        case["dim"] = rng.choice([case["width"], 2 * rng.randint(4, case["width"] // 2)])
        case |= PLAIN
        case["interleaved"] = rng.random() < 0.5
        case["base"] = rng.choice([10000.0, 500000.0])
        case["scaling"] = rng.choice(["none", "linear", "base", "bands"])
        if case["scaling"] != "none":
            case |= {"factor": rng.choice([2.0, 4.0, 8.0, 32.0]), "original": 8192, "amplitude": rng.choice([1.0, 1.25])}
    if op == "rotary":
        case["heads"] = rng.randint(1, 48)
        rows = size(1, 2 ** 24 // (case["heads"] * case["width"]))
        case["batch"] = size(1, min(rows, 64))
        case["tokens"] = max(1, rows // case["batch"])
        return case | {"start": rng.choice([0, size(1, 200000)]), "grad": rng.random() < 0.5}
    case["kv"] = rng.choice([1, 2, 3, 4, 8, 12, 16])
    case["heads"] = case["kv"] * rng.choice([1, 1, 2, 3, 4, 8])
    case["page"] = rng.choice([16, 32, 64, 128, 24, 40, rng.randint(1, 200)])
    case["padded"] = rng.random() < 0.3
    if op == "append":
        rows = size(1, 2 ** 24 // ((case["heads"] + 2 * case["kv"]) * case["width"]))
        case["batch"] = size(1, min(rows, 256))
        case["tokens"] = max(1, rows // case["batch"])
        case["length"] = rng.choice([0, size(1, max(1, 2 ** 26 // (case["batch"] * case["kv"] * case["width"])))])
        return case
    case["width"] = rng.choice([64, 128, 128, 8 * rng.randint(2, 16)])
    if op == "attend":
        case["batch"] = size(1, 128)
        case["length"] = size(1, min(65536, 2 ** 29 // (case["batch"] * case["kv"] * case["width"])))
        case["tokens"] = rng.choice([1, 1, rng.randint(2, 16), size(16, 1024)])
        limit = 2 ** 36 if case["dtype"] != "f32" else 2 ** 33        # products: at most those of the prompts, or their fp32 share
        while case["tokens"] > 1 and case["batch"] * case["heads"] * case["width"] * case["tokens"] * (case["length"] + case["tokens"]) > limit:
            case["tokens"] //= 2
        return case
    case["batch"] = size(2, 384)
    case["tokens"] = rng.choice([1, 1, 1, rng.randint(2, 4)])
    case["length"] = size(1, 512)
    most = min(16384, 2 ** 34 // (case["batch"] * case["heads"] * case["width"] * case["tokens"]))
    case["prefix"] = case["page"] * max(1, size(1, max(1, most // case["page"])))
    return case


def _lengths(case):
    """Positions in the cache before the call, and new tokens, of each sequence.  One sequence has the case's own numbers."""
    rng = random.Random(case["batch"] * 1000003 + case["length"])
    lengths, counts = [], []
    for b in range(case["batch"]):
        lengths.append(case.get("prefix", 0) + (case["length"] if b == 0 else rng.randint(case["length"] // 8, case["length"])))
        counts.append(rng.randint(0, case["tokens"]) if case["padded"] and b else case["tokens"])
    return lengths, counts


def work(case):
    size = TYPES[case["dtype"]].itemsize
    if case["op"] == "rotary":          # read and written, both again for the gradient
        n = case["batch"] * case["tokens"] * case["heads"] * case["width"]
        return {"bytes": 2 * n * size * (2 if case["grad"] else 1), "flops": 3 * n * (2 if case["grad"] else 1)}
    lengths, counts = _lengths(case)
    new, width, heads, kv = sum(counts), case["width"], case["heads"], case["kv"]
    if case["op"] == "append":          # queries, keys and values read and written
        return {"bytes": 2 * new * (heads + 2 * kv) * width * size, "flops": 3 * new * (heads + kv) * width}
    prefix = case.get("prefix", 0)
    rows = prefix + sum(n + c - prefix for n, c in zip(lengths, counts) if c)               # each key and value once
    pairs = sum(c * n + c * (c + 1) // 2 for n, c in zip(lengths, counts))
    return {"bytes": (2 * rows * kv + (new + case["batch"] * case["tokens"]) * heads) * width * size, "flops": 4 * pairs * heads * width}


# ---------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dtype, batch, tokens, width = TYPES[case["dtype"]], case["batch"], case["tokens"], case["width"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    if case["op"] == "rotary":
        x = normal(batch, tokens, case["heads"], width)
        at = torch.arange(tokens, device="cuda") + case["start"]
        at = at if case["start"] == 0 else at + 17 * torch.arange(batch, device="cuda")[:, None]     # every sequence at its own place
        return {"x": x, "positions": at, "dy": normal(*x.shape) if case["grad"] else None}
    lengths, counts = _lengths(case)
    page, kv = case["page"], case["kv"]
    prefix = case.get("prefix", 0) // page                                                          # whole pages
    needs = [-(-(n + tokens) // page) for n in lengths]
    total = prefix + sum(n - prefix for n in needs)
    order = torch.randperm(total + 3, generator=g, device="cuda").to(torch.int32).cpu()             # pages lie in any order; some are free
    table = torch.zeros(batch, max(needs), dtype=torch.int32)
    used = prefix
    for b, n in enumerate(needs):
        table[b, :prefix] = order[:prefix]
        table[b, prefix:n] = order[used:used + n - prefix]
        used += n - prefix
    made = {"k_cache": normal(total + 3, kv, page, width), "v_cache": normal(total + 3, kv, page, width), "table": table.cuda(),
            "lengths": torch.tensor(lengths, dtype=torch.int32).cuda(),
            "counts": torch.tensor(counts, dtype=torch.int32).cuda() if case["padded"] else None}
    # scores of trained heads differ by several units
    made["q"] = 2 * normal(batch, tokens, case["heads"], width)
    if case["op"] == "append":
        made |= {"k": normal(batch, tokens, kv, width), "v": normal(batch, tokens, kv, width)}
    return made


def prepare(case, seed):
    state = dict(case, **_inputs(case, seed), type=TYPES[case["dtype"]])
    if own:
        from gonn_b200 import nn

        if "dim" in case:
            state["rope"] = nn.RotaryEmbedding(case["dim"], case["base"], interleaved=case["interleaved"], scaling=case["scaling"],
                                               factor=case["factor"], original=case["original"], low=case["low"], high=case["high"],
                                               amplitude=case["amplitude"], device="cuda")
        if "k_cache" in state:
            state["cache"] = nn.KVCache.Over(state["k_cache"], state["v_cache"])
    return state


# ---------------------------------------------------------------------------------------------------------------------------
# a pass
# ---------------------------------------------------------------------------------------------------------------------------
def _turned(x, positions, s, sign=1.0):
    """x (batch, tokens, heads, width) turned, in 32 bits; angles in 64."""
    dim, base = s["dim"], s["base"]
    if s["scaling"] == "base":
        base = base * s["factor"] ** (dim / (dim - 2))
    w = base ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=x.device) / dim)
    if s["scaling"] == "linear":
        w = w / s["factor"]
    elif s["scaling"] == "bands":
        g = ((s["original"] * w / (2 * math.pi) - s["low"]) / (s["high"] - s["low"])).clamp(0, 1)
        w = w * (g + (1 - g) / s["factor"])
    angle = positions.double().unsqueeze(-1) * w
    cos = (torch.cos(angle) * s["amplitude"]).float().unsqueeze(-2)
    sin = (torch.sin(angle) * s["amplitude"] * sign).float().unsqueeze(-2)
    y = x.float().clone()
    first = slice(0, dim, 2) if s["interleaved"] else slice(0, dim // 2)
    second = slice(1, dim, 2) if s["interleaved"] else slice(dim // 2, dim)
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first] = a * cos - b * sin
    y[..., second] = a * sin + b * cos
    return y


def _plain(s):
    dtype, op = s["type"], s["op"]
    if op == "rotary":
        y = _turned(s["x"], s["positions"], s).to(dtype)
        return (y, _turned(s["dy"], s["positions"], s, -1.0).to(dtype)) if s["grad"] else y
    q, table, lengths, page = s["q"], s["table"].long(), s["lengths"].long(), s["page"]
    batch, tokens, heads, width = q.shape
    counts = torch.full_like(lengths, tokens) if s["counts"] is None else s["counts"].long()
    step = torch.arange(tokens, device=q.device)
    positions = lengths[:, None] + step
    valid = step < counts[:, None]
    if op == "append":
        q = _turned(q, positions, s) * valid[..., None, None]
        k, v, at = _turned(s["k"], positions, s)[valid], s["v"][valid], positions[valid]
        pages = table.gather(1, positions.div(page, rounding_mode="floor"))[valid]
        s["k_cache"][pages, :, at % page] = k.to(dtype)
        s["v_cache"][pages, :, at % page] = v
        return q.to(dtype), s["k_cache"], s["v_cache"]
    out = torch.zeros(batch, tokens, heads, width, device=q.device)
    kv = s["kv"]
    for b, (n, c) in enumerate(zip(*_lengths(s))):
        if c == 0:
            continue
        used = table[b, : -(-(n + c) // page)]
        k = s["k_cache"][used].float().transpose(0, 1).reshape(kv, -1, width)[:, : n + c]
        v = s["v_cache"][used].float().transpose(0, 1).reshape(kv, -1, width)[:, : n + c]
        rows = q[b, :c].float().view(c, kv, heads // kv, width).permute(1, 2, 0, 3)         # key head, its queries' heads, tokens
        scores = rows.reshape(kv, -1, width) @ k.transpose(1, 2) / math.sqrt(width)
        unseen = torch.arange(n + c, device=q.device) > n + step[:c, None]
        scores = scores.view(kv, heads // kv, c, n + c).masked_fill(unseen, -math.inf)
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        p = (p / p.sum(-1, keepdim=True)).view(kv, -1, n + c)
        out[b, :c] = (p @ v).view(kv, heads // kv, c, width).permute(2, 0, 1, 3).reshape(c, heads, width)
    return out.to(dtype)


def _own(s):
    op = s["op"]
    if op == "rotary":
        if not s["grad"]:
            return s["rope"](s["x"], s["positions"])
        x = s["x"].detach().requires_grad_()
        y = s["rope"](x, s["positions"])
        return y.detach(), torch.autograd.grad(y, x, s["dy"])[0]
    if op == "append":
        q = s["cache"].Append(s["k"], s["v"], s["table"], s["lengths"], counts=s["counts"], rotary=s["rope"], q=s["q"])
        return q, s["k_cache"], s["v_cache"]
    return s["cache"].Attend(s["q"], s["table"], s["lengths"], counts=s["counts"], shared_pages=s.get("prefix", 0) // s["page"])


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------------
def _rotation(x, positions, case, back=False):
    """Pairs as complex numbers times amplitude * exp(i p w)."""
    dim, half = case["dim"], case["dim"] // 2
    w = []
    for i in range(half):
        base = case["base"] * (case["factor"] ** (dim / (dim - 2)) if case["scaling"] == "base" else 1.0)
        f = math.exp(-2 * i / dim * math.log(base))
        if case["scaling"] == "linear":
            f /= case["factor"]
        if case["scaling"] == "bands":
            g = min(1.0, max(0.0, (case["original"] * f / (2 * math.pi) - case["low"]) / (case["high"] - case["low"])))
            f = g * f + (1 - g) * f / case["factor"]
        w.append(f)
    angle = positions.to(torch.float64)[..., None, None] * torch.tensor(w, dtype=torch.float64, device=x.device)
    turn = torch.polar(torch.full_like(angle, case["amplitude"]), -angle if back else angle)
    part = x[..., :dim].double()
    part = part.unflatten(-1, (half, 2)) if case["interleaved"] else part.unflatten(-1, (2, half)).transpose(-1, -2)
    part = torch.view_as_real(torch.view_as_complex(part.contiguous()) * turn)
    part = part.flatten(-2) if case["interleaved"] else part.transpose(-1, -2).flatten(-2)
    return torch.cat((part, x[..., dim:].double()), -1)


def exact(case, seed):
    made = _inputs(case, seed)
    if case["op"] == "rotary":
        y = _rotation(made["x"], made["positions"], case)
        return (y, _rotation(made["dy"], made["positions"], case, back=True)) if case["grad"] else y
    lengths, counts = _lengths(case)
    table, page, q = made["table"].tolist(), case["page"], made["q"]
    if case["op"] == "append":
        k_cache, v_cache, rotated = made["k_cache"].double(), made["v_cache"].double(), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        for b, (n, c) in enumerate(zip(lengths, counts)):
            at = torch.arange(n, n + c, device=q.device)
            rotated[b, :c] = _rotation(q[b, :c], at, case)
            k = _rotation(made["k"][b, :c], at, case)
            t = 0
            while t < c:                                                                   # page by page
                row = (n + t) % page
                more = min(c - t, page - row)
                where = table[b][(n + t) // page]
                k_cache[where, :, row:row + more] = k[t:t + more].transpose(0, 1)
                v_cache[where, :, row:row + more] = made["v"][b, t:t + more].double().transpose(0, 1)
                t += more
        return rotated, k_cache, v_cache
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    group, width = case["heads"] // case["kv"], case["width"]
    for b, (n, c) in enumerate(zip(lengths, counts)):
        pages = made["table"][b].long()
        for h in range(case["kv"]):
            if c == 0:
                continue
            k = made["k_cache"][pages, h].flatten(0, 1)[: n + c].double()
            v = made["v_cache"][pages, h].flatten(0, 1)[: n + c].double()
            scores = torch.einsum("tgd,nd->gtn", q[b, :c, h * group:(h + 1) * group].double(), k) * width ** -0.5
            scores += torch.full((c, n + c), -math.inf, dtype=torch.float64, device=q.device).triu(n + 1)
            out[b, :c, h * group:(h + 1) * group] = torch.einsum("gtn,nd->tgd", torch.softmax(scores, -1), v)
    return out

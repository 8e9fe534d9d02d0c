"""Measured cases of the decode-side operators: the W4A16 linear, attention of one new token over a paged key-value
cache, branching of cached sequences (free, fork, copy on write, append) and compaction of the page pool.

``run`` computes a case in plain torch operations where ``own`` is false and through the package's operators where it
is true; ``exact`` gives the same outputs from the definitions in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp8": torch.float8_e4m3fn}
_SIZE = {"bf16": 2, "f16": 2, "fp8": 1}
_FP8_MAX = 448.0


def _linear(name, m, k, n, group, dtype, bias):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "group": group, "dtype": dtype, "bias": bias}


def _attention(name, batch, q_heads, kv_heads, dim, page, longest, spread, window, sinks, dtype, cache):
    return {"name": name, "op": "attention", "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "longest": longest, "spread": spread, "window": window, "sinks": sinks, "dtype": dtype,
            "cache": cache}


def _branch(name, prompts, rows, longest, layers, kv_heads, page, dim, dtype):
    return {"name": name, "op": "branch", "prompts": prompts, "rows": rows, "longest": longest, "layers": layers,
            "kv_heads": kv_heads, "page": page, "dim": dim, "dtype": dtype}


def _compact(name, rows, longest, layers, kv_heads, page, dim, dtype, fill):
    return {"name": name, "op": "compact", "rows": rows, "longest": longest, "layers": layers, "kv_heads": kv_heads,
            "page": page, "dim": dim, "dtype": dtype, "fill": fill}


def listed():
    return [
        # one token through a small projection with an odd number of outputs: latency
        _linear("linear_one_small", 1, 1024, 1001, 64, "bf16", True),
        # one token through a feed-forward projection, the ordinary decode call
        _linear("linear_one", 1, 4096, 16384, 128, "bf16", False),
        # a batch of eighteen sequences, fine groups, half precision
        _linear("linear_batch", 18, 5120, 13824, 32, "f16", True),
        # the largest call: a full batch through the widest projection
        _linear("linear_wide", 64, 8192, 28672, 128, "bf16", False),
        # one short conversation: latency
        _attention("attention_one_short", 1, 16, 2, 128, 16, 333, 0.0, 0, 0, "bf16", "bf16"),
        # a ragged batch as a server holds it, among them an empty row and a row of one token
        _attention("attention_ragged", 64, 32, 8, 128, 16, 8000, 1.0, 0, 0, "bf16", "bf16"),
        # two very long contexts, few heads: the length has to be split
        _attention("attention_long", 2, 28, 4, 128, 64, 200001, 0.1, 0, 0, "f16", "f16"),
        # a sliding-window layer with first tokens that stay, wide heads, an 8-bit cache
        _attention("attention_window_fp8", 48, 16, 8, 256, 32, 16000, 1.0, 1024, 4, "bf16", "fp8"),
        # four samples of one prompt in a small cache
        _branch("branch_small", 1, 4, 100, 4, 2, 16, 64, "f16"),
        # resampling 128 rows of 16 prompts, all layers of a deep model
        _branch("branch_deep", 16, 128, 900, 32, 8, 16, 128, "bf16"),
        # a small pool after a few requests have left
        _compact("compact_small", 5, 60, 2, 2, 16, 64, "f16", 0.5),
        # a large pool, half of it free
        _compact("compact_deep", 24, 700, 32, 8, 16, 128, "bf16", 0.5),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "attention", "attention", "attention", "branch", "compact"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "linear":
        group = rng.choice([32, 64, 128])
        k = max(1, _spread(rng, 512, 8192) // group) * group
        case = _linear("", _spread(rng, 1, 64), k, _spread(rng, 200, 28672), group, dtype, rng.random() < 0.5)
    elif op == "attention":
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        dim = rng.choice([64, 128, 256])
        cache = rng.choice([dtype, dtype, "fp8"])
        batch = _spread(rng, 1, 96)
        # the whole cache stays below that of the largest listed case
        longest = _spread(rng, 1, max(2, min(200000, 160_000_000 // (batch * kv_heads * dim))))
        windowed = rng.random() < 0.4
        case = _attention("", batch, kv_heads * rng.choice([1, 2, 4, 5, 7, 8, 12, 16]), kv_heads, dim,
                          rng.choice([16, 32, 64, 128]), longest, rng.choice([0.0, 0.5, 1.0]),
                          _spread(rng, 1, 4096) if windowed else 0, rng.choice([0, 1, 4, 17]) if windowed else 0,
                          dtype, cache)
    elif op == "branch":
        prompts = _spread(rng, 1, 16)
        case = _branch("", prompts, prompts * rng.randint(1, 8), _spread(rng, 1, 900), rng.randint(1, 32),
                       rng.choice([1, 2, 4, 8]), rng.choice([16, 32]), rng.choice([64, 128]), dtype)
    else:
        case = _compact("", _spread(rng, 1, 24), _spread(rng, 2, 700), rng.randint(1, 32), rng.choice([1, 2, 4, 8]),
                        rng.choice([16, 32]), rng.choice([64, 128]), dtype, rng.choice([0.2, 0.5, 0.8]))
    del case["name"]
    return case


# ----------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------

def _generators(seed):
    host = torch.Generator().manual_seed(seed)
    return host, torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, gen, dtype, scale=1.0):
    """Standard normal values, made in pieces so that a large cache needs no 32-bit copy of itself."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    step = 1 << 26
    for i in range(0, flat.numel(), step):
        piece = flat[i:i + step]
        piece.copy_(torch.randn(piece.numel(), generator=gen, device="cuda") * scale)
    return out


def _lengths(c):
    """The lengths of a case's rows, a property of its sizes: from the longest down, spread evenly."""
    spread = {"attention": c.get("spread"), "branch": 0.7, "compact": 0.8}[c["op"]]
    count = {"attention": c.get("batch"), "branch": c.get("prompts"), "compact": c.get("rows")}[c["op"]]
    lens = [max(1, round(c["longest"] * (1.0 - spread * i / count))) for i in range(count)]
    if spread == 1.0 and count >= 4:
        lens[-2:] = [1, 0]               # a row of one token, a row without any
    return lens


def _shuffled_lengths(c, host):
    lens = torch.tensor(_lengths(c))
    return lens[torch.randperm(len(lens), generator=host)]


def _tables(lens, page, pages, width, host):
    """Block tables over randomly ordered pages: [rows, width] int32, -1 where a row has no page."""
    order = torch.randperm(pages, generator=host)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    used = 0
    for r, n in enumerate(lens.tolist()):
        need = -(-n // page)
        table[r, :need] = order[used:used + need].int()
        used += need
    return table, order[used:]


def _prepare_linear(c, seed):
    _, gen = _generators(seed)
    t = _TYPES[c["dtype"]]
    groups = c["k"] // c["group"]
    x = torch.randn(c["m"], c["k"], generator=gen, device="cuda")
    x[:, :: max(1, c["k"] // 7)] *= 12.0                       # a few outlier channels, as activations have
    scale = 0.002 + 0.004 * torch.rand(groups, c["n"], generator=gen, device="cuda")
    zeros = 0.004 * torch.randn(groups, c["n"], generator=gen, device="cuda")
    return {"x": x.to(t),
            "qweight": torch.randint(-128, 128, (c["n"], c["k"] // 2), generator=gen, device="cuda", dtype=torch.int8),
            "scale": scale.bfloat16(), "zeros": zeros.bfloat16(),
            "bias": torch.randn(c["n"], generator=gen, device="cuda").to(t) if c["bias"] else None}


def _prepare_attention(c, seed):
    host, gen = _generators(seed)
    t, ct = _TYPES[c["dtype"]], _TYPES[c["cache"]]
    lens = _shuffled_lengths(c, host)
    page = c["page"]
    width = -(-c["longest"] // page)
    pages = int((-(-lens // page)).sum()) + 3
    table, _ = _tables(lens, page, pages, width, host)
    shape = (pages, c["kv_heads"], page, c["dim"])
    state = {"q": _normal((c["batch"], c["q_heads"], c["dim"]), gen, t, 2.0)}
    for name in ("k", "v"):
        if c["cache"] == "fp8":
            values = _normal(shape, gen, torch.float16, 60.0).clamp_(-_FP8_MAX, _FP8_MAX).to(ct)
            state[name + "_scale"] = 0.01 + 0.01 * torch.rand(c["kv_heads"], generator=gen, device="cuda")
        else:
            values = _normal(shape, gen, ct)
            state[name + "_scale"] = None
        state[name] = values
    for r, n in enumerate(lens.tolist()):                      # what a recycled page holds past the row's end
        if n % page:
            last = int(table[r, n // page])
            for name in ("k", "v"):
                state[name][last, :, n % page:] = torch.tensor(float("nan"), device="cuda").to(ct)
    return state | {"table": table.cuda(), "lens": lens.int().cuda()}


def _refs(table, pages):
    live = table[table >= 0].long()
    return torch.bincount(live, minlength=pages).int()


def _prepare_branch(c, seed):
    host, gen = _generators(seed)
    t, page = _TYPES[c["dtype"]], c["page"]
    lens = _shuffled_lengths(c, host)
    width = c["longest"] // page + 2
    pages = int((-(-lens // page)).sum()) + c["rows"] + 5
    table, _ = _tables(lens, page, pages, width, host)
    refs = _refs(table, pages)
    table = torch.cat([table, torch.full((c["rows"], width), -1, dtype=torch.int32)])
    lens = torch.cat([lens, torch.zeros(c["rows"], dtype=torch.long)])
    shape = (c["layers"], pages, c["kv_heads"], page, c["dim"])
    new = (c["layers"], c["rows"], c["kv_heads"], c["dim"])
    return {"k": _normal(shape, gen, t), "v": _normal(shape, gen, t), "table": table.cuda(), "lens": lens.int().cuda(),
            "refs": refs.cuda(), "k_new": _normal(new, gen, t), "v_new": _normal(new, gen, t),
            "src": torch.randint(0, c["prompts"], (c["rows"],), generator=host, dtype=torch.int32).cuda(),
            "dst": (c["prompts"] + torch.arange(c["rows"], dtype=torch.int32)).cuda()}


def _prepare_compact(c, seed):
    host, gen = _generators(seed)
    t, page = _TYPES[c["dtype"]], c["page"]
    lens = _shuffled_lengths(c, host)
    used = int((-(-lens // page)).sum())
    pages = int(used / c["fill"]) + 1
    table, _ = _tables(lens, page, pages, -(-c["longest"] // page) + 1, host)
    if c["rows"] > 1:                                          # two rows share the first page of the first
        table[1, 0] = table[0, 0]
    shape = (c["layers"], pages, c["kv_heads"], page, c["dim"])
    return {"k": _normal(shape, gen, t), "v": _normal(shape, gen, t), "table": table.cuda(),
            "refs": _refs(table, pages).cuda()}


def prepare(case, seed):
    return {"case": case} | {"linear": _prepare_linear, "attention": _prepare_attention, "branch": _prepare_branch,
                             "compact": _prepare_compact}[case["op"]](case, seed)


# ----------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------

def _taken(x, *index):
    """x[index]; 8-bit floats are indexed as the bytes they are held in."""
    return x.view(torch.uint8)[index].view(x.dtype) if x.dtype == torch.float8_e4m3fn else x[index]


def _codes(qweight):
    u = qweight.view(torch.uint8)
    return torch.stack([u & 15, u >> 4], dim=-1).reshape(u.shape[0], -1)


def _plain_linear(s):
    c = s["case"]
    n, k, g = c["n"], c["k"], c["group"]
    q = _codes(s["qweight"]).float().view(n, k // g, g)
    w = (q - 8.0) * s["scale"].float().t().unsqueeze(-1) + s["zeros"].float().t().unsqueeze(-1)
    y = s["x"].float() @ w.view(n, k).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def _plain_attention(s):
    c = s["case"]
    b, hq, hk, d, page = c["batch"], c["q_heads"], c["kv_heads"], c["dim"], c["page"]
    table = s["table"].long().clamp(min=0)
    span = table.shape[1] * page
    pos = torch.arange(span, device="cuda")
    lens = s["lens"].long().unsqueeze(1)
    vis = pos < lens
    if c["window"]:
        vis &= (pos >= lens - c["window"]) | (pos < c["sinks"])
    vis = vis.view(b, 1, span)

    def gathered(name):
        x = _taken(s[name], table).transpose(1, 2).reshape(b, hk, span, d).float()
        if s[name + "_scale"] is not None:
            x = x * s[name + "_scale"].view(1, hk, 1, 1)
        return torch.where(vis.unsqueeze(-1), x, 0.0)

    q = s["q"].float().view(b, hk, hq // hk, d) * (1.0 / math.sqrt(d))
    score = q @ gathered("k").transpose(-1, -2)
    score = torch.where(vis.unsqueeze(2), score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = (p @ gathered("v")) / torch.where(total == 0, 1.0, total)
    return out.view(b, hq, d).to(s["q"].dtype)


def _plain_branch(s):
    table, lens, refs, dst = s["table"], s["lens"], s["refs"], s["dst"].long()
    src, page, n = s["src"].long(), s["case"]["page"], s["case"]["rows"]
    slot = torch.arange(table.shape[1], device="cuda")

    def count(rows, by):
        held = slot < (lens[rows].long().unsqueeze(1) + page - 1) // page
        refs.scatter_add_(0, table[rows].long().clamp(min=0).flatten(), held.int().flatten() * by)

    count(dst, -1)                                             # free
    table[dst], lens[dst] = -1, 0
    table[dst], lens[dst] = table[src], lens[src]              # fork
    count(dst, 1)
    start = lens[dst]                                          # room for one token
    at = (start // page).long()
    last = table[dst].gather(1, at.clamp(max=table.shape[1] - 1).unsqueeze(1)).squeeze(1)
    fresh = start % page == 0
    shared = ~fresh & (refs[last.long().clamp(min=0)] > 1)
    need = (fresh | shared).int()
    free = torch.sort((refs > 0).int(), stable=True).indices
    got = free[(torch.cumsum(need, 0) - need).long()].int()
    copies = torch.full((n, 2), -1, dtype=torch.int32, device="cuda")
    copies[:, 0] = torch.where(shared, last, -1)
    copies[:, 1] = torch.where(shared, got, -1)
    refs.scatter_add_(0, last.long().clamp(min=0), -shared.int())
    refs.scatter_add_(0, got.long(), need)
    where = torch.where(need.bool(), got, last)
    table[dst, at] = where
    lens[dst] = start + 1
    a, b = last[shared].long(), got[shared].long()
    for name in ("k", "v"):
        s[name][:, b] = s[name][:, a]
        s[name][:, where.long(), :, (start % page).long()] = s[name + "_new"].transpose(0, 1)
    return {"k": s["k"], "v": s["v"], "table": table, "lens": lens, "refs": refs, "start": start, "copies": copies}


def _plain_compact(s):
    refs = s["refs"]
    pages = refs.numel()
    index = torch.arange(pages, device="cuda")
    held = refs > 0
    live = held.sum()
    holes, movers = index[~held & (index < live)], index[held & (index >= live)]
    to = index.clone()
    to[movers] = holes
    table = torch.where(s["table"] >= 0, to[s["table"].long().clamp(min=0)].int(), -1)
    moves = torch.full((pages // 2, 2), -1, dtype=torch.int32, device="cuda")
    moves[:len(movers), 0], moves[:len(movers), 1] = movers.int(), holes.int()
    packed = torch.zeros_like(refs)
    packed[to[held]] = refs[held]
    for name in ("k", "v"):
        s[name][:, holes] = s[name][:, movers]
    return {"k": s["k"], "v": s["v"], "table": table, "refs": packed, "moves": moves}


def _own_linear(s):
    from comfy_quant_bench_b200 import ops
    return ops.w4a16_linear(s["x"], s["qweight"], s["scale"], s["zeros"], s["bias"], group_size=s["case"]["group"])


def _own_attention(s):
    from comfy_quant_bench_b200 import kvcache
    return kvcache.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], window=s["case"]["window"],
                                   sinks=s["case"]["sinks"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def _own_branch(s):
    from comfy_quant_bench_b200 import kvcache
    start, copies = kvcache.branch_rows(s["table"], s["lens"], s["refs"], s["src"], s["dst"], 1, s["k"], s["v"])
    kvcache.append_kv(s["k_new"], s["v_new"], s["k"], s["v"], s["table"], s["dst"], start)
    return {"k": s["k"], "v": s["v"], "table": s["table"], "lens": s["lens"], "refs": s["refs"], "start": start,
            "copies": copies}


def _own_compact(s):
    from comfy_quant_bench_b200 import kvcache
    table, refs, moves = kvcache.compact_pages(s["table"], s["refs"], s["k"], s["v"])
    return {"k": s["k"], "v": s["v"], "table": table, "refs": refs, "moves": moves}


def run(state):
    which = {"linear": (_plain_linear, _own_linear), "attention": (_plain_attention, _own_attention),
             "branch": (_plain_branch, _own_branch), "compact": (_plain_compact, _own_compact)}
    return which[state["case"]["op"]][1 if own else 0](state)


# ----------------------------------------------------------------------------------------------------------
# the work a pass cannot do without
# ----------------------------------------------------------------------------------------------------------

def _visible(n, window, sinks):
    return n if not window else min(n, window) + min(sinks, max(0, n - window))


def work(case):
    c = case
    if c["op"] == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        return {"bytes": n * k // 2 + 4 * n * (k // c["group"]) + 2 * m * k + 2 * m * n + (2 * n if c["bias"] else 0),
                "flops": 2 * m * n * k}
    if c["op"] == "attention":
        seen = sum(_visible(n, c["window"], c["sinks"]) for n in _lengths(c))
        return {"bytes": 2 * seen * c["kv_heads"] * c["dim"] * _SIZE[c["cache"]] + 4 * c["batch"] * c["q_heads"] * c["dim"],
                "flops": 4 * seen * c["q_heads"] * c["dim"]}
    page_bytes = 2 * c["layers"] * c["kv_heads"] * c["page"] * c["dim"] * 2
    held = [-(-n // c["page"]) for n in _lengths(c)]
    if c["op"] == "branch":
        # each row's last page read and written once, its new token too, and its table row
        tables = c["rows"] * 3 * 4 * (sum(held) // len(held))
        return {"bytes": 2 * c["rows"] * page_bytes * (c["page"] - 1) // c["page"] + 2 * c["rows"] * page_bytes // c["page"] + tables,
                "flops": 0}
    moved = sum(held) * (1 - c["fill"])                        # holes below the live count, pages in random order
    return {"bytes": int(2 * moved * page_bytes) + 8 * int(sum(held) / c["fill"]) + 8 * sum(held), "flops": 0}


# ----------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ----------------------------------------------------------------------------------------------------------

def _exact_linear(c, s):
    out = torch.empty(c["m"], c["n"], dtype=torch.float64, device="cuda")
    x = s["x"].double()
    raw = s["qweight"].int()
    per = torch.arange(c["k"], device="cuda") // c["group"]
    for lo in range(0, c["n"], 4096):
        rows = slice(lo, min(c["n"], lo + 4096))
        w = torch.empty(raw[rows].shape[0], c["k"], dtype=torch.float64, device="cuda")
        w[:, 0::2] = (raw[rows] % 16).double()
        w[:, 1::2] = (raw[rows] % 256 // 16).double()
        w = (w - 8) * s["scale"][:, rows].double().t()[:, per] + s["zeros"][:, rows].double().t()[:, per]
        out[:, rows] = torch.einsum("mk,nk->mn", x, w)
    return out if s["bias"] is None else out + s["bias"].double()


def _exact_attention(c, s):
    b, hk, d, page = c["batch"], c["kv_heads"], c["dim"], c["page"]
    each = c["q_heads"] // hk
    out = torch.zeros(b, c["q_heads"], d, dtype=torch.float64, device="cuda")
    for r, n in enumerate(s["lens"].tolist()):
        seen = [j for j in (range(n) if not c["window"] else
                            sorted(set(range(max(0, n - c["window"]), n)) | set(range(min(n, c["sinks"])))))]
        if not seen:
            continue
        seen = torch.tensor(seen, device="cuda")
        pg, slot = s["table"][r].long()[seen // page], seen % page
        for h in range(hk):
            k, v = _taken(s["k"], pg, h, slot).double(), _taken(s["v"], pg, h, slot).double()
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
            p = torch.softmax((s["q"][r, h * each:(h + 1) * each].double() @ k.t()) / math.sqrt(d), dim=-1)
            out[r, h * each:(h + 1) * each] = p @ v
    return out


def _exact_branch(c, s):
    page = c["page"]
    table, lens, refs = s["table"].tolist(), s["lens"].tolist(), s["refs"].tolist()
    k, v = s["k"].double(), s["v"].double()
    src, dst = s["src"].tolist(), s["dst"].tolist()
    for a, b in zip(src, dst):                                 # the destination rows start empty
        for j in range(-(-lens[a] // page)):
            table[b][j] = table[a][j]
            refs[table[a][j]] += 1
        lens[b] = lens[a]
    free = [p for p, count in enumerate(refs) if count == 0]
    counts = list(refs)
    start, copies = [], []
    for b in dst:
        at, slot = divmod(lens[b], page)
        copies.append([-1, -1])
        if slot == 0 or counts[table[b][at]] > 1:
            new = free.pop(0)
            if slot:
                copies[-1] = [table[b][at], new]
                refs[table[b][at]] -= 1
                k[:, new], v[:, new] = k[:, table[b][at]].clone(), v[:, table[b][at]].clone()
            table[b][at] = new
            refs[new] = 1
        start.append(lens[b])
        lens[b] += 1
    for i, b in enumerate(dst):
        pg, slot = table[b][start[i] // page], start[i] % page
        k[:, pg, :, slot], v[:, pg, :, slot] = s["k_new"][:, i].double(), s["v_new"][:, i].double()
    whole = {"table": table, "lens": lens, "refs": refs, "start": start, "copies": copies}
    return {"k": k, "v": v} | {n: torch.tensor(x, dtype=torch.int32) for n, x in whole.items()}


def _exact_compact(c, s):
    table, refs = s["table"].tolist(), s["refs"].tolist()
    k, v = s["k"].double(), s["v"].double()
    live = sum(count > 0 for count in refs)
    holes = [p for p in range(live) if refs[p] == 0]
    moves = []
    for p in range(live, len(refs)):
        if refs[p] > 0:
            to = holes.pop(0)
            moves.append([p, to])
            k[:, to], v[:, to] = k[:, p].clone(), v[:, p].clone()
            refs[to], refs[p] = refs[p], 0
    to = dict(moves)
    table = [[to.get(p, p) for p in row] for row in table]
    moves += [[-1, -1]] * (len(refs) // 2 - len(moves))
    whole = {"table": table, "refs": refs, "moves": moves}
    return {"k": k, "v": v} | {n: torch.tensor(x, dtype=torch.int32).reshape(-1, 2) if n == "moves" else
                               torch.tensor(x, dtype=torch.int32) for n, x in whole.items()}


def exact(case, seed):
    state = prepare(case, seed)
    return {"linear": _exact_linear, "attention": _exact_attention, "branch": _exact_branch,
            "compact": _exact_compact}[case["op"]](case, state)

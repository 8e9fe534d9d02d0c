"""Measured cases of the operators around a decode step's linears and attention: the root-mean-square norm with the
residual's addition (16-bit or 8-bit output), rotary positions with the append to a paged cache, attention of a batch
that shares a long prefix, and the choice of the next tokens from given random numbers.

``run`` computes a case in plain torch operations where ``own`` is false and through the package's operators where it
is true; ``exact`` gives the same outputs from the definitions in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4, "fp8": 1}
_TOP = {"int8": 127.0, "fp8": 448.0}


def _norm(name, rows, width, dtype, residual, quant, group):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype, "residual": residual,
            "quant": quant, "group": group}


def _rotate(name, tokens, seqs, q_heads, kv_heads, dim, rot, interleaved, normed, far, page, dtype, cache):
    return {"name": name, "op": "rotate", "tokens": tokens, "seqs": seqs, "q_heads": q_heads, "kv_heads": kv_heads,
            "dim": dim, "rot": rot, "interleaved": interleaved, "normed": normed, "far": far, "page": page,
            "dtype": dtype, "cache": cache}


def _prefix(name, batch, q_heads, kv_heads, dim, page, prefix, longest, dtype, cache):
    return {"name": name, "op": "prefix", "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "prefix": prefix, "longest": longest, "dtype": dtype, "cache": cache}


def _sample(name, rows, vocab, dtype, top_k, top_p, min_p):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "top_k": top_k, "top_p": top_p,
            "min_p": min_p}


def listed():
    return [
        # one token between two blocks: latency
        _norm("norm_one", 1, 4096, "bf16", True, "", 0),
        # a ragged batch of an odd width in half precision, codes for an 8-bit linear
        _norm("norm_odd_int8", 777, 1001, "f16", True, "int8", 0),
        # a long prompt through a wide model, 8-bit floats with a scale per 128 columns
        _norm("norm_prompt_fp8", 8192, 8192, "bf16", True, "fp8", 128),
        # one new token of one conversation: latency
        _rotate("rotate_one", 1, 1, 16, 2, 128, 128, False, False, 333, 16, "bf16", "bf16"),
        # one new token for each of 64 conversations, normed heads in pairs, an 8-bit cache
        _rotate("rotate_step", 64, 64, 32, 8, 128, 128, True, True, 8000, 16, "bf16", "fp8"),
        # a prompt far into a long context, half of each head turned
        _rotate("rotate_prompt", 16001, 2, 32, 8, 128, 64, False, False, 120000, 64, "f16", "f16"),
        # four samples of one short prompt
        _prefix("prefix_few", 4, 16, 2, 128, 16, 500, 60, "bf16", "bf16"),
        # a server's batch behind one long instruction
        _prefix("prefix_batch", 64, 32, 8, 128, 16, 16003, 700, "bf16", "bf16"),
        # wide heads, an 8-bit cache
        _prefix("prefix_wide_fp8", 40, 16, 4, 256, 32, 20000, 300, "f16", "fp8"),
        # the largest call: many samples of one long document
        _prefix("prefix_many", 256, 64, 8, 128, 16, 30011, 256, "bf16", "bf16"),
        # one token of one conversation: latency
        _sample("sample_one", 1, 32000, "bf16", 0, 0.9, 0.0),
        # a full batch over a large vocabulary, every filter in use
        _sample("sample_batch", 128, 128257, "f32", 200, 0.95, 0.02),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "rotate", "prefix", "prefix", "sample"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "norm":
        width = _spread(rng, 64, 16384)
        group = 0
        quant = rng.choice(["", "int8", "fp8"])
        if quant and rng.random() < 0.5:
            group = rng.choice([32, 64, 128])
            width = max(1, width // group) * group
        case = _norm("", _spread(rng, 1, max(2, (1 << 26) // width)), width, dtype, rng.random() < 0.8, quant, group)
    elif op == "rotate":
        dim = rng.choice([64, 128, 256])
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        q_heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
        tokens = _spread(rng, 1, max(2, 60_000_000 // (dim * (q_heads + 2 * kv_heads))))
        seqs = tokens if rng.random() < 0.5 and tokens <= 256 else rng.randint(1, min(tokens, 8))
        case = _rotate("", tokens, seqs, q_heads, kv_heads, dim, rng.choice([dim, dim, dim // 2, dim // 4]),
                       rng.random() < 0.5, rng.random() < 0.5, _spread(rng, 1, 120000), rng.choice([16, 32, 64, 128]),
                       dtype, rng.choice([dtype, dtype, "fp8"]))
        if seqs == tokens:                                     # a deep cache for every row: below 4 GB in all
            case["far"] = min(case["far"], max(1, 1_000_000_000 // (seqs * kv_heads * dim)))
    elif op == "prefix":
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        dim = rng.choice([64, 128, 256])
        q_heads = kv_heads * rng.choice([1, 2, 4, 5, 7, 8, 12])
        batch = _spread(rng, 2, 256)
        # products below those of the largest listed case, a cache below 4 GB
        prefix = _spread(rng, 1, max(2, min(60000, 60_000_000_000 // (batch * q_heads * dim))))
        longest = _spread(rng, 1, max(2, min(1000, 500_000_000 // (batch * kv_heads * dim))))
        case = _prefix("", batch, q_heads, kv_heads, dim, rng.choice([16, 32, 64, 128]), prefix, longest, dtype,
                       rng.choice([dtype, dtype, "fp8"]))
    else:
        vocab = _spread(rng, 500, 200000)
        case = _sample("", _spread(rng, 1, max(2, min(256, 16_000_000 // vocab))), vocab, rng.choice([dtype, "f32"]),
                       rng.choice([0, 1, 20, _spread(rng, 2, 1000)]), rng.choice([1.0, 0.95, round(rng.uniform(0.1, 1), 3)]),
                       rng.choice([0.0, 0.0, 0.05, round(rng.uniform(0, 0.5), 3)]))
    del case["name"]
    return case


# ----------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------

def _normal(shape, gen, dtype, scale=1.0):
    """Normal values, made in pieces so that a large cache needs no 32-bit copy of itself."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    step = 1 << 26
    for i in range(0, flat.numel(), step):
        piece = flat[i:i + step]
        x = torch.randn(piece.numel(), generator=gen, device="cuda") * scale
        piece.copy_(x.clamp_(-448.0, 448.0) if dtype == torch.float8_e4m3fn else x)
    return out


def _prepare_norm(c, host, gen):
    t, m, n = _TYPES[c["dtype"]], c["rows"], c["width"]
    x = torch.randn(m, n, generator=gen, device="cuda")
    x[:, :: max(1, n // 5)] *= 20.0                            # a few outlier channels, as activations have
    return {"x": x.to(t), "weight": (1.0 + 0.2 * torch.randn(n, generator=gen, device="cuda")).to(t),
            "residual": _normal((m, n), gen, t, 3.0) if c["residual"] else None}


def _rope(positions, rot, factor):
    """(cos, sin) of every position for rot / 2 frequencies, positions divided by `factor`: [positions, rot / 2, 2]."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    angle = torch.outer(torch.arange(positions, device="cuda", dtype=torch.float64) / factor, inv)
    return torch.stack([angle.cos(), angle.sin()], dim=-1).float()


def _prepare_rotate(c, host, gen):
    t, ct, page = _TYPES[c["dtype"]], _TYPES[c["cache"]], c["page"]
    n, seqs = c["tokens"], c["seqs"]
    each = torch.full((seqs,), n // seqs)
    each[: n % seqs] += 1
    start = torch.randint(0, c["far"] + 1, (seqs,), generator=host)
    start[0] = c["far"]
    rows = torch.repeat_interleave(torch.arange(seqs), each)
    first = torch.cumsum(each, 0) - each
    positions = start[rows] + torch.arange(n) - first[rows]
    width = (int((start + each).max()) + page - 1) // page
    # a page of the pool for each place that a new token takes, in random order; earlier pages are not looked at
    table = torch.full((seqs, width), -1, dtype=torch.int32)
    places = torch.unique(rows * width + positions // page)
    pages = int((each // page).sum()) + 2 * seqs + 3           # whatever the starts are
    table.view(-1)[places] = torch.randperm(pages, generator=host)[: len(places)].int()
    heads = c["q_heads"] + 2 * c["kv_heads"]
    qkv = _normal((n, heads, c["dim"]), gen, t, 2.0)
    shape = (pages, c["kv_heads"], page, c["dim"])
    k, v = (_normal(shape, gen, ct) for _ in range(2))
    scales = [0.02 + 0.02 * torch.rand(c["kv_heads"], generator=gen, device="cuda") if c["cache"] == "fp8" else None
              for _ in range(2)]
    weights = [(1.0 + 0.2 * torch.randn(c["dim"], generator=gen, device="cuda")).to(t) if c["normed"] else None
               for _ in range(2)]
    return {"qkv": qkv, "k": k, "v": v, "table": table.cuda(), "rows": rows.int().cuda(),
            "positions": positions.int().cuda(), "rope": _rope(c["far"] + n + 1, c["rot"], 1.0 if c["far"] < 32000 else 4.0),
            "k_scale": scales[0], "v_scale": scales[1], "q_norm": weights[0], "k_norm": weights[1]}


def _suffixes(c):
    """Each row's tokens behind the shared ones, from the longest down; where there are four rows, one has none."""
    lens = [max(1, round(c["longest"] * (1.0 - i / c["batch"]))) for i in range(c["batch"])]
    if c["batch"] >= 4:
        lens[-1] = 0
    return lens


def _prepare_prefix(c, host, gen):
    t, ct, page, prefix = _TYPES[c["dtype"]], _TYPES[c["cache"]], c["page"], c["prefix"]
    tail = torch.tensor(_suffixes(c))[torch.randperm(c["batch"], generator=host)]
    lens = prefix + tail
    whole = prefix // page                                     # pages that all rows hold; the next one is each row's own
    need = (lens + page - 1) // page
    width = int(need.max())
    pages = whole + int((need - whole).sum()) + 3
    order = torch.randperm(pages, generator=host).int()
    table = torch.full((c["batch"], width), -1, dtype=torch.int32)
    table[:, :whole] = order[:whole]
    mine = torch.arange(width).unsqueeze(0).expand(c["batch"], -1)
    mine = (mine >= whole) & (mine < need.unsqueeze(1))
    table[mine] = order[whole: whole + int(mine.sum())]
    shape = (pages, c["kv_heads"], page, c["dim"])
    state = {"q": _normal((c["batch"], c["q_heads"], c["dim"]), gen, t, 2.0)}
    behind = torch.arange(page, device="cuda")
    for name in ("k", "v"):
        if c["cache"] == "fp8":
            values = _normal(shape, gen, ct, 60.0)
            state[name + "_scale"] = 0.01 + 0.01 * torch.rand(c["kv_heads"], generator=gen, device="cuda")
        else:
            values = _normal(shape, gen, ct)
            state[name + "_scale"] = None
        raw = values.view(torch.uint8) if c["cache"] == "fp8" else values
        if prefix % page:                                      # copies of the page that the prefix ends in
            own_pages = table[:, whole].cuda().long()
            raw[own_pages, :, : prefix % page] = raw[own_pages[:1], :, : prefix % page]
        last = table[torch.arange(c["batch"]), (need - 1).clamp(min=0)].long().cuda()
        used = (lens.cuda() - 1) % page + 1
        part = (behind.unsqueeze(0) >= used.unsqueeze(1)) & (lens.cuda() % page > 0).unsqueeze(1)
        hole = part.view(-1, 1, page, 1)                       # what a recycled page holds past the row's end
        nan = torch.tensor(float("nan"), device="cuda").to(ct)
        nan = nan.view(torch.uint8) if c["cache"] == "fp8" else nan
        raw[last] = torch.where(hole, nan, raw[last])
        state[name] = values
    return state | {"table": table.cuda(), "lens": lens.int().cuda(),
                    "shared": torch.tensor([prefix], dtype=torch.int32, device="cuda")}


def _prepare_sample(c, host, gen):
    m, n = c["rows"], c["vocab"]
    x = 2.5 * torch.randn(m, n, generator=gen, device="cuda")
    likely = torch.randint(0, n, (m, 12), generator=gen, device="cuda")
    x.scatter_add_(1, likely, 4.0 + 6.0 * torch.rand(m, 12, generator=gen, device="cuda"))
    x[:, torch.randint(0, n, (max(1, n // 100),), generator=gen, device="cuda")] = float("-inf")   # tokens not allowed
    x[:, 0] = 0.0
    return {"logits": x.to(_TYPES[c["dtype"]]), "uniform": torch.rand(m, generator=gen, device="cuda"),
            "temperature": 0.5 + torch.rand(m, generator=gen, device="cuda")}


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"case": case} | {"norm": _prepare_norm, "rotate": _prepare_rotate, "prefix": _prepare_prefix,
                             "sample": _prepare_sample}[case["op"]](case, host, gen)


# ----------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------

def _plain_norm(s):
    c = s["case"]
    t, n = s["x"].dtype, c["width"]
    h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(t)
    # the product with the weight is exact in 32 bits (16-bit factors); its scale is common to the row
    product = h.float() * s["weight"].float()
    inv = torch.rsqrt(h.float().square().mean(-1, keepdim=True) + 1e-6)
    if not c["quant"]:
        return {"y": (product * inv).to(t), "h": h}
    top, group = _TOP[c["quant"]], c["group"] or n
    product = product.view(-1, n // group, group)
    most = product.abs().amax(-1, keepdim=True)
    scale = (most * inv.unsqueeze(-1) / top).squeeze(-1)
    # 64 bits: the codes next to a border, and the rank of what is held in a few bits
    code = product.double() * top / torch.where(most == 0, 1.0, most).double()
    code = code.round().to(torch.int8) if c["quant"] == "int8" else code.float().to(torch.float8_e4m3fn)
    return {"q": code.view(-1, n), "scale": scale.t().contiguous() if c["group"] else scale.view(-1), "h": h}


def _turned(x, cos, sin, rot, interleaved):
    """x [T, heads, D] in 32 bits with its first `rot` columns turned by the token's angles ([T, 1, rot / 2])."""
    head, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2), rest], dim=-1)
    a, b = head[..., : rot // 2], head[..., rot // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, rest], dim=-1)


def _put(cache, page, slot, x):
    """cache[page, :, slot] = x; 8-bit floats are moved as the bytes they are held in."""
    x = x.to(cache.dtype)
    if cache.dtype == torch.float8_e4m3fn:
        cache, x = cache.view(torch.uint8), x.view(torch.uint8)
    cache[page, :, slot] = x


def _plain_rotate(s):
    c = s["case"]
    q, k, v = s["qkv"].float().split((c["q_heads"], c["kv_heads"], c["kv_heads"]), dim=1)
    if c["normed"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * s["q_norm"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * s["k_norm"].float()
    at = s["positions"].long()
    cos, sin = s["rope"][at].unsqueeze(1).unbind(-1)
    q, k = _turned(q, cos, sin, c["rot"], c["interleaved"]), _turned(k, cos, sin, c["rot"], c["interleaved"])
    page = s["table"][s["rows"].long(), at // c["page"]].long()
    if c["cache"] == "fp8":
        k = (k / s["k_scale"].view(-1, 1)).clamp(-448.0, 448.0)
        v = (v / s["v_scale"].view(-1, 1)).clamp(-448.0, 448.0)
    _put(s["k"], page, at % c["page"], k)
    _put(s["v"], page, at % c["page"], v)
    return {"q": q.to(s["qkv"].dtype), "k": s["k"], "v": s["v"]}


def _taken(x, *index):
    """x[index]; 8-bit floats are indexed as the bytes they are held in."""
    return x.view(torch.uint8)[index].view(x.dtype) if x.dtype == torch.float8_e4m3fn else x[index]


def _plain_prefix(s):
    c = s["case"]
    b, hq, hk, d, page, prefix = c["batch"], c["q_heads"], c["kv_heads"], c["dim"], c["page"], c["prefix"]
    q = s["q"].float().view(b, hk, hq // hk, d) * (1.0 / math.sqrt(d))
    lens = s["lens"].long()
    scale = [1.0 if s[n + "_scale"] is None else s[n + "_scale"].view(hk, 1, 1) for n in ("k", "v")]
    # what all rows share, once: [hk, prefix, d]
    shared = s["table"][0, : -(-prefix // page)].long()
    k0, v0 = (_taken(s[n], shared).transpose(0, 1).reshape(hk, -1, d)[:, :prefix].float() * f for n, f in zip("kv", scale))
    score0 = torch.einsum("bhgd,hnd->bhgn", q, k0)
    # each row's own tokens
    whole = prefix // page
    table = s["table"][:, whole:].long().clamp(min=0)
    span = table.shape[1] * page
    at = whole * page + torch.arange(span, device="cuda")
    seen = ((at >= prefix) & (at < lens.unsqueeze(1))).view(b, 1, span, 1)
    k1, v1 = (torch.where(seen, _taken(s[n], table).transpose(1, 2).reshape(b, hk, span, d).float() * f, 0.0)
              for n, f in zip("kv", scale))
    score1 = torch.where(seen.transpose(2, 3), q @ k1.transpose(-1, -2), float("-inf"))
    score = torch.cat([score0, score1], dim=-1)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = torch.einsum("bhgn,hnd->bhgd", p[..., :prefix], v0) + p[..., prefix:] @ v1
    return (out / p.sum(-1, keepdim=True)).reshape(b, hq, d).to(s["q"].dtype)


def _plain_sample(s):
    c = s["case"]
    n = c["vocab"]
    x = s["logits"].double()                                   # 64 bits: sums and values next to a border
    top = x.amax(-1, keepdim=True)
    weight = torch.exp((x - top) / s["temperature"].double().unsqueeze(1))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    rank = torch.arange(n, device="cuda")
    ordered = weight.gather(1, order)
    if c["top_k"]:
        ordered = torch.where(rank < c["top_k"], ordered, 0.0)
    before = torch.cumsum(ordered, -1) - ordered
    limit = torch.tensor(c["top_p"], dtype=torch.float32, device="cuda").double()
    kept = (before < limit * ordered.sum(-1, keepdim=True)) | (rank == 0) if c["top_p"] < 1 else torch.ones_like(ordered, dtype=torch.bool)
    kept &= ordered >= torch.tensor(c["min_p"], dtype=torch.float32, device="cuda").double()
    weight = torch.zeros_like(weight).scatter(1, order, torch.where(kept, ordered, 0.0))
    run_sum = torch.cumsum(weight, -1)
    total = run_sum[:, -1:]
    token = (run_sum <= s["uniform"].double().unsqueeze(1) * total).sum(-1, keepdim=True)
    token = torch.minimum(token, torch.where(weight > 0, rank, 0).amax(-1, keepdim=True))
    return {"token": token.squeeze(1), "logprob": torch.log(weight.gather(1, token) / total).squeeze(1).float()}


def _own_norm(s):
    from comfy_quant_bench_b200 import ops
    c = s["case"]
    got = ops.add_rmsnorm(s["x"], s["weight"], s["residual"], eps=1e-6, quant=c["quant"] or None, group_size=c["group"])
    return dict(zip(("q", "scale", "h") if c["quant"] else ("y", "h"), got))


def _own_rotate(s):
    from comfy_quant_bench_b200 import kvcache
    c = s["case"]
    q, k, v = s["qkv"].split((c["q_heads"], c["kv_heads"], c["kv_heads"]), dim=1)
    q = kvcache.append_rotated(q, k, v, s["k"], s["v"], s["table"], s["rows"], s["positions"], s["rope"],
                               interleaved=c["interleaved"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6,
                               k_scale=s["k_scale"], v_scale=s["v_scale"])
    return {"q": q, "k": s["k"], "v": s["v"]}


def _own_prefix(s):
    from comfy_quant_bench_b200 import kvcache
    return kvcache.prefix_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["shared"], k_scale=s["k_scale"],
                                    v_scale=s["v_scale"])


def _own_sample(s):
    from comfy_quant_bench_b200 import ops
    c = s["case"]
    token, logprob = ops.sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"], top_k=c["top_k"],
                                       top_p=c["top_p"], min_p=c["min_p"], return_logprob=True)
    return {"token": token, "logprob": logprob}


def run(state):
    which = {"norm": (_plain_norm, _own_norm), "rotate": (_plain_rotate, _own_rotate),
             "prefix": (_plain_prefix, _own_prefix), "sample": (_plain_sample, _own_sample)}
    return which[state["case"]["op"]][1 if own else 0](state)


# ----------------------------------------------------------------------------------------------------------
# the work a pass cannot do without
# ----------------------------------------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "norm":
        cells, size = c["rows"] * c["width"], _SIZE[c["dtype"]]
        out = cells + 4 * c["rows"] * (c["width"] // c["group"] if c["group"] else 1) if c["quant"] else size * cells
        # the sum with the residual is read once and written once; without one it is the input itself
        return {"bytes": size * cells * (3 if c["residual"] else 1) + out + size * c["width"], "flops": 0}
    if c["op"] == "rotate":
        size, heads = _SIZE[c["dtype"]], c["q_heads"] + 2 * c["kv_heads"]
        moved = c["tokens"] * c["dim"] * (size * heads + size * c["q_heads"] + _SIZE[c["cache"]] * 2 * c["kv_heads"])
        return {"bytes": moved + 4 * c["rot"] * c["tokens"] + 12 * c["tokens"], "flops": 0}
    if c["op"] == "prefix":
        keys = c["prefix"] + sum(_suffixes(c))
        pairs = c["batch"] * c["prefix"] + sum(_suffixes(c))
        return {"bytes": 2 * keys * c["kv_heads"] * c["dim"] * _SIZE[c["cache"]] + 2 * _SIZE[c["dtype"]] * c["batch"] * c["q_heads"] * c["dim"],
                "flops": 4 * pairs * c["q_heads"] * c["dim"]}
    return {"bytes": c["rows"] * (c["vocab"] * _SIZE[c["dtype"]] + 20), "flops": 0}


# ----------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ----------------------------------------------------------------------------------------------------------

def _exact_norm(c, s):
    x = s["x"].double()
    if s["residual"] is not None:
        x = x + s["residual"].double()
    h = x.to(s["x"].dtype).double()                            # the residual stream holds 16 bits
    rms = torch.linalg.vector_norm(h, dim=-1, keepdim=True) / math.sqrt(c["width"])
    y = h / torch.sqrt(rms ** 2 + 1e-6) * s["weight"].double()
    if not c["quant"]:
        return {"y": y, "h": x}
    per = c["group"] or c["width"]
    blocks = y.unflatten(-1, (c["width"] // per, per))
    scale = torch.linalg.vector_norm(blocks, ord=math.inf, dim=-1) / _TOP[c["quant"]]
    q = (blocks / scale.clamp(min=1e-300).unsqueeze(-1)).flatten(-2)
    return {"q": None if c["quant"] == "int8" else q, "scale": scale.t().contiguous() if c["group"] else scale.flatten(), "h": x}


def _exact_rotate(c, s):
    hq, hk = c["q_heads"], c["kv_heads"]
    x = s["qkv"].double()
    parts = [x[:, :hq], x[:, hq: hq + hk], x[:, hq + hk:]]
    z = torch.view_as_complex(s["rope"].double())[s["positions"].long()].unsqueeze(1)
    rot = c["rot"]
    done = []
    for part, w in zip(parts[:2], (s["q_norm"], s["k_norm"])):
        if w is not None:
            part = part / torch.sqrt((part * part).sum(-1, keepdim=True) / c["dim"] + 1e-6) * w.double()
        if c["interleaved"]:
            pairs = torch.view_as_complex(part[..., :rot].unflatten(-1, (rot // 2, 2)).contiguous())
            turned = torch.view_as_real(pairs * z).flatten(-2)
        else:
            pairs = torch.complex(part[..., : rot // 2], part[..., rot // 2: rot]) * z
            turned = torch.cat([pairs.real, pairs.imag], dim=-1)
        done.append(torch.cat([turned, part[..., rot:]], dim=-1))
    q, k = done
    v = parts[2]
    if c["cache"] == "fp8":
        k, v = k / s["k_scale"].double().view(hk, 1), v / s["v_scale"].double().view(hk, 1)
        k, v = (torch.clamp(e, -448.0, 448.0) for e in (k, v))
    caches = []
    for cache, new in ((s["k"], k), (s["v"], v)):
        cache = cache.double()
        flat = cache.transpose(1, 2).reshape(-1, hk, c["dim"])   # [pages * page, hk, d]
        pos = s["positions"].long()
        flat[s["table"][s["rows"].long(), pos // c["page"]].long() * c["page"] + pos % c["page"]] = new
        caches.append(flat.view(cache.shape[0], c["page"], hk, c["dim"]).transpose(1, 2).contiguous())
    return {"q": q, "k": caches[0], "v": caches[1]}


def _exact_prefix(c, s):
    b, hk, d, page, prefix = c["batch"], c["kv_heads"], c["dim"], c["page"], c["prefix"]
    each = c["q_heads"] // hk
    out = torch.empty(b, c["q_heads"], d, dtype=torch.float64, device="cuda")
    lens = s["lens"].tolist()

    def tokens(name, row, h, lo, hi):
        at = torch.arange(lo, hi, device="cuda")
        x = _taken(s[name], s["table"][row].long()[at // page], h, at % page).double()
        return x if s[name + "_scale"] is None else x * s[name + "_scale"][h].double()

    for h in range(hk):
        k0, v0 = (tokens(n, 0, h, 0, prefix) for n in "kv")
        for lo in range(0, b, 32):                             # 32 rows' scores at a time
            rows = range(lo, min(b, lo + 32))
            shared = torch.matmul(s["q"][lo: lo + 32, h * each: (h + 1) * each].double(), k0.t()) / math.sqrt(d)
            for r in rows:
                k1, v1 = (tokens(n, r, h, prefix, lens[r]) for n in "kv")
                q = s["q"][r, h * each: (h + 1) * each].double()
                p = torch.softmax(torch.cat([shared[r - lo], q @ k1.t() / math.sqrt(d)], dim=-1), dim=-1)
                out[r, h * each: (h + 1) * each] = p[:, :prefix] @ v0 + p[:, prefix:] @ v1
    return out


def _exact_sample(c, s):
    tokens, logs = [], []
    for r in range(c["rows"]):
        x = s["logits"][r].double()
        order = torch.argsort(-x, stable=True)
        z = (x[order] - x[order[0]]) / s["temperature"][r].double()
        w = z.exp()
        keep = c["top_k"] or c["vocab"]
        w = w[:keep]
        if c["top_p"] < 1:
            target = torch.tensor(c["top_p"], dtype=torch.float32).double().cuda() * w.sum()
            ahead = torch.cat([torch.zeros(1, dtype=torch.float64, device="cuda"), w.cumsum(0)[:-1]])
            w = w[: max(1, int((ahead < target).sum()))]
        w = w[w >= torch.tensor(c["min_p"], dtype=torch.float32).double().cuda()]
        w = w[w > 0]
        ids, place = torch.sort(order[: len(w)])
        sums = w[place].cumsum(0)
        at = min(int(torch.searchsorted(sums, s["uniform"][r].double() * sums[-1], right=True)), len(w) - 1)
        tokens.append(ids[at])
        logs.append(z[place[at]] - sums[-1].log())
    return {"token": torch.stack(tokens), "logprob": torch.stack(logs)}


def exact(case, seed):
    state = prepare(case, seed)
    return {"norm": _exact_norm, "rotate": _exact_rotate, "prefix": _exact_prefix,
            "sample": _exact_sample}[case["op"]](case, state)

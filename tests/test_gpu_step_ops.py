"""The operators around a decode step's linears and attention against 64-bit implementations: the residual norm with its
8-bit outputs, rotated appends, attention behind a shared prefix, and sampling.

Bounds.  u is half a step of the output type relative to the value (2^-8 bf16, 2^-11 f16, 2^-24 f32, 2^-4 e4m3).
* Norm: h is compared exactly.  y has one output rounding after fp32 work: the sum of squares adds at most (C / 32 + 16)
  roundings of 2^-24 along a term's way (half of that in the root), a product, a root and a division a few more:
  |y - exact| <= (u + (C / 32 + 24) 2^-24) |exact|.  Scales the same without u.  int8 codes are equal; an e4m3 code is
  the rounded quotient, whose fp32 value is off by 4 x 2^-24: a step of the code where that crosses a border.
* Rotation: each of the two products and their sum is fp32, the norm before it as above:
  |y - exact| <= u |exact| + ((D / 32 + 28) 2^-24) (|a| + |b|) for the pair (a, b) turned.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
FP8 = torch.float8_e4m3fn
BOTH = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from comfy_quant_bench_b200 import _lib, ops as _ops
    _lib.load()
    return _ops


@pytest.fixture(scope="module")
def kv(ops):
    from comfy_quant_bench_b200 import kvcache
    return kvcache


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ----------------------------------------------------------------------------------------------------------
# norm
# ----------------------------------------------------------------------------------------------------------

def _norm_problem(m, c, dtype, seed=0):
    g = _gen(seed + 31 * m + c)
    x, r = (3 * torch.randn(m, c, generator=g, device="cuda") for _ in range(2))
    x[:, ::7] *= 10
    return x.to(dtype), r.to(dtype), (1 + 0.3 * torch.randn(c, generator=g, device="cuda")).to(dtype)


def _norm_holds(x, r, w, got, quant, group, eps=1e-6):
    m, c = x.numel() // x.shape[-1], x.shape[-1]
    h = x if r is None else (x.float() + r.float()).to(x.dtype)        # one fp32 sum, one rounding
    assert torch.equal(got[-1], h) and got[-1].dtype == x.dtype
    hd = h.double().reshape(m, c)
    product = hd * w.double()
    root = torch.sqrt(hd.square().mean(-1, keepdim=True) + eps)
    slack = (c / 32 + 24) * 2.0 ** -24
    if not quant:
        y = product / root
        assert got[0].shape == x.shape and got[0].dtype == x.dtype
        over = (got[0].double().reshape(m, c) - y).abs() - (U[x.dtype] + slack) * y.abs()
        assert float(over.max()) <= 2.0 ** -24                         # the spacing of subnormal f16
        return
    top, per = (127.0, 448.0)[quant == "fp8"], group or c
    p = product.view(m, c // per, per)
    most = p.abs().amax(-1, keepdim=True)
    scale = (most.squeeze(-1) / root / top)
    scale = scale.t() if group else scale.view(-1)
    assert got[1].dtype == torch.float32 and got[1].shape == scale.shape
    assert float(((got[1].double() - scale).abs() - slack * scale).max()) <= 2.0 ** -140
    quotient = (p * top / torch.where(most == 0, 1.0, most)).view(m, c)
    assert got[0].shape == x.shape
    if quant == "int8":
        assert got[0].dtype == torch.int8
        assert torch.equal(got[0].view(m, c), quotient.round().to(torch.int8))
    else:
        assert got[0].dtype == FP8
        lo, hi = ((quotient.float() * (1 + s * 4 * 2.0 ** -23)).clamp(-448, 448).to(FP8).float() for s in (-1, 1))
        q = got[0].view(m, c).float()
        assert bool(((q == lo) | (q == hi)).all())


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("m,c", [(1, 8), (3, 256), (9, 264), (2, 520), (17, 1024), (5, 1032), (2, 4096), (3, 4104), (2, 8192),
                                 (1, 8200), (2, 16384), (1, 32768), (1, 1), (5, 7), (3, 255), (7, 1001), (2, 32767)])
@pytest.mark.parametrize("quant", [None, "int8", "fp8"])
def test_norm_widths(ops, m, c, dtype, quant):
    x, r, w = _norm_problem(m, c, dtype)
    _norm_holds(x, r, w, ops.add_rmsnorm(x, w, r, quant=quant), quant, 0)
    got = ops.add_rmsnorm(x, w, quant=quant, eps=1e-5)
    assert got[-1] is x
    _norm_holds(x, None, w, got, quant, 0, 1e-5)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,c", [(1, 128), (13, 384), (300, 1152), (4, 5120), (2, 8320), (1, 24576)])
@pytest.mark.parametrize("quant", ["int8", "fp8"])
def test_norm_groups(ops, m, c, group, dtype, quant):
    x, r, w = _norm_problem(m, c, dtype)
    x[0, :group], r[0, :group] = 0, 0                                   # a group of zeros
    _norm_holds(x, r, w, ops.add_rmsnorm(x, w, r, quant=quant, group_size=group), quant, group)


@pytest.mark.parametrize("dtype", BOTH)
def test_norm_codes_on_borders(ops, dtype):
    """Quotients on and next to the borders between codes: 127 p / P = k + 1/2 where p = (2 k + 1) and P = 254."""
    p = torch.arange(1, 255, device="cuda").float()
    x = torch.cat([p, -p, torch.zeros(4, device="cuda")]).to(dtype).view(1, -1)
    w = torch.ones(x.shape[1], device="cuda").to(dtype)
    _norm_holds(x, None, w, ops.add_rmsnorm(x, w, quant="int8"), "int8", 0)
    near = x.clone()
    near[0, 253] = 254.0 + (2.0 if dtype == torch.bfloat16 else 0.125)   # P a little off: no quotient on a border
    _norm_holds(near, None, w, ops.add_rmsnorm(near, w, quant="int8"), "int8", 0)


def test_norm_extremes(ops):
    t = torch.bfloat16
    w = torch.ones(512, device="cuda", dtype=t)
    x = torch.zeros(5, 512, device="cuda", dtype=t)
    x[1, 3], x[2, 4], x[3] = float("nan"), float("inf"), 2.0 ** -120
    x[4] = 2.0 ** -130                                                  # subnormal
    y, _ = ops.add_rmsnorm(x, w)
    assert not y[0].any() and bool(y[1].isnan().all()) and bool(y[2, 4].isnan()) and not y[2, :4].any()
    for quant in ("int8", "fp8"):
        q, s, _ = ops.add_rmsnorm(x, w, quant=quant)
        assert not q[0].float().any() and s[0] == 0 and bool(s[1].isnan()) and bool(s[2].isnan())
        top = 127 if quant == "int8" else 448
        assert bool((q[3:].float() == top).all())
    empty, h = ops.add_rmsnorm(x[:0], w, x[:0])
    assert empty.shape == (0, 512) and h.shape == (0, 512)


def test_norm_strides_in_place_and_streams(ops):
    x, r, w = _norm_problem(12, 520, torch.float16)
    want = ops.add_rmsnorm(x, w, r)
    wide = torch.zeros(12, 1100, dtype=torch.float16, device="cuda")
    for off in (0, 8, 3):
        wide[:, off:off + 520] = x
        got = ops.add_rmsnorm(wide[:, off:off + 520], w.float(), r)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    every = torch.empty(24, 520, dtype=torch.float16, device="cuda")[::2].copy_(r)
    got = ops.add_rmsnorm(x.view(3, 4, 520), w, every.view(3, 4, 520))
    assert got[0].shape == (3, 4, 520) and torch.equal(got[0].view(12, 520), want[0])
    res = r.clone()
    got = ops.add_rmsnorm(x, w, res, out_residual=res)
    assert got[1] is res or got[1].data_ptr() == res.data_ptr()
    assert torch.equal(res, want[1]) and torch.equal(got[0], want[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.add_rmsnorm(x, w, r, quant="fp8")
    side.synchronize()
    assert torch.equal(got[0].view(torch.uint8), ops.add_rmsnorm(x, w, r, quant="fp8")[0].view(torch.uint8))
    odd = torch.randn(6, 77, device="cuda", dtype=torch.float16)
    buf = torch.zeros(6 * 77 + 1, device="cuda", dtype=torch.float16)[1:].view(6, 77).copy_(odd)   # 2-byte aligned
    assert torch.equal(ops.add_rmsnorm(buf, w[:77], buf)[0], ops.add_rmsnorm(odd, w[:77], odd)[0])


def test_norm_codes_feed_the_int8_gemm(ops):
    x, r, w = _norm_problem(40, 512, torch.bfloat16)
    g = _gen(5)
    qw, sw = ops.quantize_int8_convrot_weight(torch.randn(64, 512, generator=g, device="cuda"), 0)
    q, s, h = ops.add_rmsnorm(x, w, r, quant="int8")
    y = ops.gemm_rowcol(q, s, qw, sw.view(-1), b_int8=True)
    want = (q.double() @ qw.double().t()) * s.double().unsqueeze(1) * sw.double().view(1, -1)
    assert float((y.double() - want).abs().max()) <= 2.0 ** -7 * float(want.abs().max())


# ----------------------------------------------------------------------------------------------------------
# rotary positions and append
# ----------------------------------------------------------------------------------------------------------

def _turn(x, cos, sin, rot, interleaved):
    """x [T, H, D] in 64 bits, turned, and the sum of the magnitudes that each result comes from."""
    x, mag = x.clone(), x.abs()
    i, j = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., i].clone(), x[..., j].clone()
    x[..., i], x[..., j] = a * cos - b * sin, a * sin + b * cos
    mag[..., i] = mag[..., j] = a.abs() + b.abs()
    return x, mag


def _rotate_problem(t, hq, hk, d, rot, dtype, cache, seed=0, page=16, normed=True, far=40):
    g = _gen(seed + 3 * t + d)
    heads = hq + 2 * hk
    qkv = (2 * torch.randn(t, heads, d, generator=g, device="cuda")).to(dtype)
    pages = t + 5
    k, v = (torch.randn(pages, hk, page, d, generator=g, device="cuda").to(cache) for _ in range(2))
    host = torch.Generator().manual_seed(seed)
    pos = torch.randint(0, far, (t,), generator=host)
    table = torch.full((t + 1, -(-far // page)), -1, dtype=torch.int32)
    order = torch.randperm(pages, generator=host)
    rows = torch.randperm(t + 1, generator=host)[:t]
    for n in range(t):
        table[rows[n], pos[n] // page] = order[n]
    w = [(1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dtype) if normed else None for _ in range(2)]
    scales = [0.02 + 0.02 * torch.rand(hk, generator=g, device="cuda") if cache == FP8 else None for _ in range(2)]
    return qkv, k, v, table.cuda(), rows.int().cuda(), pos.int().cuda(), w, scales


def _rotate_holds(kv, problem, hq, hk, rot, interleaved, rope):
    qkv, k, v, table, rows, pos, w, scales = problem
    d, page, dtype, cache = qkv.shape[2], k.shape[2], qkv.dtype, k.dtype
    k0, v0 = k.clone(), v.clone()
    q_new, k_new, v_new = qkv.split((hq, hk, hk), dim=1)
    got, got_k = kv.append_rotated(q_new, k_new, v_new, k, v, table, rows, pos, rope, interleaved=interleaved, q_norm=w[0],
                                   k_norm=w[1], k_scale=scales[0], v_scale=scales[1], return_k=True)
    at = pos.long().clamp(min=0)
    cos, sin = rope.double()[at].unsqueeze(1).unbind(-1)
    slack = (d / 32 + 28) * 2.0 ** -24
    want = []
    for x, weight in ((q_new, w[0]), (k_new, w[1])):
        x = x.double()
        if weight is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.double()
        want.append(_turn(x, cos, sin, rot, interleaved))
    for g, (y, mag) in zip((got, got_k), want):
        assert g.dtype == dtype and g.shape == y.shape and g.is_contiguous()
        assert float(((g.double() - y).abs() - U[dtype] * y.abs() - slack * mag).max()) <= 2.0 ** -25
    placed = [n for n in range(len(pos)) if pos[n] >= 0 and pos[n] // page < table.shape[1] and 0 <= rows[n] < len(table) and
              0 <= table[rows[n], pos[n] // page] < len(k)]
    for c, c0, new, scale in ((k, k0, want[1], scales[0]), (v, v0, (v_new.double(), None), scales[1])):
        c, c0 = c.float(), c0.float()
        for n in placed:
            p, slot = int(table[rows[n], pos[n] // page]), int(pos[n]) % page
            y = new[0][n] if scale is None else (new[0][n] / scale.double().view(-1, 1)).clamp(-448, 448)
            m = y.abs() if new[1] is None else new[1][n] if scale is None else new[1][n] / scale.double().view(-1, 1)
            u = U[dtype] if scale is None else 2.0 ** -4
            tiny = 2.0 ** -25 if scale is None else 2.0 ** -10         # half the spacing of subnormal values
            assert float(((c[p, :, slot].double() - y).abs() - u * y.abs() - (slack + 2.0 ** -23) * m).max()) <= tiny
            c0[p, :, slot] = c[p, :, slot]
        assert torch.equal(c, c0)                                      # and nothing else was written


@pytest.mark.parametrize("cache", ["own", "fp8"])
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t,hq,hk,d,rot", [(1, 1, 1, 16, 16), (1, 16, 2, 128, 128), (3, 7, 1, 64, 32), (40, 32, 8, 128, 64),
                                           (5, 6, 3, 80, 80), (300, 3, 1, 96, 48), (2, 20, 4, 256, 256), (9, 64, 8, 256, 64),
                                           (4, 5, 5, 24, 16), (310, 12, 4, 128, 128)])
def test_rotated_append(kv, t, hq, hk, d, rot, interleaved, dtype, cache):
    rope = kv.rope_table(64, rot)
    for normed in (False, True):
        problem = _rotate_problem(t, hq, hk, d, rot, dtype, FP8 if cache == "fp8" else dtype, normed=normed)
        _rotate_holds(kv, problem, hq, hk, rot, interleaved, rope)


def test_rotated_append_far_positions_scaled(kv):
    rope = kv.rope_table(130000, 128, base=500000.0, scaling="parts", factor=8.0, original=8192)
    problem = list(_rotate_problem(6, 4, 2, 128, 128, torch.bfloat16, torch.bfloat16, far=129999))
    _rotate_holds(kv, problem, 4, 2, 128, False, rope)


def test_rotated_append_tokens_without_a_place(kv):
    from comfy_quant_bench_b200 import _lib
    rope = kv.rope_table(64, 64)
    problem = _rotate_problem(8, 4, 2, 64, 64, torch.float16, torch.float16)
    qkv, k, v, table, rows, pos, w, scales = problem
    pos[0], pos[1], pos[2] = -1, 63, -7                                # refused, beyond the table, refused
    rows[3], rows[4] = -1, len(table)
    table[rows[5].long(), pos[5].long() // 16] = -1
    table[rows[6].long(), pos[6].long() // 16] = len(k)
    _rotate_holds(kv, problem, 4, 2, 64, False, rope)
    kv.check()
    pos[0] = 64                                                        # no angle
    before = k.clone()
    q, k_new, v_new = qkv.split((4, 2, 2), dim=1)
    got = kv.append_rotated(q[:1], k_new[:1], v_new[:1], k, v, table, rows[:1], pos[:1], rope[:, :16].contiguous())
    assert bool(got[..., :32].isnan().all()) and torch.equal(got[..., 32:], q[:1, :, 32:]) and torch.equal(k, before)
    with pytest.raises(_lib.CQError, match="append_rotated"):
        kv.check()
    none = kv.append_rotated(q[:0], k_new[:0], v_new[:0], k, v, table, rows[:0], pos[:0], rope)
    assert none.shape == (0, 4, 64)


def test_rotated_append_strides_special_values_and_streams(kv):
    rope = kv.rope_table(64, 64)
    problem = _rotate_problem(12, 4, 2, 64, 64, torch.bfloat16, torch.bfloat16, normed=False)
    qkv, k, v, table, rows, pos, w, scales = problem
    q, k_new, v_new = qkv.split((4, 2, 2), dim=1)
    want = kv.append_rotated(q, k_new, v_new, k, v, table, rows, pos, rope)
    kc, vc = k.clone(), v.clone()
    k.zero_(), v.zero_()
    odd = torch.zeros(12, 4, 65, device="cuda", dtype=torch.bfloat16)[..., 1:].copy_(q)    # not aligned: copied
    expanded = table.t().contiguous().t()                                                  # a table of other strides
    with pytest.raises(ValueError, match="contiguous"):
        kv.append_rotated(odd, k_new, v_new, k, v, expanded, rows, pos, rope)
    got = kv.append_rotated(odd, k_new.contiguous(), v_new.transpose(0, 1).contiguous().transpose(0, 1), k, v, table, rows, pos, rope)
    assert torch.equal(got, want)
    touched = kc != 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = kv.append_rotated(q, k_new, v_new, k, v, table, rows, pos, rope)
    side.synchronize()
    assert torch.equal(again, want)
    for n in range(12):
        p, slot = int(table[rows[n], pos[n] // 16]), int(pos[n]) % 16
        assert torch.equal(k[p, :, slot], kc[p, :, slot]) and torch.equal(v[p, :, slot], vc[p, :, slot])
    assert int((k != 0).any(-1).sum()) <= 12 * 2 and touched.any()
    # values that are not finite stay in their pair
    bad = q.clone()
    bad[0, 0, 3] = float("inf")
    bad[1, 1, 40] = float("nan")
    got = kv.append_rotated(bad, k_new, v_new, k, v, table, rows, pos, rope)
    off = got != want
    assert {tuple(i) for i in off.nonzero().tolist()} <= {(0, 0, 3), (0, 0, 35), (1, 1, 8), (1, 1, 40)}
    assert bool(got[1, 1, 40].isnan()) and not bool(got[0, 0, 3].isfinite())


# ----------------------------------------------------------------------------------------------------------
# sampling: tokens are compared exactly.  Weights are rounded at 2^-45 of the largest, so the shares of a test's choice are
# off by n 2^-45 at most; numbers that near to a border (or shares that near to top-p's or min-p's) are not drawn but
# built to be exact.  log of a share: 2^-24 relative, and n 2^-44 of the share.
# ----------------------------------------------------------------------------------------------------------

def _chosen(x, u, t, k, p, m):
    """One row in 64 bits: (token, logprob)."""
    x = x.double()
    x = torch.where(x.isnan(), float("-inf"), x)
    top = x.max()
    if top == float("-inf"):
        return -1, float("-inf")
    if not t > 0:
        return int((x == top).nonzero()[0]), 0.0
    z = torch.where(x == top, 0.0, (x - top) / t)
    order = torch.sort(x, descending=True, stable=True).indices
    w = z.exp()[order]
    w = w[: k if k else len(w)]
    if p < 1:
        before = w.cumsum(0) - w
        w = w[: max(1, int((before < p * w.sum()).sum()))]
    w = w[w >= m]
    ids, place = torch.sort(order[: len(w)])
    sums = w[place].cumsum(0)
    live = (w[place] > 0).nonzero()
    at = min(int((sums <= u * sums[-1]).sum()), int(live[-1]))
    return int(ids[at]), float(z[ids[at]] - sums[-1].log())


def _sample_holds(ops, x, u, t=1.0, k=0, p=1.0, m=0.0):
    tokens, logs = ops.sample_tokens(x, u, temperature=t, top_k=k, top_p=p, min_p=m, return_logprob=True)
    assert tokens.dtype == torch.int64 and logs.dtype == torch.float32
    row = lambda v, r, f: float(v[r]) if isinstance(v, torch.Tensor) else float(torch.tensor(v, dtype=torch.float32)) if f else v  # noqa: E731
    for r in range(len(x)):
        want, log = _chosen(x[r], float(u[r]), row(t, r, True), int(row(k, r, False)), row(p, r, True), row(m, r, True))
        assert int(tokens[r]) == want, (r, int(tokens[r]), want)
        if want < 0 or math.isinf(log):
            assert float(logs[r]) == log
        else:
            assert abs(float(logs[r]) - log) <= 2.0 ** -23 * abs(log) + x.shape[1] * 2.0 ** -44 / math.exp(log)
    return tokens


def _logits(rows, vocab, dtype, seed=0, scale=2.5):
    g = _gen(seed + vocab)
    x = scale * torch.randn(rows, vocab, generator=g, device="cuda")
    x[:, ::5] = float("-inf")
    x[:, 0] = 0.5
    return x.to(dtype), torch.rand(rows, generator=g, device="cuda")


@pytest.mark.parametrize("dtype", [*BOTH, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 33, 500, 2047, 2049, 4100, 32000, 50257, 131073])
@pytest.mark.parametrize("k,p,m", [(0, 1.0, 0.0), (0, 0.9, 0.0), (40, 1.0, 0.0), (50, 0.8, 0.05), (0, 0.3, 0.2), (1, 0.5, 0.0),
                                   (0, 0.999, 0.0), (3000, 0.97, 0.0), (0, 1.0, 0.1), (0, 0.0, 0.0), (7, 1.0, 1.0)])
def test_sample(ops, vocab, dtype, k, p, m):
    x, u = _logits(6, vocab, dtype, seed=k)
    _sample_holds(ops, x, u, 0.8, k, p, m)


@pytest.mark.parametrize("scale,t", [(0.01, 1.0), (30.0, 1.0), (1.0, 0.01), (1.0, 50.0), (1.0, 1e6), (1e4, 1e4)])
def test_sample_flat_and_peaked(ops, scale, t):
    for vocab in (300, 40000):
        x, u = _logits(8, vocab, torch.float32, scale=scale)
        for k, p in ((0, 1.0), (0, 0.9), (100, 0.7), (0, 0.5)):
            _sample_holds(ops, x, u, t, k, p, 0.0)


@pytest.mark.parametrize("vocab", [64, 5000, 100001])
def test_sample_equal_logits(ops, vocab):
    """More equal logits than a border is ranked for: lowest indexes first; every border exact."""
    x = torch.full((5, vocab), -3.0, device="cuda")
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24], device="cuda")
    for k, p in ((0, 1.0), (0, 0.5), (vocab // 2, 1.0), (vocab // 4, 0.5), (17, 1.0), (0, 0.25)):
        for t in (1.0, 0.3):
            _sample_holds(ops, x, u, t, k, p, 0.0)
    x[:, ::2] = -3.0 - 1.0 / 128                                       # two values in one bin
    x[:, 7] = 30.0
    _sample_holds(ops, x, u, 40.0, vocab // 2 + 3, 1.0, 0.0)
    x = torch.where(torch.arange(vocab, device="cuda") % 2 == 0, 0.0, -0.0).expand(5, -1).contiguous()
    _sample_holds(ops, x, u, 1.0, 5, 1.0, 0.0)


def test_sample_rows_of_their_own_parameters(ops):
    n = 300
    x, u = _logits(n, 3001, torch.bfloat16)
    g = _gen(3)
    t = 0.3 + torch.rand(n, generator=g, device="cuda")
    t[::10] = 0.0
    k = torch.randint(0, 400, (n,), generator=g, device="cuda", dtype=torch.int32)
    k[::7] = 0
    p = torch.rand(n, generator=g, device="cuda")
    p[::5] = 1.0
    m = 0.3 * torch.rand(n, generator=g, device="cuda")
    m[::3] = 0.0
    tokens = _sample_holds(ops, x, u, t, k, p, m)
    for _ in range(3):
        assert torch.equal(ops.sample_tokens(x, u, temperature=t, top_k=k, top_p=p, min_p=m), tokens)


def test_sample_special_logits(ops):
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    x = torch.full((8, 4000), -inf, device="cuda")
    x[1, 3999] = -7.0                                                  # one token
    x[2, 100:200] = nan
    x[2, 150] = 1.0
    x[3, ::3], x[3, 4] = 0.0, inf                                      # one at infinity takes the row
    x[4, 9], x[4, 3000] = inf, inf
    x[5] = low                                                         # masked by the type's lowest value
    x[5, 77], x[5, 78] = 2.0, 1.0
    x[6] = nan
    x[7] = low                                                         # nothing but masked: all alike
    u = torch.full((8,), 0.6, device="cuda")
    for k, p, m in ((0, 1.0, 0.0), (2, 0.9, 0.0), (0, 0.5, 0.0), (500, 1.0, 0.5)):
        for t in (1.0, 0.0, 3.0):
            tokens = _sample_holds(ops, x, u, t, k, p, m)
            assert tokens[0] == -1 and tokens[6] == -1 and tokens[1] == 3999
    for dtype in BOTH:
        y = torch.full((3, 600), torch.finfo(dtype).min, dtype=dtype, device="cuda")
        y[1, 5], y[2, 6], y[2, 7] = 3.0, torch.finfo(dtype).max, torch.finfo(dtype).max
        for k, p in ((0, 1.0), (3, 0.9), (0, 0.7)):
            _sample_holds(ops, y, u[:3], 0.7, k, p, 0.0)


def test_sample_numbers_at_the_ends(ops):
    x = torch.tensor([[-1.0, 2.0, 2.0, -60.0]], device="cuda").expand(6, -1).contiguous()
    u = torch.tensor([0.0, -1.0, float("nan"), 1.0, 7.0, float("inf")], device="cuda")
    assert ops.sample_tokens(x, u, top_k=2).tolist() == [1, 1, 1, 2, 2, 2]
    assert ops.sample_tokens(x, u).tolist() == [0, 0, 0, 2, 2, 2]      # a weight of e^-62 cannot be chosen


def test_sample_strides_streams_and_graphs(ops):
    x, u = _logits(9, 7000, torch.float16)
    want = _sample_holds(ops, x, u, 1.0, 0, 0.9, 0.0)
    wide = torch.full((9, 7100), 60000.0, device="cuda", dtype=torch.float16)
    for off in (0, 1, 3, 8, 99):                                       # rows at every alignment; neighbours are not read
        wide.fill_(60000.0)
        wide[:, off:off + 7000] = x
        assert torch.equal(ops.sample_tokens(wide[:, off:off + 7000], u, top_p=0.9), want)
    assert torch.equal(ops.sample_tokens(x.t().contiguous().t(), u, top_p=0.9), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.sample_tokens(x, u, top_p=0.9)
    side.synchronize()
    assert torch.equal(got, want)
    assert ops.sample_tokens(x[:0], u[:0]).shape == (0,)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, logs = ops.sample_tokens(x, u, top_p=0.9, return_logprob=True)
    u.copy_(1 - u)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, ops.sample_tokens(x, u, top_p=0.9))
    assert bool((logs <= 0).all())

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
import decimal
import fractions
import math
import random

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


# ----------------------------------------------------------------------------------------------------------
# attention behind a shared prefix.  A score's fp32 error is at most err = (D + 16) 2^-23 scale sum |q| |k|; it and the
# exponential (2^-20) enter numerator and denominator; a weight in two 16-bit parts is held to 2^-16 (2^-14 for its share of
# the sums as elsewhere), in one part to u; f16 parts to 2^-32 of the running maximum beside that:
# |o - exact| <= u |exact| + A (2 max err + 2^-14 [+ u]) + n 2^-32 max |v|, A = sum p |v| / sum p.
# ----------------------------------------------------------------------------------------------------------

def _wide(table, hk, d, page, size):
    """The table with columns of no pages, so many that the call shares the prefix however few tokens the rows hold."""
    width = -(-((1 << 27) + 1) // (len(table) * hk * d * 2 * size * page))
    return torch.cat([table, table.new_full((len(table), max(0, width - table.shape[1])), -1)], dim=1)


def _prefix_problem(lens, prefix, hq, hk, d, page, dtype, cache, seed=0, holes=True, wide=True):
    """Rows of lens tokens; those with at least `prefix` of them share the first ones: whole pages, the last in copies."""
    g = _gen(seed + d + prefix)
    host = torch.Generator().manual_seed(seed)
    b = len(lens)
    width = max(1, -(-max(max(lens), 1) // page))
    whole = prefix // page
    joined = [n >= prefix for n in lens]
    need = [max(0, -(-n // page) - (whole if j else 0)) for n, j in zip(lens, joined)]
    pages = whole + sum(need) + 3
    order = torch.randperm(pages, generator=host).int()
    table = torch.full((b, width), -1, dtype=torch.int32)
    used = whole
    for r in range(b):
        skip = whole if joined[r] else 0
        table[r, :skip] = order[:skip]
        table[r, skip: skip + need[r]] = order[used: used + need[r]]
        used += need[r]
    shape = (pages, hk, page, d)
    k, v = (torch.randn(shape, generator=g, device="cuda") for _ in range(2))
    scales = [None, None]
    if cache == FP8:
        k, v = k * 40, v * 40
        scales = [0.02 + 0.02 * torch.rand(hk, generator=g, device="cuda") for _ in range(2)]
    k, v = k.to(cache), v.to(cache)
    first = next((r for r in range(b) if joined[r]), None)
    for c in (k, v):
        raw = c.view(torch.uint8) if cache == FP8 else c
        if prefix % page and first is not None:
            src = int(table[first, whole])
            for r in range(b):
                if joined[r]:
                    raw[int(table[r, whole]), :, : prefix % page] = raw[src, :, : prefix % page].clone()
        if holes:
            nan = torch.tensor(float("nan"), device="cuda").to(cache)
            nan = nan.view(torch.uint8) if cache == FP8 else nan
            for r, n in enumerate(lens):
                if n % page:
                    raw[int(table[r, n // page]), :, n % page:] = nan
    q = (1.5 * torch.randn(b, hq, d, generator=g, device="cuda")).to(dtype)
    if wide:
        table = _wide(table, hk, d, page, k.element_size())
    return q, k, v, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), scales


def _prefix_exact(q, k, v, table, lens, scales, scale=None, rows=None):
    b, hq, d = q.shape
    hk, page = k.shape[1], k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    out, lse = torch.zeros(b, hq, d, dtype=torch.float64, device="cuda"), torch.full((b, hq), -math.inf, dtype=torch.float64, device="cuda")
    slack = torch.zeros_like(out)
    tail = torch.zeros(b, hq, 1, dtype=torch.float64, device="cuda")
    for i in range(b):
        r = i if rows is None else int(rows[i])
        n = int(lens[r]) if 0 <= r < len(lens) else 0
        at = torch.arange(n, device="cuda")
        pages = table[r].long()[at // page] if n else at
        at, pages = at[(pages >= 0) & (pages < len(k))], pages[(pages >= 0) & (pages < len(k))]
        if not len(at):
            continue
        take = lambda c: (c.view(torch.uint8)[pages, :, at % page].view(FP8) if c.dtype == FP8 else c[pages, :, at % page]).double()  # noqa: E731
        kk, vv = take(k), take(v)
        if scales[0] is not None:
            kk, vv = kk * scales[0].double().view(-1, 1), vv * scales[1].double().view(-1, 1)
        kk, vv = (x.repeat_interleave(hq // hk, 1).transpose(0, 1) for x in (kk, vv))          # [hq, n, d]
        qq = q[i].double().unsqueeze(1)
        s = (qq @ kk.transpose(1, 2)).squeeze(1) * scale
        err = (d + 16) * 2.0 ** -23 * abs(scale) * (qq.abs() @ kk.abs().transpose(1, 2)).squeeze(1).amax(-1)
        p = torch.softmax(s, -1)
        out[i], lse[i] = (p.unsqueeze(1) @ vv).squeeze(1), torch.logsumexp(s, -1)
        slack[i] = (p.unsqueeze(1) @ vv.abs()).squeeze(1) * (2 * err + 2.0 ** -14).unsqueeze(-1)
        tail[i] = n * 2.0 ** -32 * vv.abs().amax()
        err_lse = err + 2.0 ** -19
        assert bool((err_lse < 0.1).all())
    share = slack / 2.0 ** -14                                          # at least A
    return out, lse, slack, share, tail


def _prefix_holds(kv, problem, prefix, rows=None, scale=None, **kw):
    q, k, v, table, lens, scales = problem
    got, lse = kv.prefix_attention(q, k, v, table, lens, prefix, rows=rows, scale=scale, k_scale=scales[0], v_scale=scales[1],
                                   return_lse=True, **kw)
    want, want_lse, slack, share, tail = _prefix_exact(q, k, v, table, lens, scales, scale, rows)
    b, hq, d = q.shape
    one_part = b * (hq // k.shape[1]) > (128 if d == 256 else 256)
    u = U[q.dtype]
    assert got.dtype == q.dtype and got.shape == q.shape
    bound = u * want.abs() + slack * (1 + u) + (u * share if one_part else 0) + tail + 2.0 ** -25
    over = ((got.double() - want).abs() - bound).max()
    assert float(over) <= 0, float(over)
    seen = ~torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), ~seen)
    assert float((lse.double() - want_lse)[seen].abs().max() if seen.any() else 0.0) <= 2.0 ** -12
    if want.numel() > 4000 and float(want.norm()) > 0:
        once = float((want.to(q.dtype).double() - want).norm() / want.norm())
        assert float((got.double() - want).norm() / want.norm()) <= (1.5 if one_part else 1.05) * once + 2.0 ** -14
    return got


@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                         (torch.bfloat16, FP8), (torch.float16, FP8)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("b,hq,hk,prefix,longest,page", [(1, 1, 1, 1, 1, 16), (2, 4, 1, 5, 3, 8), (4, 16, 2, 500, 60, 16),
                                                         (3, 6, 3, 127, 40, 16), (3, 6, 3, 128, 0, 32), (5, 8, 4, 129, 200, 64),
                                                         (40, 8, 2, 700, 30, 16), (33, 8, 1, 1111, 90, 16), (65, 12, 3, 300, 17, 128),
                                                         (20, 56, 2, 2050, 5, 16), (70, 16, 1, 640, 9, 16), (2, 8, 8, 6000, 100, 16)])
def test_prefix(kv, b, hq, hk, prefix, longest, page, d, dtype, cache):
    lens = [prefix + (longest * i) // max(1, b - 1) for i in range(b)]
    problem = _prefix_problem(lens, prefix, hq, hk, d, page, dtype, cache, wide=False)
    _prefix_holds(kv, problem, prefix)                                  # every row by itself
    problem = _prefix_problem(lens, prefix, hq, hk, d, page, dtype, cache)
    _prefix_holds(kv, problem, prefix)
    _prefix_holds(kv, problem, torch.tensor([prefix], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("b,hq,hk", [(6, 8, 2), (50, 16, 2)])
def test_prefix_of_uneven_rows(kv, b, hq, hk, d):
    """Rows without the prefix, rows of nothing, prefixes of nothing and beyond every row."""
    lens = [0, 400, 350, 3, 700, 349] + [350 + 7 * i for i in range(b - 6)]
    problem = _prefix_problem(lens, 350, hq, hk, d, 16, torch.bfloat16, torch.bfloat16)
    q, k, v, table, n, scales = problem
    for prefix in (350, 349, 200, 17, 1, 0, 100000):
        if prefix >= 350 or prefix == 0:
            _prefix_holds(kv, problem, prefix)
    lens = [260 + 7 * i for i in range(b)]
    problem = _prefix_problem(lens, 260, hq, hk, d, 16, torch.bfloat16, torch.bfloat16)
    for prefix in (260, 259, 128, 1):                                   # any shorter prefix is shared too
        _prefix_holds(kv, problem, prefix)
    rows = torch.arange(b, device="cuda", dtype=torch.int32).flip(0)
    rows[1], rows[2], rows[3] = -1, b, rows[0]                          # no row, beyond the table, the same row twice
    _prefix_holds(kv, problem, 260, rows=rows)
    _prefix_holds(kv, problem, 260, scale=-0.02)
    # a page that the table does not have, inside the prefix
    holed = problem[3].clone()
    holed[:, 3], holed[:, 9] = -1, len(problem[1])
    _prefix_holds(kv, (*problem[:3], holed, *problem[4:]), 260)


def test_prefix_agrees_with_one_row_at_a_time_and_again(kv):
    problem = _prefix_problem([900 + i for i in range(48)], 900, 32, 8, 128, 16, torch.float16, torch.float16)
    q, k, v, table, lens, _ = problem
    got = _prefix_holds(kv, problem, 900)
    plain = kv.paged_attention(q, k, v, table, lens)
    assert float((got.double() - plain.double()).norm() / plain.double().norm()) <= 2.0 ** -11
    for _ in range(4):
        assert torch.equal(kv.prefix_attention(q, k, v, table, lens, 900), got)


def test_prefix_large_scores(kv):
    """Maxima that grow from tile to tile, one key that outweighs the rest, infinities and NaN in sight."""
    lens = [1500 + i for i in range(20)]
    for d in (64, 128, 256):
        problem = _prefix_problem(lens, 1500, 8, 2, d, 16, torch.float16, torch.float16)
        q, k, v, table, n, scales = problem
        for j in range(1500):                                           # keys grow along the prefix
            if j % 16 == 0:
                k[int(table[0, j // 16])] *= 0.2 + 4 * j / 1500
        if 1500 % 16:
            src = int(table[0, 93])
            for r in range(1, 20):
                k[int(table[r, 93]), :, :12] = k[src, :, :12]
        want, lse, slack, share, tail = _prefix_exact(*problem[:5], scales)
        got = kv.prefix_attention(q, k, v, table, n, 1500)
        assert float(((got.double() - want).abs() - U[torch.float16] * want.abs() - slack * 1.01 - tail - 2.0 ** -25).max()) <= 0
        bad = v.clone()
        bad[int(table[0, 5]), 0, 3, 7] = float("inf")
        bad[int(table[0, 6]), 1, 4, 9] = float("nan")
        got = kv.prefix_attention(q, k, bad, table, n, 1500)
        off = ~torch.isfinite(got)
        assert bool(off[:, :4, 7].all()) and bool(off[:, 4:, 9].all()) and int(off.sum()) == 20 * 8
        worse = k.clone()
        worse[int(table[0, 5]), 0, 3] = float("nan")
        got = kv.prefix_attention(q, worse, v, table, n, 1500)
        assert bool(got[:, :4].isnan().all()) and bool(torch.isfinite(got[:, 4:]).all())


def test_prefix_strides_streams_graphs_and_workspaces(kv):
    b, prefix = 12, 333
    lens = [prefix + 5 * i for i in range(b)]
    problem = _prefix_problem(lens, prefix, 8, 2, 64, 16, torch.bfloat16, torch.bfloat16)
    q, k, v, table, n, scales = problem
    want = _prefix_holds(kv, problem, prefix)
    wide = torch.zeros(b, 11, 64, device="cuda", dtype=q.dtype)
    wide[:, 1:9] = q
    out = torch.full_like(q, 7.0)
    assert kv.prefix_attention(wide[:, 1:9], k, v, table, n, prefix, out=out) is out and torch.equal(out, want)
    head_last = k.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)  # [pages, page, heads, d] in memory
    value_last = v.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    assert torch.equal(kv.prefix_attention(q, head_last, value_last, table, n, prefix), want)
    odd = torch.zeros(b, 8, 65, device="cuda", dtype=q.dtype)[..., 1:].copy_(q)
    assert torch.equal(kv.prefix_attention(odd, k, v, table, n, prefix), want)
    # two graphs and an eager call on two streams, each with its own workspace
    shared = torch.tensor([prefix], dtype=torch.int32, device="cuda")
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = kv.prefix_attention(q, k, v, table, n, shared)
        graphs.append((graph, held))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
            mine = kv.prefix_attention(q, k, v, table, n, prefix)
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want) and torch.equal(mine, want)
    shared.fill_(200)                                                   # a captured step reads the prefix anew
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], kv.prefix_attention(q, k, v, table, n, 200))
    empty = kv.prefix_attention(q[:0], k, v, table, n, prefix)
    assert empty.shape == (0, 8, 64)
    assert _status() == (0, 0)


def test_prefix_offsets_past_32_bits(kv):
    """Pages more than 2^32 bytes into a cache."""
    pages, page, hk, d = 140_000, 16, 8, 128                            # 4.6 GB each
    k = torch.zeros(pages, hk, page, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    g = _gen(11)
    ids = torch.tensor([pages - 1 - 5 * i for i in range(40)], dtype=torch.int32)
    for p in ids.tolist():
        k[p], v[p] = (torch.randn(hk, page, d, generator=g, device="cuda").bfloat16() for _ in range(2))
    table = torch.full((3, 24), -1, dtype=torch.int32)
    table[:, :20] = ids[:20]
    for r in range(3):
        table[r, 20:24] = ids[20 + 4 * r: 24 + 4 * r]
    lens = torch.tensor([330, 384, 321], dtype=torch.int32, device="cuda")
    q = torch.randn(3, 16, d, generator=g, device="cuda").bfloat16()
    table = _wide(table, hk, d, page, 2)
    _prefix_holds(kv, (q, k, v, table.cuda(), lens, [None, None]), 320)


def _status():
    from comfy_quant_bench_b200 import _lib
    torch.cuda.synchronize()
    return _lib.take_device_status()


# ----------------------------------------------------------------------------------------------------------
# the operators together, in the small language model of ``textgen``.  Both ways of attending a shared prompt lie within the
# bound that test_gpu_textgen derives for a model's logits (2.3e-2 of relative L2 for two blocks), so they differ by twice it.
# ----------------------------------------------------------------------------------------------------------

def _model(**kw):
    from comfy_quant_bench_b200 import textgen
    base = dict(vocab=500, hidden=256, layers=2, heads=8, kv_heads=2, head_dim=64, ffn=512, group_size=64, max_tokens=160, rows=6,
                pages=80, page_size=16)
    return textgen.TextModel(textgen.TextConfig(**{**base, **kw}))


@pytest.mark.parametrize("kw", [{}, {"max_tokens": 70000}, {"max_tokens": 70000, "window": 24, "sinks": 3}])
def test_steps_behind_a_shared_prompt(kv, kw):
    """Rows forked from one prompt; with room for 70000 tokens a row its tokens are attended once for all rows."""
    g = _gen(5)
    prompt, tokens = torch.randint(0, 500, (37,), generator=g, device="cuda"), torch.randint(0, 500, (12, 5), generator=g, device="cuda")
    models = [_model(**kw) for _ in range(3)]
    rows = torch.arange(1, 6, dtype=torch.int32, device="cuda")
    for m in models:
        m.prompt(prompt, 0)
        m.cache.branch(torch.zeros_like(rows), rows, 0)
    shared = torch.tensor([37], dtype=torch.int32, device="cuda")
    fill, graph, held = models[2].capture(rows, shared)
    for i in range(12):
        alone, together = models[0].step(tokens[i], rows), models[1].step(tokens[i], rows, None, 37)
        assert float((alone.float() - together.float()).norm() / alone.float().norm()) <= 4.6e-2
        fill.copy_(tokens[i])
        graph.replay()
        assert torch.equal(held, together)
    for m in models:
        m.cache.check()
    assert _status() == (0, 0)


def test_generate_with_filters(ops):
    m = _model()
    prompt = torch.arange(33, device="cuda")
    u = torch.rand(10, 3, generator=_gen(1), device="cuda")
    greedy = m.generate(prompt, 3, 10)
    assert torch.equal(m.generate(prompt, 3, 10, u, top_k=1), greedy)
    assert torch.equal(m.generate(prompt, 3, 10, u, temperature=0.0), greedy)
    assert torch.equal(m.generate(prompt, 3, 10, u, min_p=1.0), greedy)
    some = m.generate(prompt, 3, 10, u, temperature=0.7, top_k=50, top_p=0.9, min_p=0.01)
    assert some.shape == (3, 10) and torch.equal(m.generate(prompt, 3, 10, u, temperature=0.7, top_k=50, top_p=0.9, min_p=0.01), some)


def test_a_long_context_model_steps(ops):
    m = _model(rope_scaling="parts", rope_factor=4.0, rope_original=40, cache_dtype=FP8)
    logits = m.prompt(torch.arange(100, device="cuda"), 0)
    step = m.step(torch.tensor([3], device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert bool(torch.isfinite(logits).all()) and bool(torch.isfinite(step).all())
    m.cache.check()


@pytest.mark.parametrize("t", [2.0 ** -149, 1e-44, 1e-40, 4e-39, 5e-39, 2.0 ** -126, 1e-37, 3e-37, 6.6e-37, 7e-37, 1e-36, 1e-30])
@pytest.mark.parametrize("vocab", [9, 700, 5000])
def test_sample_temperatures_next_to_nothing(ops, vocab, t):
    """Temperatures down to the smallest subnormal: the definition holds, for logits that differ by far more than the
    temperature (the largest, or those equal to it, share the row) and for some that differ by a few times it."""
    t = float(torch.tensor(t, dtype=torch.float32))
    x, u = _logits(6, vocab, torch.float32)
    x[1, 3::4] = x[1].max() + 1                                        # several at the maximum
    x[2] = -7.0                                                        # all of them
    g = torch.Generator().manual_seed(vocab)
    fine = torch.randn(6, vocab, generator=g, dtype=torch.float64) * 6 * t
    fine = torch.round(fine * 2.0 ** 149) * 2.0 ** -149                # multiples of the smallest number: f32 holds them
    for logits in (x, fine.float().cuda()):
        for k, p, m in ((0, 1.0, 0.0), (0, 0.9, 0.0), (0, 0.4, 0.05), (4, 1.0, 0.0), (5, 0.7, 0.0), (vocab - 1, 0.95, 0.0), (0, 0.0, 0.0)):
            tokens = _sample_holds(ops, logits, u, t, k, p, m)
            each = torch.full((6,), t, device="cuda")
            assert torch.equal(ops.sample_tokens(logits, u, temperature=each, top_k=k, top_p=p, min_p=m), tokens)


def _weights_next_to_a_choice(n):
    """[(logit, temperature, u, token)] of two tokens, the first with a logit below 0, the second with 0.  With w the first
    one's weight and W = round(2^44 w) it is chosen where W exceeds u (W + 2^44), that is where W > 2^44 u / (1 - u).  The
    quotient of logit and temperature, a fraction of two integers below 2^24, puts W next to that border, on one of its
    sides: a weight that is off by one unit more than its rounding is chosen wrongly."""
    decimal.getcontext().prec = 50
    rng, one, cases = random.Random(1), decimal.Decimal(2) ** 44, []
    while len(cases) < n:
        share = 2.0 ** (-(2 * rng.randrange(40) + 1 + rng.uniform(-0.06, 0.06)) / 128)    # halfway between table entries
        u = math.floor(share / (1 + share) * 2 ** 25) / 2 ** 25                           # an f32
        border = decimal.Decimal(u) / (1 - decimal.Decimal(u)) * one
        aim = math.floor(border) + rng.randrange(2) + decimal.Decimal(rng.uniform(-0.3, 0.3))
        x = fractions.Fraction(-(aim / one).ln()).limit_denominator((1 << 24) - 1)
        exact = one * (decimal.Decimal(-x.numerator) / decimal.Decimal(x.denominator)).exp()
        held = int(exact.to_integral_value())
        if x.numerator < 1 << 24 and abs(exact - held) <= decimal.Decimal("0.45") and decimal.Decimal("0.01") <= abs(held - border) <= 1:
            cases.append((-x.numerator * 2.0 ** -24, x.denominator * 2.0 ** -24, u, 0 if held > border else 1))
    return cases


def test_sample_weights_are_right_to_their_rounding(ops):
    cases = _weights_next_to_a_choice(600)
    x, t, u, want = (torch.tensor(c) for c in zip(*cases))
    assert 200 < int(want.sum()) < 400
    logits = torch.stack([x, torch.zeros_like(x)], dim=1).cuda()
    for width in (2, 3000):                                            # alone, and where eight CTAs hold the row
        row = torch.full((len(cases), width), float("-inf"), device="cuda")
        row[:, 0], row[:, -1] = logits[:, 0], logits[:, 1]
        for p in (1.0, 0.999):
            got = ops.sample_tokens(row, u.cuda(), temperature=t.cuda(), top_p=p)
            assert torch.equal((got > 0).long().cpu(), want), (width, p, int(((got > 0).long().cpu() != want).sum()))


def _nearest_e4m3(q):
    """The e4m3 value nearest to q (64 bits, at most 448), halves to the even one: multiples of 2^(e - 3) in [2^e, 2^(e + 1)),
    of 2^-9 below 2^-6."""
    step = torch.exp2((torch.frexp(q)[1].double() - 4).clamp(min=-9))
    return torch.round(q / step) * step


def _e4m3_codes_hold(ops, x, r, w, group):
    q, scale, h = ops.add_rmsnorm(x, w, r, quant="fp8", group_size=group)
    m, c = x.shape
    p = (h.double() * w.double()).view(m, -1, group or c)
    most = p.abs().amax(-1, keepdim=True)
    want = _nearest_e4m3(p * 448.0 / torch.where(most == 0, 1.0, most)).view(m, c)
    assert torch.equal(q.double(), want), int((q.double() != want).sum())


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("m,c,group", [(4096, 4096, 0), (4096, 4096, 32), (16384, 512, 128), (5000, 1001, 0), (700, 2049, 0), (5000, 520, 0)])
def test_norm_e4m3_codes_are_the_nearest(ops, m, c, group, dtype):
    """A code is the nearest one of the exact quotient 448 p / P (products p of 16-bit numbers), halves to the even one."""
    x, r, w = _norm_problem(m, c, dtype)
    _e4m3_codes_hold(ops, x, r, w, group)
    _e4m3_codes_hold(ops, x, None, torch.ones_like(w), group)           # products of few digits: many on a border


@pytest.mark.parametrize("dtype", BOTH)
def test_norm_e4m3_codes_on_borders(ops, dtype):
    """Quotients on borders: P = 2^a 7 gives 448 p / P = p 2^(6 - a), and other P quotients next to them; subnormal codes too."""
    p = torch.cat([(2 * torch.arange(8, 16) + 1) * 2.0 ** e for e in range(-7, 4)] + [(2 * torch.arange(0, 8) + 1) * 2.0 ** -10 / 2.0 ** 2])
    p = p[p < 100]
    for top in (112.0, 111.0, 113.0, 127.5, 119.0, 448.0, 224.0):
        x = torch.cat([p, -p, torch.tensor([top, 0.0])]).cuda().to(dtype)
        for c in (x.numel(), (x.numel() + 7) // 8 * 8):
            row = torch.zeros(2, c, dtype=dtype, device="cuda")
            row[0, : x.numel()], row[1, -x.numel():] = x, x.flip(0)
            for weight in (1.0, 1.5, 2.0 ** -100 if dtype == torch.bfloat16 else 2.0 ** -10):
                _e4m3_codes_hold(ops, row, None, torch.full((c,), weight, device="cuda").to(dtype), 0)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("quant", ["int8", "fp8"])
@pytest.mark.parametrize("c,group", [(512, 0), (512, 64), (509, 0)])
def test_norm_codes_beside_an_infinity_and_of_extreme_rows(ops, c, group, quant, dtype):
    """p / P is 0 beside an infinite P; rows near the ends of the type's range have the codes of their quotients."""
    x = torch.randn(6, c, generator=_gen(c), device="cuda")
    x[0, 5], x[1, 6] = float("inf"), float("-inf")
    ends = [1e30, 3e38, 1e-25, 1e-35] if dtype == torch.bfloat16 else [60.0, 15000.0, 1e-3, 1e-4]
    for i, size in enumerate(ends):
        x[2 + i] *= size / x[2 + i].abs().max()
    x, w = x.to(dtype), torch.ones(c, device="cuda", dtype=dtype)
    q, scale, _ = ops.add_rmsnorm(x, w, quant=quant, group_size=group)
    assert not q[0, : group or c].float()[torch.arange(group or c, device="cuda") != 5].any()
    assert not q[1, : group or c].float()[torch.arange(group or c, device="cuda") != 6].any()
    p = x[2:].double().view(4, -1, group or c)
    quotient = (p * (127.0 if quant == "int8" else 448.0) / p.abs().amax(-1, keepdim=True)).view(4, c)
    want = quotient.round() if quant == "int8" else _nearest_e4m3(quotient)
    assert torch.equal(q[2:].double(), want)


@pytest.mark.parametrize("cache", [torch.float16, FP8])
@pytest.mark.parametrize("b,hq,hk,d,prefix", [(40, 8, 8, 128, 2096), (33, 24, 8, 64, 4000), (17, 8, 8, 256, 2000), (64, 64, 8, 128, 1104)])
def test_prefix_keeps_a_tail_behind_one_strong_key(kv, b, hq, hk, d, prefix, cache):
    """f16 weights of e^-18 (2^-26) of the largest, whose own value is 0: all that is left is the tail.  A part of a weight holds
    2^-25 of 2^14, 2^-39 of the running maximum, so 2^-13 of such a weight; one part rounds it by 2^-11 besides."""
    lens = [prefix + i % 5 for i in range(b)]
    q, k, v, table, n, scales = _prefix_problem(lens, prefix, hq, hk, d, 16, torch.float16, cache, holes=False, wide=False)
    q.zero_(), k.view(torch.uint8).zero_()
    q[..., 0] = 1.0
    at = int(table[0, 0])
    k[at, :, 0, 0] = 18.0
    v.copy_((600 + 200 * torch.rand(v.shape, generator=_gen(d), device="cuda")).clamp(max=448 if cache == FP8 else 1000).to(cache))
    v[at, :, 0] = 0.0
    scales = [None if s is None else torch.ones_like(s) for s in scales]
    got = kv.prefix_attention(q, k, v, table, n, prefix, scale=1.0, k_scale=scales[0], v_scale=scales[1])
    want = _prefix_exact(q, k, v, table, n, scales, 1.0)[0]
    assert float(want.min()) > 2.0 ** -8
    assert float(((got.double() - want).abs() / want).max()) <= 2 * 2.0 ** -11 + 2.0 ** -13 + 2.0 ** -14


# ----------------------------------------------------------------------------------------------------------
# where sharing pays: more than 128 MB of shared keys and values that the rows would read one by one.  Fewer, and the results
# are those of the rows' own kernel, bit for bit, however wide the table.
# ----------------------------------------------------------------------------------------------------------

def _rows_that_pay(hk, d, prefix, cache):
    return (1 << 27) // (hk * prefix * d * 2 * (1 if cache == FP8 else 2)) + 1


@pytest.mark.parametrize("cache", [torch.bfloat16, torch.float16, FP8])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("b,hq,hk,prefix", [(6, 8, 2, 333), (33, 16, 4, 60), (3, 5, 1, 1), (12, 8, 8, 0)])
def test_prefix_short_in_a_wide_table(kv, b, hq, hk, prefix, d, cache):
    lens = [prefix + 3 * i for i in range(b)]
    dtype = torch.float16 if cache == FP8 else cache
    problem = _prefix_problem(lens, prefix, hq, hk, d, 16, dtype, cache)
    q, k, v, table, n, scales = problem
    kw = dict(k_scale=scales[0], v_scale=scales[1], return_lse=True)
    want, log = kv.paged_attention(q, k, v, table, n, **kw)
    got, same = kv.prefix_attention(q, k, v, table, n, prefix, **kw)
    assert torch.equal(got, want) and torch.equal(same, log)
    shared = torch.tensor([prefix], dtype=torch.int32, device="cuda")
    assert torch.equal(_prefix_holds(kv, problem, shared), want)
    shared.fill_(-5)
    assert torch.equal(_prefix_holds(kv, problem, shared), want)


_COMBINED = [[(torch.bfloat16, torch.bfloat16), (torch.float16, FP8)], [(torch.float16, torch.float16), (torch.bfloat16, FP8)]]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("case", list(enumerate([(8, 8, 1111, 60, 16), (8, 1, 5000, 33, 16), (16, 2, 700, 30, 16), (6, 3, 2049, 40, 64),
                                            (56, 8, 640, 17, 128), (12, 12, 129, 5, 32), (64, 8, 127, 9, 16), (8, 8, 6000, 100, 16),
                                            (2, 1, 60000, 3, 16), (64, 64, 6, 2, 8), (32, 8, 1024, 0, 16)])), ids=lambda c: str(c[1]))
def test_prefix_where_sharing_pays(kv, case, d):
    i, (hq, hk, prefix, longest, page) = case
    for dtype, cache in _COMBINED[(i + d // 128) % 2]:
        b = _rows_that_pay(hk, d, prefix, cache)
        lens = [prefix + (longest * r) // max(1, b - 1) for r in range(b)]
        problem = _prefix_problem(lens, prefix, hq, hk, d, page, dtype, cache, wide=False)
        got = _prefix_holds(kv, problem, prefix)
        q, k, v, table, n, scales = problem
        shared = torch.tensor([prefix], dtype=torch.int32, device="cuda")
        for again in (prefix, shared):
            assert torch.equal(kv.prefix_attention(q, k, v, table, n, again, k_scale=scales[0], v_scale=scales[1]), got)
        assert _status() == (0, 0)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq", [8, 40])
def test_prefix_of_uneven_rows_where_sharing_pays(kv, hq, d):
    """Rows without the prefix, rows of nothing, prefixes of nothing and beyond every row, holes in the table."""
    b = _rows_that_pay(8, d, 300, torch.bfloat16) + 6
    lens = [0, 400, 350, 3, 700, 349] + [350 + 7 * (i % 20) for i in range(b - 6)]
    problem = _prefix_problem(lens, 350, hq, 8, d, 16, torch.bfloat16, torch.bfloat16, wide=False)
    for prefix in (350, 0, 100000):
        _prefix_holds(kv, problem, prefix)
    lens = [360 + 7 * (i % 20) for i in range(b)]
    problem = _prefix_problem(lens, 360, hq, 8, d, 16, torch.bfloat16, torch.bfloat16, wide=False)
    for prefix in (360, 359, 321):                                      # any shorter prefix is shared too
        _prefix_holds(kv, problem, prefix)
    rows = torch.arange(b, device="cuda", dtype=torch.int32).flip(0)
    rows[1], rows[2], rows[3] = -1, b, rows[0]                          # no row, beyond the table, the same row twice
    _prefix_holds(kv, problem, 360, rows=rows)
    _prefix_holds(kv, problem, 360, scale=-0.02)
    holed = problem[3].clone()
    holed[:, 3], holed[:, 9] = -1, len(problem[1])                      # pages that the table does not have, inside the prefix
    _prefix_holds(kv, (*problem[:3], holed, *problem[4:]), 360)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_prefix_large_scores_where_sharing_pays(kv, d):
    """Maxima that grow from tile to tile, infinities and NaN in sight."""
    b = _rows_that_pay(8, d, 1500, torch.float16)
    problem = _prefix_problem([1500 + i % 9 for i in range(b)], 1500, 16, 8, d, 16, torch.float16, torch.float16, wide=False)
    q, k, v, table, n, scales = problem
    for j in range(0, 1500, 16):                                        # keys grow along the prefix
        k[int(table[0, j // 16])] *= 0.2 + 4 * j / 1500
    src = int(table[0, 93])
    for r in range(1, b):
        k[int(table[r, 93]), :, :12] = k[src, :, :12]
    want, lse, slack, share, tail = _prefix_exact(*problem[:5], scales)
    one_part = 2 * b > (128 if d == 256 else 256)
    got = kv.prefix_attention(q, k, v, table, n, 1500)
    u = U[torch.float16]
    assert float(((got.double() - want).abs() - u * want.abs() - slack * 1.01 - (u * share if one_part else 0) - tail - 2.0 ** -25).max()) <= 0
    bad = v.clone()
    bad[int(table[0, 5]), 0, 3, 7] = float("inf")
    bad[int(table[0, 6]), 1, 4, 9] = float("nan")
    off = ~torch.isfinite(kv.prefix_attention(q, k, bad, table, n, 1500))
    assert bool(off[:, :2, 7].all()) and bool(off[:, 2:4, 9].all()) and int(off.sum()) == b * 4
    worse = k.clone()
    worse[int(table[0, 5]), 0, 3] = float("nan")
    got = kv.prefix_attention(q, worse, v, table, n, 1500)
    assert bool(got[:, :2].isnan().all()) and bool(torch.isfinite(got[:, 2:]).all())


def test_prefix_strides_streams_and_graphs_where_sharing_pays(kv):
    b = _rows_that_pay(8, 64, 950, torch.bfloat16)
    problem = _prefix_problem([1000 + i % 30 for i in range(b)], 1000, 16, 8, 64, 16, torch.bfloat16, torch.bfloat16, wide=False)
    q, k, v, table, n, _ = problem
    want = _prefix_holds(kv, problem, 1000)
    wide = torch.zeros(b, 19, 64, device="cuda", dtype=q.dtype)
    wide[:, 1:17] = q
    out = torch.full_like(q, 7.0)
    assert kv.prefix_attention(wide[:, 1:17], k, v, table, n, 1000, out=out) is out and torch.equal(out, want)
    head_last, value_last = (c.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for c in (k, v))
    assert torch.equal(kv.prefix_attention(q, head_last, value_last, table, n, 1000), want)
    shared = torch.tensor([1000], dtype=torch.int32, device="cuda")
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = kv.prefix_attention(q, k, v, table, n, shared)
        graphs.append((graph, held))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
            mine = kv.prefix_attention(q, k, v, table, n, 1000)
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want) and torch.equal(mine, want)
    for prefix in (960, 20, 0, 1000):                                   # a captured step reads the prefix anew, and what pays
        shared.fill_(prefix)
        graphs[0][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], kv.prefix_attention(q, k, v, table, n, prefix))
    assert _status() == (0, 0)


def test_prefix_offsets_past_32_bits_where_sharing_pays(kv):
    pages, page, hk, d = 140_000, 16, 8, 128                            # 4.6 GB each
    k = torch.zeros(pages, hk, page, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    b = _rows_that_pay(hk, d, 320, torch.bfloat16)
    ids = torch.tensor([pages - 1 - 5 * i for i in range(20 + 4 * b)], dtype=torch.int32)
    g = _gen(11)
    for c in (k, v):
        c[ids.long().cuda()] = torch.randn(len(ids), hk, page, d, generator=g, device="cuda").bfloat16()
    table = torch.cat([ids[:20].expand(b, 20), ids[20:].view(b, 4)], dim=1).cuda()
    lens = torch.tensor([320 + i % 65 for i in range(b)], dtype=torch.int32, device="cuda")
    q = torch.randn(b, 16, d, generator=g, device="cuda").bfloat16()
    _prefix_holds(kv, (q, k, v, table, lens, [None, None]), 320)


def test_steps_behind_a_shared_prompt_where_sharing_pays(kv):
    """40 rows forked from a prompt of 500 tokens, eight heads of 256: its tokens are attended once for all rows."""
    g = _gen(6)
    prompt, tokens = torch.randint(0, 500, (500,), generator=g, device="cuda"), torch.randint(0, 500, (4, 40), generator=g, device="cuda")
    models = [_model(heads=8, kv_heads=8, head_dim=256, rows=41, pages=200, max_tokens=520) for _ in range(3)]
    rows = torch.arange(1, 41, dtype=torch.int32, device="cuda")
    for m in models:
        m.prompt(prompt, 0)
        m.cache.branch(torch.zeros_like(rows), rows, 0)
    shared = torch.tensor([500], dtype=torch.int32, device="cuda")
    fill, graph, held = models[2].capture(rows, shared)
    for i in range(4):
        alone, together = models[0].step(tokens[i], rows), models[1].step(tokens[i], rows, None, 500)
        assert float((alone.float() - together.float()).norm() / alone.float().norm()) <= 4.6e-2
        fill.copy_(tokens[i])
        graph.replay()
        assert torch.equal(held, together)
    for m in models:
        m.cache.check()
    assert _status() == (0, 0)


@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, torch.bfloat16), (torch.float16, FP8)])
@pytest.mark.parametrize("b,hq,hk,d,prefix", [(300, 32, 8, 64, 600), (130, 8, 4, 256, 700), (100, 64, 8, 128, 1000), (20, 8, 8, 128, 2000)])
def test_prefix_weights_in_one_part_or_two(kv, b, hq, hk, d, prefix, dtype, cache):
    """Two parts: the bound of paged attention, whatever the batch; one: u of the weights besides."""
    problem = _prefix_problem([prefix + i % 7 for i in range(b)], prefix, hq, hk, d, 16, dtype, cache, wide=False)
    q, k, v, table, n, scales = problem
    want, _, slack, share, tail = _prefix_exact(q, k, v, table, n, scales)
    u = U[dtype]
    once = float((want.to(dtype).double() - want).norm() / want.norm())
    got = {}
    for parts in (1, 2, None):
        got[parts] = kv.prefix_attention(q, k, v, table, n, prefix, k_scale=scales[0], v_scale=scales[1], weight_parts=parts)
        one = parts == 1 or (parts is None and b * (hq // hk) > (128 if d == 256 else 256))
        off = (got[parts].double() - want).abs()
        assert float((off - u * want.abs() - slack * (1 + u) - (u * share if one else 0) - tail - 2.0 ** -25).max()) <= 0
        assert float(off.norm() / want.norm()) <= (1.5 if one else 1.05) * once + 2.0 ** -14
    assert torch.equal(got[1], got[2]) == (b < _rows_that_pay(hk, d, prefix, cache))    # 20 rows in 8 bits: 82 MB, read row by row
    assert torch.equal(got[None], got[1 if b * (hq // hk) > (128 if d == 256 else 256) else 2])


def test_a_step_behind_a_shared_prompt_is_as_exact_as_alone(kv, monkeypatch):
    """The model's attention behind a prompt holds the bound of attention row by row: weights in two parts."""
    held = []
    whole = kv.prefix_attention

    def recorded(q, k, v, table, lens, prefix, rows=None, **kw):
        out = whole(q, k, v, table, lens, prefix, rows=rows, **kw)
        held.append((q.clone(), out.clone(), kv.paged_attention(q, k, v, table, lens, rows=rows)))
        return out
    monkeypatch.setattr(kv, "prefix_attention", recorded)
    m = _model(heads=32, kv_heads=4, head_dim=128, rows=41, pages=400, max_tokens=2010)
    m.prompt(torch.randint(0, 500, (2000,), generator=_gen(8), device="cuda"), 0)
    rows = torch.arange(1, 41, dtype=torch.int32, device="cuda")
    m.cache.branch(torch.zeros_like(rows), rows, 0)
    m.step(torch.arange(40, device="cuda"), rows, None, 2000)
    assert len(held) == 2
    # each holds 2^-14: two results 2^-13 apart round to neighbours, 2^-7 apart, in 2^-6 of the cases: 2^-10 in the square mean
    for q, got, want in held:
        assert float((got.double() - want.double()).norm() / want.double().norm()) <= 2.0 ** -10


def test_generate_takes_numbers_of_any_type_and_one_for_all_rows(ops):
    m = _model()
    prompt, u = torch.arange(33, device="cuda"), torch.randint(0, 128, (6, 3), generator=_gen(2), device="cuda") / 128
    want = m.generate(prompt, 3, 6, u)
    for same in (u.bfloat16(), u.half(), u.double(), u.unsqueeze(-1)):   # exact in all of them
        assert torch.equal(m.generate(prompt, 3, 6, same), want)
    one = m.generate(prompt, 3, 6, u[:, :1].expand(6, 3))
    assert torch.equal(m.generate(prompt, 3, 6, u[:, :1]), one) and torch.equal(m.generate(prompt, 3, 6, u[:, 0]), one)
    assert torch.equal(m.generate(prompt, 3, 6, torch.zeros(6, 3, dtype=torch.long, device="cuda")), m.generate(prompt, 3, 6, 0 * u))


def test_generate_with_more_tokens_than_the_sampler_takes(ops):
    m = _model(vocab=327744)
    u = torch.rand(3, 2, generator=_gen(3), device="cuda")
    got = m.generate(torch.arange(20, device="cuda"), 2, 3, u)
    assert got.shape == (2, 3) and int(got.min()) >= 0 and int(got.max()) < 327744
    logits = m.prompt(torch.arange(20, device="cuda"), 5)[-1].double().softmax(-1).cumsum(0)
    for r in range(2):                                                   # a cumulative sum in f32: off by 2^-24 a token at most
        at = int(got[r, 0])
        off = 327744 * 2.0 ** -24
        assert float(logits[at - 1] if at else 0.0) <= float(u[0, r]) + off and float(logits[at]) >= float(u[0, r]) - off
    with pytest.raises(ValueError, match="327680"):
        m.generate(torch.arange(20, device="cuda"), 2, 3, u, top_k=5)


@pytest.mark.parametrize("off", [0, 1, 3])
def test_sample_the_largest_vocabulary(ops, off):
    """327680 tokens in f32: a CTA's share and the helpers come to 202 KB, and sums of equal logits to 2^62.3."""
    n = 327680
    x, u = _logits(3, n, torch.float32)
    x[1] = -2.0
    x[2] = torch.where(torch.arange(n, device="cuda") % 3 == 0, 1.0, -8.0)
    u = torch.tensor([float(u[0]), 0.75, 0.3125], device="cuda")
    wide = torch.full((3, n + 5), 60000.0, device="cuda")               # neighbours are not read
    wide[:, off:off + n] = x
    for k, p, m in ((0, 1.0, 0.0), (0, 0.9, 0.0), (50, 0.8, 0.05), (n // 2, 0.5, 0.0), (n - 1, 1.0, 0.0), (0, 0.25, 0.5)):
        _sample_holds(ops, wide[:, off:off + n], u, 0.9, k, p, m)


@pytest.mark.parametrize("t", [3, 400])
@pytest.mark.parametrize("cache", ["own", "fp8"])
@pytest.mark.parametrize("which", [0, 1])
def test_rotated_append_norm_of_queries_or_keys_alone(kv, which, cache, t):
    dtype = torch.bfloat16
    rope = kv.rope_table(64, 64)
    problem = list(_rotate_problem(t, 6, 2, 128, 64, dtype, FP8 if cache == "fp8" else dtype))
    problem[6] = [w if i == which else None for i, w in enumerate(problem[6])]
    for interleaved in (False, True):
        _rotate_holds(kv, problem, 6, 2, 64, interleaved, rope)


@pytest.mark.parametrize("quant", ["int8", "fp8"])
@pytest.mark.parametrize("c,group", [(256, 0), (2048, 0), (2048, 64), (255, 0), (2049, 0)])
def test_norm_products_that_are_no_numbers_show_in_the_scale(ops, c, group, quant):
    """P of products with a NaN is NaN, though the row has none: a NaN weight, or an infinity times a weight of 0."""
    x = torch.randn(5, c, generator=_gen(c), device="cuda").bfloat16()
    w = torch.ones(c, device="cuda").bfloat16()
    plain = ops.add_rmsnorm(x, w, quant=quant, group_size=group)
    hurt = w.clone()
    hurt[c - 7] = float("nan")
    _, scale, _ = ops.add_rmsnorm(x, hurt, quant=quant, group_size=group)
    if group:
        assert bool(scale[-1].isnan().all()) and torch.equal(scale[:-1], plain[1][:-1])
    else:
        assert bool(scale.isnan().all())
    x[3, 9] = float("inf")
    hurt = w.clone()
    hurt[9] = 0.0
    _, scale, _ = ops.add_rmsnorm(x, hurt, quant=quant, group_size=group)
    assert bool(scale[..., 3][:1].isnan().all() if group else scale[3].isnan())
    assert bool(torch.isfinite(scale[..., [0, 1, 2, 4]]).all())

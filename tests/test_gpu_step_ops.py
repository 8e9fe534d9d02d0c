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

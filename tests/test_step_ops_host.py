"""CPU-side checks of the operators around a decode step: the C ABI rejects bad arguments before it touches a device, the
Python operators say what is wrong with their arguments and reject CPU tensors, and the tables of angles are right."""
import ctypes
import math

import pytest
import torch

BF, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def lib():
    from comfy_quant_bench_b200 import _lib
    return _lib.load()


VP = ctypes.c_void_p(256)


def test_norm_argument_checks_need_no_device(lib):
    from comfy_quant_bench_b200 import _lib as L

    def call(x=VP, ldx=64, r=VP, ldr=64, w=VP, dt=0, rows=2, width=64, kind=0, group=0, h=VP, ldh=64, out=VP, scale=VP):
        return lib.cq_add_rmsnorm(x, ldx, r, ldr, w, dt, rows, width, 1e-6, kind, group, h, ldh, out, scale, None)
    assert call(dt=2) == L.CQ_ERR_ARG and call(kind=3) == L.CQ_ERR_ARG and call(kind=-1) == L.CQ_ERR_ARG
    assert call(group=32) == L.CQ_ERR_ARG and call(kind=1, group=16) == L.CQ_ERR_ARG and call(kind=1, scale=None) == L.CQ_ERR_ARG
    assert call(kind=1, group=128) == L.CQ_ERR_SHAPE and call(width=0) == L.CQ_ERR_SHAPE and call(width=32769) == L.CQ_ERR_SHAPE
    assert call(rows=-1) == L.CQ_ERR_SHAPE and call(ldx=63) == L.CQ_ERR_SHAPE and call(ldr=8) == L.CQ_ERR_SHAPE
    assert call(ldh=8) == L.CQ_ERR_SHAPE
    assert call(x=None) == L.CQ_ERR_ARG and call(w=None) == L.CQ_ERR_ARG and call(out=None) == L.CQ_ERR_ARG
    assert call(x=ctypes.c_void_p(258)) == L.CQ_ERR_ALIGN and call(ldx=65) == L.CQ_ERR_ALIGN and call(ldr=68) == L.CQ_ERR_ALIGN
    assert call(width=63, x=ctypes.c_void_p(257)) == L.CQ_ERR_ALIGN
    assert call(rows=0, x=None, out=None) == L.CQ_OK


def test_rotated_append_argument_checks_need_no_device(lib):
    from comfy_quant_bench_b200 import _lib as L

    def call(q=VP, dt=0, t=1, hq=4, hk=2, d=64, rope=VP, rr=10, rot=64, qo=VP, cdt=0, pages=10, page=16, ts=8, rows=VP, qst=512,
             scale=None):
        return lib.cq_kv_append_rotated(q, qst, 64, VP, 512, 64, VP, 512, 64, dt, t, hq, hk, d, rope, rr, rot, 0, None, None,
                                        1e-6, qo, None, VP, VP, cdt, pages, page, 2048, 1024, 64, VP, 4, 8, ts, rows, VP, scale,
                                        scale, None)
    assert call(dt=2) == L.CQ_ERR_ARG and call(cdt=1) == L.CQ_ERR_ARG and call(q=None) == L.CQ_ERR_ARG
    assert call(rope=None) == L.CQ_ERR_ARG and call(qo=None) == L.CQ_ERR_ARG and call(rows=None) == L.CQ_ERR_ARG
    assert call(d=20) == L.CQ_ERR_SHAPE and call(d=264) == L.CQ_ERR_SHAPE and call(rot=24) == L.CQ_ERR_SHAPE
    assert call(rot=80) == L.CQ_ERR_SHAPE and call(rot=0) == L.CQ_ERR_SHAPE and call(rr=0) == L.CQ_ERR_SHAPE
    assert call(page=12) == L.CQ_ERR_SHAPE and call(ts=7) == L.CQ_ERR_SHAPE and call(t=-1) == L.CQ_ERR_SHAPE
    assert call(hq=0) == L.CQ_ERR_SHAPE and call(qst=513) == L.CQ_ERR_ALIGN and call(q=ctypes.c_void_p(264)) == L.CQ_ERR_ALIGN
    assert call(scale=ctypes.c_void_p(257), cdt=2) == L.CQ_ERR_ALIGN
    assert call(t=0, q=None) == L.CQ_OK


def test_refusals_say_what_is_wrong():
    from comfy_quant_bench_b200 import kvcache, ops
    x, w = torch.zeros(3, 96, dtype=BF), torch.ones(96, dtype=BF)
    q, k = torch.zeros(2, 4, 64, dtype=BF), torch.zeros(2, 2, 64, dtype=BF)
    kc = torch.zeros(5, 2, 16, 64, dtype=BF)
    t, r, rope = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(8, 32, 2)

    def turn(q=q, k=k, v=None, kc=kc, t=t, r=r, rope=rope, **kw):
        return kvcache.append_rotated(q, k, k if v is None else v, kc, kc, t, r, r, rope, **kw)
    for says, call in (("bf16 or f16, got Float", lambda: ops.add_rmsnorm(x.float(), w)),
                       ("96 elements", lambda: ops.add_rmsnorm(x, w[:5])),
                       ("1 to 32768", lambda: ops.add_rmsnorm(x[:, :0], w)),
                       (r"residual must be BFloat16 of shape \[3, 96\]", lambda: ops.add_rmsnorm(x, w, x[:2])),
                       ("residual must be", lambda: ops.add_rmsnorm(x, w, x.half())),
                       ("'int8' or 'fp8', got 'int4'", lambda: ops.add_rmsnorm(x, w, quant="int4")),
                       ("divide 96 with an 8-bit output, got 64", lambda: ops.add_rmsnorm(x, w, quant="int8", group_size=64)),
                       ("with an 8-bit output, got 32", lambda: ops.add_rmsnorm(x, w, group_size=32)),
                       ("goes with a residual", lambda: ops.add_rmsnorm(x, w, out_residual=x)),
                       ("out_residual must be contiguous", lambda: ops.add_rmsnorm(x, w, x, out_residual=x[:2])),
                       (r"\[T, q_heads, D\]", lambda: turn(q=q[0])),
                       ("of one shape", lambda: turn(v=k[:, :1])),
                       ("does not fit q", lambda: turn(k=k[:1])),
                       ("do not fit k", lambda: turn(kc=kc[:, :1])),
                       ("multiple of 8 from 16 to 256, got 12", lambda: turn(q=q[..., :12], k=k[..., :12], kc=kc[..., :12])),
                       ("one entry per token", lambda: turn(r=r[:1])),
                       ("rope must be contiguous f32", lambda: turn(rope=rope.double())),
                       ("multiple of 16 columns, at most D=64, got 128", lambda: turn(rope=torch.zeros(8, 64, 2))),
                       ("at most D=64, got 20", lambda: turn(rope=rope[:, :10].contiguous())),
                       ("q_norm must have 64 elements", lambda: turn(q_norm=w)),
                       ("must hold", lambda: turn(kc=kc.half()))):
        with pytest.raises(ValueError, match=says):
            call()
    for call in (lambda: ops.add_rmsnorm(x, w, x, quant="int8"), turn):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_tables_of_angles():
    from comfy_quant_bench_b200 import kvcache
    plain = kvcache.rope_table(100001, 64, device="cpu")
    assert plain.shape == (100001, 32, 2) and plain.dtype == torch.float32
    for p in (0, 1, 77, 100000):
        for i in (0, 5, 31):
            angle = p * 10000.0 ** (-2 * i / 64)
            assert abs(float(plain[p, i, 0]) - math.cos(angle)) <= 2.0 ** -24
            assert abs(float(plain[p, i, 1]) - math.sin(angle)) <= 2.0 ** -24
    linear = kvcache.rope_table(400, 64, scaling="linear", factor=4.0, device="cpu")
    assert float((linear[::4] - plain[:100]).abs().max()) <= 2.0 ** -23
    base = kvcache.rope_table(400, 64, scaling="base", factor=4.0, device="cpu")
    assert torch.equal(base[:, 0], plain[:400, 0])                       # the fastest pair stays
    assert float((base[::4, 31] - plain[:100, 31]).abs().max()) <= 2.0 ** -20    # the slowest is divided by the factor
    parts = kvcache.rope_table(400, 64, scaling="parts", factor=4.0, original=4096, device="cpu")
    size = 0.1 * math.log(4.0) + 1
    assert float((parts[:, 0] / size - plain[:400, 0]).abs().max()) <= 2.0 ** -22
    assert float((parts[::4, 31] / size - plain[:100, 31]).abs().max()) <= 2.0 ** -20
    for bad in (dict(rot_dim=7), dict(rot_dim=64, scaling="other"), dict(rot_dim=64, scaling="linear", factor=0.5),
                dict(rot_dim=64, scaling="parts", factor=2.0)):
        with pytest.raises(ValueError):
            kvcache.rope_table(4, device="cpu", **bad)

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


def test_prefix_attention_argument_checks_need_no_device(lib):
    from comfy_quant_bench_b200 import _lib as L
    size = lib.cq_prefix_attention_workspace_bytes
    assert size(4, 8, 2, 128, 100, ) == 0 and size(0, 8, 2, 128, 1 << 20) == 0          # read row by row, whole
    assert size(64, 32, 8, 128, 16000) > 64 * 32 * 132 * 4
    assert size(2, 8, 3, 128, 64) == -1 and size(2, 8, 2, 96, 64) == -1 and size(-1, 8, 2, 64, 64) == -1

    def call(q=VP, dt=0, b=64, hq=32, hk=8, d=128, cdt=0, pages=10, page=16, st=128, width=1000, ts=1000, lens=VP, prefix=VP, n=0,
             out=VP, ws=VP, wsn=1 << 40):
        return lib.cq_prefix_attention(q, 4096, 128, dt, b, hq, hk, d, VP, VP, cdt, pages, page, 16384, 2048, st, VP, 64, width, ts,
                                       None, lens, prefix, n, 1.0, None, None, out, None, ws, wsn, None)
    assert call(dt=2) == L.CQ_ERR_ARG and call(cdt=1) == L.CQ_ERR_ARG and call(q=None) == L.CQ_ERR_ARG
    assert call(lens=None) == L.CQ_ERR_ARG and call(out=None) == L.CQ_ERR_ARG and call(ws=None) == L.CQ_ERR_ARG
    assert call(page=12) == L.CQ_ERR_SHAPE and call(hq=30) == L.CQ_ERR_SHAPE and call(d=96) == L.CQ_ERR_SHAPE
    assert call(n=-1) == L.CQ_ERR_SHAPE and call(n=1 << 31) == L.CQ_ERR_SHAPE and call(wsn=1024) == L.CQ_ERR_SHAPE
    assert call(b=65536) == L.CQ_ERR_SHAPE and call(ts=999) == L.CQ_ERR_SHAPE
    assert call(q=ctypes.c_void_p(264)) == L.CQ_ERR_ALIGN and call(st=129) == L.CQ_ERR_ALIGN
    assert call(prefix=ctypes.c_void_p(258)) == L.CQ_ERR_ALIGN and call(ws=ctypes.c_void_p(128)) == L.CQ_ERR_ALIGN
    assert call(b=0, q=None, lens=None, out=None, ws=None) == L.CQ_OK


def test_sample_argument_checks_need_no_device(lib):
    from comfy_quant_bench_b200 import _lib as L

    def call(x=VP, ld=100, dt=3, rows=2, vocab=100, u=VP, k=0, tokens=VP, logs=None, ts=None):
        return lib.cq_sample(x, ld, dt, rows, vocab, u, ts, 1.0, None, k, None, 1.0, None, 0.0, tokens, logs, None)
    assert call(dt=2) == L.CQ_ERR_ARG and call(dt=4) == L.CQ_ERR_ARG and call(x=None) == L.CQ_ERR_ARG
    assert call(u=None) == L.CQ_ERR_ARG and call(tokens=None) == L.CQ_ERR_ARG
    assert call(rows=-1) == L.CQ_ERR_SHAPE and call(vocab=0) == L.CQ_ERR_SHAPE and call(vocab=327681, ld=400000) == L.CQ_ERR_SHAPE
    assert call(ld=99) == L.CQ_ERR_SHAPE and call(k=-1) == L.CQ_ERR_SHAPE
    assert call(x=ctypes.c_void_p(258)) == L.CQ_ERR_ALIGN and call(tokens=ctypes.c_void_p(260)) == L.CQ_ERR_ALIGN
    assert call(ts=ctypes.c_void_p(258)) == L.CQ_ERR_ALIGN
    assert call(rows=0, x=None, u=None, tokens=None) == L.CQ_OK


def test_more_refusals_say_what_is_wrong():
    from comfy_quant_bench_b200 import kvcache, ops
    k, n = torch.zeros(6, 2, 16, 64, dtype=BF), torch.zeros(2, dtype=torch.int32)
    t, q = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 4, 64, dtype=BF)
    x, u = torch.zeros(3, 50), torch.zeros(3)

    def attend(prefix=5, q=q, **kw):
        return kvcache.prefix_attention(q, k, k, t, n, prefix, **kw)

    def sample(x=x, u=u, **kw):
        return ops.sample_tokens(x, u, **kw)
    for says, call in (("must not be negative, got -1", lambda: attend(-1)),
                       ("int32 tensor of one element", lambda: attend(n)),
                       ("int32 tensor of one element", lambda: attend(torch.zeros(1, dtype=torch.int64))),
                       ("multiple of kv_heads", lambda: attend(q=q[:, :3])),
                       ("64, 128 or 256", lambda: attend(q=q[..., :32])),
                       ("rows must have 2 entries", lambda: attend(rows=n[:1])),
                       (r"f32 \[rows, vocab\]", lambda: sample(x=x.double())),
                       (r"f32 \[rows, vocab\]", lambda: sample(x=x[0])),
                       ("1 to 327680, got 0", lambda: sample(x=x[:, :0])),
                       (r"uniform must be f32 \[3\]", lambda: sample(u=u[:2])),
                       (r"uniform must be f32 \[3\]", lambda: sample(u=u.double())),
                       ("temperature is out of range", lambda: sample(temperature=-1.0)),
                       ("temperature is out of range", lambda: sample(temperature=float("nan"))),
                       ("top_k is out of range", lambda: sample(top_k=-3)),
                       ("top_p is out of range", lambda: sample(top_p=1.5)),
                       ("min_p is out of range", lambda: sample(min_p=-0.1)),
                       (r"top_p must be a number or Float \[3\]", lambda: sample(top_p=u[:1])),
                       (r"top_k must be a number or Int \[3\]", lambda: sample(top_k=u))):
        with pytest.raises(ValueError, match=says):
            call()
    for call in (attend, sample):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_sampling_waits_for_its_cluster_before_it_writes_to_it():
    """Another CTA's shared memory may be touched once that CTA runs: every CTA arrives at the cluster's barrier as it starts
    and waits there, on every path, before its first store to another (whose help, ``exchange``, is the first to use one)."""
    import os
    import re

    from comfy_quant_bench_b200 import build
    source = open(os.path.join(build.SRC, "sample.cu")).read()
    body = source[source.index("sample_kernel(const SampleArgs"):]
    body = body[:body.index("\nnamespace {")]
    before = re.split(r"exchange\(|there\(|cluster_sum\(|add_at_first\(|cut_in_bin<|list_up_to", body)[0]
    assert before.count("cluster_arrive()") == 1 and before.count("cluster_wait()") == 1
    assert before.index("cluster_arrive()") < before.index("grid_dep_wait()") < before.index("cluster_wait()")
    assert "return;" not in before and "cluster_sync_all()" not in before


def test_weight_parts_are_checked(lib):
    from comfy_quant_bench_b200 import _lib as L
    from comfy_quant_bench_b200 import kvcache

    def call(parts, dt=0, ws=VP):
        return lib.cq_prefix_attention_parts(VP, 4096, 128, dt, 64, 32, 8, 128, VP, VP, 0, 10, 16, 16384, 2048, 128, VP, 64, 1000,
                                             1000, None, VP, VP, 0, parts, 1.0, None, None, VP, None, ws, 1 << 40, None)
    assert call(3) == L.CQ_ERR_ARG and call(-1) == L.CQ_ERR_ARG and call(2, dt=2) == L.CQ_ERR_ARG and call(1, ws=None) == L.CQ_ERR_ARG
    k, n = torch.zeros(6, 2, 16, 64, dtype=BF), torch.zeros(2, dtype=torch.int32)
    t, q = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 4, 64, dtype=BF)
    for parts in (0, 3, -1):
        with pytest.raises(ValueError, match="weight_parts must be None, 1 or 2, got"):
            kvcache.prefix_attention(q, k, k, t, n, 5, weight_parts=parts)
    with pytest.raises(ValueError, match="CUDA"):
        kvcache.prefix_attention(q, k, k, t, n, 5, weight_parts=2)


def test_a_fraction_of_a_token_is_refused():
    from comfy_quant_bench_b200 import ops
    x, u = torch.zeros(3, 50), torch.zeros(3)
    for k in (0.5, 2.5, 49.999):
        with pytest.raises(ValueError, match="top_k must be a whole number, got"):
            ops.sample_tokens(x, u, top_k=k)
    for k in (3, 3.0, True):
        with pytest.raises(ValueError, match="CUDA"):
            ops.sample_tokens(x, u, top_k=k)


def test_sampling_arguments_without_numbers_to_sample_by_are_refused():
    from comfy_quant_bench_b200 import textgen
    model = object.__new__(textgen.TextModel)                            # refused before anything is looked at
    for kw in (dict(temperature=0.7), dict(top_k=5, top_p=0.9), dict(temprature=0.7)):
        with pytest.raises(ValueError, match=f"{next(iter(kw))}.* without uniform numbers"):
            model.generate(torch.zeros(3, dtype=torch.long), 2, 4, **kw)


@pytest.mark.parametrize("rot,base,factor,original,fast,slow", [(128, 500000.0, 8.0, 8192, 4.0, 1.0), (64, 10000.0, 16.0, 4096, 32.0, 1.0),
                                                                (128, 10000.0, 4.0, 32768, 32.0, 1.0), (16, 100.0, 2.0, 40, 1.01, 1.0), (32, 10000.0, 2.0, 5, 4.0, 2.0)])
@pytest.mark.parametrize("blend", ["turns", "pairs"])
@pytest.mark.parametrize("size", [None, 1.0, 1.25])
def test_tables_stretched_by_parts(rot, base, factor, original, fast, slow, blend, size):
    """Every angle against the formula: with a size of 1 and fast 4, slow 1, too, and with the blend over the pairs' indexes."""
    from comfy_quant_bench_b200 import kvcache
    table = kvcache.rope_table(3000, rot, base=base, scaling="parts", factor=factor, original=original, fast=fast, slow=slow,
                               blend=blend, size=size, device="cpu")
    at = [rot * math.log(original / (2 * math.pi * n)) / (2 * math.log(base)) for n in (fast, slow)]
    first, last = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
    times = (0.1 * math.log(factor) + 1) if size is None else size
    for i in range(rot // 2):
        angle = base ** (-2 * i / rot)
        if blend == "turns":
            kept = min(1.0, max(0.0, (original * angle / (2 * math.pi) - slow) / (fast - slow)))
        else:
            kept = 0.0 if last < 0 or i >= last > first else 1.0 if i <= first else 1 - (i - first) / (last - first)
        angle = angle * kept + angle / factor * (1 - kept)
        for p in (0, 1, 777, 2999):
            assert abs(float(table[p, i, 0]) - times * math.cos(p * angle)) <= times * 2.0 ** -24 + 1e-9
            assert abs(float(table[p, i, 1]) - times * math.sin(p * angle)) <= times * 2.0 ** -24 + 1e-9


def test_the_size_of_turned_columns_and_blends_are_checked():
    from comfy_quant_bench_b200 import kvcache
    plain = kvcache.rope_table(50, 32, device="cpu")
    for scaling in (None, "linear", "base"):
        kw = dict(scaling=scaling, factor=2.0 if scaling else 1.0, device="cpu")
        assert float((kvcache.rope_table(50, 32, size=1.5, **kw) - 1.5 * kvcache.rope_table(50, 32, **kw)).abs().max()) <= 1.5 * 2.0 ** -23
    assert torch.equal(kvcache.rope_table(50, 32, size=1.0, device="cpu"), plain)
    for bad in (dict(size=0.0), dict(size=-1.0), dict(size=float("nan")), dict(size=float("inf")), dict(blend="pair")):
        with pytest.raises(ValueError):
            kvcache.rope_table(4, 32, device="cpu", **bad)

"""CPU-side checks of the decode-side operators: the C ABI rejects bad arguments on the host before touching a device,
and the Python operators reject CPU tensors."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from comfy_quant_bench_b200 import _lib
    return _lib.load()


VP = ctypes.c_void_p(256)


def test_linear_argument_checks_need_no_device(lib):
    from comfy_quant_bench_b200 import _lib as L

    def call(x=VP, ldx=256, dtype=0, m=2, k=256, n=16, w=VP, s=VP, z=VP, g=64, b=None, out=VP, ws=VP, wsn=1 << 30):
        return lib.cq_w4a16_linear(x, ldx, dtype, m, k, n, w, s, z, g, b, out, ws, wsn, None)
    assert call(dtype=2) == L.CQ_ERR_ARG and call(g=16) == L.CQ_ERR_ARG and call(g=0) == L.CQ_ERR_ARG
    assert call(k=96) == L.CQ_ERR_SHAPE and call(k=0) == L.CQ_ERR_SHAPE and call(ldx=128) == L.CQ_ERR_SHAPE
    assert call(m=-1) == L.CQ_ERR_SHAPE and call(n=-1) == L.CQ_ERR_SHAPE and call(k=1 << 20, ldx=1 << 20) == L.CQ_ERR_SHAPE
    assert call(x=None) == L.CQ_ERR_ARG and call(w=None) == L.CQ_ERR_ARG and call(out=None) == L.CQ_ERR_ARG
    assert call(x=ctypes.c_void_p(264)) == L.CQ_ERR_ALIGN and call(ldx=257) == L.CQ_ERR_ALIGN
    assert call(w=ctypes.c_void_p(260)) == L.CQ_ERR_ALIGN
    need = lib.cq_w4a16_workspace_bytes(20, 256, 64)
    assert need >= 20 * 256 * 2 and lib.cq_w4a16_workspace_bytes(4, 256, 64) == 0
    assert lib.cq_w4a16_workspace_bytes(4, 200, 64) == -1 and lib.cq_w4a16_workspace_bytes(-1, 256, 64) == -1
    assert call(m=20, wsn=need - 1) == L.CQ_ERR_SHAPE and call(m=20, ws=None) == L.CQ_ERR_ARG
    assert call(m=20, ws=ctypes.c_void_p(128)) == L.CQ_ERR_ALIGN
    assert call(m=0, x=None, w=None, s=None, z=None, out=None) == L.CQ_OK
    assert call(n=0) == L.CQ_OK


def test_attention_argument_checks_need_no_device(lib):
    from comfy_quant_bench_b200 import _lib as L
    size = lib.cq_paged_attention_workspace_bytes
    assert size(2, 8, 2, 128, 100000, 0, 0) > 0 and size(0, 8, 2, 128, 100000, 0, 0) == 0
    assert size(2, 8, 2, 128, 64, 0, 0) == 0 and size(2, 8, 2, 128, 100000, 50, 4) == 0      # no row is split
    assert size(2, 8, 3, 128, 64, 0, 0) == -1 and size(2, 8, 2, 96, 64, 0, 0) == -1 and size(-1, 8, 2, 64, 64, 0, 0) == -1

    def call(q=VP, sb=1024, sh=128, dt=0, b=2, hq=8, hk=2, d=128, k=VP, v=VP, cdt=0, pages=10, page=16, sp=4096, shd=2048,
             st=128, table=VP, rows=2, width=4, ts=4, lens=VP, window=0, sinks=0, out=VP, ws=VP, wsn=1 << 40):
        return lib.cq_paged_attention(q, sb, sh, dt, b, hq, hk, d, k, v, cdt, pages, page, sp, shd, st, table, rows, width,
                                      ts, None, lens, 1.0, window, sinks, None, None, out, None, ws, wsn, None)
    assert call(dt=2) == L.CQ_ERR_ARG and call(dt=0, cdt=1) == L.CQ_ERR_ARG and call(cdt=9) == L.CQ_ERR_ARG
    assert call(window=-1) == L.CQ_ERR_ARG and call(sinks=-1) == L.CQ_ERR_ARG
    assert call(page=12) == L.CQ_ERR_SHAPE and call(page=4) == L.CQ_ERR_SHAPE and call(pages=0) == L.CQ_ERR_SHAPE
    assert call(ts=3) == L.CQ_ERR_SHAPE and call(hq=7) == L.CQ_ERR_SHAPE and call(d=96) == L.CQ_ERR_SHAPE
    assert call(b=70000) == L.CQ_ERR_SHAPE and call(wsn=-1) == L.CQ_ERR_SHAPE
    assert call(q=None) == L.CQ_ERR_ARG and call(lens=None) == L.CQ_ERR_ARG and call(table=None) == L.CQ_ERR_ARG
    assert call(q=ctypes.c_void_p(8)) == L.CQ_ERR_ALIGN and call(st=129) == L.CQ_ERR_ALIGN
    assert call(cdt=2, st=8) == L.CQ_ERR_ALIGN
    assert call(b=0, q=None, k=None, v=None, lens=None, out=None) == L.CQ_OK


def test_page_argument_checks_need_no_device(lib):
    from comfy_quant_bench_b200 import _lib as L

    def update(rows=4, width=8, ts=8, pages=10, page=16, nf=1, nk=0, nr=0, count=1, layers=0, lb=0, pb=0, wsn=1 << 20,
               table=VP, start=VP, k=None):
        return lib.cq_pages_update(table, rows, width, ts, VP, VP, pages, page, VP, nf, VP, VP, nk, VP, nr, None, count,
                                   start, VP, k, k, layers, lb, pb, VP, wsn, None)
    assert update(page=10) == L.CQ_ERR_SHAPE and update(ts=7) == L.CQ_ERR_SHAPE and update(nf=5) == L.CQ_ERR_SHAPE
    assert update(nr=1, count=-1) == L.CQ_ERR_SHAPE and update(nr=1, wsn=8) == L.CQ_ERR_SHAPE
    assert update(nr=1, layers=2, lb=64, pb=8, k=VP) == L.CQ_ERR_SHAPE
    assert update(nr=1, layers=2, lb=64, pb=32, k=None) == L.CQ_ERR_ARG
    assert update(table=None) == L.CQ_ERR_ARG and update(nr=1, start=None) == L.CQ_ERR_ARG
    assert update(pages=1 << 22) == L.CQ_ERR_CAPACITY
    assert update(nf=0) == L.CQ_OK
    assert lib.cq_pages_workspace_bytes(100, 7) >= 4 * 114 and lib.cq_pages_workspace_bytes(-1, 0) == -1
    assert lib.cq_pages_compact(VP, 4, 8, 8, VP, 8, VP, VP, 10, VP, None, None, 0, 0, 0, VP, 8, None) == L.CQ_ERR_SHAPE
    assert lib.cq_pages_compact(VP, 4, 8, 8, VP, 7, VP, VP, 10, VP, None, None, 0, 0, 0, VP, 40, None) == L.CQ_ERR_SHAPE
    assert lib.cq_pages_compact(VP, 4, 8, 8, VP, 8, None, VP, 10, VP, None, None, 0, 0, 0, VP, 40, None) == L.CQ_ERR_ARG
    assert lib.cq_pages_compact(VP, 4, 8, 8, VP, 8, VP, VP, 1 << 22, VP, None, None, 0, 0, 0, VP, 1 << 30, None) == \
        L.CQ_ERR_CAPACITY

    def append(dt=0, cdt=0, t=1, hk=2, d=64, page=16, pos=VP, k=VP, sl=0):
        return lib.cq_kv_append(k, sl, 128, 64, VP, 0, 128, 64, dt, 1, t, hk, d, VP, VP, cdt, 10, page, 0, 2048, 1024, 64,
                                VP, 4, 8, 8, VP, pos, None, None, None)
    assert append(dt=2) == L.CQ_ERR_ARG and append(cdt=1) == L.CQ_ERR_ARG and append(pos=None) == L.CQ_ERR_ARG
    assert append(page=3) == L.CQ_ERR_SHAPE and append(d=12) == L.CQ_ERR_SHAPE and append(t=-1) == L.CQ_ERR_SHAPE
    assert append(k=ctypes.c_void_p(258)) == L.CQ_ERR_ALIGN and append(sl=4) == L.CQ_ERR_ALIGN
    assert append(t=0, k=None) == L.CQ_OK


def test_operators_reject_cpu_tensors():
    from comfy_quant_bench_b200 import kvcache, ops
    with pytest.raises(ValueError, match="CUDA"):
        ops.w4a16_linear(torch.zeros(1, 128, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.int8),
                         torch.zeros(1, 8, dtype=torch.bfloat16), torch.zeros(1, 8, dtype=torch.bfloat16))
    c = kvcache.PagedKVCache(1, 4, 2, 64, 2, 40, device="cpu")
    assert c.block_table.shape == (2, 3) and int(c.block_table.max()) == -1
    one = torch.zeros(1, dtype=torch.int32)
    new = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    for bad in (lambda: c.reserve(one, 1), lambda: c.free(one), lambda: c.fork(one, one), lambda: c.compact(),
                lambda: c.branch(one, one + 1, 1), lambda: c.append(0, new, new, one, one),
                lambda: c.attend(0, new, rows=one)):
        with pytest.raises(ValueError, match="CUDA"):
            bad()


def test_refusals_say_what_is_wrong():
    from comfy_quant_bench_b200 import kvcache, ops
    x, q = torch.zeros(2, 256, dtype=torch.bfloat16), torch.zeros(16, 128, dtype=torch.int8)
    s, b = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(16, dtype=torch.bfloat16)
    k, n = torch.zeros(6, 2, 16, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    t, query = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    for says, call in (("bf16 or f16, got Float", lambda: ops.w4a16_linear(x.float(), q, s, s, b, group_size=64)),
                       ("K=128 does not match qweight K=256", lambda: ops.w4a16_linear(x[:, :128], q, s, s, b, group_size=64)),
                       ("divide K=256, got 16", lambda: ops.w4a16_linear(x, q, s, s, b, group_size=16)),
                       (r"\[4, 16\]", lambda: ops.w4a16_linear(x, q, s.float(), s, b, group_size=64)),
                       ("16 elements", lambda: ops.w4a16_linear(x, q, s, s, b[:5], group_size=64)),
                       ("multiple of kv_heads", lambda: kvcache.paged_attention(query[:, :3], k, k, t, n)),
                       ("64, 128 or 256", lambda: kvcache.paged_attention(query[..., :32], k, k, t, n)),
                       ("one entry per table row", lambda: kvcache.paged_attention(query, k, k, t, n[:1])),
                       ("2 queries for 1", lambda: kvcache.paged_attention(query, k, k, t[:1], n[:1])),
                       ("do not fit", lambda: kvcache.append_kv(query, query, k, k, t, n, n))):
        with pytest.raises(ValueError, match=says):
            call()


def test_awq_layout_is_registered_on_request():
    import types

    from comfy_quant_bench_b200 import layout
    fake = types.SimpleNamespace(QUANT_ALGOS={}, layouts={}, __name__="comfy.quant_ops")
    fake.register_layout_class = lambda name, cls: fake.layouts.__setitem__(name, cls)
    layout.register(target=fake)
    assert "awq_w4a16" not in fake.QUANT_ALGOS
    assert layout.register_w4a16(target=fake) == "comfy.quant_ops"
    algo = fake.QUANT_ALGOS["awq_w4a16"]
    assert algo["comfy_tensor_layout"] in fake.layouts and not algo["quantize_input"]
    params = algo["params_from_state_dict"]("l", None, None, {"weight_scale": 1, "weight_zeros": 2}.get,
                                            {"format": "awq_w4a16", "group_size": 32})
    assert params == {"scale": 1, "zeros": 2, "group_size": 32}
    with pytest.raises(ValueError):
        algo["params_from_state_dict"]("l", None, None, lambda name: None, {"format": "awq_w4a16"})


def test_written_tables_have_rows_of_their_own():
    """A view whose rows share memory cannot be written row by row: refused before anything else."""
    from comfy_quant_bench_b200 import kvcache
    k, refs = torch.zeros(1, 6, 1, 16, 64, dtype=torch.bfloat16), torch.zeros(6, dtype=torch.int32)
    lens, rows = torch.zeros(3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    plain = torch.zeros(3, 4, dtype=torch.int32)
    for view in (plain[:1].expand(3, 4), torch.zeros(8, dtype=torch.int32).as_strided((3, 4), (2, 1))):
        for name, call in (("block_table", lambda: kvcache.free_rows(view, lens, refs, rows, 16)),
                           ("block_table", lambda: kvcache.fork_rows(view, lens, refs, rows, rows + 1, 16)),
                           ("block_table", lambda: kvcache.reserve_tokens(view, lens, refs, rows, 1, k, k)),
                           ("block_table", lambda: kvcache.branch_rows(view, lens, refs, rows, rows + 1, 1, k, k)),
                           ("out_table", lambda: kvcache.compact_pages(plain, refs, k, k, out_table=view)),
                           ("out_table", lambda: kvcache.compact_pages(view, refs, k, k, out_table=view))):
            with pytest.raises(ValueError, match=f"{name} is written, but its rows share memory"):
                call()
    for fine in (plain[:1], torch.zeros(3, 9, dtype=torch.int32)[:, 2:6]):       # one row of any stride, rows further apart
        with pytest.raises(ValueError, match="CUDA"):
            kvcache.free_rows(fine, lens[:len(fine)], refs, rows, 16)


def test_textgen_has_a_rotary_entry_for_every_position(monkeypatch):
    """A row's last page may reach past max_tokens, and a prompt may not: an index past the table would fault the device."""
    from comfy_quant_bench_b200 import textgen
    monkeypatch.setattr(textgen.ops, "quantize_affine_w4_weight", lambda w, group: (w, w, w))
    m = textgen.TextModel(textgen.TextConfig(vocab=8, hidden=64, layers=1, heads=1, kv_heads=1, head_dim=64, ffn=64, group_size=64,
                                             max_tokens=150, rows=2, pages=4, page_size=16), device="cpu")
    positions = m.cache.block_table.shape[1] * m.cache.page_size           # what a row can reserve
    assert positions == 160 and m.rope.shape == (positions, 32, 2)
    with pytest.raises(ValueError, match="prompt of 151 tokens for rows of max_tokens = 150"):
        m.prompt(torch.zeros(151, dtype=torch.long), 0)


@pytest.mark.parametrize("pages", [(1 << 31) - 1, (1 << 31) - 31, 1 << 30])
def test_pools_near_the_integer_limit_are_refused_as_too_large(lib, pages):
    from comfy_quant_bench_b200 import _lib as L
    assert lib.cq_pages_update(VP, 4, 8, 8, VP, VP, pages, 16, VP, 1, None, None, 0, None, 0, None, 0, None, None, None, None, 0,
                               0, 0, None, 0, None) == L.CQ_ERR_CAPACITY
    assert lib.cq_pages_compact(VP, 4, 8, 8, VP, 8, VP, VP, pages, VP, None, None, 0, 0, 0, VP, 1 << 40, None) == \
        L.CQ_ERR_CAPACITY


def test_a_list_left_out_is_refused():
    """None in place of a list of rows; the page calls take their lists as optional ones."""
    from comfy_quant_bench_b200 import kvcache
    table, lens, refs = (torch.zeros(s, dtype=torch.int32) for s in ((3, 4), 3, 6))
    k, one = torch.zeros(1, 6, 1, 16, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: kvcache.free_rows(table, lens, refs, None, 16), lambda: kvcache.fork_rows(table, lens, refs, one, None, 16),
                 lambda: kvcache.fork_rows(table, lens, refs, None, one, 16),
                 lambda: kvcache.fork_rows(table, lens, refs, None, None, 16),
                 lambda: kvcache.reserve_tokens(table, lens, refs, None, 1, k, k),
                 lambda: kvcache.reserve_tokens(table, lens, refs, None, one, k, k),
                 lambda: kvcache.reserve_tokens(table, lens, refs, one, 1, k, None),
                 lambda: kvcache.branch_rows(table, lens, refs, None, one, 1, k, k),
                 lambda: kvcache.branch_rows(table, lens, refs, one, None, one, k, k)):
        with pytest.raises(ValueError, match="int32 tensor|caches are needed"):
            call()


def test_a_cache_asks_its_own_device_for_refusals(monkeypatch):
    """A cache on another device than the current one: the status word and the stream are that device's."""
    import contextlib
    import types

    from comfy_quant_bench_b200 import kvcache
    current, asked = ["cuda:0"], []

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], current[0] if d is None else str(d)
        yield
        current[0] = before

    def take(stream):
        asked.append((current[0], stream))
        return (7, 103) if current[0] == "cuda:1" else (0, 0)
    monkeypatch.setattr(kvcache.torch.cuda, "device", device)
    monkeypatch.setattr(kvcache.torch.cuda, "current_stream", lambda: types.SimpleNamespace(cuda_stream="of " + current[0]))
    monkeypatch.setattr(kvcache._lib, "take_device_status", take)
    c = kvcache.PagedKVCache(1, 4, 1, 64, 2, 32, device="cpu")
    c.k = types.SimpleNamespace(device=torch.device("cuda:1"))
    with pytest.raises(RuntimeError, match="reserve"):
        c.check()
    kvcache.check()
    assert asked == [("cuda:1", "of cuda:1"), ("cuda:0", "of cuda:0")] and current == ["cuda:0"]

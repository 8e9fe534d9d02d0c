"""Decode-side operators against 64-bit implementations: the W4A16 linear, attention of one new token over a paged
cache, and the cache's bookkeeping and page movement.

Bounds.  u is the unit roundoff of the output type (2^-8 bf16, 2^-11 f16).
* Linear: one output rounding, and fp32 products and sums with at most 300 roundings (2^-23 each, room for tensor
  cores that truncate) on the way of any term: |y - exact| <= u |exact| + 300 2^-23 (sum |x| (|q - 8| |s| + |z|) + |b|).
* Attention: a score's fp32 error is at most (D + 16) 2^-23 scale sum |q| |k|; it and the exponential (2^-20, its
  argument's rounding among it) enter numerator and denominator; weights may be split into two 16-bit parts (2^-16):
  |o - exact| <= u |exact| + A (2 max_j err_j + 2^-14), A = sum p |v| / sum p.
* Over a whole output the kernel may add at most 2^-14 of relative L2 error to what rounding the exact result costs.
Pages, tables, counts and copied data are compared exactly.
"""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
FP8 = torch.float8_e4m3fn


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


def _status():
    from comfy_quant_bench_b200 import _lib
    torch.cuda.synchronize()
    return _lib.take_device_status()


def _hold(got, want, slack, dtype):
    """Element bound and the L2 bound of the module's docstring; NaN and infinities have to agree in place."""
    assert got.dtype == dtype and got.shape == want.shape
    g = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(g), fine)
    assert torch.equal(torch.isnan(g), torch.isnan(want))
    g, w = torch.where(fine, g, 0.0), torch.where(fine, want, 0.0)
    tiny = 2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -24      # spacing of the subnormal outputs
    over = (g - w).abs() - (U[dtype] * w.abs() + slack + tiny)
    assert float(over.max()) <= 0 if over.numel() else True
    if w.numel() and float(w.norm()) > 0:
        once = float((w.to(dtype).double() - w).norm() / w.norm())
        assert float((g - w).norm() / w.norm()) <= 1.05 * once + 2.0 ** -14


# ----------------------------------------------------------------------------------------------------------
# W4A16 linear
# ----------------------------------------------------------------------------------------------------------

def _linear_problem(m, k, n, group, dtype, seed=0, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed + m + 7 * k + n)
    x = torch.randn(m, k, generator=g, device="cuda").to(dtype)
    q = torch.randint(-128, 128, (n, k // 2), generator=g, device="cuda", dtype=torch.int8)
    s = (0.01 * torch.rand(k // group, n, generator=g, device="cuda")).bfloat16()
    z = (0.01 * torch.randn(k // group, n, generator=g, device="cuda")).bfloat16()
    b = torch.randn(n, generator=g, device="cuda").to(dtype) if bias else None
    return x, q, s, z, b


def _linear_exact(x, q, s, z, b, group):
    u = q.view(torch.uint8)
    codes = torch.stack([u & 15, u >> 4], -1).reshape(u.shape[0], -1).double() - 8
    s, z = (t.double().t().repeat_interleave(group, 1) for t in (s, z))
    y, mag = x.double() @ (codes * s + z).t(), x.double().abs() @ (codes.abs() * s.abs() + z.abs()).t()
    return (y, mag) if b is None else (y + b.double(), mag + b.double().abs())


def _linear_holds(ops, x, q, s, z, b, group, y=None):
    if y is None:
        y = ops.w4a16_linear(x, q, s, z, b, group_size=group)
    want, mag = _linear_exact(x, q, s, z, b, group)
    _hold(y, want, 300 * 2.0 ** -23 * mag, x.dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 33, 64, 65])
def test_linear_token_counts(ops, m, group, dtype):
    _linear_holds(ops, *_linear_problem(m, 1152, 200, group, dtype), group)


@pytest.mark.parametrize("k,n,group", [(32, 1, 32), (32, 17, 32), (64, 16, 64), (96, 33, 32), (128, 1, 128), (160, 15, 32),
                                       (192, 129, 64), (512, 1001, 128), (2080, 31, 32), (8064, 47, 128), (32768, 65, 64)])
@pytest.mark.parametrize("m", [1, 5, 20])
def test_linear_odd_sizes(ops, m, k, n, group):
    _linear_holds(ops, *_linear_problem(m, k, n, group, torch.bfloat16, bias=n % 2 == 0), group)


@pytest.mark.parametrize("m,k,n", [(1, 4096, 12288), (4, 8192, 4096), (24, 4096, 8192), (300, 1024, 520)])
def test_linear_ordinary_sizes(ops, m, k, n):
    _linear_holds(ops, *_linear_problem(m, k, n, 128, torch.bfloat16), 128)


@pytest.mark.parametrize("m,k,n,group", [(33, 4160, 19001, 32), (64, 2112, 19100, 64), (70, 1152, 18950, 128), (40, 9600, 300, 32)])
def test_linear_many_tokens_deep_and_wide(ops, m, k, n, group):
    """More blocks of zeros and chunks than the rings hold, whole K and split, last chunks that are not full."""
    x, q, s, z, b = _linear_problem(m, k, n, group, torch.float16 if m == 64 else torch.bfloat16)
    y = ops.w4a16_linear(x, q, s, z, b, group_size=group)
    _linear_holds(ops, x, q, s, z, b, group, y)
    for _ in range(3):
        assert torch.equal(ops.w4a16_linear(x, q, s, z, b, group_size=group), y)
    assert _status()[0] == 0


def test_linear_strided_rows_leading_dims_and_out(ops):
    x, q, s, z, b = _linear_problem(6, 512, 96, 64, torch.float16)
    wide = torch.zeros(6, 1200, dtype=torch.float16, device="cuda")
    for off in (0, 8, 3):                                   # the last one is not 16-byte aligned
        wide[:, off:off + 512] = x
        _linear_holds(ops, x, q, s, z, b, 64, ops.w4a16_linear(wide[:, off:off + 512], q, s, z, b, group_size=64))
    y = ops.w4a16_linear(x.view(2, 3, 512), q, s, z, b, group_size=64)
    assert y.shape == (2, 3, 96)
    assert torch.equal(y.view(6, 96), ops.w4a16_linear(x, q, s, z, b, group_size=64))
    every_other = torch.empty(12, 512, dtype=torch.float16, device="cuda")[::2].copy_(x)
    out = torch.full((6, 96), 7.0, dtype=torch.float16, device="cuda")
    assert ops.w4a16_linear(every_other, q, s, z, b, group_size=64, out=out) is out
    assert torch.equal(out, y.view(6, 96))


def test_linear_one_row_is_the_same_in_every_batch_and_again(ops):
    x, q, s, z, b = _linear_problem(64, 2048, 300, 128, torch.bfloat16)
    whole = ops.w4a16_linear(x, q, s, z, b)
    for _ in range(3):
        assert torch.equal(ops.w4a16_linear(x, q, s, z, b), whole)


def test_linear_nonfinite_tokens_stay_in_their_rows(ops):
    x, q, s, z, b = _linear_problem(9, 256, 40, 64, torch.bfloat16)
    clean = ops.w4a16_linear(x, q, s, z, b, group_size=64)
    x[2, 5], x[7, 200] = float("nan"), float("nan")
    y = ops.w4a16_linear(x, q, s, z, b, group_size=64)
    hit = torch.zeros(9, dtype=torch.bool, device="cuda")
    hit[[2, 7]] = True
    assert bool(torch.isnan(y[hit]).all()) and torch.equal(y[~hit], clean[~hit])


def test_linear_large_activations_f16(ops):
    """Group sums far beyond f16's range stay in fp32; only the output has to fit."""
    x, q, s, z, _ = _linear_problem(3, 1024, 64, 32, torch.float16)
    x = (x * 15000).clamp(-65504, 65504)
    _linear_holds(ops, x, q, (s.float() * 2.0 ** -12).bfloat16(), (z.float() * 2.0 ** -12).bfloat16(), None, 32)


def test_linear_empty(ops):
    x, q, s, z, b = _linear_problem(1, 128, 16, 128, torch.bfloat16)
    assert ops.w4a16_linear(x[:0], q, s, z, b).shape == (0, 16)
    assert ops.w4a16_linear(x, q[:0], s[:, :0].contiguous(), z[:, :0].contiguous(), b[:0]).shape == (1, 0)


def test_linear_refusals(ops):
    x, q, s, z, b = _linear_problem(2, 256, 16, 64, torch.bfloat16)
    ok = dict(group_size=64)
    for bad in (lambda: ops.w4a16_linear(x.float(), q, s, z, b, **ok),
                lambda: ops.w4a16_linear(x[:, :128], q, s, z, b, **ok),
                lambda: ops.w4a16_linear(x, q, s, z, b, group_size=128),
                lambda: ops.w4a16_linear(x, q, s, z, b, group_size=16),
                lambda: ops.w4a16_linear(x, q, s.float(), z, b, **ok),
                lambda: ops.w4a16_linear(x, q, s.t(), z, b, **ok),
                lambda: ops.w4a16_linear(x, q.int(), s, z, b, **ok),
                lambda: ops.w4a16_linear(x, q.t().contiguous().t(), s, z, b, **ok),
                lambda: ops.w4a16_linear(x, q, s, z, b[:5], **ok),
                lambda: ops.w4a16_linear(x, q, s.cpu(), z, b, **ok),
                lambda: ops.w4a16_linear(x, q, s, z, b, out=torch.empty(2, 16, device="cuda"), **ok)):
        with pytest.raises(ValueError):
            bad()


def test_linear_on_another_stream(ops):
    x, q, s, z, b = _linear_problem(4, 1024, 512, 128, torch.bfloat16)
    want = ops.w4a16_linear(x, q, s, z, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.w4a16_linear(x, q, s, z, b)
    side.synchronize()
    assert torch.equal(got, want)


# ----------------------------------------------------------------------------------------------------------
# attention of one new token
# ----------------------------------------------------------------------------------------------------------

def _cache(lens, hk, page, d, cache_type, seed, width=None, poison=True, token_major=False):
    """Caches over randomly ordered pages; what lies past a row's end is NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = random.Random(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    order = list(range(pages))
    host.shuffle(order)
    width = width or max([1] + need)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    made = []
    for _ in range(2):
        x = torch.randn(pages, hk, page, d, generator=g, device="cuda")
        if poison:
            for r, n in enumerate(lens):
                if n % page:
                    x[int(table[r, n // page]), :, n % page:] = float("nan")
            for p in order[at:]:
                x[p] = float("nan")
        x = (x * 20).to(FP8) if cache_type == FP8 else x.to(cache_type)
        if token_major:
            x = (x.view(torch.uint8) if cache_type == FP8 else x).transpose(1, 2).contiguous().transpose(1, 2)
            x = x.view(FP8) if cache_type == FP8 else x
        made.append(x)
    return made[0], made[1], table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


def _attention_exact(q, k, v, table, lens, scale, window=0, sinks=0, ks=None, vs=None, rows=None):
    b, hq, d = q.shape
    pages, hk, page, _ = k.shape
    out = torch.zeros(b, hq, d, dtype=torch.float64, device="cuda")
    slack, lse = torch.zeros_like(out), torch.full((b, hq), -math.inf, dtype=torch.float64, device="cuda")
    k, v = k.float(), v.float()
    for i in range(b):
        r = i if rows is None else int(rows[i])
        n = int(lens[r]) if 0 <= r < len(lens) else 0
        j = torch.arange(max(0, min(n, table.shape[1] * page)), device="cuda")
        if window:
            j = j[(j >= n - window) | (j < sinks)]
        if not len(j):
            continue
        pg = table[r].long()[j // page]
        j, pg = j[(pg >= 0) & (pg < pages)], pg[(pg >= 0) & (pg < pages)]
        if not len(j):
            continue
        for h in range(hk):
            at = slice(h * (hq // hk), (h + 1) * (hq // hk))
            kk, vv = k[pg, h, j % page].double(), v[pg, h, j % page].double()
            if ks is not None:
                kk, vv = kk * ks[h].double(), vv * vs[h].double()
            qq = q[i, at].double()
            s = qq @ kk.t() * scale
            p = torch.softmax(s, -1)
            out[i, at] = p @ vv
            err = scale * float((qq.abs() @ kk.abs().t()).max()) * (d + 16) * 2.0 ** -23
            slack[i, at] = (p @ vv.abs()) * (2 * err + 2.0 ** -14)
            lse[i, at] = torch.logsumexp(s, -1)
    return out, slack, lse


def _attention_holds(kv, q, k, v, table, lens, rows=None, **kw):
    got, lse = kv.paged_attention(q, k, v, table, lens, rows=rows, return_lse=True, **kw)
    scale = kw.get("scale") or q.shape[-1] ** -0.5
    want, slack, want_lse = _attention_exact(q, k, v, table, lens, scale, kw.get("window", 0), kw.get("sinks", 0),
                                             kw.get("k_scale"), kw.get("v_scale"), rows)
    _hold(got, want, slack, q.dtype)
    seen = torch.isfinite(want_lse)
    assert torch.equal(torch.isfinite(lse), seen) and bool((lse[~seen] == -math.inf).all())
    assert float((lse.double() - want_lse)[seen].abs().max() if bool(seen.any()) else 0.0) <= 2.0 ** -10
    assert _status() == (0, 0)
    return got


def _query(b, hq, d, dtype, seed, size=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (size * torch.randn(b, hq, d, generator=g, device="cuda")).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [8, 16, 64, 1024])
def test_attention_types_dims_pages(kv, dtype, fp8, d, page):
    lens = [1, 0, page, page + 1, 2 * page - 1, 37, 300]
    k, v, table, n = _cache(lens, 2, page, d, FP8 if fp8 else dtype, seed=d + page)
    kw = {}
    if fp8:
        kw = {"k_scale": torch.tensor([0.05, 0.02], device="cuda"), "v_scale": torch.tensor([0.3, 0.04], device="cuda")}
    _attention_holds(kv, _query(len(lens), 8, d, dtype, 1), k, v, table, n, **kw)


@pytest.mark.parametrize("hq,hk", [(1, 1), (3, 3), (4, 1), (7, 1), (8, 1), (9, 1), (14, 2), (16, 1), (17, 1), (24, 2), (40, 1),
                                   (64, 8), (96, 2)])
def test_attention_head_groups(kv, hq, hk):
    lens = [129, 5, 511]
    k, v, table, n = _cache(lens, hk, 16, 128, torch.bfloat16, seed=hq)
    _attention_holds(kv, _query(3, hq, 128, torch.bfloat16, hq), k, v, table, n)


@pytest.mark.parametrize("n", list(range(1, 36)) + [63, 64, 65, 127, 128, 129, 255, 256, 257, 1000, 1023, 1025, 4097])
def test_attention_lengths(kv, n):
    k, v, table, lens = _cache([n], 2, 16, 64, torch.float16, seed=n, width=-(-n // 16) + 3)
    _attention_holds(kv, _query(1, 10, 64, torch.float16, n), k, v, table, lens)


@pytest.mark.parametrize("b,n,hk", [(1, 30011, 1), (1, 70000, 4), (3, 20000, 2), (2, 131, 8)])
def test_attention_long_and_split(kv, b, n, hk):
    lens = [n - 777 * i for i in range(b)] if n > 2000 else [n] * b
    k, v, table, ln = _cache(lens, hk, 64, 128, torch.bfloat16, seed=n)
    q = _query(b, 7 * hk, 128, torch.bfloat16, n, 3.0)
    a = _attention_holds(kv, q, k, v, table, ln)
    for _ in range(3):                                    # the join's order is fixed
        assert torch.equal(kv.paged_attention(q, k, v, table, ln), a)


@pytest.mark.parametrize("b,n,hk,d", [(40, 700, 8, 64), (40, 1300, 8, 64), (30, 1000, 8, 128), (38, 200, 8, 64), (5, 900, 8, 128),
                                      (10, 1500, 8, 64), (20, 900, 16, 64), (1, 600, 2, 256), (33, 1536, 9, 64), (1, 8300, 1, 64)])
def test_attention_ways_to_deal_the_work(kv, b, n, hk, d):
    """Runs, whole segments and clusters, at and past the sizes where one takes over from another; ragged and empty rows."""
    host = random.Random(b * n)
    lens = [n if i == 0 else host.choice([0, 1, n, n - 1, host.randint(0, n)]) for i in range(b)]
    k, v, table, ln = _cache(lens, hk, 16, d, torch.bfloat16, seed=n)
    q = _query(b, 2 * hk, d, torch.bfloat16, b)
    a = _attention_holds(kv, q, k, v, table, ln)
    assert torch.equal(kv.paged_attention(q, k, v, table, ln), a)


def test_attention_many_ragged_rows(kv):
    host = random.Random(5)
    lens = [host.choice([0, 1, 15, 16, 17, host.randint(1, 700), host.randint(1, 3000)]) for _ in range(150)]
    k, v, table, n = _cache(lens, 2, 16, 64, torch.bfloat16, seed=9)
    _attention_holds(kv, _query(150, 6, 64, torch.bfloat16, 3), k, v, table, n)


def test_attention_more_rows_than_one_pass_of_the_schedule(kv):
    lens = [(i * 7) % 40 for i in range(1500)]
    k, v, table, n = _cache(lens, 1, 8, 64, torch.float16, seed=2)
    _attention_holds(kv, _query(1500, 2, 64, torch.float16, 3), k, v, table, n)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 2), (16, 4), (17, 33), (64, 4), (100, 1000), (4096, 4), (300, 0)])
def test_attention_window_and_first_tokens(kv, window, sinks):
    lens = [1, 2, 16, 17, 90, 300, 1111, 5000]
    k, v, table, n = _cache(lens, 2, 16, 128, torch.bfloat16, seed=window)
    _attention_holds(kv, _query(len(lens), 6, 128, torch.bfloat16, sinks), k, v, table, n, window=window, sinks=sinks)


def test_attention_masked_tokens_may_hold_anything(kv):
    """Tokens outside the window, past the end and in unused pages: NaN, infinities and the type's lowest value."""
    lens = [200, 75]
    for fill in (float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min):
        k, v, table, n = _cache(lens, 1, 16, 64, torch.bfloat16, seed=4, poison=False)
        for t in (k, v):
            for r in range(2):
                for j in range(lens[r], -(-lens[r] // 16) * 16):
                    t[int(table[r, j // 16]), :, j % 16] = fill
                for j in range(3, lens[r] - 40):
                    t[int(table[r, j // 16]), :, j % 16] = fill
        _attention_holds(kv, _query(2, 4, 64, torch.bfloat16, 8), k, v, table, n, window=40, sinks=3)


def test_attention_visible_nan_and_overflow(kv):
    k, v, table, n = _cache([40, 40], 1, 16, 64, torch.float16, seed=4)
    v[int(table[0, 1]), 0, 3, 7] = float("nan")
    out = kv.paged_attention(_query(2, 2, 64, torch.float16, 1), k, v, table, n)
    assert bool(torch.isnan(out[0, :, 7]).all()) and int(torch.isnan(out).sum()) == 2
    k[int(table[0, 1]), 0, 3, 7] = float("nan")
    out = kv.paged_attention(_query(2, 2, 64, torch.float16, 1), k, v, table, n)
    assert bool(torch.isnan(out[0]).all()) and not bool(torch.isnan(out[1]).any())


def test_attention_scores_far_apart(kv):
    """One key takes all the weight, and all keys far below zero: the maximum is subtracted first."""
    k, v, table, n = _cache([600], 1, 16, 64, torch.bfloat16, seed=6)
    q = _query(1, 3, 64, torch.bfloat16, 1, 60.0)
    _attention_holds(kv, q, k, v, table, n)
    _attention_holds(kv, q, k, v, table, n, scale=5.0)
    k.copy_(torch.where(torch.isnan(k), k, -k.abs() * 30))
    _attention_holds(kv, q.abs() + 1, k, v, table, n)


def test_attention_missing_pages_bad_rows_and_long_lens(kv):
    lens = [100, 64, 33, 48]
    k, v, table, n = _cache(lens, 2, 16, 64, torch.bfloat16, seed=3)
    table[0, 2], table[1, :], table[2, 0] = -1, -1, 10 ** 6
    n[3] = 10 ** 9                                        # longer than the table is wide
    table[3, 3:] = -1
    got = _attention_holds(kv, _query(4, 4, 64, torch.bfloat16, 1), k, v, table, n)
    assert bool((got[1] == 0).all())
    n[0] = -5
    assert bool((kv.paged_attention(_query(4, 4, 64, torch.bfloat16, 1), k, v, table, n)[0] == 0).all())
    rows = torch.tensor([2, -1, 4, 0, 2, 1], dtype=torch.int32, device="cuda")
    _attention_holds(kv, _query(6, 4, 64, torch.bfloat16, 1), k, v, table, n, rows=rows)


def test_attention_strides(kv):
    """Queries as a slice of a wider projection, token-major caches, a layer of a larger cache, a wide table."""
    lens = [70, 19, 257]
    for ct, kw in ((torch.bfloat16, {}), (FP8, {"k_scale": torch.full((2,), 0.05, device="cuda"),
                                                "v_scale": torch.full((2,), 0.05, device="cuda")})):
        k, v, table, n = _cache(lens, 2, 16, 128, ct, seed=1)
        proj = torch.randn(3, 20, 128, device="cuda").bfloat16()
        q = proj[:, 3:11]
        want = _attention_holds(kv, q, k, v, table, n, **kw)
        for shifted in (proj.view(3, 2560)[:, 4:4 + 1024].view(3, 8, 128), proj[:, ::2][:, :8]):
            _attention_holds(kv, shifted, k, v, table, n, **kw)
        km, vm, tm, nm = _cache(lens, 2, 16, 128, ct, seed=1, token_major=True)
        assert torch.equal(kv.paged_attention(q, km, vm, tm, nm, **kw), want)
        big = torch.full((3, 9), -1, dtype=torch.int32, device="cuda").repeat(1, 8)
        big[:, 5:5 + table.shape[1]] = table
        assert torch.equal(kv.paged_attention(q, k, v, big[:, 5:5 + table.shape[1]], n, **kw), want)
        out = torch.empty_like(want)
        assert kv.paged_attention(q, k, v, table, n, out=out, **kw) is out and torch.equal(out, want)


def test_attention_offsets_past_31_bits(kv):
    """A layer stack whose last page lies more than 2^31 elements into the cache."""
    page_elems = 16 * 128
    pages = (1 << 31) // page_elems + 40
    k = torch.empty(pages, 1, 16, 128, dtype=FP8, device="cuda")
    v = torch.empty(pages, 1, 16, 128, dtype=FP8, device="cuda")
    used = [pages - 1, 0, pages - 33, pages // 2]
    for i, p in enumerate(used):
        for j, t in enumerate((k, v)):
            t[p] = (30 * torch.randn(1, 16, 128, generator=torch.Generator("cuda").manual_seed(2 * i + j), device="cuda")).to(FP8)
    table = torch.tensor([used], dtype=torch.int32, device="cuda")
    n = torch.tensor([61], dtype=torch.int32, device="cuda")
    sc = torch.tensor([0.02], device="cuda")
    small_k, small_v = (torch.stack([t[p].view(torch.uint8) for p in used]).view(FP8) for t in (k, v))
    q = _query(1, 4, 128, torch.bfloat16, 1)
    want = _attention_holds(kv, q, small_k, small_v, torch.arange(4, dtype=torch.int32, device="cuda")[None], n, k_scale=sc, v_scale=sc)
    assert torch.equal(kv.paged_attention(q, k, v, table, n, k_scale=sc, v_scale=sc), want)


def test_attention_empty_and_refusals(kv):
    k, v, table, n = _cache([20, 20], 2, 16, 64, torch.bfloat16, seed=1)
    q = _query(2, 4, 64, torch.bfloat16, 1)
    assert kv.paged_attention(q[:0], k, v, table, n).shape == (0, 4, 64)
    assert bool((kv.paged_attention(q, k, v, table[:, :0], n) == 0).all())
    for bad in (lambda: kv.paged_attention(q.float(), k, v, table, n), lambda: kv.paged_attention(q.half(), k, v, table, n),
                lambda: kv.paged_attention(q[:, :3], k, v, table, n), lambda: kv.paged_attention(q[..., :32], k, v, table, n),
                lambda: kv.paged_attention(q, k, v[:1], table, n), lambda: kv.paged_attention(q, k, v.half(), table, n),
                lambda: kv.paged_attention(q, k, v, table.long(), n), lambda: kv.paged_attention(q, k, v, table, n.long()),
                lambda: kv.paged_attention(q, k, v, table, n[:1]), lambda: kv.paged_attention(q, k, v, table[:1], n[:1]),
                lambda: kv.paged_attention(q, k, v, table, n, window=-1), lambda: kv.paged_attention(q, k, v, table, n, sinks=-1),
                lambda: kv.paged_attention(q, k, v, table, n, k_scale=torch.ones(2, device="cuda")),
                lambda: kv.paged_attention(q, k.cpu(), v.cpu(), table, n),
                lambda: kv.paged_attention(q, k[:, :, :12], v[:, :, :12], table, n),
                lambda: kv.paged_attention(q, k, v, table, n, rows=torch.zeros(1, dtype=torch.int32, device="cuda")),
                lambda: kv.paged_attention(q, k, v, table, n, out=torch.empty(2, 4, 64, device="cuda"))):
        with pytest.raises(ValueError):
            bad()


def test_attention_in_a_graph_follows_the_state(kv):
    """A captured step reads lengths and tables at replay."""
    k, v, table, n = _cache([500, 900], 2, 16, 128, torch.bfloat16, seed=1)
    q = _query(2, 8, 128, torch.bfloat16, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv.paged_attention(q, k, v, table, n)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kv.paged_attention(q, k, v, table, n)
    for lens in ([500, 900], [1, 0], [499, 16]):
        n.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, kv.paged_attention(q, k, v, table, n))


# ----------------------------------------------------------------------------------------------------------
# pages
# ----------------------------------------------------------------------------------------------------------

class Model:
    """The cache as its documentation describes it, on the host: bookkeeping and the content of every slot."""

    def __init__(self, layers, pages, hk, d, rows, width, page):
        self.page, self.width = page, width
        self.table = [[-1] * width for _ in range(rows)]
        self.lens, self.refs = [0] * rows, [0] * pages

    def held(self, r):
        return -(-self.lens[r] // self.page)

    def free(self, rows):
        for r in rows:
            for j in range(self.held(r)):
                self.refs[self.table[r][j]] -= 1
                self.table[r][j] = -1
            self.lens[r] = 0

    def fork(self, src, dst):
        for s, d in zip(src, dst):
            for j in range(self.held(s)):
                self.table[d][j] = self.table[s][j]
                self.refs[self.table[s][j]] += 1
            self.lens[d] = self.lens[s]

    def reserve(self, rows, counts):
        spare = [p for p, c in enumerate(self.refs) if c == 0]
        counted = list(self.refs)
        need = 0
        for r, c in zip(rows, counts):
            if self.lens[r] + c > self.width * self.page:
                return None
            need += -(-(self.lens[r] + c) // self.page) - self.held(r)
            need += bool(c and self.lens[r] % self.page and counted[self.table[r][self.held(r) - 1]] > 1)
        if need > len(spare):
            return None
        start, copies = [], []
        for r, c in zip(rows, counts):
            copies.append([-1, -1])
            last = self.held(r) - 1
            if c and self.lens[r] % self.page and counted[self.table[r][last]] > 1:
                old, new = self.table[r][last], spare.pop(0)
                copies[-1] = [old, new]
                self.refs[old] -= 1
                self.refs[new], self.table[r][last] = 1, new
            start.append(self.lens[r])
            self.lens[r] += c
            for j in range(last + 1, self.held(r)):
                self.table[r][j] = spare.pop(0)
                self.refs[self.table[r][j]] = 1
        return start, copies

    def compact(self):
        live = sum(c > 0 for c in self.refs)
        holes = [p for p in range(live) if self.refs[p] == 0]
        moves = [[p, holes.pop(0)] for p in range(live, len(self.refs)) if self.refs[p]]
        to = dict(moves)
        for a, b in moves:
            self.refs[a], self.refs[b] = 0, self.refs[a]
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return moves

    def agrees(self, c):
        assert c.block_table.tolist() == self.table
        assert c.seq_lens.tolist() == self.lens
        assert c.ref_counts.tolist() == self.refs
        counted = [0] * len(self.refs)
        for row in self.table:
            for p in row:
                if p >= 0:
                    counted[p] += 1
        assert counted == self.refs


def _rows(*r):
    return torch.tensor(list(r), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("seed", range(6))
def test_pages_random_histories(kv, seed):
    """Reserve, append, fork, branch, free and compact at random: the bookkeeping equals the model's after every step
    and every row reads back the tokens that were written to it or to the rows it came from."""
    host = random.Random(seed)
    layers, pages, hk, d, rows, page = 2, host.choice([23, 64, 100]), 2, 64, 9, host.choice([8, 16])
    c = kv.PagedKVCache(layers, pages, hk, d, rows, host.choice([120, 300]), page_size=page, dtype=torch.float16)
    m = Model(layers, pages, hk, d, rows, c.block_table.shape[1], page)
    written = [[] for _ in range(rows)]                    # the number each of a row's tokens holds
    stamp = 0
    refused = 0

    def put(rows_, counts, start):
        nonlocal stamp
        tok_rows, pos, val = [], [], []
        for r, n, s in zip(rows_, counts, start):
            for i in range(n):
                stamp += 1
                tok_rows.append(r), pos.append(s + i), val.append(stamp % 2000)
                written[r].append(stamp % 2000)
        if not val:
            return
        x = torch.tensor(val, dtype=torch.float16, device="cuda").view(-1, 1, 1).expand(-1, hk, d)
        for layer in range(layers):
            c.append(layer, x + 0.0, -x, _rows(*tok_rows), _rows(*pos))

    for _ in range(60):
        op = host.choice(["reserve", "reserve", "fork", "branch", "free", "compact"])
        used = [r for r in range(rows) if m.lens[r]]
        empty = [r for r in range(rows) if not m.lens[r]]
        if op == "reserve":
            some = host.sample(range(rows), host.randint(1, rows))
            counts = [host.choice([0, 1, 1, 3, page, 29]) for _ in some]
            want = m.reserve(some, counts)
            start = c.reserve(_rows(*some), torch.tensor(counts, dtype=torch.int32, device="cuda"))
            if want is None:
                refused += 1
                assert start.tolist() == [-1] * len(some)
                assert _status() == (7, 103)
                put([], [], [])
            else:
                assert start.tolist() == want[0]
                put(some, counts, want[0])
        elif op == "fork" and used and empty:
            dst = host.sample(empty, host.randint(1, len(empty)))
            src = [host.choice(used) for _ in dst]
            m.fork(src, dst)
            c.fork(_rows(*src), _rows(*dst))
            for s, t in zip(src, dst):
                written[t] = list(written[s])
        elif op == "branch" and len(used) > 1:
            src_rows = host.sample(used, max(1, len(used) // 2))
            dst = host.sample([r for r in range(rows) if r not in src_rows], host.randint(1, rows - len(src_rows)))
            src = [host.choice(src_rows) for _ in dst]
            m.free(dst)
            m.fork(src, dst)
            want = m.reserve(dst, [1] * len(dst))
            start = c.branch(_rows(*src), _rows(*dst), 1)
            for s, t in zip(src, dst):
                written[t] = list(written[s])
            if want is None:
                refused += 1
                assert _status() == (7, 103) and start.tolist() == [-1] * len(dst)
            else:
                assert start.tolist() == want[0]
                put(dst, [1] * len(dst), want[0])
        elif op == "free" and used:
            gone = host.sample(range(rows), host.randint(1, 3))
            m.free(gone)
            c.free(_rows(*gone))
            for r in gone:
                written[r] = []
        elif op == "compact":
            m.compact()
            c.compact()
        m.agrees(c)
        for r in range(rows):
            pos = torch.arange(m.lens[r], device="cuda")
            pg = c.block_table[r].long()[pos // page]
            for layer in range(layers):
                assert c.k[layer, pg, 1, pos % page, 5].tolist() == [float(w) for w in written[r]]
                assert c.v[layer, pg, 0, pos % page, 63].tolist() == [-float(w) for w in written[r]]
    assert _status() == (0, 0)


@pytest.mark.parametrize("pages,rows,width", [(40000, 300, 700), (5000, 2000, 9)])
def test_pages_large_pools(kv, pages, rows, width):
    host = random.Random(pages)
    c = kv.PagedKVCache(1, pages, 1, 8, rows, width * 8, page_size=8, dtype=torch.bfloat16)
    m = Model(1, pages, 1, 8, rows, width, 8)

    def both(op, *a):
        getattr(c, op)(*(torch.tensor(x, dtype=torch.int32, device="cuda") for x in a))
        want = getattr(m, op)(*a)
        m.agrees(c)
        return want

    half = list(range(0, rows, 2))
    counts = [host.randint(0, min(width * 8, pages * 8 // rows)) for _ in half]
    assert both("reserve", half, counts) is not None
    both("fork", [host.choice(half) for _ in range(1, rows, 2)], list(range(1, rows, 2)))
    some = host.sample(range(rows), rows // 2)
    both("reserve", some, [1 if m.lens[r] < width * 8 else 0 for r in some])
    both("free", host.sample(range(rows), rows // 2))
    _, _, moves = kv.compact_pages(c.block_table, c.ref_counts, c.k, c.v, out_table=c.block_table, out_refs=c.ref_counts)
    want = m.compact()
    m.agrees(c)
    assert moves.tolist() == want + [[-1, -1]] * (pages // 2 - len(want))
    assert _status() == (0, 0)


def test_pages_refusals_change_nothing(kv):
    c = kv.PagedKVCache(1, 6, 1, 64, 4, 64, page_size=16, dtype=torch.bfloat16)
    c.reserve(_rows(0, 1), 20)
    assert _status() == (0, 0)
    before = [t.clone() for t in (c.block_table, c.seq_lens, c.ref_counts, c.k.view(torch.int16))]

    def same():
        assert all(torch.equal(a, b) for a, b in zip(before, (c.block_table, c.seq_lens, c.ref_counts, c.k.view(torch.int16))))

    for call, code, site in ((lambda: c.reserve(_rows(0, 2), 64), 7, 103),        # too few free pages
                             (lambda: c.reserve(_rows(2), 65), 7, 103),           # wider than the table
                             (lambda: c.reserve(_rows(2), 2 ** 31 - 1), 7, 103),
                             (lambda: c.reserve(_rows(1, 1), 1), 1, 103),         # a row twice
                             (lambda: c.reserve(_rows(4), 1), 1, 103),
                             (lambda: c.reserve(_rows(-1), 1), 1, 103),
                             (lambda: c.reserve(_rows(2), _rows(-1)), 7, 103),
                             (lambda: c.fork(_rows(0), _rows(1)), 1, 102),        # not empty
                             (lambda: c.fork(_rows(0, 1), _rows(2, 2)), 1, 102),
                             (lambda: c.fork(_rows(7), _rows(2)), 1, 102),
                             (lambda: c.fork(_rows(2), _rows(2)), 1, 102),
                             (lambda: c.free(_rows(0, 0)), 1, 101),
                             (lambda: c.free(_rows(9)), 1, 101),
                             (lambda: c.branch(_rows(0, 1), _rows(2, 4), 1), 1, 101)):
        start = call()
        assert _status() == (code, site)
        assert start is None or bool((start == -1).all())
        same()
    with pytest.raises(RuntimeError, match="reserve"):
        c.reserve(_rows(2), 1000)
        c.check()
    c.check()
    # a refused position is skipped by the write
    x = torch.ones(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    c.append(0, x, x, _rows(2), _rows(-1))
    c.append(0, x, x, _rows(17), _rows(0))
    c.append(0, x, x, _rows(2), _rows(3))
    c.append(0, x, x, _rows(0), _rows(64))
    same()


def test_pages_host_refusals(kv):
    c = kv.PagedKVCache(1, 6, 1, 64, 4, 64, page_size=16)
    one = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    for bad in (lambda: c.reserve(_rows(0).long(), 1), lambda: c.reserve(_rows(0), -1), lambda: c.reserve(_rows(0).cpu(), 1),
                lambda: c.reserve(_rows(0, 1), _rows(1)), lambda: c.fork(_rows(0), _rows(1, 2)),
                lambda: c.reserve(_rows(0, 1, 2, 3, 0), 1),
                lambda: c.append(0, one.float(), one.float(), _rows(0), _rows(0)),
                lambda: c.append(0, one.half(), one.half(), _rows(0), _rows(0)),
                lambda: c.append(0, one, one, _rows(0, 1), _rows(0)),
                lambda: kv.append_kv(one[..., :32], one[..., :32], c.k[0], c.v[0], c.block_table, _rows(0), _rows(0)),
                lambda: kv.compact_pages(c.block_table, c.ref_counts[:3], c.k, c.v),
                lambda: kv.compact_pages(c.block_table, c.ref_counts, c.k, c.v, out_table=c.block_table[:1]),
                lambda: kv.PagedKVCache(1, 6, 1, 64, 4, 64, page_size=12),
                lambda: kv.PagedKVCache(1, 6, 1, 64, 4, 64, dtype=torch.float32)):
        with pytest.raises(ValueError):
            bad()


def test_compact_to_new_tensors_keeps_the_old_ones(kv):
    c = kv.PagedKVCache(3, 40, 2, 64, 5, 200, page_size=16, dtype=torch.float16)
    c.reserve(_rows(0, 1, 2, 3), _rows(100, 17, 60, 90))
    c.k.normal_()
    c.v.normal_()
    c.free(_rows(0, 2))
    table, refs, k, v = c.block_table.clone(), c.ref_counts.clone(), c.k.clone(), c.v.clone()
    t2, r2, moves = kv.compact_pages(c.block_table, c.ref_counts, c.k, c.v)
    assert torch.equal(c.block_table, table) and torch.equal(c.ref_counts, refs)
    for a, b in moves.tolist():
        if a >= 0:
            assert torch.equal(c.k[:, b], k[:, a]) and torch.equal(c.v[:, b], v[:, a])
    for r in (1, 3):
        for j in range(c.block_table.shape[1]):
            assert int(t2[r, j]) < 8
            if int(table[r, j]) >= 0:
                assert torch.equal(c.k[:, int(t2[r, j])], k[:, int(table[r, j])])
    assert r2.tolist() == [1] * 8 + [0] * 32
    assert kv.compact_pages(t2, r2, c.k, c.v)[2].tolist() == [[-1, -1]] * 20     # already compact


def test_append_types_strides_and_8_bits(kv):
    g = torch.Generator(device="cuda").manual_seed(3)
    proj = torch.randn(5, 12, 128, generator=g, device="cuda").bfloat16()
    k, v = proj[:, 6:8], proj[:, 8:10]                     # slices of a projection's output
    for ct in (torch.bfloat16, FP8):
        ks = torch.tensor([0.003, 0.5], device="cuda") if ct == FP8 else None
        vs = torch.tensor([1.0, 0.01], device="cuda") if ct == FP8 else None
        for token_major in (False, True):
            shape = (9, 16, 2, 128) if token_major else (9, 2, 16, 128)
            kc, vc = (torch.zeros(shape, dtype=torch.uint8, device="cuda").to(ct) for _ in range(2))
            if token_major:
                kc, vc = (x.view(torch.uint8).transpose(1, 2).view(ct) if ct == FP8 else x.transpose(1, 2) for x in (kc, vc))
            table = torch.tensor([[3, 8], [0, 5]], dtype=torch.int32, device="cuda")
            rows, pos = _rows(0, 1, 0, 1, 0), _rows(15, 31, 16, 0, 3)
            kv.append_kv(k, v, kc, vc, table, rows, pos, k_scale=ks, v_scale=vs)
            for t in range(5):
                p, s = int(table[int(rows[t]), int(pos[t]) // 16]), int(pos[t]) % 16
                for x, c, sc in ((k, kc, ks), (v, vc, vs)):
                    want = x[t] if ct != FP8 else (x[t].float() / sc[:, None]).clamp(-448, 448).to(FP8)
                    assert torch.equal(c.float()[p, :, s], want.float())
            written = {(int(table[int(r), int(q) // 16]), int(q) % 16) for r, q in zip(rows, pos)}
            for p in range(9):
                for s in range(16):
                    if (p, s) not in written:
                        assert not bool(kc.float()[p, :, s].any()) and not bool(vc.float()[p, :, s].any())
    x = torch.tensor([float("inf"), -float("inf"), float("nan"), 1e5] * 32, device="cuda").half().view(1, 1, 128)
    kc, vc = (torch.zeros(1, 1, 16, 128, dtype=torch.uint8, device="cuda").to(FP8) for _ in range(2))
    kv.append_kv(x, x, kc, vc, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), _rows(0), _rows(0))
    assert kc.float()[0, 0, 0, :2].tolist() == [448.0, -448.0] and bool(torch.isnan(kc.float()[0, 0, 0, 2]))
    assert float(kc.float()[0, 0, 0, 3]) == 448.0


def test_branch_equals_its_three_calls(kv):
    def made():
        c = kv.PagedKVCache(2, 60, 2, 64, 8, 100, page_size=16, dtype=torch.bfloat16)
        c.reserve(_rows(0, 1, 5), _rows(37, 48, 9))
        gen = torch.Generator(device="cuda").manual_seed(1)
        for t in (c.k, c.v):
            t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
        return c
    a, b = made(), made()
    src, dst = _rows(0, 0, 1, 1), _rows(5, 2, 7, 3)
    start = a.branch(src, dst, 2)
    b.free(dst)
    b.fork(src, dst)
    assert torch.equal(b.reserve(dst, 2), start) and start.tolist() == [37, 37, 48, 48]
    for x, y in zip((a.block_table, a.seq_lens, a.ref_counts, a.k, a.v), (b.block_table, b.seq_lens, b.ref_counts, b.k, b.v)):
        assert torch.equal(x, y)
    assert _status() == (0, 0)


# ----------------------------------------------------------------------------------------------------------
# tables whose rows share memory
# ----------------------------------------------------------------------------------------------------------

def _shared_views():
    """(view, the same table with rows of its own): one row for four queries, and rows that overlap by a page."""
    row = torch.tensor([[4, 1, 3]], dtype=torch.int32, device="cuda")
    run = torch.tensor([0, 5, 2, 6, 1, 3], dtype=torch.int32, device="cuda").as_strided((4, 3), (1, 1))
    return [(v, v.clone(memory_format=torch.contiguous_format)) for v in (row.expand(4, 3), run)]


@pytest.mark.parametrize("cache_type", [torch.bfloat16, FP8])
def test_attention_over_a_table_whose_rows_share_memory(kv, cache_type):
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = ((20 * torch.randn(7, 2, 16, 64, generator=g, device="cuda")).to(cache_type) for _ in range(2))
    n = torch.tensor([48, 1, 0, 33], dtype=torch.int32, device="cuda")
    q = _query(4, 6, 64, torch.bfloat16, 2, 0.1)
    for view, own in _shared_views():
        want = _attention_holds(kv, q, k, v, own, n)
        assert torch.equal(_attention_holds(kv, q, k, v, view, n), want)
        rows = _rows(3, 3, 0, 1)
        assert torch.equal(_attention_holds(kv, q, k, v, view, n, rows=rows), kv.paged_attention(q, k, v, own, n, rows=rows))


def test_append_and_compact_read_a_table_whose_rows_share_memory(kv):
    g = torch.Generator(device="cuda").manual_seed(2)
    x, y = (torch.randn(4, 2, 64, generator=g, device="cuda").bfloat16() for _ in range(2))
    rows, pos = _rows(0, 1, 2, 3), _rows(0, 17, 3, 47)
    for view, own in _shared_views():
        made = []
        for table in (own, view):
            k, v = (torch.zeros(1, 7, 2, 16, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
            kv.append_kv(x, y, k[0], v[0], table, rows, pos)
            for t in range(4):
                p, s = int(own[t, int(pos[t]) // 16]), int(pos[t]) % 16
                assert torch.equal(k[0, p, :, s], x[t]) and torch.equal(v[0, p, :, s], y[t])
            refs = torch.bincount(own.flatten(), minlength=7).int()
            made.append((k, v, *kv.compact_pages(table, refs, k, v)))
        for a, b in zip(*made):
            assert torch.equal(a, b)
    assert _status() == (0, 0)


# ----------------------------------------------------------------------------------------------------------
# weights far below the largest
# ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("b,n", [(1, 600), (30, 600), (2, 9000)])
@pytest.mark.parametrize("dtype,cache_type", [(torch.float16, torch.float16), (torch.float16, FP8), (torch.bfloat16, FP8),
                                              (torch.bfloat16, torch.bfloat16)])
def test_attention_long_tail_behind_one_strong_key(kv, dtype, cache_type, b, n):
    """One key with a value of zero takes nearly all the weight, the others e^-16 to e^-18 of it (2^-23 to 2^-26), and the
    output is made of them alone.  f16 parts of a weight are held to 2^-40 of the largest, 2^-14 of such a weight: within
    the module's bound, whose A is the tail's.  Clusters, whole segments and runs with their join."""
    k, v, table, lens = _cache([n] * b, 8, 16, 64, torch.float32, seed=n + b, poison=False)
    g = torch.Generator(device="cuda").manual_seed(4)
    k[..., 0] = -16 - 2 * torch.rand(k.shape[:-1], generator=g, device="cuda")
    v *= 20
    first = table[:, 0].long()
    k[first, :, 0, 0], v[first, :, 0] = 0.0, 0.0
    q = torch.zeros(b, 16, 64, device="cuda")
    q[..., 0] = 1.0
    kw = {}
    if cache_type == FP8:
        kw = {"k_scale": torch.ones(8, device="cuda"), "v_scale": torch.full((8,), 50.0, device="cuda")}
    _attention_holds(kv, q.to(dtype), k.to(cache_type), v.to(cache_type), table, lens, scale=1.0, **kw)


# ----------------------------------------------------------------------------------------------------------
# refused branches
# ----------------------------------------------------------------------------------------------------------

def _state(c):
    return [t.clone() for t in (c.block_table, c.seq_lens, c.ref_counts, c.k.view(torch.int16), c.v.view(torch.int16))]


def _three_rows(kv, pages=8):
    """Rows 0, 1 and 2 of 20, 33 and 5 tokens, 2 + 3 + 1 of the pages, and rows 3 and 4 without any."""
    c = kv.PagedKVCache(2, pages, 1, 64, 5, 64, page_size=16, dtype=torch.bfloat16)
    c.reserve(_rows(0, 1, 2), _rows(20, 33, 5))
    c.k.normal_(), c.v.normal_()
    assert _status() == (0, 0)
    return c


@pytest.mark.parametrize("src,dst", [((0,), (0,)), ((0, 1), (1, 2)), ((5,), (1,)), ((-1,), (1,)), ((0, 7), (1, 2)),
                                     ((2 ** 31 - 1,), (2,))])
def test_branch_with_a_wrong_source_changes_nothing(kv, src, dst):
    c = _three_rows(kv)
    before = _state(c)
    assert c.branch(_rows(*src), _rows(*dst), 1).tolist() == [-1] * len(src)
    assert _status() == (1, 102)
    assert all(torch.equal(a, b) for a, b in zip(before, _state(c)))


@pytest.mark.parametrize("free,src,dst,reserve,site", [((1, 1), (0,), (3,), (3,), 101), ((1, 9), (0,), (3,), (3,), 101),
                                                       ((1,), (0,), (2,), (2,), 102),      # neither empty nor freed
                                                       ((1,), (0, 2), (3, 3), (3,), 102), ((1,), (0,), (-2,), (3,), 102),
                                                       ((1,), (0,), (3,), (0, 0), 103), ((1,), (0,), (3,), (5,), 103),
                                                       ((1,), (0,), (3,), (-1,), 103)])
def test_a_wrong_list_stops_the_phases_before_it_too(kv, free, src, dst, reserve, site):
    from comfy_quant_bench_b200 import _lib
    c = _three_rows(kv)
    before = _state(c)
    start, copies = _lib.decode().pages_update(c.block_table, c.seq_lens, c.ref_counts, 16, _rows(*free), _rows(*src), _rows(*dst),
                                               _rows(*reserve), None, 1, c.k, c.v)
    assert _status() == (1, site) and bool((start == -1).all()) and bool((copies == -1).all())
    assert all(torch.equal(a, b) for a, b in zip(before, _state(c)))


def test_phases_on_lists_of_their_own(kv):
    """A destination may be empty or freed by the same call, a freed row may be a (then empty) source, and the rows that grow
    may be others."""
    from comfy_quant_bench_b200 import _lib
    c = _three_rows(kv)
    m = Model(2, 8, 1, 64, 5, 4, 16)
    m.reserve([0, 1, 2], [20, 33, 5])
    m.agrees(c)
    free, src, dst, reserve = [1, 2], [0, 2, 0], [3, 4, 1], [0, 4]
    m.free(free), m.fork(src, dst)
    want = m.reserve(reserve, [3, 3])
    start, copies = _lib.decode().pages_update(c.block_table, c.seq_lens, c.ref_counts, 16, _rows(*free), _rows(*src), _rows(*dst),
                                               _rows(*reserve), None, 3, c.k, c.v)
    assert _status() == (0, 0) and (start.tolist(), copies.tolist()) == want
    m.agrees(c)


def test_branch_without_room_is_completed_by_a_reservation(kv):
    """The reservation alone is refused: the rows are copies of their sources, and get their room once there is some."""
    c = _three_rows(kv, pages=6)
    c.branch(_rows(1, 1), _rows(3, 4), 1)                      # two copies of the last page of 33 tokens, no page free
    assert _status() == (7, 103)
    assert c.seq_lens.tolist() == [20, 33, 5, 33, 33]
    assert torch.equal(c.block_table[3], c.block_table[1]) and torch.equal(c.block_table[4], c.block_table[1])
    c.free(_rows(0))
    last = int(c.block_table[1, 2])
    assert c.reserve(_rows(3, 4), 1).tolist() == [33, 33] and _status() == (0, 0)
    for r in (3, 4):
        own = int(c.block_table[r, 2])
        assert own != last and torch.equal(c.k[:, own], c.k[:, last]) and torch.equal(c.v[:, own], c.v[:, last])


@pytest.mark.parametrize("pages", [392960, 393216])
def test_pages_pools_at_the_default_limit_of_shared_memory(kv, pages):
    """Bitmaps of 48 KB or just below, which fit the limit of a plain launch only without the kernels' static arrays."""
    c = kv.PagedKVCache(1, pages, 1, 8, 2, 8 * 40, page_size=8, dtype=torch.bfloat16)
    assert c.reserve(_rows(0, 1), _rows(300, 9)).tolist() == [0, 0]
    c.free(_rows(0))
    c.compact()
    assert _status() == (0, 0)
    assert c.block_table[1, :2].tolist() == [0, 1] and c.ref_counts[:3].tolist() == [1, 1, 0] and int(c.ref_counts.sum()) == 2


# ----------------------------------------------------------------------------------------------------------
# sizes near the ends of bf16's range
# ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("power", [-130, -122, -118, -110, -95, 90, 110])
@pytest.mark.parametrize("m", [1, 8, 9, 32, 33, 64])
def test_linear_tokens_of_any_size(ops, m, power):
    """Tokens of about 2^power, one of ordinary size among them, in each of the three kernels: bf16 tokens beyond eight are
    multiplied as f16 with a power of two per token, which has to bring every bf16 value into f16's range."""
    x, q, s, z, _ = _linear_problem(m, 1024, 200, 64, torch.bfloat16, seed=power)
    size = torch.full((m, 1), 2.0 ** power, device="cuda")
    size[m // 2] = 1.0 if m > 1 else size[0]
    x = (x.float() * size).bfloat16()
    _linear_holds(ops, x, q, s, z, None, 64)


@pytest.mark.parametrize("power", [-120, -110, -90, 0, 90, 110, 120])
@pytest.mark.parametrize("cache_type", [torch.bfloat16, FP8])
def test_attention_queries_of_any_size(kv, cache_type, power):
    """Queries of about 2^power and a scale that brings the scores back: a bf16 query of an 8-bit cache is multiplied as f16
    with a power of two per head."""
    k, v, table, n = _cache([300, 37], 2, 16, 64, cache_type, seed=3)
    kw = {} if cache_type != FP8 else {"k_scale": torch.tensor([0.05, 0.02], device="cuda"), "v_scale": torch.ones(2, device="cuda")}
    q = (_query(2, 8, 64, torch.bfloat16, 1).float() * 2.0 ** power).bfloat16()
    _attention_holds(kv, q, k, v, table, n, scale=2.0 ** (-power - 3), **kw)


@pytest.mark.parametrize("m", [12, 40])
def test_linear_calls_that_follow_each_other_use_their_own_tokens_sizes(ops, m):
    """The product's grid is already there when the kernel before it writes what each token was divided by; with a
    workspace that is taken again, the value before is another call's."""
    x, q, s, z, b = _linear_problem(m, 512, 384, 64, torch.bfloat16)
    sizes = [1.0, 2.0 ** 30, 2.0 ** -30, 2.0 ** 7]
    wants = [ops.w4a16_linear((x.float() * p).bfloat16(), q, s, z, group_size=64) for p in sizes]
    torch.cuda.synchronize()
    many = [(i, ops.w4a16_linear((x.float() * sizes[i]).bfloat16(), q, s, z, group_size=64)) for i in [0, 1, 2, 3] * 25]
    for i, y in many:
        assert torch.equal(y, wants[i])
    for p, y in zip(sizes, wants):
        assert torch.equal((y.double() / p).bfloat16(), wants[0])


# ----------------------------------------------------------------------------------------------------------
# infinities
# ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("m", [3, 8, 9, 32, 33, 70])
def test_linear_infinite_tokens_are_not_finite_and_stay_in_their_rows(ops, m, group, dtype):
    """In each of the three kernels: rows with an infinity or a NaN have no finite output, the others do not change."""
    x, q, s, z, b = _linear_problem(m, 384, 140, group, dtype)
    clean = ops.w4a16_linear(x, q, s, z, b, group_size=group)
    hit = torch.zeros(m, dtype=torch.bool, device="cuda")
    hit[[0, m - 1]] = True
    for one, two in ((float("inf"), -float("inf")), (float("nan"), float("inf"))):
        x[0, 383], x[m - 1, 7] = one, two
        y = ops.w4a16_linear(x, q, s, z, b, group_size=group)
        assert not bool(torch.isfinite(y[hit]).any()) and torch.equal(y[~hit], clean[~hit])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [40, 700, 20000])
def test_attention_infinite_keys_and_values_in_sight(kv, dtype, n):
    """An infinite value leaves its element of the output not finite and the others as they were; a key whose score is
    -infinity weighs nothing."""
    k, v, table, lens = _cache([n, n], 1, 16, 64, dtype, seed=8)
    q = _query(2, 2, 64, dtype, 1)
    clean = kv.paged_attention(q, k, v, table, lens)
    held = v.clone()
    at = int(table[0, 1]), 0, 3
    for value in (float("inf"), -float("inf")):
        v[at + (9,)] = value
        out = kv.paged_attention(q, k, v, table, lens)
        bad = ~torch.isfinite(out)
        assert bool(bad[0, :, 9].all()) and int(bad.sum()) == 2 and torch.equal(out[~bad], clean[~bad])
    v.copy_(held)
    q[..., 5] = q[..., 5].abs() + 0.5
    k[at + (5,)] = -float("inf")
    got = _attention_holds(kv, q, k, v, table, lens)
    assert bool(torch.isfinite(got).all())


# ----------------------------------------------------------------------------------------------------------
# calls that overlap
# ----------------------------------------------------------------------------------------------------------

def test_calls_on_two_streams_do_not_share_anything(ops, kv):
    """The three linears (workspaces for two of them), split and short attention and a cache's bookkeeping, on two streams at
    a time, against the same calls one after the other."""
    linears = [_linear_problem(m, 2048, 640, 64, dt, seed=i) for i, (m, dt) in
               enumerate([(4, torch.bfloat16), (20, torch.bfloat16), (64, torch.float16), (40, torch.bfloat16)])]
    k, v, table, n = _cache([5000, 300, 0, 9000], 2, 16, 128, torch.bfloat16, seed=1)
    short = _cache([40, 9], 2, 16, 128, torch.bfloat16, seed=2)
    q = _query(4, 8, 128, torch.bfloat16, 1)

    def work(c):
        out = [ops.w4a16_linear(*p, group_size=64) for p in linears]
        out.append(kv.paged_attention(q, k, v, table, n))
        out.append(kv.paged_attention(q[:2], *short))
        out.append(c.reserve(_rows(0, 1), _rows(20, 33)))
        out.append(c.branch(_rows(0, 1), _rows(2, 3), 1))
        c.free(_rows(0))
        c.compact()
        return out + [c.block_table.clone(), c.seq_lens.clone(), c.ref_counts.clone()]

    def cache():
        return kv.PagedKVCache(2, 30, 1, 64, 5, 64, page_size=16, dtype=torch.bfloat16)
    want = work(cache())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    caches = [cache() for _ in range(40)]
    torch.cuda.synchronize()
    got = []
    for i, c in enumerate(caches):
        with torch.cuda.stream(streams[i % 2]):
            got.append(work(c))
    torch.cuda.synchronize()
    for each in got:
        assert all(torch.equal(a, b) for a, b in zip(each, want))
    assert _status() == (0, 0)

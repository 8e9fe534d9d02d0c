"""The decode-side operators together, in the small language model of ``textgen``: a step's logits against the whole
sequence computed densely in fp32 from the dequantized weights, branches against rows of their own, and a captured step
against an eager one.

Bound: activations are rounded to bf16 (2^-8) about ten times per block on the way to the logits; with independent
roundings over 2 blocks the relative L2 error stays below sqrt(2 x 10 + 4) x 2^-8 x 0.3 (the rounding's RMS share) x 4
(the residual branches' gain) = 2.3e-2."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BOUND = 2.3e-2


@pytest.fixture(scope="module")
def tg():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from comfy_quant_bench_b200 import textgen
    return textgen


def _config(tg, **kw):
    base = dict(vocab=500, hidden=256, layers=2, heads=8, kv_heads=2, head_dim=64, ffn=512, group_size=64, max_tokens=160, rows=6,
                pages=80, page_size=16)
    return tg.TextConfig(**{**base, **kw})


def _dense(lin):
    u = lin.q.view(torch.uint8)
    codes = torch.stack([u & 15, u >> 4], -1).reshape(u.shape[0], -1).float() - 8
    return codes * lin.s.float().t().repeat_interleave(lin.group, 1) + lin.z.float().t().repeat_interleave(lin.group, 1)


def _reference(m, tokens):
    """Logits of the whole sequence, fp32."""
    c = m.cfg

    def norm(x):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6)

    n = len(tokens)
    x = m.embed[tokens].float()
    rope = torch.view_as_complex(m.rope[:n].contiguous()).unsqueeze(1)
    pos = torch.arange(n, device="cuda")
    at = pos.view(-1, 1) - pos.view(1, -1)
    for b in m.blocks:
        y = (norm(x) @ _dense(b.qkv).t()).view(n, c.heads + 2 * c.kv_heads, c.head_dim)
        q, k, v = y.split((c.heads, c.kv_heads, c.kv_heads), dim=1)
        q, k = (torch.view_as_real(torch.view_as_complex(norm(t).reshape(n, t.shape[1], -1, 2)) * rope).flatten(-2) for t in (q, k))
        k, v = (t.repeat_interleave(c.heads // c.kv_heads, 1) for t in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) * c.head_dim ** -0.5
        seen = at >= 0
        if b.window:
            seen = seen & ((at < b.window) | (pos.view(1, -1) < b.sinks))
        a = torch.einsum("hij,jhd->ihd", s.masked_fill(~seen, float("-inf")).softmax(-1), v)
        x = x + a.reshape(n, -1) @ _dense(b.out).t()
        gate, up = (norm(x) @ _dense(b.up).t()).chunk(2, -1)
        x = x + (torch.nn.functional.silu(gate) * up) @ _dense(b.down).t()
    return norm(x) @ _dense(m.head).t()


def _rel(a, b):
    return float((a.float() - b).norm() / b.norm())


@pytest.mark.parametrize("kw", [{}, {"window": 24, "sinks": 3}])
def test_prompt_and_steps_match_the_whole_sequence(tg, kw):
    m = tg.TextModel(_config(tg, **kw))
    g = torch.Generator(device="cuda").manual_seed(3)
    tokens = torch.randint(0, 500, (75,), generator=g, device="cuda")
    want = _reference(m, tokens)
    row = torch.tensor([2], dtype=torch.int32, device="cuda")
    assert _rel(m.prompt(tokens[:40], 2), want[:40]) <= BOUND
    for i in range(40, 75):
        assert _rel(m.step(tokens[i:i + 1], row)[0], want[i]) <= 1.5 * BOUND      # one row: fewer values to average over
    m.cache.check()


def test_8_bit_cache_stays_near(tg):
    """e4m3 keys and values (relative rounding 2^-4) move the logits by less than a tenth."""
    m = tg.TextModel(_config(tg, cache_dtype=torch.float8_e4m3fn))
    tokens = torch.arange(50, device="cuda")
    want = _reference(m, tokens)
    m.prompt(tokens[:30], 0)
    row = torch.zeros(1, dtype=torch.int32, device="cuda")
    for i in range(30, 50):
        assert _rel(m.step(tokens[i:i + 1], row)[0], want[i]) <= 0.1


def test_branches_equal_rows_of_their_own(tg):
    """Rows forked from a shared prompt (37 tokens, so the last page is shared and copied) give the logits of rows that
    read the prompt themselves."""
    m = tg.TextModel(_config(tg))
    g = torch.Generator(device="cuda").manual_seed(5)
    prompt = torch.randint(0, 500, (37,), generator=g, device="cuda")
    next_tokens = torch.randint(0, 500, (4, 12), generator=g, device="cuda")
    m.prompt(prompt, 0)
    rows = torch.arange(1, 5, dtype=torch.int32, device="cuda")
    positions = m.cache.branch(torch.zeros_like(rows), rows, 1)
    got = [m.step(next_tokens[:, 0], rows, positions)] + [m.step(next_tokens[:, i], rows) for i in range(1, 12)]
    m.cache.check()
    own = tg.TextModel(_config(tg))
    for r in range(1, 5):
        own.prompt(prompt, r)
    for i in range(12):
        assert torch.equal(own.step(next_tokens[:, i], rows), got[i])
    m.cache.compact()
    own.cache.compact()
    more = torch.randint(0, 500, (4,), generator=g, device="cuda")
    assert torch.equal(own.step(more, rows), m.step(more, rows))


def test_captured_step_equals_an_eager_one(tg):
    a, b = tg.TextModel(_config(tg)), tg.TextModel(_config(tg))
    rows = torch.tensor([3, 1], dtype=torch.int32, device="cuda")
    for m in (a, b):
        m.prompt(torch.arange(20, device="cuda"), 1)
        m.prompt(torch.arange(7, 22, device="cuda"), 3)
    tokens, graph, logits = a.capture(rows)
    for i in range(20):
        tokens.copy_(torch.tensor([i, 40 + i]))
        graph.replay()
        assert torch.equal(logits, b.step(torch.tensor([i, 40 + i], device="cuda"), rows))
    assert torch.equal(a.cache.block_table, b.cache.block_table) and torch.equal(a.cache.seq_lens, b.cache.seq_lens)
    a.cache.check()


def test_generate(tg):
    m = tg.TextModel(_config(tg))
    prompt = torch.arange(33, device="cuda")
    greedy = m.generate(prompt, 3, 10)
    assert greedy.shape == (3, 10) and bool((greedy == greedy[:1]).all())
    assert torch.equal(m.generate(prompt, 3, 10), greedy)
    u = torch.rand(10, 3, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    sampled = m.generate(prompt, 3, 10, u)
    assert torch.equal(m.generate(prompt, 3, 10, u), sampled) and not bool((sampled == sampled[:1]).all())
    with pytest.raises(ValueError, match="cache rows"):
        m.generate(prompt, 6, 2)
    with pytest.raises(RuntimeError, match="reserve"):       # the pool has no room for so long a continuation
        m.generate(prompt, 5, 130)


def test_awq_layer_of_a_checkpoint_runs(tg):
    """The layout registered for awq_w4a16: state dict -> Linear -> the kernel."""
    import json

    from comfy_quant_bench_b200 import comfy_ops, layout, ops
    layout.register_w4a16()
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.randn(96, 256, generator=g, device="cuda")
    q, s, z = ops.quantize_affine_w4_weight(w, 64)
    bias = torch.randn(96, generator=g, device="cuda").bfloat16()
    conf = torch.tensor(list(json.dumps({"format": "awq_w4a16", "group_size": 64}).encode()), dtype=torch.uint8)
    lin = comfy_ops.Linear(256, 96)
    lin.load_state_dict({"weight": q, "weight_scale": s, "weight_zeros": z, "bias": bias, "comfy_quant": conf})
    lin.weight, lin.bias = lin.weight.to("cuda"), torch.nn.Parameter(bias, requires_grad=False)
    x = torch.randn(3, 256, generator=g, device="cuda").bfloat16()
    assert torch.equal(lin(x), ops.w4a16_linear(x, q, s, z, bias, group_size=64))
    dense = lin.weight.dequantize().float()
    want = x.float() @ dense.t() + bias.float()
    assert _rel(lin(x), want) <= 2.0 ** -7                   # the dequantized weight is rounded to bf16
    out = comfy_ops.linear_input_act(lin, torch.randn(3, 512, generator=g, device="cuda").bfloat16(), "swiglu")
    assert out.shape == (3, 96)
    with pytest.raises(ValueError, match="input_act"):
        lin.weight.linear(x, bias, input_act="swiglu")


def test_rows_fill_their_last_page(tg):
    """Steps at and past max_tokens, up to the end of the row's last page; the next one is refused."""
    m = tg.TextModel(_config(tg, max_tokens=40, pages=8))
    tokens = torch.arange(48, device="cuda")
    want = _reference(m, tokens)
    m.prompt(tokens[:38], 1)
    row = torch.ones(1, dtype=torch.int32, device="cuda")
    for i in range(38, 48):
        assert _rel(m.step(tokens[i:i + 1], row)[0], want[i]) <= 1.5 * BOUND
    m.cache.check()
    m.step(tokens[:1], row)
    with pytest.raises(RuntimeError, match="reserve"):
        m.cache.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16, torch.bfloat16])
def test_awq_layer_returns_the_type_it_is_given(tg, dtype):
    """With and without a weight patch.  Other types are rounded to bf16 on the way in; the patched path takes the weight
    rounded to bf16."""
    from comfy_quant_bench_b200 import comfy_ops, layout, ops
    layout.register_w4a16()
    g = torch.Generator(device="cuda").manual_seed(6)
    q, s, z = ops.quantize_affine_w4_weight(torch.randn(96, 256, generator=g, device="cuda"), 64)
    bias = torch.randn(96, generator=g, device="cuda").bfloat16()
    params = layout.get_layout_class("B200AwqW4A16Layout").Params(scale=s, zeros=z, orig_dtype=torch.bfloat16, orig_shape=(96, 256),
                                                                  group_size=64)
    lin = comfy_ops.Linear.from_quantized(layout.QuantizedWeight(q, "B200AwqW4A16Layout", params), bias)
    for tokens in (1, 3, 40):
        x = torch.randn(tokens, 256, generator=g, device="cuda").to(dtype)
        y = lin(x)
        held = x if dtype in (torch.bfloat16, torch.float16) else x.bfloat16()
        assert y.dtype == dtype and torch.equal(y, ops.w4a16_linear(held, q, s, z, bias, group_size=64).to(dtype))
        lin.weight_function = [lambda w: w]
        patched = lin(x)
        lin.weight_function = []
        assert patched.dtype == dtype and _rel(y, patched.float()) <= 2.0 ** -7

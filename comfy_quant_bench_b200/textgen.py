"""A small decoder language model on the decode-side operators: 4-bit weights, 16-bit activations, a paged cache.

The models beside a DiT that write or encode its prompts run like this: a prompt goes through once, then one token per
sequence and step.  With x the residual stream [tokens, hidden] (bf16), a block is

    y = RMSNorm(x) * w1;  q, k, v = Wqkv y;  q, k = rope(RMSNorm per head)
    x = x + Wo attention(q, cache of k and v)
    y = RMSNorm(x) * w2;  x = x + Wd (silu(Wg y) * Wu y)

Every linear is ``ops.w4a16_linear``, every addition to the stream and the norm after it ``ops.add_rmsnorm``; the heads'
norms, the rotary embedding and the cache's append are ``kvcache.append_rotated``.  Keys and values live in a
``kvcache.PagedKVCache`` and a step's attention reads them there.  Every second block may see only a window and the first
few tokens (``window``, ``sinks``).  Weights are random: the module shows how the operators go together, and
``python -m comfy_quant_bench_b200.textgen`` times a step.

``generate`` writes several continuations of one prompt: the prompt's row is forked, its pages are shared, and a row's
last page is copied when the row first writes to it; attention reads the prompt once for all of them
(``kvcache.prefix_attention``), and ``ops.sample_tokens`` chooses the tokens.  A step works on device state alone, so
``capture`` turns it into one CUDA graph.
"""
from __future__ import annotations

import argparse
import time
from dataclasses import dataclass

import torch
import torch.nn.functional as F

from . import kvcache, ops


@dataclass(frozen=True)
class TextConfig:
    vocab: int = 32000
    hidden: int = 2048
    layers: int = 8
    heads: int = 16
    kv_heads: int = 4
    head_dim: int = 128
    ffn: int = 5632
    group_size: int = 128
    window: int = 0              # > 0: every second block sees this many tokens and the first `sinks`
    sinks: int = 0
    rope_base: float = 10000.0
    rope_scaling: str | None = None      # kvcache.rope_table's, with its factor, original context and so on
    rope_factor: float = 1.0
    rope_original: int = 0
    rope_fast: float = 32.0
    rope_slow: float = 1.0
    rope_blend: str = "turns"
    rope_size: float | None = None
    max_tokens: int = 2048
    rows: int = 16
    pages: int = 1024
    page_size: int = 16
    cache_dtype: torch.dtype = torch.bfloat16


class _Linear:
    """A random W4A16 linear."""

    def __init__(self, n: int, k: int, cfg: TextConfig, gen: torch.Generator):
        w = torch.randn(n, k, generator=gen, device=gen.device) * k ** -0.5
        self.group = cfg.group_size
        self.q, self.s, self.z = ops.quantize_affine_w4_weight(w, self.group)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        return ops.w4a16_linear(x, self.q, self.s, self.z, group_size=self.group)


class _Block:
    def __init__(self, cfg: TextConfig, index: int, gen: torch.Generator):
        d, kv = cfg.heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim
        self.qkv = _Linear(d + 2 * kv, cfg.hidden, cfg, gen)
        self.out = _Linear(cfg.hidden, d, cfg, gen)
        self.up = _Linear(2 * cfg.ffn, cfg.hidden, cfg, gen)
        self.down = _Linear(cfg.hidden, cfg.ffn, cfg, gen)
        ones = lambda n: torch.ones(n, dtype=torch.bfloat16, device=gen.device)  # noqa: E731
        self.norm1, self.norm2 = ones(cfg.hidden), ones(cfg.hidden)
        self.norm_q, self.norm_k = ones(cfg.head_dim), ones(cfg.head_dim)
        windowed = cfg.window > 0 and index % 2 == 1
        self.window, self.sinks = (cfg.window, cfg.sinks) if windowed else (0, 0)


class TextModel:
    def __init__(self, cfg: TextConfig = TextConfig(), seed: int = 0, device="cuda"):
        if cfg.heads % cfg.kv_heads:
            raise ValueError(f"heads ({cfg.heads}) must be a multiple of kv_heads ({cfg.kv_heads})")
        gen = torch.Generator(device=device).manual_seed(seed)
        self.cfg, self.device = cfg, torch.device(device)
        self.embed = torch.randn(cfg.vocab, cfg.hidden, generator=gen, device=device).to(torch.bfloat16)
        self.blocks = [_Block(cfg, i, gen) for i in range(cfg.layers)]
        self.norm = torch.ones(cfg.hidden, dtype=torch.bfloat16, device=device)
        self.head = _Linear(cfg.vocab, cfg.hidden, cfg, gen)
        scale = torch.full((cfg.kv_heads,), 0.02, device=device) if cfg.cache_dtype == torch.float8_e4m3fn else None
        self.cache = kvcache.PagedKVCache(cfg.layers, cfg.pages, cfg.kv_heads, cfg.head_dim, cfg.rows, cfg.max_tokens,
                                          cfg.page_size, cfg.cache_dtype, device, scale, scale)
        room = self.cache.block_table.shape[1] * cfg.page_size               # max_tokens up to whole pages: any position
        self.rope = kvcache.rope_table(room, cfg.head_dim, base=cfg.rope_base, scaling=cfg.rope_scaling, factor=cfg.rope_factor,
                                       original=cfg.rope_original, fast=cfg.rope_fast, slow=cfg.rope_slow,
                                       blend=cfg.rope_blend, size=cfg.rope_size, device=device)      # [tokens, D/2, 2]

    def _forward(self, tokens, rows, positions, attention) -> torch.Tensor:
        """Logits [tokens, vocab] (bf16); ``attention(layer, block, q)`` after the tokens' keys and values are cached."""
        c = self.cfg
        out, x = self.embed[tokens], None                        # what the last linear gave, and the stream before it
        for layer, b in enumerate(self.blocks):
            y, x = ops.add_rmsnorm(out, b.norm1, x)
            y = b.qkv(y).view(len(tokens), c.heads + 2 * c.kv_heads, c.head_dim)
            q, k, v = y.split((c.heads, c.kv_heads, c.kv_heads), dim=1)
            q, k = self.cache.append_rotated(layer, q, k, v, rows, positions, self.rope, interleaved=True, q_norm=b.norm_q,
                                             k_norm=b.norm_k, return_k=True)
            y, x = ops.add_rmsnorm(b.out(attention(layer, b, q, k, v).reshape(len(tokens), c.heads * c.head_dim)), b.norm2, x)
            gate, up = b.up(y).chunk(2, dim=-1)
            out = b.down(F.silu(gate) * up)
        return self.head(ops.add_rmsnorm(out, self.norm, x)[0])

    def prompt(self, tokens: torch.Tensor, row: int) -> torch.Tensor:
        """A prompt [tokens] into the empty cache row; logits [tokens, vocab]."""
        n = len(tokens)
        if n > self.cfg.max_tokens:
            raise ValueError(f"a prompt of {n} tokens for rows of max_tokens = {self.cfg.max_tokens}")
        where = torch.tensor([row], dtype=torch.int32, device=self.device)
        self.cache.reserve(where, n)
        positions = torch.arange(n, dtype=torch.int32, device=self.device)
        at = positions.view(-1, 1) - positions.view(1, -1)

        def attention(layer, b, q, k, v):
            seen = at >= 0
            if b.window:
                seen &= (at < b.window) | (positions.view(1, -1) < b.sinks)
            q, k, v = (t.transpose(0, 1).unsqueeze(0) for t in (q, k, v))
            return F.scaled_dot_product_attention(q, k, v, attn_mask=seen, enable_gqa=True)[0].transpose(0, 1)

        return self._forward(tokens, where.expand(n).contiguous(), positions, attention)

    def step(self, tokens: torch.Tensor, rows: torch.Tensor, positions: torch.Tensor | None = None,
             prefix: int | torch.Tensor | None = None) -> torch.Tensor:
        """One token for each of the cache rows (int32): logits [rows, vocab].  ``positions``: where the tokens go, if
        they are reserved already.  ``prefix``: the rows' first so many tokens are the same (an int, or one int32 on the
        device)."""
        if positions is None:
            positions = self.cache.reserve(rows, 1)

        def attention(layer, b, q, k, v):
            if prefix is None or b.window:
                return self.cache.attend(layer, q, rows, window=b.window, sinks=b.sinks)
            return self.cache.attend_prefix(layer, q, prefix, rows, weight_parts=2)      # as exact as ``attend``

        return self._forward(tokens, rows, positions, attention)

    def capture(self, rows: torch.Tensor, prefix: int | torch.Tensor | None = None):
        """A step of these rows as one CUDA graph: (tokens to fill in, graph, logits)."""
        tokens = torch.zeros(len(rows), dtype=torch.long, device=self.device)
        start = self.cache.seq_lens[rows.long()].clone()         # warm-up: written at the rows' ends, nothing reserved
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self.step(tokens, rows, torch.full_like(start, -1), prefix)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = self.step(tokens, rows, None, prefix)
        return tokens, graph, logits

    def _choose(self, logits: torch.Tensor, uniform: torch.Tensor, sampling: dict) -> torch.Tensor:
        """The next tokens of logits [rows, vocab] by a number for each row, or one for all."""
        uniform = uniform.reshape(-1).float().expand(len(logits))
        if self.cfg.vocab <= 327680 or sampling:
            return ops.sample_tokens(logits, uniform, **sampling)
        total = logits.float().softmax(-1).cumsum(-1)            # more tokens than ``sample_tokens`` takes
        return torch.searchsorted(total, uniform.view(-1, 1) * total[:, -1:]).squeeze(1).clamp(max=self.cfg.vocab - 1)

    def generate(self, prompt: torch.Tensor, samples: int, steps: int, uniform: torch.Tensor | None = None,
                 **sampling) -> torch.Tensor:
        """``samples`` continuations of ``steps`` tokens of one prompt: [samples, steps].  ``uniform`` [steps, samples] (or one
        number a step) in [0, 1) chooses the tokens (``ops.sample_tokens``, with its temperature, top_k, top_p and min_p); without it each is
        the likeliest."""
        if uniform is None and sampling:
            raise ValueError(f"{', '.join(sampling)} without uniform numbers: the likeliest tokens are not sampled")
        if samples + 1 > self.cfg.rows:
            raise ValueError(f"{samples} samples and the prompt need {samples + 1} cache rows, there are {self.cfg.rows}")
        rows = torch.arange(1, samples + 1, dtype=torch.int32, device=self.device)
        every = torch.arange(samples + 1, dtype=torch.int32, device=self.device)
        self.cache.free(every)
        logits = self.prompt(prompt, 0)[-1:].expand(samples, -1)
        positions = self.cache.branch(torch.zeros_like(rows), rows, 1)
        out = []
        for i in range(steps):
            out.append(logits.argmax(-1) if uniform is None else self._choose(logits, uniform[i], sampling))
            if i + 1 < steps:
                logits = self.step(out[-1], rows, positions, len(prompt))
                positions = None
        self.cache.check()
        return torch.stack(out, dim=1)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--samples", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=500, help="tokens of the prompt")
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--layers", type=int, default=TextConfig.layers)
    a = ap.parse_args()
    cfg = TextConfig(layers=a.layers, window=256, sinks=4)
    model = TextModel(cfg)
    g = torch.Generator(device="cuda").manual_seed(1)
    prompt = torch.randint(0, cfg.vocab, (a.prompt,), generator=g, device="cuda")
    tokens = model.generate(prompt, a.samples, 4)
    rows = torch.arange(1, a.samples + 1, dtype=torch.int32, device="cuda")
    fill, graph, _ = model.capture(rows, a.prompt)
    fill.copy_(tokens[:, -1])
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(a.steps):
        graph.replay()
    torch.cuda.synchronize()
    ms = (time.perf_counter() - t) * 1e3 / a.steps
    model.cache.check()
    print(f"{a.samples} rows after a prompt of {a.prompt}: {ms:.3f} ms per step of {cfg.layers} blocks, "
          f"{a.samples / ms * 1e3:.0f} tokens/s")


if __name__ == "__main__":
    main()

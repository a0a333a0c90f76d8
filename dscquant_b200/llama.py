"""Llama-2-architecture decoder stack with every linear on the W4A4 path: the prefill workload of the
benchmark (random-init weights, batch 1 x seqlen token ids).

The reference applies its QuantLinear to the linears of a Hugging Face LlamaForCausalLM
(core/model_ops.py:3-6 walks model.model.layers; core/linear.py:48-52 is each wrapped linear). This
module builds the same architecture directly around this package's QuantLinear so that a prefill can
run without the transformers model code or a checkpoint:

    h = embed[ids]
    per layer:  x = RMSNorm(h)
                q, k, v = Wq x, Wk x, Wv x       one rotate+quantize of x shared by the three GEMMs
                q, k = RoPE(q), RoPE(k)
                a = causal attention(q, k, v)      bf16 (torch scaled_dot_product_attention)
                h = h + Wo a                       residual added in the GEMM epilogue
                x = RMSNorm(h)
                g, u = Wg x, Wu x                  one rotate+quantize shared by the two GEMMs
                h = h + Wd (silu(g) * u)           residual added in the GEMM epilogue
    logits = Wlm RMSNorm(h)

All seven projections of every layer and the LM head are W4A4 (symmetric per-token activations,
online Hadamard rotation, symmetric per-channel int4 weights). RMSNorm, RoPE and the SiLU gate are
single-pass bf16 kernels of this package (ops.rmsnorm / rope_ / silu_mul, the same rounding steps as
the torch expressions rms_norm / apply_rope below, which the tests compare them with); causal
attention is torch's scaled_dot_product_attention in bf16.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn.functional as F

from . import ops
from .kvcache import PagedKV4
from .linear import QuantConfig, QuantLinear


@dataclass
class LlamaConfig:
    vocab: int = 32000
    hidden: int = 4096
    heads: int = 32
    kv_heads: int = 32
    intermediate: int = 11008
    layers: int = 32
    rope_theta: float = 10000.0
    eps: float = 1e-5

    @property
    def head_dim(self) -> int:
        return self.hidden // self.heads


def random_quant_linear(N: int, K: int, gen: torch.Generator, device, std: float = 0.02) -> QuantLinear:
    """A prepared W4A4 QuantLinear with N(0, std) bf16 weights (only the packed weight is kept)."""
    base = torch.nn.Linear(K, N, bias=False, dtype=torch.bfloat16, device=device)
    with torch.no_grad():
        base.weight.copy_((torch.randn(N, K, generator=gen, device=device) * std).to(torch.bfloat16))
    ql = QuantLinear(base, QuantConfig())
    ql.enabled = True
    ql.prepare()
    base.weight.data = torch.empty(0, dtype=torch.bfloat16, device=device)
    return ql


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)).to(x.dtype) * weight


def rope_tables(seq: int, head_dim: int, theta: float, device) -> tuple[torch.Tensor, torch.Tensor]:
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, device=device, dtype=torch.float32) / head_dim))
    f = torch.outer(torch.arange(seq, device=device, dtype=torch.float32), inv)
    emb = torch.cat((f, f), dim=-1)
    return emb.cos().to(torch.bfloat16), emb.sin().to(torch.bfloat16)


def apply_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x [S, H, D]; rotate-half form of rotary embeddings."""
    d = x.shape[-1] // 2
    rot = torch.cat((-x[..., d:], x[..., :d]), dim=-1)
    return x * cos[:, None, :] + rot * sin[:, None, :]


class DecoderLayer:
    def __init__(self, cfg: LlamaConfig, gen: torch.Generator, device):
        H, I, kv = cfg.hidden, cfg.intermediate, cfg.kv_heads * cfg.head_dim
        self.cfg = cfg
        self.q = random_quant_linear(H, H, gen, device)
        self.k = random_quant_linear(kv, H, gen, device)
        self.v = random_quant_linear(kv, H, gen, device)
        self.o = random_quant_linear(H, H, gen, device)
        self.gate = random_quant_linear(I, H, gen, device)
        self.up = random_quant_linear(I, H, gen, device)
        self.down = random_quant_linear(H, I, gen, device)
        self.norm1 = (1.0 + 0.1 * torch.randn(H, generator=gen, device=device)).to(torch.bfloat16)
        self.norm2 = (1.0 + 0.1 * torch.randn(H, generator=gen, device=device)).to(torch.bfloat16)

    def project(self, h: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """q [S, heads, D], k and v [S, kv_heads, D] of the normalised input, before the rotation."""
        cfg, S = self.cfg, h.shape[0]
        qx = self.q.quantize_input(ops.rmsnorm(h, self.norm1, cfg.eps))
        return (self.q.forward_quantized(qx, S).view(S, cfg.heads, cfg.head_dim),
                self.k.forward_quantized(qx, S).view(S, cfg.kv_heads, cfg.head_dim),
                self.v.forward_quantized(qx, S).view(S, cfg.kv_heads, cfg.head_dim))

    def finish(self, h: torch.Tensor, a: torch.Tensor) -> torch.Tensor:
        """The rest of the layer behind its attention output a [S, hidden]."""
        cfg, S = self.cfg, h.shape[0]
        h = self.o.forward_quantized(self.o.quantize_input(a), S, residual=h)
        x = ops.rmsnorm(h, self.norm2, cfg.eps)
        gx = self.gate.quantize_input(x)
        g = self.gate.forward_quantized(gx, S)
        u = self.up.forward_quantized(gx, S)
        m = ops.silu_mul(g, u)
        return self.down.forward_quantized(self.down.quantize_input(m), S, residual=h)

    def __call__(self, h: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
        cfg, S = self.cfg, h.shape[0]
        q, k, v = self.project(h)
        ops.rope_(q, k, cos, sin)
        a = F.scaled_dot_product_attention(q.transpose(0, 1)[None], k.transpose(0, 1)[None], v.transpose(0, 1)[None],
                                           is_causal=True, enable_gqa=cfg.kv_heads != cfg.heads)
        return self.finish(h, a[0].transpose(0, 1).reshape(S, cfg.hidden))

    def step(self, h: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, cache: PagedKV4, where: tuple,
             max_q: int | None = None) -> torch.Tensor:
        """The layer on new tokens of a batch of sequences, keys and values kept in `cache`; `where` is
        (page_table, q_start, lengths) as ops.kv4_append takes them, cos / sin are tables by position."""
        q, k, v = self.project(h)
        q = ops.kv4_append(cache, q, k, v, cos, sin, *where)
        a = ops.kv4_attention(cache, q, *where, max_q=max_q)
        return self.finish(h, a.view(h.shape[0], self.cfg.hidden))


class LlamaW4A4:
    """Random-init Llama-2 stack (LlamaConfig) on one GPU; __call__(ids [S]) -> logits [S, vocab] bf16."""

    def __init__(self, cfg: LlamaConfig, device, seed: int = 0):
        self.cfg = cfg
        self.device = torch.device(device)
        gen = torch.Generator(device=self.device)
        gen.manual_seed(seed)
        self.embed = (torch.randn(cfg.vocab, cfg.hidden, generator=gen, device=self.device) * 0.02).to(torch.bfloat16)
        self.layers = [DecoderLayer(cfg, gen, self.device) for _ in range(cfg.layers)]
        self.norm = (1.0 + 0.1 * torch.randn(cfg.hidden, generator=gen, device=self.device)).to(torch.bfloat16)
        self.lm_head = random_quant_linear(cfg.vocab, cfg.hidden, gen, self.device)
        self._rope = {}

    def rope(self, S: int):
        if S not in self._rope:
            self._rope[S] = rope_tables(S, self.cfg.head_dim, self.cfg.rope_theta, self.device)
        return self._rope[S]

    @torch.no_grad()
    def __call__(self, ids: torch.Tensor) -> torch.Tensor:
        S = ids.shape[0]
        cos, sin = self.rope(S)
        h = self.embed[ids]
        for layer in self.layers:
            h = layer(h, cos, sin)
        x = ops.rmsnorm(h, self.norm, self.cfg.eps)
        return self.lm_head.forward_quantized(self.lm_head.quantize_input(x), S)

    def graph(self, S: int) -> "PrefillGraph":
        """The prefill of S tokens captured once as a CUDA graph (see PrefillGraph)."""
        return PrefillGraph(self, S)

    # ------------------------------------------------------------------ generation and scoring
    def caches(self, pages: int, page_size: int = 64) -> list[PagedKV4]:
        """An empty 4-bit cache of `pages` pages for every layer."""
        c = self.cfg
        return [PagedKV4.allocate(pages, c.kv_heads, c.head_dim, page_size, torch.bfloat16, self.device)
                for _ in self.layers]

    @torch.no_grad()
    def step(self, ids: torch.Tensor, caches: list[PagedKV4], page_table: torch.Tensor, q_start: torch.Tensor,
             lengths: torch.Tensor, max_q: int | None = None) -> torch.Tensor:
        """Logits [T, vocab] of new tokens ids [T] of a batch of sequences (described as for ops.kv4_append;
        `lengths` counts them in), which join the caches."""
        positions = max(page_table.shape[1] * caches[0].page_size, 1)
        # tables are kept (captured steps read them) and of a power of two, so that page tables of all widths share a few
        cos, sin = self.rope(1 << (positions - 1).bit_length())
        h = self.embed[ids]
        for layer, cache in zip(self.layers, caches):
            h = layer.step(h, cos, sin, cache, (page_table, q_start, lengths), max_q)
        x = ops.rmsnorm(h, self.norm, self.cfg.eps)
        return self.lm_head.forward_quantized(self.lm_head.quantize_input(x), ids.shape[0])

    def generate(self, prompts: list[torch.Tensor], new_tokens: int, page_size: int = 64):
        """Greedy continuation of each prompt (1-D ids, at least one): (ids [prompts, new_tokens], their log
        probabilities). The prompts run as one ragged step, the tokens behind the first through DecodeGraph."""
        counts = [len(p) for p in prompts]
        if new_tokens < 1 or not counts or min(counts) < 1:
            raise ValueError("generate needs at least one prompt, one id in each and one new token")
        used = [-(-(n + new_tokens) // page_size) for n in counts]
        caches = self.caches(sum(used), page_size)
        table = torch.full((len(prompts), max(used)), -1, dtype=torch.int32)
        for b, n in enumerate(used):
            table[b, :n] = torch.arange(sum(used[:b]), sum(used[:b]) + n, dtype=torch.int32)
        table = table.to(self.device)
        lengths = torch.tensor(counts, dtype=torch.int32, device=self.device)
        ends = lengths.cumsum(0)
        q_start = F.pad(ends, (1, 0)).to(torch.int32)
        logits = self.step(torch.cat([p.to(self.device) for p in prompts]), caches, table, q_start, lengths, max(counts))
        first = ops.token_logprobs(logits[ends - 1], torch.full_like(ends, -1), top_k=1)
        ids, logprobs = [first.top_ids], [first.top_logprobs]
        if new_tokens > 1:
            graph = DecodeGraph(self, caches, table, lengths, first.top_ids[:, 0])
            for _ in range(new_tokens - 1):
                i, lp = graph()
                ids.append(i.clone())
                logprobs.append(lp.clone())
        return torch.cat(ids[:new_tokens], 1), torch.cat(logprobs[:new_tokens], 1)

    def score(self, ids: torch.Tensor, top_k: int = 0) -> "ops.TokenLogprobs":
        """Log probability of every token of ids [S >= 2] but the first given those before it, with the entropy and the
        top_k alternatives at each place; exp(-mean) of the log probabilities is the text's perplexity."""
        return ops.token_logprobs(self(ids)[:-1], ids[1:].contiguous(), top_k)

    def linear_ops(self, S: int) -> float:
        """Integer ops of all W4A4 GEMMs of one prefill of S tokens (2 * S * N * K each)."""
        c = self.cfg
        kv = c.kv_heads * c.head_dim
        per_layer = 2 * S * (c.hidden * c.hidden * 2 + 2 * kv * c.hidden + 3 * c.intermediate * c.hidden)
        return float(per_layer * c.layers + 2 * S * c.vocab * c.hidden)


class PrefillGraph:
    """One CUDA graph holding a whole prefill of S tokens: every kernel of __call__ (rotate+quantize,
    W4A4 GEMMs, RMSNorm, RoPE, attention, SiLU gate, LM head) recorded once and replayed without the
    host issuing each op. The ids are copied into a static buffer, and the logits come back in a
    static buffer that the next replay overwrites. One eager pass runs first on a side stream: the
    first call per device and K builds the rotate+quantize operand, which cannot be captured."""

    def __init__(self, model: LlamaW4A4, S: int):
        dev = model.device
        self.ids = torch.zeros(S, dtype=torch.long, device=dev)
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            model(self.ids)
        torch.cuda.current_stream(dev).wait_stream(side)
        torch.cuda.synchronize(dev)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.logits = model(self.ids)

    def __call__(self, ids: torch.Tensor) -> torch.Tensor:
        self.ids.copy_(ids)
        self.graph.replay()
        return self.logits


class DecodeGraph:
    """One CUDA graph of a greedy decode step for a batch of sequences: each call appends the current token of every
    sequence, runs the model over the caches and picks the next tokens, whose ids [B, 1] and log probabilities
    come back in static buffers that the next call overwrites. Lengths and tokens advance on the device, so
    calls need no host work; page_table must already map the positions they reach, and may be changed in place."""

    def __init__(self, model: LlamaW4A4, caches: list[PagedKV4], page_table: torch.Tensor, lengths: torch.Tensor,
                 ids: torch.Tensor):
        dev, B = model.device, lengths.shape[0]
        self.lengths, self.ids, self.page_table = lengths.clone(), ids.clone(), page_table
        q_start = torch.arange(B + 1, dtype=torch.int32, device=dev)
        nobody = torch.full((B,), -1, dtype=torch.long, device=dev)
        self._held = model, caches, q_start, nobody  # the captured kernels go on using them

        def step():
            self.lengths.add_(1)
            r = ops.token_logprobs(model.step(self.ids, caches, page_table, q_start, self.lengths, max_q=1), nobody, top_k=1)
            self.ids.copy_(r.top_ids[:, 0])
            return r.top_ids, r.top_logprobs

        side = torch.cuda.Stream(dev)  # once eagerly: it builds what cannot be built in a capture, and is undone
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side), torch.no_grad():
            step()
            self.lengths.copy_(lengths)
            self.ids.copy_(ids)
        torch.cuda.current_stream(dev).wait_stream(side)
        torch.cuda.synchronize(dev)
        self.graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(self.graph):
            self.out = step()

    def __call__(self) -> tuple[torch.Tensor, torch.Tensor]:
        self.graph.replay()
        return self.out

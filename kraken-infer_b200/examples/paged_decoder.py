"""A small decoder served from the paged 8-bit KV cache: ragged prompts in one
call, then one token per sequence and step, each drawn with its own settings.

    python kraken-infer_b200/examples/paged_decoder.py

Random K-quant weights; the point is how the calls go together.  A step is one
graph scope of the context: embedding rows, then per layer norm, projections,
kvq8_append (rotates q and k, quantises k and v into the pages), kvq8_attention
over the pages, and the feed-forward; then the logits of each sequence's last
row, and sample.  The same step serves prompts, chunks of prompts, verify runs
and single tokens, mixed as they come: only row_start tells them apart.
Sequences take pages from a pool as they grow and give them back at their end.
"""
import os
import sys
from dataclasses import dataclass, field

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import numpy as np  # noqa: E402
import torch  # noqa: E402

import kib  # noqa: E402


@dataclass
class Config:
    vocab: int = 1000
    width: int = 512
    layers: int = 2
    heads: int = 8
    kv_heads: int = 2
    head_dim: int = 64
    ffn: int = 768
    page_tokens: int = 32
    pages: int = 64
    context: int = 256  # positions a sequence may reach
    eps: float = 1e-6
    theta: float = 1e4


@dataclass
class Sequence:
    """A running sequence and how its tokens are drawn."""
    temperature: float = 0.8
    top_k: int = 40
    top_p: float = 0.95
    min_p: float = 0.0
    length: int = 0
    pages: list = field(default_factory=list)


class PagedDecoder:
    def __init__(self, ctx: kib.Context, cfg: Config = Config(), seed: int = 0):
        self.ctx, self.cfg = ctx, cfg
        rng = np.random.default_rng(seed)
        q_width, kv_width = cfg.heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim

        def matrix(rows, cols, qtype=kib.Q4_K):
            w = rng.standard_normal((rows, cols)).astype(np.float32) / np.sqrt(cols)
            return qtype, torch.from_numpy(kib.quantize(qtype, w)).cuda(), rows, cols

        def norm():
            return torch.from_numpy((1.0 + 0.1 * rng.standard_normal(cfg.width)).astype(np.float32)).cuda()

        self.embed, self.head, self.norm = matrix(cfg.vocab, cfg.width, kib.Q6_K), matrix(cfg.vocab, cfg.width, kib.Q6_K), norm()
        self.layers = [dict(norm=norm(), q=matrix(q_width, cfg.width), k=matrix(kv_width, cfg.width), v=matrix(kv_width, cfg.width),
                            o=matrix(cfg.width, q_width), ffn_norm=norm(), gate=matrix(cfg.ffn, cfg.width),
                            up=matrix(cfg.ffn, cfg.width), down=matrix(cfg.width, cfg.ffn)) for _ in range(cfg.layers)]
        shape = (cfg.pages, cfg.kv_heads, cfg.page_tokens, cfg.head_dim)
        self.caches = [kib.KvQ8Cache(*(torch.zeros(shape, dtype=torch.int8, device="cuda") for _ in range(2)),
                                     *(torch.zeros(shape[:2], device="cuda") for _ in range(2))) for _ in range(cfg.layers)]
        half = cfg.head_dim // 2
        self.inv_freq = (1.0 / cfg.theta ** (torch.arange(half, dtype=torch.float32) / half)).cuda()
        self.rope = kib.Rope(self.inv_freq)
        self.free = list(range(cfg.pages))
        # torch's part of a step (copies, the gather of last rows) goes to the context's stream
        self.stream = torch.cuda.ExternalStream(ctx.lib.kib_stream(ctx.h))
        self.workspace = None
        torch.cuda.synchronize()

    def release(self, seq: Sequence):
        self.free += seq.pages
        seq.pages, seq.length = [], 0

    def _place(self, seqs, tokens):
        """Pages for the new tokens, and the batch that describes them."""
        cfg = self.cfg
        grown = [s.length + len(t) for s, t in zip(seqs, tokens)]
        need = [max(0, -(-n // cfg.page_tokens) - len(s.pages)) for s, n in zip(seqs, grown)]
        if max(grown) > cfg.context or sum(need) > len(self.free):
            raise RuntimeError("no room for these tokens")
        table = np.full((len(seqs), -(-cfg.context // cfg.page_tokens)), -1, np.int32)
        for i, (s, n) in enumerate(zip(seqs, need)):
            s.pages += [self.free.pop() for _ in range(n)]
            s.length = grown[i]
            table[i, :len(s.pages)] = s.pages
        start = np.cumsum([0] + [len(t) for t in tokens]).astype(np.int32)
        dev = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()  # noqa: E731
        batch = kib.KvQ8Batch(dev(table), dev(grown), dev(start), int(start[-1]), max(len(t) for t in tokens),
                              max(grown), sum(grown))
        return batch, dev(np.concatenate(tokens)), dev(start[1:] - 1).long()

    def step(self, seqs, tokens, uniform):
        """Runs tokens[i] (at least one each) of seqs[i]; draws a token per
        sequence with uniform[i].  Returns tokens, their probabilities, logits."""
        cfg, ctx = self.cfg, self.ctx
        with torch.cuda.stream(self.stream):
            batch, ids, last = self._place(seqs, tokens)
            n, count = batch.rows, len(seqs)
            new = lambda *shape: torch.empty(*shape, device="cuda")  # noqa: E731
            x, h = new(n, cfg.width), new(n, cfg.width)
            q, out = new(n, cfg.heads, cfg.head_dim), new(n, cfg.heads, cfg.head_dim)
            k, v = new(n, cfg.kv_heads, cfg.head_dim), new(n, cfg.kv_heads, cfg.head_dim)
            gate, up = new(n, cfg.ffn), new(n, cfg.ffn)
            need = ctx.kvq8_attention_workspace(self.caches[0], batch, q)
            if self.workspace is None or self.workspace.numel() < need:
                self.workspace = torch.empty(need, dtype=torch.uint8, device="cuda")
            per = lambda name, dtype: torch.tensor([getattr(s, name) for s in seqs], dtype=dtype).cuda()  # noqa: E731
            settings = dict(temperature=per("temperature", torch.float32), top_k=per("top_k", torch.int32),
                            top_p=per("top_p", torch.float32), min_p=per("min_p", torch.float32))
            uniform = torch.tensor(uniform, dtype=torch.float32).cuda()
            token, prob = torch.empty(count, dtype=torch.int32, device="cuda"), new(count)
            logits, tail, normed = new(count, cfg.vocab), new(count, cfg.width), new(count, cfg.width)
            mul = lambda w, a, o, rows=n: ctx.matmul_kquant(*w, rows, a, o)  # noqa: E731
            norm = lambda w, a, o, rows=n: ctx.call("kib_rms_norm_f32_f32_batched", a, w, rows, cfg.width, cfg.eps, o)  # noqa: E731
            add = lambda a, b: ctx.call("kib_binary_f32_in_place", 0, a, b, a.numel(), cfg.width)  # noqa: E731

            # the calls from here to commit_graph only enqueue: no waits, and nothing that waits (an allocation) between them
            ctx.begin_graph()
            qtype, weight, rows, cols = self.embed
            ctx.dequantize_rows(qtype, weight, rows, ids, n, cols, x)
            for layer, cache in zip(self.layers, self.caches):
                norm(layer["norm"], x, h)
                mul(layer["q"], h, q)
                mul(layer["k"], h, k)
                mul(layer["v"], h, v)
                ctx.kvq8_append(cache, batch, k, v, q=q, q_out=q, rope=self.rope)
                ctx.kvq8_attention(cache, batch, q, out, cfg.head_dim ** -0.5, workspace=self.workspace)
                mul(layer["o"], out, h)
                add(x, h)
                norm(layer["ffn_norm"], x, h)
                mul(layer["gate"], h, gate)
                mul(layer["up"], h, up)
                ctx.call("kib_silu_mul_f32_in_place", gate, up, gate.numel())
                mul(layer["down"], gate, h)
                add(x, h)
            torch.index_select(x, 0, last, out=tail)
            norm(self.norm, tail, normed, count)
            mul(self.head, normed, logits, count)
            ctx.sample(logits, uniform, token, prob, **settings)
            ctx.commit_graph()
            return token.cpu().numpy(), prob.cpu().numpy(), logits


def main():
    rng = np.random.default_rng(1)
    model = PagedDecoder(kib.Context(0))
    seqs = [Sequence(), Sequence(temperature=0.0), Sequence(top_k=0, top_p=0.5), Sequence(min_p=0.2)]
    tokens = [rng.integers(0, model.cfg.vocab, n) for n in (70, 5, 33, 1)]
    texts = [[] for _ in seqs]
    for _ in range(24):
        drawn, prob, _ = model.step(seqs, tokens, rng.random(len(seqs)))
        for text, t in zip(texts, drawn):
            text.append(int(t))
        tokens = [[t] for t in drawn]
    for s, text, p in zip(seqs, texts, prob):
        print(f"{s.length:4d} positions, {len(s.pages)} pages, last probability {p:.3f}:", *text)
        model.release(s)


if __name__ == "__main__":
    main()

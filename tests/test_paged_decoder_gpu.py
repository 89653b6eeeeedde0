"""The example that serves a small decoder from the paged 8-bit cache: append,
attention and sampling as they are used together.

Tolerance of the logits against a model in 64 bits without quantised keys and
values: a page's largest value is about 4 standard deviations, so a code's
rounding is 4 / 127 / sqrt(12) = 0.9 % of one, at keys and at values, at most
twice that where a grown scale rounds again; a residual stream of two layers
carries that to the logits at about the same relative size.  8 % of the logits'
root mean square leaves twice the sum of all four; a position, page or head
taken wrongly moves them by the order of 100 %."""
import importlib.util
import os

import numpy as np
import pytest
import torch

import kib

gpu = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    path = os.path.join(ROOT, "kraken-infer_b200", "examples", "paged_decoder.py")
    spec = importlib.util.spec_from_file_location("paged_decoder", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def plain_logits(model, tokens):
    """Logits of the last token, in 64 bits, with exact keys and values."""
    cfg, ctx = model.cfg, model.ctx

    def dense(w):
        qtype, data, rows, cols = w
        out = torch.empty(rows, cols, device="cuda")
        ctx.dequantize_rows(qtype, data, rows, torch.arange(rows, dtype=torch.int32, device="cuda"), rows, cols, out)
        return out.double().cpu()

    def norm(x, w):
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + cfg.eps) * w.double().cpu()

    n, half = len(tokens), cfg.head_dim // 2
    angle = torch.arange(n).double()[:, None] * model.inv_freq.double().cpu()[None]
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def rotate(x):
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    x = dense(model.embed)[torch.as_tensor(np.asarray(tokens), dtype=torch.long)]
    mask = torch.full((n, n), -torch.inf).double().triu(1)
    for layer in model.layers:
        h = norm(x, layer["norm"])
        q = rotate((h @ dense(layer["q"]).T).view(n, cfg.heads, -1))
        k = rotate((h @ dense(layer["k"]).T).view(n, cfg.kv_heads, -1))
        v = (h @ dense(layer["v"]).T).view(n, cfg.kv_heads, -1)
        k, v = (t.repeat_interleave(cfg.heads // cfg.kv_heads, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) * cfg.head_dim ** -0.5 + mask
        x = x + torch.einsum("hqk,khd->qhd", s.softmax(-1), v).reshape(n, -1) @ dense(layer["o"]).T
        h = norm(x, layer["ffn_norm"])
        x = x + (torch.nn.functional.silu(h @ dense(layer["gate"]).T) * (h @ dense(layer["up"]).T)) @ dense(layer["down"]).T
    return norm(x[-1:], model.norm)[0] @ dense(model.head).T


@gpu
def test_ragged_prompts_chunks_and_steps(example):
    model = example.PagedDecoder(kib.Context(0))
    cfg, rng = model.cfg, np.random.default_rng(3)
    S = example.Sequence
    seqs = [S(temperature=0.0), S(top_k=5), S(top_k=0, top_p=0.5), S(min_p=0.3, top_k=0, top_p=1.0)]
    # a prompt over pages, one token, a prompt to a page's edge, one in two chunks
    text = [list(rng.integers(0, cfg.vocab, n)) for n in (70, 1, 64, 90)]
    tokens = [text[0], text[1], text[2], text[3][:41]]
    drawn, _, _ = model.step(seqs, tokens, [0.5] * 4)
    tokens = [[t] for t in drawn[:3]] + [text[3][41:]]
    for t, d in zip(text, drawn[:3]):
        t.append(int(d))
    for step in range(6):
        drawn, prob, logits = model.step(seqs, tokens, rng.random(4))
        assert ((drawn >= 0) & (drawn < cfg.vocab)).all() and ((prob > 0) & (prob <= 1)).all()
        values = logits.cpu().numpy()
        assert drawn[0] == values[0].argmax()
        assert (values[1] > values[1][drawn[1]]).sum() < 5
        assert values[3].max() - values[3][drawn[3]] <= 0.8 * -np.log(0.3) + 1e-5
        if step in (0, 5):
            for i in range(4):
                want = plain_logits(model, text[i]).numpy()
                assert np.sqrt(((values[i] - want) ** 2).mean()) <= 0.08 * np.sqrt((want ** 2).mean())
        for t, d in zip(text, drawn):
            t.append(int(d))
        tokens = [[t] for t in drawn]
    assert [len(s.pages) for s in seqs] == [-(-s.length // cfg.page_tokens) for s in seqs]
    for s in seqs:
        model.release(s)
    assert sorted(model.free) == list(range(cfg.pages))


@gpu
def test_a_sequence_does_not_depend_on_its_neighbours_pages(example):
    """The same greedy sequence alone, and in pages that others used before."""
    rng = np.random.default_rng(5)
    prompt, other = rng.integers(0, 1000, 50), rng.integers(0, 1000, 200)
    got = []
    for used in (False, True):
        model = example.PagedDecoder(kib.Context(0))
        if used:
            s = example.Sequence()
            model.step([s], [other], [0.1])
            model.release(s)
        s, tokens, drawn = example.Sequence(temperature=0.0), [prompt], []
        for _ in range(8):
            t, _, _ = model.step([s], tokens, [0.0])
            drawn.append(int(t[0]))
            tokens = [t]
        got.append(drawn)
    assert got[0] == got[1]


@gpu
def test_no_room(example):
    model = example.PagedDecoder(kib.Context(0))
    with pytest.raises(RuntimeError):
        model.step([example.Sequence()], [np.zeros(model.cfg.context + 1, np.int64)], [0.0])

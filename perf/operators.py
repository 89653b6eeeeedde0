"""Serving operators over a paged 8-bit KV cache, and token sampling: cases, plain forms and calls.

Three operators that one step of a serving loop runs after another:

* append: rotates the new keys (and the queries) by their positions, quantises keys and values to 8 bits with one
  scale per page and KV head, and writes them into the pages of a block table.  A page's scale grows when a larger
  value arrives; the codes that the page already holds are then rounded again to the new scale.
* attend: causal grouped-query attention of the new rows over the 8-bit pages, ragged over the sequences.
* sample: a token per row of logits by temperature, top-k, top-p and min-p from a given uniform number.

`run` computes them with elementary torch operations in 32 bits (own = False) or by the calls that a user makes of
the kib package (own = True)."""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
FLOAT = {"f32": torch.float32, "f16": torch.float16}
VOCAB = 248320  # the benchmark model's vocabulary
ONE = 1 << 40   # the weight of a row's largest token: weights are 40-bit fixed point, so their sums are exact


def listed():
    kv = dict(heads=8, kv_heads=2, head_dim=256, page=64)
    return [
        # one decode step of 32 slots at about 2048 positions (the batched-decode workload): launch latency
        dict(name="append_slots_32", op="append", type="f32", seqs=32, rows=1, ctx=2048, mix=1, **kv),
        # a whole prompt of 8192 tokens written into fresh pages (the prefill workload)
        dict(name="append_prompt_8192", op="append", type="f32", seqs=1, rows=8192, ctx=8192, mix=0, **kv),
        # ragged prompt chunks of 13 sequences that start and end inside small pages, half-precision rows
        dict(name="append_ragged_13", op="append", type="f16", seqs=13, rows=701, ctx=1999, mix=2, heads=16, kv_heads=4,
             head_dim=128, page=16),
        # one sequence decoding at 4096 positions (the bs1 workload): the smallest attention call
        dict(name="attend_one_4096", op="attend", type="f32", seqs=1, rows=1, ctx=4096, mix=0, **kv),
        # the batched-decode workload's step: 32 slots at about 2048 positions
        dict(name="attend_slots_32", op="attend", type="f32", seqs=32, rows=1, ctx=2048, mix=1, **kv),
        # long ragged contexts, half-precision rows: the cache is read at the rate of memory
        dict(name="attend_long_64", op="attend", type="f16", seqs=64, rows=1, ctx=32768, mix=3, **kv),
        # speculative verify of up to 5 tokens in 17 sequences, pages of 16 tokens, narrower heads
        dict(name="attend_verify_17", op="attend", type="f32", seqs=17, rows=5, ctx=8190, mix=4, heads=16, kv_heads=4,
             head_dim=128, page=16),
        # the last 1024-token prefill chunk of a 32768-token prompt
        dict(name="attend_chunk_1024", op="attend", type="f16", seqs=1, rows=1024, ctx=32768, mix=0, **kv),
        # ragged prompts of odd lengths from their first token, f32 rows
        dict(name="attend_prompts_5", op="attend", type="f32", seqs=5, rows=3001, ctx=3001, mix=5, heads=8, kv_heads=2,
             head_dim=256, page=32),
        # one decoded token: one row of the vocabulary
        dict(name="sample_one", op="sample", rows=1, vocab=VOCAB, mix=6),
        # 32 slots with their own settings, greedy rows and banned tokens among them
        dict(name="sample_slots_32", op="sample", rows=32, vocab=VOCAB, mix=7),
        # a full serving batch
        dict(name="sample_batch_256", op="sample", rows=256, vocab=VOCAB, mix=8),
    ]


def draw(rng):
    def between(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("append", "attend", "sample"))
    mix = rng.randrange(1, 1 << 20)
    if op == "sample":
        return dict(op=op, rows=between(1, 256), vocab=rng.choice((VOCAB, VOCAB, between(1000, VOCAB))), mix=mix)
    kv_heads = rng.choice((1, 2, 4))
    shape = dict(type=rng.choice(("f32", "f16")), heads=kv_heads * rng.choice((1, 2, 4, 8)), kv_heads=kv_heads,
                 head_dim=rng.choice((64, 128, 256)), page=rng.choice((16, 32, 64, 128)), mix=mix)
    if op == "append":
        rows = between(1, 4096)
        return dict(op=op, seqs=between(1, max(1, 8192 // rows)), rows=rows, ctx=rows + between(1, 4096), **shape)
    if rng.random() < 0.5:  # single tokens and short verify runs
        ctx = between(1, 32768)
        return dict(op=op, seqs=between(1, max(1, min(256, 524288 // ctx))), rows=rng.choice((1, 1, 1, 2, 3, 5, 8)),
                    ctx=ctx + 8, **shape)
    rows = between(16, 2048)
    shape["heads"] = kv_heads * min(shape["heads"] // kv_heads, 16 // kv_heads)
    return dict(op=op, seqs=between(1, max(1, 4096 // rows)), rows=rows, ctx=rows + between(1, 4096), **shape)


def sizes(case):
    """Lengths after the call and new rows of each sequence: from the case alone; mix 0 keeps the largest everywhere."""
    n, rows, ctx = case["seqs"], case["rows"], case["ctx"]
    if not case["mix"]:
        return [ctx] * n, [rows] * n
    r = random.Random(case["mix"])
    new = [rows] + [r.randint(max(1, rows // 4), rows) for _ in range(n - 1)]
    length = [ctx] + [max(new[i], r.randint(ctx // 4, ctx)) for i in range(1, n)]
    return length, new


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    uni = lambda *s: torch.rand(*s, generator=g, device=DEV)  # noqa: E731
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        r = random.Random(case["mix"])
        logits = rnd(rows, vocab) * 2.0
        # a few strong candidates per row, as a trained model's head gives
        top = torch.randint(0, vocab, (rows, 24), generator=g, device=DEV)
        logits.scatter_add_(1, top, 6.0 + 5.0 * uni(rows, 24))
        # a tenth of the rows forbid a tenth of the vocabulary
        ban = (uni(rows, 1) < 0.1) & (uni(rows, vocab) < 0.1)
        logits.masked_fill_(ban, -math.inf)
        pick = lambda *of: torch.tensor([r.choice(of) for _ in range(rows)], device=DEV)  # noqa: E731
        return dict(op="sample", logits=logits, uniform=uni(rows),
                    temperature=pick(0.6, 0.7, 0.8, 1.0, 1.0, 1.3) * (pick(*[1.0] * 9, 0.0) if rows > 1 else 1.0),
                    top_k=pick(0, 0, 20, 50, 1000).to(torch.int32), top_p=pick(0.8, 0.9, 0.95, 1.0),
                    min_p=pick(0.0, 0.0, 0.05, 0.1))
    heads, kv, hd, page, seqs = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["seqs"]
    dt = FLOAT[case["type"]]
    length, new = sizes(case)
    need = [-(-x // page) for x in length]
    pages = sum(need) + 3
    width = max(need) + 1
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((seqs, width), -1, dtype=torch.int32, device=DEV)
    cum = [0]
    for x in need:
        cum.append(cum[-1] + x)
    at = torch.arange(width, device=DEV)
    first = torch.tensor(cum[:-1], device=DEV)[:, None]
    held = at[None, :] < torch.tensor(need, device=DEV)[:, None]
    table[held] = order[(first + at)[held]]
    starts = [0]
    for x in new:
        starts.append(starts[-1] + x)
    rows = starts[-1]
    s = dict(op=case["op"], rows=rows, table=table, lengths=torch.tensor(length, dtype=torch.int32, device=DEV),
             row_start=torch.tensor(starts, dtype=torch.int32, device=DEV), max_rows=max(new), page=page,
             max_length=max(length), total_length=sum(length), scale=1.0 / math.sqrt(hd))
    # codes as quantised keys and values look: near-normal with the page's largest value at 127, scales around 0.02
    codes = lambda: (rnd(pages, kv, page, hd) * 34.0).clamp_(-127, 127).round_().to(torch.int8)  # noqa: E731
    scales = lambda: 0.012 * torch.exp(0.3 * rnd(pages, kv)) + 0.012  # noqa: E731
    s.update(k=codes(), v=codes(), k_scale=scales(), v_scale=scales())
    if case["op"] == "attend":
        s["q"] = (rnd(rows, heads, hd) * 2.0).to(dt)
        return s
    # a few channels are larger than the rest, as keys have them
    wide = 1.0 + 3.0 * (torch.arange(hd, device=DEV) % 37 == 5).float()
    s.update(q_in=(rnd(rows, heads, hd)).to(dt), k_in=(rnd(rows, kv, hd) * wide).to(dt), v_in=rnd(rows, kv, hd).to(dt))
    # rotation of the leading quarter of a head, as the benchmark model has it (64 of 256)
    half = hd // 8
    s["inv_freq"] = 1.0 / 1e7 ** (torch.arange(half, device=DEV, dtype=torch.float32) / half)
    # the pages that the new rows reach, for reading back what they hold after the call
    reach = [[i, p] for i in range(seqs) for p in range((length[i] - new[i]) // page, need[i])]
    reach = torch.tensor(reach, device=DEV)
    s["reached"] = table[reach[:, 0], reach[:, 1]].contiguous()
    return s


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 32 * case["rows"], "flops": 3 * n}
    length, new = sizes(case)
    heads, kv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    width = 4 if case["type"] == "f32" else 2
    rows = sum(new)
    if case["op"] == "append":
        # rows in, rotated queries out, codes out; then the reached pages read once and their values (16 bits) written
        reached = sum(-(-length[i] // page) - (length[i] - new[i]) // page for i in range(len(new))) * page * kv * hd
        return {"bytes": rows * (heads * 2 + kv * 2) * hd * width + rows * kv * hd * 2 + reached * 2 * 3,
                "flops": rows * (heads + 2 * kv) * hd * 3}
    pairs = sum(n * (L - n) + n * (n + 1) // 2 for L, n in zip(length, new))
    return {"bytes": sum(length) * kv * hd * 2 + rows * heads * hd * 2 * width, "flops": 4 * pairs * heads * hd}


# ------------------------------------------------------------------ plain forms


def rotate(x, angle):
    """x [rows][heads][head_dim], the leading 2 * angles of a head rotated in pairs (i, i + angles)."""
    half = angle.shape[1]
    c, s = torch.cos(angle)[:, None, :], torch.sin(angle)[:, None, :]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat((a * c - b * s, b * c + a * s, x[..., 2 * half:]), -1)


def row_places(s):
    """Of each new row: its sequence and its position in the cache."""
    rows = torch.arange(s["rows"], device=DEV)
    seq = torch.searchsorted(s["row_start"][1:].long().contiguous(), rows, right=True)
    new = (s["row_start"][1:] - s["row_start"][:-1]).long()
    pos = s["lengths"].long()[seq] - new[seq] + rows - s["row_start"].long()[seq]
    return seq, pos


def plain_store(x, codes, scales, page, seq, pos, table):
    """Quantises x [rows][kv_heads][head_dim] into the pages in place."""
    at = table.long()[seq, pos // page]
    off = pos % page
    big = torch.zeros_like(scales).index_reduce_(0, at, x.abs().amax(-1), "amax", include_self=True)
    first = torch.full((codes.shape[0],), page, device=DEV, dtype=torch.int64)
    first.scatter_reduce_(0, at, off, "amin", include_self=True)  # where the new rows of a page begin
    touched = first < page
    old = torch.where((first > 0)[:, None], scales, torch.zeros_like(scales))
    now = torch.maximum(old, big / 127.0)
    now = torch.where(touched[:, None], now, scales)
    # codes that a touched page already holds move to its new scale
    ids = touched.nonzero()[:, 0]
    ratio = torch.where(now[ids] > 0, old[ids] / now[ids], torch.zeros_like(now[ids]))
    kept = torch.arange(page, device=DEV)[None, :] < first[ids][:, None]
    held = codes[ids]
    again = torch.round(held.float() * ratio[:, :, None, None]).to(torch.int8)
    codes[ids] = torch.where(kept[:, None, :, None], again, held)
    inv = torch.where(now[at] > 0, 1.0 / now[at], torch.zeros_like(now[at]))
    codes[at, :, off] = torch.round(x * inv[..., None]).clamp(-127, 127).to(torch.int8)
    scales.copy_(now)


def plain_append(s):
    seq, pos = row_places(s)
    angle = pos.float()[:, None] * s["inv_freq"][None, :]
    q = rotate(s["q_in"].float(), angle).to(s["q_in"].dtype)
    plain_store(rotate(s["k_in"].float(), angle), s["k"], s["k_scale"], s["page"], seq, pos, s["table"])
    plain_store(s["v_in"].float(), s["v"], s["v_scale"], s["page"], seq, pos, s["table"])
    ids = s["reached"].long()
    return dict(q=q, k=(s["k"][ids].float() * s["k_scale"][ids][:, :, None, None]).half(),
                v=(s["v"][ids].float() * s["v_scale"][ids][:, :, None, None]).half())


def plain_attend(s):
    q = s["q"].float()
    heads, hd = q.shape[1:]
    n, width = s["table"].shape
    kv, page, most = s["k"].shape[1], s["page"], s["max_rows"]
    ids = s["table"].clamp(min=0).long()
    keys = (s["k"][ids].float() * s["k_scale"][ids][..., None, None]).permute(0, 2, 1, 3, 4).reshape(n, kv, width * page, hd)
    values = (s["v"][ids].float() * s["v_scale"][ids][..., None, None]).permute(0, 2, 1, 3, 4).reshape(n, kv, width * page, hd)
    row = s["row_start"][:-1].long()[:, None] + torch.arange(most, device=DEV)
    live = row < s["row_start"][1:].long()[:, None]
    new = (s["row_start"][1:] - s["row_start"][:-1]).long()
    pos = torch.where(live, (s["lengths"].long() - new)[:, None] + torch.arange(most, device=DEV), -1)
    padded = q[torch.where(live, row, 0)]  # [n][most][heads][hd]
    padded = padded.reshape(n, most, kv, heads // kv, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, heads // kv * most, hd)
    score = torch.matmul(padded, keys.transpose(-1, -2)).reshape(n, kv, heads // kv, most, width * page) * s["scale"]
    seen = torch.arange(width * page, device=DEV)[None, None, :] <= pos[:, :, None]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(p.reshape(n, kv, -1, width * page), values).reshape(n, kv, heads // kv, most, hd)
    return o.permute(0, 3, 1, 2, 4).reshape(n, most, heads, hd)[live].to(s["q"].dtype)


def plain_sample(s):
    logits = s["logits"]
    logits = torch.where(torch.isnan(logits), -math.inf, logits)
    rows, vocab = logits.shape
    top = logits.amax(-1, keepdim=True)
    greedy = s["temperature"] <= 1e-6
    t = torch.where(greedy, 1.0, s["temperature"])[:, None]
    e = torch.exp((logits - top) * (1.0 / t))
    w = (e * float(ONE)).to(torch.int64)
    by, order = torch.sort(logits, dim=-1, descending=True, stable=True)
    ws, es = w.gather(1, order), e.gather(1, order)
    rank = torch.arange(vocab, device=DEV)[None, :]
    k = s["top_k"].long()[:, None]
    keep = (rank < k) | (k <= 0)
    ws = torch.where(keep, ws, 0)
    run = torch.cumsum(ws, -1)
    limit = (run[:, -1:].double() * s["top_p"].double()[:, None]).to(torch.int64)
    keep &= (run - ws < limit) | (s["top_p"][:, None] >= 1)
    keep &= es >= s["min_p"][:, None]
    keep |= rank == 0
    w = torch.where(torch.zeros_like(keep).scatter(1, order, keep), w, 0)
    run = torch.cumsum(w, -1)
    total = run[:, -1:]
    aim = torch.minimum((total.double() * s["uniform"].double()[:, None]).to(torch.int64), total - 1)
    token = (run <= aim).sum(-1).clamp(max=vocab - 1)
    prob = w.gather(1, token[:, None])[:, 0].double() / total[:, 0].double()
    token = torch.where(greedy, torch.where(logits == top, rank, vocab).amin(-1), token)
    return dict(token=token.to(torch.int32), prob=torch.where(greedy, 1.0, prob.float()))


# ------------------------------------------------------------------ the framework's calls

_kib = []


def kib_context():
    """The package and one context, kept by the process."""
    if not _kib:
        sys.path.insert(0, os.path.join(os.getcwd(), "kraken-infer_b200"))
        import kib
        _kib.extend((kib, kib.Context(0)))
    return _kib


def own_cache(s):
    kib, ctx = kib_context()
    if "cache" not in s:
        s["cache"] = kib.KvQ8Cache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        s["batch"] = kib.KvQ8Batch(s["table"], s["lengths"], s["row_start"], s["rows"], s["max_rows"],
                                   s["max_length"], s["total_length"])
    return kib, ctx, s["cache"], s["batch"], torch.cuda.current_stream().cuda_stream


def own_append(s):
    kib, ctx, cache, batch, stream = own_cache(s)
    q = torch.empty_like(s["q_in"])
    ctx.kvq8_append(cache, batch, s["k_in"], s["v_in"], q=s["q_in"], q_out=q, rope=kib.Rope(s["inv_freq"]), stream=stream)
    k = torch.empty((len(s["reached"]),) + s["k"].shape[1:], dtype=torch.float16, device=DEV)
    v = torch.empty_like(k)
    ctx.kvq8_read_pages(cache, s["reached"], k, v, stream=stream)
    return dict(q=q, k=k, v=v)


def own_attend(s):
    kib, ctx, cache, batch, stream = own_cache(s)
    out = torch.empty_like(s["q"])
    ctx.kvq8_attention(cache, batch, s["q"], out, s["scale"], stream=stream)
    return out


def own_sample(s):
    kib, ctx = kib_context()
    rows = s["logits"].shape[0]
    token = torch.empty(rows, dtype=torch.int32, device=DEV)
    prob = torch.empty(rows, device=DEV)
    ctx.sample(s["logits"], s["uniform"], token, prob, temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
               min_p=s["min_p"], stream=torch.cuda.current_stream().cuda_stream)
    return dict(token=token, prob=prob)


def run(state):
    if own:
        return {"append": own_append, "attend": own_attend, "sample": own_sample}[state["op"]](state)
    return {"append": plain_append, "attend": plain_attend, "sample": plain_sample}[state["op"]](state)


# ------------------------------------------------------------------ in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return exact_sample(s)
    length, new = sizes(case)
    page = case["page"]
    if case["op"] == "attend":
        heads, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
        outs, at = [], 0
        for i in range(case["seqs"]):
            pos = torch.arange(length[i], device=DEV)
            p = s["table"][i].long()[pos // page]
            key = s["k"][p, :, pos % page].double() * s["k_scale"][p].double()[..., None]   # [L][kv][hd]
            val = s["v"][p, :, pos % page].double() * s["v_scale"][p].double()[..., None]
            q = s["q"][at:at + new[i]].double().reshape(new[i], kv, heads // kv, hd)
            score = torch.einsum("tkgd,lkd->kgtl", q, key) * s["scale"]
            t = torch.arange(new[i], device=DEV) + length[i] - new[i]
            score.masked_fill_(pos[None, :] > t[:, None], -math.inf)
            outs.append(torch.einsum("kgtl,lkd->tkgd", torch.softmax(score, -1), val).reshape(new[i], heads, hd))
            at += new[i]
        return torch.cat(outs)
    # the rotation angle is the product of position and frequency in 32 bits, as the framework's rotation defines it
    pos = torch.cat([torch.arange(length[i] - new[i], length[i], device=DEV) for i in range(case["seqs"])])
    angle = (pos.float()[:, None] * s["inv_freq"]).double()

    def turn(x):
        x, half = x.double().clone(), angle.shape[1]
        a, b = x[..., :half].clone(), x[..., half:2 * half].clone()
        x[..., :half] = a * angle.cos()[:, None] - b * angle.sin()[:, None]
        x[..., half:2 * half] = a * angle.sin()[:, None] + b * angle.cos()[:, None]
        return x

    q = turn(s["q_in"])
    got = []
    for x, codes, scales in ((turn(s["k_in"]), s["k"], s["k_scale"]), (s["v_in"].double(), s["v"], s["v_scale"])):
        codes, scales, at = codes.double(), scales.double(), 0
        for i in range(case["seqs"]):
            p0, p1 = length[i] - new[i], length[i]
            while p0 < p1:
                stop = min(p1, (p0 // page + 1) * page)
                p, o = int(s["table"][i, p0 // page]), p0 % page
                part = x[at:at + stop - p0].transpose(0, 1)  # [kv][rows][hd]
                was = scales[p] if o else torch.zeros_like(scales[p])
                now = torch.maximum(was, part.abs().amax((1, 2)) / 127)
                codes[p, :, :o] = torch.round(codes[p, :, :o] * (was / now)[:, None, None])
                codes[p, :, o:o + stop - p0] = torch.round(part / now[:, None, None]).clamp(-127, 127)
                scales[p] = now
                at, p0 = at + stop - p0, stop
        ids = s["reached"].long()
        got.append(codes[ids] * scales[ids][:, :, None, None])
    return dict(q=q, k=got[0], v=got[1])


def exact_sample(s):
    tokens, probs = [], []
    for i in range(s["logits"].shape[0]):
        x = s["logits"][i].double()
        t = float(s["temperature"][i])
        value, order = torch.sort(x, descending=True, stable=True)
        if t <= 1e-6:
            tokens.append(int(order[0]))
            probs.append(1.0)
            continue
        p = torch.exp((value - value[0]) / t)
        n = int(s["top_k"][i])
        if n > 0:
            p = p[:n]
        keep = p >= float(s["min_p"][i])
        if float(s["top_p"][i]) < 1:
            keep &= torch.cumsum(p, 0) - p < float(s["top_p"][i]) * p.sum()
        keep[0] = True
        left = torch.zeros_like(x)
        left[order[:len(p)][keep]] = p[keep]
        run_ = torch.cumsum(left, 0)
        token = int((run_ <= float(s["uniform"][i]) * run_[-1]).sum())
        tokens.append(token)
        probs.append(float(left[token] / run_[-1]))
    return dict(token=torch.tensor(tokens, dtype=torch.int32), prob=torch.tensor(probs, dtype=torch.float64))

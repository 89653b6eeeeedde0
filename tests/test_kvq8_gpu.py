"""The paged 8-bit KV cache (kib_kvq8_*) against plain forms in 64 bits: append
with rotation, reading pages, ragged causal attention, and their refusals.

Tolerances.  Codes: the quotient x / scale is known to 2e-4 (127 times the
rounding of the rotated value, 12 half-ulps of fp32, of its scale and of the
reciprocal), so a code equals the 64-bit one unless that quotient lies within
2e-4 of a half-integer, and is off by at most one there; a code that is rounded
again to a grown scale has twice that.  Attention: a score carries at most 2^-20 of
sum |q_i k_i| * scale (16 half-ulps of fp32 over the absolute sum), a softmax
weight twice that relatively, the sums 2^-19; half rows add 2^-11 for the
weights and 2^-11 for the result.  All relative to the largest |v| attended."""
import math

import numpy as np
import pytest
import torch

import kib

gpu = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16}


class Case:
    """Sequences with lengths (new rows included) and new rows, their cache on
    the GPU, and copies of everything in numpy for the oracle."""

    def __init__(self, lengths, new, heads=4, kv=2, hd=64, page=16, dtype="f32", seed=0, layout="packed", spread=1.0):
        r = np.random.default_rng(seed)
        self.lengths, self.new, self.heads, self.kv, self.hd, self.page = lengths, new, heads, kv, hd, page
        n = len(lengths)
        need = [max(0, -(-x // page)) for x in lengths]
        self.pages = sum(need) + 2
        self.width = max(need + [1]) + 1
        order = r.permutation(self.pages)
        self.table = np.full((n, self.width), -1, np.int32)
        at = 0
        for i in range(n):
            self.table[i, :need[i]] = order[at:at + need[i]]
            at += need[i]
        self.codes = [r.integers(-127, 128, (self.pages, kv, page, hd)).astype(np.int8) for _ in range(2)]
        self.scales = [(0.01 + 0.02 * r.random((self.pages, kv))).astype(np.float32) for _ in range(2)]
        self.start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        rows = int(self.start[-1])
        rnd = lambda h: torch.from_numpy((r.standard_normal((rows, h, hd)) * spread).astype(np.float32)).to(DT[dtype])  # noqa: E731
        self.q, self.k, self.v = rnd(heads), rnd(kv), rnd(kv)
        self.dtype, self.rows = dtype, rows
        dev = []
        for c in self.codes:
            if layout == "packed":
                dev.append(torch.from_numpy(c).cuda())
            elif layout == "token_major":  # [page][token][head][d] in memory
                dev.append(torch.from_numpy(c).permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3))
            else:  # padded rows, and other layers' pages in between
                big = torch.zeros(self.pages, 3, kv, page, hd + 16, dtype=torch.int8, device="cuda")
                view = big[:, 1, :, :, :hd]
                view.copy_(torch.from_numpy(c))
                dev.append(view)
        self.dev = dev + [torch.from_numpy(s.copy()).cuda() for s in self.scales]
        self.cache = kib.KvQ8Cache(*self.dev)
        cuda = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()  # noqa: E731
        self.lengths_dev = cuda(lengths)
        self.batch = kib.KvQ8Batch(cuda(self.table), self.lengths_dev, cuda(self.start), rows, max(list(new) + [0]))

    def positions(self, i):
        """Cache positions of sequence i's new rows."""
        return np.arange(self.lengths[i] - self.new[i], self.lengths[i])


def rotate64(x, angle):
    x, half = x.astype(np.float64).copy(), angle.shape[-1]
    c, s = np.cos(angle)[:, None, :], np.sin(angle)[:, None, :]
    a, b = x[..., :half].copy(), x[..., half:2 * half].copy()
    x[..., :half], x[..., half:2 * half] = a * c - b * s, b * c + a * s
    return x


def oracle_append(c, x, codes, scales):
    """Quotients (before rounding) and scales after the rows x (64-bit) are
    stored; quotients of everything not touched are its codes."""
    quo, scales = codes.astype(np.float64), scales.astype(np.float64)
    fresh = np.zeros(codes.shape, bool)
    for i in range(len(c.lengths)):
        p, stop, row = max(0, c.lengths[i] - c.new[i]), c.lengths[i], c.start[i] + max(0, c.new[i] - c.lengths[i])
        while p < stop:
            end = min(stop, (p // c.page + 1) * c.page)
            page, lo = c.table[i, p // c.page], p % c.page
            part = x[row:row + end - p]  # [rows][kv][hd]
            row, n, p = row + end - p, end - p, end
            if page < 0:
                continue
            big = np.where(np.isfinite(part), np.abs(part), 0).max((0, 2))
            old = scales[page] if lo else np.zeros_like(big)
            now = np.maximum(old, big / 127)
            with np.errstate(all="ignore"):
                ratio = np.where(now > 0, old / now, 0)
                inv = np.where(now > 0, 1 / now, 0)
                quo[page, :, :lo] *= ratio[:, None, None]
                y = part * inv[None, :, None]
            quo[page, :, lo:lo + n] = np.where(np.isnan(part), 0, np.clip(np.nan_to_num(y, nan=0), -127, 127)).transpose(1, 0, 2)
            fresh[page, :, lo:lo + n] = True
            scales[page] = now
    return quo, scales, fresh


def check_codes(got, quo, fresh):
    want = np.rint(quo)
    edge = np.abs(np.abs(quo - np.floor(quo)) - 0.5)
    diff = np.abs(got.astype(np.int64) - want)
    assert diff.max() <= 1
    assert not (diff[fresh] > 0)[edge[fresh] > 2e-4].any()
    assert not (diff[~fresh] > 0)[edge[~fresh] > 4e-4].any()


def inv_freq(pairs, theta=1e4):
    return (1.0 / theta ** (np.arange(pairs) / pairs)).astype(np.float32)


def run_append(ctx, c, pairs=8, sections=(0, 0, 0, 0), positions=None, in_place=False, stream=None):
    q, k, v = c.q.cuda(), c.k.cuda(), c.v.cuda()
    q_out = q if in_place else torch.empty_like(q)
    rope = None
    if pairs:
        rope = kib.Rope(torch.from_numpy(inv_freq(pairs)).cuda(), sections,
                        None if positions is None else torch.from_numpy(positions).cuda())
    torch.cuda.synchronize()
    ctx.kvq8_append(c.cache, c.batch, k, v, q=q, q_out=q_out, rope=rope, stream=stream)
    torch.cuda.synchronize()
    return q_out.cpu().float().numpy()


def check_append(ctx, c, pairs=8, sections=(0, 0, 0, 0), positions=None, **kw):
    got_q = run_append(ctx, c, pairs, sections, positions, **kw)
    pos = np.concatenate([c.positions(i) for i in range(len(c.lengths))])
    if positions is None:
        per = np.repeat(pos[:, None], max(pairs, 1), 1)
    else:
        tot = sum(sections)
        stream = [0 if not tot else (0 if j % tot < sections[0] else 1 if j % tot < sum(sections[:2]) else
                                     2 if j % tot < sum(sections[:3]) else 3) for j in range(pairs)]
        per = np.stack([positions[s] for s in stream], 1)
    angle = (per[:, :pairs].astype(np.float32) * inv_freq(pairs)[None] if pairs else np.zeros((c.rows, 0))).astype(np.float64)
    kept = pos >= 0
    q, k = rotate64(c.q.float().numpy(), angle), rotate64(c.k.float().numpy(), angle)
    tol = 1e-6 * np.abs(q).max(-1, keepdims=True) + (2.0 ** -11 * np.abs(q) + 2.0 ** -25 if c.dtype == "f16" else 0)
    assert (np.abs(got_q - q) <= tol)[kept].all()
    for x, at in ((k, 0), (c.v.float().numpy().astype(np.float64), 1)):
        quo, scales, fresh = oracle_append(c, x, c.codes[at], c.scales[at])
        assert np.allclose(c.dev[2 + at].cpu().numpy(), scales, rtol=2e-6, atol=0)
        check_codes(c.dev[at].cpu().numpy(), quo, fresh)
    # read back: code * scale
    ids = torch.arange(-1, c.pages + 1, dtype=torch.int32, device="cuda")
    shape = (c.pages + 2, c.kv, c.page, c.hd)
    out = [torch.full(shape, 7.0, dtype=DT[c.dtype], device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    ctx.kvq8_read_pages(c.cache, ids, out[0], out[1])
    for x, codes, scales in zip(out, c.dev[:2], c.dev[2:]):
        assert (x[0] == 0).all() and (x[-1] == 0).all()
        assert torch.equal(x[1:-1], (codes.float() * scales[:, :, None, None]).to(DT[c.dtype]))


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd,page,layout", [(64, 16, "packed"), (128, 32, "token_major"), (256, 64, "padded"),
                                            (256, 128, "packed"), (128, 16, "padded")])
def test_append(ctx, dtype, hd, page, layout):
    # runs inside a page, ending at its edge, over many pages, one row, none, from the first position
    c = Case([5, page, 3 * page + 7, 2 * page, 1, 40], [5, 1, 2 * page + 9, 0, 1, 3], heads=6, kv=2, hd=hd, page=page,
             dtype=dtype, seed=hd + page, layout=layout)
    check_append(ctx, c, pairs=hd // 8)


@gpu
def test_append_rotation_positions_and_in_place(ctx):
    c = Case([33, 20], [30, 20], hd=64, seed=5)
    r = np.random.default_rng(1)
    check_append(ctx, c, pairs=32, sections=(11, 11, 10, 0), positions=r.integers(0, 200000, (4, 50)).astype(np.int32),
                 in_place=True)
    check_append(ctx, Case([33, 20], [30, 20], hd=64, seed=6), pairs=0)
    check_append(ctx, Case([9], [9], hd=64, seed=7, dtype="f16"), pairs=5, in_place=True)


@gpu
def test_append_positions_before_the_first_are_dropped(ctx):
    # more new rows than positions: the first rows have no place
    check_append(ctx, Case([10, 3], [14, 3], seed=8))


@gpu
def test_append_one_by_one_grows_the_scale(ctx):
    """Rows of growing size: each one enlarges the scale, the codes before it
    are rounded again; the page stays within the sum of the roundings."""
    c = Case([1], [1], kv=1, heads=1, hd=64, seed=3)
    r = np.random.default_rng(0)
    rows = r.standard_normal((16, 64)) * (1.0 + np.arange(16)[:, None])
    rows = rows.astype(np.float32)
    for i in range(16):
        c.lengths_dev.fill_(i + 1)
        x = torch.from_numpy(rows[i]).cuda().reshape(1, 1, 64)
        torch.cuda.synchronize()
        ctx.kvq8_append(c.cache, c.batch, x, x)
    page = c.table[0, 0]
    s = float(c.dev[2][page, 0])
    assert s == pytest.approx(np.abs(rows).max() / 127, rel=1e-6)
    got = c.dev[0][page, 0].cpu().numpy() * s
    # each of at most 16 roundings costs half a unit of a scale no larger than the last
    assert np.abs(got - rows).max() <= 16 * 0.5 * s
    assert np.abs(got[15] - rows[15]).max() <= 0.5 * s * (1 + 1e-5)


@gpu
def test_append_values_that_are_not_finite(ctx):
    c = Case([20], [20], kv=1, heads=1, seed=4)
    c.k[3, 0, 20], c.k[4, 0, 21], c.k[5, 0, 22] = math.inf, -math.inf, math.nan
    c.v[:] = 0
    run_append(ctx, c, pairs=0)
    quo, scales, fresh = oracle_append(c, c.k.numpy().astype(np.float64), c.codes[0], c.scales[0])
    check_codes(c.dev[0].cpu().numpy(), quo, fresh)
    page = c.table[0, 0]
    assert [int(c.dev[0][page, 0, t, d]) for t, d in ((3, 20), (4, 21), (5, 22))] == [127, -127, 0]
    assert np.allclose(c.dev[2].cpu().numpy(), scales, rtol=2e-6)
    # all zeros: scale 0, codes 0
    assert float(c.dev[3][page, 0]) == 0.0 and not c.dev[1][page, 0].any()


@gpu
def test_append_skips_absent_pages_and_strided_rows(ctx):
    c = Case([40], [40], kv=2, heads=4, seed=9)
    c.table[0, 1] = -1
    c.batch.tensors[0].copy_(torch.from_numpy(c.table))
    before = [x.clone() for x in c.dev]
    joined = torch.cat([c.q, c.k, c.v], 1).cuda()  # one row holds q | k | v
    q, k, v = joined[:, :4], joined[:, 4:6], joined[:, 6:]
    torch.cuda.synchronize()
    ctx.kvq8_append(c.cache, c.batch, k, v, q=q, q_out=q)
    for x, at in ((c.k, 0), (c.v, 1)):
        quo, scales, fresh = oracle_append(c, x.numpy().astype(np.float64), c.codes[at], c.scales[at])
        check_codes(c.dev[at].cpu().numpy(), quo, fresh)
        lost = [p for p in range(c.pages) if p not in c.table[0]]
        assert torch.equal(c.dev[at][lost], before[at][lost]) and torch.equal(c.dev[2 + at][lost], before[2 + at][lost])


def oracle_attend(c, scale):
    """Outputs and the largest error allowed, per row and head."""
    q = c.q.float().numpy().astype(np.float64)
    out, tol = np.zeros_like(q), np.zeros(q.shape[:2])
    codes = [x.cpu().numpy().astype(np.float64) for x in c.dev[:2]]
    scales = [x.cpu().numpy().astype(np.float64) for x in c.dev[2:]]
    for i in range(len(c.lengths)):
        L, n = max(0, c.lengths[i]), c.new[i]
        pos = np.arange(L)
        page = c.table[i][pos // c.page] if L else np.zeros(0, np.int64)
        here = (page >= 0) & (page < c.pages)
        pos, page = pos[here], page[here]
        key, val = ((x[page, :, pos % c.page] * s[page][..., None]) for x, s in zip(codes, scales))  # [L][kv][hd]
        for t in range(n):
            row, end = c.start[i] + t, np.searchsorted(pos, c.lengths[i] - n + t, side="right")
            if end == 0:
                continue
            for h in range(c.heads):
                g = h // (c.heads // c.kv)
                sc = key[:end, g] @ q[row, h] * scale
                big = np.abs(key[:end, g]) @ np.abs(q[row, h]) * abs(scale)
                p = np.exp(sc - sc.max())
                p /= p.sum()
                out[row, h] = p @ val[:end, g]
                tol[row, h] = (2 * 2.0 ** -20 * big.max() + 2.0 ** -19 + (2.0 ** -10 if c.dtype == "f16" else 0)) * np.abs(
                    val[:end, g]).max()
    return out, tol


def run_attend(ctx, c, scale, stream=None, workspace=None):
    q = c.q.cuda()
    out = torch.full_like(q, 77.0)
    torch.cuda.synchronize()
    ctx.kvq8_attention(c.cache, c.batch, q, out, scale, stream=stream, workspace=workspace)
    torch.cuda.synchronize()
    return out


def check_attend(ctx, c, scale=None):
    scale = scale if scale is not None else 1.0 / math.sqrt(c.hd)
    got = run_attend(ctx, c, scale).cpu().float().numpy()
    want, tol = oracle_attend(c, scale)
    err = np.abs(got - want).max(-1)
    assert (err <= tol).all(), float((err - tol).max())
    return got


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv,hd,page,layout", [(8, 2, 256, 64, "packed"), (4, 4, 64, 16, "token_major"),
                                                     (6, 2, 128, 32, "padded"), (16, 1, 256, 128, "packed"),
                                                     (5, 1, 64, 16, "padded"), (8, 8, 128, 16, "packed")])
def test_attention_single_rows(ctx, dtype, heads, kv, hd, page, layout):
    lengths = [1, 17, 0, page, 3 * page + 1, 700, 63]
    check_attend(ctx, Case(lengths, [1] * 7, heads, kv, hd, page, dtype, seed=heads + hd, layout=layout, spread=1.5))


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd,page", [(256, 64), (128, 16), (64, 128)])
def test_attention_few_rows(ctx, dtype, hd, page):
    # verify runs of several rows, sequences without rows, more rows than positions
    check_attend(ctx, Case([5, 100, 300, 2, 64, 33], [5, 3, 0, 4, 8, 2], 8, 2, hd, page, dtype, seed=hd))


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv,hd,page", [(8, 2, 256, 64), (4, 4, 128, 16), (6, 1, 64, 32), (8, 2, 256, 16),
                                              (16, 2, 128, 128)])
def test_attention_many_rows(ctx, dtype, heads, kv, hd, page):
    # prompts from their first position, chunks late in a sequence, ragged with single rows
    check_attend(ctx, Case([77, 300, 1, 513, 130], [77, 44, 1, 150, 129], heads, kv, hd, page, dtype, seed=hd + page))


@gpu
@pytest.mark.parametrize("rows", [1, 90])
def test_attention_absent_pages_and_masked_junk(ctx, rows):
    """Absent pages are left out; codes past the length and the scales of
    pages that are not reached (NaN, infinity) change nothing."""
    c = Case([200, 150], [rows, rows], seed=11, hd=128)
    c.table[0, 2] = c.pages + 5
    c.table[1, 0] = -7
    c.batch.tensors[0].copy_(torch.from_numpy(c.table))
    used = set(c.table[0]) | set(c.table[1])
    for p in range(c.pages):
        if p not in used:
            c.dev[2][p], c.dev[3][p] = math.nan, math.inf
    a = check_attend(ctx, c)
    last = c.table[0, 199 // c.page]
    for x in c.dev[:2]:
        x[last, :, 199 % c.page + 1:] = -128
    assert np.array_equal(check_attend(ctx, c), a)


@gpu
def test_attention_rows_whose_every_key_is_absent_are_zero(ctx):
    c = Case([40, 40], [1, 40], seed=12)
    c.table[:] = -1
    c.batch.tensors[0].copy_(torch.from_numpy(c.table))
    assert not run_attend(ctx, c, 0.125).any()


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows", [1, 70])
def test_attention_scales_far_apart(ctx, dtype, rows):
    """Pages whose scales differ by factors of 1e5, zero scales, and scores so
    sharp that one key takes all the weight."""
    c = Case([400, 129], [rows, rows], hd=128, seed=13, dtype=dtype)
    r = np.random.default_rng(3)
    c.dev[3].copy_(torch.from_numpy((10.0 ** r.uniform(-6, -1, c.scales[1].shape)).astype(np.float32)))
    c.dev[3][c.table[0, 3]] = 0.0
    c.dev[2][c.table[0, 1]] = 0.0
    check_attend(ctx, c)
    check_attend(ctx, c, scale=2.0)
    check_attend(ctx, c, scale=-0.1)
    check_attend(ctx, c, scale=0.0)


@gpu
def test_attention_is_the_same_every_time_and_on_another_stream(ctx):
    c = Case([3000, 1, 777, 2048], [1, 1, 6, 1], 8, 2, 256, 64, seed=14)
    a = run_attend(ctx, c, 0.06)
    for _ in range(3):
        assert torch.equal(run_attend(ctx, c, 0.06), a)
    side = torch.cuda.Stream()
    q = c.q.cuda()
    need = ctx.kvq8_attention_workspace(c.cache, c.batch, q)
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device="cuda")
    assert torch.equal(run_attend(ctx, c, 0.06, stream=side.cuda_stream, workspace=ws), a)
    assert torch.equal(run_attend(ctx, c, 0.06, stream=0), a)


@gpu
@pytest.mark.parametrize("rows", [1, 100])
def test_append_and_attention_in_a_captured_graph(ctx, rows):
    """Enqueued on a capturing stream and replayed on new inputs."""
    c = Case([300, 140], [rows, rows], 8, 2, 128, 32, seed=15)
    q, k, v = c.q.cuda(), c.k.cuda(), c.v.cuda()
    out = torch.empty_like(q)
    ws = torch.empty(max(ctx.kvq8_attention_workspace(c.cache, c.batch, q), 256), dtype=torch.uint8, device="cuda")

    def step(stream):
        ctx.kvq8_append(c.cache, c.batch, k, v, stream=stream)
        ctx.kvq8_attention(c.cache, c.batch, q, out, 0.09, workspace=ws, stream=stream)

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    step(side.cuda_stream)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step(torch.cuda.current_stream().cuda_stream)
    q.mul_(0.5)
    k.mul_(1.5)
    g.replay()
    torch.cuda.synchronize()
    replayed = out.clone()
    out.zero_()
    torch.cuda.synchronize()
    step(None)
    assert torch.equal(out, replayed)


@gpu
def test_refusals(ctx):
    c = Case([33, 20], [1, 2], 8, 2, 64, 16, seed=1)
    q, k, v = c.q.cuda(), c.k.cuda(), c.v.cuda()
    out = torch.empty_like(q)
    lib = ctx.lib

    def refused(rc, word):
        assert rc == kib.KIB_ERR_INVALID_ARGUMENT
        assert word in lib.kib_last_error(ctx.h).decode()

    def attend(cache=c.cache, batch=c.batch, kind=0, heads=8, qp=q.data_ptr(), qs=0, scale=0.1, op=out.data_ptr(), os_=0,
               ws=None, size=0):
        need = ctx.kvq8_attention_workspace(c.cache, c.batch, q)
        if ws is None:
            attend.ws = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
            ws, size = attend.ws.data_ptr(), need
        return lib.kib_kvq8_attention(ctx.h, cache.c, batch.c, kind, heads, qp, qs, scale, op, os_, ws, size, None)

    def with_cache(**kw):
        x = kib.KvQ8Cache(*c.dev)
        for n, val in kw.items():
            setattr(x.c, n, val)
        return x

    def with_batch(**kw):
        x = kib.KvQ8Batch(*c.batch.tensors, c.rows, 2)
        for n, val in kw.items():
            setattr(x.c, n, val)
        return x

    assert attend() == kib.KIB_OK
    refused(attend(cache=with_cache(head_dim=96)), "head_dim")
    refused(attend(cache=with_cache(page_tokens=48)), "page_tokens")
    refused(attend(cache=with_cache(kv_heads=0)), "kv_heads")
    refused(attend(cache=with_cache(pages=0)), "pages")
    refused(attend(cache=with_cache(k=None)), "null")
    refused(attend(cache=with_cache(token_stride=72)), "16")
    refused(attend(cache=with_cache(token_stride=32)), "smaller")
    refused(attend(cache=with_cache(v=c.dev[1].data_ptr() + 1)), "16")
    refused(attend(batch=with_batch(lengths=None)), "null")
    refused(attend(batch=with_batch(block_table=None)), "block table")
    refused(attend(batch=with_batch(max_rows=0)), "max_rows")
    refused(attend(batch=with_batch(max_rows=4)), "max_rows")
    refused(attend(batch=with_batch(sequences=1 << 20)), "sequences")
    refused(attend(batch=with_batch(table_stride=1 << 29)), "2^31")
    refused(attend(kind=12), "type")
    refused(attend(heads=7), "heads")
    refused(attend(heads=0), "heads")
    refused(attend(qp=None), "null")
    refused(attend(qp=q.data_ptr() + 4), "16")
    refused(attend(qs=100), "smaller")
    refused(attend(os_=514), "16")
    refused(attend(scale=math.nan), "finite")
    need = ctx.kvq8_attention_workspace(c.cache, c.batch, q)
    if need:
        refused(attend(ws=attend.ws.data_ptr(), size=need - 1), "workspace")
        refused(attend(ws=attend.ws.data_ptr() + 16, size=need), "workspace")

    def append(cache=c.cache, rope=None, kind=0, heads=8, qp=q.data_ptr(), kp=k.data_ptr(), op=out.data_ptr(), ks=0, os_=0):
        return lib.kib_kvq8_append(ctx.h, cache.c, c.batch.c, rope.c if rope else None, kind, heads, qp, 0, kp, ks,
                                   v.data_ptr(), 0, op, os_, None)

    freq = torch.ones(40, device="cuda")
    refused(append(kind=14), "type")
    refused(append(kp=None), "null")
    refused(append(op=None), "together")
    refused(append(heads=0), "heads")
    refused(append(ks=64), "smaller")
    refused(append(op=q.data_ptr(), os_=1024), "in-place")
    refused(append(rope=kib.Rope(freq)), "pairs")
    refused(append(rope=kib.Rope(freq[:8], sections=(1000, 0, 0, 0))), "sections")
    ids = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = torch.empty(1, 2, 16, 64, device="cuda")
    refused(lib.kib_kvq8_read_pages(ctx.h, c.cache.c, ids.data_ptr(), 1, 7, x.data_ptr(), x.data_ptr(), None), "type")
    refused(lib.kib_kvq8_read_pages(ctx.h, c.cache.c, None, 1, 0, x.data_ptr(), x.data_ptr(), None), "null")
    refused(lib.kib_kvq8_read_pages(ctx.h, c.cache.c, ids.data_ptr(), 1, 0, x.data_ptr() + 4, x.data_ptr(), None), "16")
    # nothing to do is not an error
    empty = kib.KvQ8Batch(torch.zeros(0, 1, dtype=torch.int32, device="cuda"), ids[:0], ids, 0, 0)
    ctx.kvq8_append(c.cache, empty, k[:0], v[:0])
    ctx.kvq8_attention(c.cache, empty, q[:0], out[:0], 0.1)
    ctx.kvq8_read_pages(c.cache, ids[:0], x[:0], x[:0])


def test_wrapper_checks_shapes_and_types():
    z = lambda *s, t=torch.int8: torch.zeros(*s, dtype=t)  # noqa: E731
    s = z(4, 2, t=torch.float32)
    kib.KvQ8Cache(z(4, 2, 16, 64), z(4, 2, 16, 64), s, s)
    for bad in ((z(4, 2, 16, 64), z(4, 2, 16, 128), s, s), (z(4, 2, 16, 64, t=torch.uint8), z(4, 2, 16, 64), s, s),
                (z(4, 2, 64, 16).transpose(2, 3), z(4, 2, 64, 16).transpose(2, 3), s, s),
                (z(4, 2, 16, 64), z(4, 2, 16, 64), s[:3], s), (z(4, 2, 16, 64), z(4, 2, 16, 64), s, s.double())):
        with pytest.raises(ValueError):
            kib.KvQ8Cache(*bad)
    i = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
    kib.KvQ8Batch(i(3, 5), i(3), i(4), 7, 3)
    for bad in ((i(2, 5), i(3), i(4)), (i(3, 5).float(), i(3), i(4)), (i(3, 5), i(3), i(3)), (i(3, 10)[:, ::2], i(3), i(4)),
                (i(3, 10)[:, :5], i(3), i(4))):
        with pytest.raises(ValueError):
            kib.KvQ8Batch(*bad, 7, 3)
    with pytest.raises(TypeError):
        kib._row_type(torch.zeros(2, 3, 64, dtype=torch.float64))
    with pytest.raises(ValueError):
        kib._row_type(torch.zeros(2, 3, 128)[:, :, ::2])
    assert kib._row_type(torch.zeros(5, 10, 64)[:, 2:6]) == (kib.TYPE_F32, 640)


@gpu
@pytest.mark.parametrize("dtype,hd,heads,kv", [("f32", 256, 8, 2), ("f16", 256, 8, 2), ("f16", 64, 6, 6), ("f32", 128, 16, 1)])
@pytest.mark.parametrize("length,rows", [(900, 900), (700, 129), (65, 65), (128, 64), (129, 1)])
def test_attention_one_sequence(ctx, dtype, hd, heads, kv, length, rows):
    # a prompt, a late chunk, row tiles that end with one row, a single row with many heads on one
    check_attend(ctx, Case([length], [rows], heads, kv, hd, 32, dtype, seed=length + rows + hd))


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows", [[1, 7, 8, 9, 2, 3], [15, 16, 17, 1, 2], [63, 64, 65, 1]])
def test_attention_where_sequences_change_sides(ctx, dtype, rows):
    """Rows times heads around the multiples of eight that a unit takes and
    around the bound between the two kernels, in one batch."""
    lengths = [n + 37 * i for i, n in enumerate(rows)]
    for heads, kv, hd in ((8, 1, 64), (4, 1, 128), (3, 3, 256)):
        check_attend(ctx, Case(lengths, rows, heads, kv, hd, 16, dtype, seed=rows[0] + hd))


@gpu
@pytest.mark.parametrize("rows", [1, 5, 40])
def test_attention_long_absent_stretches(ctx, rows):
    # 130 of a sequence's pages in a row absent: at its start, in its middle, up to its end
    c = Case([2500, 2500, 2500, 300], [rows] * 4, 4, 2, 64, 16, seed=31)
    c.table[0, :130] = -1
    c.table[1, 15:145] = 1 << 30
    c.table[2, 26:] = -5
    c.batch.tensors[0].copy_(torch.from_numpy(c.table))
    check_attend(ctx, c)


@gpu
@pytest.mark.parametrize("rows", [[1], [1, 3], [1, 40]])
def test_attention_many_sequences(ctx, rows):
    n = 700
    new = [rows[i % len(rows)] if i % 5 else 0 for i in range(n)]
    lengths = [max(x, (i * 37) % 90) for i, x in enumerate(new)]
    check_attend(ctx, Case(lengths, new, 4, 2, 64, 16, seed=len(rows) + rows[-1]))


@gpu
@pytest.mark.parametrize("rows", [1, 70])
def test_a_cache_whose_offsets_pass_32_bits(ctx, rows):
    """Pages 2^30 bytes apart: the last of nine lies 8 GB behind the first."""
    c = Case([100, 80], [rows, rows], 8, 2, 128, 32, seed=33)
    hold, dev = [], []
    for x in c.codes:
        big = torch.empty((c.pages - 1 << 30) + x[0].size, dtype=torch.int8, device="cuda")
        view = torch.as_strided(big, x.shape, (1 << 30, x.shape[2] * x.shape[3], x.shape[3], 1))
        view.copy_(torch.from_numpy(x))
        hold.append(big)
        dev.append(view)
    c.dev[:2] = dev
    c.cache = kib.KvQ8Cache(*c.dev)
    check_attend(ctx, c)
    check_append(ctx, c)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 256), (8, 1, 64), (6, 2, 128)])
def test_attention_short_sequences_beside_long_ones(ctx, dtype, heads, kv, hd):
    """Enough work that long runs go to the tensor-core path, with sequences
    of every short kind in the same batch."""
    new = [500, 1, 65, 0, 128, 129, 16, 33, 300]
    lengths = [900, 1, 65, 40, 128, 200, 16, 1000, 300]
    check_attend(ctx, Case(lengths, new, heads, kv, hd, 16, dtype, seed=hd))


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows", [140, 200, 260])
def test_attention_around_the_work_that_one_kernel_takes_alone(ctx, dtype, rows):
    for length in (rows, rows + 250):
        check_attend(ctx, Case([length], [rows], 8, 2, 256, 64, dtype, seed=rows + length))


@gpu
@pytest.mark.parametrize("hd,spread", [(64, 1.0), (128, 2.0), (256, 2.0), (256, 0.0)])
@pytest.mark.parametrize("alike", [False, True])
def test_attention_long_prompts_keep_fp32_accuracy(ctx, hd, spread, alike):
    """A prompt so long that a CTA's runs are up to 48 tiles.  The cut sums of
    the tensor core may lose 4.3e-8 of O at each of 128 steps between two
    roundings, of which 2e-8 is made up for, and 1.5e-6 is left for q's, p's and
    the scores' 22 bits: 4.4e-6 of the result's norm."""
    n, heads, kv, page = 6144, 8, 2, 64
    g = torch.Generator(device="cuda").manual_seed(hd)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    codes = [(rnd(n // page, kv, page, hd) * 34).clamp_(-127, 127).round_().to(torch.int8) for _ in range(2)]
    if alike:
        codes[1].fill_(100)
    scales = [0.012 * torch.exp(0.3 * rnd(n // page, kv)) + 0.012 for _ in range(2)]
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = kib.KvQ8Batch(torch.randperm(n // page, generator=g, device="cuda").to(torch.int32)[None], i32([n]), i32([0, n]), n, n)
    q = rnd(n, heads, hd) * spread
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    ctx.kvq8_attention(kib.KvQ8Cache(*codes, *scales), batch, q, out, hd ** -0.5)
    order = batch.tensors[0][0].long()
    k, v = ((c.double() * s.double()[..., None, None])[order].permute(1, 0, 2, 3).reshape(kv, n, hd) for c, s in zip(codes, scales))
    for rows in (torch.arange(n - 64, n, device="cuda"), torch.arange(3000, 3064, device="cuda")):
        s = torch.einsum("rgxd,gkd->rgxk", q[rows].double().view(64, kv, heads // kv, hd), k) * hd ** -0.5
        s.masked_fill_(torch.arange(n, device="cuda") > rows[:, None, None, None], -torch.inf)
        want = torch.einsum("rgxk,gkd->rgxd", s.softmax(-1), v).reshape(64, heads, hd)
        assert (out[rows] - want).norm() <= 4.4e-6 * want.norm()


@gpu
def test_a_graph_on_the_contexts_workspace_outlives_its_growth():
    """A small call captured on the context's own workspace, then a larger call
    that outgrows it, then the replay."""
    own = kib.Context(0)
    small, large = Case([300, 140], [1, 1], 8, 2, 128, 32, seed=15), Case([900, 700], [900, 300], 8, 2, 128, 32, seed=16)
    q = small.q.cuda()
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()

    def step(stream):
        own.kvq8_attention(small.cache, small.batch, q, out, 0.09, stream=stream)

    g = torch.cuda.CUDAGraph()
    with pytest.raises(ValueError, match="captured"):  # nothing there yet, and no allocation now
        with torch.cuda.graph(g, stream=side):
            step(torch.cuda.current_stream().cuda_stream)
    step(side.cuda_stream)
    torch.cuda.synchronize()
    want, at = out.clone(), own._workspace[0]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step(torch.cuda.current_stream().cuda_stream)
    run_attend(own, large, 0.09)
    assert own._workspace[0] != at and own._kept == [at]  # only then may the graph run
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    del g
    own.close()


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("lengths,rows", [([300, 90], [1, 1]), ([2500, 40], [3, 1]), ([400, 150], [140, 140]), ([3000, 2900], [2000, 900])])
def test_attention_rows_that_are_not_numbers(ctx, dtype, lengths, rows):
    """A query with a NaN, or an infinity (whose scores are infinite of both
    signs), gives NaN, whichever kernel and however many CTAs take the row; its
    neighbours and other heads are as ever."""
    c = Case(lengths, rows, 8, 2, 128, 32, dtype, seed=41)
    bad = {(0, 1): math.nan, (rows[0] - 1, 6): math.inf, (c.rows - 1, 3): -math.inf, (c.rows // 2, 0): math.nan}
    clean = c.q.clone()
    for (row, head), x in bad.items():
        c.q[row, head, 77] = x
    got = run_attend(ctx, c, 0.09)
    c.q = clean
    plain = run_attend(ctx, c, 0.09)
    for row, head in bad:
        assert got[row, head].isnan().all()
        got[row, head] = plain[row, head]
    # a neighbour's reference may move at another tile: 22-bit (half: 11-bit) weights, rounded differently
    step = 2.0 ** -10 if dtype == "f16" else 2.0 ** -18
    assert (got - plain).abs().max() <= step * 127 * max(float(s.max()) for s in c.dev[3:])


@gpu
@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("lengths,rows", [([300, 90], [1, 1]), ([5000, 40], [2, 1]), ([400, 150], [140, 140])])
def test_attention_over_a_page_whose_scale_is_not_a_number(ctx, lengths, rows, which):
    """Every row that sees such a page gives NaN, wherever the page's keys fall
    among the warps and CTAs; sequences without it are as ever."""
    for at in (0, 1, lengths[0] // 32):
        c = Case(lengths, rows, 8, 2, 128, 32, seed=42)
        clean = run_attend(ctx, c, 0.09)
        c.dev[which][c.table[0, at], 1] = math.nan
        got = run_attend(ctx, c, 0.09)
        sees = torch.from_numpy(c.positions(0) >= at * 32).cuda()
        assert got[:rows[0], 4:][sees].isnan().all()
        assert torch.equal(got[rows[0]:], clean[rows[0]:]) and not got[:rows[0], :4].isnan().any()


@gpu
@pytest.mark.parametrize("size", [1e-30, 3e-36, 2e-37, 1e-38, 2e-41, 1e-43, 1e-45])
def test_append_of_tiny_values(ctx, size):
    """Pages whose largest value is so small that the scale is subnormal (its
    reciprocal infinite) or 0.  A scale is then known to half of 2^-149 only, and
    so is every value read back to 127 of those and half a scale; zeros stay 0."""
    c = Case([20], [20], kv=2, heads=1, seed=43)
    c.v = (c.k.double().clamp(-2, 2) / 2 * size).float()
    c.v[::3, :, ::5] = 0.0
    c.v[2, 1, 7] = math.inf
    run_append(ctx, c, pairs=0)
    v = c.v.numpy().astype(np.float64)
    ulp = 2.0 ** -149
    for head in range(2):
        for page, lo, hi in ((c.table[0, 0], 0, 16), (c.table[0, 1], 16, 20)):
            part = v[lo:hi, head]
            big = np.where(np.isfinite(part), np.abs(part), 0).max()
            s = float(c.dev[3][page, head].double())
            assert abs(s - big / 127) <= 1e-6 * big / 127 + ulp / 2
            got = c.dev[1][page, head, :hi - lo].cpu().numpy().astype(np.int64)
            assert (got[part == 0] == 0).all() and (got[np.isinf(part)] == (127 if s > 0 else 0)).all()
            ok = np.isfinite(part)
            assert (np.abs(got * s - part)[ok] <= 0.5 * s * (1 + 1e-4) + (128 * ulp if s < 1e-36 else 0)).all()


@gpu
def test_attention_of_few_rows_with_lengths_that_the_host_did_not_announce(ctx):
    """Wrong lengths on the device read nothing outside the tensors: keys past
    the table's span are none, positions before the first see nothing."""
    c = Case([100, 64, 80, 33], [1, 3, 2, 1], 8, 2, 128, 16, seed=44)
    want = run_attend(ctx, c, 0.1)
    c.lengths_dev[1:].copy_(torch.tensor([1 << 30, -2 ** 31, -7], dtype=torch.int32))
    got = run_attend(ctx, c, 0.1)
    assert torch.equal(got[:1], want[:1]) and not got[4:].any() and got.isfinite().all()
    # a length past the table sees every key of it
    c.lengths_dev[1] = c.width * c.page + 2
    assert torch.equal(got[1:4], run_attend(ctx, c, 0.1)[1:4])


@gpu
def test_attention_of_many_rows_with_lengths_that_the_host_did_not_announce(ctx):
    """300 sequences whose lengths (and their sums, past 32 bits) the workspace
    has no room for, row starts that go back and past the rows: the sequences
    that fit are right, the others read nothing outside the tensors."""
    n, rows = 300, 70
    c = Case([200] + [rows] * (n - 1), [rows] * n, 4, 2, 64, 128, seed=45)
    table = torch.full((n, 1 << 17), -1, dtype=torch.int32, device="cuda")  # spans 2^24 positions
    table[:, :c.width] = torch.from_numpy(c.table).cuda()
    starts = c.start.copy()
    starts[200], starts[250], starts[n] = 100, 1 << 30, 2 ** 31 - 1
    lengths = [200] + [1 << 30] * 149 + [-2 ** 31] * 75 + [1 << 24] * 75
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = kib.KvQ8Batch(table, i32(lengths), i32(starts.tolist()), c.rows, rows, total_length=rows * n + 200)
    q = c.q.cuda()
    out = torch.full_like(q, 77.0)
    torch.cuda.synchronize()
    ctx.kvq8_attention(c.cache, batch, q, out, 0.1)
    torch.cuda.synchronize()
    want, tol = oracle_attend(c, 0.1)
    assert (np.abs(out[:rows].cpu().numpy() - want[:rows]).max(-1) <= tol[:rows]).all()
    assert out.isfinite().all()


@gpu
def test_rows_of_no_sequence_are_nothing_to_do(ctx):
    c = Case([40], [20], seed=46)
    q, none = c.q.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 7.0)
    for rows in (20, 1):
        batch = kib.KvQ8Batch(torch.zeros(0, 3, dtype=torch.int32, device="cuda"), none[:0], none, rows, rows)
        ctx.kvq8_append(c.cache, batch, c.k.cuda()[:rows], c.v.cuda()[:rows])
        ctx.kvq8_attention(c.cache, batch, q[:rows], out[:rows], 0.1)
    assert (out == 7.0).all()


def row_errors(ctx, n, new, hd, kind, alike, dtype="f32"):
    """Errors against 64 bits, relative to the row's norm, of rows over
    long sequences whose scores are exact but for their last rounding: a query
    is a power of two in one dimension, so that a key's weight is the choice of
    its code there.  equal: all weights alike; peak: the fourth key holds over
    0.999 of them; tail: some 0.97."""
    page, kv, heads, S = 64, 2, 8, len(n)
    need = [x // page for x in n]
    pages = sum(need)
    g = torch.Generator(device="cuda").manual_seed(hd + S)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    k = torch.zeros(pages, kv, page, hd, dtype=torch.int8, device="cuda")
    low, high = dict(equal=(0, 0), peak=(-32, -16), tail=(-8, 8))[kind]
    k[..., 5] = torch.randint(low, high + 1, k.shape[:3], generator=g, device="cuda")
    v = (rnd(pages, kv, page, hd) * 34).clamp_(-127, 127).round_().to(torch.int8)
    if alike:
        v.fill_(100)
    first = np.concatenate([[0], np.cumsum(need)])
    if kind != "equal":
        k[first[:-1], :, 3, 5] = 127
    ks = torch.full((pages, kv), 2.0 ** -5, device="cuda")
    vs = 0.012 * torch.exp(0.3 * rnd(pages, kv)) + 0.012
    table = torch.full((S, max(need)), -1, dtype=torch.int32)
    for i in range(S):
        table[i, :need[i]] = torch.arange(first[i], first[i + 1])
    start = np.concatenate([[0], np.cumsum(new)])
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = kib.KvQ8Batch(table.cuda(), i32(n), i32(start.tolist()), int(start[-1]), max(new), max(n), sum(n))
    q = torch.zeros(int(start[-1]), heads, hd, device="cuda")
    q[..., 5] = 32.0
    q = q.to(DT[dtype])
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    ctx.kvq8_attention(kib.KvQ8Cache(k, v, ks, vs), batch, q, out, 0.125)
    errors = []
    for i in range(0, S, max(1, S // 5)):
        val = (v[first[i]:first[i + 1]].double() * vs[first[i]:first[i + 1]].double()[..., None, None]).permute(1, 0, 2, 3).reshape(kv, n[i], hd)
        score = (k[first[i]:first[i + 1]].double()[..., 5] * 0.125).permute(1, 0, 2).reshape(kv, n[i])  # 2^-5 * 32 * 0.125
        for t in sorted({0, new[i] // 3, new[i] // 2, new[i] - 1}):
            end = n[i] - new[i] + t + 1
            p = torch.softmax(score[:, :end], -1)
            want = torch.einsum("gk,gkd->gd", p, val[:, :end]).repeat_interleave(heads // kv, 0)
            if kind == "peak":
                assert p.max(-1).values.min() > 0.999 or end < 4
            errors.append(((out[start[i] + t].double() - want).norm(dim=-1) / want.norm(dim=-1)).max())
    return float(torch.stack(errors).max())


@gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("kind", ["equal", "peak", "tail"])
@pytest.mark.parametrize("alike", [False, True])
def test_attention_of_few_rows_keeps_fp32_accuracy_on_long_runs(ctx, hd, rows, kind, alike):
    """Runs of 29700 keys a CTA.  A tile's sum on the tensor cores loses 2^-23 of
    itself twice at most (2.4e-7); some 80 rounded additions to O in a row
    deviate by sqrt(80) 2^-24 / sqrt(3) (3e-7), the normaliser's by 1e-7, the
    weights' 22 bits and the joins by less: together below 1e-6 of the result."""
    assert row_errors(ctx, [32768] * 64, [rows] * 64, hd, kind, alike) <= 1e-6


@gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n,rows", [(6144, 6144), (32768, 1024)])
@pytest.mark.parametrize("kind", ["equal", "peak", "tail"])
@pytest.mark.parametrize("alike", [False, True])
def test_attention_of_many_rows_keeps_fp32_accuracy_on_long_runs(ctx, hd, n, rows, kind, alike):
    """A prompt, and a chunk after a long context.  The tensor cores cut 16
    products a step at a quarter of the sum's last bit, 2^-22 of it together:
    eight steps of a tile lose 1.9e-6 at most where V are all alike, and random
    signs cancel to a tenth of it.  Up to 110 rounded additions of tiles deviate
    by sqrt(110) 2^-24 / sqrt(3) (4e-7), the weights' 22 bits and the joins by
    less."""
    assert row_errors(ctx, [n], [rows], hd, kind, alike) <= (2.5e-6 if alike else 1e-6)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_batches_go_to_the_kernel_that_is_faster_for_them(ctx, hd, dtype):
    """Told by the workspace, which holds unpacked keys for the many-row path
    only: batches whose times by the two kernels differ by over a fifth."""
    i32 = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")  # noqa: E731

    def unpacks(n, rows, length):
        pages = -(-length // 32)
        cache = kib.KvQ8Cache(*(torch.empty(1, 2, 32, hd, dtype=torch.int8, device="cuda") for _ in range(2)),
                              *(torch.empty(1, 2, device="cuda") for _ in range(2)))
        batch = kib.KvQ8Batch(i32(n, pages), i32(n), i32(n + 1), n * rows, rows, length, n * length)
        q = torch.empty(1, 8, hd, dtype=DT[dtype], device="cuda").expand(1, 8, hd)
        one = kib.KvQ8Batch(i32(n, pages), i32(n), i32(n + 1), n * 16, 16, length, n * length)  # 64 rows a KV head: never
        return ctx.kvq8_attention_workspace(cache, batch, q) > ctx.kvq8_attention_workspace(cache, one, q)

    for few in ((1, 32, 32), (1, 32, 16000), (1, 24, 32000), (1, 100, 100), (1, 40, 4000), (1, 64, 1000)):
        assert not unpacks(*few), few
    for many in ((1, 500, 500), (30, 20, 500), (8, 200, 200), (3, 500, 500), (1, 1024, 32768), (5, 3001, 3001)):
        assert unpacks(*many), many


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 256])
def test_attention_of_many_rows_with_scales_far_apart_and_absent_pages(ctx, dtype, hd):
    c = Case([1500, 700], [1300, 500], 2, 1, hd, 64, seed=47, dtype=dtype)
    r = np.random.default_rng(4)
    c.dev[3].copy_(torch.from_numpy((10.0 ** r.uniform(-6, -1, c.scales[1].shape)).astype(np.float32)))
    c.dev[3][c.table[0, 3]] = 0.0
    c.dev[2][c.table[0, 1]] = 0.0
    c.table[0, 5], c.table[1, 0], c.table[1, 1] = -1, c.pages, 1 << 30
    c.batch.tensors[0].copy_(torch.from_numpy(c.table))
    for scale in (None, 2.0, -0.1, 0.0):
        check_attend(ctx, c, scale)


@gpu
@pytest.mark.parametrize("sequences,n,rows,hd", [(1, 131072, 1024, 128), (2, 131072, 2048, 64), (3, 70000 // 64 * 64, 1500, 256)])
@pytest.mark.parametrize("kind", ["equal", "peak", "tail"])
@pytest.mark.parametrize("alike", [False, True])
def test_attention_of_many_half_rows_over_very_long_runs(ctx, sequences, n, rows, hd, kind, alike):
    """Runs of up to 900 tiles a CTA.  2^-11 each for the weights and the
    result, and 256 tiles of eight steps that lose 2^-22 of the sum at most
    (4.9e-4; a tenth of it where the values' signs are random)."""
    assert row_errors(ctx, [n] * sequences, [rows] * sequences, hd, kind, alike, "f16") <= 2.0 ** -10 + (4.9e-4 if alike else 4.9e-5)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("length,rows", [(700, 2), (1500, 1400)])
def test_attention_where_scores_are_huge(ctx, dtype, hd, length, rows):
    """Scores far beyond 2^24: the largest take all the weight (equals share it).
    They are exact but for their last rounding, being single products."""
    c = Case([length], [rows], 4, 1, hd, 64, dtype, seed=48)
    for x in (c.dev[2], c.dev[3]):
        x.fill_(2.0 ** -5)
    c.q.zero_()
    c.q[..., 3] = torch.tensor([1.0, -0.5, 2.0, -4.0])
    pages = torch.from_numpy(c.table[0][:-(-length // 64)]).long().cuda()
    key, val = (x[pages, 0].reshape(-1, hd)[:length].double() / 32 for x in c.dev[:2])
    masked = torch.arange(length, device="cuda") > torch.arange(length - rows, length, device="cuda")[:, None, None]
    for scale in (1e4, 3e6, 1e7, -2e8, 1e12, 1e30):
        got = run_attend(ctx, c, scale).double()
        score = (c.q.cuda().double()[..., 3, None] * key[:, 3] * scale).masked_fill(masked, -math.inf)
        want = torch.softmax(score, -1) @ val
        # rounding a result and its weights to half, or fp32 rows' 22 bits of a weight
        assert (got - want).abs().max() <= (2.0 ** -10 if dtype == "f16" else 2.0 ** -19) * val.abs().max(), scale


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("length,rows", [(1, 1), (300, 3), (1500, 1500)])
def test_attention_where_every_score_is_far_below_zero(ctx, dtype, length, rows):
    c = Case([length], [rows], 4, 1, 64, 64, dtype, seed=49)
    c.dev[0][..., 3] = -torch.randint(40, 127, c.dev[0].shape[:3], device="cuda").to(torch.int8)
    for x in (c.dev[2], c.dev[3]):
        x.fill_(2.0 ** -5)
    c.q.zero_()
    c.q[..., 3] = 1.0
    pages = torch.from_numpy(c.table[0][:-(-length // 64)]).long().cuda()
    key, val = (x[pages, 0].reshape(-1, 64)[:length].double() / 32 for x in c.dev[:2])
    masked = torch.arange(length, device="cuda") > torch.arange(length - rows, length, device="cuda")[:, None]
    for scale in (1.0, 1e10, 1e31, 1e36):
        got = run_attend(ctx, c, scale).double()
        want = torch.softmax((key[:, 3] * scale).expand(rows, -1).masked_fill(masked, -math.inf), -1) @ val
        assert (got - want[:, None]).abs().max() <= (2.0 ** -10 if dtype == "f16" else 2.0 ** -19) * val.abs().max(), scale

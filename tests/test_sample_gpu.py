"""kib_sample_f32 against the definition in 64 bits.

The kernel's weights are trunc(2^40 exp(..)) of a 32-bit exponential, off by a
few 2^-24 relatively and by 2^-40 absolutely.  So against the 64-bit weights a
token's share of [0, 1) has to hold the uniform number to within MARGIN = 1e-5
(16 to 100 times that error), with the cuts at top_p and min_p or MARGIN to
either side of them.  Where the weights are exact (equal logits), so is the comparison; and the
tokens equal those of the same integers summed by torch."""
import math

import numpy as np
import pytest
import torch

import kib

MARGIN = 1e-5


def oracle(x, t=1.0, k=0, p=1.0, m=0.0):
    """The possible weights of the kept, in index order; empty where nothing is left."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if x.max() == -np.inf:
        return []
    if t <= 1e-6:
        w = np.zeros(len(x))
        w[np.argmax(x)] = 1
        return [w]
    order = np.lexsort((np.arange(len(x)), -x))
    with np.errstate(invalid="ignore"):
        e = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / t))
    e[x == -np.inf] = 0
    first = (np.arange(len(x)) < k) if k > 0 else np.ones(len(x), bool)
    es = np.where(first, e[order], 0)
    before = np.cumsum(es) - es
    found = []
    for dp in (0, -MARGIN, MARGIN) if p < 1 else (0,):
        for dm in (0, -MARGIN, MARGIN) if m > 0 else (0,):
            keep = first & (es >= min(m, 1.0) * (1 + dm))
            if p < 1:
                keep &= before < (p + dp) * es.sum()
            keep[0] = True
            w = np.zeros(len(x))
            w[order[keep]] = e[order[keep]]
            found.append(w / w.sum())
    return found


def sample(ctx, x, u, t=None, k=None, p=None, m=None, stream=None, stride=0):
    rows, vocab = x.shape
    f = lambda a, d=np.float32: None if a is None else torch.from_numpy(np.asarray(a, d)).cuda()  # noqa: E731
    if stride:
        wide = torch.full((rows, stride), 99.0, device="cuda")
        wide[:, :vocab] = torch.from_numpy(x).cuda()
        dev = wide[:, :vocab]
    else:
        dev = torch.from_numpy(x).cuda()
    tok = torch.full((rows,), -5, dtype=torch.int32, device="cuda")
    prob = torch.full((rows,), -5.0, device="cuda")
    args = (f(t), f(k, np.int32), f(p), f(m))
    u = f(u)
    torch.cuda.synchronize()
    ctx.sample(dev, u, tok, prob, *args, stream=stream)
    torch.cuda.synchronize()
    return tok.cpu().numpy(), prob.cpu().numpy()


def check(ctx, x, u, t=None, k=None, p=None, m=None, **kw):
    tok, prob = sample(ctx, x, u, t, k, p, m, **kw)
    at = lambda a, i, d: d if a is None else float(np.float32(a[i]))  # noqa: E731

    def fits(w, n, q, u):
        run = np.cumsum(w)
        return run[n] - w[n] - MARGIN <= u <= run[n] + MARGIN and abs(q - w[n]) <= 2 * MARGIN * max(w[n], MARGIN)

    for i in range(len(x)):
        found = oracle(x[i], at(t, i, 1.0), int(at(k, i, 0)), at(p, i, 1.0), at(m, i, 0.0))
        if not found:
            assert tok[i] == -1 and prob[i] == 0
            continue
        assert 0 <= tok[i] < x.shape[1]
        assert any(fits(w, tok[i], prob[i], np.float32(u[i])) for w in found), (i, tok[i])
    return tok


def by_torch(x, u, t, k, p, m):
    """The tokens of the definition's integers, summed and compared by torch."""
    x = torch.from_numpy(x).cuda() + 0.0
    f = lambda a, d=torch.float32: torch.as_tensor(np.asarray(a)).to(d).cuda()[:, None]  # noqa: E731
    t, k, p, m, u = f(t), f(k, torch.int64), f(p), f(m), f(u)
    e = torch.exp((x - x.amax(-1, keepdim=True)) * (1.0 / t))
    w = (e * 2.0 ** 40).to(torch.int64)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    rank = torch.arange(x.shape[1], device="cuda")[None]
    keep = (rank < k) | (k <= 0)
    ws = torch.where(keep, w.gather(1, order), 0)
    run = ws.cumsum(-1)
    keep &= (run - ws < (run[:, -1:].double() * p.double()).to(torch.int64)) | (p >= 1)
    keep &= e.gather(1, order) >= m
    keep |= rank == 0
    w = torch.where(torch.zeros_like(keep).scatter(1, order, keep), w, 0)
    run = w.cumsum(-1)
    aim = torch.minimum((run[:, -1:].double() * u.double()).to(torch.int64), run[:, -1:] - 1)
    return (run <= aim).sum(-1).cpu().numpy()


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 33, 1000, 4097, 65536, 248320])
@pytest.mark.parametrize("spread", [0.01, 3.0])
def test_sample_equals_the_integer_definition(ctx, vocab, spread):
    r = np.random.default_rng(vocab)
    x = (r.standard_normal((40, vocab)) * spread).astype(np.float32)
    pick = lambda *a: r.choice(np.float32(a), 40)  # noqa: E731
    for args in (dict(t=pick(0.4, 1, 1.7), k=pick(0, 1, 3, 50, 2000, 30000), p=pick(0.01, 0.6, 0.9, 0.999, 1), m=pick(0, 0, 0.05, 0.3)),
                 dict(t=pick(1), k=pick(0), p=pick(1), m=pick(0)), dict(t=pick(1), k=pick(0), p=pick(0.5, 0.95), m=pick(0))):
        u = r.random(40).astype(np.float32)
        assert np.array_equal(sample(ctx, x, u, **args)[0], by_torch(x, u, **args))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 2, 31, 257, 1000, 4097, 50001, 248320])
def test_sample_random_settings(ctx, vocab):
    r = np.random.default_rng(vocab)
    rows = 24 if vocab > 100000 else 60
    x = (r.standard_normal((rows, vocab)) * 2.5).astype(np.float32)
    hot = r.integers(0, vocab, (rows, min(vocab, 12)))
    np.put_along_axis(x, hot, r.uniform(5, 12, hot.shape).astype(np.float32), 1)
    pick = lambda *a: r.choice(a, rows)  # noqa: E731
    check(ctx, x, r.random(rows).astype(np.float32), pick(0.0, 0.3, 0.7, 1.0, 2.0), pick(0, 1, 5, 40, 100000),
          pick(0.0, 0.3, 0.9, 0.95, 1.0), pick(0.0, 0.02, 0.2, 1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,rows,stride", [(300001, 9, 0), (262145, 3, 262150), (262144, 75, 0), (40000, 400, 0), (99999, 150, 100003)])
def test_sample_long_rows_and_large_batches(ctx, vocab, rows, stride):
    """Long rows, odd strides, and more rows than SMs."""
    r = np.random.default_rng(vocab)
    x = (r.standard_normal((rows, vocab)) * 3).astype(np.float32)
    x[0] = 1.25                      # all equal
    x[1, ::3] = -np.inf
    x[2, 5] = np.nan
    pick = lambda *a: r.choice(np.float32(a), rows)  # noqa: E731
    u = r.random(rows).astype(np.float32)
    for args in (dict(t=pick(0.5, 1, 1.7), k=pick(0, 1, 50, 20000), p=pick(0.01, 0.9, 0.99, 1), m=pick(0, 0.05)),
                 dict(t=pick(1), k=pick(0), p=pick(1), m=pick(0))):
        clean = np.where(np.isnan(x), -np.inf, x).astype(np.float32)
        assert np.array_equal(sample(ctx, x, u, **args, stride=stride)[0], by_torch(clean, u, **args))
    tok, prob = sample(ctx, x, u, t=np.zeros(rows), stride=stride)
    assert np.array_equal(tok, np.nanargmax(x, 1)) and (prob == 1).all()
    dead = np.full((rows, vocab), -np.inf, np.float32)
    assert (sample(ctx, dead, u)[0] == -1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [270000])
def test_sample_long_rows_of_equals(ctx, vocab):
    r = np.random.default_rng(8)
    x = r.choice(np.array([-1.0, -0.0, 0.0, 0.5], np.float32), (6, vocab))
    # logits that differ and round to one weight: the order is theirs, then the index's
    x[5] = np.nextafter(np.float32(1e-3), np.float32(1), dtype=np.float32) * r.choice(np.float32([1, 1 - 2.0 ** -23, 1 - 2.0 ** -22]), vocab)
    u, one, none = r.random(6).astype(np.float32), np.ones(6), np.zeros(6)
    for k, p in ((r.integers(1, vocab, 6), one), (none, r.uniform(0.05, 0.99, 6)), (r.integers(1, vocab, 6), r.uniform(0.05, 0.99, 6))):
        assert np.array_equal(sample(ctx, x, u, one, k, p, none)[0], by_torch(x, u, one, k, p, none))
        assert np.array_equal(sample(ctx, x[:, :9000].copy(), u, one, k % 9000 + 1, p, none)[0],
                              by_torch(x[:, :9000].copy(), u, one, k % 9000 + 1, p, none))


@pytest.mark.gpu
@pytest.mark.parametrize("stride", [0, 1003, 1024])
def test_sample_defaults_and_strides(ctx, stride):
    r = np.random.default_rng(2)
    x = r.standard_normal((50, 1001)).astype(np.float32)
    u = r.random(50).astype(np.float32)
    check(ctx, x, u, stride=stride)
    for one in (dict(t=r.uniform(0.2, 3, 50)), dict(k=r.integers(1, 50, 50)), dict(p=r.uniform(0.1, 0.99, 50)),
                dict(m=r.uniform(0.01, 0.9, 50))):
        check(ctx, x, u, stride=stride, **one)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [64, 70000])
def test_sample_ties_go_to_the_lowest_index(ctx, vocab):
    # few distinct values (-0 and 0 among them): every cut falls inside a group of equals
    r = np.random.default_rng(3)
    x = r.choice(np.array([-1.0, -0.0, 0.0, 0.5], np.float32), (60, vocab))
    u = r.random(60).astype(np.float32)
    one, none = np.ones(60), np.zeros(60)
    for k, p, m in ((r.integers(1, vocab, 60), one, none), (none, r.uniform(0.05, 0.99, 60), none),
                    (r.integers(1, vocab, 60), r.uniform(0.05, 0.99, 60), r.choice([0.0, 0.7], 60))):
        tok = check(ctx, x, u, one, k, p, m)
        assert np.array_equal(tok, by_torch(x, u, one, k, p, m))
    same = np.zeros((4, vocab), np.float32)
    assert list(sample(ctx, same, np.float32([0, 0.5, 0.999, 0]), t=[0, 1, 1, 1], k=[0, 1, 2, 3])[0]) == [0, 0, 1, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [5, 1000, 150001])
def test_sample_equal_logits_exactly(ctx, vocab):
    """All weights equal: the token is the floor(u * n)-th of the n kept, in whole numbers."""
    r = np.random.default_rng(vocab)
    x = np.where(r.random((40, vocab)) < 0.6, np.float32(1.5), -np.inf).astype(np.float32)
    x[:, -1] = 1.5
    u, k = r.random(40).astype(np.float32), r.integers(0, vocab, 40)
    p = r.uniform(0.05, 1.0, 40).astype(np.float32)
    tok, prob = sample(ctx, x, u, t=[0.9] * 40, k=k, p=p, m=[1.0] * 40)
    for i in range(40):
        at = np.flatnonzero(x[i] > 0)
        n = min(len(at), int(k[i])) if k[i] > 0 else len(at)
        limit = int(float(n << 40) * float(p[i])) if p[i] < 1 else n << 40
        n = max(1, -(-limit >> 40))
        assert tok[i] == at[min(int(float(n << 40) * float(u[i])) >> 40, n - 1)]
        assert prob[i] == np.float32(1.0 / n)


@pytest.mark.gpu
def test_sample_uniform_at_its_ends(ctx):
    x = np.log(np.array([[1, 2, 3, 4]] * 6, np.float32))
    u = np.float32([0.0, 0.0999, 0.1001, 0.5999, 0.6001, 0.99999994])
    assert list(sample(ctx, x, u)[0]) == [0, 0, 1, 2, 3, 3]
    # out of range numbers stay inside the row
    assert list(sample(ctx, x[:3], np.float32([-1.0, 1.0, math.nan]))[0]) == [0, 3, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [7, 300, 100001])
def test_sample_banned_and_broken_rows(ctx, vocab):
    r = np.random.default_rng(4)
    x = r.standard_normal((8, vocab)).astype(np.float32)
    x[0] = -np.inf                     # nothing left
    x[1] = np.nan
    x[2, :-1] = -np.inf                # one left
    x[3, ::2] = np.nan                 # half unusable
    x[4, 3] = np.inf                   # all weight on one
    x[5, 2] = x[5, 5] = np.inf         # on two
    x[6] = -3.4e38
    x[6, 4] = 3.4e38
    x[7] = np.finfo(np.float32).min
    u = r.random(8).astype(np.float32)
    u[5] = 0.75
    for t in (0.0, 1.0, 1e-5, 1e30, np.inf):
        tok, prob = sample(ctx, x, u, t=[t] * 8, p=[0.9999] * 8, k=[vocab] * 8)
        assert list(tok[:3]) == [-1, -1, vocab - 1] and list(prob[:3]) == [0, 0, 1]
        assert np.isfinite(x[3, tok[3]]) and tok[4] == 3 and tok[5] == (2 if t == 0 else 5)
        assert tok[6] == 4 or t >= 1e30
        assert 0 <= tok[7] < vocab
        for i, q in enumerate(prob):
            assert 0 <= q <= 1
    check(ctx, x[3:4], u[3:4])
    check(ctx, x[7:], u[7:])


@pytest.mark.gpu
def test_sample_probabilities_follow_the_weights(ctx):
    """Many uniform numbers over one row: the counts are the rounded shares."""
    n = 4096
    w = np.array([0.5, 0.25, 0.125, 0.125])
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    tok, prob = sample(ctx, np.tile(np.log(w).astype(np.float32), (n, 1)), u)
    assert list(np.bincount(tok, minlength=4)) == [2048, 1024, 512, 512]
    assert np.allclose(prob, w[tok], rtol=1e-6)


@pytest.mark.gpu
def test_sample_same_every_time_other_streams_and_graphs(ctx):
    r = np.random.default_rng(5)
    x = (r.standard_normal((40, 30000)) * 2).astype(np.float32)
    u, p, k = r.random(40).astype(np.float32), r.uniform(0.5, 1, 40), r.integers(0, 500, 40)
    a = sample(ctx, x, u, p=p, k=k)
    side = torch.cuda.Stream()
    for s in (None, 0, side.cuda_stream):
        b = sample(ctx, x, u, p=p, k=k, stream=s)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    dev, ud = torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda()
    tok = torch.zeros(40, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ctx.sample(dev, ud, tok, stream=side.cuda_stream)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        ctx.sample(dev, ud, tok, stream=torch.cuda.current_stream().cuda_stream)
    dev.neg_()
    tok.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert np.array_equal(tok.cpu().numpy(), sample(ctx, -x, u)[0])


@pytest.mark.gpu
def test_sample_refusals(ctx):
    x = torch.zeros(2, 8, device="cuda")
    u = torch.zeros(2, device="cuda")
    tok = torch.zeros(2, dtype=torch.int32, device="cuda")

    def call(lp=x.data_ptr(), rows=2, vocab=8, stride=0, up=u.data_ptr(), tp=tok.data_ptr()):
        return ctx.lib.kib_sample_f32(ctx.h, lp, rows, vocab, stride, up, None, None, None, None, tp, None, None)

    assert call() == kib.KIB_OK
    for kw, word in ((dict(vocab=0), "vocab"), (dict(vocab=(1 << 23) + 1), "vocab"), (dict(stride=7), "stride"),
                     (dict(lp=None), "null"), (dict(up=None), "null"), (dict(tp=None), "null"), (dict(rows=1 << 40), "rows")):
        assert call(**kw) == kib.KIB_ERR_INVALID_ARGUMENT
        assert word in ctx.lib.kib_last_error(ctx.h).decode()
    assert call(rows=0, lp=None) == kib.KIB_OK
    for bad in (dict(temperature=u.double()), dict(top_k=u), dict(top_p=u[:1])):
        with pytest.raises(ValueError):
            ctx.sample(x, u, tok, **bad)
    with pytest.raises(ValueError):
        ctx.sample(x[:, ::2], u, tok)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 5, 18, 37, 74, 75])
@pytest.mark.parametrize("vocab", [40003, 8192])
def test_sample_every_split_of_a_row(ctx, rows, vocab):
    """Row counts that give a row 16, 8, 4, 2 and 1 CTAs; top-k around the
    number of a CTA's threads and of the tokens that are left."""
    r = np.random.default_rng(rows + vocab)
    x = (r.standard_normal((rows, vocab)) * 3).astype(np.float32)
    x[rows // 2, r.random(vocab) < 0.95] = -np.inf
    x[rows // 3] = np.round(x[rows // 3])  # groups of equals
    pick = lambda *a: r.choice(np.float32(a), rows)  # noqa: E731
    for k in (1, 7, 1023, 1024, 1025, 5000, vocab - 1, vocab):
        u = r.random(rows).astype(np.float32)
        args = dict(t=pick(0.7, 1, 1.3), k=np.full(rows, k, np.float32), p=pick(0.3, 0.9, 1), m=pick(0, 0.02))
        assert np.array_equal(sample(ctx, x, u, **args)[0], by_torch(x, u, **args))


@pytest.mark.gpu
def test_sample_where_no_logit_stands_out(ctx):
    """Weights that fill one bin, or spread over every value of it."""
    r = np.random.default_rng(21)
    x = (1.0 + r.random((4, 100000)) * np.float32([[0.0], [1e-6], [1e-3], [0.02]])).astype(np.float32)
    for k, p in ((0, 0.37), (700, 0.9), (30000, 1.0), (30000, 0.61)):
        u = r.random(4).astype(np.float32)
        args = dict(t=np.ones(4), k=np.full(4, k), p=np.full(4, p), m=np.zeros(4))
        assert np.array_equal(sample(ctx, x, u, **args)[0], by_torch(x, u, **args))

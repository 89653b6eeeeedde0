"""What the Python calls of the paged 8-bit cache and of sampling hand to the
C entries: nothing is launched here, a stand-in takes the entries' place."""
import pytest
import torch

import kib


class Entries:
    """Stands in for the C library: notes the calls, and answers that all is well."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append((name, args))
            return kib.KIB_OK
        return entry


@pytest.fixture
def ctx():
    c = kib.Context.__new__(kib.Context)
    c.lib, c.h, c.device, c._workspace, c.children = Entries(), None, -1, (None, 0), ()  # -1: tensors in host memory
    return c


ROWS, KV, HD, PAGE = 6, 2, 64, 16
i32 = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
codes = lambda: torch.zeros(4, KV, PAGE, HD, dtype=torch.int8)  # noqa: E731


def cache(k=None, v=None):
    return kib.KvQ8Cache(codes() if k is None else k, codes() if v is None else v, torch.zeros(4, KV), torch.zeros(4, KV))


def batch():
    return kib.KvQ8Batch(i32(2, 3), i32(2), i32(3), ROWS, 3)


def test_expanded_tensors_are_not_taken_for_packed_ones(ctx):
    """A stride of 0 means "packed" to the C entries, which would read (and
    write) past the one row that an expanded tensor has."""
    row = lambda heads: torch.zeros(1, heads, HD).expand(ROWS, heads, HD)  # noqa: E731
    full = lambda heads: torch.zeros(ROWS, heads, HD)  # noqa: E731
    for args, kw in (((row(KV), full(KV)), {}), ((full(KV), row(KV)), {}), ((full(KV), full(KV)), dict(q=row(4), q_out=full(4))),
                     ((full(KV), full(KV)), dict(q=full(4), q_out=row(4)))):
        with pytest.raises(ValueError, match="overlap"):
            ctx.kvq8_append(cache(), batch(), *args, **kw)
    for q, out in ((row(4), full(4)), (full(4), row(4))):
        with pytest.raises(ValueError, match="overlap"):
            ctx.kvq8_attention(cache(), batch(), q, out, 0.1, workspace=torch.zeros(1024, dtype=torch.uint8))
    with pytest.raises(ValueError, match="overlap"):
        ctx.sample(torch.zeros(1, 100).expand(ROWS, 100), torch.zeros(ROWS), i32(ROWS))
    for k in (torch.zeros(HD, dtype=torch.int8).expand(4, KV, PAGE, HD), codes()[:1].expand(4, KV, PAGE, HD),
              codes()[:, :, :1].expand(4, KV, PAGE, HD)):
        with pytest.raises(ValueError, match="overlap"):
            cache(k, k)
    assert not ctx.lib.calls
    # rows apart, and one row whose stride says nothing, are fine
    ctx.sample(torch.zeros(ROWS, 120)[:, :100], torch.zeros(ROWS), i32(ROWS))
    ctx.sample(torch.zeros(1, 100).expand(1, 100), torch.zeros(1), i32(1))
    assert [c[1][4] for c in ctx.lib.calls] == [120, 0]


def test_tensors_on_another_device_are_refused(ctx):
    """A kernel would fault on a host tensor's address."""
    full = lambda heads: torch.zeros(ROWS, heads, HD)  # noqa: E731
    ctx.device = 0
    rope = kib.Rope(torch.ones(8))
    for call in (lambda: ctx.kvq8_append(cache(), batch(), full(KV), full(KV), rope=rope),
                 lambda: ctx.kvq8_attention(cache(), batch(), full(4), full(4), 0.1),
                 lambda: ctx.kvq8_attention(cache(), batch(), full(4), full(4), 0.1, workspace=torch.zeros(4096, dtype=torch.uint8)),
                 lambda: ctx.kvq8_read_pages(cache(), i32(1), torch.zeros(1, KV, PAGE, HD), torch.zeros(1, KV, PAGE, HD)),
                 lambda: ctx.sample(torch.zeros(ROWS, 100), torch.zeros(ROWS), i32(ROWS))):
        with pytest.raises(ValueError, match="device"):
            call()
    assert not ctx.lib.calls

    class Elsewhere(torch.Tensor):
        def get_device(self):
            return 1

    with pytest.raises(ValueError, match="device"):
        kib.KvQ8Cache(codes(), codes(), torch.zeros(4, KV), torch.zeros(4, KV).as_subclass(Elsewhere))

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
    c.lib, c.h, c.device, c._workspace, c._kept, c.children = Entries(), None, -1, (None, 0), [], ()  # -1: tensors in host memory
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


class Memory(Entries):
    """The entries that the context's own workspace needs, with buffers that are only numbers."""

    def __init__(self):
        super().__init__()
        self.need, self.live, self.made, self.used, self.captured, self.capturing = 0, set(), 0, [], set(), False

    def kib_kvq8_attention_workspace(self, h, cache, batch, kind, heads, need):
        need._obj.value = self.need
        return kib.KIB_OK

    def kib_make_buffer(self, h, size, out):
        assert not self.capturing
        self.made += 1
        out._obj.value = 4096 * self.made
        self.live.add(out._obj.value)
        return kib.KIB_OK

    def kib_free_buffer(self, h, where):
        assert not self.capturing
        self.live.remove(where)
        return kib.KIB_OK

    def kib_kvq8_attention_captured(self, h, where, stream, captured, capturing):
        captured._obj.value, capturing._obj.value = where in self.captured, self.capturing
        return kib.KIB_OK

    def kib_kvq8_attention(self, *args):
        where = args[10]
        assert where in self.live
        self.used.append(where)
        if self.capturing:
            self.captured.add(where)
        return kib.KIB_OK

    def kib_destroy(self, h):
        pass


def test_a_workspace_that_a_graph_replays_on_is_not_freed(ctx):
    """The context's own workspace: outgrown, it goes, but not while a captured
    call's graph holds its address; and nothing is allocated during a capture."""
    ctx.lib = m = Memory()
    q = torch.zeros(ROWS, 4, HD)

    def call(need, capturing=False):
        m.need, m.capturing = need, capturing
        try:
            ctx.kvq8_attention(cache(), batch(), q, torch.zeros_like(q), 0.1, stream=7)
        finally:
            m.capturing = False

    call(100)
    call(200)
    assert len(m.live) == 1 and len(m.used) == 2  # outgrown and never captured: freed
    call(150, capturing=True)
    graph = m.used[-1]
    call(1000)
    assert graph in m.live and m.used[-1] != graph  # a replay may still write there
    call(5000)
    assert graph in m.live and len(m.live) == 2
    with pytest.raises(ValueError, match="workspace of 9000 bytes"):
        call(9000, capturing=True)
    call(4000, capturing=True)
    call(9000)
    assert len(m.live) == 3
    ctx.h = 1
    ctx.close()
    assert not m.live

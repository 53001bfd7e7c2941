"""CacheContext.bind_stream without a GPU: which stream waits for which, by stand-ins that
record it.  A context's calls share one workspace, so each has to come after the last."""
import pytest

from xwen_amd import _lib, tree


class Stream:
    def __init__(self, handle, log):
        self.cuda_stream, self.log, self.capturing = handle, log, False

    def wait_stream(self, other):
        assert self.capturing == other.capturing, "an edge between a graph and work outside it"
        self.log.append((self.cuda_stream, other.cuda_stream))


class FakeCuda:
    """torch.cuda as bind_stream uses it."""

    def __init__(self, current):
        self.now = [current]

    def init(self):
        pass

    def current_stream(self, device=None):
        return self.now[-1]

    def is_current_stream_capturing(self):
        return self.now[-1].capturing

    def stream(self, s):
        cuda = self

        class On:
            def __enter__(self):
                cuda.now.append(s)

            def __exit__(self, *exc):
                cuda.now.pop()
        return On()


@pytest.fixture
def bench(monkeypatch):
    log, bound = [], []
    streams = [Stream(h, log) for h in (0, 11, 12, 13)]

    class Torch:
        cuda = FakeCuda(streams[0])

    class Lib:
        @staticmethod
        def xs_cache_create(device, dims, h):
            return _lib.XS_OK

        @staticmethod
        def xs_cache_set_stream(h, s):
            bound.append(s.value or 0)
            return _lib.XS_OK

    monkeypatch.setattr(tree, "_torch", lambda: Torch)
    monkeypatch.setattr(_lib, "load", lambda: Lib)
    ctx = tree.CacheContext(max_seqs=1, max_nodes=1, q_heads=1, kv_heads=1, head_dim=8, capacity=1)

    def call(s):
        with Torch.cuda.stream(s):
            ctx.bind_current_stream()
        assert bound[-1] == s.cuda_stream
    return streams, log, call


def test_calls_outside_a_graph_wait_for_the_last(bench):
    (null, a, b, c), log, call = bench
    for s in (null, null, a, b, b, null):
        call(s)
    assert log == [(11, 0), (12, 11), (0, 12)]


def test_forks_of_one_capture_wait_for_each_other(bench):
    (null, a, b, c), log, call = bench
    call(null)
    a.capturing = b.capturing = True
    call(a)
    assert log == []        # the device has run dry; a graph cannot wait for work outside it
    call(b)
    call(a)
    assert log == [(12, 11), (11, 12)]


def test_a_stream_used_before_and_in_its_capture(bench):
    (null, a, b, c), log, call = bench
    call(a)
    a.capturing = b.capturing = True
    call(a)
    call(b)
    assert log == [(12, 11)]
    a.capturing = b.capturing = False
    call(c)                 # outside again: after a's calls of before
    assert log[1:] == [(13, 11)]


def test_a_graph_ends_and_another_begins(bench):
    (null, a, b, c), log, call = bench
    call(null)
    a.capturing = b.capturing = True
    call(a)
    call(b)
    a.capturing = b.capturing = False
    call(null)
    del log[:]
    a.capturing = True      # b is not in this one
    call(a)
    assert log == []
    c.capturing = True
    call(c)
    assert log == [(13, 11)]


def test_a_call_outside_while_another_stream_captures(bench):
    (null, a, b, c), log, call = bench
    call(c)
    a.capturing = b.capturing = True
    call(a)
    call(null)              # waits for c's calls, not for the graph's
    call(b)                 # in the graph: after a's
    assert log == [(0, 13), (12, 11)]

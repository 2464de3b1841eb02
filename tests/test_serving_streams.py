"""Serving operators and streams: where a call's memory comes from, and how long it is kept.

The host side runs on the CPU with a recorder in place of CUDA's streams and of
the library; the GPU tests run the same situations."""
import contextlib
from types import SimpleNamespace

import pytest
import torch

import serving_ref as ref
import sparse_computation_b200 as sc
from sparse_computation_b200 import serving


class Stream:
    def __init__(self, raw):
        self.cuda_stream, self.device = raw, SimpleNamespace(index=-1)

    def synchronize(self):
        pass


MAIN, SIDE = Stream(1), Stream(2)


@pytest.fixture
def recorder(monkeypatch):
    """Streams without a GPU (CPU tensors are on device -1): ``made`` lists (raw stream, tensor) of what calls
    allocate, ``kept`` (raw stream, data pointer) of record_stream, ``launched`` the raw streams of the C calls."""
    log = SimpleNamespace(now=MAIN, made=[], kept=[], launched=[])

    @contextlib.contextmanager
    def current(stream):
        before, log.now = log.now, stream
        yield
        log.now = before

    new_empty = torch.Tensor.new_empty

    def allocate(self, *shape, **kw):
        t = new_empty(self, *shape, **kw)
        log.made.append((log.now.cuda_stream, t))
        return t

    monkeypatch.setattr(torch.Tensor, "new_empty", allocate)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: log.kept.append((s.cuda_stream, t.data_ptr())),
                        raising=False)
    monkeypatch.setattr(torch.cuda, "stream", current)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: log.now)
    monkeypatch.setattr(serving, "_current", lambda device: log.now.cuda_stream)
    return log


def handle(log, cls, kept=(), **fields):
    """A handle of ``cls`` without the library behind it."""
    h = cls.__new__(cls)
    h.device = -1
    h._call = lambda handle, args, stream: log.launched.append(stream)
    for name, value in fields.items():
        setattr(h, name, value)
    h._kept, h._streams = tuple(kept), {MAIN.cuda_stream}
    return h


def calls(log):
    """name -> (a call with stream=..., its tensors), for each operator; tokens enough for scratch."""
    n, h, d = 300, 2, 8
    x = torch.zeros(n, h, d)
    ints, table = torch.zeros(n, dtype=torch.int32), torch.zeros(n, 1, dtype=torch.int32)
    pools, work, memory = torch.zeros(2, 4, h, 4, d), torch.zeros(64, dtype=torch.uint8), torch.zeros(64, dtype=torch.uint8)
    cache = handle(log, sc.PagedKVCache, pools, k=pools[0], v=pools[1], kv_heads=h, head_dim=d)
    plan = handle(log, sc.DecodeAttention, (work, *pools), cache=cache, q_heads=h, max_seqs=n, _work=work)
    adapters = handle(log, sc.LowRankAdapters, (memory,), in_features=8, out_features=6, _memory=memory)
    adapters._scratch = (n, 128)
    cols = torch.zeros(8, n)
    return {
        "append": (lambda **kw: cache.append(x, x, ints, table, q=x, **kw), [x, ints, table, cache.k, cache.v]),
        "attend": (lambda **kw: plan.attend(x, table, ints, return_lse=True, **kw),
                   [x, table, ints, cache.k, cache.v, plan._work]),
        "apply": (lambda **kw: adapters.apply(cols, ints, **kw), [cols, ints, adapters._memory]),
    }


@pytest.mark.parametrize("name,allocations", [("append", 1), ("attend", 2), ("apply", 2)])
def test_a_call_on_another_stream_allocates_there(recorder, name, allocations):
    """Outputs and scratch of a call with stream= come from that stream's memory, and outputs are kept for the stream
    that was current; its inputs are kept for the stream that reads them."""
    call, given = calls(recorder)[name]
    got = call(stream=SIDE)
    assert recorder.launched == [SIDE.cuda_stream] and recorder.now is MAIN
    assert [raw for raw, _ in recorder.made] == [SIDE.cuda_stream] * allocations
    for t in given:
        assert (SIDE.cuda_stream, t.data_ptr()) in recorder.kept
    for t in got if isinstance(got, tuple) else (got,):
        assert (MAIN.cuda_stream, t.data_ptr()) in recorder.kept


@pytest.mark.parametrize("name", ["append", "attend", "apply"])
def test_a_call_on_the_current_stream_records_nothing(recorder, name):
    call, _ = calls(recorder)[name]
    for kw in ({}, {"stream": MAIN}):
        recorder.launched.clear()
        call(**kw)
        assert recorder.launched == [MAIN.cuda_stream] and not recorder.kept


@pytest.mark.parametrize("name,owned", [("append", slice(3, 5)), ("attend", slice(3, 6)), ("apply", slice(2, 3))])
@pytest.mark.parametrize("explicit", [False, True])
def test_memory_of_a_handle_is_kept_for_every_stream_it_is_used_on(recorder, name, owned, explicit):
    """Under torch.cuda.stream(side) as with stream=side: dropping the handle then gives nothing back that side's
    kernels still use."""
    call, given = calls(recorder)[name]
    if explicit:
        call(stream=SIDE)
    else:
        with torch.cuda.stream(SIDE):
            call()
    for t in given[owned]:
        assert (SIDE.cuda_stream, t.data_ptr()) in recorder.kept
    recorder.kept.clear()
    with torch.cuda.stream(SIDE):
        call()
    assert recorder.launched == [SIDE.cuda_stream] * 2
    assert not recorder.kept  # the allocator remembers a stream until the memory is freed


@pytest.mark.parametrize("name", ["append", "attend", "apply"])
def test_a_stream_of_another_device_is_refused(recorder, name):
    call, _ = calls(recorder)[name]
    other = Stream(3)
    other.device = SimpleNamespace(index=1)
    with pytest.raises(sc.ScError) as e:
        call(stream=other)
    assert e.value.code == sc.SC_ERR_ARG and not recorder.launched


def test_a_plan_made_on_another_stream_than_its_cache(recorder, monkeypatch):
    """The cache's memory is kept for the plan's stream too, although the plan's own workspace comes from there."""
    def size(cache, heads, seqs, out):
        out._obj.value = 64
        return 0

    fake = SimpleNamespace(sc_attn_workspace=size, sc_attn_create_in=lambda *a: 0, sc_attn_free=lambda h: None,
                           sc_attn_decode=lambda h, args, stream: recorder.launched.append(stream))
    monkeypatch.setattr(serving, "lib", lambda: fake)
    pools = torch.zeros(2, 4, 2, 4, 8)
    cache = handle(recorder, sc.PagedKVCache, pools, k=pools[0], v=pools[1], kv_heads=2, head_dim=8)
    cache._h = None
    q, table, lens = torch.zeros(3, 2, 8), torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with torch.cuda.stream(SIDE):
        plan = sc.DecodeAttention(cache, 2, 3)
        plan.attend(q, table, lens)
    assert recorder.launched == [SIDE.cuda_stream]
    for t in pools:
        assert (SIDE.cuda_stream, t.data_ptr()) in recorder.kept


def test_scratch_sizes_of_two_threads_stay_apart(recorder, monkeypatch):
    """Another thread's call with more tokens between any two steps of a size lookup does not change its answer."""
    class Shared(sc.LowRankAdapters):
        stored = (-1, 0)

        @property
        def _scratch(self):
            return self.stored

        @_scratch.setter
        def _scratch(self, pair):
            self.stored = (999, 999 * 8)  # the other thread's, put there right after ours

    def size(h, n, out):
        out._obj.value = n * 8
        return 0

    monkeypatch.setattr(serving, "lib", lambda: SimpleNamespace(sc_adapters_workspace=size))
    s = handle(recorder, Shared)
    s._h = None
    assert [s._workspace(n) for n in (300, 400, 999)] == [300 * 8, 400 * 8, 999 * 8]


# -------------------------------------------------------------------- GPU --

@pytest.mark.gpu
def test_adapters_of_two_streams_do_not_share_scratch(cuda):
    """Batches of different size and order on the current stream and on another one, without a wait between them."""
    gen = torch.Generator().manual_seed(20)
    down = [torch.randn(8, 256, generator=gen) / 16 for _ in range(3)]
    up = [torch.randn(128, 8, generator=gen) / 3 for _ in range(3)]
    s = sc.LowRankAdapters([a.cuda() for a in down], [b.cuda() for b in up], [1.0, 0.5, 2.0])
    batches = []
    for n in (2000, 300):
        x, ids = torch.randn(256, n, generator=gen), torch.randint(-1, 3, (n,), generator=gen).int()
        batches.append((x.cuda(), ids.cuda(), *ref.adapters(x, ids, down, up, [1.0, 0.5, 2.0], None, torch.float32)))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        got.append((s.apply(*batches[0][:2]), s.apply(*batches[1][:2], stream=side)))
    torch.cuda.synchronize()
    s.check()
    for pair in got:
        for y, (_, _, want, tol) in zip(pair, batches):
            assert ((y.cpu().double() - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("explicit", [False, True])
def test_a_dropped_handle_keeps_its_memory_until_its_streams_are_done(cuda, explicit):
    side = torch.cuda.Stream()
    q, table = torch.ones(4, 2, 64, device=cuda), torch.zeros(4, 4, dtype=torch.int32, device=cuda)
    ids, x = torch.zeros(4, dtype=torch.int32, device=cuda), torch.ones(256, 4, device=cuda)
    torch.cuda.synchronize()

    def use(call):
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)  # about 0.1 s
            if not explicit:
                return call()
        return call(stream=side)

    cache = sc.PagedKVCache.allocate(4, 16, 2, 64)

    def plan():
        p = sc.DecodeAttention(cache, 2, 4)
        use(lambda **kw: p.attend(q, table, ids, **kw))
        return p._work

    def adapters():
        s = sc.LowRankAdapters([torch.ones(64, 256, device=cuda)], [torch.ones(1000, 64, device=cuda)], [1.0])
        use(lambda **kw: s.apply(x, ids, **kw))
        return s._memory

    for make in (plan, adapters):
        make()  # loads the kernels
        torch.cuda.synchronize()
        t = make()  # the handle is gone when this returns
        at, n = t.data_ptr(), t.numel()
        del t
        again = torch.empty(n, dtype=torch.uint8, device=cuda)
        assert not side.query()  # or the test shows nothing
        assert not at <= again.data_ptr() < at + n
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_outputs_on_another_stream_take_no_block_of_the_current_one(cuda):
    """A block freed on the current stream, whose last kernel is still ahead, is not what the other stream's output gets."""
    cache = sc.PagedKVCache.allocate(4, 16, 2, 64)
    plan = sc.DecodeAttention(cache, 2, 300)
    s = sc.LowRankAdapters([torch.ones(4, 256, device=cuda)], [torch.ones(128, 4, device=cuda)], [1.0])
    q, table = torch.ones(300, 2, 64, device=cuda), torch.zeros(300, 4, dtype=torch.int32, device=cuda)
    ids, x = torch.zeros(300, dtype=torch.int32, device=cuda), torch.ones(256, 300, device=cuda)
    side = torch.cuda.Stream()
    for call in (lambda: cache.append(q[:4], q[:4], ids[:4] - 1, table, q=q[:4], stream=side),
                 lambda: plan.attend(q, table, ids, stream=side),
                 lambda: s.apply(x, ids, stream=side)):
        size = call().numel()  # and loads the kernels
        torch.cuda.synchronize()
        freed = torch.empty(size, device=cuda)
        torch.cuda._sleep(200_000_000)  # about 0.1 s
        freed.add_(1)
        at = freed.data_ptr()
        del freed
        out = call()
        assert not at <= out.data_ptr() < at + 4 * size
        torch.cuda.synchronize()

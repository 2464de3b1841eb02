"""Entry points and ways of calling the serving operators that the other tests do not take: the C calls that allocate
their own memory, the ones that are given it, graphs of every operator, windows that begin anywhere in a page."""
import ctypes
import math
from struct import pack

import pytest
import torch

import serving_ref as ref
import sparse_computation_b200 as sc

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def arrays(down, up):
    n = len(down)
    i64, vp = ctypes.c_int64 * n, ctypes.c_void_p * n
    return (i64(*[a.shape[0] for a in down]), 0, vp(*[a.data_ptr() for a in down]), i64(*[a.stride(0) for a in down]),
            vp(*[b.data_ptr() for b in up]), i64(*[b.stride(0) for b in up]))


def last_error():
    return sc.lib().sc_last_error_string().decode()


def test_attention_through_the_c_calls(cuda):
    """sc_attn_create, whose workspace is its own, gives the plan that DecodeAttention is; sc_attn_create_in refuses a
    workspace that is short or off a 256-byte boundary, and takes one of just the size."""
    gen, L = torch.Generator().manual_seed(60), sc.lib()
    k, v = (torch.randn(6, 2, 16, 64, generator=gen) for _ in range(2))
    q = torch.randn(3, 4, 64, generator=gen)
    cache = sc.PagedKVCache(k.cuda(), v.cuda())
    table, lens = torch.tensor([[0, 1, 2], [3, 0, 0], [4, 5, 0]], dtype=torch.int32), [40, 0, 32]
    want, lse, tol, ltol = ref.attend(q, k, v, table, lens, 0.125)
    qg, tg, lg = q.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    size, h = ctypes.c_int64(), ctypes.c_void_p()
    assert L.sc_attn_workspace(cache._h, 4, 3, ctypes.byref(size)) == sc.SC_OK and size.value > 0
    block = torch.empty(size.value + 512, dtype=torch.uint8, device=cuda)
    at = (block.data_ptr() + 255) // 256 * 256
    for start, n in ((at, size.value - 1), (at + 16, size.value), (at, 0)):
        assert L.sc_attn_create_in(cache._h, 4, 3, 0.0, 0, start, n, ctypes.byref(h)) == sc.SC_ERR_ARG
        assert "workspace" in last_error() and not h.value
    assert L.sc_attn_create_in(cache._h, 4, 3, 0.0, 0, None, size.value, ctypes.byref(h)) == sc.SC_ERR_ARG
    torch.cuda.synchronize()
    for create in (lambda: L.sc_attn_create(cache._h, 4, 3, 0.0, 0, ctypes.byref(h)),
                   lambda: L.sc_attn_create_in(cache._h, 4, 3, 0.0, 0, at, size.value, ctypes.byref(h))):
        assert create() == sc.SC_OK
        out, s = torch.full_like(qg, 7.0), torch.zeros(3, 4, device=cuda)
        args = pack("15q", 3, 0, qg.data_ptr(), *qg.stride(), out.data_ptr(), *out.stride(), s.data_ptr(), tg.data_ptr(), 3,
                    3, lg.data_ptr())
        assert L.sc_attn_decode(h, args, torch.cuda.current_stream().cuda_stream) == sc.SC_OK
        status = ctypes.c_int32(5)
        assert L.sc_attn_status(h, ctypes.byref(status)) == sc.SC_OK and status.value == 0
        assert ((out.cpu().double() - want).abs() <= tol).all()
        full = lse != -math.inf
        assert ((s.cpu().double() - lse)[full].abs() <= ltol[full]).all() and (s.cpu()[~full] == -math.inf).all()
        L.sc_attn_free(h)


@pytest.mark.parametrize("tokens", [20, 300])
def test_adapters_through_the_c_calls(cuda, tokens):
    gen, L = torch.Generator().manual_seed(61), sc.lib()
    down = [torch.randn(r, 40, generator=gen) for r in (3, 8)]
    up = [torch.randn(24, r, generator=gen) for r in (3, 8)]
    dg, ug = [a.cuda() for a in down], [b.cuda() for b in up]
    ranks, kind, dp, dl, upp, ul = arrays(dg, ug)
    scales = (ctypes.c_float * 2)(1.0, -2.0)
    x, ids = torch.randn(40, tokens, generator=gen), torch.randint(-1, 2, (tokens,), generator=gen).int()
    want, tol = ref.adapters(x, ids, down, up, [1.0, -2.0], None, F32)
    xg, ig = x.cuda(), ids.cuda()
    stream = torch.cuda.current_stream().cuda_stream
    size, h, need = ctypes.c_int64(), ctypes.c_void_p(), ctypes.c_int64()
    assert L.sc_adapters_size(40, 24, 2, ranks, kind, ctypes.byref(size)) == sc.SC_OK and size.value > 0
    block = torch.empty(size.value + 512, dtype=torch.uint8, device=cuda)
    at = (block.data_ptr() + 255) // 256 * 256
    given = lambda start, n: L.sc_adapters_create_in(0, 40, 24, 2, ranks, kind, dp, dl, upp, ul, scales, stream, start, n,
                                                     ctypes.byref(h))
    for start, n in ((at, size.value - 1), (at + 128, size.value), (None, size.value)):
        assert given(start, n) == sc.SC_ERR_ARG and not h.value
    for create in (lambda: L.sc_adapters_create(0, 40, 24, 2, ranks, kind, dp, dl, upp, ul, scales, stream, ctypes.byref(h)),
                   lambda: given(at, size.value)):
        assert create() == sc.SC_OK
        assert L.sc_adapters_workspace(h, tokens, ctypes.byref(need)) == sc.SC_OK
        assert (need.value == 0) == (tokens <= 256)
        work = torch.empty(need.value + 16, dtype=torch.uint8, device=cuda)
        out = torch.zeros(24, tokens, device=cuda)
        args = lambda n: pack("14q", tokens, 0, xg.data_ptr(), *xg.stride(), 0, 0, 0, out.data_ptr(), *out.stride(),
                              ig.data_ptr(), work.data_ptr(), n)
        if need.value:
            assert L.sc_adapters_apply(h, args(need.value - 1), stream) == sc.SC_ERR_ARG and "workspace" in last_error()
        assert L.sc_adapters_apply(h, args(need.value), stream) == sc.SC_OK
        status = ctypes.c_int32(5)
        assert L.sc_adapters_status(h, ctypes.byref(status)) == sc.SC_OK and status.value == 0
        assert ((out.cpu().double() - want).abs() <= tol).all()
        L.sc_adapters_free(h)


# ----------------------------------------------------------------- graphs --

def captured(call):
    """A graph of one call; its kernels have run before."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = call()
    return g, got


@pytest.mark.parametrize("layout", ["tokens", "features", "any"])
def test_append_in_a_graph(cuda, layout):
    """Replays with other rows, positions and sequences."""
    gen = torch.Generator().manual_seed(62)
    cache = sc.PagedKVCache.allocate(8, 4, 2, 64, BF16)
    angle = torch.rand(32, 32, generator=gen) * 6
    rope = sc.RotaryTable(angle.cos().cuda(), angle.sin().cuda())
    table = torch.randperm(8, generator=gen).int().view(2, 4).cuda()
    made = lambda h: torch.zeros(6, h, 64).cuda() if layout == "tokens" else \
        torch.zeros(h * 64, 6).cuda().view(h, 64, 6).permute(2, 0, 1) if layout == "features" else \
        torch.zeros(6, 64, h).cuda().transpose(1, 2)
    k, v, q = made(2), made(2), made(6)
    ids, pos = torch.zeros(6, dtype=torch.int32).cuda(), torch.zeros(6, dtype=torch.int32).cuda() - 1
    g, out = captured(lambda: cache.append(k, v, pos, table, seq_ids=ids, rope=rope, q=q))
    for spread in ([3, 0, 7, 12, 15, 1], [2, 5, 9, 10, 4, 14]):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=gen))
        pos.copy_(torch.tensor(spread))
        ids.copy_(torch.tensor([0, 1, 0, 1, 1, 0]))
        cache.k.zero_(), cache.v.zero_()
        g.replay()
        got, kept = out.clone(), (cache.k.clone(), cache.v.clone())
        cache.k.zero_(), cache.v.zero_()
        assert torch.equal(got, cache.append(k, v, pos, table, seq_ids=ids, rope=rope, q=q))
        assert torch.equal(kept[0], cache.k) and torch.equal(kept[1], cache.v) and kept[0].abs().sum() > 0
    cache.check()


@pytest.mark.parametrize("tokens", [40, 700])
@pytest.mark.parametrize("types", [(F32, F32), (F32, F16), (BF16, BF16)])
def test_adapters_in_a_graph(cuda, tokens, types):
    """Replays with other tokens and adapters; with scratch, a sort and its dependent launch from 257 tokens on."""
    gen = torch.Generator().manual_seed(63)
    down = [torch.randn(r, 200, generator=gen).to(types[1]) / 14 for r in (3, 8, 20)]
    up = [torch.randn(120, r, generator=gen).to(types[1]) / 3 for r in (3, 8, 20)]
    s = sc.LowRankAdapters([a.cuda() for a in down], [b.cuda() for b in up], [1.0, 0.5, 2.0])
    x, base = torch.zeros(200, tokens, dtype=types[0]).cuda(), torch.zeros(120, tokens, dtype=types[0]).cuda()
    ids = torch.zeros(tokens, dtype=torch.int32).cuda()
    g, out = captured(lambda: s.apply(x, ids, base=base))
    for _ in range(3):
        xs, bs = torch.randn(200, tokens, generator=gen).to(types[0]), torch.randn(120, tokens, generator=gen).to(types[0])
        which = torch.randint(-1, 3, (tokens,), generator=gen).int()
        x.copy_(xs), base.copy_(bs), ids.copy_(which)
        g.replay()
        g.replay()  # one after the other: the second sort waits for the first call's tiles
        want, tol = ref.adapters(xs, which, down, up, [1.0, 0.5, 2.0], bs, types[0])
        assert ((out.cpu().double() - want).abs() <= tol).all()
    s.check()


# ---------------------------------------------------------------- windows --

@pytest.mark.parametrize("types", [(F32, F32), (F32, BF16), (F16, F16)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 12, 32])
def test_windows_that_begin_anywhere_in_sixteen_keys(cuda, types, d, page):
    """From the eighth key of sixteen on, a step of eight keys holds none of the window's."""
    gen = torch.Generator().manual_seed(64)
    window = 50
    lens = [window + f for f in (0, 1, 7, 8, 9, 12, 15, 16, 24, 31)]
    need = [-(-n // page) for n in lens]
    table, at = torch.zeros(len(lens), max(need), dtype=torch.int32), 0
    for i, c in enumerate(need):
        table[i, :c] = torch.arange(at, at + c).int()
        at += c
    k, v = (torch.randn(at, 2, page, d, generator=gen).to(types[1]) for _ in range(2))
    q = torch.randn(len(lens), 6, d, generator=gen).to(types[0])
    want, lse, tol, ltol = ref.attend(q, k, v, table, lens, 1 / math.sqrt(d), window)
    for i, n in enumerate(lens):  # what the window leaves out is not looked at
        for j in range(n - window):
            k[table[i, j // page], :, j % page] = math.nan
            v[table[i, j // page], :, j % page] = math.nan
    plan = sc.DecodeAttention(sc.PagedKVCache(k.cuda(), v.cuda()), 6, len(lens), window=window)
    out, s = plan.attend(q.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), return_lse=True)
    plan.check()
    assert ((out.cpu().double() - want).abs() <= tol).all()
    assert ((s.cpu().double() - lse).abs() <= ltol).all()

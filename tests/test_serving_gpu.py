"""Serving operators on the GPU against plain 64-bit restatements
(tests/serving_ref.py, which derives the tolerances): cache append with the
rotary rotation, decode attention over a paged cache, low-rank adapters."""
import math

import pytest
import torch

import serving_ref as ref
import sparse_computation_b200 as sc

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPE_PAIRS = [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (F16, F16), (BF16, F32), (F16, BF16)]


def randn(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype)


def rows(x, layout):
    """The same values on the GPU as a token-major tensor, a view of a feature-major one, or one with padded strides."""
    t, h, d = x.shape
    if layout == "features":
        return x.permute(1, 2, 0).reshape(h * d, t).contiguous().cuda().view(h, d, t).permute(2, 0, 1)
    if layout == "padded":
        wide = torch.zeros(t, h + 1, d + 3, dtype=x.dtype).cuda()
        wide[:, :h, :d] = x.cuda()
        return wide[:, :h, :d]
    return x.cuda()


def pool_of(x, order):
    """[pages, heads, slots, dim] on the GPU, or a permuted view of slot-major pages."""
    return x.cuda() if order == "heads" else x.transpose(1, 2).contiguous().cuda().transpose(1, 2)


def tables(half, n=4096):
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(1, half))
    ang = torch.arange(n, dtype=torch.float64)[:, None] * freq
    return ang.cos().float(), ang.sin().float()


# ----------------------------------------------------------------- append --

APPEND = [
    # types, kv heads, q heads, dim, rotary, interleaved, page, layout, pool order, sequence spans (cached, new)
    (TYPE_PAIRS[0], 8, 8, 64, 64, False, 16, "features", "heads", [(0, 1)]),
    (TYPE_PAIRS[1], 2, 8, 128, 128, False, 16, "features", "slots", [(3, 1), (15, 1), (16, 1), (31, 1)]),
    (TYPE_PAIRS[2], 1, 5, 40, 20, True, 1, "tokens", "heads", [(0, 7), (5, 1), (2, 0), (9, 30)]),
    (TYPE_PAIRS[3], 4, 4, 80, 32, True, 24, "tokens", "heads", [(10, 61), (0, 23), (47, 2)]),
    (TYPE_PAIRS[4], 3, 12, 96, 96, False, 64, "padded", "slots", [(60, 9), (0, 130)]),
    (TYPE_PAIRS[5], 2, 2, 256, 128, False, 7, "features", "heads", [(6, 33)]),
    (TYPE_PAIRS[6], 1, 1, 8, 2, False, 3, "tokens", "heads", [(1, 2), (2, 3)]),
    (TYPE_PAIRS[1], 8, 32, 128, 128, False, 64, "tokens", "heads", [(100, 70), (0, 1), (63, 2)]),
    (TYPE_PAIRS[3], 2, 6, 72, 36, False, 16, "features", "heads", [(0, 19), (4, 130)]),
    (TYPE_PAIRS[4], 2, 4, 64, 0, False, 16, "tokens", "heads", [(3, 20)]),
]


@pytest.mark.parametrize("types,h,hq,d,rotary,pairs,page,layout,order,spans", APPEND)
@pytest.mark.parametrize("with_q", [True, False])
def test_append(cuda, types, h, hq, d, rotary, pairs, page, layout, order, spans, with_q):
    kind, stored = types
    gen = torch.Generator().manual_seed(1)
    need = [-(-(a + n) // page) for a, n in spans]
    pool = sum(need) + 3
    perm = torch.randperm(pool, generator=gen)
    table = torch.full((len(spans), max(need) + 1), -7, dtype=torch.int32)  # unused entries are never read
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = perm[at:at + c].int()
        at += c
    ids = torch.tensor([i for i, (_, n) in enumerate(spans) for _ in range(n)], dtype=torch.int32)
    pos = torch.tensor([p for a, n in spans for p in range(a, a + n)], dtype=torch.int32)
    t = len(pos)
    shuffle = torch.randperm(t, generator=gen)
    ids, pos = ids[shuffle], pos[shuffle]
    if t > 2:
        pos[1] = -1  # a padding token
    k, v, q = (randn(gen, t, n, d, dtype=kind) for n in (h, h, hq))
    k0, v0 = (randn(gen, pool, h, page, d, dtype=stored) for _ in range(2))
    cos, sin = tables(rotary // 2)
    kp, vp = pool_of(k0, order), pool_of(v0, order)
    cache = sc.PagedKVCache(kp, vp)
    rope = sc.RotaryTable(cos.cuda(), sin.cuda(), interleaved=pairs) if rotary else None
    alone = len(set(ids.tolist())) == t and ids.tolist() == list(range(t))
    got = cache.append(rows(k, layout), rows(v, layout), pos.cuda(), table.cuda(),
                       seq_ids=None if alone else ids.cuda(), rope=rope, q=rows(q, layout) if with_q else None)
    cache.check()
    kr, kmag = ref.rotate(k, pos, cos, sin, pairs)
    want_k, want_v, free = k0.clone().double(), v0.clone(), torch.ones(pool, page, dtype=torch.bool)
    tol_k = torch.zeros_like(want_k)
    for i in range(t):
        p = int(pos[i])
        if p < 0:
            continue
        pg, sl = int(table[ids[i], p // page]), p % page
        free[pg, sl] = False
        want_k[pg, :, sl] = kr[i]
        tol_k[pg, :, sl] = 2.0 ** -22 * kmag[i] + ref.rounding(kr[i], stored) + ref.rounding(kr[i], stored) * 2.0 ** -6
        want_v[pg, :, sl] = v[i].float().to(stored)
    assert torch.equal(vp.cpu(), want_v)
    assert ((kp.cpu().double() - want_k).abs() <= tol_k).all()
    assert torch.equal(kp.cpu().transpose(1, 2)[free], k0.transpose(1, 2)[free])
    if with_q:
        qr, qmag = ref.rotate(q, pos, cos, sin, pairs)
        qr[pos < 0] = 0
        tol = (2.0 ** -22 * qmag + ref.rounding(qr, kind) * (1 + 2.0 ** -6)) * (pos >= 0)[:, None, None]
        assert got.dtype == kind and got.shape == q.shape
        assert ((got.cpu().double() - qr).abs() <= tol).all()
    else:
        assert got is None


@pytest.mark.parametrize("layout", ["tokens", "features", "padded"])
def test_append_rotates_q_in_place(cuda, layout):
    gen = torch.Generator().manual_seed(2)
    k, v, q = (randn(gen, 9, n, 64) for n in (2, 2, 6))
    cos, sin = tables(32)
    cache = sc.PagedKVCache.allocate(4, 16, 2, 64)
    pos, table = torch.arange(9, dtype=torch.int32).cuda(), torch.arange(4, dtype=torch.int32).view(1, 4).cuda()
    ids, rope = torch.zeros(9, dtype=torch.int32).cuda(), sc.RotaryTable(cos.cuda(), sin.cuda())
    args = (rows(k, layout), rows(v, layout), pos, table, ids, rope)
    apart = cache.append(*args, q=rows(q, layout))
    mine = rows(q, layout)
    assert cache.append(*args, q=mine, q_out=mine) is mine
    assert torch.equal(mine, apart)


def test_append_out_of_range_places_are_skipped(cuda):
    """A page-table entry outside the pool, a position beyond the table, a
    sequence beyond it, or a position without rotation rows: status, nothing stored."""
    cache = sc.PagedKVCache.allocate(4, 16, 1, 64)
    k = torch.ones(3, 1, 64).cuda()
    rope = sc.RotaryTable(*(x.cuda() for x in tables(32, n=40)))
    table = torch.tensor([[0, 9, 1], [-1, 2, 3]], dtype=torch.int32).cuda()
    def put(pos, seq):
        q = cache.append(k, k, torch.tensor(pos, dtype=torch.int32).cuda(), table,
                         seq_ids=torch.tensor(seq, dtype=torch.int32).cuda(), rope=rope, q=k)
        return q, cache.status(), cache.status()
    for pos, seq, code in (([17, 0, 1], [0, 0, 0], 8), ([48, 0, 1], [0, 0, 0], 8), ([0, 0, 1], [2, 0, 0], 8),
                           ([0, 0, 1], [-1, 0, 0], 8), ([5, 0, 1], [1, 0, 0], 8), ([41, 0, 1], [0, 0, 0], 9),
                           ([2, 0, 1], [0, 0, 0], 0)):
        q, first, second = put(pos, seq)
        assert (first, second) == (code, 0)
        assert (q[0] == 0).all().item() == (code != 0)
        assert not (q[1:] == 0).all()
    cache.k.zero_()
    put([17, 33, 18], [0, 0, 0])
    assert cache.k[[0, 2, 3]].abs().sum() == 0 and cache.k[1].abs().sum() > 0


# ----------------------------------------------------------------- attend --

ATTEND = [
    # types, kv heads, q heads, dim, page, window, layout, pool order, lengths
    (TYPE_PAIRS[0], 8, 8, 64, 16, 0, "features", "heads", [1, 0, 16, 17, 200]),
    (TYPE_PAIRS[0], 2, 10, 128, 16, 0, "tokens", "slots", [31, 32, 33, 700]),
    (TYPE_PAIRS[0], 1, 3, 20, 5, 0, "padded", "heads", [4, 5, 6, 64, 65]),
    (TYPE_PAIRS[0], 2, 2, 256, 16, 40, "features", "heads", [0, 39, 40, 41, 300]),
    (TYPE_PAIRS[1], 2, 8, 128, 64, 0, "features", "heads", [1, 63, 64, 65, 1000]),
    (TYPE_PAIRS[1], 1, 8, 96, 24, 100, "tokens", "heads", [99, 100, 101, 500]),
    (TYPE_PAIRS[1], 1, 16, 64, 16, 0, "tokens", "slots", [77, 300]),
    (TYPE_PAIRS[2], 2, 6, 80, 1, 0, "features", "heads", [1, 2, 15, 90]),
    (TYPE_PAIRS[2], 1, 12, 32, 7, 0, "tokens", "heads", [50, 333]),
    (TYPE_PAIRS[3], 8, 32, 128, 16, 0, "tokens", "heads", [5, 129, 2049]),
    (TYPE_PAIRS[3], 2, 2, 8, 16, 0, "tokens", "heads", [3, 40]),
    (TYPE_PAIRS[3], 1, 40, 192, 48, 0, "padded", "slots", [47, 48, 49, 260]),
    (TYPE_PAIRS[4], 5, 25, 80, 48, 100, "tokens", "heads", [0, 1, 99, 600]),
    (TYPE_PAIRS[4], 4, 4, 256, 128, 0, "features", "heads", [127, 400]),
    (TYPE_PAIRS[5], 2, 4, 64, 16, 0, "tokens", "heads", [90]),
    (TYPE_PAIRS[6], 2, 4, 64, 16, 0, "tokens", "heads", [90, 1]),
]


def scattered(gen, lens, page, pool_extra=3):
    need = [-(-n // page) for n in lens]
    pool = sum(need) + pool_extra
    perm = torch.randperm(pool, generator=gen)
    table = torch.full((len(lens), max(need) + 2), 1 << 30, dtype=torch.int32)  # never read beyond the length
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = perm[at:at + c].int()
        at += c
    return table, pool


def poisoned(x, table, lens, page, first):
    """x with NaN and infinity everywhere that no sequence attends to."""
    keep = torch.zeros(x.shape[0], page, dtype=torch.bool)
    for i, n in enumerate(lens):
        for j in range(first[i], n):
            keep[table[i, j // page], j % page] = True
    y = torch.full_like(x, float("nan"))
    y[:, :, ::2] = float("inf")
    y.transpose(1, 2)[keep] = x.transpose(1, 2)[keep]
    return y


def attend_case(types, h, hq, d, page, window, layout, order, lens, seed=3, sharp=1.0, scale=None):
    kind, stored = types
    gen = torch.Generator().manual_seed(seed)
    table, pool = scattered(gen, lens, page)
    k, v = (randn(gen, pool, h, page, d, dtype=stored) for _ in range(2))
    q = randn(gen, len(lens), hq, d, dtype=kind, scale=sharp)
    first = [max(0, n - window) if window else 0 for n in lens]
    kg = pool_of(poisoned(k, table, lens, page, first), order)
    vg = pool_of(poisoned(v, table, lens, page, first), order)
    plan = sc.DecodeAttention(sc.PagedKVCache(kg, vg), hq, len(lens), scale=scale, window=window)
    want = ref.attend(q, k, v, table, lens, scale or 1 / math.sqrt(d), window)
    return plan, rows(q, layout), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), want


def close(out, lse, want):
    w, wl, tol, ltol = want
    assert ((out.cpu().double() - w).abs() <= tol).all(), ((out.cpu().double() - w).abs() / tol.clamp_min(1e-300)).max()
    lse = lse.cpu().double()
    empty = wl == float("-inf")
    assert torch.equal(lse == float("-inf"), empty)
    assert ((lse - wl)[~empty].abs() <= ltol[~empty]).all()


@pytest.mark.parametrize("types,h,hq,d,page,window,layout,order,lens", ATTEND)
def test_attend(cuda, types, h, hq, d, page, window, layout, order, lens):
    plan, q, table, sl, want = attend_case(types, h, hq, d, page, window, layout, order, lens)
    out, lse = plan.attend(q, table, sl, return_lse=True)
    plan.check()
    assert out.dtype == types[0]
    close(out, lse, want)
    again, lse2 = plan.attend(q, table, sl, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)  # the same bits every time
    fm = rows(torch.zeros(out.shape, dtype=out.dtype), "features")
    assert plan.attend(q, table, sl, out=fm) is fm
    assert torch.equal(fm, out)


@pytest.mark.parametrize("types", TYPE_PAIRS[:5])
@pytest.mark.parametrize("lens", [[20000], [9000, 1, 0, 3000], [5] * 300, [0], [0, 0, 0]])
def test_attend_splits(cuda, types, lens):
    """One long sequence, a ragged batch and many short ones: how the work is cut must not show."""
    plan, q, table, sl, want = attend_case(types, 2, 6, 64, 16, 0, "tokens", "heads", lens)
    for _ in range(3):
        close(*plan.attend(q, table, sl, return_lse=True), want)


@pytest.mark.parametrize("types", TYPE_PAIRS[:5])
@pytest.mark.parametrize("sharp,scale", [(60.0, None), (1e-3, None), (1.0, 3.0), (1.0, 1e-6)])
def test_attend_sharp_and_flat(cuda, types, sharp, scale):
    plan, q, table, sl, want = attend_case(types, 2, 4, 64, 16, 0, "tokens", "heads", [300, 7], sharp=sharp,
                                           scale=scale)
    close(*plan.attend(q, table, sl, return_lse=True), want)


def test_attend_few_of_max_seqs_and_reuse(cuda):
    """A plan of many sequences serves fewer; calls of other sizes follow one another."""
    kind = TYPE_PAIRS[1]
    plan, q, table, sl, want = attend_case(kind, 2, 8, 64, 16, 0, "tokens", "heads", [400, 3000, 0, 17, 64])
    for n in (5, 1, 3, 5):
        out, lse = plan.attend(q[:n], table[:n], sl[:n], return_lse=True)
        close(out, lse, tuple(x[:n] for x in want))


def test_attend_page_entries_out_of_range_are_absent(cuda):
    """Keys on a page outside the pool, or beyond the table, count as absent and set the status."""
    gen = torch.Generator().manual_seed(5)
    k, v, q = randn(gen, 6, 1, 16, 64), randn(gen, 6, 1, 16, 64), randn(gen, 1, 2, 64)
    plan = sc.DecodeAttention(sc.PagedKVCache(k.cuda(), v.cuda()), 2, 1)
    run = lambda t, n: plan.attend(q.cuda(), torch.tensor([t], dtype=torch.int32).cuda(),
                                   torch.tensor([n], dtype=torch.int32).cuda(), return_lse=True)
    full = torch.tensor([[0, 1, 2]])
    close(*run([0, 1, 2], 48), ref.attend(q, k, v, full, [48], 0.125))
    assert plan.status() == 0
    close(*run([0, 1, 2], 60), ref.attend(q, k, v, full, [48], 0.125))  # longer than the table
    assert plan.status() == 8
    for bad in (6, -1, 1 << 30):
        close(*run([0, 1, bad], 40), ref.attend(q, k, v, full[:, :2], [32], 0.125))
        assert plan.status() == 8 and plan.status() == 0
    out, lse = run([-1, 99, -5], 48)  # nothing left
    assert (out == 0).all() and (lse == float("-inf")).all()


def test_attend_non_finite_keys_follow_the_formula(cuda):
    """A NaN key makes its heads' rows NaN, not others'; a score of -inf takes no part."""
    gen = torch.Generator().manual_seed(6)
    k, v, q = randn(gen, 4, 2, 16, 64), randn(gen, 4, 2, 16, 64), randn(gen, 2, 2, 64).abs()
    k[0, 0, 3] = float("nan")
    plan = sc.DecodeAttention(sc.PagedKVCache(k.cuda(), v.cuda()), 2, 2)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32).cuda()
    out = plan.attend(q.cuda(), table, torch.tensor([20, 30], dtype=torch.int32).cuda())
    assert out[0, 0].isnan().all() and out[0, 1].isfinite().all() and out[1].isfinite().all()


@pytest.mark.parametrize("types", [TYPE_PAIRS[0], TYPE_PAIRS[3]])
def test_attend_beyond_32_bit_offsets(cuda, types):
    """Pages whose element offsets pass 2^31 and 2^32 bytes."""
    kind, stored = types
    gen = torch.Generator().manual_seed(7)
    d, page = 128, 64
    pages = 2 ** 31 // (page * d) + 5
    k = torch.empty(pages, 1, page, d, dtype=stored, device="cuda")
    v = torch.empty(pages, 1, page, d, dtype=stored, device="cuda")
    small = [randn(gen, 3, 1, page, d, dtype=stored) for _ in range(2)]
    at = [pages - 1, 2 ** 30 // (page * d), pages - 3]
    q = randn(gen, 1, 4, d, dtype=kind)
    for i, p in enumerate(at):
        k[p], v[p] = small[0][i].cuda(), small[1][i].cuda()
    plan = sc.DecodeAttention(sc.PagedKVCache(k, v), 4, 1)
    out, lse = plan.attend(q.cuda(), torch.tensor([at], dtype=torch.int32).cuda(),
                           torch.tensor([180], dtype=torch.int32).cuda(), return_lse=True)
    close(out, lse, ref.attend(q, *small, torch.tensor([[0, 1, 2]]), [180], 1 / math.sqrt(d)))
    new = randn(gen, 1, 1, d, dtype=kind)
    plan.cache.append(new.cuda(), new.cuda(), torch.tensor([181], dtype=torch.int32).cuda(),
                      torch.tensor([at], dtype=torch.int32).cuda())
    assert torch.equal(k[at[2], 0, 181 - 128].cpu(), new[0, 0].to(stored))


def test_serving_on_another_stream_and_in_a_graph(cuda):
    kind = TYPE_PAIRS[1]
    plan, q, table, sl, want = attend_case(kind, 2, 8, 128, 16, 0, "features", "heads", [900, 33, 0, 128])
    plain = plan.attend(q, table, sl)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = plan.attend(q, table, sl, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(plain, other)
    out, g = torch.zeros_like(plain), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan.attend(q, table, sl, out=out)
    for _ in range(2):
        out.zero_()
        g.replay()
        assert torch.equal(out, plain)


# --------------------------------------------------------------- adapters --

ADAPTERS = [
    # types, in, out, ranks, ids, token-major
    (TYPE_PAIRS[0], 512, 512, [4, 8, 6], [0, 2, -1, 1], False),
    (TYPE_PAIRS[0], 37, 53, [1, 0, 7], [0, 1, 2, 2, -1], False),
    (TYPE_PAIRS[0], 2048, 512, [256, 16], [1, 0, 0] * 11, True),
    (TYPE_PAIRS[1], 512, 2048, [4, 64, 17, 8], [3, 2, 1, 0, -1] * 13, False),
    (TYPE_PAIRS[1], 129, 257, [33, 5], [0] * 40 + [1] * 37, False),
    (TYPE_PAIRS[2], 1000, 904, [16, 24, 9], [0] * 100 + [-1] * 3 + [2] * 90 + [1] * 64, True),
    (TYPE_PAIRS[3], 4096, 1024, [8, 64, 12], [0, 1, 2, 1], True),
    (TYPE_PAIRS[3], 520, 512, [1, 3], [1, 0] * 150, False),
    (TYPE_PAIRS[4], 96, 40, [10], [0], True),
    (TYPE_PAIRS[4], 64, 8, [2, 200], [-1, -1, 1, 0], False),
    (TYPE_PAIRS[5], 100, 60, [4, 9], [0, 1, 1], False),
    (TYPE_PAIRS[6], 100, 60, [4, 9], [0, 1, 1], True),
]


def adapter_set(gen, types, k, m, ranks):
    down = [randn(gen, r, k, dtype=types[1], scale=k ** -0.5) for r in ranks]
    up = [randn(gen, m, r, dtype=types[1], scale=max(1, r) ** -0.5) for r in ranks]
    scales = [(-1.0) ** i * 2.0 / (i + 1) for i in range(len(ranks))]
    return down, up, scales


@pytest.mark.parametrize("types,k,m,ranks,ids,token_major", ADAPTERS)
@pytest.mark.parametrize("with_base", ["apart", "in place", "none"])
def test_adapters(cuda, types, k, m, ranks, ids, token_major, with_base):
    gen = torch.Generator().manual_seed(8)
    down, up, scales = adapter_set(gen, types, k, m, ranks)
    n = len(ids)
    x, base = randn(gen, k, n, dtype=types[0]), randn(gen, m, n, dtype=types[0])
    turn = (lambda y: y.t().contiguous().cuda().t()) if token_major else (lambda y: y.cuda())
    s = sc.LowRankAdapters([a.cuda() for a in down], [b.cuda() for b in up], scales)
    i = torch.tensor(ids, dtype=torch.int32)
    b = None if with_base == "none" else turn(base)
    got = s.apply(turn(x), i.cuda(), base=b, out=b if with_base == "in place" else None)
    s.check()
    want, tol = ref.adapters(x, i, down, up, scales, None if b is None else base, types[0])
    assert got.dtype == types[0] and got.shape == (m, n)
    assert ((got.cpu().double() - want).abs() <= tol).all()
    if with_base != "in place":
        assert torch.equal(got, s.apply(turn(x), i.cuda(), base=b))  # the same bits every time


def test_adapters_odd_strides_and_ids_beyond_the_set(cuda):
    gen = torch.Generator().manual_seed(9)
    down, up, scales = adapter_set(gen, TYPE_PAIRS[1], 200, 120, [8, 20])
    s = sc.LowRankAdapters([a.cuda() for a in down], [b.t().contiguous().cuda().t() for b in up], scales)
    x, base = randn(gen, 200, 2 * 21), randn(gen, 120, 3 * 21)
    ids = torch.tensor([0, 1, 7, -3, 1, 2, 0] * 3, dtype=torch.int32)
    got = s.apply(x.cuda()[:, ::2], ids.cuda(), base=base.cuda()[:, 1::3])
    assert s.status() == 10 and s.status() == 0
    want, tol = ref.adapters(x[:, ::2], ids, down, up, scales, base[:, 1::3], F32)
    assert ((got.cpu().double() - want).abs() <= tol).all()
    out = torch.zeros(120, 2 * 21).cuda()[:, ::2]
    assert torch.equal(s.apply(x.cuda()[:, ::2], ids.cuda(), base=base.cuda()[:, 1::3], out=out), got)


def test_adapters_other_tokens_do_not_leak(cuda):
    """NaN and infinity in a token, or in an adapter that a token does not use, stay there."""
    gen = torch.Generator().manual_seed(10)
    down, up, scales = adapter_set(gen, TYPE_PAIRS[0], 64, 64, [8, 8, 8])
    down[1].fill_(float("nan"))
    s = sc.LowRankAdapters([a.cuda() for a in down], [b.cuda() for b in up], scales)
    x = randn(gen, 64, 40)
    x[:, 5] = float("inf")
    x[:, 6] = float("nan")
    ids = torch.tensor([0, 2] * 20, dtype=torch.int32)
    ids[6], ids[9] = -1, 1
    base = randn(gen, 64, 40)
    y = s.apply(x.cuda(), ids.cuda(), base=base.cuda()).cpu()
    bad = ~y.isfinite().all(0)
    assert bad.tolist() == [i in (5, 9) for i in range(40)]
    assert torch.equal(y[:, 6], base[:, 6])


# ---------------------------------------------------------- a whole layer --

def test_decoding_steps_of_a_pruned_layer(cuda):
    """Sparse q/k/v/o projections with adapters, cache append and attention
    for several steps, against the same in 64 bits from the whole history."""
    from sparse_computation_b200 import workloads as wl
    from parity import to_csr_handle
    heads, d, n, steps = 8, 64, 4, 5
    gen = torch.Generator().manual_seed(11)
    dense, plans, sets, raw = {}, {}, {}, {}
    for i, name in enumerate("qkvo"):
        a = wl.magnitude_pruned(512, 512, 0.80, 0.05, 40 + i)
        plans[name] = sc.SpMMPlan(sc.csr_to_compressed_format_converter(to_csr_handle(a), 4, 1), n)
        w = torch.zeros(512, 512, dtype=torch.float64)
        r = torch.repeat_interleave(torch.arange(512), torch.from_numpy(a[2]).diff().long())
        w[r, torch.from_numpy(a[3]).long()] = torch.from_numpy(a[4])
        dense[name] = w
        raw[name] = adapter_set(gen, (F32, F32), 512, 512, [4, 8])
        sets[name] = sc.LowRankAdapters([x.cuda() for x in raw[name][0]], [x.cuda() for x in raw[name][1]], raw[name][2])
    ids = torch.tensor([0, -1, 1, 0], dtype=torch.int32)
    cos, sin = tables(32)
    rope = sc.RotaryTable(cos.cuda(), sin.cuda())
    cache = sc.PagedKVCache.allocate(12, 2, heads, d)
    attention = sc.DecodeAttention(cache, heads, n)
    table = torch.randperm(12, generator=gen).int().view(4, 3).cuda()

    def project(name, x):
        return sets[name].apply(x, ids.cuda(), base=plans[name].spmm(x))

    def project64(name, x):
        y = dense[name] @ x
        for t in range(n):
            a = int(ids[t])
            if a >= 0:
                y[:, t] += raw[name][2][a] * (raw[name][1][a].double() @ (raw[name][0][a].double() @ x[:, t]))
        return y

    split = lambda y: y.view(heads, d, n).permute(2, 0, 1)
    ks, vs = [], []
    for step in range(steps):
        x = randn(gen, 512, n)
        pos = torch.full((n,), step, dtype=torch.int32)
        xg = x.cuda()
        q = cache.append(split(project("k", xg)), split(project("v", xg)), pos.cuda(), table, rope=rope,
                         q=split(project("q", xg)))
        mixed = torch.empty(512, n, device="cuda")
        attention.attend(q, table, (pos + 1).cuda(), out=split(mixed))
        y = project("o", mixed).cpu().double()
        q64, _ = ref.rotate(split(project64("q", x.double())), pos, cos, sin, False)
        k64, _ = ref.rotate(split(project64("k", x.double())), pos, cos, sin, False)
        ks.append(k64)
        vs.append(split(project64("v", x.double())))
        z = torch.einsum("thd,sthd->ths", q64, torch.stack(ks)) / 8.0
        o = torch.einsum("ths,sthd->thd", torch.softmax(z, -1), torch.stack(vs))
        want = project64("o", o.permute(1, 2, 0).reshape(512, n))
        # four chained fp32 products of about 100 terms each: 2^-24 * sqrt-free worst case ~ 4 * 110 * 2^-24 of their
        # absolute sums, which stay below 20 times the result's largest value
        assert (y - want).abs().max() <= 4 * 110 * 2.0 ** -24 * 20 * want.abs().max()
    cache.check()
    attention.check()


# ------------------------------------------- adapters of many tokens -----

MANY = [
    # types, in, out, ranks, tokens of each adapter and without one (last), token-major, mixed
    (TYPE_PAIRS[0], 5000, 300, [9, 40, 17], [700, 300, 400, 100], False, False),  # five chunks of columns a block
    (TYPE_PAIRS[1], 5000, 300, [9, 40, 17], [700, 300, 400, 100], True, True),
    (TYPE_PAIRS[2], 700, 1100, [200, 70], [200, 150, 3], False, False),  # more than 64 ranks
    (TYPE_PAIRS[3], 576, 200, [256, 1, 0, 65], [100, 90, 80, 70, 30], True, False),
    (TYPE_PAIRS[4], 520, 4000, [33, 64], [257, 0, 0], False, True),
    (TYPE_PAIRS[5], 130, 70, [8], [300, 5], True, True),
    (TYPE_PAIRS[1], 5000, 90, [12, 30], [3, 2, 1], False, True),  # few tokens, two chunks of columns a block
]


@pytest.mark.parametrize("types,k,m,ranks,counts,token_major,mixed", MANY)
def test_adapters_many_tokens(cuda, types, k, m, ranks, counts, token_major, mixed):
    gen = torch.Generator().manual_seed(12)
    down, up, scales = adapter_set(gen, types, k, m, ranks)
    ids = torch.tensor([i if i < len(ranks) else -1 for i, c in enumerate(counts) for _ in range(c)], dtype=torch.int32)
    if mixed:
        ids = ids[torch.randperm(len(ids), generator=gen)]
    n = len(ids)
    x, base = randn(gen, k, n, dtype=types[0]), randn(gen, m, n, dtype=types[0])
    turn = (lambda y: y.t().contiguous().cuda().t()) if token_major else (lambda y: y.cuda())
    s = sc.LowRankAdapters([a.cuda() for a in down], [b.cuda() for b in up], scales)
    got = s.apply(turn(x), ids.cuda(), base=turn(base))
    s.check()
    want, tol = ref.adapters(x, ids, down, up, scales, base, types[0])
    assert ((got.cpu().double() - want).abs() <= tol).all()
    assert torch.equal(got, s.apply(turn(x), ids.cuda(), base=turn(base)))


@pytest.mark.parametrize("tokens", [200, 600])
def test_adapters_many_adapters(cuda, tokens):
    """More adapters than a sorting block counts in shared memory, most of them unused; ids beyond the set are none."""
    gen = torch.Generator().manual_seed(13)
    count = 2100
    down = [randn(gen, 1 + i % 3, 24) for i in range(count)]
    up = [randn(gen, 40, 1 + i % 3) for i in range(count)]
    s = sc.LowRankAdapters([a.cuda() for a in down], [b.cuda() for b in up], [0.5] * count)
    ids = torch.randint(-1, count, (tokens,), generator=gen).int()
    ids[7], ids[8] = 2099, 2100
    x = randn(gen, 24, tokens)
    got = s.apply(x.cuda(), ids.cuda())
    assert s.status() == 10
    want, tol = ref.adapters(x, ids, down, up, [0.5] * count, None, F32)
    assert ((got.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("types", [TYPE_PAIRS[0], TYPE_PAIRS[1], TYPE_PAIRS[3], TYPE_PAIRS[4]])
def test_attend_more_sequences_than_threads(cuda, types):
    """The scan over the lengths takes several rounds; empty, tiny and longer sequences alternate."""
    lens = [(i * 37) % 50 if i % 3 else (i % 2) for i in range(900)]
    plan, q, table, sl, want = attend_case(types, 1, 2, 32, 16, 0, "tokens", "heads", lens)
    close(*plan.attend(q, table, sl, return_lse=True), want)


@pytest.mark.parametrize("page", [1, 2, 3, 8, 16, 17, 32, 100])
def test_attend_page_sizes(cuda, page):
    plan, q, table, sl, want = attend_case(TYPE_PAIRS[1], 2, 6, 64, page, 0, "tokens", "slots", [1, 31, 257, 1000])
    close(*plan.attend(q, table, sl, return_lse=True), want)


@pytest.mark.parametrize("t", [1, 3, 5, 9, 17, 40, 700])
@pytest.mark.parametrize("layout", ["tokens", "features"])
def test_append_token_counts(cuda, t, layout):
    gen = torch.Generator().manual_seed(14)
    h, d, page = 2, 64, 16
    k, v, q = (randn(gen, t, n, d, dtype=BF16) for n in (h, h, 4))
    pages = -(-t // page)
    cache = sc.PagedKVCache.allocate(pages + 1, page, h, d, BF16)
    cos, sin = tables(16)
    pos = torch.arange(t, dtype=torch.int32)
    table = torch.randperm(pages + 1, generator=gen)[:pages].int().view(1, -1)
    got = cache.append(rows(k, layout), rows(v, layout), pos.cuda(), table.cuda(), torch.zeros(t, dtype=torch.int32).cuda(),
                       rope=sc.RotaryTable(cos.cuda(), sin.cuda()), q=rows(q, layout))
    cache.check()
    for given, out in ((q, got.cpu()), (k, cache.k.cpu()[table[0].long()].transpose(1, 2).reshape(-1, h, d)[:t])):
        want, mag = ref.rotate(given, pos, cos, sin, False)
        assert ((out.double() - want).abs() <= 2.0 ** -22 * mag + ref.rounding(want, BF16) * (1 + 2.0 ** -6)).all()
    assert torch.equal(cache.v.cpu()[table[0].long()].transpose(1, 2).reshape(-1, h, d)[:t], v)


def test_decode_demo(cuda, capsys):
    from sparse_computation_b200 import decode_demo
    assert decode_demo.main(["--requests", "4", "--steps", "6", "--layers", "2", "--page", "4"]) > 0
    assert "4 requests, 2 layers, bf16 cache" in capsys.readouterr().out

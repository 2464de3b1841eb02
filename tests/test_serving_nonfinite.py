"""Infinities and NaN among the operands: results follow the formulas, as sums and products of fp32 numbers do.

A kernel that splits an operand into parts meets differences of infinities that
the formula does not have; such results have to come out as the formula's."""
import math

import pytest
import torch

import serving_ref as ref
import sparse_computation_b200 as sc

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF, NAN = float("inf"), float("nan")


# --------------------------------------------------------------- adapters --

def formula(x, ids, down, up, scale, base):
    """base + scale up (down x) in fp64, product by product."""
    y = base.double().clone()
    for t in range(x.shape[1]):
        a = int(ids[t])
        if a >= 0:
            v = (down[a].double() * x[:, t].double()).sum(1) * scale
            y[:, t] += (up[a].double() * v).sum(1)
    return y


@pytest.mark.parametrize("kind,stored", [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("tokens", [200, 300, 600])
@pytest.mark.parametrize("token_major", [False, True])
def test_adapters_with_infinities(cuda, kind, stored, tokens, token_major):
    """In x, in base, in `down` (adapter 1) and in `up` (adapter 2); whole columns of one sign leave infinities, mixed ones NaN."""
    gen = torch.Generator().manual_seed(50)
    k, m, r = 1100, 72, 5
    down = [torch.randn(r, k, generator=gen).to(stored) for _ in range(4)]
    up = [torch.randn(m, r, generator=gen).to(stored) for _ in range(4)]
    down[0], up[0] = down[0].abs(), up[0].abs()
    up[0][40:] *= -1
    down[1][2, 1000] = INF
    up[2][3, 1], up[2][50, 2], up[2][51, 0] = INF, -INF, NAN
    x, base = torch.randn(k, tokens, generator=gen).to(kind), torch.randn(m, tokens, generator=gen).to(kind)
    ids = torch.randint(-1, 4, (tokens,), generator=gen).int()
    ids[:8] = torch.tensor([0, 0, 3, 0, 3, -1, 0, 0])
    x[9, 0], x[1099, 1], x[500, 2], x[700, 3], x[3, 4], x[3, 5] = INF, -INF, INF, NAN, NAN, INF
    base[5, 6], base[6, 7] = INF, NAN
    turn = (lambda y: y.t().contiguous().cuda().t()) if token_major else (lambda y: y.cuda())
    s = sc.LowRankAdapters([a.cuda() for a in down], [b.cuda() for b in up], [0.5] * 4)
    got = s.apply(turn(x), ids.cuda(), base=turn(base)).cpu().double()
    s.check()
    want = formula(x, ids, down, up, 0.5, base)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got == INF, want == INF) and torch.equal(got == -INF, want == -INF)
    assert (want[:, 0].abs() == INF).all() and want[:, 2].isnan().any() and want[:, 5].isfinite().all()
    fine = want.isfinite()
    x, base = x.clone(), base.clone()
    x[~x.isfinite()], base[~base.isfinite()] = 0, 0  # the bound of what is finite
    for w in down + up:
        w[~w.isfinite()] = 0
    y, tol = ref.adapters(x, ids, down, up, [0.5] * 4, base, kind)
    clean = fine & want.isclose(y, rtol=1e-9, atol=1e-9)
    assert clean.sum() > 0.5 * clean.numel()
    assert ((got - want).abs() <= tol)[clean].all()


# -------------------------------------------------------------- attention --

TYPES = [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (F16, F16), (BF16, F16)]
# cached keys: one warp's segment, a block's, several blocks'; a sequence without keys between them
LENGTHS = [[20, 0, 7], [700, 0, 130], [9000, 0, 40]]


def case(kind, stored, d, lens, page, seed):
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pool = sum(need)
    perm = torch.randperm(pool, generator=gen)
    table = torch.full((len(lens), max(need)), 1 << 30, dtype=torch.int32)
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = perm[at:at + c].int()
        at += c
    k, v = (torch.randn(pool, 2, page, d, generator=gen).to(stored) for _ in range(2))
    q = torch.randn(len(lens), 6, d, generator=gen).abs().to(kind)
    return q, k, v, table


def attend(q, k, v, table, lens):
    plan = sc.DecodeAttention(sc.PagedKVCache(k.cuda(), v.cuda()), q.shape[1], len(lens))
    out, lse = plan.attend(q.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), return_lse=True)
    plan.check()
    return out.cpu().double(), lse.cpu().double()


def without(k, v, table, lens, page, gone):
    """The same keys and values but those of sequence 0 at the places `gone`, in new pages."""
    kept = [[j for j in range(n) if i or j not in gone] for i, n in enumerate(lens)]
    need = [-(-len(x) // page) for x in kept]
    k2, v2 = torch.zeros(sum(need), *k.shape[1:], dtype=k.dtype), torch.zeros(sum(need), *v.shape[1:], dtype=v.dtype)
    t2 = torch.zeros(len(lens), max(need), dtype=torch.int32)
    at = 0
    for i, c in enumerate(need):
        t2[i, :c] = torch.arange(at, at + c).int()
        at += c
        for a, j in enumerate(kept[i]):
            k2[t2[i, a // page], :, a % page] = k[table[i, j // page], :, j % page]
            v2[t2[i, a // page], :, a % page] = v[table[i, j // page], :, j % page]
    return k2, v2, t2, [len(x) for x in kept]


@pytest.mark.parametrize("kind,stored", TYPES)
@pytest.mark.parametrize("d,page", [(64, 16), (128, 16), (40, 5)])
@pytest.mark.parametrize("lens", LENGTHS)
def test_scores_of_minus_infinity_take_no_part(cuda, kind, stored, d, page, lens):
    q, k, v, table = case(kind, stored, d, lens, page, 51)
    gone = {0, 3, lens[0] // 2, lens[0] - 1}
    want = ref.attend(q, *without(k, v, table, lens, page, gone), 1 / math.sqrt(d))
    for j in gone:  # q is positive: -inf is the score of these keys, whatever their values
        k[table[0, j // page], :, j % page, j % d] = -INF
        v[table[0, j // page], :, j % page] = 1000.0
    out, lse = attend(q, k, v, table, lens)
    w, wl, tol, ltol = want
    assert ((out - w).abs() <= tol).all()
    assert torch.equal(lse == -INF, wl == -INF)
    there = wl != -INF
    assert ((lse - wl)[there].abs() <= ltol[there]).all()


@pytest.mark.parametrize("kind,stored", TYPES)
@pytest.mark.parametrize("d,page", [(64, 16), (128, 16), (40, 5)])
@pytest.mark.parametrize("lens", LENGTHS)
def test_infinite_values_and_keys(cuda, kind, stored, d, page, lens):
    """kv head 0 of sequence 0: values of +inf, -inf and both; kv head 1: a key of +inf, so that its rows are NaN.
    Sequence 2 has a NaN value, and a query row with a NaN."""
    q, k, v, table = case(kind, stored, d, lens, page, 52)
    want = ref.attend(q, k, v, table, lens, 1 / math.sqrt(d))
    put = lambda pool, s, j, h, i, x: pool[table[s, j // page], h, j % page].__setitem__(i, x)
    last = lens[0] - 1
    put(v, 0, 2, 0, 1, INF)
    put(v, 0, last, 0, 5, -INF)
    put(v, 0, 1, 0, d - 1, INF)
    put(v, 0, last, 0, d - 1, -INF)
    put(k, 0, last // 2, 1, 7, INF)
    put(v, 2, 4, 1, 3, NAN)
    q[2, 1, 6] = NAN
    out, lse = attend(q, k, v, table, lens)
    w, wl, tol, ltol = want
    w, tol = w.clone(), tol.clone()
    w[0, :3, 1], w[0, :3, 5], w[0, :3, d - 1], w[0, 3:], w[2, 3:, 3], w[2, 1] = INF, -INF, NAN, NAN, NAN, NAN
    assert torch.equal(out.isnan(), w.isnan())
    assert torch.equal(out == INF, w == INF) and torch.equal(out == -INF, w == -INF)
    fine = w.isfinite()
    assert ((out - w).abs() <= tol)[fine].all()
    sure = torch.ones_like(wl, dtype=torch.bool)
    sure[0, 3:], sure[2, 1], sure[1] = False, False, False
    assert ((lse - wl).abs() <= ltol)[sure].all()
    assert not lse[0, 3:].isfinite().any() and lse[2, 1].isnan() and (lse[1] == -INF).all()

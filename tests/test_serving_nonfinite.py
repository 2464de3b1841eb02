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



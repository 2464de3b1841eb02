"""Operands of unequal size in one row: what is small beside a row's largest value keeps its digits.

The tolerances are those of serving_ref.py.  They go by the products that a
result really has (sums of |q k|, |p v|, |up down x|), so a large operand that
meets a zero does not widen them."""
import math

import pytest
import torch

import serving_ref as ref
import sparse_computation_b200 as sc

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def attention(q, k, v, lens, page, scale=None):
    """(out, lse) on the GPU of contiguous pages, and the 64-bit answer with its bounds."""
    each = -(-max(lens) // page)
    table = torch.arange(len(lens) * each).int().view(len(lens), each)
    plan = sc.DecodeAttention(sc.PagedKVCache(k.cuda(), v.cuda()), q.shape[1], len(lens), scale=scale)
    out, lse = plan.attend(q.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), return_lse=True)
    plan.check()
    return out.cpu().double(), lse.cpu().double(), ref.attend(q, k, v, table, lens, scale or 1 / math.sqrt(q.shape[2]))


def held(out, lse, want):
    w, wl, tol, ltol = want
    assert ((out - w).abs() <= tol).all(), ((out - w).abs() / tol).max()
    assert ((lse - wl).abs() <= ltol).all()


# types of queries and cache
WIDE = [(F32, F32), (F32, BF16), (F32, F16), (BF16, F16)]


@pytest.mark.parametrize("kind,stored", WIDE)
@pytest.mark.parametrize("n", [40, 1500])
def test_weights_far_below_a_sink(cuda, kind, stored, n):
    """One key takes nearly all of the weight, with a value of zero; the result is made of weights of e^-16 (2^-23)."""
    gen = torch.Generator().manual_seed(40)
    d, page = 64, 16
    pages = -(-n // page)
    k, v = (torch.randn(pages, 2, page, d, generator=gen).to(stored) for _ in range(2))
    q = torch.randn(1, 2, d, generator=gen).to(kind)
    k *= 0.25
    x = q[0].float()
    k[0, :, 5] = (x * (16 * 8 / x.square().sum(-1, keepdim=True))).to(stored)
    v[0, :, 5] = 0
    held(*attention(q, k, v, [n], page))


@pytest.mark.parametrize("kind,stored", WIDE)
def test_a_query_with_an_outlier_that_meets_zeros(cuda, kind, stored):
    gen = torch.Generator().manual_seed(41)
    d, page = 64, 16
    k, v = (torch.randn(3, 2, page, d, generator=gen).to(stored) for _ in range(2))
    q = torch.randn(1, 4, d, generator=gen).to(kind)
    q[:, :, 9] = 2.0 ** 18
    k[..., 9] = 0
    held(*attention(q, k, v, [40], page))


ADAPTERS = [(F32, F32), (F32, BF16), (F32, F16), (BF16, F16)]


@pytest.mark.parametrize("kind,stored", ADAPTERS)
@pytest.mark.parametrize("tokens", [40, 300])
@pytest.mark.parametrize("where", ["x", "v"])
def test_adapters_with_an_outlier_that_meets_zeros(cuda, kind, stored, tokens, where):
    """A feature of x that `down` does not read, or a rank that `up` does not read, 2^14 times larger than the others."""
    gen = torch.Generator().manual_seed(42)
    k, m, r = 64, 72, 12
    down, up = (torch.randn(r, k, generator=gen) / 8).to(stored), (torch.randn(m, r, generator=gen) / 3).to(stored)
    x = torch.randn(k, tokens, generator=gen).to(kind)
    if where == "x":
        x[7] = 2.0 ** 14
        down[:, 7] = 0
    else:
        down[3] = 2.0 ** 14 * torch.sign(down[3].float()).to(stored)
        x[:] = x.abs() * torch.sign(down[3].float()).to(kind)[:, None]
        up[:, 3] = 0
    s = sc.LowRankAdapters([down.cuda()], [up.cuda()], [1.0])
    ids = torch.zeros(tokens, dtype=torch.int32)
    got = s.apply(x.cuda(), ids.cuda()).cpu().double()
    want, tol = ref.adapters(x, ids, [down], [up], [1.0], None, kind)
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()

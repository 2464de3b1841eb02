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


# fp32 operands are split into two parts of 11 bits.  Rounding a part errs either way; cutting it off takes 0.9 units of
# 2^-23 of each operand's binade on average (0.6 of its size), always towards zero: 7e-8 an operand, and a product of
# two such tails that is left out another 1e-7.  Below, every sum has one product, so that nothing but the split and
# three or four roundings of 2^-24, which average out over 4096 results, and the constants' own (1.3e-8) is in the mean.

def spread(gen, *shape):
    """Numbers of either sign with mantissas spread evenly."""
    sign = torch.randint(0, 2, shape, generator=gen).float() * 2 - 1
    return sign * (1 + torch.rand(*shape, generator=gen)) * torch.randint(0, 4, shape, generator=gen).float().exp2()


def mean_off(got, want):
    return ((got - want) / want).mean().abs()


def test_scores_and_values_of_fp32_are_split_without_a_bias(cuda):
    gen = torch.Generator().manual_seed(43)
    seqs, heads, d = 64, 64, 64
    q, k = torch.zeros(seqs, heads, d), torch.zeros(seqs, heads, 16, d)
    at = torch.arange(heads)
    q[:, at, at] = spread(gen, seqs, heads)
    k[:, at, 0, at] = spread(gen, seqs, heads)
    v = spread(gen, seqs, heads, 16, d)
    out, lse, _ = attention(q, k, v, [1] * seqs, 16)
    z = q[:, at, at].double() * k[:, at, 0, at].double() / 8
    assert mean_off(lse, z) <= 2.0 ** -24
    assert mean_off(out, v[:, :, 0].double()) <= 2.0 ** -25


def test_adapters_of_fp32_are_split_without_a_bias(cuda):
    gen = torch.Generator().manual_seed(44)
    k, m, tokens = 64, 64, 512
    down, x = torch.zeros(1, k), torch.zeros(k, tokens)
    x[3] = spread(gen, tokens)
    sets = [(spread(gen, 1), spread(gen, m, 1)) for _ in range(8)]
    want, got = [], []
    for w, up in sets:
        down[0, 3] = w
        s = sc.LowRankAdapters([down.cuda()], [up.cuda()], [1.0])
        got.append(s.apply(x.cuda(), torch.zeros(tokens, dtype=torch.int32, device=cuda)).cpu().double())
        want.append(up.double() * (w.double() * x[3].double()))
    assert mean_off(torch.stack(got), torch.stack(want)) <= 2.0 ** -24

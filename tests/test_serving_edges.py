"""Serving operators at the edges of their arguments and values, against the 64-bit restatements of serving_ref.py."""
import math

import pytest
import torch

import serving_ref as ref
import sparse_computation_b200 as sc

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def test_adapter_weights_may_be_expanded_or_overlap(cuda):
    """Rows that share memory: one row for all ranks, one column for all ranks, sliding rows of one vector."""
    gen = torch.Generator().manual_seed(30)
    k, m, r = 40, 24, 6
    line = torch.randn(k + m + r, generator=gen)
    down = [line[:k].expand(r, k), line.as_strided((r, k), (1, 1)), torch.randn(r, k, generator=gen)]
    up = [torch.randn(m, r, generator=gen), line[:m].unsqueeze(1).expand(m, r), line[:r].expand(m, r)]
    on_gpu = line.cuda()
    down_gpu = [on_gpu[:k].expand(r, k), on_gpu.as_strided((r, k), (1, 1)), down[2].cuda()]
    up_gpu = [up[0].cuda(), on_gpu[:m].unsqueeze(1).expand(m, r), on_gpu[:r].expand(m, r)]
    s = sc.LowRankAdapters(down_gpu, up_gpu, [1.0, -0.5, 2.0])
    x, ids = torch.randn(k, 9, generator=gen), torch.tensor([0, 1, 2, 2, 1, 0, -1, 0, 2], dtype=torch.int32)
    got = s.apply(x.cuda(), ids.cuda())
    want, tol = ref.adapters(x, ids, down, up, [1.0, -0.5, 2.0], None, F32)
    assert ((got.cpu().double() - want).abs() <= tol).all()


def test_refusals_of_weights_without_two_dimensions(cuda):
    w = torch.zeros(4, 8, device=cuda)
    for down, up in ((torch.zeros((), device=cuda), w.t()), (w, torch.zeros((), device=cuda)), (w, torch.zeros(8, device=cuda))):
        with pytest.raises(sc.ScError) as e:
            sc.LowRankAdapters([down], [up], [1.0])
        assert e.value.code == sc.SC_ERR_ARG


def test_a_scale_beyond_fp32_is_refused(cuda):
    cache = sc.PagedKVCache.allocate(4, 16, 2, 64)
    for scale in (1e39, 3e38, 1e308):  # 3e38 / ln 2 is beyond fp32 too
        with pytest.raises(sc.ScError) as e:
            sc.DecodeAttention(cache, 4, 4, scale=scale)
        assert e.value.code == sc.SC_ERR_ARG
    sc.DecodeAttention(cache, 4, 4, scale=1e38)


@pytest.mark.parametrize("kind,stored", [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (F16, F16), (BF16, F16)])
@pytest.mark.parametrize("scale,size", [(1e-50, 1.0), (1e-9, 0.0), (1e-9, 2.0 ** -120), (1e-30, 1.0)])
def test_scales_and_queries_near_zero_weigh_all_keys_alike(cuda, kind, stored, scale, size):
    """A product of scale and query below fp32's smallest number is a score of zero, also beside keys that are masked."""
    gen = torch.Generator().manual_seed(31)
    lens, page, d = [21, 1, 0, 300], 16, 64
    need = [-(-n // page) for n in lens]
    table, at = torch.zeros(len(lens), max(need), dtype=torch.int32), 0
    for i, c in enumerate(need):
        table[i, :c] = torch.arange(at, at + c).int()
        at += c
    k, v = (torch.randn(at, 2, page, d, generator=gen).to(stored) for _ in range(2))
    q = (torch.randn(len(lens), 4, d, generator=gen) * size).to(kind)
    plan = sc.DecodeAttention(sc.PagedKVCache(k.cuda(), v.cuda()), 4, len(lens), scale=scale)
    out, lse = plan.attend(q.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), return_lse=True)
    plan.check()
    w, wl, tol, ltol = ref.attend(q, k, v, table, lens, scale)
    assert ((out.cpu().double() - w).abs() <= tol).all()
    there = wl != -math.inf
    assert torch.equal(lse.cpu() != -math.inf, there)
    assert ((lse.cpu().double() - wl)[there].abs() <= ltol[there]).all()

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

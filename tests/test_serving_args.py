"""Refusals of the serving operators: wrong arguments end in a status (ScError), never in a kernel."""
import ctypes
from struct import pack

import pytest
import torch

import sparse_computation_b200 as sc


def create(k=4096, v=8192, pages=4, page=16, heads=2, dim=64, ks=(2048, 1024, 64), vs=(2048, 1024, 64), kind=0):
    h = ctypes.c_void_p()
    code = sc.lib().sc_kv_cache_create(pack("13q", k, v, pages, page, heads, dim, *ks, *vs, kind), 0, ctypes.byref(h))
    return code, sc.lib().sc_last_error_string().decode()


@pytest.mark.parametrize("change,code,words", [
    (dict(k=0), sc.SC_ERR_ARG, "null"), (dict(kind=5), sc.SC_ERR_ARG, "type"), (dict(pages=0), sc.SC_ERR_ARG, "positive"),
    (dict(page=-1), sc.SC_ERR_ARG, "positive"), (dict(dim=260), sc.SC_ERR_UNSUPPORTED, "256"),
    (dict(dim=6), sc.SC_ERR_UNSUPPORTED, "16 bytes"), (dict(dim=36, kind=1), sc.SC_ERR_UNSUPPORTED, "16 bytes"),
    (dict(ks=(2048, 1024, 66)), sc.SC_ERR_UNSUPPORTED, "strides"), (dict(v=8200), sc.SC_ERR_UNSUPPORTED, "aligned"),
    (dict(pages=1 << 28), sc.SC_ERR_UNSUPPORTED, "slots"), (dict(vs=(-2048, 1024, 64)), sc.SC_ERR_UNSUPPORTED, "strides"),
    (dict(heads=70000), sc.SC_ERR_UNSUPPORTED, "heads"),
])
def test_cache_is_checked_before_any_gpu_call(change, code, words):
    got, text = create(**change)
    assert got == code and words in text


def test_null_handles_are_refused():
    L = sc.lib()
    h, n = ctypes.c_void_p(), ctypes.c_int64()
    assert L.sc_kv_cache_create(None, 0, ctypes.byref(h)) == sc.SC_ERR_ARG
    assert L.sc_kv_append(None, None, None) == sc.SC_ERR_ARG
    assert L.sc_attn_create(None, 8, 4, 0.0, 0, ctypes.byref(h)) == sc.SC_ERR_ARG
    assert L.sc_attn_decode(None, None, None) == sc.SC_ERR_ARG
    assert L.sc_adapters_apply(None, None, None) == sc.SC_ERR_ARG
    assert L.sc_adapters_workspace(None, 4, ctypes.byref(n)) == sc.SC_ERR_ARG
    for free in (L.sc_kv_cache_free, L.sc_attn_free, L.sc_adapters_free):
        free(None)


def adapters(ranks=(4,), k=8, m=8, kind=0, down=1, ld=8, count=1, uld=4):
    n = max(1, count)
    h = ctypes.c_void_p()
    i64, vp = ctypes.c_int64 * n, ctypes.c_void_p * n
    code = sc.lib().sc_adapters_create(0, k, m, count, i64(*ranks), kind, vp(down * 4096), i64(ld), vp(4096), i64(uld),
                                       (ctypes.c_float * n)(1.0), None, ctypes.byref(h))
    return code


@pytest.mark.parametrize("change,code", [
    (dict(count=0), sc.SC_ERR_ARG), (dict(k=0), sc.SC_ERR_ARG), (dict(m=-1), sc.SC_ERR_ARG), (dict(kind=3), sc.SC_ERR_ARG),
    (dict(ranks=(257,)), sc.SC_ERR_UNSUPPORTED), (dict(ranks=(-1,)), sc.SC_ERR_UNSUPPORTED), (dict(ld=7), sc.SC_ERR_ARG),
    (dict(down=0), sc.SC_ERR_ARG), (dict(uld=3), sc.SC_ERR_ARG),
])
def test_adapter_sets_are_checked_before_any_gpu_call(change, code):
    assert adapters(**change) == code


def test_python_checks_need_no_gpu():
    k = torch.zeros(2, 2, 16, 64)
    for args in ((k, k), (k[0], k[0]), (k, k.half()), (k.double(), k.double()), (k, k[:1])):
        with pytest.raises(sc.ScError) as e:
            sc.PagedKVCache(*args)
        assert e.value.code == sc.SC_ERR_ARG
    for args in ((k[0, 0], k[0, 0]), (k[0, 0].half(), k[0, 0])):
        with pytest.raises(sc.ScError):
            sc.RotaryTable(*args)
    a, b = torch.zeros(4, 8), torch.zeros(6, 4)
    for args in (([a], [b], [1.0]), ([], [], []), ([a], [], [1.0]), ([a], [b], [])):
        with pytest.raises(sc.ScError) as e:
            sc.LowRankAdapters(*args)
        assert e.value.code == sc.SC_ERR_ARG


@pytest.mark.gpu
def test_append_refusals(cuda):
    cache = sc.PagedKVCache.allocate(4, 16, 2, 64)
    x = torch.zeros(3, 2, 64, device=cuda)
    pos, table = torch.arange(3, dtype=torch.int32, device=cuda), torch.zeros(3, 2, dtype=torch.int32, device=cuda)
    q = torch.zeros(3, 4, 64, device=cuda)
    rope = sc.RotaryTable(torch.zeros(50, 40, device=cuda), torch.zeros(50, 40, device=cuda))
    good = dict(k=x, v=x, positions=pos, page_table=table, q=q)
    cache.append(**good)
    for change in (dict(k=x[:, :1]), dict(v=x.half()), dict(k=x.double(), v=x.double()), dict(k=x.cpu()), dict(v=x[:2]),
                   dict(positions=pos.long()), dict(positions=pos[:2]), dict(positions=pos.cpu()),
                   dict(page_table=table[:2]), dict(page_table=table.long()), dict(page_table=table[0]),
                   dict(seq_ids=pos[:1]), dict(q=q.half()), dict(q=q[..., :32]), dict(q=q[0]), dict(q_out=q[:2]),
                   dict(q_out=torch.zeros(1, 1, 64, device=cuda).expand(3, 4, 64)), dict(rope=rope),
                   dict(q=None, q_out=q), dict(q=q.transpose(0, 1).contiguous().transpose(0, 1), q_out=q[:, :2])):
        with pytest.raises(sc.ScError) as e:
            cache.append(**{**good, **change})
        assert e.value.code == sc.SC_ERR_ARG
    none = x[:0]
    assert cache.append(none, none, pos[:0], table, q=q[:0]).shape == (0, 4, 64)


@pytest.mark.gpu
def test_attend_refusals(cuda):
    cache = sc.PagedKVCache.allocate(4, 16, 2, 64)
    for args in ((3, 4), (0, 4), (4, 0), (4, 1 << 21)):
        with pytest.raises(sc.ScError) as e:
            sc.DecodeAttention(cache, *args)
        assert e.value.code == sc.SC_ERR_ARG
    for kw in (dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1)):
        with pytest.raises(sc.ScError):
            sc.DecodeAttention(cache, 4, 4, **kw)
    plan = sc.DecodeAttention(cache, 4, 4)
    q, lens = torch.zeros(3, 4, 64, device=cuda), torch.ones(3, dtype=torch.int32, device=cuda)
    table = torch.zeros(3, 2, dtype=torch.int32, device=cuda)
    good = dict(q=q, page_table=table, seq_lens=lens)
    plan.attend(**good)
    for change in (dict(q=q[:, :2]), dict(q=q.double()), dict(q=q.cpu()), dict(q=torch.zeros(5, 4, 64, device=cuda)),
                   dict(page_table=table[:2]), dict(page_table=table.long()), dict(page_table=table.t().contiguous().t()),
                   dict(seq_lens=lens.long()), dict(seq_lens=lens[:2]), dict(out=q.half()), dict(out=q[:2]),
                   dict(out=q[:1].expand(3, 4, 64))):
        with pytest.raises(sc.ScError) as e:
            plan.attend(**{**good, **change})
        assert e.value.code == sc.SC_ERR_ARG
    out, lse = plan.attend(q[:0], table, lens[:0], return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


@pytest.mark.gpu
def test_adapters_refusals(cuda):
    s = sc.LowRankAdapters([torch.zeros(4, 8, device=cuda)], [torch.zeros(6, 4, device=cuda)], [1.0])
    x, base, ids = torch.zeros(8, 5, device=cuda), torch.zeros(6, 5, device=cuda), torch.zeros(5, dtype=torch.int32, device=cuda)
    good = dict(x=x, ids=ids, base=base)
    s.apply(**good)
    for change in (dict(x=x[:7]), dict(x=x.double()), dict(x=x.cpu()), dict(x=x[0]), dict(ids=ids.long()), dict(ids=ids[:4]),
                   dict(base=base.half()), dict(base=base[:5]), dict(out=base[:, :4]), dict(out=base[:1].expand(6, 5)),
                   dict(out=base.t().contiguous().t()[:5])):
        with pytest.raises(sc.ScError) as e:
            s.apply(**{**good, **change})
        assert e.value.code == sc.SC_ERR_ARG
    with pytest.raises(sc.ScError):
        sc.LowRankAdapters([torch.zeros(4, 8, device=cuda)], [torch.zeros(6, 5, device=cuda)], [1.0])
    assert s.apply(x[:, :0], ids[:0]).shape == (6, 0)

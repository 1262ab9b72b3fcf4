"""Refusals of the paged batch-decode operators: every bad argument is answered before any
device work, at the C entry points and in the Python calls (CPU only)."""
import ctypes

import pytest
import torch

import hyperion_b200 as hb
from hyperion_b200 import ops

P = ctypes.c_void_p(4096)  # a non-null, 16-byte aligned pointer that is never followed
ODD = ctypes.c_void_p(4104)


def _plan(L, **kw):
    a = dict(cached=P, new=P, n_req=4, page=16, n_pages=8, free=P, n_free=8, table=P, max_blocks=4, pos0=0, max_rows=8,
             a=P, b=P, c=P, d=P, e=P, f=P)
    a.update(kw)
    return L.hyb_paged_plan(*a.values(), None)


@pytest.mark.parametrize("kw", [dict(cached=None), dict(table=None), dict(free=None), dict(n_free=-1), dict(n_req=0),
                                dict(n_req=8193), dict(page=0), dict(n_pages=0), dict(max_blocks=0), dict(max_rows=0),
                                dict(pos0=-1), dict(n_pages=1 << 27), dict(max_blocks=1 << 27),
                                dict(pos0=(1 << 31) - 10), dict(f=None)])
def test_plan_refuses(built_lib, kw):
    assert _plan(built_lib, **kw) == hb.INVALID_ARGUMENT
    assert hb.last_error()


def _post(L, **kw):
    a = dict(qkv=P, T=4, ld=256, H=2, nkv=1, hd=64, vfk=0, qn=P, kn=P, inv=P, pos=P, slot=P, n_slots=64, eps=1e-6, q=P, k=P,
             v=P)
    a.update(kw)
    return L.hyb_qkv_post_paged(*a.values(), None)


@pytest.mark.parametrize("kw", [dict(qkv=None), dict(v=None), dict(T=0), dict(H=0), dict(nkv=0), dict(n_slots=0), dict(ld=255),
                                dict(ld=260), dict(qkv=ODD), dict(k=ODD), dict(qn=ODD)])
def test_post_refuses(built_lib, kw):
    assert _post(built_lib, **kw) == hb.INVALID_ARGUMENT


@pytest.mark.parametrize("hd", [32, 96, 512])
def test_post_unsupported_head_dim(built_lib, hd):
    assert _post(built_lib, hd=hd, ld=4096) == hb.UNSUPPORTED


def _attn(L, **kw):
    a = dict(q=P, k=P, v=P, n_pages=8, page=16, pt=P, plen=20, bt=P, max_blocks=2, own=P, start=P, pos=P, T=2, n_req=2, max_q=1,
             max_own=32, H=2, nkv=1, hd=64, window=0, scale=1.0, softcap=0.0, out=P, scratch=P, nbytes=1 << 30)
    a.update(kw)
    return L.hyb_sdpa_shared_prefix(*a.values(), None)


@pytest.mark.parametrize("kw", [dict(q=None), dict(scratch=None), dict(pt=None), dict(T=0), dict(n_req=0), dict(n_req=1025), dict(max_q=0),
                                dict(max_own=-1), dict(plen=-1), dict(H=3, nkv=2), dict(window=-1), dict(n_pages=0),
                                dict(max_blocks=0), dict(n_pages=1 << 28), dict(q=ODD), dict(out=ODD), dict(scratch=ODD),
                                dict(plen=(1 << 31) - 1), dict(nbytes=64)])
def test_attn_refuses(built_lib, kw):
    assert _attn(built_lib, **kw) == hb.INVALID_ARGUMENT


def test_attn_refuses_too_many_steps(built_lib):
    # 1024 requests of one row each, their own keys of 2^25 tokens: 2^31 steps of 16 keys
    kw = dict(T=1024, n_req=1024, max_q=1, plen=0, pt=None, nbytes=1 << 40)
    assert _attn(built_lib, max_own=1 << 25, **kw) == hb.INVALID_ARGUMENT
    assert "steps of 16 keys" in hb.last_error()


@pytest.mark.parametrize("kw", [dict(hd=32), dict(hd=512), dict(page=8), dict(page=48), dict(page=512)])
def test_attn_unsupported(built_lib, kw):
    assert _attn(built_lib, **kw) == hb.UNSUPPORTED


def test_scratch_bytes(built_lib):
    f = built_lib.hyb_sdpa_shared_prefix_scratch_bytes
    assert f(0, 1, 1, 1, 1, 2, 1, 64) == 0 and f(1, 1, 1, 1, 1, 2, 1, 96) == 0 and f(1, 1, 1, 1, 1, 3, 2, 64) == 0
    assert f(1, 1, 1, 0, 0, 2, 1, 64) > 0
    for T, n, q, own, pre, H, nkv, hd in [(64, 64, 1, 1024, 16384, 32, 16, 128), (2048, 8, 300, 600, 8192, 16, 8, 256)]:
        assert 0 < f(T, n, q, own, pre, H, nkv, hd) < 1 << 30


def _sample(L, **kw):
    a = dict(x=P, f32=0, rows=2, vocab=100, ld=100, u=P, t=P, k=P, p=P, m=P, tok=P, kept=P, prob=P)
    a.update(kw)
    return L.hyb_sample_batch(*a.values(), None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(u=None), dict(tok=None), dict(rows=0), dict(vocab=0), dict(ld=99),
                                dict(vocab=(1 << 19) + 1, ld=1 << 20), dict(x=ctypes.c_void_p(4098), f32=1),
                                dict(x=ctypes.c_void_p(4097))])
def test_sample_refuses(built_lib, kw):
    assert _sample(built_lib, **kw) == hb.INVALID_ARGUMENT


def test_python_calls_refuse_cpu_tensors(built_lib):
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_plan(i, i, i, torch.zeros(2, 2, dtype=torch.int32), 4, 16, 8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.sample_batch(torch.zeros(2, 8), torch.zeros(2))
    with pytest.raises(ValueError):
        ops.sample_batch(torch.zeros(2, 8, dtype=torch.float16), torch.zeros(2))
    with pytest.raises(ValueError):
        ops.paged_plan(i, i, i, i, 4, 16, 8)
    pool = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.qkv_post_paged(torch.zeros(2, 64, dtype=torch.bfloat16), 2, 1, 64, False, None, None, None, i, i, pool, pool)
    with pytest.raises(ValueError, match="CUDA"):
        ops.sdpa_shared_prefix(torch.zeros(2, 2, 64, dtype=torch.bfloat16), pool, pool, None, 0, torch.zeros(2, 2, dtype=torch.int32),
                               i, torch.zeros(3, dtype=torch.int32), i, 1, 16)

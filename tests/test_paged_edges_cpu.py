"""Refusals of the paged batch-decode operators for calls whose arguments do not go together (CPU only)."""
import ctypes

import pytest
import torch

import hyperion_b200 as hb
from hyperion_b200 import ops

AT = {n: 1 << 20 | i << 16 for i, n in enumerate(["cached", "new", "free", "table", "row_start", "row_req", "row_pos", "slot_map",
                                                  "total_lens", "status"])}  # addresses that are never followed


def _plan(L, at):
    p = {k: ctypes.c_void_p(v) for k, v in at.items()}
    return L.hyb_paged_plan(p["cached"], p["new"], 4, 16, 8, p["free"], 8, p["table"], 4, 0, 32, p["row_start"], p["row_req"], p["row_pos"],
                            p["slot_map"], p["total_lens"], p["status"], None)


@pytest.mark.parametrize("moved,onto,by", [
    ("cached", "total_lens", 0),          # a step fed with its own lengths
    ("new", "total_lens", 12), ("cached", "row_start", 16), ("new", "row_pos", 124), ("free", "slot_map", -28), ("free", "status", 12),
    ("cached", "table", 60), ("free", "table", -4), ("status", "total_lens", 0), ("row_req", "slot_map", 4), ("row_start", "row_req", -16),
    ("total_lens", "table", 32)])
def test_plan_refuses_overlapping_outputs(built_lib, moved, onto, by):
    at = dict(AT)
    at[moved] = at[onto] + by
    assert _plan(built_lib, at) == hb.INVALID_ARGUMENT
    assert "overlap" in hb.last_error()


@pytest.mark.parametrize("n_single,chunk,own,prefix,H,nkv,hd,most", [
    (63, 2000, 4096, 2048, 16, 8, 256, 100), (63, 2048, 4096, 16384, 32, 16, 128, 100), (255, 2048, 4096, 2048, 16, 8, 256, 150),
    (1023, 2048, 4096, 16384, 32, 16, 128, 300), (1023, 8192, 8192, 0, 4, 4, 64, 60)])
def test_scratch_of_single_rows_beside_a_chunk(built_lib, n_single, chunk, own, prefix, H, nkv, hd, most):
    """At most what the rows can touch: a float output and two statistics of every (row, head) once for the 128-row kernel
    (in 148 parts at most over its tiles), and of the 16-row units, rows / 16 + requests + shares. In MB."""
    f = built_lib.hyb_sdpa_shared_prefix_scratch_bytes
    T, n = n_single + chunk, n_single + 1
    got = f(T, n, chunk, own, prefix, H, nkv, hd)
    wide = 4 * (hd + 2) * H * (T + 148 * 128)
    small = 4 * (hd + 2) * 16 * nkv * (T * (H // nkv) / 16 + n + 592 / nkv + 1) + 8 * (T * (H // nkv) / 16 + n + 1)
    assert 0 < got <= wide + small + 4096
    assert got < most << 20


def test_scratch_bounds_hold_for_uniform_batches(built_lib):
    """No larger than a tile a request, where all requests have as many rows."""
    f = built_lib.hyb_sdpa_shared_prefix_scratch_bytes
    for n, q, H, nkv, hd in [(64, 1, 32, 16, 128), (1024, 1, 16, 1, 64), (300, 3, 8, 4, 256)]:
        G = H // nkv
        units = n * -(-q * G // 16)
        assert f(n * q, n, q, 200, 0, H, nkv, hd) <= 4 * (hd + 2) * 16 * nkv * (units + 592 / nkv + 1) + 8 * units + 4096


@pytest.mark.parametrize("i,v", [(4, 1 << 32), (5, (1 << 32) + 16), (6, 1 << 31), (7, 1 << 40), (7, -(1 << 32))])
def test_plan_sizes_are_not_cut_to_32_bits(built_lib, i, v):
    x = torch.zeros(2, dtype=torch.int32)
    args = [x, x, x, torch.zeros(2, 2, dtype=torch.int32), 4, 16, 8, 0]
    args[i] = v
    with pytest.raises(ValueError, match="2\\^31"):
        ops.paged_plan(*args)


@pytest.mark.parametrize("kw", [dict(window=(1 << 32) + 1), dict(window=1 << 32), dict(max_own=1 << 32), dict(max_q=(1 << 33) + 1),
                                dict(prefix_len=1 << 32)])
def test_attention_sizes_are_not_cut_to_32_bits(built_lib, kw):
    i, pool = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16)
    a = dict(q=torch.zeros(2, 2, 64, dtype=torch.bfloat16), k_pool=pool, v_pool=pool, prefix_table=None, prefix_len=0, block_table=i[None],
             own_lens=i, row_start=i, row_pos=i, max_q=1, max_own=16)
    a.update(kw)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.sdpa_shared_prefix(**a)


def test_scratch_sizes_are_not_cut_to_32_bits(built_lib):
    good = [4, 2, 2, 100, 100, 4, 2, 64]
    assert ops.SharedPrefixScratch(*good, device="cpu").nbytes > 0
    for i in range(8):
        bad = list(good)
        bad[i] += 1 << 32
        with pytest.raises(ValueError, match="2\\^31"):
            ops.SharedPrefixScratch(*bad, device="cpu")
        bad[i] = -1
        with pytest.raises(ValueError):
            ops.SharedPrefixScratch(*bad, device="cpu")


def test_post_sizes_are_not_cut_to_32_bits(built_lib):
    pool = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16)
    for kw in ((1 << 32 | 2, 1, 64), (2, 1 << 32 | 1, 64), (2, 1, 1 << 32 | 64)):
        with pytest.raises(ValueError, match="2\\^31"):
            ops.qkv_post_paged(torch.zeros(2, 256, dtype=torch.bfloat16), *kw, False, None, None, None, None, None, pool, pool)


@pytest.mark.parametrize("moved,onto,by", [("prob", "u", 0), ("token", "top_k", 0), ("kept", "token", 4), ("prob", "temperature", -8),
                                           ("u", "kept", 8), ("token", "logits", 1200), ("prob", "min_p", 8), ("kept", "top_p", 0)])
def test_sample_refuses_overlapping_outputs(built_lib, moved, onto, by):
    at = {n: 1 << 20 | i << 16 for i, n in enumerate(["logits", "u", "temperature", "top_k", "top_p", "min_p", "token", "kept", "prob"])}
    at[moved] = at[onto] + by
    p = {k: ctypes.c_void_p(v) for k, v in at.items()}
    assert built_lib.hyb_sample_batch(p["logits"], 1, 3, 100, 104, p["u"], p["temperature"], p["top_k"], p["top_p"], p["min_p"], p["token"],
                                      p["kept"], p["prob"], None) == hb.INVALID_ARGUMENT
    assert "overlap" in hb.last_error()

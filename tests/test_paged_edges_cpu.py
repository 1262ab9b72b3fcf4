"""Refusals of the paged batch-decode operators for calls whose arguments do not go together (CPU only)."""
import ctypes

import pytest

import hyperion_b200 as hb

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

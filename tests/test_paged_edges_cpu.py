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

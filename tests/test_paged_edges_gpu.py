"""Calls of the paged batch-decode operators at the edges of what their documentation allows.

Roundings as in test_paged_gpu.py: bf16 half a step is 2^-8 of the value, fp32 2^-24.
"""
import numpy as np
import pytest

from tests.conftest import has_gpu
from tests.test_paged_gpu import Batch, _no_timeouts, run_plan, run_sample  # noqa: F401

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not has_gpu(), reason="no CUDA device")]


# ---------------------------------------------------------------------------------- plan
@pytest.mark.parametrize("page,cached,new", [(2 ** 31 - 1, [2 ** 30 + 5, 2, 2 ** 31 - 4, 0], [3, 1, 3, 2]), (2 ** 30 + 1, [2 ** 30 - 1, 0], [2, 4]),
                                             (1000, [2147482990, 2147482000, 0], [5, 3, 1])])
def test_plan_lengths_whose_rounding_up_passes_32_bits(built_lib, page, cached, new):
    width = (2 ** 31 - 1) // page
    n = len(cached)
    table = np.zeros((n, width), np.int64)
    for b in range(n):
        table[b, -1] = b % width  # pages of the pool: 0 .. width - 1
    run_plan(np.array(cached), np.array(new), np.arange(n) % width, table, width, page, sum(new) + 2)


def test_plan_most_rows(built_lib):
    """2^31 - 1 rows: every one behind the last is -1, up to the end of each array."""
    import torch
    from hyperion_b200 import ops
    rows = 2 ** 31 - 1
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    plan = ops.paged_plan(i32(0, 7), i32(3, 2), i32(5, 6, 7), torch.zeros(2, 4, dtype=torch.int32, device="cuda"), 8, 16, rows)
    assert plan.row_start.tolist() == [0, 3, 5] and plan.status.tolist() == [1, 5, 0, 0]
    assert plan.row_pos[:5].tolist() == [0, 1, 2, 7, 8] and plan.slot_map[:5].tolist() == [80, 81, 82, 7, 8]
    for x in (plan.row_req, plan.row_pos, plan.slot_map):
        assert all(int(x[i:i + 2 ** 29].max()) == -1 == int(x[i:i + 2 ** 29].min()) for i in range(5, rows, 2 ** 29))
    del plan, x
    torch.cuda.empty_cache()


def test_plan_stepped_from_its_own_lengths(built_lib):
    """total_lens is the next step's cached_lens: of the same plan refused, of two in turn right."""
    import torch
    import hyperion_b200 as hb
    from hyperion_b200 import ops
    n, page, rows = 1000, 16, 3000
    rng = np.random.default_rng(1)
    table = torch.zeros(n, 8, dtype=torch.int32, device="cuda")
    free = torch.arange(4000, dtype=torch.int32, device="cuda")
    lens, done = torch.zeros(n, dtype=torch.int32, device="cuda"), np.zeros(n, np.int64)
    plans = [ops.PagedPlan(n, rows), ops.PagedPlan(n, rows)]
    for i in range(6):
        new = rng.integers(0, 4, n)
        plan = ops.paged_plan(lens, torch.tensor(new, dtype=torch.int32, device="cuda"), free, table, 4000, page, rows, plan=plans[i % 2])
        done += new
        assert plan.total_lens.tolist() == done.tolist() and plan.status[1:].tolist() == [int(new.sum()), 0, 0]
        free, lens = free[int(plan.status[0]):].contiguous(), plan.total_lens
        with pytest.raises(hb.HypError, match="overlap"):
            ops.paged_plan(lens, torch.ones(n, dtype=torch.int32, device="cuda"), free, table, 4000, page, rows, plan=plan)


def test_plan_empty_free_list_overlaps_nothing(built_lib):
    import torch
    import hyperion_b200 as hb
    from hyperion_b200 import ops
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    cached, new, table, plan = i32(3, 5), i32(1, 2), i32(4, 7), ops.PagedPlan(2, 4)
    hb.check(built_lib.hyb_paged_plan(cached.data_ptr(), new.data_ptr(), 2, 16, 8, plan.slot_map.data_ptr() + 4, 0, table.data_ptr(), 1, 0, 4,
                                      *plan._at, torch.cuda.current_stream().cuda_stream))
    assert plan.slot_map.tolist() == [4 * 16 + 3, 7 * 16 + 5, 7 * 16 + 6, -1] and plan.status.tolist() == [0, 3, 0, 0]


# ----------------------------------------------------------------------------- attention
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("B,q,prefix", [(2, 150, 300), (2, 1, 30), (40, 1, 300), (4, 1, 300)])
def test_attn_output_on_any_16_byte_boundary(built_lib, hd, B, q, prefix):
    """An output 16, 32 or 48 bytes into a buffer gets the bits of an aligned one; nothing beside it is written."""
    import torch
    b = Batch(8, 4, hd, 16, prefix, [160] * B, [q] * B, seed=hd + B)
    want = b.call()
    n = want.numel()
    for off in (8, 16, 24):
        flat = torch.full((n + 32,), 7.0, dtype=torch.bfloat16, device="cuda")
        out = flat[off:off + n].view(want.shape)
        assert out.data_ptr() % 32 == (16 if off % 16 else 0)
        b.call(out=out)
        assert torch.equal(out, want)
        assert (flat[:off] == 7.0).all() and (flat[off + n:] == 7.0).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("B,q,prefix,own", [(3, 1, 0, 80), (3, 1, 100, 300), (40, 1, 100, 300), (2, 70, 100, 300)])
def test_attn_pages_that_no_row_sees(built_lib, hd, B, q, prefix, own):
    """Rows that stand before their request's last keys: the pages behind them are not looked at."""
    import torch
    start = prefix + own - q - 33  # two pages and more end unseen
    b = Batch(4, 2, hd, 16, prefix, [own] * B, [q] * B, seed=hd + B, positions=np.tile(start + np.arange(q), B))
    for page in (-1, 10 ** 6):
        c = b.table.copy()
        b.table[:, (own - 1) // 16] = page
        got = b.call()
        b.table = c
        b.check(got, rows=list(range(min(b.T, 12))) + [b.T - 1])
        assert torch.isfinite(got).all()


@pytest.mark.parametrize("prefix", [300, 700])
def test_attn_prefix_pages_that_no_row_sees(built_lib, prefix):
    b = Batch(4, 2, 64, 16, prefix, [3, 2], [1, 1], seed=prefix, positions=[100, 90])
    tab = b.ptab.copy()
    b.ptab[7:] = -1
    got = b.call()
    b.ptab = tab
    b.check(got)


@pytest.mark.parametrize("hd,window,softcap", [(64, 0, 0.0), (128, 0, 20.0), (128, 300, 0.0), (256, 0, 0.0)])
@pytest.mark.parametrize("prefix,chunk", [(0, 900), (30, 40), (400, 900), (2000, 300), (2000, 40)])
def test_attn_decode_rows_beside_a_chunk(built_lib, hd, window, softcap, prefix, chunk):
    """One step of many single rows and one request's long chunk of new rows; the scratch is used within its bounds."""
    import torch
    from hyperion_b200 import ops
    rng = np.random.default_rng(hd)
    own = rng.integers(1, 200, 40)
    q = np.ones(40, np.int64)
    q[:3], q[17], q[39] = [0, 2, 1], chunk, 19
    own[17], own[0], own[39] = chunk + 50, 30, 20
    b = Batch(8, 4, hd, 32, prefix, own, q, seed=hd + window, window=window, softcap=softcap, lead=1, pad_rows=3)
    scratch = ops.SharedPrefixScratch(b.T, 40, chunk, int(own.max()), prefix, 8, 4, hd)
    whole = torch.full((scratch.nbytes + 4096,), 77, dtype=torch.uint8, device="cuda")
    scratch.buf = whole[:scratch.nbytes]
    first = int(b.start[17])
    rows = list(range(1, first + 3, 3)) + [first + chunk // 2 - 1, first + chunk - 3, first + chunk - 2, first + chunk - 1, first + chunk]
    b.check(b.call(scratch=scratch), rows=rows + list(range(int(b.start[39]), int(b.start[40]), 6)) + [b.T - 4])
    assert (whole[scratch.nbytes:] == 77).all()


@pytest.mark.parametrize("H,nkv,hd,B,prefix,softcap", [(8, 4, 64, 200, 3000, 0.0), (8, 4, 128, 200, 3000, 0.0), (16, 8, 256, 96, 3001, 0.0),
                                                       (8, 4, 128, 200, 3000, 30.0), (32, 16, 128, 64, 2500, 0.0)])
def test_attn_window_of_a_large_decode_batch(built_lib, H, nkv, hd, B, prefix, softcap):
    """Tiles of 128 rows of many requests at different positions, whose windows reach into the prefix or not; the pages
    in front of every window are gone. All of these go the way of the prefix by whole-batch tiles of the 128-row
    kernel, the own keys by the 16-row kernel and a merge."""
    import torch
    rng = np.random.default_rng(B + hd)
    own = rng.integers(1, 120, B)
    own[::7] = rng.integers(1000, 1400, len(own[::7]))  # around the window
    own[3:6], own[-1] = [1023, 1024, 1025], 1400
    b = Batch(H, nkv, hd, 16, prefix, own, [1] * B, seed=hd, window=1024, softcap=softcap)
    tab, table = b.ptab.copy(), b.table.copy()
    b.ptab[:(prefix - 1024 + 1) // 16] = -1
    for i in range(B):
        b.table[i, :max(0, int(own[i]) - 1024) // 16] = 10 ** 6
    got = b.call()
    b.ptab, b.table = tab, table
    assert torch.isfinite(got).all()
    b.check(got, rows=sorted({0, 3, 4, 5, 7, 63, 64, B - 1} | set(rng.choice(B, 12, replace=False).tolist())))


@pytest.mark.parametrize("H,nkv,hd,B,prefix", [(4, 2, 64, 2, 600), (4, 2, 256, 3, 600), (8, 4, 64, 200, 3000), (32, 16, 128, 64, 2500)])
def test_attn_rows_of_no_request_widen_no_window(built_lib, H, nkv, hd, B, prefix):
    """Rows before the first and behind the last request, with stale positions, share the tiles of the others: what
    they would see of the prefix is not looked at."""
    import torch
    own = np.random.default_rng(B).integers(1, 40, B)
    own[-1] = min(1400, 7 * B)
    window = 50 if B < 10 else 1024
    b = Batch(H, nkv, hd, 16, prefix, own, [1] * B, seed=hd, window=window, lead=1, pad_rows=2)
    assert (b.pos[[0, -2, -1]] == 5).all()
    tab = b.ptab.copy()
    for page in (None, -1):  # NaN in the slots, then pages that are gone, in front of every window
        if page is not None:
            b.ptab[:(prefix - window + 1) // 16] = page
        got = b.call()
        saved, b.ptab = b.ptab, tab
        b.check(got, rows=sorted({1, 2, B // 2, B}))
        assert torch.isfinite(got).all() and (got[[0, -2, -1]] == 7.0).all()
        b.ptab = saved


# ------------------------------------------------------------------------------ sampling
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("min_p", [1e-12, 1e-14, 1e-20, 1e-37])
def test_min_p_below_the_weights_resolution(built_lib, dtype, min_p):
    """exp((x - M) / T) >= min_p down to where the weights of 44 bits are all zero."""
    import torch
    rng = np.random.default_rng(3)
    x = np.stack([np.linspace(-130, 4, 5001), rng.permutation(np.linspace(-130, 4, 5001)), rng.standard_normal(5001) * 30,
                  np.where(np.arange(5001) % 3, -np.inf, np.linspace(-100, 100, 5001))]).astype(np.float32)
    run_sample(x, [0.2, 0.9, 0.5, 0.7], [1.0, 1.3, 0.7, 2.5], 0, 0.0, min_p, getattr(torch, dtype))
    run_sample(x, [0.2, 0.9, 0.5, 0.7], [1.0, 1.3, 0.7, 2.5], [0, 4000, 30, 0], [0.9999, 0.0, 0.0, 0.5], min_p, getattr(torch, dtype))


@pytest.mark.parametrize("min_p", [0.3, 0.5, 0.77, 0.9])
def test_min_p_between_neighbouring_logits(built_lib, min_p):
    """Thousands of neighbouring fp32 logits on both sides of M + T ln(min_p): the kept ones are those above it,
    whatever the roundings of their weights."""
    import torch
    rng = np.random.default_rng(int(min_p * 100))
    rows = []
    for M in (0.0, 0.25, 1.0):
        at = np.float32(M + np.log(np.float64(np.float32(min_p))))
        near = (at.view(np.int32) + np.arange(-3000, 3000, dtype=np.int32)).view(np.float32)
        rows.append(np.concatenate([rng.permutation(near), np.float32([M])]))
    run_sample(np.stack(rows), [0.25, 0.5, 0.75], 1.0, 0, 0.0, min_p, torch.float32)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_min_p_around_zero_logits(built_lib, dtype):
    """The least kept logit is a zero, of either sign."""
    import torch
    x = np.zeros((6, 300), np.float32)
    x[:, ::2] = -0.0
    x[:, 100:200] = -1e-3
    x[1, 7] = x[4, 7] = np.log(4.0)
    x[2:4, 150] = 1e-38
    x[3, 151] = -1e-38
    run_sample(x, [0.1, 0.2, 0.5, 0.6, 0.9, 0.99], [1.0, 1.0, 1e-3, 1e-3, 2.0, 1e-5], 0, 0.0, [1.0, 0.25, 1.0, 0.5, 0.5, 1.0],
               getattr(torch, dtype))

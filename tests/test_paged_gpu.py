"""The paged batch-decode operators (hyb_paged_plan, hyb_qkv_post_paged, hyb_sdpa_shared_prefix,
hyb_sample_batch) against plain 64-bit implementations, and a serving step of all four.

Roundings counted by the tolerances: bf16 half a step is 2^-8 of the value, fp32 2^-24.
"""
import numpy as np
import pytest

from tests.conftest import has_gpu

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not has_gpu(), reason="no CUDA device")]

BF = 2.0 ** -8   # half a bf16 step, relative
F32 = 2.0 ** -24


@pytest.fixture(autouse=True)
def _no_timeouts(built_lib):
    import ctypes

    import hyperion_b200 as hb
    yield
    n = ctypes.c_int64()
    hb.check(built_lib.hyb_wait_timeouts(ctypes.byref(n)))
    assert n.value == 0


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ---------------------------------------------------------------------------------- plan
def plan_ref(cached, new, free, table, n_pages, page, max_rows, pos0):
    """The documented rules, one request after the other."""
    n, width = table.shape
    table = table.copy()
    row_req, row_pos, slots = (np.full(max_rows, -1, np.int64) for _ in range(3))
    start, total, taken, refused, bad, at, short = [0], [], 0, 0, 0, 0, False
    for b in range(n):
        c, a = int(cached[b]), int(new[b])
        if c < 0 or a < 0:
            refused += 1
            total.append(max(c, 0))
            start.append(min(at, max_rows))
            continue
        have, want = -(-c // page), -(-(c + a) // page)
        ok = c + a <= width * page and at + a <= max_rows
        if ok and want > have and (short or taken + want - have > len(free)):
            ok, short = False, True
        if not ok and min(at, max_rows) + a <= max_rows and a == 0 and c <= width * page:
            ok = True  # nothing to place
        if ok:
            if a and c % page:
                bad += not 0 <= table[b, c // page] < n_pages
            table[b, have:want] = free[taken:taken + want - have]
            bad += int(((free[taken:taken + want - have] < 0) | (free[taken:taken + want - have] >= n_pages)).sum())
            taken += want - have
        refused += not ok
        total.append(c + a if ok else c)
        for i in range(a):
            r = at + i
            if r >= max_rows:
                break
            row_req[r], row_pos[r] = b, pos0 + c + i
            if ok:
                pg = table[b, (c + i) // page]
                if 0 <= pg < n_pages:
                    slots[r] = pg * page + (c + i) % page
        at += a
        start.append(min(at, max_rows))
    return dict(table=table, row_start=start, row_req=row_req, row_pos=row_pos, slot_map=slots, total_lens=total,
                status=[taken, min(at, max_rows), refused, bad])


def run_plan(cached, new, free, table, n_pages, page, max_rows, pos0=0):
    from hyperion_b200 import ops
    t = dev(table.astype(np.int32))
    args = (dev(np.int32(cached)), dev(np.int32(new)), dev(np.int32(free)), t, n_pages, page, max_rows, pos0)
    plan = ops.paged_plan(*args)
    got = {k: getattr(plan, k).cpu().numpy() for k in ("row_start", "row_req", "row_pos", "slot_map", "total_lens", "status")}
    got["table"] = t.cpu().numpy()
    again = ops.paged_plan(*args, plan=plan)  # the same lengths once more: the same tables
    assert again is plan
    for k in ("row_start", "row_req", "row_pos", "slot_map", "total_lens", "status"):
        assert np.array_equal(getattr(plan, k).cpu().numpy(), got[k])
    assert np.array_equal(t.cpu().numpy(), got["table"])
    want = plan_ref(np.int64(cached), np.int64(new), np.int64(free), table, n_pages, page, max_rows, pos0)
    for k, v in want.items():
        assert np.array_equal(got[k], np.asarray(v)), (k, got[k], v)
    return got


@pytest.mark.parametrize("n,page,c_hi,a_hi,pos0", [(1, 16, 0, 1, 0), (3, 1, 5, 4, 7), (64, 16, 300, 1, 4097), (65, 64, 500, 9, 0),
                                                   (1025, 32, 100, 40, 100), (8192, 16, 40, 3, 0), (7, 48, 1000, 5000, 0)])
def test_plan(built_lib, n, page, c_hi, a_hi, pos0):
    rng = np.random.default_rng(n * page + a_hi)
    cached, new = rng.integers(0, c_hi + 1, n), rng.integers(0, a_hi + 1, n)
    cached[: n // 8] = cached[: n // 8] // page * page  # full last pages
    have = -(-cached // page)
    width = -(-(c_hi + a_hi) // page) + 2
    n_pages = int((-(-(cached + new) // page)).sum()) + 5
    perm = rng.permutation(n_pages)
    table = rng.integers(-5, n_pages + 5, (n, width))  # stale entries behind the held ones
    at = 0
    for b in range(n):
        table[b, :have[b]] = perm[at:at + have[b]]
        at += have[b]
    run_plan(cached, new, perm[at:], table, n_pages, page, int(new.sum()) + 3, pos0)


@pytest.mark.parametrize("case", ["negative", "table", "rows", "free", "free_none", "bad_free", "bad_old", "huge"])
def test_plan_refused_requests(built_lib, case):
    page, n_pages, width = 16, 64, 4
    cached = np.array([5, 16, 0, 31, 20, 7])
    new = np.array([3, 1, 20, 1, 0, 30])
    table = np.arange(24).reshape(6, 4)
    free, max_rows = np.arange(30, 50), 80
    if case == "negative":
        cached[1], new[2] = -3, -1
    if case == "table":
        new[2], cached[4] = 65, 70
    if case == "rows":
        max_rows = 24  # request 2 ends on the border, request 3 is past it
    if case == "free":
        free = free[:2]
    if case == "free_none":
        free = free[:0]
    if case == "bad_free":
        free[0], free[2] = 64, -1
    if case == "bad_old":
        table[0, 0], table[3, 1] = 64, -2
    if case == "huge":
        new[1], new[3], cached[5] = 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 2
    got = run_plan(cached, new, free, table, n_pages, page, max_rows)
    assert got["status"][2] > 0 or case.startswith("bad")


# -------------------------------------------------------------------------------- append
@pytest.mark.parametrize("H,nkv,hd,v_from_k,T,pad", [(4, 2, 64, False, 1, 0), (4, 1, 128, True, 5, 8), (16, 8, 256, False, 33, 0),
                                                     (5, 5, 64, True, 17, 64), (33, 3, 128, False, 9, 0), (1, 1, 256, False, 130, 24)])
def test_qkv_post_paged(built_lib, H, nkv, hd, v_from_k, T, pad):
    import torch
    from hyperion_b200 import ops
    rng = np.random.default_rng(H * hd + T)
    cols = (H + (1 if v_from_k else 2) * nkv) * hd
    g = torch.Generator().manual_seed(T)
    wide = torch.randn(T, cols + pad, generator=g) * 3
    wide[T // 2] = 0  # a row of zeros: eps decides
    wide = wide.bfloat16().cuda()
    x = wide[:, :cols]
    qn, kn = (torch.randn(hd, generator=g).bfloat16().cuda() for _ in range(2))
    inv = dev((10000.0 ** (-np.arange(0, hd, 2) / hd)).astype(np.float32))
    inv[-3:] = 0  # identity pairs
    n_pages, page = T // 16 + 3, 16
    slots = rng.permutation(n_pages * page)[:T].astype(np.int32)
    pos = rng.integers(0, 2 ** 20, T).astype(np.int32)
    pos[0] = 0
    if T > 4:
        pos[1], slots[2], slots[3], pos[T - 1] = -1, -1, n_pages * page, 2 ** 31 - 1
    k = torch.randn(n_pages, page, nkv, hd, generator=g).bfloat16().cuda()
    v = torch.randn(n_pages, page, nkv, hd, generator=g).bfloat16().cuda()
    k0, v0 = k.clone(), v.clone()
    q = torch.full((T, H, hd), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.qkv_post_paged(x, H, nkv, hd, v_from_k, qn, kn, inv, dev(pos), dev(slots), k, v, q_out=q)
    # 64-bit reference
    xd = x.cpu().double().numpy().reshape(T, -1, hd)
    unit = xd / np.sqrt((xd ** 2).mean(-1, keepdims=True) + np.float64(np.float32(1e-6)))
    ang = pos.astype(np.float64)[:, None] * inv.cpu().numpy().astype(np.float64)[None]
    cs, sn = np.cos(ang)[:, None], np.sin(ang)[:, None]

    def turned(h, w):
        h = h * w.cpu().double().numpy()
        a, b = h[..., : hd // 2], h[..., hd // 2:]
        size = np.tile(np.abs(a) + np.abs(b), 2)
        return np.concatenate([a * cs - b * sn, a * sn + b * cs], -1), size

    # fp32: the sum of squares (hd/16 + 5 additions deep, halved by the root), rsqrtf 2 steps, three
    # products, one addition; the angle: its float (pi * 2^-24) and sincospif (2 steps): below
    # 32 roundings of 2^-24 of |a| + |b|; then one bf16 rounding
    def close(got, want, size):
        got = got.cpu().double().numpy()
        assert (np.abs(got - want) <= BF * np.abs(want) + 32 * F32 * size + 1e-30).all()

    live = pos >= 0
    wq, sq = turned(unit[:, :H], qn)
    wk, sk = turned(unit[:, H:H + nkv], kn)
    wv = unit[:, H:H + nkv] if v_from_k else unit[:, H + nkv:H + 2 * nkv]
    close(q[torch.from_numpy(live).cuda()], wq[live], sq[live])
    assert (q[torch.from_numpy(~live).cuda()] == 7.0).all()
    kept = live & (slots >= 0) & (slots < n_pages * page)
    at = torch.from_numpy(slots[kept].astype(np.int64)).cuda()
    close(k.view(-1, nkv, hd)[at], wk[kept], sk[kept])
    close(v.view(-1, nkv, hd)[at], wv[kept], np.abs(wv[kept]))
    rest = torch.ones(n_pages * page, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert torch.equal(k.view(-1, nkv, hd)[rest], k0.view(-1, nkv, hd)[rest])
    assert torch.equal(v.view(-1, nkv, hd)[rest], v0.view(-1, nkv, hd)[rest])


# ----------------------------------------------------------------------------- attention
class Batch:
    """A random batch; the pools hold NaN wherever no row looks."""

    def __init__(self, H, nkv, hd, page, prefix, own, q_lens, seed=0, window=0, softcap=0.0, scale=None, pad_rows=0, lead=0,
                 positions=None):
        import torch
        rng = np.random.default_rng(seed)
        self.H, self.nkv, self.hd, self.page, self.prefix = H, nkv, hd, page, prefix
        self.window, self.softcap = window, softcap
        self.scale = hd ** -0.5 if scale is None else scale
        self.own = np.array(own, np.int32)
        self.q_lens = np.array(q_lens, np.int32)
        n = len(own)
        self.start = (lead + np.concatenate([[0], np.cumsum(self.q_lens)])).astype(np.int32)
        self.T = int(self.start[-1]) + pad_rows
        self.pos = np.full(self.T, 5, np.int32)
        for b in range(n):
            for i in range(q_lens[b]):
                self.pos[self.start[b] + i] = max(0, prefix + own[b] - q_lens[b] + i)
        if positions is not None:
            self.pos[:] = positions
        pb = -(-prefix // page)
        blocks = [-(-max(0, int(o)) // page) for o in own]
        self.n_pages = pb + sum(blocks) + 2
        perm = rng.permutation(self.n_pages).astype(np.int32)
        self.ptab = perm[:pb]
        self.width = max(blocks + [1]) + 1
        self.table = np.full((n, self.width), 10 ** 9, np.int32)
        at = pb
        for b in range(n):
            self.table[b, :blocks[b]] = perm[at:at + blocks[b]]
            at += blocks[b]
        shape = (self.n_pages, page, nkv, hd)
        g = torch.Generator().manual_seed(seed)
        self.k, self.v = torch.randn(shape, generator=g).bfloat16(), torch.randn(shape, generator=g).bfloat16()
        self.q = torch.randn(self.T, H, hd, generator=g).bfloat16()
        # what no row sees holds NaN
        seen = np.zeros(self.n_pages * page, bool)
        for t, b, keys, slots in self.rows():
            seen[slots] = True
        for x in (self.k, self.v):
            x.view(-1, nkv, hd)[torch.from_numpy(~seen)] = float("nan")

    def rows(self):
        """(row, request, visible key positions, their slots) of every row of a request."""
        pj = np.arange(self.prefix)
        pslot = self.ptab[pj // self.page].astype(np.int64) * self.page + pj % self.page if self.prefix else np.zeros(0, np.int64)
        for b in range(len(self.own)):
            j = np.arange(max(0, self.own[b]))
            oslot = self.table[b, j // self.page].astype(np.int64) * self.page + j % self.page
            key, slot = np.concatenate([pj, self.prefix + j]), np.concatenate([pslot, oslot])
            for t in range(self.start[b], self.start[b + 1]):
                ok = key <= self.pos[t]
                if self.window:
                    ok &= key > int(self.pos[t]) - self.window
                yield t, b, key[ok], slot[ok]

    def call(self, max_q=None, max_own=None, **kw):
        import torch
        from hyperion_b200 import ops
        out = kw.pop("out", None)
        if out is None:
            out = torch.full((self.T, self.H, self.hd), 7.0, dtype=torch.bfloat16, device="cuda")
        ops.sdpa_shared_prefix(self.q.cuda(), self.k.cuda(), self.v.cuda(), dev(self.ptab) if self.prefix else None, self.prefix,
                               dev(self.table), dev(self.own), dev(self.start), dev(self.pos),
                               max(1, int(self.q_lens.max())) if max_q is None else max_q,
                               max(0, int(self.own.max())) if max_own is None else max_own, window=self.window, scale=self.scale,
                               softcap=self.softcap, out=out, **kw)
        return out

    def check(self, got, rows=None):
        import torch
        got = got.cpu().double().numpy()
        G = self.H // self.nkv
        k, v = (x.view(-1, self.nkv, self.hd).double().numpy() for x in (self.k, self.v))
        q = self.q.double().numpy()
        touched = np.zeros(self.T, bool)
        for t, b, keys, slots in self.rows():
            touched[t] = True
            if rows is not None and t not in rows:
                continue
            if len(keys) == 0:
                assert (got[t] == 0).all()
                continue
            kk, vv = np.repeat(k[slots], G, 1), np.repeat(v[slots], G, 1)
            dot = np.einsum("hd,jhd->hj", q[t], kk)
            mag = np.einsum("hd,jhd->hj", np.abs(q[t]), np.abs(kk)).max(1)
            s = dot * self.scale
            if self.softcap:
                s = self.softcap * np.tanh(s / self.softcap)
            w = np.exp(s - s.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            o, A = np.einsum("hj,jhd->hd", w, vv), np.einsum("hj,jhd->hd", w, np.abs(vv))
            # a probability is off by its bf16 rounding, by its score's error (an fp32 dot product of
            # hd terms, and the few roundings of scale, softcap and maximum: hd + 16 roundings of the
            # terms' magnitude) and by ex2 (2^-22); the sums add the roundings of a few
            # hundred fp32 additions (tile by tile); o moves by that share of sum w |v - o| <= A + |o|
            eps = BF + (self.hd + 16) * F32 * mag[:, None] * abs(self.scale) + 2.0 ** -22 + 512 * F32
            tol = BF * np.abs(o) + eps * (A + np.abs(o)) * (1 + 4 * BF)
            err = np.abs(got[t] - o)
            assert (err <= tol).all(), (t, b, float((err / tol).max()))
        if rows is None:
            assert (got[~touched] == 7.0).all()


GEOM = [(4, 2, 64), (4, 1, 128), (16, 8, 256), (3, 3, 64), (16, 1, 128), (33, 1, 64), (24, 2, 256)]


@pytest.mark.parametrize("H,nkv,hd", GEOM)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_attn_decode(built_lib, H, nkv, hd, page):
    b = Batch(H, nkv, hd, page, 75, [1, 16, 17, 63, 64, 65, 200, 333], [1] * 8, seed=H + page)
    b.check(b.call())


@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 63, 64, 127, 128, 129, 1000])
def test_attn_prefix_lengths(built_lib, prefix, page):
    b = Batch(4, 2, 128, page, prefix, [1, 2, 40], [1, 1, 1], seed=prefix)
    b.check(b.call())


@pytest.mark.parametrize("H,nkv,hd", GEOM)
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_attn_ragged_rows(built_lib, H, nkv, hd, softcap):
    b = Batch(H, nkv, hd, 32, 130, [9, 0, 3, 70, 100, 31], [9, 0, 3, 1, 64, 17], seed=hd + H, softcap=softcap, pad_rows=5, lead=2)
    b.check(b.call())


@pytest.mark.parametrize("window", [1, 7, 64, 100, 5000])
@pytest.mark.parametrize("hd,q", [(64, 1), (128, 5), (256, 40)])
def test_attn_window(built_lib, window, hd, q):
    b = Batch(4, 2, hd, 16, 333, [q, q + 1, 64 + q, 150 + q], [q] * 4, seed=window + q, window=window)
    b.check(b.call())


@pytest.mark.parametrize("hd,B", [(64, 40), (128, 64), (256, 70)])
def test_attn_many_rows_long_prefix(built_lib, hd, B):
    rng = np.random.default_rng(B)
    b = Batch(8, 4, hd, 64, 2050, rng.integers(1, 90, B), [1] * B, seed=B)
    b.check(b.call())


@pytest.mark.parametrize("hd", [64, 256])
def test_attn_prefill_rows(built_lib, hd):
    b = Batch(8, 2, hd, 64, 517, [150, 200, 1], [150, 133, 1], seed=hd)
    b.check(b.call(), rows=[0, 1, 31, 32, 63, 64, 149, 150, 250, 282, 283])


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attn_many_blocks(built_lib, hd):
    """Hundreds of key blocks in one pass, with and without parts, and several tiles per SM."""
    b = Batch(16, 8, hd, 128, 3001, [64] * 40, [64] * 40, seed=hd)  # 320 tiles, one part each
    b.check(b.call(), rows=[0, 63, 64, 1281, 2559])
    b = Batch(4, 2, hd, 64, 20011, [80, 100], [64, 64], seed=hd + 1)  # few tiles, many parts
    b.check(b.call(), rows=[0, 1, 63, 64, 127])
    b = Batch(150, 150, hd, 256, 6000, [64], [64], seed=hd + 2)  # 150 heads: one long part each
    b.check(b.call(), rows=[0, 63])


@pytest.mark.parametrize("n,window", [(300, 0), (1024, 0), (257, 20)])
@pytest.mark.parametrize("prefix", [0, 70, 700])
def test_attn_many_requests(built_lib, n, window, prefix):
    """Requests without rows, without keys, with one key and with hundreds, in shares that cross them."""
    rng = np.random.default_rng(n + prefix)
    own = rng.choice([0, 0, 1, 5, 16, 17, 40, 300], n)
    q = np.where(rng.random(n) < 0.2, 0, 1 + (rng.random(n) < 0.1))
    q[:3], own[:3] = 0, 50
    b = Batch(4, 2, 64, 16, prefix, own, q, seed=n, window=window, pad_rows=2)
    got = b.call()
    b.check(got, rows=sorted(rng.choice(b.T - 2, 60, replace=False).tolist()) + [b.T - 3])
    assert (got[-2:] == 7.0).all()


def test_attn_scores_far_apart(built_lib):
    """Scores of some hundreds, growing along the keys (every tile moves the maximum) and falling."""
    for order in (1, -1):
        b = Batch(4, 2, 128, 32, 700, [40, 3], [1, 1], seed=5, scale=1.0)
        ramp = np.linspace(0.1, 3.0, 700)[::order].copy()
        import torch
        slots = b.ptab[np.arange(700) // 32].astype(np.int64) * 32 + np.arange(700) % 32
        flat = b.k.view(-1, 2, 128)
        flat[torch.from_numpy(slots)] = (flat[torch.from_numpy(slots)].float() * torch.from_numpy(ramp)[:, None, None]).bfloat16()
        b.check(b.call())


def test_attn_rows_without_keys(built_lib):
    b = Batch(4, 2, 64, 16, 0, [0, 5, -4, 3], [1, 2, 1, 3], seed=1)
    got = b.call(max_own=5)
    b.check(got)
    # a window that ends before the first key of the request
    b = Batch(4, 2, 64, 16, 0, [4, 4], [1, 1], seed=2, window=3, positions=[20, 3])
    b.check(b.call())
    # nothing anywhere
    b = Batch(4, 2, 256, 16, 0, [0, 0], [1, 1], seed=3)
    b.check(b.call(max_own=0))


def test_attn_padding_rows_stay(built_lib):
    import torch
    b = Batch(4, 2, 128, 16, 40, [8, 9, 10], [2, 2, 2], seed=4)
    b.pos[3] = -1
    got = b.call()
    assert (got[3] == 7.0).all()
    b.check(got, rows=[0, 1, 2, 4, 5])
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("q", [1, 40])
def test_attn_broken_bounds_are_nan(built_lib, q):
    import torch
    b = Batch(4, 2, 64, 16, 20, [50, 60, 70], [q, q, q], seed=6)
    got = b.call(max_own=60)  # request 2 has more keys than the bound
    assert torch.isnan(got[2 * q:]).all()
    b.check(got, rows=list(range(2 * q)))
    b.own[1] = b.width * 16 + 1  # more keys than its table holds
    got = b.call(max_own=10 ** 6)
    assert torch.isnan(got[q:2 * q]).all()
    if q > 1:
        b = Batch(4, 2, 64, 16, 20, [50, 60], [3, 5], seed=7)
        got = b.call(max_q=4)
        assert torch.isnan(got[7]).all()
        b.check(got, rows=range(7))


@pytest.mark.parametrize("B,q", [(3, 1), (40, 1), (2, 70)])
@pytest.mark.parametrize("page_id", [-1, 10 ** 6])
def test_attn_bad_pages_are_nan(built_lib, B, q, page_id):
    import torch
    b = Batch(4, 2, 64, 16, 100, [80] * B, [q] * B, seed=8)
    b.table[1, 2] = page_id
    got = b.call()
    assert torch.isnan(got[q:2 * q]).all() if q == 1 else torch.isnan(got[2 * q - 1]).all()
    assert torch.isfinite(got[:q]).all()
    b = Batch(4, 2, 64, 16, 100, [80] * B, [q] * B, seed=8)
    b.ptab[3] = page_id
    assert torch.isnan(b.call()).all()


def test_attn_slots_past_32_bits(built_lib):
    """Element offsets of the last pages beyond 2^32 (a pool of 9 GB per side)."""
    import torch
    from hyperion_b200 import ops
    nkv, hd, page = 8, 256, 64
    n_pages = 2 ** 32 // (page * nkv * hd) + 40
    k = torch.zeros(n_pages, page, nkv, hd, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(n_pages, page, nkv, hd, dtype=torch.bfloat16, device="cuda")
    for B in (2, 40):
        b = Batch(16, nkv, hd, page, 200, [70] * B, [1] * B, seed=9)
        far = n_pages - 1 - np.arange(b.n_pages) if b.n_pages <= 38 else np.concatenate(
            [n_pages - 1 - np.arange(38), 100 + np.arange(b.n_pages - 38)])
        at = torch.from_numpy(far.astype(np.int64)).cuda()
        k[at], v[at] = b.k.cuda(), b.v.cuda()
        table = np.where(b.table < b.n_pages, far[np.minimum(b.table, b.n_pages - 1)], 0).astype(np.int32)
        got = ops.sdpa_shared_prefix(b.q.cuda(), k, v, dev(far[b.ptab].astype(np.int32)), 200, dev(table), dev(b.own), dev(b.start),
                                     dev(b.pos), 1, 70, scale=b.scale)
        b.check(got, rows=[0, 1, B - 1])
    # and the cache write
    slot = n_pages * page - 3
    qkv = torch.randn(1, (16 + 16) * hd, device="cuda").bfloat16()
    one = torch.ones(hd, dtype=torch.bfloat16, device="cuda")
    ops.qkv_post_paged(qkv, 16, nkv, hd, False, one, one, torch.zeros(hd // 2, device="cuda"), dev(np.int32([3])),
                       dev(np.int32([slot])), k, v)
    want = qkv.float().view(32, hd)[24:]
    want = want * torch.rsqrt((want * want).mean(-1, keepdim=True) + 1e-6)
    assert torch.allclose(v.view(-1, nkv, hd)[slot].float(), want, rtol=2 * BF, atol=0)


# ------------------------------------------------------------------------------ sampling
def sample_ref(x, u, t, k, p, mp):
    """(token, kept, prob, distance of the draw from the nearest border, distance of the cuts)."""
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    V = len(x)
    if x.max() == -np.inf:
        return -1, 0, 0.0
    if not t > 0:
        return int(np.argmax(x)), 1, 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / np.float64(t)))
    order = np.argsort(-x, kind="stable")
    m = V
    if 0 < p < 1:
        cum = np.cumsum(w[order])
        m = min(m, int(np.searchsorted(cum, np.float64(p) * cum[-1], side="left")) + 1)
    if mp > 0:
        m = min(m, int((w >= min(np.float64(mp), 1.0)).sum()))
    if k > 0:
        m = min(m, int(k))
    ids = np.sort(order[:m])
    cum = np.cumsum(w[ids])
    at = int(np.searchsorted(cum, np.float64(u) * cum[-1], side="right"))
    if at >= m:
        at = int(np.nonzero(w[ids])[0][-1])
    return int(ids[at]), m, w[ids[at]] / cum[-1]


def run_sample(x, u, t, k, p, mp, dtype, pad=0, offset=0):
    import torch
    from hyperion_b200 import ops
    n, V = x.shape
    flat = torch.full((offset + n * (V + pad),), float("inf"), dtype=dtype, device="cuda")
    view = torch.as_strided(flat, (n, V), (V + pad, 1), offset)
    view.copy_(torch.from_numpy(x))
    f = lambda a, ty: dev(np.broadcast_to(np.asarray(a, ty), (n,)))  # noqa: E731
    tok, kept, prob = ops.sample_batch(view, f(u, np.float32), f(t, np.float32), f(k, np.int32), f(p, np.float32), f(mp, np.float32))
    vals = view.float().cpu().numpy()
    tok, kept, prob = tok.cpu().numpy(), kept.cpu().numpy(), prob.cpu().numpy()
    B = lambda a, i: np.broadcast_to(np.asarray(a), (n,))[i]  # noqa: E731
    for i in range(n):
        want = sample_ref(vals[i], np.float32(B(u, i)), np.float32(B(t, i)), B(k, i), np.float32(B(p, i)), np.float32(B(mp, i)))
        assert (tok[i], kept[i]) == want[:2], (i, tok[i], kept[i], want)
        # a weight is an integer of 2^-44 of the largest (half a unit: 2^-45 absolute over a sum
        # >= 1), and the share is rounded to fp32 once
        assert abs(prob[i] - want[2]) <= 2 * F32 * want[2] + 2.0 ** -44
    return tok, kept, prob


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("V", [1, 2, 31, 100, 4096, 8191, 32003, 100001, 262144])
def test_sample_batch(built_lib, V, dtype):
    import torch
    rng = np.random.default_rng(V)
    n = 12
    x = 30 * np.tanh(rng.standard_normal((n, V)).astype(np.float32) * 0.1)
    x[:, rng.integers(0, V, max(0, min(3, V - 1)))] = -np.inf
    t = np.resize([0.8, 1.0, 0.0, 1.7, 0.3, 1.0], n)
    k = np.resize([40, 0, 0, 7, 1000000, 1, 2], n)
    p = np.resize([0.95, 0.0, 0.5, 0.999, 1.0, 0.1, 0.7], n)
    mp = np.resize([0.0, 0.0, 0.2, 0.01], n)
    run_sample(x, rng.random(n, dtype=np.float32), t, k, p, mp, getattr(torch, dtype), pad=5 if V % 2 else 0, offset=1 if V == 8191 else 0)


def test_sample_batch_largest_vocabulary(built_lib):
    import torch
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, 1 << 19)).astype(np.float32) * 2
    for dtype in (torch.bfloat16, torch.float32):
        run_sample(x, [0.3, 0.9999], [1.0, 0.7], [0, 500], [0.9, 0.0], 0.0, dtype)


def test_sample_batch_many_rows(built_lib):
    import torch
    rng = np.random.default_rng(4)
    x = rng.standard_normal((700, 1000)).astype(np.float32) * 3
    run_sample(x, rng.random(700, dtype=np.float32), rng.random(700), rng.integers(0, 50, 700), rng.random(700), 0.0, torch.bfloat16)


@pytest.mark.parametrize("V", [7, 5000, 70000])
def test_sample_batch_edges(built_lib, V):
    import torch
    rng = np.random.default_rng(V)
    x = rng.standard_normal((12, V)).astype(np.float32)
    x[0] = -np.inf                       # nothing to draw from
    x[1] = np.nan
    x[2] = 1.25                          # all tied
    x[3] = np.where(np.arange(V) % 2, 0.0, -0.0)  # both zeros are equal
    x[4, : V // 2] = np.nan              # NaN counts as -inf
    x[5] = -np.inf
    x[5, V - 1] = -3.0                   # one finite logit
    x[6] = 2.0
    x[6, 3] = 2.5
    x[7] = np.linspace(-300, 300, V)     # most weights vanish
    x[8, [1, V - 2]] = np.inf            # +inf shares all the weight
    u = np.float32([0.5, 0.5, 0.37, 0.999, 0.1, 0.9, 0.6, 0.5, 0.75, 0.0, 1 - 2 ** -24, 0.5])
    for t, k, p, mp in [(1.0, 0, 0.0, 0.0), (1.0, 3, 0.0, 0.0), (0.7, 0, 0.5, 0.0), (1.0, 0, 0.0, 1.0), (0.5, 5, 0.9, 0.3),
                        (0.0, 0, 0.0, 0.0), (100.0, V - 1, 0.99, 0.0), (1e-3, 4, 0.5, 0.1)]:
        run_sample(x, u, t, k, p, mp, torch.float32)
        run_sample(x, u, t, k, p, mp, torch.bfloat16)


@pytest.mark.parametrize("V,offset", [(131072, 0), (131063, 3)])
def test_sample_batch_values_that_repeat(built_lib, V, offset):
    """A value that fills a whole slice of the row, and ones that fill halves and quarters of it."""
    import torch
    rng = np.random.default_rng(V)
    x = rng.standard_normal((80, V)).astype(np.float32)
    x[0] = 0.5
    x[1] = -2.0
    x[1, 7] = 1.0
    x[2] = np.where(np.arange(V) % 2, 3.0, 2.0)
    x[3] = np.where(np.arange(V) < 70000, 1.5, -1.5)
    x[4] = np.where(np.arange(V) % 4, 0.0, -0.0)
    x[5] = np.repeat(np.float32([1, 2, 3, 4]), V // 4 + 1)[:V]
    x[6, : V // 2] = -np.inf
    x[7, 5000:] = np.nan
    t = np.resize([1.0, 0.6, 0.0], 80)
    k = np.resize([0, 50000, 0, 100000, 3], 80)
    p = np.resize([0.0, 0.9, 0.0, 0.5], 80)
    mp = np.resize([0.0, 0.0, 0.0, 0.0, 0.0, 0.3], 80)
    run_sample(x, rng.random(80, dtype=np.float32), t, k, p, mp, torch.bfloat16, pad=offset, offset=offset)
    run_sample(x[:8], rng.random(8, dtype=np.float32), 1.0, 0, 0.7, 0.0, torch.bfloat16)


def test_sample_batch_defaults_and_strange_settings(built_lib):
    import torch
    from hyperion_b200 import ops
    x = torch.randn(4, 500, device="cuda")
    u = torch.tensor([float("nan"), -1.0, 2.0, 0.5], device="cuda")
    tok, kept, prob = ops.sample_batch(x, u)
    xs = x.double().cpu().numpy()
    assert kept.tolist() == [500] * 4 and tok[:3].tolist() == [0, 0, 499]
    assert tok[3].item() == sample_ref(xs[3], 0.5, 1.0, 0, 0.0, 0.0)[0]
    nan = torch.full((4,), float("nan"), device="cuda")
    tok, kept, prob = ops.sample_batch(x, u, temperature=nan, top_p=nan, min_p=nan)
    assert torch.equal(tok, x.argmax(-1).int()) and kept.tolist() == [1] * 4
    tok, kept, _ = ops.sample_batch(x, u, min_p=torch.full((4,), 7.0, device="cuda"))
    assert torch.equal(tok, x.argmax(-1).int()) and kept.tolist() == [1] * 4


# ------------------------------------------------------------------------- all together
class Step:
    """One layer of a serving step: plan, append, attend, sample, on static buffers."""

    def __init__(self, seed=0):
        import torch
        from hyperion_b200 import ops
        self.H, self.nkv, self.hd, self.page, self.prefix, n = 8, 4, 128, 16, 90, 5
        g = torch.Generator().manual_seed(seed)
        self.n, self.rows, self.n_pages = n, 16, 60
        shape = (self.n_pages, self.page, self.nkv, self.hd)
        self.k, self.v = (torch.randn(shape, generator=g).bfloat16().cuda() for _ in range(2))
        perm = torch.randperm(self.n_pages, generator=g).int().cuda()
        self.ptab, self.free = perm[:6].contiguous(), perm[6:].contiguous()
        self.table = torch.zeros(n, 8, dtype=torch.int32, device="cuda")
        self.cached = torch.zeros(n, dtype=torch.int32, device="cuda")
        self.new = torch.zeros(n, dtype=torch.int32, device="cuda")
        self.qkv = torch.randn(self.rows, (self.H + 2 * self.nkv) * self.hd, generator=g).bfloat16().cuda()
        self.qn = torch.ones(self.hd, dtype=torch.bfloat16, device="cuda")
        self.inv = torch.linspace(1, 0.001, self.hd // 2, device="cuda")
        self.head = (torch.randn(self.H * self.hd, 1000, generator=g) * 0.1).cuda()
        self.u = torch.rand(self.rows, generator=g).cuda()
        self.plan = ops.PagedPlan(n, self.rows)
        self.scratch = ops.SharedPrefixScratch(self.rows, n, 8, 128, self.prefix, self.H, self.nkv, self.hd)
        self.q = torch.zeros(self.rows, self.H, self.hd, dtype=torch.bfloat16, device="cuda")
        self.out = torch.zeros_like(self.q)
        self.logits = torch.zeros(self.rows, 1000, device="cuda")
        self.drawn = (torch.zeros(self.rows, dtype=torch.int32, device="cuda"), torch.zeros(self.rows, dtype=torch.int32, device="cuda"),
                      torch.zeros(self.rows, device="cuda"))

    def __call__(self, stream=None):
        import torch
        from hyperion_b200 import ops
        p = ops.paged_plan(self.cached, self.new, self.free, self.table, self.n_pages, self.page, self.rows, pos0=self.prefix,
                           plan=self.plan, stream=stream)
        ops.qkv_post_paged(self.qkv, self.H, self.nkv, self.hd, False, self.qn, self.qn, self.inv, p.row_pos, p.slot_map, self.k,
                           self.v, q_out=self.q, stream=stream)
        ops.sdpa_shared_prefix(self.q, self.k, self.v, self.ptab, self.prefix, self.table, p.total_lens, p.row_start, p.row_pos, 8,
                               128, scale=self.hd ** -0.5, scratch=self.scratch, out=self.out, stream=stream)
        with torch.cuda.stream(stream if stream is not None else torch.cuda.current_stream()):
            torch.mm(self.out.view(self.rows, -1).float(), self.head, out=self.logits)
        ops.sample_batch(self.logits, self.u, top_k=None, out=self.drawn, stream=stream)

    def advance(self):
        taken = int(self.plan.status[0])
        assert self.plan.status[2:].tolist() == [0, 0]
        self.free.copy_(self.free.roll(-taken))
        self.cached.copy_(self.plan.total_lens)



STEPS = [[3, 0, 8, 1, 2], [1, 1, 1, 1, 1], [1, 5, 0, 8, 1], [2, 2, 2, 2, 2], [0, 0, 0, 0, 0], [1, 1, 1, 1, 1]]


def _drive(step, run):
    """Several steps; returns what each wrote, and checks it against an unpaged 64-bit run."""
    import torch
    logs = []
    hist = [dict(k=[], v=[]) for _ in range(step.n)]  # each request's own keys, unpaged
    pk = step.k[step.ptab.long()].view(-1, step.nkv, step.hd)[:step.prefix].cpu().double()
    pv = step.v[step.ptab.long()].view(-1, step.nkv, step.hd)[:step.prefix].cpu().double()
    for i, new in enumerate(STEPS):
        step.new.copy_(torch.tensor(new, dtype=torch.int32))
        step.qkv.copy_(torch.randn(step.qkv.shape, generator=torch.Generator().manual_seed(i)))
        step.out.fill_(7.0)
        run()
        torch.cuda.synchronize()
        T = int(step.plan.row_start[-1])
        assert T == sum(new)
        x = step.qkv.cpu().double().view(step.rows, -1, step.hd)
        x = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + 1e-6)
        half, r = step.hd // 2, 0
        for b in range(step.n):
            for _ in range(new[b]):
                ang = (step.prefix + len(hist[b]["k"])) * step.inv.cpu().double()
                c, s = torch.cos(ang), torch.sin(ang)
                rot = lambda h: torch.cat([h[..., :half] * c - h[..., half:] * s, h[..., :half] * s + h[..., half:] * c], -1)  # noqa: E731
                q, k, v = rot(x[r, :step.H]), rot(x[r, step.H:step.H + step.nkv]), x[r, step.H + step.nkv:]
                hist[b]["k"].append(k)
                hist[b]["v"].append(v)
                K = torch.cat([pk, torch.stack(hist[b]["k"])]).repeat_interleave(2, 1)
                V = torch.cat([pv, torch.stack(hist[b]["v"])]).repeat_interleave(2, 1)
                sc = torch.einsum("hd,jhd->hj", q, K) * step.hd ** -0.5
                w = torch.softmax(sc, -1)
                o, A = torch.einsum("hj,jhd->hd", w, V), torch.einsum("hj,jhd->hd", w, V.abs())
                # q, k and v are bf16 (a score moves by 2 * 2^-8 of its terms' magnitude, v by 2^-8),
                # the probability and the output once more
                mag = torch.einsum("hd,jhd->hj", q.abs(), K.abs()).amax(1, keepdim=True) * step.hd ** -0.5
                tol = (2 * BF * mag * 1.05 + 3 * BF) * (A + o.abs())
                assert ((step.out[r].cpu().double() - o).abs() <= tol).all(), (i, b, r)
                r += 1
        assert (step.out[T:] == 7.0).all()
        for r in range(T):
            assert step.drawn[0][r].item() == sample_ref(step.logits[r].cpu().numpy(), step.u[r].item(), 1.0, 0, 0.0, 0.0)[0]
        logs.append((step.out.clone(), step.k.clone(), step.drawn[0][:T].clone(), step.table.clone()))
        step.advance()
    return logs


def test_serving_steps(built_lib):
    """Steps of the four operators in a row: eager, on another stream, and as one captured graph
    replayed while the lengths change; all three write the same bits."""
    import torch
    first = Step()
    logs = _drive(first, first)
    side = torch.cuda.Stream()
    second = Step()
    torch.cuda.synchronize()
    logs2 = _drive(second, lambda: (side.wait_stream(torch.cuda.current_stream()), second(stream=side)))
    third = Step()
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        third()
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third()
    logs3 = _drive(third, graph.replay)
    for a, b, c in zip(logs, logs2, logs3):
        for x, y, z in zip(a, b, c):
            assert torch.equal(x, y) and torch.equal(x, z)


def test_two_graphs_share_a_workspace(built_lib):
    """Two captured attention calls of different sizes that use one scratch, replayed in turn."""
    import torch
    from hyperion_b200 import ops
    a = Batch(4, 2, 64, 16, 300, [40, 50], [1, 1], seed=1)
    b = Batch(16, 8, 256, 64, 600, [20] * 12, [3] * 12, seed=2)
    scratch = ops.SharedPrefixScratch(b.T, 12, 3, 20, 600, 16, 8, 256)
    need = ops.SharedPrefixScratch(a.T, 2, 1, 50, 300, 4, 2, 64)
    assert need.nbytes <= scratch.nbytes
    graphs, outs = [], []
    for x in (a, b):
        out = torch.full((x.T, x.H, x.hd), 7.0, dtype=torch.bfloat16, device="cuda")
        held = [x.q.cuda(), x.k.cuda(), x.v.cuda(), dev(x.ptab), dev(x.table), dev(x.own), dev(x.start), dev(x.pos)]

        def call(h=held, x=x, out=out):
            ops.sdpa_shared_prefix(h[0], h[1], h[2], h[3], x.prefix, h[4], h[5], h[6], h[7], int(x.q_lens.max()), int(x.own.max()),
                                   scale=x.scale, scratch=scratch, out=out)
        call()
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            call()
        graphs.append((gr, held))
        outs.append(out)
    for _ in range(3):
        for out in outs:
            out.fill_(7.0)
        for gr, _held in graphs:
            gr.replay()
        torch.cuda.synchronize()
        a.check(outs[0])
        b.check(outs[1])


def test_results_do_not_depend_on_the_run(built_lib):
    import torch
    b = Batch(32, 16, 128, 16, 1500, [100] * 33, [1] * 33, seed=3)
    first = b.call()
    for _ in range(3):
        assert torch.equal(first, b.call())


def test_python_checks(built_lib):
    import torch
    from hyperion_b200 import ops
    b = Batch(4, 2, 64, 16, 20, [5, 6], [1, 1], seed=1)
    args = lambda: [b.q.cuda(), b.k.cuda(), b.v.cuda(), dev(b.ptab), 20, dev(b.table), dev(b.own), dev(b.start), dev(b.pos), 1, 6]  # noqa: E731
    for i, bad in [(0, b.q), (0, b.q.cuda().float()), (0, b.q.cuda()[:1]), (3, dev(b.ptab)[:1]), (5, dev(b.table).long()),
                   (6, dev(b.own)[:1]), (7, dev(b.start)[:2]), (8, dev(b.pos).cpu()), (2, b.v.cuda()[:, :8])]:
        a = args()
        a[i] = bad
        with pytest.raises(ValueError):
            ops.sdpa_shared_prefix(*a)
    x = torch.zeros(4, 100, device="cuda")
    for kw in (dict(u=torch.zeros(3, device="cuda")), dict(u=torch.zeros(4, device="cuda"), top_k=torch.zeros(4, device="cuda")),
               dict(u=torch.zeros(4))):
        with pytest.raises(ValueError):
            ops.sample_batch(x, **kw)
    with pytest.raises(ValueError):
        ops.sample_batch(x.t(), torch.zeros(100, device="cuda"))
    with pytest.raises(ValueError):
        ops.sample_batch(x.expand(4, 100)[:1].expand(4, 100), torch.zeros(4, device="cuda"))
    if torch.cuda.device_count() > 1:
        with pytest.raises(ValueError):
            ops.sample_batch(x, torch.zeros(4, device="cuda:1"))

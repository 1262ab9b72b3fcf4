"""Cases, plain forms and 64-bit values of the paged batch-decode operators.

A serving step over a paged KV cache whose requests share a long prompt prefix:

* ``paged_plan``          block tables, slot map and row tables from the requests' lengths;
* ``qkv_post_paged``      QK-norm, RoPE and the cache write through the slot map;
* ``sdpa_shared_prefix``  attention of every row over the shared prefix and its own pages;
* ``sample_batch``        temperature / top-k / top-p / min-p sampling from given uniforms.

With ``own`` false every operator runs in its plain form (elementary torch operations in 32
or 64 bits, rounded once); with ``own`` true the framework's entry points are called.
"""
import math

import numpy as np
import torch

own = False

# (query heads, KV heads, head_dim) of the framework's own decoders: the 12B- and 27B-shaped
# ones and the two tiny test geometries
LAYOUTS = {"12b": (16, 8, 256), "27b": (32, 16, 128), "tiny": (4, 2, 64), "tiny_global": (4, 1, 128)}
VOCAB = 262144


# ------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one decode step of 64 running requests: a row each, pages taken now and then
        dict(name="plan_step_b64", op="plan", n_req=64, new_lo=1, new_hi=1, cached_hi=8192, page=64),
        # a prefill wave: 512 requests admitted with a few hundred new tokens each
        dict(name="plan_prefill_b512", op="plan", n_req=512, new_lo=1, new_hi=1023, cached_hi=2048, page=16),
        # the rows of one decode step of the 27B-shaped decoder
        dict(name="append_step_27b", op="append", layout="27b", rows=64, page=64, v_from_k=False, far=16384),
        # one 2048-token prefill chunk of the 12B-shaped decoder
        dict(name="append_chunk_12b", op="append", layout="12b", rows=2048, page=64, v_from_k=False, far=131072),
        # the smallest call: one request of the tiny decoder, where only latency counts
        dict(name="attn_one_tiny", op="attn", layout="tiny", n_req=1, q_lo=1, q_hi=1, prefix=33, own_hi=17, page=16,
             window=0, softcap=0.0, q_rms=1.0),
        # an ordinary small batch behind a system prompt
        dict(name="attn_step_12b_b8", op="attn", layout="12b", n_req=8, q_lo=1, q_hi=1, prefix=2048, own_hi=700, page=64,
             window=0, softcap=0.0, q_rms=0.25),
        # the largest decode batch over a long shared document, ragged answers
        dict(name="attn_step_27b_b64", op="attn", layout="27b", n_req=64, q_lo=1, q_hi=1, prefix=16384, own_hi=1024,
             page=16, window=0, softcap=0.0, q_rms=0.25),
        # speculative verify rows of a sliding-window layer, odd prefix
        dict(name="attn_verify_12b_window", op="attn", layout="12b", n_req=16, q_lo=2, q_hi=9, prefix=4097, own_hi=513,
             page=32, window=1024, softcap=0.0, q_rms=0.25),
        # the users' own prompts prefilled behind the shared prefix
        dict(name="attn_prefill_12b", op="attn", layout="12b", n_req=8, q_lo=200, q_hi=300, prefix=8192, own_hi=600,
             page=128, window=0, softcap=0.0, q_rms=0.25),
        # one stream's next token over the whole vocabulary
        dict(name="sample_one", op="sample", rows=1, vocab=VOCAB, dtype="bf16", mix=False, sigma=3.0),
        # the largest decode batch, every row with settings of its own
        dict(name="sample_b64", op="sample", rows=64, vocab=VOCAB, dtype="bf16", mix=True, sigma=3.0),
        # 32-bit logits of a smaller, odd vocabulary
        dict(name="sample_f32_odd", op="sample", rows=16, vocab=32003, dtype="f32", mix=True, sigma=3.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attn", "attn", "attn", "sample", "sample"])
    if op == "plan":
        hi = _log(rng, 1, 1023)
        return dict(op=op, n_req=_log(rng, 1, 512), new_lo=rng.choice([0, 1]), new_hi=hi, cached_hi=_log(rng, 1, 8192),
                    page=rng.choice([16, 32, 64, 128, 256]))
    if op == "append":
        return dict(op=op, layout=rng.choice(sorted(LAYOUTS)), rows=_log(rng, 1, 2048), page=rng.choice([16, 32, 64, 128, 256]),
                    v_from_k=rng.choice([False, True]), far=_log(rng, 64, 131072))
    if op == "sample":
        dtype = rng.choice(["bf16", "f32"])
        return dict(op=op, rows=_log(rng, 1, 64 if dtype == "bf16" else 32), vocab=_log(rng, 100, VOCAB), dtype=dtype,
                    mix=rng.choice([False, True]), sigma=rng.choice([1.0, 2.0, 3.0, 5.0]))
    while True:
        kind = rng.choice(["step", "step", "verify", "prefill"])
        q_lo, q_hi = {"step": (1, 1), "verify": (2, 9), "prefill": (1, _log(rng, 16, 300))}[kind]
        case = dict(op=op, layout=rng.choice(sorted(LAYOUTS)), n_req=_log(rng, 1, 64), q_lo=q_lo, q_hi=q_hi,
                    prefix=_log(rng, 1, 16384), own_hi=max(q_hi, _log(rng, 1, 1024)), page=rng.choice([16, 32, 64, 128, 256]),
                    window=rng.choice([0, 0, 1024]), softcap=rng.choice([0.0, 0.0, 50.0]), q_rms=rng.choice([0.1, 0.25, 1.0]))
        w = work(case)
        if w["flops"] <= 2.5e11 and w["bytes"] <= 4e8:
            return case


# ----------------------------------------------------------------------------- the inputs
def _rng(case, seed):
    return np.random.default_rng([seed, 7919])


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _lens(case, rng):
    """New rows (evenly spread over the case's range, in any order) and total own tokens of each
    request (host arrays)."""
    new = rng.permutation(np.round(np.linspace(case["q_lo"], case["q_hi"], case["n_req"])).astype(np.int64))
    total = np.maximum(new, rng.integers(1, case["own_hi"] + 1, case["n_req"]))
    return new.astype(np.int32), total.astype(np.int32)


def _plan_inputs(case, seed):
    rng = _rng(case, seed)
    n, page = case["n_req"], case["page"]
    cached = rng.integers(0, case["cached_hi"] + 1, n).astype(np.int32)
    new = rng.integers(case["new_lo"], case["new_hi"] + 1, n).astype(np.int32)
    blocks = -(-cached // page)
    need = -(-(cached + new) // page) - blocks
    max_blocks = -(-(case["cached_hi"] + case["new_hi"]) // page) + 1
    n_pages = int(blocks.sum() + need.sum()) + 64
    perm = rng.permutation(n_pages).astype(np.int32)
    table = np.full((n, max_blocks), -1, np.int32)
    held = np.arange(max_blocks)[None, :] < blocks[:, None]
    table[held] = perm[:int(blocks.sum())]
    free = perm[int(blocks.sum()):]
    return cached, new, free, table, n_pages, n * max(1, case["new_hi"])


def _append_inputs(case, seed):
    rng, g = _rng(case, seed), _gen(seed)
    H, nkv, hd = LAYOUTS[case["layout"]]
    rows, page = case["rows"], case["page"]
    cols = (H + (1 if case["v_from_k"] else 2) * nkv) * hd
    qkv = torch.randn(rows, cols, device="cuda", generator=g).bfloat16()
    qn = (1 + 0.02 * torch.randn(hd, device="cuda", generator=g)).bfloat16()
    kn = (1 + 0.02 * torch.randn(hd, device="cuda", generator=g)).bfloat16()
    inv = _dev((10000.0 ** (-np.arange(0, hd, 2) / hd)).astype(np.float32))
    n_pages = -(-rows // page) + 2
    slots = rng.permutation(n_pages * page)[:rows].astype(np.int32)
    pos = (rng.integers(0, case["far"]) + np.arange(rows)).astype(np.int32)
    k = torch.randn(n_pages, page, nkv, hd, device="cuda", generator=g).bfloat16()
    v = torch.randn(n_pages, page, nkv, hd, device="cuda", generator=g).bfloat16()
    return dict(qkv=qkv, qn=qn, kn=kn, inv=inv, slots=_dev(slots), pos=_dev(pos), k=k, v=v)


def _attn_inputs(case, seed):
    rng, g = _rng(case, seed), _gen(seed)
    H, nkv, hd = LAYOUTS[case["layout"]]
    page, lp, n = case["page"], case["prefix"], case["n_req"]
    new, total = _lens(case, rng)
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    T = int(start[-1])
    pos = np.concatenate([lp + total[b] - new[b] + np.arange(new[b]) for b in range(n)]).astype(np.int32)
    blocks, pblocks = -(-total // page), -(-lp // page)
    n_pages = int(blocks.sum()) + pblocks + 3
    perm = rng.permutation(n_pages).astype(np.int32)
    table = np.zeros((n, int(blocks.max())), np.int32)
    table[np.arange(table.shape[1])[None, :] < blocks[:, None]] = perm[pblocks:pblocks + int(blocks.sum())]
    # queries and keys as the QK norms leave them: rows of unit mean square, the queries scaled
    q = torch.randn(T, H, hd, device="cuda", generator=g)
    q = (q * torch.rsqrt((q * q).mean(-1, keepdim=True)) * case["q_rms"]).bfloat16()
    k = torch.randn(n_pages, page, nkv, hd, device="cuda", generator=g).bfloat16()
    v = torch.randn(n_pages, page, nkv, hd, device="cuda", generator=g).bfloat16()
    return dict(q=q, k=k, v=v, prefix_table=_dev(perm[:pblocks]), table=_dev(table), own_lens=_dev(total),
                row_start=_dev(start), row_pos=_dev(pos), max_q=int(new.max()), max_own=int(total.max()))


def _sample_inputs(case, seed):
    rng, g = _rng(case, seed), _gen(seed)
    n, V = case["rows"], case["vocab"]
    x = 30.0 * torch.tanh(torch.randn(n, V, device="cuda", generator=g) * (case["sigma"] / 30.0))
    banned = torch.randint(0, V, (n, 3), device="cuda", generator=g)
    x.scatter_(1, banned, float("-inf"))  # tokens that a request rules out
    x = x.bfloat16() if case["dtype"] == "bf16" else x
    t, k = np.full(n, 0.8, np.float32), np.full(n, 40, np.int32)
    p, mp = np.full(n, 0.95, np.float32), np.zeros(n, np.float32)
    if case["mix"]:
        t = rng.choice([0.0, 0.5, 0.7, 1.0, 1.3], n).astype(np.float32)
        k = np.minimum(V, rng.choice([0, 0, 1, 40, 200, 5000], n)).astype(np.int32)
        p = rng.choice([0.0, 0.5, 0.9, 0.95, 0.999], n).astype(np.float32)
        mp = rng.choice([0.0, 0.0, 0.01, 0.1], n).astype(np.float32)
    else:
        k = np.minimum(V, k)
    u = rng.random(n, dtype=np.float32)
    return dict(x=x, u=_dev(u), t=_dev(t), k=_dev(k), p=_dev(p), mp=_dev(mp))


def prepare(case, seed):
    op = case["op"]
    if op == "plan":
        cached, new, free, table, n_pages, max_rows = _plan_inputs(case, seed)
        st = dict(cached=_dev(cached), new=_dev(new), free=_dev(free), table=_dev(table), n_pages=n_pages, max_rows=max_rows)
    else:
        st = {"append": _append_inputs, "attn": _attn_inputs, "sample": _sample_inputs}[op](case, seed)
    st["case"] = case
    return st


# ------------------------------------------------------------------------- the plain forms
def _plain_plan(st):
    c, page = st["case"], st["case"]["page"]
    cached, new, free, table, n_pages, max_rows = (st[k] for k in ("cached", "new", "free", "table", "n_pages", "max_rows"))
    dev = cached.device
    n, width = table.shape
    rows_end = torch.cumsum(new, 0)
    row_start = torch.cat([torch.zeros_like(rows_end[:1]), rows_end])
    held = (cached + page - 1) // page
    total = cached + new
    need = (total + page - 1) // page - held
    end = torch.cumsum(need, 0)
    first = end - need
    j = torch.arange(width, device=dev)[None, :]
    fresh = (j >= held[:, None]) & (j < (held + need)[:, None])
    src = (first[:, None] + j - held[:, None]).clamp(0, max(0, free.numel() - 1))
    table.copy_(torch.where(fresh, free[src], table))
    r = torch.arange(max_rows, device=dev)
    live = r < rows_end[-1]
    req = torch.searchsorted(rows_end, r, right=True).clamp(max=n - 1)
    local = cached[req] + (r - row_start[req])
    page_of = table[req, (local // page).clamp(0, width - 1)]
    none = torch.full_like(r, -1)
    slot = torch.where(live, page_of * page + local % page, none)
    taken, rows = end[-1], rows_end[-1]
    status = torch.stack([taken, rows, torch.zeros_like(taken), torch.zeros_like(taken)])
    i32 = torch.int32
    return dict(table=table, row_start=row_start.to(i32), row_req=torch.where(live, req, none).to(i32),
                row_pos=torch.where(live, local, none).to(i32), slot_map=slot.to(i32), total_lens=total.to(i32),
                status=status.to(i32))


def _plain_append(st):
    c = st["case"]
    H, nkv, hd = LAYOUTS[c["layout"]]
    rows, half = c["rows"], hd // 2
    x = st["qkv"].float()
    q = x[:, :H * hd].view(rows, H, hd)
    k = x[:, H * hd:(H + nkv) * hd].view(rows, nkv, hd)
    v = k if c["v_from_k"] else x[:, (H + nkv) * hd:].view(rows, nkv, hd)
    eps = 1e-6
    q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + eps) * st["qn"].float()
    kr = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + eps) * st["kn"].float()
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps)
    ang = st["pos"].double()[:, None] * st["inv"].double()[None, :]
    cs, sn = torch.cos(ang).float()[:, None, :], torch.sin(ang).float()[:, None, :]
    q = torch.cat([q[..., :half] * cs - q[..., half:] * sn, q[..., :half] * sn + q[..., half:] * cs], -1)
    kr = torch.cat([kr[..., :half] * cs - kr[..., half:] * sn, kr[..., :half] * sn + kr[..., half:] * cs], -1)
    at = st["slots"].long()
    st["k"].view(-1, nkv, hd)[at] = kr.bfloat16()
    st["v"].view(-1, nkv, hd)[at] = v.bfloat16()
    return dict(q=q.bfloat16(), k_pool=st["k"], v_pool=st["v"])


def _plain_attn(st):
    c = st["case"]
    H, nkv, hd = LAYOUTS[c["layout"]]
    G, page, lp, n, max_q, max_own = H // nkv, c["page"], c["prefix"], c["n_req"], st["max_q"], st["max_own"]
    q, dev = st["q"], st["q"].device
    T = q.shape[0]
    k, v = st["k"].view(-1, nkv, hd), st["v"].view(-1, nkv, hd)
    pos = st["row_pos"].long()
    jp, jo = torch.arange(lp, device=dev), torch.arange(max_own, device=dev)
    at_p = st["prefix_table"].long()[jp // page] * page + jp % page
    at_o = st["table"].long()[:, jo // page] * page + jo % page                     # [n, max_own]
    start = st["row_start"].long()
    r = torch.arange(T, device=dev)
    req = torch.searchsorted(start[1:], r, right=True)
    i = r - start[req]
    q4 = q.float().view(T, nkv, G, hd)
    qb = torch.zeros(n, max_q, nkv, G, hd, device=dev)
    qb[req, i] = q4
    s_p = torch.einsum("tkgd,jkd->tkgj", q4, k[at_p].float())
    s_o = torch.einsum("bqkgd,bjkd->bqkgj", qb, k[at_o].float())[req, i]
    s = torch.cat([s_p, s_o], -1)
    if c["softcap"] > 0:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    key = torch.cat([jp, lp + jo])[None, :]
    see = (key <= pos[:, None]) & (key < lp + st["own_lens"].long()[req][:, None])
    if c["window"] > 0:
        see = see & (key > pos[:, None] - c["window"])
    s = torch.where(see[:, None, None, :], s, torch.full_like(s, float("-inf")))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    l = p.sum(-1, keepdim=True)
    o = torch.einsum("tkgj,jkd->tkgd", p[..., :lp], v[at_p].float())
    pb = torch.zeros(n, max_q, nkv, G, max_own, device=dev)
    pb[req, i] = p[..., lp:]
    o = o + torch.einsum("bqkgj,bjkd->bqkgd", pb, v[at_o].float())[req, i]
    return (o / l).reshape(T, H, hd).bfloat16()


def _plain_sample(st):
    x = st["x"].double()
    n, V = x.shape
    t, p, mp = st["t"].double()[:, None], st["p"].double()[:, None], st["mp"].double()[:, None]
    k = st["k"].long()[:, None]
    greedy = t <= 0
    w = torch.exp((x - x.amax(-1, keepdim=True)) / torch.where(greedy, torch.ones_like(t), t))
    order = torch.sort(st["x"], dim=-1, descending=True, stable=True).indices
    cum = torch.cumsum(w.gather(1, order), -1)
    every = torch.full_like(k, V)
    m_p = torch.where((p > 0) & (p < 1), 1 + (cum < p * cum[:, -1:]).sum(-1, keepdim=True), every)
    m_m = torch.where(mp > 0, (w >= mp).sum(-1, keepdim=True), every)
    m = torch.minimum(torch.minimum(m_p, m_m), torch.where(k > 0, k, every))
    m = torch.where(greedy, torch.ones_like(m), m).clamp(1, V)
    rank = torch.empty_like(order)
    rank.scatter_(1, order, torch.arange(V, device=x.device).expand(n, V))
    kept = torch.where(rank < m, w, torch.zeros_like(w))
    run_sum = torch.cumsum(kept, -1)
    whole = run_sum[:, -1:]
    token = (run_sum <= st["u"].double()[:, None] * whole).sum(-1, keepdim=True).clamp(max=V - 1)
    prob = kept.gather(1, token) / whole
    return dict(token=token[:, 0].int(), kept=m[:, 0].int(), prob=prob[:, 0].float())


# ------------------------------------------------------------------------- the entry points
def _own_plan(st):
    from hyperion_b200 import ops
    plan = ops.paged_plan(st["cached"], st["new"], st["free"], st["table"], st["n_pages"], st["case"]["page"], st["max_rows"])
    return dict(table=st["table"], row_start=plan.row_start, row_req=plan.row_req, row_pos=plan.row_pos,
                slot_map=plan.slot_map, total_lens=plan.total_lens, status=plan.status)


def _own_append(st):
    from hyperion_b200 import ops
    c = st["case"]
    H, nkv, hd = LAYOUTS[c["layout"]]
    q = ops.qkv_post_paged(st["qkv"], H, nkv, hd, c["v_from_k"], st["qn"], st["kn"], st["inv"], st["pos"], st["slots"],
                           st["k"], st["v"])
    return dict(q=q, k_pool=st["k"], v_pool=st["v"])


def _own_attn(st):
    from hyperion_b200 import ops
    c = st["case"]
    return ops.sdpa_shared_prefix(st["q"], st["k"], st["v"], st["prefix_table"], c["prefix"], st["table"], st["own_lens"],
                                  st["row_start"], st["row_pos"], st["max_q"], st["max_own"], window=c["window"],
                                  softcap=c["softcap"])


def _own_sample(st):
    from hyperion_b200 import ops
    token, kept, prob = ops.sample_batch(st["x"], st["u"], st["t"], st["k"], st["p"], st["mp"])
    return dict(token=token, kept=kept, prob=prob)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"plan": _own_plan, "append": _own_append, "attn": _own_attn, "sample": _own_sample}[op](state)
    return {"plan": _plain_plan, "append": _plain_append, "attn": _plain_attn, "sample": _plain_sample}[op](state)


# --------------------------------------------------------------------- the definition, 64 bits
def _exact_plan(case, seed):
    cached, new, free, table, n_pages, max_rows = _plan_inputs(case, seed)
    page, n = case["page"], case["n_req"]
    table = table.copy()
    req, pos, slot = (np.full(max_rows, -1, np.int32) for _ in range(3))
    start, taken = [0], 0
    for b in range(n):
        c, a = int(cached[b]), int(new[b])
        have, want = -(-c // page), -(-(c + a) // page)
        table[b, have:want] = free[taken:taken + want - have]
        taken += want - have
        at = start[-1]
        local = np.arange(c, c + a)
        req[at:at + a], pos[at:at + a] = b, local
        slot[at:at + a] = table[b, local // page] * page + local % page
        start.append(at + a)
    return dict(table=table, row_start=np.array(start, np.int32), row_req=req, row_pos=pos, slot_map=slot,
                total_lens=(cached + new).astype(np.int32), status=np.array([taken, start[-1], 0, 0], np.int32))


def _exact_append(case, seed):
    a = _append_inputs(case, seed)
    H, nkv, hd = LAYOUTS[case["layout"]]
    rows, half = case["rows"], hd // 2
    x = a["qkv"].double().view(rows, -1, hd)
    unit = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / hd + 1e-6)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), a["pos"].double()[:, None] * a["inv"].double())
    def rotated(h):
        z = torch.complex(h[..., :half], h[..., half:]) * turn[:, None, :]
        return torch.cat([z.real, z.imag], -1)
    k, v = a["k"].double().view(-1, nkv, hd), a["v"].double().view(-1, nkv, hd)
    k[a["slots"].long()] = rotated(unit[:, H:H + nkv] * a["kn"].double())
    v[a["slots"].long()] = unit[:, H:H + nkv] if case["v_from_k"] else unit[:, H + nkv:]
    return dict(q=rotated(unit[:, :H] * a["qn"].double()), k_pool=k.view(a["k"].shape), v_pool=v.view(a["v"].shape))


def _exact_attn(case, seed):
    a = _attn_inputs(case, seed)
    H, nkv, hd = LAYOUTS[case["layout"]]
    page, lp = case["page"], case["prefix"]
    k, v = a["k"].view(-1, nkv, hd), a["v"].view(-1, nkv, hd)
    start, lens = a["row_start"].tolist(), a["own_lens"].tolist()
    out = torch.empty(a["q"].shape, dtype=torch.float64, device="cuda")
    def slots(pages, length):
        return (pages.long()[:, None] * page + torch.arange(page, device="cuda")).flatten()[:length]
    at_p = slots(a["prefix_table"], lp)
    kp, vp = k[at_p].double(), v[at_p].double()
    for b, length in enumerate(lens):
        at = slots(a["table"][b], length)
        kb, vb = torch.cat([kp, k[at].double()]), torch.cat([vp, v[at].double()])
        rows = slice(start[b], start[b + 1])
        q, pos = a["q"][rows].double(), a["row_pos"][rows].long()[:, None]
        key = torch.arange(lp + length, device="cuda")[None, :]
        hidden = key > pos
        if case["window"]:
            hidden = hidden | (key <= pos - case["window"])
        for h in range(nkv):
            g = slice(h * H // nkv, (h + 1) * H // nkv)
            s = q[:, g] @ kb[:, h].T
            if case["softcap"]:
                s = case["softcap"] * torch.tanh(s / case["softcap"])
            out[rows, g] = torch.softmax(s.masked_fill(hidden[:, None], -math.inf), -1) @ vb[:, h]
    return out


def _exact_sample(case, seed):
    a = _sample_inputs(case, seed)
    x = a["x"].double().cpu().numpy()
    t, k, p, mp, u = (a[n].cpu().numpy() for n in ("t", "k", "p", "mp", "u"))
    n, V = x.shape
    token, kept, prob = np.zeros(n, np.int32), np.zeros(n, np.int32), np.zeros(n)
    for r in range(n):
        if t[r] <= 0:
            token[r], kept[r], prob[r] = int(np.argmax(x[r])), 1, 1.0
            continue
        w = np.exp((x[r] - x[r].max()) / np.float64(t[r]))
        order = np.argsort(-x[r], kind="stable")
        m = V
        if 0 < p[r] < 1:
            cum = np.cumsum(w[order])
            m = min(m, int(np.searchsorted(cum, np.float64(p[r]) * cum[-1], side="left")) + 1)
        if mp[r] > 0:
            m = min(m, int((w >= np.float64(mp[r])).sum()))
        if k[r] > 0:
            m = min(m, int(k[r]))
        m = max(m, 1)
        ids = np.sort(order[:m])
        cum = np.cumsum(w[ids])
        at = min(int(np.searchsorted(cum, np.float64(u[r]) * cum[-1], side="right")), m - 1)
        token[r], kept[r], prob[r] = ids[at], m, w[ids[at]] / cum[-1]
    return dict(token=token, kept=kept, prob=prob)


def exact(case, seed):
    return {"plan": _exact_plan, "append": _exact_append, "attn": _exact_attn, "sample": _exact_sample}[case["op"]](case, seed)


# --------------------------------------------------------------------------------- the work
def work(case):
    """Bytes that have to be read and written once, and operations of the products (expected sizes
    where lengths are drawn)."""
    op = case["op"]
    if op == "plan":
        new = (case["new_lo"] + case["new_hi"]) / 2
        rows, n = case["n_req"] * new, case["n_req"]
        most = n * max(1, case["new_hi"])
        pages = rows / case["page"]
        # lengths in; row tables out; the pages taken are read and entered; the old entry of a row's page is read
        return {"bytes": 4 * (2 * n + 2 * n + 1 + 3 * most + 2 * pages + n + 4), "flops": 8 * rows}
    if op == "append":
        H, nkv, hd = LAYOUTS[case["layout"]]
        cols_in = (H + (1 if case["v_from_k"] else 2) * nkv) * hd
        cols_out = (H + 2 * nkv) * hd
        return {"bytes": case["rows"] * (2 * cols_in + 2 * cols_out + 8) + 8 * hd,
                "flops": case["rows"] * 8 * cols_out}
    if op == "sample":
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": case["rows"] * (case["vocab"] * size + 32), "flops": 4 * case["rows"] * case["vocab"]}
    H, nkv, hd = LAYOUTS[case["layout"]]
    q = (case["q_lo"] + case["q_hi"]) / 2
    T, own_mean = case["n_req"] * q, max(q, case["own_hi"] / 2)
    seen = case["prefix"] + own_mean - q / 2
    prefix_read, own_read = case["prefix"], own_mean
    if case["window"]:
        # the window reaches back over the own tokens first, then into the prefix; of the
        # prefix the row with the fewest own tokens reads most
        seen = min(seen, case["window"])
        own_read = min(own_read, case["window"] + q)
        prefix_read = min(prefix_read, case["window"])
    kv = 2 * nkv * hd * 2
    return {"bytes": kv * (prefix_read + case["n_req"] * own_read) + 2 * T * H * hd * 2,
            "flops": 4 * T * H * hd * seen}

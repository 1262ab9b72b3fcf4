"""Op-level calls into libhyperion_mlx.so on torch CUDA tensors.

torch is used only to own device memory and streams; every computation runs in
the library's sm_100a kernels through the hyperion_b200.h C ABI.
"""
from __future__ import annotations

import ctypes

import torch

from . import check, lib


def _p(t: torch.Tensor):
    return ctypes.c_void_p(t.data_ptr())


def _stream(stream=None) -> ctypes.c_void_p:
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def quantized_matmul(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor,
                     out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """y = x @ dequant(w).T for affine Q4/g64 (x bf16 [M,K], w int32/uint32 [N,K/8])."""
    M, K = x.shape
    N = w.shape[0]
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    check(lib().hyb_quantized_matmul(_p(x), _p(w), _p(scales), _p(biases), _p(out), M, K, N, 64, 4,
                                     _stream(stream)))
    return out


def qmv_fused(x, w, scales, biases, prologue=0, epilogue=0, norm_w=None, resid=None, post_w=None, scalar=None,
              h_out=None, eps=1e-6, out=None, stream=None):
    """Batch-1 qmv with the decode engine's fused norm prologue / GeGLU epilogue."""
    K = x.numel()
    N = w.shape[0]
    if out is None:
        out = torch.empty(N // 2 if epilogue == 1 else N, dtype=torch.bfloat16, device=x.device)
    opt = lambda t: _p(t) if t is not None else None
    check(lib().hyb_qmv_fused(_p(x), _p(w), _p(scales), _p(biases), _p(out), K, N, prologue, epilogue,
                              opt(norm_w), opt(resid), opt(post_w), opt(scalar), opt(h_out), eps, _stream(stream)))
    return out


def qmv_pack(w, scales, biases, stream=None) -> torch.Tensor:
    """Repack MLX-layout Q4/g64 weights into the decode engine's packed layout (uint8 tensor)."""
    N, K8 = w.shape
    K = K8 * 8
    out = torch.empty(lib().hyb_qmv_packed_bytes(K, N), dtype=torch.uint8, device=w.device)
    check(lib().hyb_qmv_pack(_p(w), _p(scales), _p(biases), K, N, _p(out), _stream(stream)))
    return out


def qmv_unpack(packed, K, N, stream=None):
    """The MLX layout (w [N, K/8] uint32, scales/biases [N, K/64] bf16) of a packed matrix."""
    w = torch.empty((N, K // 8), dtype=torch.int32, device=packed.device)
    s = torch.empty((N, K // 64), dtype=torch.bfloat16, device=packed.device)
    b = torch.empty((N, K // 64), dtype=torch.bfloat16, device=packed.device)
    check(lib().hyb_qmv_unpack(_p(packed), K, N, _p(w), _p(s), _p(b), _stream(stream)))
    return w, s, b


def embed_packed(ids, packed, H, N, embed_scale_bits, stream=None):
    """Embedding rows of a packed [N, H] table (dequantised, x embed scale): [L, H] bf16."""
    L = ids.numel()
    out = torch.empty((L, H), dtype=torch.bfloat16, device=packed.device)
    check(lib().hyb_embed_packed(_p(ids), L, _p(packed), H, N, embed_scale_bits, _p(out), _stream(stream)))
    return out


def qmv_packed(x, packed, K, N, prologue=0, epilogue=0, norm_w=None, resid=None, post_w=None, scalar=None,
               h_out=None, eps=1e-6, out=None, stream=None):
    """Batch-1 qmv over packed weights (TMA-streamed kernel), same options as qmv_fused."""
    if out is None:
        out = torch.empty(N // 2 if epilogue == 1 else N, dtype=torch.bfloat16, device=x.device)
    opt = lambda t: _p(t) if t is not None else None
    check(lib().hyb_qmv_packed(_p(x), _p(packed), _p(out), K, N, prologue, epilogue, opt(norm_w), opt(resid),
                               opt(post_w), opt(scalar), opt(h_out), eps, _stream(stream)))
    return out


def qmv_batched(x, packed, K, N, geglu=False, out=None, stream=None):
    """Batched decode qmv over packed weights: x [B, K] bf16 -> [B, N] (or [B, N/2] with GeGLU)."""
    B = x.shape[0]
    if out is None:
        out = torch.empty((B, N // 2 if geglu else N), dtype=torch.bfloat16, device=x.device)
    check(lib().hyb_qmv_batched(_p(x), B, x.stride(0), _p(packed), _p(out), out.stride(0), K, N, 1 if geglu else 0,
                                _stream(stream)))
    return out


class DecodeScratch:
    """Device workspace for hyb_sdpa_decode (zeroed once)."""

    def __init__(self, n_heads, n_kv, hd, max_keys, device="cuda"):
        n = lib().hyb_sdpa_decode_scratch_bytes(n_heads, n_kv, hd, max_keys)
        self.buf = torch.zeros(n, dtype=torch.uint8, device=device)
        self.nbytes = n


def sdpa_decode(q, k_cache, v_cache, last_pos: int, n_keys: int, scratch: DecodeScratch, scale=1.0,
                softcap=0.0, rounding=0, out=None, stream=None):
    H, hd = q.shape
    cap, nkv, _ = k_cache.shape
    if out is None:
        out = torch.empty_like(q)
    check(lib().hyb_sdpa_decode(_p(q), _p(k_cache), _p(v_cache), _p(out), H, nkv, hd, cap, last_pos, n_keys,
                                scale, softcap, rounding, _p(scratch.buf), scratch.nbytes, _stream(stream)))
    return out


def sdpa_decode_fused(qkv, v_from_k, q_norm, k_norm, inv_freq, k_cache, v_cache, pos, n_keys, n_heads, eps=1e-6,
                      scale=1.0, softcap=0.0, rounding=0, out=None, stream=None):
    """Fused decode step: norms + RoPE + cache append + attention (cluster kernel)."""
    cap, nkv, hd = k_cache.shape
    if out is None:
        out = torch.empty((n_heads, hd), dtype=torch.bfloat16, device=qkv.device)
    check(lib().hyb_sdpa_decode_fused(_p(qkv), int(v_from_k), _p(q_norm), _p(k_norm), _p(inv_freq), eps,
                                      _p(k_cache), _p(v_cache), cap, pos, n_keys, n_heads, nkv, hd, scale, softcap,
                                      rounding, _p(out), _stream(stream)))
    return out


def sdpa_prefill(q, k, v, q_pos0: int, k_pos0: int, window: int, scale=1.0, softcap=0.0, rounding=0,
                 out=None, stream=None):
    Lq, H, hd = q.shape
    Lk, nkv, _ = k.shape
    if out is None:
        out = torch.empty_like(q)
    check(lib().hyb_sdpa_prefill(_p(q), _p(k), _p(v), _p(out), Lq, Lk, H, nkv, hd, q_pos0, k_pos0, window,
                                 scale, softcap, rounding, _stream(stream)))
    return out


def rms_norm(x, w, eps=1e-6, out=None, stream=None):
    rows = x.numel() // x.shape[-1]
    if out is None:
        out = torch.empty_like(x)
    check(lib().hyb_rms_norm(_p(x), _p(w) if w is not None else None, _p(out), rows, x.shape[-1], eps,
                             _stream(stream)))
    return out


def qkv_post(qkv, n_heads, n_kv, hd, v_from_k, q_norm, k_norm, inv_freq, pos0, eps=1e-6, k_cache=None,
             v_cache=None, cache_first=0, stream=None):
    L, ld = qkv.shape
    q_out = torch.empty((L, n_heads, hd), dtype=torch.bfloat16, device=qkv.device)
    k_out = torch.empty((L, n_kv, hd), dtype=torch.bfloat16, device=qkv.device)
    v_out = torch.empty((L, n_kv, hd), dtype=torch.bfloat16, device=qkv.device)
    cap = k_cache.shape[0] if k_cache is not None else 0
    check(lib().hyb_qkv_post(_p(qkv), L, ld, n_heads, n_kv, hd, int(v_from_k), _p(q_norm), _p(k_norm),
                             _p(inv_freq), pos0, eps, _p(q_out), _p(k_out), _p(v_out),
                             _p(k_cache) if k_cache is not None else None,
                             _p(v_cache) if v_cache is not None else None, cap, cache_first, _stream(stream)))
    return q_out, k_out, v_out


# ---------------------------------------------------------------- batch decode over a paged cache
# A decode step calls these every few microseconds of GPU work, so the checks are written for the
# host's time: one comparison chain per tensor, plain integers for the C arguments, and a stream
# or device switch only where the call asks for one.
_I32, _F32, _BF16 = torch.int32, torch.float32, torch.bfloat16


def _bad(name, t, dtype, shape, dev):
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{dev}")
    if t.dtype != dtype:
        raise ValueError(f"{name} is {t.dtype}, expected {dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    raise ValueError(f"{name} must be contiguous")


def _ck(name, t, dtype, shape, dev):
    """The pointer of a contiguous tensor of this type, shape and device."""
    if t.get_device() != dev or t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        _bad(name, t, dtype, shape, dev)
    return t.data_ptr()


def _ck_opt(name, t, dtype, shape, dev):
    return None if t is None else _ck(name, t, dtype, shape, dev)


def _ck_int(names, bits):
    """ctypes would cut a count to its lower 32 bits. `bits` is the or of them all: out of range where one is and
    none is negative, and a negative one is refused by the entry point."""
    if bits >> 31 not in (0, -1):
        raise ValueError(f"{names} must be below 2^31")


def _device(t):
    dev = t.get_device()
    if dev < 0:
        raise ValueError("the paged ops take CUDA tensors")
    return dev


def _switch(dev, stream):
    """None where the call can go to the current stream as it is; otherwise the context that makes
    its device and stream current, so that what the call allocates belongs to them."""
    if stream is None:
        return None if dev == torch._C._cuda_getDevice() else torch.cuda.device(dev)
    if stream.device.index != dev:
        raise ValueError(f"the stream is on {stream.device}, the tensors on cuda:{dev}")
    return torch.cuda.stream(stream)


def _here(dev):
    return torch._C._cuda_getCurrentRawStream(dev)


class PagedPlan:
    """The row tables of a step (int32, on the device): row_start [n_req + 1], row_req, row_pos
    and slot_map [max_rows], total_lens [n_req], status [4] (pages taken, rows, requests
    refused, bad pages). Reused from step to step by passing it back as `plan`."""

    def __init__(self, n_req: int, max_rows: int, device="cuda"):
        whole = torch.empty(2 * n_req + 3 * max_rows + 5, dtype=_I32, device=device)
        (self.row_start, self.row_req, self.row_pos, self.slot_map, self.total_lens, self.status) = whole.split_with_sizes(
            [n_req + 1, max_rows, max_rows, max_rows, n_req, 4])
        # the parts' addresses, in the order of the C arguments
        a = whole.data_ptr()
        b = a + 4 * (n_req + 1)
        r = 4 * max_rows
        self._at = (a, b, b + r, b + 2 * r, b + 3 * r, b + 3 * r + 4 * n_req)
        self._key = (n_req, max_rows, whole.get_device())


def paged_plan(cached_lens, new_lens, free_pages, block_table, n_pages: int, page_size: int, max_rows: int, pos0=0,
               plan: PagedPlan | None = None, stream=None) -> PagedPlan:
    """Block tables (in place) and the row tables of a step from the requests' lengths. The lengths may be
    another plan's total_lens, not those of the `plan` that is written."""
    _ck_int("n_pages, page_size, max_rows, pos0", n_pages | page_size | max_rows | pos0)
    dev, n = _device(cached_lens), cached_lens.numel()
    if block_table.dim() != 2 or free_pages.dim() != 1:
        raise ValueError("block_table is [n_req, max_blocks], free_pages [n_free]")
    width, n_free = block_table.shape[1], free_pages.shape[0]
    _ck_int("the lengths of cached_lens, block_table and free_pages", n | width | n_free)
    c, a = _ck("cached_lens", cached_lens, _I32, (n,), dev), _ck("new_lens", new_lens, _I32, (n,), dev)
    f, b = _ck("free_pages", free_pages, _I32, (n_free,), dev), _ck("block_table", block_table, _I32, (n, width), dev)
    ctx = _switch(dev, stream)
    if ctx is not None:
        with ctx:
            return paged_plan(cached_lens, new_lens, free_pages, block_table, n_pages, page_size, max_rows, pos0, plan)
    if plan is None:
        plan = PagedPlan(n, max_rows, cached_lens.device)
    if plan._key != (n, max_rows, dev):
        raise ValueError(f"plan is for (requests, rows, device) {plan._key}, the call has {(n, max_rows, dev)}")
    check(lib().hyb_paged_plan(c, a, n, page_size, n_pages, f, n_free, b, width, pos0, max_rows, *plan._at, _here(dev)))
    return plan


def qkv_post_paged(qkv, n_heads, n_kv, hd, v_from_k, q_norm, k_norm, inv_freq, row_pos, slot_map, k_pool, v_pool, eps=1e-6,
                   q_out=None, stream=None):
    """QK-norm, RoPE at row_pos and the cache write to slot_map of the pools [n_pages, page_size,
    n_kv, hd]; returns q [T, n_heads, hd]. qkv [T, ld] may have padded rows (its stride is used)."""
    _ck_int("n_heads, n_kv, hd", n_heads | n_kv | hd)
    dev = _device(qkv)
    if qkv.dim() != 2 or qkv.dtype is not _BF16 or qkv.stride(1) != 1:
        raise ValueError("qkv is bf16 [T, columns] with unit column stride")
    T, cols = qkv.shape
    ld = qkv.stride(0) if T > 1 else -(-cols // 8) * 8
    if ld < cols or cols < (n_heads + (1 if v_from_k else 2) * n_kv) * hd:
        raise ValueError("qkv has overlapping rows or fewer columns than q, k and v need")
    shape = k_pool.shape
    if len(shape) != 4 or shape[2] != n_kv or shape[3] != hd:
        raise ValueError("k_pool is [n_pages, page_size, n_kv, hd]")
    _ck_int("the rows of qkv, their stride and the slots of the pools", T | ld | shape[0] * shape[1])
    ctx = _switch(dev, stream)
    if ctx is not None:
        with ctx:
            return qkv_post_paged(qkv, n_heads, n_kv, hd, v_from_k, q_norm, k_norm, inv_freq, row_pos, slot_map, k_pool, v_pool,
                                  eps, q_out)
    if q_out is None:
        q_out = torch.empty((T, n_heads, hd), dtype=_BF16, device=qkv.device)
    check(lib().hyb_qkv_post_paged(qkv.data_ptr(), T, ld, n_heads, n_kv, hd, 1 if v_from_k else 0,
                                   _ck("q_norm", q_norm, _BF16, (hd,), dev), _ck("k_norm", k_norm, _BF16, (hd,), dev),
                                   _ck("inv_freq", inv_freq, _F32, (hd // 2,), dev), _ck("row_pos", row_pos, _I32, (T,), dev),
                                   _ck("slot_map", slot_map, _I32, (T,), dev), shape[0] * shape[1], eps,
                                   _ck("q_out", q_out, _BF16, (T, n_heads, hd), dev), _ck("k_pool", k_pool, _BF16, shape, dev),
                                   _ck("v_pool", v_pool, _BF16, shape, dev), _here(dev)))
    return q_out


class SharedPrefixScratch:
    """Device workspace for sdpa_shared_prefix calls of these sizes (contents do not matter). A
    larger one serves any call that needs no more bytes."""

    def __init__(self, T, n_req, max_q, max_own, prefix_len, n_heads, n_kv, hd, device="cuda"):
        _ck_int("T, n_req, max_q, max_own, prefix_len, n_heads, n_kv, hd", T | n_req | max_q | max_own | prefix_len | n_heads | n_kv | hd)
        n = lib().hyb_sdpa_shared_prefix_scratch_bytes(T, n_req, max_q, max_own, prefix_len, n_heads, n_kv, hd)
        if n == 0:
            raise ValueError("sdpa_shared_prefix: bad shape")
        self.buf = torch.empty(n, dtype=torch.uint8, device=device)
        self.nbytes = n


def sdpa_shared_prefix(q, k_pool, v_pool, prefix_table, prefix_len: int, block_table, own_lens, row_start, row_pos, max_q: int,
                       max_own: int, window=0, scale=1.0, softcap=0.0, scratch: SharedPrefixScratch | None = None, out=None,
                       stream=None):
    """Attention of rows q [T, H, hd] over the shared prefix and their requests' own pages."""
    _ck_int("prefix_len, max_q, max_own, window", prefix_len | max_q | max_own | window)
    dev = _device(q)
    shape = q.shape
    if len(shape) != 3 or k_pool.dim() != 4 or block_table.dim() != 2:
        raise ValueError("q is [T, H, hd], the pools [n_pages, page_size, n_kv, hd], block_table [n_req, max_blocks]")
    T, H, hd = shape
    pool = k_pool.shape
    n_pages, page, nkv, _ = pool
    n, width = own_lens.numel(), block_table.shape[1]
    _ck_int("the sizes of q, the pools and block_table", T | H | n_pages | page | n | width)
    if prefix_len < 0 or (prefix_len > 0 and (prefix_table is None or prefix_table.numel() * page < prefix_len)):
        raise ValueError("prefix_table does not hold prefix_len keys")
    if pool[3] != hd:
        raise ValueError(f"q has head_dim {hd}, the pools {pool[3]}")
    ctx = _switch(dev, stream)
    if ctx is not None:
        with ctx:
            return sdpa_shared_prefix(q, k_pool, v_pool, prefix_table, prefix_len, block_table, own_lens, row_start, row_pos,
                                      max_q, max_own, window, scale, softcap, scratch, out)
    L = lib()
    if out is None:
        out = torch.empty(shape, dtype=_BF16, device=q.device)
    if scratch is None:
        scratch = SharedPrefixScratch(T, n, max_q, max_own, prefix_len, H, nkv, hd, q.device)
    if scratch.buf.get_device() != dev:
        raise ValueError(f"scratch is on {scratch.buf.device}, expected cuda:{dev}")
    check(L.hyb_sdpa_shared_prefix(_ck("q", q, _BF16, shape, dev), _ck("k_pool", k_pool, _BF16, pool, dev),
                                   _ck("v_pool", v_pool, _BF16, pool, dev), n_pages, page,
                                   None if prefix_table is None else _ck("prefix_table", prefix_table, _I32, (prefix_table.numel(),), dev),
                                   prefix_len, _ck("block_table", block_table, _I32, (n, width), dev), width,
                                   _ck("own_lens", own_lens, _I32, (n,), dev), _ck("row_start", row_start, _I32, (n + 1,), dev),
                                   _ck("row_pos", row_pos, _I32, (T,), dev), T, n, max_q, max_own, H, nkv, hd, window, scale,
                                   softcap, _ck("out", out, _BF16, shape, dev), scratch.buf.data_ptr(), scratch.nbytes, _here(dev)))
    return out


def sample_batch(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, out=None, stream=None):
    """(token, kept, prob) of every row of logits [rows, vocab] (bf16 or float32, rows may be
    padded), from uniforms u [rows] and per-row settings (None: off, temperature 1)."""
    dev, dtype = _device(logits), logits.dtype
    if logits.dim() != 2 or (dtype is not _BF16 and dtype is not _F32) or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits is bf16 or float32 [rows, vocab] with unit column stride")
    n, V = logits.shape
    _ck_int("the sizes of logits", n | V)
    ld = logits.stride(0) if n > 1 else V
    if ld < V:
        raise ValueError("the rows of logits overlap")
    rows = (n,)
    args = (_ck("u", u, _F32, rows, dev), _ck_opt("temperature", temperature, _F32, rows, dev), _ck_opt("top_k", top_k, _I32, rows, dev),
            _ck_opt("top_p", top_p, _F32, rows, dev), _ck_opt("min_p", min_p, _F32, rows, dev))
    ctx = _switch(dev, stream)
    if ctx is not None:
        with ctx:
            return sample_batch(logits, u, temperature, top_k, top_p, min_p, out)
    if out is None:
        where = logits.device
        out = (torch.empty(n, dtype=_I32, device=where), torch.empty(n, dtype=_I32, device=where),
               torch.empty(n, dtype=_F32, device=where))
    token, kept, prob = out
    check(lib().hyb_sample_batch(logits.data_ptr(), 1 if dtype is _F32 else 0, n, V, ld, *args, _ck("token", token, _I32, rows, dev),
                                 _ck("kept", kept, _I32, rows, dev), _ck("prob", prob, _F32, rows, dev), _here(dev)))
    return out

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
def _on(ref: torch.Tensor, **tensors):
    """Checks of the paged ops' arguments: every given tensor (value: tensor, dtype, shape or
    None) sits on `ref`'s CUDA device, has its dtype and shape and is contiguous."""
    if not ref.is_cuda:
        raise ValueError("the paged ops take CUDA tensors")
    for name, (t, dtype, shape) in tensors.items():
        if t is None:
            continue
        if t.device != ref.device:
            raise ValueError(f"{name} is on {t.device}, expected {ref.device}")
        if t.dtype != dtype:
            raise ValueError(f"{name} is {t.dtype}, expected {dtype}")
        if shape is not None and tuple(t.shape) != tuple(shape):
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")


class _Launch:
    """The device and the stream of a call: `stream` or the device's current one, made current
    so that what the call allocates belongs to that stream."""

    def __init__(self, device, stream):
        self.stream = stream if stream is not None else torch.cuda.current_stream(device)
        if self.stream.device != device:
            raise ValueError(f"the stream is on {self.stream.device}, the tensors on {device}")
        self.ctx = torch.cuda.stream(self.stream)

    def __enter__(self):
        self.ctx.__enter__()
        return ctypes.c_void_p(self.stream.cuda_stream)

    def __exit__(self, *exc):
        self.ctx.__exit__(*exc)


def _opt(t):
    return _p(t) if t is not None else None


class PagedPlan:
    """The row tables of a step (int32, on the device): row_start [n_req + 1], row_req, row_pos
    and slot_map [max_rows], total_lens [n_req], status [4] (pages taken, rows, requests
    refused, bad pages). Reused from step to step by passing it back as `plan`."""

    def __init__(self, n_req: int, max_rows: int, device="cuda"):
        sizes = [n_req + 1, max_rows, max_rows, max_rows, n_req, 4]
        parts = torch.empty(sum(sizes), dtype=torch.int32, device=device).split(sizes)
        self.row_start, self.row_req, self.row_pos, self.slot_map, self.total_lens, self.status = parts


def paged_plan(cached_lens, new_lens, free_pages, block_table, n_pages: int, page_size: int, max_rows: int, pos0=0,
               plan: PagedPlan | None = None, stream=None) -> PagedPlan:
    """Block tables (in place) and the row tables of a step from the requests' lengths."""
    i32, n = torch.int32, cached_lens.numel()
    if block_table.dim() != 2 or free_pages.dim() != 1:
        raise ValueError("block_table is [n_req, max_blocks], free_pages [n_free]")
    _on(cached_lens, cached_lens=(cached_lens, i32, (n,)), new_lens=(new_lens, i32, (n,)), free_pages=(free_pages, i32, None),
        block_table=(block_table, i32, (n, block_table.shape[1])))
    with _Launch(cached_lens.device, stream) as st:
        if plan is None:
            plan = PagedPlan(n, max_rows, cached_lens.device)
        _on(cached_lens, row_start=(plan.row_start, i32, (n + 1,)), row_req=(plan.row_req, i32, (max_rows,)),
            row_pos=(plan.row_pos, i32, (max_rows,)), slot_map=(plan.slot_map, i32, (max_rows,)),
            total_lens=(plan.total_lens, i32, (n,)), status=(plan.status, i32, (4,)))
        check(lib().hyb_paged_plan(_p(cached_lens), _p(new_lens), n, page_size, n_pages, _p(free_pages), free_pages.numel(),
                                   _p(block_table), block_table.shape[1], pos0, max_rows, _p(plan.row_start), _p(plan.row_req),
                                   _p(plan.row_pos), _p(plan.slot_map), _p(plan.total_lens), _p(plan.status), st))
    return plan


def qkv_post_paged(qkv, n_heads, n_kv, hd, v_from_k, q_norm, k_norm, inv_freq, row_pos, slot_map, k_pool, v_pool, eps=1e-6,
                   q_out=None, stream=None):
    """QK-norm, RoPE at row_pos and the cache write to slot_map of the pools [n_pages, page_size,
    n_kv, hd]; returns q [T, n_heads, hd]. qkv [T, ld] may have padded rows (its stride is used)."""
    bf, i32 = torch.bfloat16, torch.int32
    if qkv.dim() != 2 or qkv.stride(1) != 1 or qkv.dtype != bf or (qkv.shape[0] > 1 and qkv.stride(0) < qkv.shape[1]):
        raise ValueError("qkv is bf16 [T, columns] with unit column stride")
    T = qkv.shape[0]
    if qkv.shape[1] < (n_heads + (1 if v_from_k else 2) * n_kv) * hd:
        raise ValueError("qkv has fewer columns than q, k and v need")
    if k_pool.dim() != 4 or k_pool.shape[2:] != (n_kv, hd):
        raise ValueError("k_pool is [n_pages, page_size, n_kv, hd]")
    _on(qkv, q_norm=(q_norm, bf, (hd,)), k_norm=(k_norm, bf, (hd,)), inv_freq=(inv_freq, torch.float32, (hd // 2,)),
        row_pos=(row_pos, i32, (T,)), slot_map=(slot_map, i32, (T,)), k_pool=(k_pool, bf, None),
        v_pool=(v_pool, bf, k_pool.shape), q_out=(q_out, bf, (T, n_heads, hd)))
    with _Launch(qkv.device, stream) as st:
        if q_out is None:
            q_out = torch.empty((T, n_heads, hd), dtype=bf, device=qkv.device)
        ld = qkv.stride(0) if T > 1 else -(-qkv.shape[1] // 8) * 8
        check(lib().hyb_qkv_post_paged(_p(qkv), T, ld, n_heads, n_kv, hd, int(v_from_k), _p(q_norm), _p(k_norm), _p(inv_freq),
                                       _p(row_pos), _p(slot_map), k_pool.shape[0] * k_pool.shape[1], eps, _p(q_out),
                                       _p(k_pool), _p(v_pool), st))
    return q_out


class SharedPrefixScratch:
    """Device workspace for sdpa_shared_prefix calls of at most these sizes (contents do not matter)."""

    def __init__(self, T, n_req, max_q, max_own, prefix_len, n_heads, n_kv, hd, device="cuda"):
        n = lib().hyb_sdpa_shared_prefix_scratch_bytes(T, n_req, max_q, max_own, prefix_len, n_heads, n_kv, hd)
        if n == 0:
            raise ValueError("sdpa_shared_prefix: bad shape")
        self.buf = torch.empty(n, dtype=torch.uint8, device=device)
        self.nbytes = n


def sdpa_shared_prefix(q, k_pool, v_pool, prefix_table, prefix_len: int, block_table, own_lens, row_start, row_pos, max_q: int,
                       max_own: int, window=0, scale=1.0, softcap=0.0, scratch: SharedPrefixScratch | None = None, out=None,
                       stream=None):
    """Attention of rows q [T, H, hd] over the shared prefix and their requests' own pages."""
    bf, i32 = torch.bfloat16, torch.int32
    if q.dim() != 3 or k_pool.dim() != 4 or block_table.dim() != 2:
        raise ValueError("q is [T, H, hd], the pools [n_pages, page_size, n_kv, hd], block_table [n_req, max_blocks]")
    T, H, hd = q.shape
    n_pages, page, nkv, _ = k_pool.shape
    n = own_lens.numel()
    _on(q, q=(q, bf, None), k_pool=(k_pool, bf, (n_pages, page, nkv, hd)), v_pool=(v_pool, bf, k_pool.shape),
        prefix_table=(prefix_table, i32, None), block_table=(block_table, i32, (n, block_table.shape[1])),
        own_lens=(own_lens, i32, (n,)), row_start=(row_start, i32, (n + 1,)), row_pos=(row_pos, i32, (T,)), out=(out, bf, q.shape))
    if prefix_len < 0 or (prefix_len > 0 and (prefix_table is None or prefix_table.numel() * page < prefix_len)):
        raise ValueError("prefix_table does not hold prefix_len keys")
    with _Launch(q.device, stream) as st:
        if out is None:
            out = torch.empty_like(q)
        if scratch is None:
            scratch = SharedPrefixScratch(T, n, max_q, max_own, prefix_len, H, nkv, hd, q.device)
        _on(q, scratch=(scratch.buf, torch.uint8, None))
        check(lib().hyb_sdpa_shared_prefix(_p(q), _p(k_pool), _p(v_pool), n_pages, page, _opt(prefix_table), prefix_len,
                                           _p(block_table), block_table.shape[1], _p(own_lens), _p(row_start), _p(row_pos), T, n,
                                           max_q, max_own, H, nkv, hd, window, scale, softcap, _p(out), _p(scratch.buf),
                                           scratch.nbytes, st))
    return out


def sample_batch(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, out=None, stream=None):
    """(token, kept, prob) of every row of logits [rows, vocab] (bf16 or float32, rows may be
    padded), from uniforms u [rows] and per-row settings (None: off, temperature 1)."""
    f32, i32 = torch.float32, torch.int32
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, f32) or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits is bf16 or float32 [rows, vocab] with unit column stride")
    n, V = logits.shape
    if n > 1 and logits.stride(0) < V:
        raise ValueError("the rows of logits overlap")
    _on(logits, u=(u, f32, (n,)), temperature=(temperature, f32, (n,)), top_k=(top_k, i32, (n,)), top_p=(top_p, f32, (n,)),
        min_p=(min_p, f32, (n,)))
    with _Launch(logits.device, stream) as st:
        if out is None:
            out = (torch.empty(n, dtype=i32, device=logits.device), torch.empty(n, dtype=i32, device=logits.device),
                   torch.empty(n, dtype=f32, device=logits.device))
        token, kept, prob = out
        _on(logits, token=(token, i32, (n,)), kept=(kept, i32, (n,)), prob=(prob, f32, (n,)))
        check(lib().hyb_sample_batch(_p(logits), int(logits.dtype == f32), n, V, logits.stride(0) if n > 1 else V, _p(u),
                                     _opt(temperature), _opt(top_k), _opt(top_p), _opt(min_p), _p(token), _p(kept), _p(prob),
                                     st))
    return token, kept, prob

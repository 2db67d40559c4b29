"""The paged fp8 key/value cache: writing it, reading it back, attending over it.

Sequences of any length share one pool of pages.  A page holds ``page_size`` tokens of every K/V head in fp8, with
one scale per page and head for K and one for V (x = descale * x8).  A call is about the last n_b tokens of every
sequence b, its new ones: ``seqlens`` [batch] are the lengths with them, ``cu_seqlens`` [batch + 1] where their rows
begin in the token-major tensors ([tokens, heads, head_dim]; None: the tokens divided evenly), ``page_table``
[batch, pages] which page holds tokens p * page_size ... of a sequence.  So a decoding step is

    paged_kv_append(cache, k, v, page_table, seqlens)
    o = flash_attention_paged_kv(q, cache, page_table, seqlens, True, scale)[0]

and a batch of prompts, or of prompts and single tokens, the same with cu_seqlens (which kernel attends goes by the mean
number of new tokens: many single tokens beside a long prompt are faster as a call of their own).  The numbers in the three int32
tensors stay on the device (the calls can be captured into a CUDA graph and replayed with others in their place); one
that is out of range is left out by the kernels and raises in check_status() or at the next call.
"""
from __future__ import annotations

import ctypes
from typing import List, NamedTuple, Optional, Tuple

import torch

from . import _lib
from .api import _check_input, _native, status_word

PAGE_SIZES = (16, 32, 64, 128)
_FP8 = {torch.float8_e4m3fn: _lib.FA8_FP8_E4M3, torch.float8_e5m2: _lib.FA8_FP8_E5M2}
_HALF = {torch.float16: _lib.FA8_DTYPE_FP16, torch.bfloat16: _lib.FA8_DTYPE_BF16}


class PagedKVCache(NamedTuple):
    """The pool: k, v float8_e4m3fn or float8_e5m2 [num_pages, heads_kv, page_size, head_dim] (page_size 16, 32, 64 or
    128; head_dim a multiple of 32 up to 256) and k_descale, v_descale float32 [num_pages, heads_kv], 0 or from 2^-64 to
    2^64 where a token of the page is held, all contiguous on one device.  The operators take any four tensors like these.  A page needs no initialisation: its first token
    starts it anew."""
    k: torch.Tensor
    v: torch.Tensor
    k_descale: torch.Tensor
    v_descale: torch.Tensor

    @classmethod
    def empty(cls, num_pages: int, heads_kv: int, head_dim: int, page_size: int = 64,
              dtype: torch.dtype = torch.float8_e4m3fn, device=None) -> "PagedKVCache":
        """A pool of its own on `device` (default: the current one)."""
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        shape = (num_pages, heads_kv, page_size, head_dim)
        cache = cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device),
                    torch.empty(shape[:2], dtype=torch.float32, device=device),
                    torch.empty(shape[:2], dtype=torch.float32, device=device))
        _check_cache(*cache)
        return cache


def _check_cache(k, v, k_descale, v_descale):
    for name, t in (("cache.k", k), ("cache.v", v), ("cache.k_descale", k_descale), ("cache.v_descale", v_descale)):
        _check_input(t, name)
        if t.device != k.device:
            raise RuntimeError("the cache's tensors must be on the same device")
    if k.dtype not in _FP8 or v.dtype != k.dtype:
        raise RuntimeError(f"cache.k and cache.v must both be float8_e4m3fn or both float8_e5m2, got {k.dtype} and {v.dtype}")
    if k.dim() != 4 or v.shape != k.shape:
        raise RuntimeError(f"cache.k and cache.v must be [num_pages, heads_kv, page_size, head_dim] alike; they are "
                           f"{tuple(k.shape)} and {tuple(v.shape)}")
    if k.numel() == 0:
        raise RuntimeError(f"the cache has no pages: cache.k is {tuple(k.shape)}")
    if k.shape[2] not in PAGE_SIZES:
        raise RuntimeError(f"page_size must be one of {PAGE_SIZES}, got {k.shape[2]}")
    if k.shape[3] % 32 != 0 or k.shape[3] > 256:
        raise RuntimeError(f"head_dim must be a multiple of 32 up to 256, got {k.shape[3]}")
    for name, t in (("cache.k_descale", k_descale), ("cache.v_descale", v_descale)):
        if t.dtype != torch.float32 or t.shape != k.shape[:2]:
            raise RuntimeError(f"{name} must be float32 [num_pages, heads_kv] = {tuple(k.shape[:2])}, got {t.dtype} {tuple(t.shape)}")


def _check_tables(device, page_table, seqlens, cu_seqlens, tokens):
    given = [("page_table", page_table, 2), ("seqlens", seqlens, 1)]
    if cu_seqlens is not None:
        given.append(("cu_seqlens", cu_seqlens, 1))
    for name, t, dim in given:
        if t.device != device:
            raise RuntimeError(f"{name} must be on the cache's device")
        if t.dtype != torch.int32 or t.dim() != dim or t.stride(-1) != 1 and t.shape[-1] > 1:
            raise RuntimeError(f"{name} must be int32 with {dim} dimension{'s' if dim > 1 else ''} and contiguous rows")
    batch = seqlens.shape[0]
    if page_table.shape[0] != batch:
        raise RuntimeError(f"page_table has {page_table.shape[0]} rows, seqlens {batch} entries")
    if cu_seqlens is not None and cu_seqlens.shape[0] != batch + 1:
        raise RuntimeError(f"cu_seqlens must have batch + 1 = {batch + 1} entries, got {cu_seqlens.shape[0]}")
    if tokens > 0 and (batch == 0 or page_table.shape[1] == 0):
        raise RuntimeError("there are tokens but no sequences or no pages to hold them")
    if batch > 1 and page_table.stride(0) < page_table.shape[1]:
        raise RuntimeError("page_table's rows must not overlap")
    if batch > 1 and page_table.stride(0) > 0x7fffffff:
        raise RuntimeError(f"page_table's rows are {page_table.stride(0)} entries apart: more than 32 bits hold")
    if cu_seqlens is None and batch > 0 and tokens % batch != 0:
        raise RuntimeError(f"{tokens} tokens cannot be divided evenly over {batch} sequences: give cu_seqlens")


def _check_rows(t, name, device, heads, head_dim):
    if not isinstance(t, torch.Tensor) or t.device != device:
        raise RuntimeError(f"{name} must be a tensor on the cache's device")
    if t.dtype not in _HALF:
        raise RuntimeError(f"{name} must be float16 or bfloat16, got {t.dtype}")
    if t.dim() != 3 or t.shape[2] != head_dim or (heads is not None and t.shape[1] != heads):
        raise RuntimeError(f"{name} must be [tokens, {'heads' if heads is None else heads}, {head_dim}], got {tuple(t.shape)}")
    if t.numel() > 0 and (t.stride(2) != 1 or t.stride(0) % 8 or t.stride(1) % 8 or t.data_ptr() % 16):
        raise RuntimeError(f"{name} needs contiguous rows of head_dim that start at multiples of 16 bytes; its strides are {t.stride()}")
    if torch.is_grad_enabled() and t.requires_grad:
        raise RuntimeError(f"{name} requires a gradient, and there is no backward pass through the cache")


def _params(cache, page_table, seqlens, cu_seqlens, tokens):
    k, v, k_descale, v_descale = cache
    return _lib.Fa8KvCache(
        k=k.data_ptr(), v=v.data_ptr(), k_descale=k_descale.data_ptr(), v_descale=v_descale.data_ptr(),
        num_pages=k.shape[0], heads_kv=k.shape[1], page_size=k.shape[2], head_dim=k.shape[3], fp8_format=_FP8[k.dtype],
        batch=seqlens.shape[0], page_table=page_table.data_ptr(), table_width=page_table.shape[1],
        table_stride=page_table.stride(0) if seqlens.shape[0] > 1 else page_table.shape[1], seqlens=seqlens.data_ptr(),
        cu_seqlens=(cu_seqlens.data_ptr() if cu_seqlens is not None else None), tokens=tokens,
        status_word=status_word(k.device).data_ptr())


def _raise_if(rc: int) -> None:
    # FA8_ERR_DEVICE_TIMEOUT and FA8_ERR_BAD_INDEX are about an EARLIER launch on the device; this call was not enqueued
    if rc != _lib.FA8_OK:
        raise RuntimeError(_lib.error_message(rc))


def paged_kv_append(cache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, seqlens: torch.Tensor, *,
                    cu_seqlens: Optional[torch.Tensor] = None) -> None:
    """Quantises the new tokens' keys and values into their pages.

    cache: PagedKVCache (or four tensors like it).  k, v: float16 or bfloat16 [tokens, heads_kv, head_dim], views with
    strides allowed (parts of a fused projection).  Per page and head, and K and V apart, the scale is the smallest
    power of two 2^e, -64 <= e <= 64, by which the largest finite |x| written to the page fits the fp8 range.  It starts
    anew with the page's first token and otherwise only grows; when it does, the page's older tokens are rounded anew.
    x8 = fp8(x / descale), to the nearest, infinities (and what is beyond 2^64 times the range) as the largest number.  No two sequences may write to the same page.
    Stream-ordered; one kernel, nothing allocated."""
    native = _native()
    if native:
        try:
            done = native._kv_append(*cache, k, v, page_table, seqlens, cu_seqlens)
        except TypeError:
            done = None
        if done is not None:
            return _raise_if(done)
    lib = _lib.load()
    _check_cache(*cache)
    device, heads, head_dim = cache[0].device, cache[0].shape[1], cache[0].shape[3]
    _check_rows(k, "k", device, heads, head_dim)
    _check_rows(v, "v", device, heads, head_dim)
    if v.dtype != k.dtype or v.shape != k.shape:
        raise RuntimeError("k and v must have the same type and shape")
    tokens = k.shape[0]
    _check_tables(device, page_table, seqlens, cu_seqlens, tokens)
    if tokens == 0:
        return
    p = _params(cache, page_table, seqlens, cu_seqlens, tokens)
    with torch.cuda.device(device):
        _raise_if(lib.fa8_kv_append(ctypes.byref(p), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                                    _HALF[k.dtype], torch.cuda.current_stream(device).cuda_stream))


def paged_kv_read(cache, page_table: torch.Tensor, seqlens: torch.Tensor, tokens: int, *,
                  cu_seqlens: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The last n_b tokens of every sequence back from the cache: (k, v), float16 or bfloat16 [tokens, heads_kv,
    head_dim], x8 * descale rounded once.  `tokens`: their number in all (the rows to allocate); whole sequences are
    read with cu_seqlens the running sum of seqlens.  Rows outside cu_seqlens are left as allocated."""
    native = _native()
    if native and dtype in _HALF:
        try:
            done = native._kv_read(*cache, page_table, seqlens, tokens, cu_seqlens, dtype == torch.bfloat16)
        except TypeError:
            done = None
        if type(done) is tuple:
            return done
        if done is not None:
            _raise_if(done)
    lib = _lib.load()
    _check_cache(*cache)
    device = cache[0].device
    if dtype not in _HALF:
        raise RuntimeError(f"dtype must be float16 or bfloat16, got {dtype}")
    tokens = int(tokens)
    if not 0 <= tokens <= 0x7fffffff:
        raise RuntimeError(f"tokens must be a number of rows, got {tokens}")
    _check_tables(device, page_table, seqlens, cu_seqlens, tokens)
    k, v = (torch.empty((tokens, cache[0].shape[1], cache[0].shape[3]), dtype=dtype, device=device) for _ in range(2))
    if tokens > 0:
        p = _params(cache, page_table, seqlens, cu_seqlens, tokens)
        with torch.cuda.device(device):
            _raise_if(lib.fa8_kv_read(ctypes.byref(p), k.data_ptr(), v.data_ptr(), _HALF[dtype],
                                      torch.cuda.current_stream(device).cuda_stream))
    return k, v


def flash_attention_paged_kv(q: torch.Tensor, cache, page_table: torch.Tensor, seqlens: torch.Tensor,
                             is_causal: bool = False, softmax_scale: float = 1.0, *,
                             cu_seqlens: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                             return_lse: bool = False) -> List[torch.Tensor]:
    """Attention of the new tokens' queries over their sequences' pages.

    q: float16 or bfloat16 [tokens, heads, head_dim], a view with strides allowed; heads a multiple of the cache's (query
    head h reads K/V head h // (heads // heads_kv)).  With is_causal new token i of sequence b sees the keys up to its
    own position, seqlens[b] - n_b + i; without it every key of its sequence.  A row that sees no key is zeros (its
    log-sum-exp -inf); a NaN reaches the rows that see its key and no others (an infinity, which an e5m2 cache may hold, too, as an
    infinity or a NaN).  Scores, softmax and sums are fp32; K and V enter exactly as the cache holds them.
    Returns [O], O in q's type [tokens, heads, head_dim] (`out` if given: contiguous), and with return_lse the fp32
    [tokens, heads] log-sum-exp of the scaled scores.  Rows outside cu_seqlens are left as they were.  Stream-ordered;
    nothing synchronises."""
    native = _native()
    if native:
        try:
            done = native._kv_attention(q, *cache, page_table, seqlens, is_causal, softmax_scale, cu_seqlens, out, return_lse)
        except TypeError:
            done = None
        if type(done) is list:
            return done
        if done is not None:
            _raise_if(done)
    lib = _lib.load()
    _check_cache(*cache)
    device, heads_kv, head_dim = cache[0].device, cache[0].shape[1], cache[0].shape[3]
    _check_rows(q, "q", device, None, head_dim)
    tokens, heads = q.shape[:2]
    if heads == 0 or heads % heads_kv != 0:
        raise RuntimeError(f"q must have a multiple of the cache's {heads_kv} heads, got {heads}")
    _check_tables(device, page_table, seqlens, cu_seqlens, tokens)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
    else:
        _check_input(out, "out")
        if out.dtype != q.dtype or out.shape != q.shape or out.device != device or out.data_ptr() % 16:
            raise RuntimeError("out must be a contiguous tensor of q's type, shape and device, aligned to 16 bytes")
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=device) if return_lse else None
    if tokens > 0:
        with torch.cuda.device(device):
            need = lib.fa8_kv_attention_workspace(seqlens.shape[0], tokens, heads, heads_kv, head_dim, cache[0].shape[2], page_table.shape[1],
                                                  torch.cuda.get_device_properties(device).multi_processor_count)
            if need < 0:
                _raise_if(need)
            # of the caching allocator: a captured call's is its graph's own
            workspace = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
            p = _lib.Fa8KvAttentionParams(
                cache=_params(cache, page_table, seqlens, cu_seqlens, tokens), q=q.data_ptr(), q_token_stride=q.stride(0),
                q_head_stride=q.stride(1), o=out.data_ptr(), lse=(lse.data_ptr() if return_lse else None), dtype=_HALF[q.dtype],
                heads=heads, is_causal=int(bool(is_causal)), softmax_scale=float(softmax_scale),
                workspace=(workspace.data_ptr() if need > 0 else None), workspace_bytes=need)
            _raise_if(lib.fa8_kv_attention(ctypes.byref(p), torch.cuda.current_stream(device).cuda_stream))
    return [out, lse] if return_lse else [out]

"""Paged KV cache: requests of different lengths in one pool of pages.

The dense cache of ``ddq_b200.attention`` keeps a batch of equal positions.
Here every request has a length of its own and a row of a block table that
lists its pages, so prompts, chunks of prompts and single tokens share a step,
and a long common prefix is stored (and, when decoding, read) once:

* ``plan_step``         - new pages, slots and positions of a step from the request lengths
* ``rope_kv_write``     - rotary embedding of q and k, k and v into their pages
* ``prefill_attention`` - the new tokens of ragged requests over their pages
* ``decode_attention``  - one token per sequence over a shared prefix and its own pages

They take the place of the reference's q/k RoPE (``RoPe_d.cu:12-68``), cache
write (``engine.py:126-130``) and attention (``engine.py:225-251``) where the
requests differ.  Nothing here reads a length on the host: every call is
stream-ordered and can be captured in a CUDA graph.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib

PAGE_SIZES = (16, 32, 64, 128, 256)
_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}


class StepPlan(NamedTuple):
    """What ``plan_step`` returns (device tensors)."""
    cu_new: torch.Tensor     # int32 [R + 1] first token row of each request
    lens: torch.Tensor       # int32 [R] tokens in the cache after the step
    slots: torch.Tensor      # int64 [T] page * page_size + row; -1: none
    positions: torch.Tensor  # int64 [T]
    seq_ids: torch.Tensor    # int32 [T] request of the row; -1 behind the last
    free_head: torch.Tensor  # int32 [1] first page of the free list not handed out


def _need(cond, msg):
    if not cond:
        raise RuntimeError(msg)


def _on(t, device):
    return isinstance(t, torch.Tensor) and t.is_cuda and t.device == device


def _vector(t, n, dtype, device, what):
    _need(_on(t, device) and t.dtype == dtype and t.dim() == 1 and
          (n is None or t.numel() == n) and t.is_contiguous(), what)


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _ptr(t):
    return t.data_ptr() if t is not None else None


def plan_step(cached: torch.Tensor, new: torch.Tensor, block_table: torch.Tensor,
              free_pages: torch.Tensor, page_size: int, num_tokens: int,
              free_head: Optional[torch.Tensor] = None, prefix_len: int = 0) -> StepPlan:
    """The pages, slots and positions of a step (``ddq_plan_step``).

    ``cached`` and ``new`` int32 [R]: tokens a request has in the cache and
    tokens of this step (0 allowed); ``block_table`` int32 [R, width] holds the
    pages of the cached tokens and is extended in place; ``free_pages`` int32
    [F] with ``free_head`` int32 [1] (default 0) its first unused entry;
    ``num_tokens`` the token rows of the step (at least ``new.sum()``: a padded
    count for a captured graph is fine); ``prefix_len`` the positions of a
    shared prefix in front of every request.  A token that gets no page (list
    exhausted, table row full) has slot -1; ``free_head`` of the result then
    exceeds F, or the request's length its table row."""
    _need(isinstance(cached, torch.Tensor) and cached.is_cuda, "plan_step: cached must be CUDA")
    dev, R = cached.device, cached.numel()
    _vector(cached, None, torch.int32, dev, "plan_step: cached must be int32 CUDA [R]")
    _vector(new, R, torch.int32, dev, "plan_step: new must be int32 CUDA [R]")
    _need(_on(block_table, dev) and block_table.dtype == torch.int32 and
          block_table.dim() == 2 and block_table.shape[0] == R and block_table.shape[1] > 0 and
          block_table.stride(1) == 1 and
          (R == 1 or block_table.stride(0) >= block_table.shape[1]),
          "plan_step: block_table must be int32 CUDA [R, width] with distinct rows")
    _vector(free_pages, None, torch.int32, dev, "plan_step: free_pages must be int32 CUDA [F]")
    if free_head is not None:
        _vector(free_head, 1, torch.int32, dev, "plan_step: free_head must be int32 CUDA [1]")
    _need(R >= 1, "plan_step: at least one request")
    _need(page_size in PAGE_SIZES, f"plan_step: page_size must be one of {PAGE_SIZES}")
    _need(num_tokens >= 0 and prefix_len >= 0, "plan_step: negative count")
    T = int(num_tokens)
    i32 = torch.empty(2 * R + 2 + T, dtype=torch.int32, device=dev)
    cu, lens, head, seq = i32.split([R + 1, R, 1, T])
    i64 = torch.empty(2, T, dtype=torch.int64, device=dev)
    with torch.cuda.device(dev):
        st = _lib.load().ddq_plan_step(
            cached.data_ptr(), new.data_ptr(), block_table.data_ptr(),
            block_table.stride(0) if R > 1 else block_table.shape[1], block_table.shape[1],
            free_pages.data_ptr(), free_pages.numel(), _ptr(free_head), int(page_size),
            int(prefix_len), cu.data_ptr(), lens.data_ptr(), i64[0].data_ptr(),
            i64[1].data_ptr(), seq.data_ptr(), head.data_ptr(), R, T, _stream(dev))
    _lib.check(st, "plan_step")
    return StepPlan(cu, lens, i64[0], i64[1], seq, head)


def _strides(t, dims):
    """Element strides of the outer dimensions; a dimension of one element has
    no stride that matters (torch leaves any there)."""
    return [t.stride(i) if t.shape[i] > 1 else t.shape[-1] for i in dims]


def _cache(k_pages, v_pages, what) -> _lib.PagedCache:
    _need(isinstance(k_pages, torch.Tensor) and k_pages.is_cuda and k_pages.dtype in _DTYPES and
          k_pages.dim() == 4, f"{what}: k_pages must be fp16 or bf16 CUDA [P, Hkv, page_size, D]")
    _need(_on(v_pages, k_pages.device) and v_pages.dtype == k_pages.dtype and
          v_pages.shape == k_pages.shape,
          f"{what}: k_pages and v_pages must have the same type and shape")
    P, Hkv, ps, D = k_pages.shape
    _need(ps in PAGE_SIZES, f"{what}: page_size must be one of {PAGE_SIZES}")
    _need(D in (64, 128), f"{what}: head_dim must be 64 or 128")
    strides = _strides(k_pages, (0, 1, 2))
    _need(k_pages.stride(3) == 1 and all(s % 8 == 0 for s in strides),
          f"{what}: pages need a unit inner stride and outer strides that are multiples of 8")
    _need(strides == _strides(v_pages, (0, 1, 2)) and v_pages.stride(3) == 1,
          f"{what}: k_pages and v_pages must have the same strides")
    return _lib.PagedCache(k_pages.data_ptr(), v_pages.data_ptr(), P, ps, Hkv, D, *strides,
                           _DTYPES[k_pages.dtype])


def rope_kv_write(qkv: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                  cos: torch.Tensor, sin: torch.Tensor, slots: torch.Tensor,
                  positions: torch.Tensor, num_heads: int, num_kv_heads: int, head_dim: int,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary embedding and cache write of a step's tokens (``ddq_paged_rope_kv``).

    ``qkv`` [T, (Hq + 2 Hkv) * D]; ``k_pages``/``v_pages`` [P, Hkv, page_size, D]
    (any strides with D contiguous); ``cos``/``sin`` fp32 [max_pos, D] tables;
    ``slots`` and ``positions`` int64 [T] as ``plan_step`` gives them (a negative
    slot writes nothing; a slot must not occur twice).  Returns rope(q)
    [T, Hq, D]."""
    c = _cache(k_pages, v_pages, "rope_kv_write")
    dev = k_pages.device
    width = (num_heads + 2 * num_kv_heads) * head_dim
    _need(num_kv_heads == c.Hkv and head_dim == c.D and num_heads >= 1,
          "rope_kv_write: heads do not match the pages")
    _need(_on(qkv, dev) and qkv.dtype == k_pages.dtype and qkv.dim() == 2 and
          qkv.shape[1] == width and qkv.stride(1) == 1,
          "rope_kv_write: qkv must be [T, (Hq + 2 Hkv) * D] of the pages' type, unit inner stride")
    T = qkv.shape[0]
    for t in (cos, sin):
        _need(_on(t, dev) and t.dtype == torch.float32 and t.dim() == 2 and
              t.shape == cos.shape and t.shape[1] == head_dim and t.is_contiguous(),
              "rope_kv_write: cos and sin must be contiguous fp32 CUDA [max_pos, D]")
    _vector(slots, T, torch.int64, dev, "rope_kv_write: slots must be int64 CUDA [T]")
    _vector(positions, T, torch.int64, dev, "rope_kv_write: positions must be int64 CUDA [T]")
    if out is None:
        out = torch.empty((T, num_heads, head_dim), dtype=qkv.dtype, device=dev)
    _need(_on(out, dev) and out.dtype == qkv.dtype and out.is_contiguous() and
          tuple(out.shape) == (T, num_heads, head_dim),
          "rope_kv_write: out must be contiguous [T, Hq, D] of the pages' type")
    with torch.cuda.device(dev):
        st = _lib.load().ddq_paged_rope_kv(
            qkv.data_ptr(), qkv.stride(0) if T > 1 else width, ctypes.byref(c), cos.data_ptr(),
            sin.data_ptr(), cos.shape[0], slots.data_ptr(), positions.data_ptr(), out.data_ptr(),
            T, num_heads, _stream(dev))
    _lib.check(st, "rope_kv_write")
    return out


def _check_attention(q, k_pages, block_table, lens, rows, slopes, softcap, out, what):
    dev = k_pages.device
    Hkv, D = k_pages.shape[1], k_pages.shape[3]
    _need(_on(q, dev) and q.dtype == k_pages.dtype and q.dim() == 3 and q.shape[2] == D and
          q.shape[1] >= 1 and q.shape[1] % Hkv == 0 and q.stride(2) == 1,
          f"{what}: q must be [T, Hq, D] of the pages' type, Hq a multiple of Hkv")
    _need(_on(block_table, dev) and block_table.dtype == torch.int32 and
          block_table.dim() == 2 and block_table.shape[0] == rows and block_table.shape[1] > 0 and
          block_table.stride(1) == 1,
          f"{what}: block_table must be int32 CUDA [requests, width]")
    _need(rows <= 1 or block_table.stride(0) >= block_table.shape[1],
          f"{what}: block_table rows must not overlap")
    _vector(lens, rows, torch.int32, dev, f"{what}: lens must be int32 CUDA [requests]")
    if slopes is not None:
        _vector(slopes, q.shape[1], torch.float32, dev, f"{what}: slopes must be fp32 CUDA [Hq]")
    _need(0.0 <= softcap < float("inf"), f"{what}: softcap must be finite and not negative")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    _need(_on(out, dev) and out.dtype == q.dtype and out.shape == q.shape and
          out.stride(2) == 1, f"{what}: out must have the shape and type of q")
    return out


def _check_prefix(prefix_pages, prefix_len, c, dev, what):
    prefix_len = int(prefix_len)
    _need(prefix_len >= 0, f"{what}: prefix_len must not be negative")
    if prefix_len:
        _need(prefix_pages is not None, f"{what}: prefix_len needs prefix_pages")
        _vector(prefix_pages, None, torch.int32, dev,
                f"{what}: prefix_pages must be int32 CUDA [pages]")
        _need(prefix_pages.numel() * c.page_size >= prefix_len,
              f"{what}: prefix_pages holds fewer than prefix_len keys")
    return prefix_len


def _workspace(nbytes, device):
    """Partial results of a split key axis: from the caching allocator for each
    call, so calls on different streams and captured graphs never share it."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def prefill_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                      block_table: torch.Tensor, cu_new: torch.Tensor, lens: torch.Tensor,
                      scale: float, softcap: float = 0.0, slopes: Optional[torch.Tensor] = None,
                      bidir: Optional[torch.Tensor] = None,
                      prefix_pages: Optional[torch.Tensor] = None, prefix_len: int = 0,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the new tokens of ragged requests over their pages
    (``ddq_paged_prefill_attention``).

    ``q`` [T, Hq, D] holds the requests' new tokens one after another: rows
    ``cu_new[r] .. cu_new[r + 1] - 1`` are the last tokens of request r, whose
    ``lens[r]`` keys and values (the new ones included) lie in the pages that
    ``block_table[r]`` lists; in front of them stand ``prefix_len`` keys that all
    requests share (pages ``prefix_pages`` int32; the prefix may end inside a
    page).  A row at position p attends the keys j of the prefix and of its own
    request with ``j <= p`` (and, with ``bidir`` int32 [R], the first ``bidir[r]``
    own keys whatever its position); scores ``scale * q.k``, with ``softcap`` > 0 capped to ``softcap *
    tanh(s / softcap)``, minus ``slopes[h] * |p - j|`` with ``slopes`` fp32 [Hq].
    A row without keys is zero.  Rows of ``out`` behind ``cu_new[R]`` are left
    as they are.  Keys and values of a request must be finite; the rest of its
    last page may hold anything."""
    c = _cache(k_pages, v_pages, "prefill_attention")
    dev = k_pages.device
    _need(_on(cu_new, dev) and cu_new.dtype == torch.int32 and cu_new.dim() == 1 and
          cu_new.numel() >= 1 and cu_new.is_contiguous(),
          "prefill_attention: cu_new must be int32 CUDA [R + 1]")
    R = cu_new.numel() - 1
    out = _check_attention(q, k_pages, block_table, lens, R, slopes, softcap, out,
                           "prefill_attention")
    if bidir is not None:
        _vector(bidir, R, torch.int32, dev, "prefill_attention: bidir must be int32 CUDA [R]")
    prefix_len = _check_prefix(prefix_pages, prefix_len, c, dev, "prefill_attention")
    T, Hq, D = q.shape
    W = block_table.shape[1]
    L = _lib.load()
    with torch.cuda.device(dev):
        nws = L.ddq_paged_prefill_attention_workspace_size(T, R, Hq, c.Hkv, D, W, c.page_size,
                                                           prefix_len)
        ws = _workspace(nws, dev)
        st = L.ddq_paged_prefill_attention(
            q.data_ptr(), *_strides(q, (0, 1)), ctypes.byref(c), block_table.data_ptr(),
            block_table.stride(0) if R > 1 else W, W, cu_new.data_ptr(), lens.data_ptr(), _ptr(bidir),
            _ptr(prefix_pages) if prefix_len else None, prefix_len, _ptr(slopes), float(scale),
            float(softcap), out.data_ptr(), *_strides(out, (0, 1)), T, R, Hq, _ptr(ws), nws,
            _stream(dev))
    _lib.check(st, "prefill_attention")
    return out


def decode_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                     block_table: torch.Tensor, lens: torch.Tensor, scale: float,
                     prefix_pages: Optional[torch.Tensor] = None, prefix_len: int = 0,
                     softcap: float = 0.0, slopes: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one token per sequence (``ddq_paged_decode_attention``).

    ``q`` [B, Hq, D]; sequence b attends ``prefix_len`` keys that the whole batch
    shares (in the pages of ``prefix_pages`` int32; read once for all of them),
    then its own ``lens[b]`` keys (the new token's included) in the pages of
    ``block_table[b]``; its query stands at position ``prefix_len + lens[b] - 1``.
    The prefix may end inside a page: the own keys start in pages of their own.
    ``softcap`` and ``slopes`` as in ``prefill_attention``.  A sequence without
    keys gives zeros."""
    c = _cache(k_pages, v_pages, "decode_attention")
    dev = k_pages.device
    _need(isinstance(q, torch.Tensor) and q.dim() == 3, "decode_attention: q must be [B, Hq, D]")
    out = _check_attention(q, k_pages, block_table, lens, q.shape[0], slopes, softcap, out,
                           "decode_attention")
    prefix_len = _check_prefix(prefix_pages, prefix_len, c, dev, "decode_attention")
    B, Hq, D = q.shape
    W = block_table.shape[1]
    L = _lib.load()
    with torch.cuda.device(dev):
        nws = L.ddq_paged_decode_attention_workspace_size(B, Hq, c.Hkv, D, W, c.page_size,
                                                          prefix_len)
        ws = _workspace(nws, dev)
        st = L.ddq_paged_decode_attention(
            q.data_ptr(), *_strides(q, (0, 1)), ctypes.byref(c), block_table.data_ptr(),
            block_table.stride(0) if B > 1 else W, W, lens.data_ptr(),
            _ptr(prefix_pages) if prefix_len else None, prefix_len, _ptr(slopes), float(scale),
            float(softcap), out.data_ptr(), *_strides(out, (0, 1)), B, Hq, _ptr(ws), nws,
            _stream(dev))
    _lib.check(st, "decode_attention")
    return out

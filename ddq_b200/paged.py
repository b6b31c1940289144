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
from .gemm_fp8 import _stream_ptr

PAGE_SIZES = (16, 32, 64, 128, 256)
_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_ws_sizes: dict = {}   # (entry, device index, shape) -> workspace bytes

# A small step is bound by the host (a call's kernels take 3 to 10 us), so the
# entry points test what a correct call has in as few attribute reads as
# possible; what is wrong with one that fails is found out afterwards.


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


def _vec(t, dtype, index):
    return (t.dtype is dtype and t.get_device() == index and t.dim() == 1 and t.is_contiguous())


def _vector(t, n, dtype, index, what):
    _need(_vec(t, dtype, index) and (n is None or t.numel() == n), what)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _call(name, device, *args):
    """The library entry on the tensors' device and its current stream."""
    fn = getattr(_lib.load(), "ddq_" + name)
    if torch.cuda.current_device() == device.index:
        return fn(*args, _stream_ptr(device))
    with torch.cuda.device(device):
        return fn(*args, _stream_ptr(device))


def _size(name, device, *shape):
    key = (name, device.index, shape)
    n = _ws_sizes.get(key)
    if n is None:
        with torch.cuda.device(device):
            n = getattr(_lib.load(), f"ddq_{name}_workspace_size")(*shape)
        if len(_ws_sizes) > 4096:   # lengths vary from call to call
            _ws_sizes.clear()
        _ws_sizes[key] = n
    return n


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
    index, R, T = cached.get_device(), cached.numel(), int(num_tokens)
    _need(index >= 0 and _vec(cached, torch.int32, index),
          "plan_step: cached must be int32 CUDA [R]")
    _vector(new, R, torch.int32, index, "plan_step: new must be int32 CUDA [R]")
    shape, stride = block_table.shape, block_table.stride()
    _need(block_table.dtype is torch.int32 and block_table.get_device() == index and
          len(shape) == 2 and shape[0] == R and shape[1] > 0 and
          (stride[1] == 1 or shape[1] == 1) and (R == 1 or stride[0] >= shape[1]),
          "plan_step: block_table must be int32 CUDA [R, width] with distinct rows")
    _vector(free_pages, None, torch.int32, index, "plan_step: free_pages must be int32 CUDA [F]")
    if free_head is not None:
        _vector(free_head, 1, torch.int32, index, "plan_step: free_head must be int32 CUDA [1]")
    _need(R >= 1, "plan_step: at least one request")
    _need(page_size in PAGE_SIZES, f"plan_step: page_size must be one of {PAGE_SIZES}")
    _need(T >= 0 and prefix_len >= 0, "plan_step: negative count")
    dev = cached.device
    i32 = torch.empty(2 * R + 2 + T, dtype=torch.int32, device=dev)
    i64 = torch.empty((2, T), dtype=torch.int64, device=dev)
    p32, p64 = i32.data_ptr(), i64.data_ptr()
    st = _call("plan_step", dev, cached.data_ptr(), new.data_ptr(), block_table.data_ptr(),
               stride[0] if R > 1 else shape[1], shape[1], free_pages.data_ptr(),
               free_pages.numel(), _ptr(free_head), page_size, prefix_len, p32,
               p32 + 4 * (R + 1), p64, p64 + 8 * T, p32 + 4 * (2 * R + 2),
               p32 + 4 * (2 * R + 1), R, T)
    if st:
        _lib.check(st, "plan_step")
    cu, lens, head, seq = i32.split_with_sizes((R + 1, R, 1, T))
    slots, positions = i64.unbind(0)
    return StepPlan(cu, lens, slots, positions, seq, head)


def _strides(shape, stride):
    """Element strides of the outer dimensions; a dimension of one element has
    no stride that matters (torch leaves any there)."""
    return tuple(s if n > 1 else shape[-1] for n, s in zip(shape[:-1], stride))


def _cache(k_pages, v_pages, what):
    """(ddq_paged_cache, device index, shape) of a pool."""
    shape, dtype, index = k_pages.shape, k_pages.dtype, k_pages.get_device()
    code = _DTYPES.get(dtype)
    _need(index >= 0 and code is not None and len(shape) == 4,
          f"{what}: k_pages must be fp16 or bf16 CUDA [P, Hkv, page_size, D]")
    _need(v_pages.dtype is dtype and v_pages.get_device() == index and v_pages.shape == shape,
          f"{what}: k_pages and v_pages must have the same type and shape")
    P, Hkv, ps, D = shape
    _need(ps in PAGE_SIZES, f"{what}: page_size must be one of {PAGE_SIZES}")
    _need(D == 64 or D == 128, f"{what}: head_dim must be 64 or 128")
    sk, sv = k_pages.stride(), v_pages.stride()
    a, b, c = _strides(shape, sk)
    _need(sk[3] == 1 and (a | b | c) % 8 == 0,
          f"{what}: pages need a unit inner stride and outer strides that are multiples of 8")
    _need(sk == sv or (sv[3] == 1 and _strides(shape, sv) == (a, b, c)),
          f"{what}: k_pages and v_pages must have the same strides")
    return _lib.PagedCache(k_pages.data_ptr(), v_pages.data_ptr(), P, ps, Hkv, D, a, b, c,
                           code), index, shape


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
    c, index, (_, Hkv, _, D) = _cache(k_pages, v_pages, "rope_kv_write")
    dtype, shape, stride = k_pages.dtype, qkv.shape, qkv.stride()
    width = (num_heads + 2 * num_kv_heads) * head_dim
    _need(num_kv_heads == Hkv and head_dim == D and num_heads >= 1,
          "rope_kv_write: heads do not match the pages")
    _need(qkv.dtype is dtype and qkv.get_device() == index and len(shape) == 2 and
          shape[1] == width and stride[1] == 1,
          "rope_kv_write: qkv must be [T, (Hq + 2 Hkv) * D] of the pages' type, unit inner stride")
    T, rot = shape[0], cos.shape
    _need(cos.dtype is torch.float32 and cos.get_device() == index and len(rot) == 2 and
          rot[1] == D and cos.is_contiguous() and sin.dtype is torch.float32 and
          sin.get_device() == index and sin.shape == rot and sin.is_contiguous(),
          "rope_kv_write: cos and sin must be contiguous fp32 CUDA [max_pos, D]")
    _vector(slots, T, torch.int64, index, "rope_kv_write: slots must be int64 CUDA [T]")
    _vector(positions, T, torch.int64, index, "rope_kv_write: positions must be int64 CUDA [T]")
    dev = k_pages.device
    if out is None:
        out = torch.empty((T, num_heads, D), dtype=dtype, device=dev)
    else:
        _need(out.dtype is dtype and out.get_device() == index and out.is_contiguous() and
              tuple(out.shape) == (T, num_heads, D),
              "rope_kv_write: out must be contiguous [T, Hq, D] of the pages' type")
    st = _call("paged_rope_kv", dev, qkv.data_ptr(), stride[0] if T > 1 else width,
               ctypes.byref(c), cos.data_ptr(), sin.data_ptr(), rot[0], slots.data_ptr(),
               positions.data_ptr(), out.data_ptr(), T, num_heads)
    if st:
        _lib.check(st, "rope_kv_write")
    return out


def _check_attention(q, k_pages, index, kshape, block_table, lens, rows, slopes, softcap, out,
                     what):
    """(out, shape and outer strides of q, row stride of the table, strides of out)"""
    dtype, shape, stride = k_pages.dtype, q.shape, q.stride()
    _need(q.dtype is dtype and q.get_device() == index and len(shape) == 3 and
          shape[2] == kshape[3] and shape[1] >= 1 and shape[1] % kshape[1] == 0 and
          stride[2] == 1, f"{what}: q must be [T, Hq, D] of the pages' type, Hq a multiple of Hkv")
    if rows is None:
        rows = shape[0]
    ts, tst = block_table.shape, block_table.stride()
    _need(block_table.dtype is torch.int32 and block_table.get_device() == index and
          len(ts) == 2 and ts[0] == rows and ts[1] > 0 and (tst[1] == 1 or ts[1] == 1) and
          (rows <= 1 or tst[0] >= ts[1]),
          f"{what}: block_table must be int32 CUDA [requests, width], its rows apart")
    _vector(lens, rows, torch.int32, index, f"{what}: lens must be int32 CUDA [requests]")
    if slopes is not None:
        _vector(slopes, shape[1], torch.float32, index, f"{what}: slopes must be fp32 CUDA [Hq]")
    _need(0.0 <= softcap < float("inf"), f"{what}: softcap must be finite and not negative")
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=k_pages.device)
        ost = (shape[1] * shape[2], shape[2])
    else:
        _need(out.get_device() == index and out.dtype is dtype and out.shape == shape and
              out.stride(2) == 1, f"{what}: out must have the shape and type of q")
        ost = _strides(shape, out.stride())
    return out, shape, _strides(shape, stride), tst[0] if rows > 1 else ts[1], ts[1], ost


def _check_prefix(prefix_pages, prefix_len, ps, index, what):
    prefix_len = int(prefix_len)
    _need(prefix_len >= 0, f"{what}: prefix_len must not be negative")
    if prefix_len:
        _need(prefix_pages is not None, f"{what}: prefix_len needs prefix_pages")
        _vector(prefix_pages, None, torch.int32, index,
                f"{what}: prefix_pages must be int32 CUDA [pages]")
        _need(prefix_pages.numel() * ps >= prefix_len,
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
    c, index, kshape = _cache(k_pages, v_pages, "prefill_attention")
    _need(_vec(cu_new, torch.int32, index) and cu_new.numel() >= 1,
          "prefill_attention: cu_new must be int32 CUDA [R + 1]")
    R = cu_new.numel() - 1
    out, (T, Hq, D), qst, tst, W, ost = _check_attention(
        q, k_pages, index, kshape, block_table, lens, R, slopes, softcap, out,
        "prefill_attention")
    if bidir is not None:
        _vector(bidir, R, torch.int32, index, "prefill_attention: bidir must be int32 CUDA [R]")
    prefix_len = _check_prefix(prefix_pages, prefix_len, kshape[2], index, "prefill_attention")
    dev = k_pages.device
    nws = _size("paged_prefill_attention", dev, T, R, Hq, kshape[1], D, W, kshape[2], prefix_len)
    ws = _workspace(nws, dev)
    st = _call("paged_prefill_attention", dev, q.data_ptr(), qst[0], qst[1], ctypes.byref(c),
               block_table.data_ptr(), tst, W, cu_new.data_ptr(), lens.data_ptr(), _ptr(bidir),
               prefix_pages.data_ptr() if prefix_len else None, prefix_len, _ptr(slopes), scale,
               softcap, out.data_ptr(), ost[0], ost[1], T, R, Hq, _ptr(ws), nws)
    if st:
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
    c, index, kshape = _cache(k_pages, v_pages, "decode_attention")
    out, (B, Hq, D), qst, tst, W, ost = _check_attention(
        q, k_pages, index, kshape, block_table, lens, None, slopes, softcap, out,
        "decode_attention")
    prefix_len = _check_prefix(prefix_pages, prefix_len, kshape[2], index, "decode_attention")
    dev = k_pages.device
    nws = _size("paged_decode_attention", dev, B, Hq, kshape[1], D, W, kshape[2], prefix_len)
    ws = _workspace(nws, dev)
    st = _call("paged_decode_attention", dev, q.data_ptr(), qst[0], qst[1], ctypes.byref(c),
               block_table.data_ptr(), tst, W, lens.data_ptr(),
               prefix_pages.data_ptr() if prefix_len else None, prefix_len, _ptr(slopes), scale,
               softcap, out.data_ptr(), ost[0], ost[1], B, Hq, _ptr(ws), nws)
    if st:
        _lib.check(st, "decode_attention")
    return out

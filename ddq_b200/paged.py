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

from typing import NamedTuple, Optional

import torch

from . import _lib


class StepPlan(NamedTuple):
    """What ``plan_step`` returns (device tensors)."""
    cu_new: torch.Tensor     # int32 [R + 1] first token row of each request
    lens: torch.Tensor       # int32 [R] tokens in the cache after the step
    slots: torch.Tensor      # int64 [T] page * page_size + row; -1: none
    positions: torch.Tensor  # int64 [T]
    seq_ids: torch.Tensor    # int32 [T] request of the row; -1 behind the last
    free_head: torch.Tensor  # int32 [1] first page of the free list not handed out


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
    return StepPlan._make(_lib.load_paged().plan_step(
        cached, new, block_table, free_pages, page_size, num_tokens, free_head, prefix_len))


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
    return _lib.load_paged().rope_kv_write(qkv, k_pages, v_pages, cos, sin, slots, positions,
                                           num_heads, num_kv_heads, head_dim, out)


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
    request with ``j <= p`` (and, with ``bidir`` int32 [R], the prefix and the
    first ``bidir[r]`` own keys whatever its position); scores ``scale * q.k``, with
    ``softcap`` > 0 capped to ``softcap * tanh(s / softcap)``, minus
    ``slopes[h] * |p - j|`` with ``slopes`` fp32 [Hq].
    A row without keys is zero.  Rows of ``out`` behind ``cu_new[R]`` are left
    as they are; where ``cu_new`` exceeds T (a step planned with too few token
    rows) the rows that exist keep their positions.  Keys and values of a request
    must be finite; the rest of its last page may hold anything.

    The key axis is split by what ``block_table`` could hold: where the longest
    request is known on the host, pass the columns that it uses
    (``block_table[:, :n]``, no copy).  Scores and softmax statistics are fp32; a weight is rounded once to the type of
    the pages on its way to the weighted sum (``ddq_b200.h`` says how exact the rest
    is)."""
    return _lib.load_paged().prefill_attention(q, k_pages, v_pages, block_table, cu_new, lens,
                                               scale, softcap, slopes, bidir, prefix_pages,
                                               prefix_len, out)


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
    keys gives zeros.  At most 8192 sequences.  The weights of the own keys reach the
    weighted sum in two parts (22 bits in fp16, 16 in bf16), those of the prefix in one."""
    return _lib.load_paged().decode_attention(q, k_pages, v_pages, block_table, lens, scale,
                                              prefix_pages, prefix_len, softcap, slopes, out)

"""Host-side mirror of the reference's operator wrappers (``python/hogwild/attention.py:12-90``).

Same function names, argument order and meaning as the reference, so code written against
``hogwild.attention`` can import this module instead.  Every function ends in a
``torch.ops.libhogatt.*`` call that is served by the CUDA library of this package; there is no
eager / CPU implementation here (the reference's ``hogwild_sdpa_pt`` lives on as the test oracle
only), and importing this module fails loudly when the compiled library cannot be loaded.
"""
from __future__ import annotations

import os
from typing import List, Optional, Sequence, Tuple

import torch

_PKG = os.path.dirname(os.path.abspath(__file__))
TORCH_LIB = os.path.join(_PKG, "hogatt.abi3.so")


def _load_ops() -> None:
    if hasattr(torch.ops, "libhogatt") and hasattr(torch.ops.libhogatt, "hogwild_fused"):
        return
    if not os.path.exists(TORCH_LIB):
        raise ImportError(f"{TORCH_LIB} is missing: run `python -m inference_lib_b200._build` (no fallback exists)")
    torch.ops.load_library(TORCH_LIB)


_load_ops()

# the operators' overloads, looked up once: a call through torch.ops.libhogatt.<name> finds them anew, 1 us of a 13 us decode call
_SDPA = torch.ops.libhogatt.hogwild_sdpa.default
_ROPE = torch.ops.libhogatt.hogwild_rope.default
_FUSED = torch.ops.libhogatt.hogwild_fused.default
_FUSED_PLANNED = torch.ops.libhogatt.hogwild_fused_planned.default
_PAGED_SDPA = torch.ops.libhogatt.hogwild_paged_sdpa.default
_VARLEN_PAGED_SDPA = torch.ops.libhogatt.hogwild_varlen_paged_sdpa.default
_COPY_TO_BLOCKS = torch.ops.libhogatt.copy_to_blocks.default
_COPY_TO_BLOCKS_NEW_ROWS = torch.ops.libhogatt.copy_to_blocks.new_rows
_PAGED_SDPA_Q4 = torch.ops.libhogatt.hogwild_paged_sdpa_q4.default
_VARLEN_PAGED_SDPA_Q4 = torch.ops.libhogatt.hogwild_varlen_paged_sdpa_q4.default
_PAGED_SDPA_Q4_NEW = torch.ops.libhogatt.hogwild_paged_sdpa_q4.new
_VARLEN_PAGED_SDPA_Q4_NEW = torch.ops.libhogatt.hogwild_varlen_paged_sdpa_q4.new
_COPY_TO_BLOCKS_Q4 = torch.ops.libhogatt.copy_to_blocks_q4.default
_COPY_FROM_BLOCKS_Q4_NEW = torch.ops.libhogatt.copy_from_blocks_q4.new
_STEP_BLOCKS = torch.ops.libhogatt.step_blocks.default
_STEP_BLOCKS_NEW = torch.ops.libhogatt.step_blocks.new
_COMPACT_BLOCKS = torch.ops.libhogatt.compact_blocks.default
_COMPACT_BLOCKS_NEW = torch.ops.libhogatt.compact_blocks.new
fragment_append = torch.ops.libhogatt.fragment_append.default              # FragmentCache.update's two steps
fragment_step_plan = torch.ops.libhogatt.fragment_step_plan.default


def hogwild_fused(queries: torch.Tensor, locations: torch.Tensor, keys: List[torch.Tensor], values: List[torch.Tensor],
                  scale: float, fragment_lengths: torch.Tensor, cosines: torch.Tensor, sines: torch.Tensor, *,
                  rotated_queries: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """Query RoPE per fragment + attention over all fragments (``attention.py:19-23``).

    ``queries [W,Hq,S,E]`` un-rotated; ``rotated_queries [F,W,Hq,S,E]`` and ``out [W,Hq,S,Ev]`` are
    caller-owned buffers that are overwritten.
    """
    _FUSED(out, rotated_queries, scale, locations, queries.contiguous(), fragment_lengths,
           keys, values, cosines, sines)
    return out


def hogwild_fused_planned(queries: torch.Tensor, locations: torch.Tensor, keys: List[torch.Tensor],
                          values: List[torch.Tensor], scale: float, fragment_lengths: torch.Tensor, cosines: torch.Tensor,
                          sines: torch.Tensor, *, rotated_queries: torch.Tensor, out: torch.Tensor,
                          host_lengths: List[int], stable_fragments: int = 0) -> torch.Tensor:
    """:func:`hogwild_fused` for fragments kept in preallocated slabs ``[Hkv, capacity, E]`` (no copies are made;
    the slabs must be contiguous).  ``host_lengths[f]`` is an upper bound, known on the host, of fragment ``f``'s
    current length (the true lengths stay on the device in ``fragment_lengths``); ``stable_fragments`` leading
    fragments are not written by work enqueued before this call, e.g. the shared prompt.  With both, the kernel
    starts streaming keys and values without reading anything from device memory first.  No counterpart in the
    reference, whose fragment tensors always end at the fragment's length."""
    _FUSED_PLANNED(out, rotated_queries, scale, locations, queries.contiguous(),
                   fragment_lengths, keys, values, cosines, sines,
                   [int(x) for x in host_lengths], int(stable_fragments))
    return out


def hogwild_sdpa(queries: torch.Tensor, locations: torch.Tensor, keys: List[torch.Tensor], values: List[torch.Tensor],
                 scale: float, fragment_lengths: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention over fragments with already-rotated ``queries [F,W,Hq,S,E]`` (``attention.py:26-35``)."""
    if out is None:
        out = torch.empty((queries.size(1), queries.size(2), queries.size(3), values[0].size(-1)),
                          dtype=queries.dtype, device=queries.device)
    if fragment_lengths is None:
        fragment_lengths = torch.tensor([k.size(-2) for k in keys], dtype=torch.int32, device=queries.device)
    keys = [k.contiguous() for k in keys]
    values = [v.contiguous() for v in values]
    _SDPA(out, scale, locations, queries.contiguous(), fragment_lengths, keys, values)
    return out


def hogwild_rope(queries: torch.Tensor, cosines: torch.Tensor, sines: torch.Tensor,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``[W,Hq,S,E]`` queries -> ``[F,W,Hq,S,E]``, one rotation per fragment (``attention.py:70-74``)."""
    if out is None:
        out = torch.empty((cosines.size(0), queries.size(0), queries.size(1), queries.size(2), queries.size(3)),
                          dtype=queries.dtype, device=queries.device)
    _ROPE(out, queries, cosines, sines)
    return out


def hogwild_paged_sdpa(queries: torch.Tensor, locations: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                       block_table: torch.Tensor, scale: float, fragment_lengths: torch.Tensor,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Paged attention: ``queries [F,W,Hq,S,E]`` (rotated), worker ``w`` reads the paged sequence
    ``block_table[w]`` of ``key_cache / value_cache [NumBlocks,Hkv,bs,E]``.  The reference registers this
    operator (``src/binding.cu:368-369``) but ships no Python wrapper for it."""
    if out is None:
        out = torch.empty((queries.size(1), queries.size(2), queries.size(3), value_cache.size(3)),
                          dtype=queries.dtype, device=queries.device)
    _PAGED_SDPA(out, scale, locations, queries.contiguous(), fragment_lengths, key_cache,
                value_cache, block_table)
    return out


def hogwild_varlen_paged_sdpa(queries: torch.Tensor, locations: torch.Tensor, key_cache: torch.Tensor,
                              value_cache: torch.Tensor, block_table: torch.Tensor, scale: float,
                              fragment_lengths: torch.Tensor, cu_seqlens_q: torch.Tensor,
                              cu_seqlens_k: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Packed-query paged attention: ``queries [F,total_q,Hq,E]``, ``locations [F,total_q]``,
    ``fragment_lengths [F,W]``, ``cu_seqlens_q [W+1]`` (``src/binding.cu:372-374``)."""
    if out is None:
        out = torch.empty((queries.size(1), queries.size(2), value_cache.size(3)), dtype=queries.dtype, device=queries.device)
    if cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens_q
    _VARLEN_PAGED_SDPA(out, scale, locations, queries.contiguous(), fragment_lengths, key_cache,
                       value_cache, block_table, cu_seqlens_q, cu_seqlens_k)
    return out


def copy_to_blocks(key_states: torch.Tensor, value_states: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                   block_table: torch.Tensor, seq_lengths: torch.Tensor, *, new_rows: Optional[torch.Tensor] = None) -> None:
    """Append ``key_states / value_states [B,Hkv,S_new,E]`` to the paged caches at ``seq_lengths[b] + t``
    (``src/binding.cu:370-371``).  Rows whose page the table does not name are dropped; ``new_rows [B]``: rows from there on stay out (what
    :func:`step_blocks` returns as ``room``)."""
    if new_rows is not None:
        _COPY_TO_BLOCKS_NEW_ROWS(key_states.contiguous(), value_states.contiguous(), key_cache, value_cache, block_table, seq_lengths, new_rows)
        return
    _COPY_TO_BLOCKS(key_states.contiguous(), value_states.contiguous(), key_cache, value_cache,
                    block_table, seq_lengths)


# ---- a paged cache in 4 bits (no counterpart in the reference) -----------------------------------------------------
# Codes ``uint8 [NumBlocks,Hkv,bs,E/2]`` (two e2m1 values a byte, the even channel in the low half), scales ``float8_e4m3fn
# [NumBlocks,Hkv,bs,E/16]``, one per 16 channels: value = e2m1(code) * scale * unit.  ``key_unit`` / ``value_unit`` are powers of two that
# belong to a cache (1 suits magnitudes from 0.1 to 2,688).  ``status`` (optional, int32) gets the C ABI's status bits ORed in.

def hogwild_paged_sdpa_q4(queries: torch.Tensor, locations: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                          key_scales: torch.Tensor, value_scales: torch.Tensor, block_table: torch.Tensor, scale: float,
                          fragment_lengths: torch.Tensor, out: Optional[torch.Tensor] = None, *, key_unit: float = 1.0,
                          value_unit: float = 1.0, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`hogwild_paged_sdpa` over a 4-bit cache: ``queries [F,W,Hq,S,E]`` (rotated) and ``out [W,Hq,S,Ev]`` in fp32, fp16 or bf16."""
    if out is None:
        return _PAGED_SDPA_Q4_NEW(scale, locations, queries.contiguous(), fragment_lengths, key_cache, value_cache, key_scales, value_scales,
                                  block_table, key_unit, value_unit, status)
    _PAGED_SDPA_Q4(out, scale, locations, queries.contiguous(), fragment_lengths, key_cache, value_cache, key_scales, value_scales,
                   block_table, key_unit, value_unit, status)
    return out


def hogwild_varlen_paged_sdpa_q4(queries: torch.Tensor, locations: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                                 key_scales: torch.Tensor, value_scales: torch.Tensor, block_table: torch.Tensor, scale: float,
                                 fragment_lengths: torch.Tensor, cu_seqlens_q: torch.Tensor, out: Optional[torch.Tensor] = None, *,
                                 key_unit: float = 1.0, value_unit: float = 1.0, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`hogwild_varlen_paged_sdpa` over a 4-bit cache: ``queries [F,total_q,Hq,E]``, ``locations [F,total_q]``,
    ``fragment_lengths [F,W]``, ``cu_seqlens_q [W+1]``.  Rows of ``out`` behind the last sequence are left as they are."""
    if out is None:
        return _VARLEN_PAGED_SDPA_Q4_NEW(scale, locations, queries.contiguous(), fragment_lengths, key_cache, value_cache, key_scales,
                                         value_scales, block_table, cu_seqlens_q, key_unit, value_unit, status)
    _VARLEN_PAGED_SDPA_Q4(out, scale, locations, queries.contiguous(), fragment_lengths, key_cache, value_cache, key_scales, value_scales,
                          block_table, cu_seqlens_q, key_unit, value_unit, status)
    return out


def copy_to_blocks_q4(key_states: torch.Tensor, value_states: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                      key_scales: torch.Tensor, value_scales: torch.Tensor, block_table: torch.Tensor, seq_lengths: torch.Tensor, *,
                      cu_seqlens: Optional[torch.Tensor] = None, new_rows: Optional[torch.Tensor] = None, key_unit: float = 1.0,
                      value_unit: float = 1.0, status: Optional[torch.Tensor] = None) -> None:
    """:func:`copy_to_blocks` into a 4-bit cache: row ``t`` of sequence ``b`` is stored at position ``seq_lengths[b] + t``.  The states
    are ``[B,Hkv,S,E]`` with any strides (the transposed view of a projection's output is taken as it is) or, with ``cu_seqlens [B+1]``,
    packed ``[T,Hkv,E]``.  ``new_rows [B]``: rows from there on stay out (what :func:`step_blocks` returns as ``room``).  Rows whose page
    the table does not name are dropped."""
    _COPY_TO_BLOCKS_Q4(key_states, value_states, key_cache, value_cache, key_scales, value_scales, block_table, seq_lengths, cu_seqlens,
                       new_rows, key_unit, value_unit, status)


def copy_from_blocks_q4(key_cache: torch.Tensor, value_cache: torch.Tensor, key_scales: torch.Tensor, value_scales: torch.Tensor,
                        block_table: torch.Tensor, first_rows: torch.Tensor, rows: int, *, dtype: torch.dtype = torch.bfloat16,
                        key_unit: float = 1.0, value_unit: float = 1.0,
                        status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The numbers that a 4-bit cache holds: rows ``first_rows[b]`` ... ``first_rows[b] + rows - 1`` of every sequence of ``block_table``,
    as keys ``[B,Hkv,rows,E]`` and values ``[B,Hkv,rows,Ev]``.  Rows without a page are NaN."""
    return _COPY_FROM_BLOCKS_Q4_NEW(key_cache, value_cache, key_scales, value_scales, block_table, first_rows, rows, dtype, key_unit, value_unit,
                                    status)


# ---- the pages of a paged cache of any type (no counterpart in the reference) ------------------------------------------
# ``block_refs[p]`` counts the block-table entries that name page ``p`` (plus what a caller adds to keep a page); 0: free.  A row without
# pages has -1 in its table: append with ``new_rows=room``, and let queries over 16-bit pages see no further than ``lengths + room``.

def step_blocks(block_refs: torch.Tensor, block_table: torch.Tensor, seq_lengths: torch.Tensor, caches: Sequence[torch.Tensor],
                block_size: int, *, source: Optional[torch.Tensor] = None, new_tokens: Optional[torch.Tensor] = None,
                out: Optional[Sequence[torch.Tensor]] = None,
                status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """One step of a batch's pages: row ``w`` of the new table is row ``source[w]`` of the old one (``None``: every row stays; negative: an
    empty row; several rows may take over the same one and then share its pages; rows that nobody takes over are freed), and every
    row gets the pages for ``new_tokens[w]`` tokens behind its length, lowest free page first.  A last page that is partly filled and
    shared is copied, in all ``caches`` (every tensor ``[NumBlocks,...]`` of every layer: keys, values, scales), unless its row is the last
    holder.  Returns ``(block_refs, block_table, seq_lengths, room)`` in new tensors or in ``out``: lengths without the new tokens, and
    ``room[w]`` = ``new_tokens[w]`` where the row has its pages, otherwise 0 (rows are served in order until the pool is empty).  ``out`` may
    hold the inputs themselves where there is no ``source``; ``block_refs`` always.  Nothing is read back from the device."""
    if out is None:
        return _STEP_BLOCKS_NEW(block_refs, block_table, seq_lengths, source, new_tokens, block_size, caches, status)
    refs, table, lengths, room = out
    _STEP_BLOCKS(block_refs, block_table, seq_lengths, source, new_tokens, block_size, caches, refs, table, lengths, room, status)
    return refs, table, lengths, room


def compact_blocks(block_refs: torch.Tensor, block_table: torch.Tensor, caches: Sequence[torch.Tensor], *,
                   out: Optional[Sequence[torch.Tensor]] = None,
                   status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Moves the held pages to the front of ``caches`` (in place) and returns ``(block_refs, block_table, moved)`` in new tensors or in
    ``out`` (which may hold the inputs): ``moved[p]`` is page ``p``'s new number, -1 for a free one.  The pages that are held end up as
    ``0 .. n-1``; one that was there already stays."""
    if out is None:
        return _COMPACT_BLOCKS_NEW(block_refs, block_table, caches, status)
    refs, table, moved = out
    _COMPACT_BLOCKS(block_refs, block_table, caches, refs, table, moved, status)
    return refs, table, moved


def rotate_half(x: torch.Tensor) -> torch.Tensor:
    """``attention.py:77-81``."""
    h = x.shape[-1] // 2
    return torch.cat((-x[..., h:], x[..., :h]), dim=-1)


def apply_rotary_pos_emb(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, unsqueeze_dim: int = 1) -> torch.Tensor:
    """Key-side RoPE used when new keys are written to a fragment (``attention.py:84-90``, call site ``:315``)."""
    cos, sin = cos.unsqueeze(unsqueeze_dim), sin.unsqueeze(unsqueeze_dim)
    r = cos.shape[-1]
    head, tail = x[..., :r], x[..., r:]
    return torch.cat(((head * cos) + (rotate_half(head) * sin), tail), dim=-1).to(x.dtype)

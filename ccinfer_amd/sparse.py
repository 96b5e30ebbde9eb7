"""Decode over the blocks of a long context that a cheap score selects.

Beside each layer's K lie its key_bounds, bf16 [blocks, heads, 2, head_dim]: the smallest and the
largest of each block's keys, element by element. A step writes its token (write_kv_cache and the
like), renews the bounds of the block that it fell into, scores the row's blocks, selects and
attends:

    update_key_bounds(k, bounds, table, ctx)
    scores = score_kv_blocks(q, bounds, table, ctx)
    selected = select_kv_blocks(scores, ctx, 128)
    o = sparse_decode_attention(q, k, v, table, ctx, selected)

Conventions are those of `ops`; blocks of 16 tokens, head dims in multiples of 8 up to 256 (64 and
128 over an fp8 cache). Several query tokens of one request are rows of their own in all of these
calls, with the same table row and the context length that each sees.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .drafts import _one_layer, _table
from .ops import (CcinferError, _require, _size, _stream, _workspace, current_device,
                  fp8_scale_numel)
from .pages import _index

_I32 = torch.int32
_BF16 = torch.bfloat16


def _bounds(key_bounds: torch.Tensor, dev: int, op: str):
    """(blocks, heads, head_dim) of key bounds."""
    _require(key_bounds.dim() == 4 and key_bounds.dtype is _BF16 and key_bounds.get_device() == dev
             and key_bounds.is_contiguous() and key_bounds.shape[2] == 2, op)
    blocks, hkv, _, d = key_bounds.shape
    _require(blocks < 2 ** 31 > hkv and d < 2 ** 31, op)
    return blocks, hkv, d


def _query(q: torch.Tensor, rows: int, d, dev: int, op: str) -> int:
    """Query heads of a decode batch's q."""
    _require(q.dim() == 3 and q.dtype is _BF16 and q.get_device() == dev and q.is_contiguous()
             and q.shape[0] == rows and q.shape[2] == d and q.shape[1] < 2 ** 31, op)
    return q.shape[1]


def update_key_bounds(k_cache: torch.Tensor, key_bounds: torch.Tensor, block_table: torch.Tensor,
                      context_lens: torch.Tensor,
                      query_start_loc: Optional[torch.Tensor] = None,
                      k_scale: Optional[torch.Tensor] = None, cache_block_size: int = 16) -> None:
    """Renews key_bounds of the blocks that hold each row's newest tokens: one token a row, or
    query_start_loc[b + 1] - query_start_loc[b] (as a prefill or a tree of drafts wrote; after
    accept_draft_tokens the tree's own query_start_loc with the shorter contexts), from all
    their positions below the context length. Rows may share blocks (a row for each query token of a
    request): the longest context counts. A NaN key makes both bounds of its element NaN."""
    op = "update_key_bounds"
    _require(k_cache.is_cuda, op)
    dev = current_device()
    blocks, hkv, d = _bounds(key_bounds, dev, op)
    rows, width = _table(block_table, context_lens, dev, op)
    dims = k_cache.dim()
    _require(3 <= dims <= 4 and k_cache.dtype is (_BF16 if k_scale is None else torch.uint8)
             and k_cache.get_device() == dev and k_cache.is_contiguous()
             and k_cache.shape[-2:] == (hkv, d) and 0 < cache_block_size < 2 ** 31
             and (dims == 3 or k_cache.shape[1] == cache_block_size)
             and k_cache.numel() <= blocks * cache_block_size * hkv * d
             and (query_start_loc is None or _index(query_start_loc, dev, op) == rows + 1), op)
    if k_scale is not None:
        slots = k_cache.numel() // max(1, hkv * d)
        _require(k_scale.dtype is torch.float32 and k_scale.get_device() == dev
                 and k_scale.is_contiguous() and k_scale.numel() >= fp8_scale_numel(slots, hkv), op)
    code = _lib.load().ccinfer_update_key_bounds(
        k_cache.data_ptr() or None, None if k_scale is None else k_scale.data_ptr(),
        key_bounds.data_ptr() or None, block_table.data_ptr() or None,
        context_lens.data_ptr() or None,
        None if query_start_loc is None else query_start_loc.data_ptr(), rows, width, hkv, d,
        cache_block_size, _stream())
    if code:
        raise CcinferError(code, op)


def score_kv_blocks(q: torch.Tensor, key_bounds: torch.Tensor, block_table: torch.Tensor,
                    context_lens: torch.Tensor, cache_block_size: int = 16,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """float32 [rows, kv heads, max_blocks_per_req]: the largest logit that any key within a
    block's bounds could have with any query head of the kv head, sum_d max(q_d lo_d, q_d hi_d) /
    sqrt(head_dim). -inf past the context, for negative table entries, and for rows whose context
    the table does not hold; NaN for NaN bounds, NaN or an infinity for infinite ones. q [rows, q
    heads, head_dim]."""
    op = "score_kv_blocks"
    _require(q.is_cuda, op)
    dev = current_device()
    _, hkv, d = _bounds(key_bounds, dev, op)
    rows, width = _table(block_table, context_lens, dev, op)
    hq = _query(q, rows, d, dev, op)
    _require(0 < cache_block_size < 2 ** 31, op)
    if out is None:
        out = torch.empty(rows, hkv, width, dtype=torch.float32, device=q.device)
    else:
        _require(out.dtype is torch.float32 and out.get_device() == dev and out.is_contiguous()
                 and out.shape == (rows, hkv, width), op)
    code = _lib.load().ccinfer_score_kv_blocks(
        q.data_ptr() or None, key_bounds.data_ptr() or None, block_table.data_ptr() or None,
        context_lens.data_ptr() or None, out.data_ptr() or None, rows, width, hq, hkv, d,
        cache_block_size, _stream())
    if code:
        raise CcinferError(code, op)
    return out


def select_kv_blocks(scores: torch.Tensor, context_lens: torch.Tensor, num_selected: int,
                     first_blocks: int = 1, last_blocks: int = 1, cache_block_size: int = 16,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """int32 [rows, kv heads, num_selected]: numbers within the row of its first `first_blocks` and
    last `last_blocks` blocks and of the others with the highest scores (NaN before all others,
    equal ones by the lower number), ascending; -1 behind them where the row has fewer."""
    op = "select_kv_blocks"
    _require(scores.is_cuda, op)
    dev = current_device()
    _require(scores.dim() == 3 and scores.dtype is torch.float32 and scores.get_device() == dev
             and scores.is_contiguous(), op)
    rows, hkv, width = scores.shape
    _require(_index(context_lens, dev, op) == rows and rows < 2 ** 31 > hkv and width < 2 ** 31
             and 0 < num_selected < 2 ** 31 and 0 <= first_blocks < 2 ** 31
             and 0 <= last_blocks < 2 ** 31 and 0 < cache_block_size < 2 ** 31, op)
    if out is None:
        out = torch.empty(rows, hkv, num_selected, dtype=_I32, device=scores.device)
    else:
        _index(out, dev, op)
        _require(out.shape == (rows, hkv, num_selected), op)
    code = _lib.load().ccinfer_select_kv_blocks(
        scores.data_ptr() or None, context_lens.data_ptr() or None, rows, width, hkv, num_selected,
        first_blocks, last_blocks, cache_block_size, out.data_ptr() or None, _stream())
    if code:
        raise CcinferError(code, op)
    return out


def sparse_decode_workspace_size(batch_size: int, num_q_heads: int, num_kv_heads: int,
                                 head_dim: int, num_selected: int,
                                 cache_block_size: int = 16) -> int:
    """Workspace bytes of sparse_decode_attention (0: none needed, or an invalid shape)."""
    return int(_lib.load().ccinfer_sparse_decode_workspace_size(
        batch_size, num_q_heads, num_kv_heads, head_dim, num_selected, cache_block_size))


def sparse_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                            block_table: torch.Tensor, context_lens: torch.Tensor,
                            selected: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                            v_scale: Optional[torch.Tensor] = None,
                            output: Optional[torch.Tensor] = None, cache_block_size: int = 16,
                            workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """decode_attention of each (row, kv head) over the positions in its blocks `selected` (int32
    [rows, kv heads, n], numbers within the row; ones outside the context are passed over, one that
    is named twice counts twice). Zeros for a row that sees nothing; returns output."""
    op = "sparse_decode_attention"
    _require(q.is_cuda, op)
    dev = current_device()
    rows, width = _table(block_table, context_lens, dev, op)
    d = q.shape[-1]
    hq = _query(q, rows, d, dev, op)
    hkv = _one_layer(k_cache, v_cache, k_scale, v_scale, d, cache_block_size, dev, op)
    _index(selected, dev, op)
    _require(selected.dim() == 3 and selected.shape[:2] == (rows, hkv)
             and 0 < selected.shape[2] < 2 ** 31 > hkv and 0 < cache_block_size < 2 ** 31, op)
    take = selected.shape[2]
    if output is None:
        output = torch.empty_like(q)
    else:
        _require(output.dtype is _BF16 and output.get_device() == dev and output.is_contiguous()
                 and output.shape == q.shape, op)
    ws, ws_bytes = _workspace(_size(sparse_decode_workspace_size, rows, hq, hkv, d, take,
                                          cache_block_size), q.device, workspace)
    code = _lib.load().ccinfer_sparse_decode_attention(
        q.data_ptr() or None, k_cache.data_ptr() or None, v_cache.data_ptr() or None,
        None if k_scale is None else k_scale.data_ptr(),
        None if v_scale is None else v_scale.data_ptr(), block_table.data_ptr() or None,
        context_lens.data_ptr() or None, selected.data_ptr(), output.data_ptr() or None, rows,
        width, hq, hkv, d, take, cache_block_size, None if ws is None else ws.data_ptr(), ws_bytes,
        _stream())
    if code:
        raise CcinferError(code, op)
    return output

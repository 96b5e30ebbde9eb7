"""Steps that check several drafted tokens a request: trees of drafts, their attention over the
paged cache, and what the model confirms of them.

Conventions are those of `ops` and `pages`: device tensors on the current device, work on torch's
current stream, nothing synchronised, CcinferError with the reference's codes for what the host can
see and a device status word a request for what it cannot.

  parents           [total] int32: the request's node that each node goes on from, -1: the context
  query_start_loc   [requests + 1] int32: rows of each request's nodes
  context_lens      [requests] int32, the nodes counted: node i of n lies at position context - n + i
  tree_mask         [total, words] int32: bit j of a row, bit j % 32 of word j // 32: it sees node j
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .ops import (INVALID_ARGUMENT, CcinferError, _require, _size, _stream, _workspace,
                  current_device, fp8_scale_numel)
from .pages import _index, _layers

_I32 = torch.int32


def _one_layer(k_cache, v_cache, k_scale, v_scale, head_dim: int, block_size: int, dev: int,
               op: str) -> int:
    """Checks one layer's cache ([slots, heads, head_dim] or [blocks, block_size, heads, head_dim]);
    returns its kv heads."""
    dtype = torch.bfloat16 if k_scale is None else torch.uint8
    shape = k_cache.shape
    _require(3 <= len(shape) <= 4 and k_cache.dtype is dtype and v_cache.dtype is dtype
             and v_cache.shape == shape and shape[-1] == head_dim
             and (len(shape) == 3 or shape[1] == block_size)
             and k_cache.get_device() == dev and v_cache.get_device() == dev
             and k_cache.is_contiguous() and v_cache.is_contiguous()
             and (k_scale is None) == (v_scale is None), op)
    hkv = shape[-2]
    if k_scale is not None:
        slots = shape[0] if len(shape) == 3 else shape[0] * shape[1]
        need = fp8_scale_numel(slots, hkv)
        for s in (k_scale, v_scale):
            _require(s.dtype is torch.float32 and s.get_device() == dev and s.is_contiguous()
                     and s.numel() >= need, op)
    return hkv


def _table(block_table: torch.Tensor, context_lens: torch.Tensor, dev: int, op: str):
    """(rows, max_blocks_per_req) of a block table that fits its contexts."""
    if block_table.dim() != 2:
        raise CcinferError(INVALID_ARGUMENT, op)
    rows, width = block_table.shape
    _index(block_table, dev, op)
    _require(_index(context_lens, dev, op) == rows and rows < 2 ** 31 > width, op)
    return rows, width


def build_draft_tree(parents: torch.Tensor, query_start_loc: torch.Tensor,
                     context_lens: torch.Tensor, block_table: torch.Tensor, max_nodes: int,
                     cache_block_size: int = 16, out: Optional[dict] = None) -> dict:
    """What a step needs of its trees, once for all layers: int32 device tensors tree_mask
    [total, words] (each node sees its ancestors and itself; words covers max_nodes), positions
    [total] (for rotary embeddings: committed tokens + depth), slot_mapping [total] (for the cache
    write) and status [requests]: 0, or 6 for a request with more than max_nodes nodes or fewer
    context tokens than nodes (its rows: no mask, -1, -1), with a parent that is no earlier node
    (taken as -1) or without a block for a node (slot -1). Rows of no request (a padded batch): no
    mask, -1, -1. At most 2048 nodes a request. `out` reuses tensors of an earlier call."""
    op = "build_draft_tree"
    _require(parents.is_cuda, op)
    dev = current_device()
    total = _index(parents, dev, op)
    rows, width = _table(block_table, context_lens, dev, op)
    _require(_index(query_start_loc, dev, op) == rows + 1 and 0 < max_nodes < 2 ** 31
             and total < 2 ** 31 and 0 < cache_block_size < 2 ** 31, op)
    words = -(-max_nodes // 32)
    if out is None:
        device = parents.device
        out = {"tree_mask": torch.empty(total, words, dtype=_I32, device=device),
               "positions": torch.empty(total, dtype=_I32, device=device),
               "slot_mapping": torch.empty(total, dtype=_I32, device=device),
               "status": torch.empty(rows, dtype=_I32, device=device)}
    mask = out["tree_mask"]
    _index(mask, dev, op)
    _require(mask.dim() == 2 and mask.shape[0] == total and words <= mask.shape[1] < 2 ** 31
             and _index(out["positions"], dev, op) == total
             and _index(out["slot_mapping"], dev, op) == total
             and _index(out["status"], dev, op) == rows, op)
    code = _lib.load().ccinfer_build_draft_tree(
        parents.data_ptr() or None, query_start_loc.data_ptr(), context_lens.data_ptr() or None,
        block_table.data_ptr() or None, rows, total, width, max_nodes, mask.shape[1],
        cache_block_size, mask.data_ptr(), out["positions"].data_ptr(),
        out["slot_mapping"].data_ptr(), out["status"].data_ptr(), _stream())
    if code:
        raise CcinferError(code, op)
    return out


def tree_attention_workspace_size(batch_size: int, total_query_tokens: int,
                                  max_blocks_per_req: int, mask_words: int, num_q_heads: int,
                                  num_kv_heads: int, head_dim: int,
                                  cache_block_size: int = 16) -> int:
    """Workspace bytes of tree_attention (0 for a shape that it does not take)."""
    return int(_lib.load().ccinfer_tree_attention_workspace_size(
        batch_size, total_query_tokens, max_blocks_per_req, mask_words, num_q_heads, num_kv_heads,
        head_dim, cache_block_size))


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   block_table: torch.Tensor, query_start_loc: torch.Tensor,
                   context_lens: torch.Tensor, tree_mask: torch.Tensor,
                   k_scale: Optional[torch.Tensor] = None,
                   v_scale: Optional[torch.Tensor] = None,
                   output: Optional[torch.Tensor] = None, cache_block_size: int = 16,
                   workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """prefill_attention of a request's new tokens with a mask among them in place of their order:
    each sees the committed context and the new tokens that its row of tree_mask names (written to
    the cache before the call, as in prefill). bf16 cache, or an fp8 one with k_scale and v_scale
    (head dims 64 and 128); at most 1024 requests; returns output.

    Rows that see nothing become zeros. Rows of no request, and of requests with fewer context
    tokens than nodes, keep the contents of `output` (uninitialised when `output` is None). K and V
    of nodes that a row does not see do not reach it, whatever they hold."""
    op = "tree_attention"
    _require(q.is_cuda and q.dim() == 3, op)
    dev = current_device()
    total, hq, d = q.shape
    hkv = _one_layer(k_cache, v_cache, k_scale, v_scale, d, cache_block_size, dev, op)
    rows, width = _table(block_table, context_lens, dev, op)
    _index(tree_mask, dev, op)
    _require(q.dtype is torch.bfloat16 and q.get_device() == dev and q.is_contiguous()
             and total < 2 ** 31 > hq and hkv < 2 ** 31 and 0 < cache_block_size < 2 ** 31
             and _index(query_start_loc, dev, op) == rows + 1 and tree_mask.dim() == 2
             and tree_mask.shape[0] == total and tree_mask.shape[1] < 2 ** 31, op)
    if output is None:
        output = torch.empty_like(q)
    else:
        _require(output.dtype is torch.bfloat16 and output.get_device() == dev
                 and output.is_contiguous() and output.shape == q.shape, op)
    words = tree_mask.shape[1]
    ws, ws_bytes = _workspace(_size(tree_attention_workspace_size, rows, total, width, words,
                                          hq, hkv, d, cache_block_size), q.device, workspace)
    code = _lib.load().ccinfer_tree_attention(
        q.data_ptr() or None, k_cache.data_ptr() or None, v_cache.data_ptr() or None,
        None if k_scale is None else k_scale.data_ptr(),
        None if v_scale is None else v_scale.data_ptr(), block_table.data_ptr() or None,
        query_start_loc.data_ptr(), context_lens.data_ptr() or None, tree_mask.data_ptr() or None,
        output.data_ptr() or None, rows, total, width, words, hq, hkv, d, cache_block_size,
        None if ws is None else ws.data_ptr(), ws_bytes, _stream())
    if code:
        raise CcinferError(code, op)
    return output


def accept_draft_tokens(draft_tokens: torch.Tensor, target_tokens: torch.Tensor,
                        parents: torch.Tensor, query_start_loc: torch.Tensor,
                        context_lens: torch.Tensor, block_table: torch.Tensor,
                        k_cache: Optional[torch.Tensor] = None,
                        v_cache: Optional[torch.Tensor] = None,
                        k_scale: Optional[torch.Tensor] = None,
                        v_scale: Optional[torch.Tensor] = None, cache_block_size: int = 16,
                        out: Optional[dict] = None,
                        status: Optional[torch.Tensor] = None) -> dict:
    """What the model confirms of the trees. draft_tokens [total]: the nodes' tokens; target_tokens
    [total]: what the model says after each node. A request's path starts at node 0 (the token that
    the last step ended with) and goes on to the lowest child whose drafted token is the target of
    its parent. The K and V of the path's nodes move to the positions right behind the committed
    tokens, in every layer of the caches (all layers, or one, as in `pages`).

    Returns int32 device tensors accepted [requests] (nodes of the path), accepted_nodes [total]
    (the path, from the request's first row on, -1 behind it), tokens [total] (the step's new
    tokens: the targets of those nodes, -1 behind them; the last is the next step's node 0) and
    context_lens [requests], the contexts without the rejected nodes: `lengths` of
    update_block_tables, which gives back the blocks that they filled. A request without nodes, or
    with more than 2048, accepts 0. Layers held one by one: the same call for each of them, with
    the context_lens that counts the nodes. `out` reuses tensors of an earlier call (none of them an
    input of this one); rows of no request keep what they hold there.

    `status`: the plan's. A request that the plan refused (status not 0) was not written to the cache,
    or not all of it, and what the model says after its nodes means nothing: it accepts 0, and its
    context loses the nodes. Without `status` such a request is walked like any other."""
    op = "accept_draft_tokens"
    _require(draft_tokens.is_cuda, op)
    dev = current_device()
    total = _index(draft_tokens, dev, op)
    rows, width = _table(block_table, context_lens, dev, op)
    _require(_index(target_tokens, dev, op) == total and _index(parents, dev, op) == total
             and _index(query_start_loc, dev, op) == rows + 1 and total < 2 ** 31
             and 0 < cache_block_size < 2 ** 31
             and (status is None or _index(status, dev, op) == rows), op)
    if k_cache is None:
        _require(v_cache is None and k_scale is None and v_scale is None, op)
        cache = (None, None, None, None, 0, 0, 0, 0, 0, 0, cache_block_size)
    else:
        _require(v_cache is not None, op)
        cache = _layers(k_cache, v_cache, k_scale, v_scale, cache_block_size, dev, op)
    if out is None:
        device = draft_tokens.device
        out = {"accepted": torch.empty(rows, dtype=_I32, device=device),
               "accepted_nodes": torch.empty(total, dtype=_I32, device=device),
               "tokens": torch.empty(total, dtype=_I32, device=device),
               "context_lens": torch.empty(rows, dtype=_I32, device=device)}
    lengths = out["context_lens"]
    _require(_index(out["accepted"], dev, op) == rows
             and _index(out["accepted_nodes"], dev, op) == total
             and _index(out["tokens"], dev, op) == total and _index(lengths, dev, op) == rows
             and (rows == 0 or lengths.data_ptr() != context_lens.data_ptr()), op)
    code = _lib.load().ccinfer_accept_planned_tokens(
        draft_tokens.data_ptr() or None, target_tokens.data_ptr() or None,
        parents.data_ptr() or None, query_start_loc.data_ptr(), context_lens.data_ptr() or None,
        block_table.data_ptr() or None, None if status is None else status.data_ptr(), rows, total,
        width, *cache, out["accepted"].data_ptr(), out["accepted_nodes"].data_ptr(),
        out["tokens"].data_ptr(), lengths.data_ptr(), _stream())
    if code:
        raise CcinferError(code, op)
    return out

"""Pages of the paged KV cache over the C ABI: blocks copied, block tables changed with counted
references, the pool compacted, for all layers in one call.

Conventions are those of `ops`: device tensors on the current device, work on torch's current
stream, nothing synchronised, CcinferError with the reference's codes for what the host can see
and a device status word for what it cannot (as in build_batch_metadata).

  k_cache, v_cache   one layer [slots, heads, head_dim] or [blocks, block_size, heads, head_dim],
                     or all layers [layers, blocks, block_size, heads, head_dim] (the layers may
                     lie apart, each is contiguous); bf16, or uint8 with k_scale / v_scale
                     (float32, [layers, fp8_scale_numel] beside caches of all layers)
  block_table        [rows, max_blocks_per_req] int32, -1 padded; context_lens [rows] int32
  ref_counts         [blocks] int32: owners of each block, 0 = free; a block given up more often
                     than it was counted is below 0 and not handed out again
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .ops import (INVALID_ARGUMENT, CcinferError, _check, _known_size, _require, _stream,
                  _workspace, current_device)

_I32 = torch.int32

KV_EXHAUSTED = 12      # status: not enough free blocks
KV_INVALID_TABLE = 14  # status: a table row that the pool does not hold


def _layers(k_cache, v_cache, k_scale, v_scale, block_size: int, dev: int, op: str):
    """The cache arguments of the C ABI: pointers, layers, strides, blocks, heads, head_dim,
    block_size."""
    fp8 = k_scale is not None
    dtype = torch.uint8 if fp8 else torch.bfloat16
    shape, stride = k_cache.shape, k_cache.stride()
    dims = len(shape)
    _require(3 <= dims <= 5 and 0 < block_size < 2 ** 31 and k_cache.dtype is dtype
             and v_cache.dtype is dtype and v_cache.shape == shape
             and k_cache.get_device() == dev and v_cache.get_device() == dev
             and fp8 == (v_scale is not None), op)
    h, d = shape[-2], shape[-1]
    layers, layer_stride, scale_stride = 1, 0, 0
    if dims == 5:
        layers, nb, bs = shape[:3]
        layer_stride = stride[0] * (1 if fp8 else 2)
        vstride = v_cache.stride()
        inner = (bs * h * d, h * d, d, 1)
        _require((stride == vstride or layers == 1 or vstride[0] == stride[0])
                 and (stride[1:] == inner or k_cache[0].is_contiguous())
                 and (vstride[1:] == inner or v_cache[0].is_contiguous())
                 and bs == block_size and layers < 2 ** 31 > nb and h < 2 ** 31 > d, op)
    else:
        nb, bs = (shape[0], shape[1]) if dims == 4 else (shape[0] // block_size, block_size)
        _require((dims == 4 or nb * bs == shape[0]) and k_cache.is_contiguous()
                 and v_cache.is_contiguous() and bs == block_size
                 and nb < 2 ** 31 > h and d < 2 ** 31, op)
    ksp = vsp = None
    if fp8:
        need = nb * h * 16
        for s in (k_scale, v_scale):
            _require(s.dtype is torch.float32 and s.get_device() == dev, op)
            if layers == 1:
                _require(s.is_contiguous() and s.numel() >= need, op)
            else:
                _require(s.dim() == 2 and s.shape[0] == layers and s.shape[1] >= need
                         and s.stride() == k_scale.stride() and s.stride(1) == 1, op)
        scale_stride = k_scale.stride(0) if layers > 1 else 0
        ksp, vsp = k_scale.data_ptr(), v_scale.data_ptr()
    return (k_cache.data_ptr(), v_cache.data_ptr(), ksp, vsp, layers, layer_stride, scale_stride,
            nb, h, d, bs)


def _index(t: torch.Tensor, dev: int, op: str) -> int:
    """Elements of a contiguous int32 tensor on the device."""
    if t.dtype is not _I32 or t.get_device() != dev or not t.is_contiguous():
        raise CcinferError(INVALID_ARGUMENT, op)
    return t.numel()


def copy_kv_blocks(k_cache: torch.Tensor, v_cache: torch.Tensor, src_blocks: torch.Tensor,
                   dst_blocks: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                   v_scale: Optional[torch.Tensor] = None, cache_block_size: int = 16,
                   status: Optional[torch.Tensor] = None) -> None:
    """Block dst_blocks[i] of every layer becomes a copy of src_blocks[i] (int32 [n]; K, V and
    the scales of an fp8 cache). Pairs with a block outside the pool (-1, say) are skipped, as
    are pairs that depend on an order: a destination that is another pair's destination with
    another source, or another pair's source. `status` (int32 [1]), if given, becomes 6 then
    and is left alone otherwise."""
    op = "copy_kv_blocks"
    _require(k_cache.is_cuda, op)
    dev = current_device()
    n = _index(src_blocks, dev, op)
    _require(2 ** 31 > _index(dst_blocks, dev, op) == n
             and (status is None or _index(status, dev, op) == 1), op)
    cache = _layers(k_cache, v_cache, k_scale, v_scale, cache_block_size, dev, op)
    code = _lib.load().ccinfer_copy_kv_blocks(
        *cache[:4], src_blocks.data_ptr() or None, dst_blocks.data_ptr() or None, n, *cache[4:],
        None if status is None else status.data_ptr(), _stream())
    if code:
        raise CcinferError(code, op)


def update_tables_workspace_size(num_items: int, max_blocks_per_req: int, num_blocks: int) -> int:
    """Workspace bytes of update_block_tables (0 for an invalid shape)."""
    return int(_lib.load().ccinfer_update_tables_workspace_size(num_items, max_blocks_per_req,
                                                                num_blocks))


def update_block_tables(block_table: torch.Tensor, context_lens: torch.Tensor,
                        ref_counts: torch.Tensor, dst_rows: torch.Tensor,
                        src_rows: Optional[torch.Tensor], lengths: Optional[torch.Tensor],
                        k_cache: Optional[torch.Tensor] = None,
                        v_cache: Optional[torch.Tensor] = None,
                        k_scale: Optional[torch.Tensor] = None,
                        v_scale: Optional[torch.Tensor] = None, cache_block_size: int = 16,
                        workspace: Optional[torch.Tensor] = None,
                        status: Optional[torch.Tensor] = None,
                        copies: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
                        ) -> torch.Tensor:
    """Makes row dst_rows[i] hold the first min(lengths[i], source's context) tokens of row
    src_rows[i] as it was before the call, then blocks for the tokens up to lengths[i]; changes
    block_table, context_lens and ref_counts in place. src_rows None: of the row itself, an
    entry -1: of none; lengths None or an entry -1: the source's context.

    So one call forks (child, parent, -1), admits (row, -1, tokens), grows and truncates
    (row, row, tokens), releases (row, -1, 0) and reorders beams (row, beam it continues, -1),
    any of them for different rows at once. Whole blocks are shared and counted; a last block
    filled in part, where it would be shared, is copied to one of the row's own. New blocks are
    the lowest-numbered that were free before the call, in item order; blocks it releases are
    free after it. Returns `status` (int32 [1]): 0, or, with nothing changed, 6 (a row or length
    out of range, a row twice in dst_rows, a copy needed but neither caches nor lists given), 14
    (a row with a context or blocks that the pool does not hold) or 12 (not enough free blocks).

    `copies`: two int32 tensors of as many elements as dst_rows, which receive the block that
    each item copied and its copy (-1, -1: none). With them the caches may be None: where layers
    are held one by one, copy_kv_blocks(layer's k, v, *copies) for each of them does the copies."""
    op = "update_block_tables"
    _require(block_table.is_cuda, op)
    dev = current_device()
    shape, n, nb = block_table.shape, dst_rows.numel(), ref_counts.numel()
    _require(len(shape) == 2 and block_table.dtype is _I32 and context_lens.dtype is _I32
             and ref_counts.dtype is _I32 and dst_rows.dtype is _I32
             and block_table.get_device() == dev and context_lens.get_device() == dev
             and ref_counts.get_device() == dev and dst_rows.get_device() == dev
             and block_table.is_contiguous() and context_lens.is_contiguous()
             and ref_counts.is_contiguous() and dst_rows.is_contiguous()
             and context_lens.numel() == shape[0]
             and (src_rows is None or _index(src_rows, dev, op) == n)
             and (lengths is None or _index(lengths, dev, op) == n)
             and (status is None or _index(status, dev, op) == 1), op)
    rows, width = shape
    _require(rows < 2 ** 31 > width and n < 2 ** 31 > nb and 0 < cache_block_size < 2 ** 31, op)
    if status is None:
        status = torch.empty(1, dtype=_I32, device=block_table.device)
    copy_src = copy_dst = None
    if copies is not None:
        _require(_index(copies[0], dev, op) == n and _index(copies[1], dev, op) == n, op)
        copy_src, copy_dst = copies[0].data_ptr() or None, copies[1].data_ptr() or None
    if k_cache is None:
        _require(v_cache is None and k_scale is None and v_scale is None, op)
        cache = (None, None, None, None, 0, 0, 0, nb, 0, 0, cache_block_size)
    else:
        _require(v_cache is not None, op)
        cache = _layers(k_cache, v_cache, k_scale, v_scale, cache_block_size, dev, op)
        _require(cache[7] == nb, op)
    ws, ws_bytes = _workspace(_known_size(update_tables_workspace_size, n, width, nb),
                              block_table.device, workspace)
    code = _lib.load().ccinfer_update_block_tables(
        block_table.data_ptr(), context_lens.data_ptr(), ref_counts.data_ptr(),
        dst_rows.data_ptr() or None, None if src_rows is None else src_rows.data_ptr() or None,
        None if lengths is None else lengths.data_ptr() or None, n, rows, width, *cache,
        copy_src, copy_dst, status.data_ptr(), None if ws is None else ws.data_ptr(), ws_bytes, _stream())
    if code:
        raise CcinferError(code, op)
    return status


def compact_workspace_size(num_blocks: int) -> int:
    """Workspace bytes of compact_kv_blocks (0 for an invalid shape)."""
    return int(_lib.load().ccinfer_compact_workspace_size(num_blocks))


def compact_kv_blocks(block_table: torch.Tensor, ref_counts: torch.Tensor, k_cache: torch.Tensor,
                      v_cache: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                      v_scale: Optional[torch.Tensor] = None, cache_block_size: int = 16,
                      workspace: Optional[torch.Tensor] = None,
                      out: Optional[dict] = None) -> dict:
    """Moves the live blocks (count not 0) to the front of the pool, the ones past it, lowest
    first, into the free blocks, lowest first; returns int32 device tensors block_table and ref_counts
    with the new numbers, remap [blocks] (each block's new number, -1 for a free one) and
    num_live [1]. Table entries of free blocks become -1, negative ones stay. `out` reuses
    tensors of an earlier call; its block_table and ref_counts may be the inputs."""
    op = "compact_kv_blocks"
    _require(block_table.is_cuda, op)
    dev = current_device()
    _index(block_table, dev, op)
    _index(ref_counts, dev, op)
    _require(block_table.dim() == 2, op)
    rows, width = block_table.shape
    _require(rows < 2 ** 31 > width, op)
    cache = _layers(k_cache, v_cache, k_scale, v_scale, cache_block_size, dev, op)
    nb = cache[7]
    _require(ref_counts.numel() == nb, op)
    if out is None:
        out = {"block_table": torch.empty_like(block_table),
               "ref_counts": torch.empty_like(ref_counts), "remap": torch.empty_like(ref_counts),
               "num_live": torch.empty(1, dtype=torch.int32, device=block_table.device)}
    table, refs, remap, live = (out["block_table"], out["ref_counts"], out["remap"],
                                out["num_live"])
    _index(table, dev, op)
    _require(table.shape == block_table.shape and _index(refs, dev, op) == nb
             and _index(remap, dev, op) == nb and _index(live, dev, op) == 1, op)
    ws, ws_bytes = _workspace(_known_size(compact_workspace_size, nb), block_table.device,
                              workspace)
    _check(_lib.load().ccinfer_compact_kv_blocks(
        block_table.data_ptr() or None, ref_counts.data_ptr(), rows, width, *cache,
        table.data_ptr() or None, refs.data_ptr(), remap.data_ptr(), live.data_ptr(),
        None if ws is None else ws.data_ptr(), ws_bytes, _stream()), op)
    return out

"""Rotary positions over the C ABI: the table, the rotation of q and k, and the rotation with the
norms of each head and the write of K and V into the cache in the same pass.

Conventions are those of `ops`: device tensors on the current device, work on torch's current
stream, CcinferError with the reference's codes. Everything between the rows read and the rows
written is float32, rounded once; `qkv_prologue` of `ops` follows the reference's roundings.
"""
from __future__ import annotations

import ctypes
from typing import List, Optional, Tuple

import torch

from . import _lib
from .ops import _check, _dev_tensor, _kv_shape, _require, _stream, current_device, fp8_scale_numel

ROPE_SCALINGS = ("none", "linear", "ntk", "yarn", "bands", "factors")
_PARAMS = 5  # doubles before the pairs' own factors (enum ccinfer_rope_scaling)
_KEYS = {"type", "factor", "original_max_position", "fast", "slow", "magnitude", "factors"}


def _frequencies(rotary_dim: int, theta: float, scaling: Optional[dict], op: str):
    """(ctypes array of frequencies, magnitude)."""
    _require(2 <= rotary_dim <= 512 and rotary_dim % 2 == 0, op)
    pairs = rotary_dim // 2
    freq = (ctypes.c_double * pairs)()
    magnitude = ctypes.c_double()
    kind, params = 0, None
    if scaling is not None:
        _require(scaling.get("type") in ROPE_SCALINGS and not set(scaling) - _KEYS, op)
        kind = ROPE_SCALINGS.index(scaling["type"])
        own = scaling.get("factors", ())
        _require(len(own) == (pairs if kind == 5 else 0), op)
        params = (ctypes.c_double * (_PARAMS + len(own)))(
            scaling.get("factor", 1.0), scaling.get("original_max_position", 0.0),
            scaling.get("fast", 32.0 if kind == 3 else 4.0), scaling.get("slow", 1.0),
            scaling.get("magnitude", 0.0), *own)
    _check(_lib.load().ccinfer_rope_frequencies(rotary_dim, theta, kind, params, freq,
                                                ctypes.byref(magnitude)), op)
    return freq, magnitude.value


def rope_frequencies(rotary_dim: int, theta: float = 10000.0,
                     scaling: Optional[dict] = None) -> Tuple[List[float], float]:
    """Radians a position of each of the rotary_dim / 2 pairs, and the factor of cos and sin, in
    double precision on the host. `scaling` for contexts past the trained length:

      None or {"type": "none"}   theta^(-2p / rotary_dim)
      {"type": "linear", "factor": s}   every frequency over s
      {"type": "ntk", "factor": s}      theta grows by s^(rotary_dim / (rotary_dim - 2))
      {"type": "yarn", "factor": s, "original_max_position": n}   slow pairs over s, fast ones
          kept, a ramp over the pairs between those that turn "fast" (32) and "slow" (1) times
          over n positions; the factor of cos and sin is 0.1 ln s + 1
      {"type": "bands", "factor": s, "original_max_position": n}   the same by turns: kept at
          "fast" (4) turns and more, over s at "slow" (1) and fewer, blended between
      {"type": "factors", "factors": [...]}   each pair's frequency over its own factor

    "magnitude" sets the factor of cos and sin."""
    freq, magnitude = _frequencies(rotary_dim, theta, scaling, "rope_frequencies")
    return list(freq), magnitude


def build_rope_cache(max_position: int, rotary_dim: int, theta: float = 10000.0,
                     scaling: Optional[dict] = None, first_position: int = 0,
                     out: Optional[torch.Tensor] = None, device=None) -> torch.Tensor:
    """The table [max_position, rotary_dim / 2, 2] float32 of (cos, sin) at the positions
    first_position .. first_position + max_position - 1, frequencies as in rope_frequencies,
    built on the device with angles in double precision (the reference builds an unscaled one
    on the host in float32, src/model/rope/rope_cache.cpp)."""
    op = "build_rope_cache"
    freq, magnitude = _frequencies(rotary_dim, theta, scaling, op)
    shape = (max_position, rotary_dim // 2, 2)
    _require(max_position > 0, op)
    if out is None:
        out = torch.empty(shape, dtype=torch.float32,
                          device=torch.device("cuda") if device is None else device)
    _dev_tensor(out, torch.float32, op)
    _require(tuple(out.shape) == shape and out.get_device() == current_device(), op)
    _check(_lib.load().ccinfer_build_rope_cache(freq, rotary_dim, magnitude, first_position,
                                                max_position, out.data_ptr(), _stream()), op)
    return out


def _table(rope_cache: torch.Tensor, head_dim: int, op: str) -> Tuple[int, int]:
    """(positions, rotary_dim) of a table."""
    _dev_tensor(rope_cache, torch.float32, op)
    shape = rope_cache.shape
    _require(len(shape) == 3 and shape[2] == 2 and 2 <= 2 * shape[1] <= head_dim, op)
    return shape[0], 2 * shape[1]


def _rows(x: torch.Tensor, op: str):
    """Shape and strides of [tokens, heads, head_dim] rows."""
    _require(x.dtype is torch.bfloat16 and x.is_cuda and x.dim() == 3, op)
    shape, stride = x.shape, x.stride()
    _require(stride[2] == 1 or shape[2] == 1, op)
    return shape, stride


def _out_rows(x: torch.Tensor, shape, stride, out: Optional[torch.Tensor], op: str):
    """The output rows of x and their strides; no two of them may share memory."""
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=x.device)
        return out, out.stride()
    oshape, ostride = _rows(out, op)
    t, h, d = shape
    st, sh, _ = ostride
    apart = (sh >= d and st >= h * sh) or (st >= d and sh >= t * st) \
        or (h == 1 and st >= d) or (t == 1 and sh >= d) or (t == 1 and h == 1)
    same = out.data_ptr() == x.data_ptr()
    _require(oshape == shape and apart and (not same or ostride == stride), op)
    return out, ostride


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                     rope_cache: torch.Tensor, interleaved: bool = False, inverse: bool = False,
                     q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None):
    """Rotates q [tokens, num_q_heads, head_dim] and k [tokens, num_kv_heads, head_dim] (or None)
    bf16 by row positions[t] of rope_cache [max_position, rotary_dim / 2, 2] (launch_rope,
    src/kernel/pos/rope.cu:14-43); returns (q_out, k_out).

    Pairs are (p, p + rotary_dim / 2), or (2p, 2p + 1) with `interleaved`; elements from
    rotary_dim on, and rows at positions outside the table, are copied. `inverse` turns the
    other way: the gradient of the rotation, and the way back for cached keys. q and k may be
    views whose heads are contiguous (slices of the packed projection); q_out = q and k_out = k
    rotate in place, any other outputs lie apart from the inputs."""
    op = "rotary_embedding"
    shape, qs = _rows(q, op)
    t, hq, d = shape
    max_pos, rotary_dim = _table(rope_cache, d, op)
    _dev_tensor(positions, torch.int32, op)
    dev = q.get_device()
    _require(t > 0 and positions.numel() == t and dev == current_device()
             and positions.get_device() == dev and rope_cache.get_device() == dev, op)
    q_out, qos = _out_rows(q, shape, qs, q_out, op)
    if k is None:
        _require(k_out is None, op)
        hkv, ks, kos, kp, kop = 0, (0, 0), (0, 0), None, None
    else:
        kshape, ks = _rows(k, op)
        hkv = kshape[1]
        _require(kshape[0] == t and kshape[2] == d and k.get_device() == dev, op)
        k_out, kos = _out_rows(k, kshape, ks, k_out, op)
        kp, kop = k.data_ptr(), k_out.data_ptr()
        _require(k_out.get_device() == dev, op)
    _require(q_out.get_device() == dev, op)
    _check(_lib.load().ccinfer_rotary_embedding(
        q.data_ptr(), qs[0], qs[1], kp, ks[0], ks[1], positions.data_ptr(),
        rope_cache.data_ptr(), q_out.data_ptr(), qos[0], qos[1], kop, kos[0], kos[1], t, hq, hkv,
        d, rotary_dim, max_pos, interleaved, inverse, _stream()), op)
    return q_out, k_out


def _norm_weight(w: Optional[torch.Tensor], heads: int, d: int, dev: int, op: str):
    """(pointer, whether each head has its own) of a norm weight."""
    if w is None:
        return None, 0
    _dev_tensor(w, torch.bfloat16, op)
    shape = tuple(w.shape)
    _require((shape == (d,) or shape == (heads, d)) and w.get_device() == dev, op)
    return w.data_ptr(), len(shape) == 2


def qkv_norm_rope(qkv: torch.Tensor, q_norm_weight: Optional[torch.Tensor],
                  k_norm_weight: Optional[torch.Tensor], positions: torch.Tensor,
                  rope_cache: torch.Tensor, slot_mapping: torch.Tensor, k_cache: torch.Tensor,
                  v_cache: torch.Tensor, num_q_heads: int, eps: float = 1e-6,
                  interleaved: bool = False, weight_offset: float = 0.0,
                  k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                  q_out: Optional[torch.Tensor] = None,
                  max_slots: Optional[int] = None) -> torch.Tensor:
    """One launch for an attention layer's prologue: split of the packed projection, RMSNorm of
    each q and k head (y = x rsqrt(mean x^2 + eps) (w + weight_offset); a None weight: no norm),
    the rotation of rotary_embedding, K and V into their cache slots. Returns q
    [num_tokens, num_q_heads, head_dim].

    The prologue of `ops.qkv_prologue` for tables narrower than the head, interleaved pairs,
    weights of [heads, head_dim], row-strided qkv and fp8 caches (uint8, with k_scale and
    v_scale as in ops.write_kv_cache_fp8). It computes in float32 and rounds once, where
    qkv_prologue rounds as the reference's five kernels do, so the two differ in last places.
    A bf16 cache takes K as the rows that rotary_embedding would return; an fp8 one is
    quantised from float32. No two tokens may have the same slot."""
    op = "qkv_norm_rope"
    _require(qkv.dtype is torch.bfloat16 and qkv.is_cuda and qkv.dim() == 2, op)
    _dev_tensor(positions, torch.int32, op)
    _dev_tensor(slot_mapping, torch.int32, op)
    fp8 = k_scale is not None
    for c in (k_cache, v_cache):
        _dev_tensor(c, torch.uint8 if fp8 else torch.bfloat16, op)
    slots, hkv, d = _kv_shape(k_cache)
    max_pos, rotary_dim = _table(rope_cache, d, op)
    t, width = qkv.shape
    stride = qkv.stride()
    dev = qkv.get_device()
    _require(t > 0 and num_q_heads > 0 and width == (num_q_heads + 2 * hkv) * d and stride[1] == 1,
             op)
    _require(v_cache.shape == k_cache.shape and positions.numel() == t
             and slot_mapping.numel() == t, op)
    _require(dev == current_device() == k_cache.get_device() == v_cache.get_device()
             == positions.get_device() == slot_mapping.get_device() == rope_cache.get_device(), op)
    _require(max_slots is None or max_slots <= slots, op)
    ksp = vsp = None
    _require(fp8 == (v_scale is not None), op)
    if fp8:
        for s in (k_scale, v_scale):
            _dev_tensor(s, torch.float32, op)
            _require(s.numel() >= fp8_scale_numel(slots, hkv) and s.get_device() == dev, op)
        ksp, vsp = k_scale.data_ptr(), v_scale.data_ptr()
    qw, q_each = _norm_weight(q_norm_weight, num_q_heads, d, dev, op)
    kw, k_each = _norm_weight(k_norm_weight, hkv, d, dev, op)
    if q_out is None:
        q_out = torch.empty((t, num_q_heads, d), dtype=torch.bfloat16, device=qkv.device)
    else:
        _dev_tensor(q_out, torch.bfloat16, op)
        _require(q_out.numel() == t * num_q_heads * d and q_out.get_device() == dev, op)
    _check(_lib.load().ccinfer_qkv_norm_rope(
        qkv.data_ptr(), stride[0] if t > 1 else width, qw, q_each, kw, k_each,
        positions.data_ptr(), rope_cache.data_ptr(), slot_mapping.data_ptr(), q_out.data_ptr(),
        k_cache.data_ptr(), v_cache.data_ptr(), ksp, vsp, t, num_q_heads, hkv, d, rotary_dim,
        max_pos, slots if max_slots is None else max_slots, interleaved, eps, weight_offset,
        _stream()), op)
    return q_out

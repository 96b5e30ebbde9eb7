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
from .ops import (CcinferError, _check, _dev_tensor, _require, _stream, current_device,
                  fp8_scale_numel)

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
        if kind == 0 and "magnitude" in scaling:  # plain frequencies are linear ones over 1
            scaling, kind = {"magnitude": scaling["magnitude"]}, 1
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
    _require(max_position > 0 and 0 <= first_position < 2 ** 31 - max_position, op)
    if out is None:
        out = torch.empty(shape, dtype=torch.float32,
                          device=torch.device("cuda") if device is None else device)
    _dev_tensor(out, torch.float32, op)
    _require(tuple(out.shape) == shape and out.get_device() == current_device(), op)
    _check(_lib.load().ccinfer_build_rope_cache(freq, rotary_dim, magnitude, first_position,
                                                max_position, out.data_ptr(), _stream()), op)
    return out


# The smallest calls below take 2 us on the GPU, so their host side bounds them: the checks are
# single expressions of few interpreter steps. Host time
# of a call, launch included: rotary_embedding 9.3 -> 7.9 us, qkv_norm_rope 11.6 -> 10.3 us.

_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32


def _out_stride(x, shape, stride, out, dev: int, op: str):
    """Strides of the output rows `out` of x; no two of them may share memory."""
    t, h, d = shape
    ostride = out.stride()
    if ostride == (h * d, d, 1):
        apart = True
    else:
        st, sh, sd = ostride if out.dim() == 3 else (0, 0, 0)
        apart = sd == 1 and ((sh >= d and st >= h * sh) or (st >= d and sh >= t * st)
                             or (h == 1 and st >= d) or (t == 1 and sh >= d) or t * h == 1)
    _require(apart and out.dtype is _BF16 and out.shape == shape and out.get_device() == dev
             and (out.data_ptr() != x.data_ptr() or ostride == stride), op)
    return ostride


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
    _require(q.is_cuda, op)
    dev = current_device()
    shape, qs, table = q.shape, q.stride(), rope_cache.shape
    _require(len(shape) == 3 == len(table) and table[2] == 2 and qs[2] == 1
             and shape[1] < 2 ** 31 > table[0] and 2 * table[1] <= shape[2] <= 1024
             and q.dtype is _BF16 and positions.dtype is _I32 and rope_cache.dtype is _F32
             and q.get_device() == dev and positions.get_device() == dev
             and rope_cache.get_device() == dev and positions.is_contiguous()
             and rope_cache.is_contiguous()
             and 2 ** 31 > positions.numel() == shape[0] > 0, op)
    t, hq, d = shape
    if q_out is None:
        q_out = torch.empty(shape, dtype=_BF16, device=q.device)
        qos = q_out.stride()
    else:
        qos = _out_stride(q, shape, qs, q_out, dev, op)
    if k is None:
        _require(k_out is None, op)
        hkv, ks, kos, kp, kop = 0, (0, 0), (0, 0), None, None
    else:
        kshape, ks = k.shape, k.stride()
        _require(len(kshape) == 3 and kshape[0] == t and kshape[2] == d and ks[2] == 1
                 and kshape[1] < 2 ** 31
                 and k.dtype is _BF16 and k.get_device() == dev, op)
        hkv = kshape[1]
        if k_out is None:
            k_out = torch.empty(kshape, dtype=_BF16, device=k.device)
            kos = k_out.stride()
        else:
            kos = _out_stride(k, kshape, ks, k_out, dev, op)
        kp, kop = k.data_ptr(), k_out.data_ptr()
    code = _lib.load().ccinfer_rotary_embedding(
        q.data_ptr(), qs[0], qs[1], kp, ks[0], ks[1], positions.data_ptr(),
        rope_cache.data_ptr(), q_out.data_ptr(), qos[0], qos[1], kop, kos[0], kos[1], t, hq, hkv,
        d, 2 * table[1], table[0], interleaved, inverse, _stream())
    if code:
        raise CcinferError(code, op)
    return q_out, k_out


def _norm_weight(w: Optional[torch.Tensor], heads: int, d: int, dev: int, op: str):
    """(pointer, whether each head has its own) of a norm weight."""
    if w is None:
        return None, 0
    shape = w.shape
    each = len(shape) == 2
    _require(shape[-1:] == (d,) and (len(shape) == 1 or each and shape[0] == heads)
             and w.dtype is _BF16 and w.is_contiguous() and w.get_device() == dev, op)
    return w.data_ptr(), each


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
    quantised from float32. A row whose sum of squares passes float32's largest number becomes
    zeros. No two tokens may have the same slot."""
    op = "qkv_norm_rope"
    _require(qkv.is_cuda, op)
    dev = current_device()
    shape, table, cache = qkv.shape, rope_cache.shape, k_cache.shape
    stride = qkv.stride()
    fp8 = k_scale is not None
    kind = torch.uint8 if fp8 else _BF16
    _require(len(shape) == 2 and len(table) == 3 and table[2] == 2 and stride[1] == 1
             and 3 <= len(cache) <= 4 and qkv.dtype is _BF16 and k_cache.dtype is kind
             and v_cache.dtype is kind and positions.dtype is _I32 and slot_mapping.dtype is _I32
             and rope_cache.dtype is _F32 and qkv.get_device() == dev
             and k_cache.get_device() == dev and v_cache.get_device() == dev
             and positions.get_device() == dev and slot_mapping.get_device() == dev
             and rope_cache.get_device() == dev and k_cache.is_contiguous()
             and v_cache.is_contiguous() and positions.is_contiguous()
             and slot_mapping.is_contiguous() and rope_cache.is_contiguous()
             and v_cache.shape == cache and fp8 == (v_scale is not None), op)
    hkv, d = cache[-2], cache[-1]
    slots = cache[0] if len(cache) == 3 else cache[0] * cache[1]
    t, width = shape
    if max_slots is None:
        max_slots = slots
    _require(2 ** 31 > t > 0 and num_q_heads > 0 and width == (num_q_heads + 2 * hkv) * d
             and width < 2 ** 31 > table[0] and 2 * table[1] <= d and positions.numel() == t
             and slot_mapping.numel() == t and 0 < max_slots <= slots and max_slots < 2 ** 31, op)
    ksp = vsp = None
    if fp8:
        need = fp8_scale_numel(slots, hkv)
        for s in (k_scale, v_scale):
            _require(s.dtype is _F32 and s.is_contiguous() and s.numel() >= need
                     and s.get_device() == dev, op)
        ksp, vsp = k_scale.data_ptr(), v_scale.data_ptr()
    qw, q_each = _norm_weight(q_norm_weight, num_q_heads, d, dev, op)
    kw, k_each = _norm_weight(k_norm_weight, hkv, d, dev, op)
    if q_out is None:
        q_out = torch.empty((t, num_q_heads, d), dtype=_BF16, device=qkv.device)
    else:
        _require(q_out.dtype is _BF16 and q_out.is_contiguous()
                 and q_out.numel() == t * num_q_heads * d and q_out.get_device() == dev, op)
    code = _lib.load().ccinfer_qkv_norm_rope(
        qkv.data_ptr(), stride[0] if t > 1 else width, qw, q_each, kw, k_each,
        positions.data_ptr(), rope_cache.data_ptr(), slot_mapping.data_ptr(), q_out.data_ptr(),
        k_cache.data_ptr(), v_cache.data_ptr(), ksp, vsp, t, num_q_heads, hkv, d, 2 * table[1],
        table[0], max_slots, interleaved, eps, weight_offset, _stream())
    if code:
        raise CcinferError(code, op)
    return q_out

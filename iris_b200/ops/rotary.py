"""Head norms, position rotation and cache writes between the QKV projection and attention (``csrc/kernels/rotary.cu``):
bf16 / fp16 tensors, fp32 arithmetic, one rounding.  Used by the decoder (``iris_b200/models/tp_block.py``); no counterpart in
the reference."""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional

import torch

from .. import _native
from .paged import may_overlap, same_strides

_DT = {torch.bfloat16: 0, torch.float16: 1}
_ARGS = struct.Struct("@28qd")


def rotary_table(positions: int, rotary_dim: int, theta: float = 10000.0, *, scaling: Optional[str] = None,
                 factor: float = 1.0, original_positions: int = 0, slow: float = 1.0, fast: float = 32.0,
                 device=None) -> torch.Tensor:
    """Cosines and sines of every position's angles, ``[positions, rotary_dim]`` fp32: ``rotary_dim / 2`` cosines, then the
    sines.  Pair ``i`` turns by ``theta ** (-2 i / rotary_dim)`` per position, computed in 64 bits.  For contexts longer than a
    model was trained on:

    * ``scaling="linear"``: all angles divided by ``factor``;
    * ``scaling="theta"``: ``theta`` enlarged by ``factor ** (rotary_dim / (rotary_dim - 2))``, so that the slowest pair turns
      ``factor`` times slower and the fastest as before;
    * ``scaling="parts"``: pairs that turn fewer than ``slow`` times within ``original_positions`` are slowed down by
      ``factor``, those that turn more than ``fast`` times are left, those between are mixed linearly by their turns.
    """
    if positions < 1 or rotary_dim < 16 or rotary_dim % 16:
        raise ValueError("need at least one position and a rotary dimension that is a multiple of 16")
    if not (theta > 0 and factor > 0 and math.isfinite(theta) and math.isfinite(factor)):
        raise ValueError("theta and factor must be positive")
    half = rotary_dim // 2
    exponents = torch.arange(half, dtype=torch.float64, device=device) / half
    if scaling == "theta":
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    speed = theta ** -exponents
    if scaling == "linear":
        speed = speed / factor
    elif scaling == "parts":
        if original_positions < 1 or not 0 < slow < fast:
            raise ValueError('scaling="parts" needs original_positions, and slow < fast')
        kept = ((original_positions * speed / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        speed = speed * (kept + (1 - kept) / factor)
    elif scaling not in (None, "theta"):
        raise ValueError(f"scaling must be None, 'linear', 'theta' or 'parts', got {scaling!r}")
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * speed
    return torch.cat([angle.cos(), angle.sin()], 1).to(torch.float32)


def _weight(w: torch.Tensor, head_dim: int, dtype: torch.dtype) -> int:
    if w.dtype is not dtype or w.nbytes != 2 * head_dim or not w.is_contiguous():
        raise ValueError(f"norm weights must be contiguous [{head_dim}] of the type of qkv")
    return w.data_ptr()


def qk_norm_rope(qkv: torch.Tensor, out: torch.Tensor, positions: torch.Tensor, table: Optional[torch.Tensor], heads: int, kv_heads: int,
                 head_dim: int, *, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-6, interleaved: bool = False, k_cache: Optional[torch.Tensor] = None,
                 v_cache: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """One pass over the projection's output: every query and key head normalised and rotated by its token's position, keys and
    values stored into a paged cache.

    ``qkv`` is ``[tokens, (heads + 2 kv_heads) * head_dim]`` (Q | K | V column blocks; rows may be strided), ``positions`` int32
    ``[tokens]``, ``table`` a :func:`rotary_table` whose width says how much of a head is rotated (its first components; pairs
    ``(i, i + width / 2)``, or ``(2 i, 2 i + 1)`` if ``interleaved``; ``None``: nothing is).  ``q_weight`` / ``k_weight`` ``[head_dim]``: the head is
    first divided by the root of its mean square (plus ``eps``) and multiplied by the weight; ``None``: no norm.  ``out``: all
    columns like ``qkv``; ``qkv`` itself (in place); or the query columns alone.  ``k_cache`` / ``v_cache``: pages
    ``[pages, page_size, kv_heads, head_dim]`` with equal strides, in any order with contiguous heads; token ``t`` goes to slot
    ``slots[t]`` (int32, distinct; page * page_size + place), and to none if that is negative.  Rows whose position is negative
    are left as they were, in ``out`` and in the cache.  A position behind the table or a slot behind the cache is skipped and
    recorded in ``status`` (an ``Iris`` context's status block) if that is given.
    """
    # (every look at a tensor costs the host 0.06 to 0.12 us, on a path of 8: sizes of vectors in bytes, no shape twice)
    dtype = qkv.dtype
    if dtype not in _DT or out.dtype is not dtype:
        raise TypeError("qkv and out must both be bfloat16 or both float16")
    (tokens, width), (ld_in, one) = qkv.shape, qkv.stride()
    (out_rows, out_width), (ld_out, out_one) = out.shape, out.stride()
    if heads < 1 or kv_heads < 1 or head_dim < 16 or head_dim % 16 or head_dim > 512:
        raise ValueError("need heads, and a head dimension that is a multiple of 16, at most 512")
    if width != (heads + 2 * kv_heads) * head_dim or out_rows != tokens or (out_width != width and out_width != heads * head_dim):
        raise ValueError(f"expected qkv [tokens, {(heads + 2 * kv_heads) * head_dim}] and out like it or [tokens, "
                         f"{heads * head_dim}], got {tuple(qkv.shape)} and {tuple(out.shape)}")
    if (positions.dtype is not torch.int32 or positions.nbytes != 4 * tokens or not positions.is_contiguous() or one != 1 or
            out_one != 1):
        raise ValueError(f"positions must be int32 [{tokens}], and they and the rows of qkv and out contiguous")
    device = qkv.get_device()
    same = out.get_device() == device and positions.get_device() == device
    turns = table_ptr = table_pitch = rotary = 0
    if table is not None:
        (turns, rotary), (table_pitch, one) = table.shape, table.stride()
        if table.dtype is not torch.float32 or one != 1 or rotary > head_dim or rotary % 16:
            raise ValueError("table must be fp32 [positions, rotary dimension] with contiguous rows, the latter a multiple of 16 within "
                             "the head")
        same = same and table.get_device() == device
        table_ptr = table.data_ptr()
    q_ptr = k_ptr = 0
    if q_weight is not None:
        same = same and q_weight.get_device() == device
        q_ptr = _weight(q_weight, head_dim, dtype)
    if k_weight is not None:
        same = same and k_weight.get_device() == device
        k_ptr = _weight(k_weight, head_dim, dtype)
    k_cache_ptr = v_cache_ptr = slots_ptr = page = slot = head = pages = size = 0
    if k_cache is not None or v_cache is not None or slots is not None:
        if k_cache is None or v_cache is None or slots is None:
            raise ValueError("k_cache, v_cache and slots belong together")
        if k_cache.dtype is not dtype or v_cache.dtype is not dtype:
            raise TypeError("the cache must have the type of qkv")
        cache_shape = pages, size, cache_heads, cache_dim = k_cache.shape
        if cache_heads != kv_heads or cache_dim != head_dim or v_cache.shape != cache_shape:
            raise ValueError(f"the cache must be [pages, page_size, {kv_heads}, {head_dim}]")
        strides = page, slot, head, one = k_cache.stride()
        if one != 1 or (v_cache.stride() != strides and not same_strides(k_cache, v_cache)):
            raise ValueError("k_cache and v_cache must have the same strides, with contiguous heads")
        if slots.dtype is not torch.int32 or slots.nbytes != 4 * tokens or not slots.is_contiguous():
            raise ValueError(f"slots must be contiguous int32 [{tokens}]")
        same = same and k_cache.get_device() == device and v_cache.get_device() == device and slots.get_device() == device
        k_cache_ptr, v_cache_ptr, slots_ptr = k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr()
    elif out_width != width:
        raise ValueError("an output of queries alone needs a cache for the keys and values")
    status_ptr = 0
    if not same:
        raise ValueError("all tensors must be on one device")
    if status is not None:
        status_ptr = _native.status_block(status, device)
    if tokens == 0:
        return out
    qkv_ptr, out_ptr = qkv.data_ptr(), out.data_ptr()
    in_place = out_ptr == qkv_ptr and (ld_out == ld_in or tokens == 1)
    if tokens > 1 and ld_out < out_width:
        raise ValueError("rows of out must not overlap")
    if not in_place and may_overlap(tokens, qkv_ptr, ld_in, width, out_ptr, ld_out, out_width):
        raise ValueError("out must be qkv itself, or share no memory with it")
    if device != _native.current_device(device):
        with torch.cuda.device(device):
            return qk_norm_rope(qkv, out, positions, table, heads, kv_heads, head_dim, q_weight=q_weight, k_weight=k_weight,
                                eps=eps, interleaved=interleaved, k_cache=k_cache, v_cache=v_cache, slots=slots, status=status,
                                stream=stream)
    rc = _native.entry("iris_k_qk_norm_rope")(_ARGS.pack(
        qkv_ptr, out_ptr, positions.data_ptr(), table_ptr, q_ptr, k_ptr, k_cache_ptr, v_cache_ptr, slots_ptr, status_ptr,
        torch._C._cuda_getCurrentRawStream(device) if stream is None else stream, ld_in, ld_out, table_pitch, page, slot, head,
        heads + kv_heads if in_place and out_width == width else out_width // head_dim, turns, rotary, 1 if interleaved else 0,
        pages, size, tokens, heads, kv_heads, head_dim, _DT[dtype], eps))
    if rc:
        lib = _native.kernels()
        lib.iris_rotary_last_error.restype = ctypes.c_char_p
        raise RuntimeError("qk_norm_rope: " + (lib.iris_rotary_last_error().decode() or f"launch failed ({rc})"))
    return out

"""Head norms, position rotation and cache writes between the QKV projection and attention (``csrc/kernels/rotary.cu``):
bf16 / fp16 tensors, fp32 arithmetic, one rounding.  Used by the decoder (``iris_b200/models/tp_block.py``); no counterpart in
the reference."""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from .. import _native
from .paged import same_strides

_DT = {torch.bfloat16: 0, torch.float16: 1}
_P, _L, _I, _F = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float
_ARGTYPES = [_P, _L, _P, _L, _I, _P, _P, _L, _L, _I, _I, _P, _P, _F, _P, _P, _L, _L, _L, _L, _I, _P, _L, _I, _I, _I, _I, _P, _P]


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


def _may_overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two matrices of 16-bit elements share memory; column blocks of one matrix, with its pitch, do not."""
    rows, pitch, size = a.shape[0], a.stride(0), 2
    a0, b0 = a.data_ptr(), b.data_ptr()
    a1, b1 = a0 + ((rows - 1) * pitch + a.shape[1]) * size, b0 + ((rows - 1) * b.stride(0) + b.shape[1]) * size
    if a1 <= b0 or b1 <= a0:
        return False
    if pitch == b.stride(0) and rows > 1:
        off = (b0 - a0) % (pitch * size)
        return off < a.shape[1] * size or off + b.shape[1] * size > pitch * size
    return True


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
    if qkv.dtype not in _DT or out.dtype != qkv.dtype:
        raise TypeError("qkv and out must both be bfloat16 or both float16")
    if qkv.dim() != 2 or out.dim() != 2 or qkv.stride(1) != 1 or out.stride(1) != 1:
        raise ValueError("qkv and out must be 2-D with contiguous rows")
    tokens, width = qkv.shape
    if heads < 1 or kv_heads < 1 or head_dim < 16 or head_dim % 16 or head_dim > 512:
        raise ValueError("need heads, and a head dimension that is a multiple of 16, at most 512")
    if width != (heads + 2 * kv_heads) * head_dim or out.shape[0] != tokens or out.shape[1] not in (width, heads * head_dim):
        raise ValueError(f"expected qkv [tokens, {(heads + 2 * kv_heads) * head_dim}] and out like it or [tokens, "
                         f"{heads * head_dim}], got {tuple(qkv.shape)} and {tuple(out.shape)}")
    device = qkv.get_device()
    if positions.dtype != torch.int32 or positions.shape != (tokens,) or (tokens > 1 and positions.stride(0) != 1):
        raise ValueError(f"positions must be contiguous int32 [{tokens}]")
    same = out.get_device() == device and positions.get_device() == device
    turns = table_ptr = table_pitch = rotary = 0
    if table is not None:
        if table.dtype != torch.float32 or table.dim() != 2 or table.stride(1) != 1 or table.shape[1] > head_dim or table.shape[1] % 16:
            raise ValueError("table must be fp32 [positions, rotary dimension], at most as wide as a head, a multiple of 16")
        same = same and table.get_device() == device
        (turns, rotary), table_ptr, table_pitch = table.shape, table.data_ptr(), table.stride(0)
    for w in (q_weight, k_weight):
        if w is not None:
            if w.dtype != qkv.dtype or w.shape != (head_dim,) or w.stride(0) != 1:
                raise ValueError(f"norm weights must be [{head_dim}] of the type of qkv")
            same = same and w.get_device() == device
    in_place = False
    if tokens:
        in_place = out.data_ptr() == qkv.data_ptr() and out.stride(0) == qkv.stride(0)
        if tokens > 1 and out.stride(0) < out.shape[1]:
            raise ValueError("rows of out must not overlap")
        if not in_place and _may_overlap(qkv, out):
            raise ValueError("out must be qkv itself, or share no memory with it")
    k_ptr = v_ptr = slots_ptr = 0
    page = slot = head = pages = size = 0
    if k_cache is not None or v_cache is not None or slots is not None:
        if k_cache is None or v_cache is None or slots is None:
            raise ValueError("k_cache, v_cache and slots belong together")
        if k_cache.dtype != qkv.dtype or v_cache.dtype != qkv.dtype:
            raise TypeError("the cache must have the type of qkv")
        if k_cache.dim() != 4 or k_cache.shape[2:] != (kv_heads, head_dim) or v_cache.shape != k_cache.shape:
            raise ValueError(f"the cache must be [pages, page_size, {kv_heads}, {head_dim}]")
        page, slot, head, one = k_cache.stride()
        if one != 1 or not same_strides(k_cache, v_cache):
            raise ValueError("k_cache and v_cache must have the same strides, with contiguous heads")
        if slots.dtype != torch.int32 or slots.shape != (tokens,) or (tokens > 1 and slots.stride(0) != 1):
            raise ValueError(f"slots must be contiguous int32 [{tokens}]")
        same = same and k_cache.get_device() == device and v_cache.get_device() == device and slots.get_device() == device
        pages, size = k_cache.shape[0], k_cache.shape[1]
        k_ptr, v_ptr, slots_ptr = k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr()
    elif out.shape[1] != width:
        raise ValueError("an output of queries alone needs a cache for the keys and values")
    if not same or (status is not None and status.get_device() != device):
        raise ValueError("all tensors must be on one device")
    if tokens == 0:
        return out
    if device != _native.current_device(device):
        with torch.cuda.device(device):
            return qk_norm_rope(qkv, out, positions, table, heads, kv_heads, head_dim, q_weight=q_weight, k_weight=k_weight,
                                eps=eps, interleaved=interleaved, k_cache=k_cache, v_cache=v_cache, slots=slots, status=status,
                                stream=stream)
    out_heads = heads + kv_heads if in_place and out.shape[1] == width else out.shape[1] // head_dim
    lib = _native.kernels()
    fn = _native.typed(lib.iris_k_qk_norm_rope, _ARGTYPES)
    rc = fn(qkv.data_ptr(), qkv.stride(0), out.data_ptr(), out.stride(0), out_heads, positions.data_ptr(), table_ptr,
            table_pitch, turns, rotary, 1 if interleaved else 0,
            0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr(), eps, k_ptr, v_ptr,
            page, slot, head, pages, size, slots_ptr, tokens, heads, kv_heads, head_dim, _DT[qkv.dtype],
            0 if status is None else status.data_ptr(), _native.current_stream(device) if stream is None else stream)
    if rc:
        lib.iris_rotary_last_error.restype = ctypes.c_char_p
        raise RuntimeError("qk_norm_rope: " + (lib.iris_rotary_last_error().decode() or f"launch failed ({rc})"))
    return out

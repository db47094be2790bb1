"""Self-attention forward on the tcgen05 kernel of ``csrc/kernels/attention.cu`` (head dimension 128, bf16 / fp16): causal or
full, and causal with a sliding window and first keys that stay visible.

No counterpart in the reference, which has no model code; the tensor-parallel decoder block
(``iris_b200/models/tp_block.py``) uses it for the attention core between its fused all-gather -> GEMM (which produces
``qkv``) and its fused GEMM -> all-reduce (which consumes ``out``), so that no phase of the block is a library kernel.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional

import torch

from .. import _native
from .paged import may_overlap

HEAD_DIM = 128
_DT = {torch.bfloat16: 0, torch.float16: 1}
_ARGTYPES = [ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_int, ctypes.c_int,
             ctypes.c_int, ctypes.c_int, ctypes.c_void_p, ctypes.c_uint64, ctypes.c_void_p]


def attention_fwd(qkv: torch.Tensor, out: torch.Tensor, batch: int, seq: int, heads: int, causal: bool = True,
                  status: Optional[torch.Tensor] = None, timeout_ms: float = 2000.0, stream=None) -> torch.Tensor:
    """``out[b*seq + s, h*128:(h+1)*128] = softmax(q . k^T / sqrt(128)) . v`` per batch ``b`` and head ``h``.

    ``qkv`` is ``[batch * seq, 3 * heads * 128]`` with the Q, K and V column blocks side by side (head ``h`` in columns
    ``h * 128 ..`` of each block), ``out`` is ``[batch * seq, heads * 128]``; rows may be strided views.  ``seq`` must be
    a multiple of 128.  ``status``: the int32 status block of an ``Iris`` context (``ctx.status``), in which a bounded
    wait of the kernel records a time-out; ``None``: not recorded.
    """
    if qkv.dtype not in _DT or out.dtype != qkv.dtype:
        raise TypeError("qkv and out must both be bfloat16 or both float16")
    if qkv.dim() != 2 or out.dim() != 2 or qkv.stride(1) != 1 or out.stride(1) != 1:
        raise ValueError("qkv and out must be 2-D with contiguous rows")
    if qkv.shape != (batch * seq, 3 * heads * HEAD_DIM) or out.shape != (batch * seq, heads * HEAD_DIM):
        raise ValueError(f"expected qkv [{batch * seq}, {3 * heads * HEAD_DIM}] and out [{batch * seq}, "
                         f"{heads * HEAD_DIM}], got {tuple(qkv.shape)} and {tuple(out.shape)}")
    lib = _native.kernels()
    fn = _native.typed(lib.iris_k_attention_fwd, _ARGTYPES)
    st = _native.current_stream(qkv.get_device()) if stream is None else stream
    rc = fn(qkv.data_ptr(), qkv.stride(0), out.data_ptr(), out.stride(0), batch, seq, heads, int(bool(causal)),
            _DT[qkv.dtype], status.data_ptr() if status is not None else 0, int(timeout_ms * 1e6), st)
    if rc != 0:
        lib.iris_attention_last_error.restype = ctypes.c_char_p
        raise RuntimeError(lib.iris_attention_last_error().decode() or f"attention launch failed ({rc})")
    return out


_WINDOW_ARGS = struct.Struct("@14q")


def attention_window_fwd(qkv: torch.Tensor, out: torch.Tensor, batch: int, seq: int, heads: int, kv_heads: Optional[int] = None, *,
                         window: int, sinks: int = 0, status: Optional[torch.Tensor] = None, timeout_ms: float = 2000.0,
                         stream=None) -> torch.Tensor:
    """Causal self-attention in which query ``i`` of a sequence sees its keys ``j <= i`` with ``j > i - window`` or
    ``j < sinks`` (``window >= seq``: all of them); :func:`iris_b200.ops.paged.paged_attention` is the form for one new token.

    ``qkv`` is ``[batch * seq, (heads + 2 * kv_heads) * 128]`` with the Q, K and V column blocks side by side, query head ``h``
    reading key head ``h // (heads // kv_heads)``; ``out`` is ``[batch * seq, heads * 128]``; rows may be strided views.
    ``seq``: any length.  ``out`` may be the query columns of ``qkv`` themselves.  ``status``: as for :func:`attention_fwd`, at
    least 32 bytes.  A masked key weighs exactly nothing; a masked *value* that is infinite or NaN still reaches the queries of its
    sequence whose window shares its tile of 128 keys (zero times it), so the rows of padding have to be finite.
    """
    kv_heads = heads if kv_heads is None else kv_heads
    dtype, shape = qkv.dtype, qkv.shape
    if dtype not in _DT or out.dtype is not dtype:
        raise TypeError("qkv and out must both be bfloat16 or both float16")
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError("query heads must be a multiple of key heads")
    if batch < 0 or seq < 0 or shape != (batch * seq, (heads + 2 * kv_heads) * HEAD_DIM) or \
            out.shape != (batch * seq, heads * HEAD_DIM):
        raise ValueError(f"expected qkv [{batch * seq}, {(heads + 2 * kv_heads) * HEAD_DIM}] and out [{batch * seq}, "
                         f"{heads * HEAD_DIM}], got {tuple(shape)} and {tuple(out.shape)}")
    (ld_in, one), (ld_out, out_one) = qkv.stride(), out.stride()
    if one != 1 or out_one != 1:
        raise ValueError("rows of qkv and out must be contiguous")
    if window < 1 or sinks < 0:
        raise ValueError("a window has at least one key, the number of first keys is not negative")
    device = qkv.get_device()
    if out.get_device() != device:
        raise ValueError("all tensors must be on one device")
    status_ptr = 0 if status is None else _native.status_block(status, device)
    rows = batch * seq
    if rows == 0:
        return out
    qkv_ptr, out_ptr = qkv.data_ptr(), out.data_ptr()
    if rows > 1 and ld_out < heads * HEAD_DIM or not (out_ptr == qkv_ptr and (ld_out == ld_in or rows == 1)) and may_overlap(
            rows, qkv_ptr, ld_in, (heads + 2 * kv_heads) * HEAD_DIM, out_ptr, ld_out, heads * HEAD_DIM):
        raise ValueError("rows of out must not overlap, nor lie over qkv but for the query columns themselves")
    if device != _native.current_device(device):
        with torch.cuda.device(device):
            return attention_window_fwd(qkv, out, batch, seq, heads, kv_heads, window=window, sinks=sinks, status=status,
                                        timeout_ms=timeout_ms, stream=stream)
    rc = _native.entry("iris_k_attention_window_fwd")(_WINDOW_ARGS.pack(
        qkv_ptr, out_ptr, status_ptr,
        torch._C._cuda_getCurrentRawStream(device) if stream is None else stream, ld_in, ld_out, batch, seq, heads, kv_heads,
        window, sinks, _DT[dtype], int(timeout_ms * 1e6)))
    if rc != 0:
        lib = _native.kernels()
        lib.iris_attention_last_error.restype = ctypes.c_char_p
        raise RuntimeError(lib.iris_attention_last_error().decode() or f"attention launch failed ({rc})")
    return out

"""A paged key-value cache: its pages (:class:`PagedCache`), their bookkeeping on the GPU (:func:`reserve_slots`,
:func:`release_slots`, ``csrc/kernels/paged_cache.cu``) and the attention of one new token per sequence over them
(:func:`paged_attention`, ``csrc/kernels/paged_attention.cu``).

Nothing here waits for the GPU: which pages a request holds, how long it is and how many pages are free live on the device, so
a decode step, the taking of new pages included, can be recorded into a CUDA graph and replayed
(``TPDecoder.capture``).  No counterpart in the reference.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional

import torch

from .. import _native

HEAD_DIMS = (64, 128, 256)   # of paged_attention
_DT = {torch.bfloat16: 0, torch.float16: 1}
_P, _L, _I = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int
_ATTENTION, _RESERVE, _LIMITS = struct.Struct("@34qd"), struct.Struct("@17q"), struct.Struct("@2q")
_RELEASE = [_P, _P, _P, _L, _L, _P, _L, _P, _I, _L, _P]


def _ints(t: torch.Tensor, name: str, shape) -> torch.Tensor:
    if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 {list(shape)}, got {t.dtype} {list(t.shape)}")
    return t


def _rows(table: torch.Tensor, batch: int):
    """Shape and strides of a block table."""
    shape, strides = table.shape, table.stride()
    if table.dtype is not torch.int32 or len(shape) != 2 or shape[0] != batch or (strides[1] != 1 and shape[1] > 1) or \
            (strides[0] < shape[1] and batch > 1):
        raise ValueError(f"block_table must be int32 [{batch}, pages of a request] with contiguous rows that do not overlap")
    return shape, strides


def same_strides(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of one shape are laid out alike (along one element, a stride says nothing)."""
    return a.stride() == b.stride() or all(x == y or n < 2 for x, y, n in zip(a.stride(), b.stride(), a.shape))


def may_overlap(rows: int, a: int, a_pitch: int, a_width: int, b: int, b_pitch: int, b_width: int) -> bool:
    """Whether two matrices of 16-bit elements (address, pitch and width in elements) share memory; column blocks of one matrix,
    with its pitch, do not."""
    if a + ((rows - 1) * a_pitch + a_width) * 2 <= b or b + ((rows - 1) * b_pitch + b_width) * 2 <= a:
        return False
    if a_pitch == b_pitch and rows > 1:
        off = (b - a) % (a_pitch * 2) if a_pitch else 0
        return off < a_width * 2 or off + b_width * 2 > a_pitch * 2
    return True


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    lens: torch.Tensor, out: torch.Tensor, *, window: int = 0, sinks: int = 0, scale: Optional[float] = None,
                    lse: Optional[torch.Tensor] = None, longest: Optional[int] = None, status: Optional[torch.Tensor] = None,
                    timeout_ms: float = 2000.0, stream=None) -> torch.Tensor:
    """Attention of every sequence's newest token over its cached keys and values.

    ``q`` and ``out`` are ``[batch, heads, head_dim]`` (any strides with contiguous heads, e.g. the query columns of a
    projection), ``k_cache`` / ``v_cache`` ``[pages, page_size, kv_heads, head_dim]`` with equal strides, in any order with
    contiguous heads; ``head_dim`` 64, 128 or 256, ``page_size`` a power of two, query head ``h`` reads key head
    ``h // (heads // kv_heads)``.  ``block_table`` int32 ``[batch, max_pages]``: key ``j`` of a sequence lies in page
    ``block_table[b, j // page_size]``; ``lens`` int32 ``[batch]``: keys of each sequence, the newest token's included.  With
    ``window`` the token sees the last ``window`` keys (its own among them) and the first ``sinks``.  ``scale`` defaults to
    ``head_dim ** -0.5``.  ``lse`` fp32 ``[batch, heads]``: receives the logarithm of the softmax's sum.

    A sequence of no keys gets zeros (and minus infinity in ``lse``); a length beyond the table's width is cut to it, a negative
    one counts as 0.  Keys and values behind a sequence's last key, or out of its window, reach nothing, NaN or not; a seen value
    that is infinite makes its component infinite or NaN.  A key whose table entry is no page is left out and recorded in ``status``
    (an ``Iris`` context's status block) if that is given, as is a bounded wait of the kernel that ran out (the output then means
    nothing).  ``out`` may be ``q`` itself; otherwise what is written shares no memory with anything else.  ``longest``: what the lengths are
    expected not to exceed, where that is much less than the table's width; it is for speed alone.
    """
    dtype, shape, cache_shape = q.dtype, q.shape, k_cache.shape
    if dtype not in _DT or out.dtype is not dtype or k_cache.dtype is not dtype or v_cache.dtype is not dtype:
        raise TypeError("q, out and the cache must all be bfloat16 or all float16")
    if len(shape) != 3 or out.shape != shape or len(cache_shape) != 4 or v_cache.shape != cache_shape:
        raise ValueError("expected q and out [batch, heads, head_dim] and a cache [pages, page_size, kv_heads, head_dim]")
    batch, heads, dim = shape
    pages, size, kv_heads, cache_dim = cache_shape
    if cache_dim != dim or kv_heads < 1 or heads < 1 or heads % kv_heads or dim not in HEAD_DIMS:
        raise ValueError(f"{heads} query heads of {dim} do not go with {kv_heads} key heads of {cache_dim} (64, 128 or 256)")
    q_batch, q_head, q_one = q.stride()
    out_batch, out_head, out_one = out.stride()
    strides = page, slot, head, one = k_cache.stride()
    if one != 1 or q_one != 1 or out_one != 1 or (v_cache.stride() != strides and not same_strides(k_cache, v_cache)):
        raise ValueError("k_cache and v_cache must have the same strides, and all heads be contiguous")
    (rows, wide), (table_pitch, table_one) = block_table.shape, block_table.stride()
    if (block_table.dtype is not torch.int32 or rows != batch or (table_one != 1 and wide > 1) or lens.dtype is not torch.int32 or
            lens.nbytes != 4 * batch or not lens.is_contiguous()):
        raise ValueError(f"block_table must be int32 [{batch}, pages of a sequence] with contiguous rows, lens contiguous int32 [{batch}]")
    if (batch > 1 and out_batch < dim) or (heads > 1 and out_head < dim):
        raise ValueError("rows of out must not overlap")
    device = q.get_device()
    same = (out.get_device() == device and k_cache.get_device() == device and v_cache.get_device() == device and
            block_table.get_device() == device and lens.get_device() == device)
    lse_ptr = lse_batch = status_ptr = 0
    if lse is not None:
        (lse_batch, lse_one) = lse.stride()
        if (lse.dtype is not torch.float32 or lse.shape != (batch, heads) or (lse_one != 1 and heads > 1) or
                (batch > 1 and lse_batch < heads)):
            raise ValueError(f"lse must be fp32 [{batch}, {heads}], with rows that are contiguous and do not overlap")
        same = same and lse.get_device() == device
        lse_ptr = lse.data_ptr()
    if not same:
        raise ValueError("all tensors must be on one device")
    if status is not None:
        status_ptr = _native.status_block(status, device)
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must not be negative")
    if batch == 0:
        return out
    if device != _native.current_device(device):
        with torch.cuda.device(device):
            return paged_attention(q, k_cache, v_cache, block_table, lens, out, window=window, sinks=sinks, scale=scale, lse=lse,
                                   longest=longest, status=status, timeout_ms=timeout_ms, stream=stream)
    fn = _native.entry("iris_k_paged_attention")
    current = torch._C._cuda_getCurrentRawStream(device)
    work_ptr = work_bytes = 0
    while True:
        rc = fn(_ATTENTION.pack(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), lens.data_ptr(), out.data_ptr(), lse_ptr,
            work_ptr, status_ptr, current if stream is None else stream, q_batch, q_head, page, slot, head, table_pitch, out_batch,
            out_head, lse_batch, batch, heads, dim, pages, size, kv_heads, wide, _DT[dtype], window, sinks, longest or 0,
            -1, work_bytes, device, int(timeout_ms * 1e6), dim ** -0.5 if scale is None else scale))
        if rc <= 0 or work_bytes:
            break
        # sums of sequences that several CTAs share: memory of this call alone, and of the stream that it runs on
        if stream is None or stream == current:
            work = torch.empty(rc, dtype=torch.uint8, device=q.device)
        else:
            with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=q.device)):
                work = torch.empty(rc, dtype=torch.uint8, device=q.device)
        work_ptr, work_bytes = work.data_ptr(), rc
    if rc:
        lib = _native.kernels()
        lib.iris_paged_attention_last_error.restype = ctypes.c_char_p
        raise RuntimeError(lib.iris_paged_attention_last_error().decode() or f"paged attention failed ({rc})")
    return out


def reserve_slots(lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                  free_count: torch.Tensor, page_size: int, slots: torch.Tensor, positions: torch.Tensor, *,
                  row_stride: int = 0, lens_out: Optional[torch.Tensor] = None, free_count_out: Optional[torch.Tensor] = None,
                  max_len: Optional[int] = None, fresh: bool = False, stream=None) -> None:
    """Takes pages for ``new_lens[b]`` further tokens of every request ``b``, and says where those tokens go.

    Request ``b`` holds ``lens[b]`` tokens in pages ``block_table[b, :]``.  In the requests' order, each takes the pages it lacks
    from the end of the ``free_count[0]`` entries of ``free_pages``; they are written into ``block_table``.  ``slots`` and
    ``positions`` receive, for the row of every new token, page * page_size + place in the page, and the token's position in its
    request: with ``row_stride`` 0 the requests' tokens are packed one behind the other, else request ``b`` has rows
    ``b * row_stride`` on.  Rows of no token get -1 in both.  ``lens_out`` / ``free_count_out`` (default: ``lens`` and
    ``free_count``, in place) receive the new lengths and count; nothing else that is written may share memory.  ``new_lens`` below 0
    count as 0.

    A request for which the free pages do not last (nor for any later one that lacks a page), whose tokens do not fit its row of
    the table, or have not enough rows, or which would hold more than ``max_len`` tokens, gets nothing: its length stays, its rows
    get -1.  With ``fresh`` neither does a request that holds tokens already.  All tensors int32.
    """
    # (every look at a tensor costs the host 0.06 to 0.12 us, on a path of 7: sizes in bytes and straight chains, not shapes and loops)
    i32 = torch.int32
    lens_out = lens if lens_out is None else lens_out
    free_count_out = free_count if free_count_out is None else free_count_out
    if not (lens.dtype is i32 and new_lens.dtype is i32 and free_pages.dtype is i32 and free_count.dtype is i32 and
            slots.dtype is i32 and positions.dtype is i32 and lens_out.dtype is i32 and free_count_out.dtype is i32 and
            lens.is_contiguous() and new_lens.is_contiguous() and free_pages.is_contiguous() and slots.is_contiguous() and
            positions.is_contiguous() and lens_out.is_contiguous()):
        raise ValueError("all tensors must be int32 and contiguous (block_table: its rows)")
    size, rows = lens.nbytes, slots.nbytes
    if new_lens.nbytes != size or lens_out.nbytes != size or positions.nbytes != rows or free_count.nbytes != 4 or free_count_out.nbytes != 4:
        raise ValueError("lens, new_lens and lens_out must be of one length, as slots and positions, and the counts of one element")
    batch, tokens = size // 4, rows // 4
    table_shape, (pitch, one) = _rows(block_table, batch)
    if page_size < 1 or page_size & (page_size - 1):
        raise ValueError("page_size must be a power of two")
    if row_stride < 0 or tokens < batch * row_stride:
        raise ValueError(f"{tokens} rows do not hold {batch} requests of {row_stride}")
    if max_len is not None and max_len < 0:
        raise ValueError("max_len must not be negative")
    device = lens.get_device()
    if not (new_lens.get_device() == device and block_table.get_device() == device and free_pages.get_device() == device and
            free_count.get_device() == device and slots.get_device() == device and positions.get_device() == device and
            lens_out.get_device() == device and free_count_out.get_device() == device):
        raise ValueError("all tensors must be on one device")
    if batch == 0 or table_shape[1] == 0:
        raise ValueError("no requests, or no room in the block table")
    if device != _native.current_device(device):
        with torch.cuda.device(device):
            return reserve_slots(lens, new_lens, block_table, free_pages, free_count, page_size, slots, positions,
                                 row_stride=row_stride, lens_out=lens_out, free_count_out=free_count_out, max_len=max_len,
                                 fresh=fresh, stream=stream)
    args = _RESERVE.pack(
        lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(),
        slots.data_ptr(), positions.data_ptr(), lens_out.data_ptr(), free_count_out.data_ptr(),
        torch._C._cuda_getCurrentRawStream(device) if stream is None else stream, pitch, table_shape[1], free_pages.nbytes // 4,
        page_size, batch, tokens, row_stride)
    if max_len is None and not fresh:
        rc = _native.entry("iris_k_reserve_slots")(args)
    else:
        rc = _native.entry("iris_k_reserve_slots_within")(args + _LIMITS.pack(0x7fffffff if max_len is None else min(max_len, 0x7fffffff), fresh))
    if rc:
        _raise("reserve_slots", rc)


def release_slots(lens: torch.Tensor, which: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                  free_count: torch.Tensor, page_size: int, *, stream=None) -> None:
    """Gives the pages of the requests with ``which[b] != 0`` (int32) back to the end of the list of free pages; their lengths
    become 0 and their entries of the table -1.  A request whose pages the list has no room for keeps them (that, and all later
    ones that hold any).  Negative entries are no pages: a program may put back pages of a row itself (those that a window has left
    behind) and write -1 in their places.  ``which`` may be ``lens``; nothing else shares memory."""
    batch = lens.shape[0] if lens.dim() == 1 else -1
    _ints(lens, "lens", (batch,))
    _ints(which, "which", (batch,))
    table_shape, (pitch, one) = _rows(block_table, batch)
    if free_pages.dim() != 1:
        raise ValueError("free_pages must be 1-D")
    _ints(free_pages, "free_pages", free_pages.shape)
    _ints(free_count, "free_count", (1,))
    if page_size < 1 or page_size & (page_size - 1):
        raise ValueError("page_size must be a power of two")
    device = lens.get_device()
    for t in (which, block_table, free_pages, free_count):
        if t.get_device() != device:
            raise ValueError("all tensors must be on one device")
    if batch == 0 or table_shape[1] == 0:
        raise ValueError("no requests, or no room in the block table")
    if device != _native.current_device(device):
        with torch.cuda.device(device):
            return release_slots(lens, which, block_table, free_pages, free_count, page_size, stream=stream)
    lib = _native.kernels()
    rc = _native.typed(lib.iris_k_release_slots, _RELEASE)(
        lens.data_ptr(), which.data_ptr(), block_table.data_ptr(), pitch, table_shape[1],
        free_pages.data_ptr(), free_pages.shape[0], free_count.data_ptr(), page_size, batch,
        _native.current_stream(device) if stream is None else stream)
    if rc:
        _raise("release_slots", rc)


def _raise(what: str, rc: int):
    lib = _native.kernels()
    lib.iris_pages_last_error.restype = ctypes.c_char_p
    raise RuntimeError(f"{what}: " + (lib.iris_pages_last_error().decode() or f"launch failed ({rc})"))


class PagedCache:
    """Keys and values of up to ``max_batch`` requests in pages that all layers share out alike: page ``i`` of the list is page
    ``i`` in every layer.  ``k(layer)`` / ``v(layer)``: ``[pages, page_size, kv_heads, head_dim]``.  No request gets more than
    ``max_len`` tokens, whatever room its last page has."""

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, max_batch: int, max_len: int,
                 dtype: torch.dtype = torch.bfloat16, device=None):
        if min(layers, pages, page_size, kv_heads, head_dim, max_batch, max_len) < 1 or page_size & (page_size - 1):
            raise ValueError("sizes must be positive, page_size a power of two")
        if dtype not in _DT:
            raise TypeError("the cache holds bfloat16 or float16")
        self.page_size = page_size
        self.max_len = max_len
        self.data = torch.zeros((layers, 2, pages, page_size, kv_heads, head_dim), dtype=dtype, device=device)
        ints = dict(dtype=torch.int32, device=device)
        self.block_table = torch.full((max_batch, math.ceil(max_len / page_size)), -1, **ints)
        self.lens = torch.zeros(max_batch, **ints)
        self.free_pages = torch.arange(pages - 1, -1, -1, **ints)
        self.free_count = torch.full((1,), pages, **ints)

    def k(self, layer: int) -> torch.Tensor:
        return self.data[layer, 0]

    def v(self, layer: int) -> torch.Tensor:
        return self.data[layer, 1]

    def reserve(self, new_lens: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor, row_stride: int = 0,
                fresh: bool = False, stream=None) -> None:
        """:func:`reserve_slots` on this cache's requests, up to ``max_len`` tokens each; lengths and free pages are updated in place."""
        reserve_slots(self.lens, new_lens, self.block_table, self.free_pages, self.free_count, self.page_size, slots, positions,
                      row_stride=row_stride, max_len=self.max_len, fresh=fresh, stream=stream)

    def release(self, which: torch.Tensor, stream=None) -> None:
        """:func:`release_slots` on this cache's requests."""
        release_slots(self.lens, which, self.block_table, self.free_pages, self.free_count, self.page_size, stream=stream)

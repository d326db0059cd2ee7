"""8-bit paged caches: e4m3 or int8 codes with one scale for each block.

A block is one page's rows of one KV head, of K or of V.  A layer is a paged
tensor in ``kv_layout`` pages ([pages, 2, page_size, Hkv, D] or [pages, 2, Hkv,
page_size, D]) of float8_e4m3fn or int8 with its scales [pages, 2, Hkv] in
float32; a value is its code times the block's scale.

``append_quantized`` is ``write_suffix_kv`` / ``set_kv_buffer`` for such layers
(flashinfer_full_verify.py:844-855, sglang_page_attention.py:187-194),
``commit_quantized`` the route commit (target_runtime.py:910-912);
``paged_attention.paged_attention`` reads them.  A private copy of a partial page
(the tail-page copy-on-write) is the page's bytes (``kv_ops.move_slots`` on the
layers viewed as bytes) and its row of the scales.

Scales are powers of two.  The scale of a block is the least under which its largest
value fits the codes (e4m3: 448, int8: 127); rows that come later raise it when they
need to, and the rows that are there are rounded to the new scale.  Raising by a
power of two costs an e4m3 value nothing but what falls below the format's normal
range, and all the roundings of an int8 value together are off by less than one step
of its last scale.
"""

from __future__ import annotations

import ctypes
from operator import attrgetter
from typing import Sequence

import torch

from . import _lib
from .kv_ops import check_kv_layout, rows_contiguous
from .paged_attention import CACHE_CODES, _i32, cache_geometry
from .tree_attention import _host_lists


def alloc_quantized_layers(num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, *,
                           dtype: torch.dtype = torch.float8_e4m3fn, device, kv_layout: str = "NHD"):
    """(layers, scales): zeroed codes, and scales of 1, in one allocation each."""
    check_kv_layout(kv_layout)
    if dtype not in CACHE_CODES:
        raise TypeError(f"a quantised cache holds float8_e4m3fn or int8, not {dtype}")
    inner = (page_size, num_kv_heads) if kv_layout == "NHD" else (num_kv_heads, page_size)
    codes = torch.zeros((num_layers, num_pages, 2, *inner, head_dim), dtype=torch.uint8, device=device).view(dtype)
    scales = torch.ones((num_layers, num_pages, 2, num_kv_heads), dtype=torch.float32, device=device)
    return list(codes.unbind(0)), list(scales.unbind(0))


_dtype = attrgetter("dtype")


def _alike(tensors: Sequence[torch.Tensor], first: torch.Tensor) -> bool:
    """Whether all have ``first``'s shape, strides, dtype and (HIP) device."""
    if len(tensors) == 1 and tensors[0] is first:
        return True
    # (dense tensors of one shape have the same strides wherever those matter)
    dense = first.is_contiguous()
    return (set(map(torch.Tensor.size, tensors)) == {first.shape}
            and (all(map(torch.Tensor.is_contiguous, tensors)) if dense
                 else set(map(torch.Tensor.stride, tensors)) == {first.stride()})
            and set(map(_dtype, tensors)) == {first.dtype}
            and set(map(torch.Tensor.get_device, tensors)) == {first.get_device()})


def _pointers(tensors: Sequence[torch.Tensor]):
    return (ctypes.c_void_p * len(tensors))(*map(torch.Tensor.data_ptr, tensors))


def _check_layers(layers: Sequence[torch.Tensor], scales: Sequence[torch.Tensor], kv_layout: str, what: str):
    """The device and the arguments that describe the layers."""
    if not layers or len(scales) != len(layers):
        raise ValueError("one tensor of scales per layer is required")
    first, s0 = layers[0], scales[0]
    base, v_offset, (page_stride, token_stride, head_stride), (pages, page_size, hkv, d) = cache_geometry(first, kv_layout)
    device = _lib.require_device(first, s0, what=what)
    if first.dtype not in CACHE_CODES:
        raise TypeError(f"{what} writes float8_e4m3fn or int8 layers, not {first.dtype}")
    if not _alike(layers, first):
        raise ValueError("every layer must have the first layer's shape, strides, dtype and device")
    if s0.dtype != torch.float32 or s0.shape != (pages, 2, hkv) or not _alike(scales, s0):
        raise ValueError(f"every layer's scales must be float32 [{pages}, 2, {hkv}] of the same strides on {device}")
    return device, hkv, d, pages, page_size, (
        _pointers(layers), _pointers(scales), len(layers),
        CACHE_CODES[first.dtype], page_size, page_stride, v_offset, token_stride, head_stride, *s0.stride())


def append_quantized(
    layers: Sequence[torch.Tensor],
    scales: Sequence[torch.Tensor],
    k_src: Sequence[torch.Tensor],
    v_src: Sequence[torch.Tensor],
    append_indptr: torch.Tensor,
    kv_indptr: torch.Tensor,
    kv_indices: torch.Tensor,
    kv_last_page_len: torch.Tensor,
    *,
    max_append: int | None = None,
    kv_layout: str = "NHD",
) -> None:
    """Write K / V rows ([nnz, Hkv, D] fp16 or bf16 per layer) at the ends of a
    batch's requests, every layer in one launch.

    Request b's rows ``append_indptr[b] .. append_indptr[b + 1] - 1`` go to its last
    positions: ``kv_indptr`` and ``kv_last_page_len`` (int32 device tensors, as
    for the attention that follows) already count them.  ``max_append`` is the most
    rows of one request (read back from the device when left out); rows past it are not
    written.  Pages must not be shared by two requests that both write to them.

    Rows are rounded to nearest, ties to even.  Infinities become the largest
    code and do not count for a scale; NaN stays NaN in e4m3 and becomes 0 in int8."""
    device, hkv, d, pages, page_size, args = _check_layers(layers, scales, kv_layout, "append_quantized")
    where = layers[0].get_device()
    if len(k_src) != len(layers) or len(v_src) != len(layers):
        raise ValueError("one K and one V source per layer are required")
    first = k_src[0]
    if first.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"K/V rows must be float16 or bfloat16, got {first.dtype}")
    if first.ndim != 3 or tuple(first.shape[1:]) != (hkv, d) or not rows_contiguous(first):
        raise ValueError(f"K/V rows must be [nnz, {hkv}, {d}] with contiguous (Hkv, D), got {tuple(first.shape)}")
    if first.device != device or not _alike(k_src, first) or not _alike(v_src, first):
        raise ValueError(f"every K/V source must have the first one's shape, strides and dtype and be on {device}")
    nnz, stride, dtype = first.shape[0], first.stride(), first.dtype
    batch = kv_last_page_len.numel()
    if batch == 0:
        raise ValueError("the batch must hold at least one request")
    _i32(append_indptr, "append_indptr", batch + 1, where)
    _i32(kv_indptr, "kv_indptr", batch + 1, where)
    _i32(kv_last_page_len, "kv_last_page_len", batch, where)
    _i32(kv_indices, "kv_indices", kv_indices.numel(), where)
    if nnz == 0:
        return
    if max_append is None:
        rows, = _host_lists(append_indptr)
        max_append = max(b - a for a, b in zip(rows, rows[1:]))
    if max_append < 0:
        raise ValueError("max_append must not be negative")
    with _lib.on_device(device):
        rc = _lib.load().atlas_kv_append_quantized(
            *args, _pointers(k_src), _pointers(v_src),
            stride[0] if nnz > 1 else hkv * d, _lib.dtype_code(dtype), hkv, d, append_indptr.data_ptr(),
            kv_indptr.data_ptr(), kv_indices.data_ptr(), kv_last_page_len.data_ptr(), batch, int(max_append), nnz, pages,
            kv_indices.numel(), _lib.stream_of(device))
    _lib.check(rc, "atlas_kv_append_quantized")


def commit_quantized(
    layers: Sequence[torch.Tensor],
    scales: Sequence[torch.Tensor],
    src_pos: torch.Tensor,
    dst_pos: torch.Tensor,
    item_indptr: torch.Tensor,
    kv_indptr: torch.Tensor,
    kv_indices: torch.Tensor,
    *,
    max_items: int | None = None,
    kv_layout: str = "NHD",
) -> None:
    """Move rows of a batch's requests, every layer in one launch: row
    ``src_pos[i]`` of request b goes to ``dst_pos[i]`` for ``item_indptr[b] <= i <
    item_indptr[b + 1]`` (int64 positions, int32 ``item_indptr``, device
    tensors).  All of a request's sources are read before any row of it is written.

    A destination block's scale becomes the largest of its own and those of the
    blocks its rows come from; when it grows, the block's other rows are rounded to
    it.  Of rows with one destination the last stays.  At most 64 rows of one request; ``max_items`` is the most of any (read
    back when left out), rows past it stay where they are.  Requests must not
    share the pages they write to."""
    device, hkv, d, pages, page_size, args = _check_layers(layers, scales, kv_layout, "commit_quantized")
    where = layers[0].get_device()
    for t, name in ((src_pos, "src_pos"), (dst_pos, "dst_pos")):
        if t.dtype != torch.int64 or not t.is_contiguous() or t.get_device() != where:
            raise TypeError(f"{name} must be a contiguous int64 tensor on {device}")
    n = src_pos.numel()
    if dst_pos.numel() != n:
        raise ValueError("source and destination position counts differ")
    batch = item_indptr.numel() - 1
    if batch < 1:
        raise ValueError("the batch must hold at least one request")
    _i32(item_indptr, "item_indptr", batch + 1, where)
    _i32(kv_indptr, "kv_indptr", batch + 1, where)
    _i32(kv_indices, "kv_indices", kv_indices.numel(), where)
    if n == 0:
        return
    if max_items is None:
        items, = _host_lists(item_indptr)
        max_items = max(b - a for a, b in zip(items, items[1:]))
    if max_items < 0:
        raise ValueError("max_items must not be negative")
    with _lib.on_device(device):
        rc = _lib.load().atlas_kv_commit_quantized(
            *args, hkv, d, src_pos.data_ptr(), dst_pos.data_ptr(), item_indptr.data_ptr(), kv_indptr.data_ptr(),
            kv_indices.data_ptr(), batch, int(max_items), n, pages, kv_indices.numel(), _lib.stream_of(device))
    _lib.check(rc, "atlas_kv_commit_quantized")


def dequantize_layer(layer: torch.Tensor, scales: torch.Tensor, kv_layout: str = "NHD") -> torch.Tensor:
    """The layer's values in float32, in its own shape."""
    check_kv_layout(kv_layout)
    s = scales[:, :, None, :, None] if kv_layout == "NHD" else scales[:, :, :, None, None]
    return layer.float() * s


__all__ = ["alloc_quantized_layers", "append_quantized", "commit_quantized", "dequantize_layer"]

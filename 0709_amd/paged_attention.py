"""Paged attention from device-side metadata, with scored and 8-bit variants.

``paged_attention`` takes the page-table arrays of FlashInfer's paged metadata
(``qo_indptr``, ``kv_indptr``, ``kv_indices``, ``kv_last_page_len``) as device
tensors and needs no plan: the kernel reads every request's lengths itself, so a
call costs no host work per request, can be captured in a HIP graph and replayed
with other lengths, page tables and inputs in the same buffers.

For a request with n queries and L keys, query i stands at position L - n + i::

    s = sm_scale * q . k
    s = logits_soft_cap * tanh(s / logits_soft_cap)
    s = s - alibi_slopes[head] * |position(q) - position(k)|

and the output is the softmax of s over the keys the query sees, times V.  Over an
8-bit cache (e4m3 or int8 codes, ``quantized_kv.py``) k and v are the codes times
their block's scale.

The calls it extends: the Drafter's decode
(src/atlas_0709/flashinfer_paged/sglang_page_attention.py:171-209, which passes
``logits_soft_cap``, ``k_scale`` and ``v_scale`` per layer) and the Target's verify
(flashinfer_full_verify.py:953-985).
"""

from __future__ import annotations

import math
import struct

import torch

from . import _lib
from .tree_attention import _host_lists

# Most packed query rows (query token * group + head of the group) of a workgroup:
# one token per request; few rows, over 8-bit caches, over 16-bit ones, and where the page
# size is no multiple of 16; many rows.
DECODE_ROWS = 16
STREAM_ROWS_8BIT = 48
STREAM_ROWS_16BIT = 32
STREAM_ROWS_PAGES = 16
WIDE_ROWS = 256
# Requests whose rows make several such blocks stream their keys once for each; the kernel
# of many rows reads them once and takes longer to start.  It is taken when the blocks
# would stream more keys than this in all (16 bits, one request of 1000 keys and 96 rows: 13.6 us
# against 19.8; 8 of 4096 keys: 87 against 51), 8-bit caches up to MAX_STREAM_ROWS never
# (8 x 4096 keys, 192 rows: 60 us against 66; 240 rows: 79 against 71).
STREAM_KEYS_16BIT = 1 << 17
STREAM_KEYS_8BIT = 1 << 19
MAX_STREAM_ROWS = 192
# Single tokens and few rows: splits as long as one workgroup per CU makes them, between
# these (8 requests of 4096 keys: 63 us whole, 28.7 in 4 splits, 35.5 in 6; short splits even out
# requests of different lengths: 32 of 1189 to 15893 keys take 119, 105 and 118 us with at most
# 1024, 1536 and 2048 keys a split).  A request of a single token whose keys and values of a head
# are no more than WHOLE_BYTES is not split: the join costs what the splits gain (1000 codes of
# 64: 9.9 us).
CUS = 256
MIN_SPLIT_KEYS = 256
MAX_DECODE_SPLIT = 1536
MAX_STREAM_SPLIT = 4096
WHOLE_BYTES = 256 << 10
# Many rows: the workgroups that run at once (two chunks of 512 tokens: 139 us, with twice as
# many 145, three times 163).
BLOCK_WORKGROUPS = 256
MAX_SPLITS = 256
MAX_WORKGROUPS = 16384  # (splits of requests of a large batch, whose states take memory)

# A capped score is cap * (1 - 2 / (1 + e^(2 s / cap))) in 32 bits, off by up to cap * 2^-21
# however small the score: 2^-11 here, as much as a weight's rounding to fp16.
MAX_SOFT_CAP = _lib.PAGED_ATTN_MAX_SOFT_CAP

CACHE_CODES = {torch.float8_e4m3fn: _lib.CACHE_E4M3, torch.int8: _lib.CACHE_INT8}

# atlas_paged_attn_t: 14 pointers, 15 int64, 15 int32, 2 floats
_ARGS = struct.Struct("=14Q15q15i2f4x")


def launch_shape(batch: int, kv_heads: int, group: int, max_q_len: int, max_kv_len: int, *, tree: bool = False,
                 window_left: int = -1, row_bytes: int = 256, quantized: bool = False,
                 page_size: int = 16) -> tuple[bool, int, int, int, int]:
    """(single token?, rows of a block, row blocks, most splits, least keys of a split) of a
    call.  ``row_bytes`` is a cache row's size.

    One query token per request takes blocks of 16 packed rows, more take equal
    blocks.  A request takes as many splits as its own length asks for.  Behind a window
    the splits are sized for its keys; a visible prefix in front of it, which only the
    device knows, is taken to be short (a long one makes the splits longer)."""
    if window_left >= 0:
        max_kv_len = min(max_kv_len, window_left + max_q_len)
    single = max_q_len <= 1 and not tree
    rows = max(1, max_q_len * group)
    if single:
        most_rows = DECODE_ROWS
    else:
        most_rows = STREAM_ROWS_PAGES if page_size % 16 else (STREAM_ROWS_8BIT if quantized else STREAM_ROWS_16BIT)
        streamed = -(-rows // most_rows) * batch * kv_heads * max_kv_len
        if rows > most_rows and streamed > (STREAM_KEYS_8BIT if quantized else STREAM_KEYS_16BIT) and not (
                quantized and rows <= MAX_STREAM_ROWS and page_size % 16 == 0):
            most_rows = WIDE_ROWS
    blocks = -(-rows // most_rows)
    block_rows = 16 * -(-rows // (16 * blocks))
    items = batch * kv_heads * blocks
    longest = max(1, max_kv_len)
    if most_rows == WIDE_ROWS:
        keys = max(MIN_SPLIT_KEYS, -(-longest // max(1, BLOCK_WORKGROUPS // items)))
    elif single and 2 * row_bytes * longest <= WHOLE_BYTES:
        keys = longest
    else:
        keys = max(MIN_SPLIT_KEYS, -(-longest // max(1, CUS // items)))
        keys = min(keys, MAX_DECODE_SPLIT if single else MAX_STREAM_SPLIT)
    keys = max(keys, -(-longest // max(1, min(MAX_SPLITS, MAX_WORKGROUPS // items))))
    keys = -(-keys // 64) * 64
    return single, block_rows, blocks, -(-longest // keys), keys


def workspace_bytes(batch: int, kv_heads: int, head_dim: int, shape: tuple[bool, int, int, int, int]) -> int:
    """Bytes of the split states of a call of ``shape`` (``launch_shape``)."""
    _, block_rows, blocks, splits, _ = shape
    return 0 if splits == 1 else batch * kv_heads * blocks * splits * block_rows * (4 * head_dim + 4)


def _i32(t: torch.Tensor, name: str, count: int, where: int) -> None:
    """``t`` must hold ``count`` contiguous int32 on device ``where`` (``get_device()``)."""
    if t.dtype != torch.int32 or not t.is_contiguous():
        raise TypeError(f"{name} must be a contiguous int32 tensor")
    if t.get_device() != where:
        raise ValueError(f"{name} is on {t.device}, not on the cache's device")
    if t.numel() != count:
        raise ValueError(f"{name} has {t.numel()} entries, expected {count}")


def cache_geometry(paged_kv_cache, kv_layout: str):
    """(K pages, V's byte offset, (page, token, head) byte strides, (pages, page
    size, KV heads, head_dim)) of an NHD / HND cache, one tensor or a (K, V) pair."""
    if kv_layout not in ("NHD", "HND"):
        raise NotImplementedError(f"paged layout {kv_layout!r}: NHD and HND are supported")
    if isinstance(paged_kv_cache, (tuple, list)):
        base, v = paged_kv_cache
        if base.shape != v.shape or base.stride() != v.stride() or base.dtype != v.dtype or base.device != v.device:
            raise ValueError("K and V caches must have the same shape, strides, dtype and device")
        if base.ndim != 4:
            raise ValueError("tuple KV caches must be 4-dimensional")
        v_offset = v.data_ptr() - base.data_ptr()
    else:
        base = paged_kv_cache
        if base.ndim != 5 or base.shape[1] != 2:
            raise ValueError(f"kv cache must be [pages, 2, ...] of {kv_layout} pages, got {tuple(base.shape)}")
        v_offset = base.stride(1) * base.element_size()
    es = base.element_size()
    st, sh = base.stride(), base.shape
    td, hd = (-3, -2) if kv_layout == "NHD" else (-2, -3)
    if st[-1] != 1:
        raise ValueError("kv cache head rows (D) must be contiguous")
    return base, v_offset, (st[0] * es, st[td] * es, st[hd] * es), (sh[0], sh[td], sh[hd], sh[-1])


def paged_attention(
    q: torch.Tensor,
    paged_kv_cache,
    qo_indptr: torch.Tensor,
    kv_indptr: torch.Tensor,
    kv_indices: torch.Tensor,
    kv_last_page_len: torch.Tensor,
    *,
    max_q_len: int | None = None,
    max_kv_len: int | None = None,
    kv_block_scales: torch.Tensor | None = None,
    causal: bool = False,
    tree_mask: torch.Tensor | None = None,
    mask_col_start: torch.Tensor | None = None,
    window_left: int = -1,
    prefix_lens: torch.Tensor | None = None,
    logits_soft_cap: float | None = None,
    alibi_slopes: torch.Tensor | None = None,
    sm_scale: float | None = None,
    kv_layout: str = "NHD",
    out: torch.Tensor | None = None,
    lse: torch.Tensor | None = None,
    return_lse: bool = False,
    workspace: torch.Tensor | None = None,
):
    """Attention of a batch over its pages; returns ``out`` [nnz, Hq, D] (and
    ``lse`` [nnz, Hq], natural logarithm).

    ``q`` is [nnz, Hq, D] in fp16 or bf16, ``paged_kv_cache`` one tensor
    [pages, 2, ...] or a (K, V) pair in ``kv_layout`` pages, of q's type or of
    8-bit codes (float8_e4m3fn, int8) with ``kv_block_scales`` [pages, 2, Hkv]
    in float32.  The four metadata arrays are int32 device tensors.

    ``max_q_len`` and ``max_kv_len`` size the launch: of a request with more queries
    than ``max_q_len`` only the first are sure to be computed, one with more keys
    than ``max_kv_len`` is right but slower.  Left out, they are read back from the
    metadata, which waits for the device (and cannot be captured).

    Masks: none; ``causal`` with an optional ``window_left`` (keys more than that
    far behind the query are hidden) and ``prefix_lens`` [batch] (keys below it
    are visible to every query, also behind the window and ahead of the query); or
    ``tree_mask`` with ``mask_col_start`` [batch] as the verify plans hold them: int64
    [nnz] (bit j: key mask_col_start + j) or [nnz, words] (word j: keys
    64 * (mask_col_start // 64 + j) ..).  A row that sees no key gets 0 and an
    lse of -inf.  Rows past the last request's are left as they were.

    ``workspace`` (uint8, ``workspace_bytes``) holds the split states; left out, it
    comes from torch's allocator.  Calls that overlap must not share one."""
    base, v_offset, (page_stride, token_stride, head_stride), (pages, page_size, hkv, d) = cache_geometry(
        paged_kv_cache, kv_layout)
    device = _lib.require_device(q, base, what="paged attention")
    where = q.get_device()
    if q.ndim != 3 or q.stride(-1) != 1:
        raise ValueError("q must be [nnz, Hq, D] with contiguous rows")
    nnz, hq, qd = q.shape
    if qd != d or hkv == 0 or hq % hkv != 0 or hq == 0:
        raise ValueError(f"q {tuple(q.shape)} does not fit a cache of {hkv} KV heads of {d}")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"q must be float16 or bfloat16, got {q.dtype}")
    ss = (0, 0, 0)
    if base.dtype in CACHE_CODES:
        cache = CACHE_CODES[base.dtype]
        s = kv_block_scales
        if s is None:
            raise ValueError("an 8-bit cache needs kv_block_scales")
        if s.dtype != torch.float32 or s.shape != (pages, 2, hkv) or s.get_device() != where:
            raise ValueError(f"kv_block_scales must be float32 [{pages}, 2, {hkv}] on {device}")
        ss = s.stride()
    elif base.dtype == q.dtype:
        cache, s = _lib.CACHE_16BIT, None
        if kv_block_scales is not None:
            raise ValueError("kv_block_scales goes with an 8-bit cache")
    else:
        raise TypeError(f"a cache of {base.dtype} does not go with q of {q.dtype}")
    batch = kv_last_page_len.numel()
    if batch == 0:
        raise ValueError("the batch must hold at least one request")
    _i32(qo_indptr, "qo_indptr", batch + 1, where)
    _i32(kv_indptr, "kv_indptr", batch + 1, where)
    _i32(kv_last_page_len, "kv_last_page_len", batch, where)
    _i32(kv_indices, "kv_indices", kv_indices.numel(), where)
    mode, words = _lib.MASK_NONE, 1
    if tree_mask is not None:
        if causal or alibi_slopes is not None:
            raise ValueError("a tree mask goes with neither causal nor a distance bias (its nodes stand in no order)")
        if mask_col_start is None:
            raise ValueError("tree_mask needs mask_col_start")
        mode = _lib.MASK_TREE
        words = 1 if tree_mask.ndim == 1 else tree_mask.shape[1]
        if tree_mask.dtype != torch.int64 or not tree_mask.is_contiguous() or tree_mask.ndim > 2 or \
                tree_mask.shape[0] < nnz or words < 1 or tree_mask.device != device:
            raise ValueError(f"tree_mask must be contiguous int64 [{nnz}] or [{nnz}, words] on {device}")
        _i32(mask_col_start, "mask_col_start", batch, where)
    elif causal:
        mode = _lib.MASK_CAUSAL
    if mode != _lib.MASK_CAUSAL and (window_left != -1 or prefix_lens is not None):
        raise ValueError("window_left and prefix_lens go with causal=True")
    if window_left < -1:
        raise ValueError("window_left must be -1 (none) or not negative")
    window_left = min(int(window_left), 1 << 30)
    if prefix_lens is not None:
        _i32(prefix_lens, "prefix_lens", batch, where)
    if alibi_slopes is not None and (alibi_slopes.dtype != torch.float32 or alibi_slopes.numel() != hq
                                     or not alibi_slopes.is_contiguous() or alibi_slopes.device != device):
        raise ValueError(f"alibi_slopes must be contiguous float32 [{hq}] on {device}")
    cap = 0.0 if logits_soft_cap is None else float(logits_soft_cap)
    scale = 1.0 / math.sqrt(d) if sm_scale is None else float(sm_scale)
    if not (cap == 0.0 or 1e-37 <= cap <= MAX_SOFT_CAP) or not abs(scale) <= 1e37:
        raise ValueError(f"logits_soft_cap must be 0 (none) or lie in [1e-37, {MAX_SOFT_CAP}], sm_scale in [-1e37, 1e37]")
    if out is None:
        out = torch.empty((nnz, hq, d), dtype=q.dtype, device=device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(-1) != 1 or out.device != device:
        raise ValueError("out must have q's shape, dtype and device and contiguous rows")
    if lse is None:
        lse = torch.empty((nnz, hq), dtype=torch.float32, device=device) if return_lse else None
    elif lse.dtype != torch.float32 or tuple(lse.shape) != (nnz, hq) or not lse.is_contiguous() or lse.device != device:
        raise ValueError(f"lse must be contiguous float32 [{nnz}, {hq}]")
    else:
        return_lse = True
    if nnz == 0:
        return (out, lse) if return_lse else out
    if max_q_len is None or max_kv_len is None:
        qo, kvp, last = _host_lists(qo_indptr, kv_indptr, kv_last_page_len)
        if max_q_len is None:
            max_q_len = max(b - a for a, b in zip(qo, qo[1:]))
        if max_kv_len is None:
            max_kv_len = max((b - a - 1) * page_size + n if b > a else 0 for a, b, n in zip(kvp, kvp[1:], last))
    if max_q_len < 0 or max_kv_len < 0:
        raise ValueError("max_q_len and max_kv_len must not be negative")
    if max_q_len == 0:
        return (out, lse) if return_lse else out
    max_q_len, max_kv_len = min(int(max_q_len), nnz), min(int(max_kv_len), kv_indices.numel() * page_size)
    shape = launch_shape(batch, hkv, hq // hkv, max_q_len, max_kv_len, tree=mode == _lib.MASK_TREE,
                         window_left=window_left, row_bytes=d * base.element_size(), quantized=s is not None, page_size=page_size)
    need = workspace_bytes(batch, hkv, d, shape)
    if need:
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
        elif workspace.device != device or not workspace.is_contiguous() or \
                workspace.numel() * workspace.element_size() < need:
            raise ValueError(f"the workspace must hold {need} contiguous bytes on {device}")
    args = _ARGS.pack(
        q.data_ptr(), base.data_ptr(), s.data_ptr() if s is not None else 0, qo_indptr.data_ptr(), kv_indptr.data_ptr(),
        kv_indices.data_ptr(), kv_last_page_len.data_ptr(), tree_mask.data_ptr() if tree_mask is not None else 0,
        mask_col_start.data_ptr() if mode == _lib.MASK_TREE else 0,
        prefix_lens.data_ptr() if prefix_lens is not None else 0,
        alibi_slopes.data_ptr() if alibi_slopes is not None else 0, out.data_ptr(),
        lse.data_ptr() if lse is not None else 0, workspace.data_ptr() if need else 0,
        need, q.stride(0), q.stride(1), out.stride(0), out.stride(1), page_stride, v_offset, token_stride, head_stride,
        *ss, pages, kv_indices.numel(), nnz,
        batch, hq, hkv, d, page_size, _lib.dtype_code(q.dtype), cache, mode, words, window_left,
        *shape, scale, cap)
    with _lib.on_device(device):
        rc = _lib.load().atlas_paged_attn(args, _lib.stream_of(device))
    _lib.check(rc, "atlas_paged_attn")
    return (out, lse) if return_lse else out


def default_alibi_slopes(num_qo_heads: int, device: torch.device) -> torch.Tensor:
    """The usual slopes: 2^(-8 i / n), i = 1 .. n, for a power of two n of heads;
    otherwise those of the next smaller power of two, then every other one of the next
    larger."""
    def geometric(n):
        return [2.0 ** (-8.0 * i / n) for i in range(1, n + 1)]

    n = 1 << (int(num_qo_heads).bit_length() - 1)
    slopes = geometric(n) + geometric(2 * n)[0::2][: int(num_qo_heads) - n]
    return torch.tensor(slopes, dtype=torch.float32, device=device)


__all__ = ["paged_attention", "launch_shape", "workspace_bytes", "default_alibi_slopes"]

"""Refusals of paged attention and of the 8-bit cache's writes, and launch shapes, without
a device: the C entries reject before any launch, the Python checks run over host
tensors in front of a library that records its calls."""

import contextlib
import ctypes
import math

import pytest
import torch

from helpers import pkg

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn
EINVAL, EUNSUPPORTED = 1, 2


def i32(v):
    return torch.as_tensor(v, dtype=torch.int32)


# ------------------------------------------------------------------ C entries
def attn_args(**changes):
    """A valid decode call of 2 requests; pointers are never followed."""
    pa = pkg("paged_attention")
    p = 1 << 20
    fields = dict(q=p, kv=p, scales=0, qo=p, kvp=p, idx=p, last=p, tree=0, col=0, prefix=0, slopes=0, out=p, lse=0, ws=0,
                  ws_bytes=0, qst=512, qsh=128, ost=512, osh=128, page=65536, voff=32768, token=512, head=256, sp=0, sk=0,
                  sh=0, pages=10, indices=8, nnz=2, batch=2, hq=4, hkv=2, d=128, ps=16, dtype=pkg("_lib").dtype_code(BF16),
                  cache=0, mode=0, words=1, window=-1, single=1, rows=16, blocks=1, splits=1, keys=1024, sm=0.1, cap=0.0)
    assert set(changes) <= set(fields), changes
    fields.update(changes)
    return pa._ARGS.pack(*fields.values())


@pytest.mark.parametrize("changes,code", [
    (dict(q=0), EINVAL), (dict(kv=0), EINVAL), (dict(out=0), EINVAL), (dict(qo=0), EINVAL), (dict(kvp=0), EINVAL),
    (dict(last=0), EINVAL), (dict(idx=0), EINVAL), (dict(batch=0), EINVAL), (dict(nnz=-1), EINVAL), (dict(hkv=3), EINVAL),
    (dict(hq=0), EINVAL), (dict(d=96), EUNSUPPORTED), (dict(ps=0), EINVAL), (dict(pages=0), EINVAL),
    (dict(dtype=7), EINVAL), (dict(cache=3), EINVAL), (dict(cache=-1), EINVAL), (dict(cache=1), EINVAL),
    (dict(mode=3), EINVAL), (dict(mode=1, single=0), EINVAL), (dict(mode=1, tree=8, col=8), EINVAL),
    (dict(mode=1, tree=8, col=8, words=0, single=0), EINVAL), (dict(window=3), EINVAL), (dict(prefix=8), EINVAL),
    (dict(mode=1, tree=8, col=8, single=0, slopes=8), EINVAL), (dict(rows=8), EINVAL), (dict(rows=32), EINVAL),
    (dict(rows=272, single=0), EINVAL), (dict(blocks=0), EINVAL), (dict(splits=0), EINVAL), (dict(keys=100), EINVAL),
    (dict(keys=0), EINVAL), (dict(cap=-1.0), EINVAL), (dict(q=(1 << 20) + 2), EINVAL), (dict(qst=4), EINVAL),
    (dict(out=(1 << 20) + 8), EINVAL), (dict(osh=4), EINVAL), (dict(kv=(1 << 20) + 8), EINVAL), (dict(page=8), EINVAL),
    (dict(voff=8), EINVAL), (dict(token=264), EINVAL), (dict(token=128), EINVAL), (dict(head=8), EINVAL),
    (dict(indices=1 << 27), EUNSUPPORTED), (dict(nnz=1 << 30), EUNSUPPORTED), (dict(token=1 << 27), EUNSUPPORTED),
    (dict(splits=1 << 22), EUNSUPPORTED), (dict(splits=4), EINVAL), (dict(splits=4, ws=1 << 20, ws_bytes=100), EINVAL),
    (dict(splits=4, ws=(1 << 20) + 4, ws_bytes=1 << 30), EINVAL), (dict(cap=math.nan), EINVAL), (dict(cap=1e-40), EINVAL), (dict(cap=1025.0), EINVAL), (dict(sm=math.nan), EINVAL),
    (dict(sm=-2e37), EINVAL), (dict(indices=(1 << 27) - 256), EUNSUPPORTED),
])
def test_attention_entry_refuses(changes, code):
    lib, L = pkg("_lib").load(), pkg("_lib")
    want = L.ATLAS_EINVAL if code == EINVAL else L.ATLAS_EUNSUPPORTED
    assert lib.atlas_paged_attn(attn_args(**changes), None) == want
    assert lib.atlas_last_error()


def test_attention_entry_accepts_nothing_to_do():
    lib = pkg("_lib").load()
    assert lib.atlas_paged_attn(attn_args(nnz=0), None) == 0


def test_struct_matches_the_header():
    """The packed arguments are as long as the C struct (every field in its place)."""
    pa = pkg("paged_attention")
    assert pa._ARGS.size == 14 * 8 + 15 * 8 + 15 * 4 + 2 * 4 + 4


def write_args(commit=False, **changes):
    p = 1 << 20
    n = changes.pop("num_layers", 1)
    table = (ctypes.c_void_p * max(1, n))(*[changes.pop("layer", p)] * n) if n > 0 else None
    scales = (ctypes.c_void_p * max(1, n))(*[changes.pop("scale", p)] * n) if n > 0 else None
    src = (ctypes.c_void_p * max(1, n))(*[changes.pop("src", p)] * n) if n > 0 else None
    f = dict(cache=1, ps=16, page=65536, voff=32768, token=256, head=128, sp=4, sk=2, sh=1, src_stride=256,
             dtype=pkg("_lib").dtype_code(BF16), hkv=2, d=128, ap=p, kvp=p, idx=p, last=p, batch=2, most=3, nnz=4, pages=10,
             indices=6, src_pos=p, dst_pos=p, items=p)
    assert set(changes) <= set(f), changes
    f.update(changes)
    head = (table, scales, n, f["cache"], f["ps"], f["page"], f["voff"], f["token"], f["head"], f["sp"], f["sk"], f["sh"])
    if commit:
        return (*head, f["hkv"], f["d"], f["src_pos"], f["dst_pos"], f["items"], f["kvp"], f["idx"], f["batch"], f["most"],
                f["nnz"], f["pages"], f["indices"], None)
    return (*head, src, src, f["src_stride"], f["dtype"], f["hkv"], f["d"], f["ap"], f["kvp"], f["idx"], f["last"], f["batch"],
            f["most"], f["nnz"], f["pages"], f["indices"], None)


COMMON = [(dict(num_layers=0), EINVAL), (dict(layer=0), EINVAL), (dict(layer=(1 << 20) + 8), EINVAL), (dict(scale=0), EINVAL),
          (dict(cache=0), EINVAL), (dict(cache=5), EINVAL), (dict(ps=0), EINVAL), (dict(pages=0), EINVAL), (dict(hkv=0), EINVAL),
          (dict(d=80), EUNSUPPORTED), (dict(page=8), EINVAL), (dict(voff=8), EINVAL), (dict(token=8), EINVAL),
          (dict(head=8), EINVAL), (dict(kvp=0), EINVAL), (dict(idx=0), EINVAL), (dict(batch=0), EINVAL), (dict(most=-1), EINVAL),
          (dict(nnz=-1), EINVAL)]


@pytest.mark.parametrize("changes,code", COMMON + [
    (dict(src=0), EINVAL), (dict(src=(1 << 20) + 8), EINVAL), (dict(dtype=9), EINVAL), (dict(src_stride=260), EINVAL),
    (dict(src_stride=128), EINVAL), (dict(ap=0), EINVAL), (dict(last=0), EINVAL),
    (dict(batch=1 << 23), EUNSUPPORTED)])
def test_append_entry_refuses(changes, code):
    lib, L = pkg("_lib").load(), pkg("_lib")
    want = L.ATLAS_EINVAL if code == EINVAL else L.ATLAS_EUNSUPPORTED
    assert lib.atlas_kv_append_quantized(*write_args(**changes)) == want


@pytest.mark.parametrize("changes,code", COMMON + [
    (dict(src_pos=0), EINVAL), (dict(dst_pos=0), EINVAL), (dict(items=0), EINVAL), (dict(most=65), EUNSUPPORTED),
    (dict(batch=1 << 25), EUNSUPPORTED)])
def test_commit_entry_refuses(changes, code):
    lib, L = pkg("_lib").load(), pkg("_lib")
    want = L.ATLAS_EINVAL if code == EINVAL else L.ATLAS_EUNSUPPORTED
    assert lib.atlas_kv_commit_quantized(*write_args(commit=True, **changes)) == want


@pytest.mark.parametrize("commit", [False, True])
@pytest.mark.parametrize("changes", [dict(nnz=0), dict(most=0)])
def test_write_entries_accept_nothing_to_do(commit, changes):
    lib = pkg("_lib").load()
    fn = lib.atlas_kv_commit_quantized if commit else lib.atlas_kv_append_quantized
    assert fn(*write_args(commit=commit, **changes)) == 0


# ------------------------------------------------------------------ Python checks
class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append((name, args))
            return 0

        return entry


@pytest.fixture
def lib(monkeypatch):
    """Host tensors pass for device tensors in front of a library that launches nothing."""
    L, rec = pkg("_lib"), Recorder()

    def device_of(*tensors, what):
        return tensors[0].device

    monkeypatch.setattr(L, "load", lambda: rec)
    monkeypatch.setattr(L, "require_device", device_of)
    monkeypatch.setattr(L, "on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(L, "stream_of", lambda device: None)
    return rec


def attn_call(**changes):
    kw = dict(q=torch.zeros((2, 4, 128), dtype=BF16), paged_kv_cache=torch.zeros((5, 2, 16, 2, 128), dtype=BF16),
              qo_indptr=i32([0, 1, 2]), kv_indptr=i32([0, 2, 3]), kv_indices=i32([0, 1, 2]), kv_last_page_len=i32([4, 9]),
              max_q_len=1, max_kv_len=20)
    kw.update(changes)
    return pkg("paged_attention").paged_attention(**kw)


CODES = torch.zeros((5, 2, 16, 2, 128), dtype=torch.uint8).view(E4M3)
SCALES = torch.ones((5, 2, 2))


@pytest.mark.parametrize("changes,error", [
    (dict(q=torch.zeros((2, 512), dtype=BF16)), ValueError),
    (dict(q=torch.zeros((2, 4, 64), dtype=BF16)), ValueError),
    (dict(q=torch.zeros((2, 3, 128), dtype=BF16)), ValueError),
    (dict(q=torch.zeros((2, 4, 256), dtype=BF16)[..., ::2]), ValueError),
    (dict(q=torch.zeros((2, 4, 128))), TypeError),
    (dict(q=torch.zeros((2, 4, 128), dtype=torch.float16)), TypeError),
    (dict(paged_kv_cache=torch.zeros((5, 16, 2, 128), dtype=BF16)), ValueError),
    (dict(paged_kv_cache=(torch.zeros((5, 16, 2, 128), dtype=BF16), torch.zeros((4, 16, 2, 128), dtype=BF16))), ValueError),
    (dict(paged_kv_cache=(torch.zeros((2, 5, 2, 16, 128), dtype=BF16),) * 2), ValueError),
    (dict(paged_kv_cache=torch.zeros((5, 2, 16, 2, 256), dtype=BF16)[..., ::2]), ValueError),
    (dict(kv_layout="NDH"), NotImplementedError),
    (dict(paged_kv_cache=CODES), ValueError),
    (dict(paged_kv_cache=CODES, kv_block_scales=SCALES.half()), ValueError),
    (dict(paged_kv_cache=CODES, kv_block_scales=SCALES[:4]), ValueError),
    (dict(paged_kv_cache=CODES.view(torch.uint8), kv_block_scales=SCALES), TypeError),
    (dict(kv_block_scales=SCALES), ValueError),
    (dict(kv_last_page_len=i32([])), ValueError),
    (dict(qo_indptr=torch.tensor([0, 1, 2])), TypeError),
    (dict(qo_indptr=i32([0, 1])), ValueError),
    (dict(kv_indptr=i32([0, 1, 2, 3])), ValueError),
    (dict(kv_indices=torch.tensor([0, 1, 2])), TypeError),
    (dict(kv_indices=i32([0, 0, 1, 1, 2, 2])[::2]), TypeError),
    (dict(tree_mask=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(tree_mask=torch.zeros(2, dtype=torch.int64), mask_col_start=i32([0, 0]), causal=True), ValueError),
    (dict(tree_mask=torch.zeros(2, dtype=torch.int64), mask_col_start=i32([0, 0]), alibi_slopes=torch.ones(4)), ValueError),
    (dict(tree_mask=torch.zeros(1, dtype=torch.int64), mask_col_start=i32([0, 0])), ValueError),
    (dict(tree_mask=torch.zeros(2, dtype=torch.int32), mask_col_start=i32([0, 0])), ValueError),
    (dict(tree_mask=torch.zeros((2, 1, 1), dtype=torch.int64), mask_col_start=i32([0, 0])), ValueError),
    (dict(tree_mask=torch.zeros((2, 0), dtype=torch.int64), mask_col_start=i32([0, 0])), ValueError),
    (dict(tree_mask=torch.zeros(2, dtype=torch.int64), mask_col_start=i32([0])), ValueError),
    (dict(window_left=4), ValueError), (dict(prefix_lens=i32([1, 1])), ValueError),
    (dict(causal=True, window_left=-2), ValueError), (dict(causal=True, prefix_lens=i32([1])), ValueError),
    (dict(alibi_slopes=torch.ones(3)), ValueError), (dict(alibi_slopes=torch.ones(4).double()), ValueError),
    (dict(logits_soft_cap=-1.0), ValueError), (dict(logits_soft_cap=math.inf), ValueError),
    (dict(logits_soft_cap=math.nan), ValueError), (dict(logits_soft_cap=1e-50), ValueError),
    (dict(logits_soft_cap=1025.0), ValueError), (dict(sm_scale=1e39), ValueError), (dict(sm_scale=math.inf), ValueError), (dict(sm_scale=math.nan), ValueError),
    (dict(out=torch.zeros((2, 4, 128))), ValueError), (dict(out=torch.zeros((1, 4, 128), dtype=BF16)), ValueError),
    (dict(lse=torch.zeros((2, 4), dtype=BF16)), ValueError), (dict(lse=torch.zeros((4, 2)).T), ValueError),
    (dict(max_q_len=-1), ValueError), (dict(max_kv_len=-1), ValueError),
    (dict(max_kv_len=9000, kv_indices=i32([0] * 600), workspace=torch.zeros(10, dtype=torch.uint8)), ValueError),
])
def test_attention_refuses(lib, changes, error):
    with pytest.raises(error):
        attn_call(**changes)
    assert not lib.calls


def test_attention_calls(lib):
    """Sizes read back, one launch per call, none without rows; padding rows are part of the output."""
    out, lse = attn_call(max_q_len=None, max_kv_len=None, return_lse=True)
    assert out.shape == (2, 4, 128) and lse.shape == (2, 4) and len(lib.calls) == 1
    attn_call(q=torch.zeros((0, 4, 128), dtype=BF16), qo_indptr=i32([0, 0, 0]))
    attn_call(max_q_len=0)
    assert len(lib.calls) == 1
    attn_call(paged_kv_cache=CODES, kv_block_scales=SCALES, causal=True, window_left=1 << 40)
    assert len(lib.calls) == 2
    attn_call(max_q_len=1 << 40, max_kv_len=1 << 40)  # (no more than the tokens and the table hold)
    assert len(lib.calls) == 3


def append_call(**changes):
    kw = dict(layers=[CODES.clone(), CODES.clone()], scales=[SCALES.clone(), SCALES.clone()],
              k_src=[torch.zeros((3, 2, 128), dtype=BF16)] * 2, v_src=[torch.zeros((3, 2, 128), dtype=BF16)] * 2,
              append_indptr=i32([0, 2, 3]), kv_indptr=i32([0, 2, 3]), kv_indices=i32([0, 1, 2]), kv_last_page_len=i32([4, 9]),
              max_append=2)
    kw.update(changes)
    return pkg("quantized_kv").append_quantized(**kw)


ROWS = torch.zeros((3, 2, 128), dtype=BF16)
LAYER_FAULTS = [
    (dict(layers=[], scales=[]), ValueError), (dict(scales=[SCALES]), ValueError),
    (dict(layers=[CODES, CODES.view(torch.int8)]), ValueError), (dict(layers=[CODES, CODES[:4]]), ValueError),
    (dict(layers=[CODES, torch.zeros((5, 2, 16, 4, 128), dtype=torch.uint8).view(E4M3)[:, :, :, ::2]]), ValueError),
    (dict(layers=[torch.zeros((5, 2, 16, 2, 128), dtype=BF16)] * 2), TypeError),
    (dict(scales=[SCALES, SCALES.half()]), ValueError), (dict(scales=[SCALES[:4], SCALES[:4]]), ValueError),
    (dict(scales=[SCALES, torch.ones((5, 2, 4))[:, :, ::2]]), ValueError), (dict(kv_layout="NDH"), NotImplementedError),
    (dict(kv_indptr=i32([0, 1])), ValueError), (dict(kv_indices=torch.tensor([0, 1, 2])), TypeError),
]


@pytest.mark.parametrize("changes,error", LAYER_FAULTS + [
    (dict(k_src=[ROWS]), ValueError), (dict(v_src=[ROWS, ROWS[:2]]), ValueError), (dict(k_src=[ROWS, ROWS.half()]), ValueError),
    (dict(k_src=[ROWS.float()] * 2, v_src=[ROWS.float()] * 2), TypeError),
    (dict(k_src=[ROWS[:, :1]] * 2, v_src=[ROWS[:, :1]] * 2), ValueError),
    (dict(v_src=[ROWS, torch.zeros((3, 4, 128), dtype=BF16)[:, :2]]), ValueError),
    (dict(append_indptr=i32([0, 3])), ValueError), (dict(kv_last_page_len=i32([])), ValueError),
    (dict(max_append=-1), ValueError),
])
def test_append_refuses(lib, changes, error):
    with pytest.raises(error):
        append_call(**changes)
    assert not lib.calls


def commit_call(**changes):
    kw = dict(layers=[CODES.clone(), CODES.clone()], scales=[SCALES.clone(), SCALES.clone()], src_pos=torch.tensor([5, 6]),
              dst_pos=torch.tensor([1, 2]), item_indptr=i32([0, 1, 2]), kv_indptr=i32([0, 2, 3]), kv_indices=i32([0, 1, 2]),
              max_items=1)
    kw.update(changes)
    return pkg("quantized_kv").commit_quantized(**kw)


@pytest.mark.parametrize("changes,error", LAYER_FAULTS + [
    (dict(src_pos=i32([5, 6])), TypeError), (dict(dst_pos=torch.tensor([1, 0, 2, 0])[::2]), TypeError),
    (dict(dst_pos=torch.tensor([1])), ValueError), (dict(item_indptr=i32([0])), ValueError),
    (dict(item_indptr=torch.tensor([0, 1, 2])), TypeError), (dict(max_items=-1), ValueError),
])
def test_commit_refuses(lib, changes, error):
    with pytest.raises(error):
        commit_call(**changes)
    assert not lib.calls


def test_writes_call_once(lib):
    append_call(max_append=None)
    commit_call(max_items=None)
    append_call(k_src=[ROWS[:0]] * 2, v_src=[ROWS[:0]] * 2)
    commit_call(src_pos=torch.tensor([], dtype=torch.int64), dst_pos=torch.tensor([], dtype=torch.int64))
    assert [name for name, _ in lib.calls] == ["atlas_kv_append_quantized", "atlas_kv_commit_quantized"]


def test_layers_with_other_strides_and_pairs(lib):
    """Layers that are slices of one wider tensor, alike in their strides."""
    wide = torch.zeros((5, 2, 16, 4, 128), dtype=torch.uint8).view(E4M3)
    append_call(layers=[wide[:, :, :, :2], wide[:, :, :, 2:]], scales=[torch.ones((5, 2, 4))[:, :, :2]] * 2)
    assert len(lib.calls) == 1


# ------------------------------------------------------------------ launch shapes
@pytest.mark.parametrize("batch", [1, 3, 32, 300])
@pytest.mark.parametrize("hkv,group", [(8, 4), (1, 1), (2, 71)])
@pytest.mark.parametrize("tree,quantized,page", [(False, False, 16), (True, True, 16), (False, True, 7)])
def test_launch_shapes_are_accepted(batch, hkv, group, tree, quantized, page):
    """Every shape covers its rows and keys and stays within what the entry takes."""
    pa = pkg("paged_attention")
    for rows in (0, 1, 2, 12, 48, 200, 5000):
        for keys in (0, 1, 64, 1000, 16384, 1 << 22):
            single, block, blocks, splits, per = pa.launch_shape(batch, hkv, group, rows, keys, tree=tree,
                                                                 quantized=quantized, page_size=page)
            assert single == (rows <= 1 and not tree)
            assert block % 16 == 0 and 16 <= block <= (16 if single else 256) and block * blocks >= rows * group
            assert per % 64 == 0 and 1 <= splits <= pa.MAX_SPLITS and splits * per >= keys
            assert splits == 1 or batch * hkv * blocks * splits <= pa.MAX_WORKGROUPS


def test_window_sizes_the_splits():
    pa = pkg("paged_attention")
    full = pa.launch_shape(1, 8, 4, 1, 100000)
    assert full[3] > 8
    assert pa.launch_shape(1, 8, 4, 1, 100000, window_left=99)[3] == 1


def test_default_slopes():
    pa = pkg("paged_attention")
    s = pa.default_alibi_slopes(8, torch.device("cpu"))
    assert torch.equal(s, torch.tensor([2.0 ** -i for i in range(1, 9)]))
    t = pa.default_alibi_slopes(12, torch.device("cpu"))
    assert torch.equal(t[:8], s) and torch.allclose(t[8:], torch.tensor([2.0 ** -(i + 0.5) for i in range(4)]))

"""The prefill and decode wrappers with capped, windowed and biased scores and
8-bit caches: against 64 bits, and their refusals."""

import math

import pytest
import torch

from helpers import pkg
from test_gpu_paged_attention import build, check

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.as_tensor(v, dtype=torch.int32)


def workspace(dev, mb=64):
    return torch.empty(mb << 20, dtype=torch.uint8, device=dev)


def slopes_of(hq):
    return pkg("paged_attention").default_alibi_slopes(hq, torch.device("cpu"))


OPTIONS = [
    (dict(logits_soft_cap=30.0), dict(soft_cap=30.0)),
    (dict(window_left=37, causal=True), dict(window_left=37)),
    (dict(pos_encoding_mode="ALIBI", causal=True), dict(slopes=True)),
    (dict(pos_encoding_mode="ALIBI", logits_soft_cap=20.0, window_left=0, causal=True),
     dict(slopes=True, soft_cap=20.0, window_left=0)),
    (dict(logits_soft_cap=50.0, sm_scale=0.2, causal=True), dict(soft_cap=50.0, sm_scale=0.2)),
]


@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("opts,want", OPTIONS)
@pytest.mark.parametrize("cache", ["same", torch.float8_e4m3fn], ids=str)
def test_prefill(dev, layout, opts, want, cache):
    ta = pkg("tree_attention")
    s = build(101, [70, 1, 5], [300, 65, 5], hq=8, hkv=2, layout=layout, cache=cache)
    w = ta.BatchPrefillWithPagedKVCacheWrapper(workspace(dev), layout)
    w.plan(i32(s["qo"]), i32(s["kvp"]), s["table"], i32(s["last"]), 8, 2, 128, 16, q_data_type=torch.bfloat16,
           kv_data_type=None if cache == "same" else "float8_e4m3fn", **opts)
    scales = None if s["scales"] is None else s["scales"].to(dev)
    # two padded rows behind the batch stay as they were
    q = torch.cat((s["q"], torch.zeros((2, 8, 128), dtype=s["q"].dtype))).to(dev)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=dev)
    w.run(q, s["cache"].to(dev), out=out, lse=lse, kv_block_scales=scales)
    torch.cuda.synchronize()
    assert bool((out[-2:] == 7).all()) and bool((lse[-2:] == 7).all())
    want = dict(want)
    if want.pop("slopes", False):
        want["slopes"] = slopes_of(8)
    check(s, (out[:-2].cpu(), lse[:-2].cpu()), causal=opts.get("causal", False), **want)


@pytest.mark.parametrize("nodes", [12, 100])
@pytest.mark.parametrize("cache,cap", [(torch.int8, 0.0), (torch.float8_e4m3fn, 30.0), ("same", 30.0)], ids=str)
def test_prefill_with_a_tree(dev, nodes, cache, cap):
    """A draft tree's mask over an 8-bit cache, and with capped scores."""
    ta = pkg("tree_attention")
    befores = [130, 40]
    s = build(111, [nodes, nodes], [p + nodes for p in befores], hq=8, hkv=2, cache=cache)
    g = torch.Generator().manual_seed(3)
    masks = []
    for p in befores:
        parent = [int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for i in range(nodes)]
        seen = torch.zeros((nodes, nodes), dtype=torch.bool)
        for i in range(nodes):
            if parent[i] >= 0:
                seen[i] = seen[parent[i]]
            seen[i, i] = True
        masks.append(torch.cat((torch.ones((nodes, p), dtype=torch.bool), seen), 1))
    flat = torch.cat([m.reshape(-1) for m in masks])
    w = ta.BatchPrefillWithPagedKVCacheWrapper(workspace(dev), "NHD")
    w.plan(i32(s["qo"]), i32(s["kvp"]), s["table"], i32(s["last"]), 8, 2, 128, 16, custom_mask=flat.to(dev),
           q_data_type=torch.bfloat16, kv_data_type=None if cache == "same" else cache, logits_soft_cap=cap)
    got = w.run(s["q"].to(dev), s["cache"].to(dev), return_lse=True,
                kv_block_scales=None if s["scales"] is None else s["scales"].to(dev))
    torch.cuda.synchronize()
    check(s, tuple(t.cpu() for t in got), visible=masks, soft_cap=cap)


@pytest.mark.parametrize("opts,want", OPTIONS)
@pytest.mark.parametrize("cache", ["same", torch.int8], ids=str)
def test_decode(dev, opts, want, cache):
    da = pkg("decode_attention")
    s = build(121, [1] * 5, [700, 1, 64, 33, 0], hq=8, hkv=2, cache=cache, layout="HND")
    opts = {k: v for k, v in opts.items() if k != "causal"}
    want = dict(want)
    if want.pop("slopes", False):
        want["slopes"] = slopes_of(8)
    w = da.BatchDecodeWithPagedKVCacheWrapper(workspace(dev), "HND")
    w.plan(i32(s["kvp"]), s["table"], i32(s["last"]), 8, 2, 128, 16, q_data_type=torch.bfloat16,
           kv_data_type=None if cache == "same" else cache, **opts)
    scales = None if s["scales"] is None else s["scales"].to(dev)
    got = w.run(s["q"].to(dev), s["cache"].to(dev), return_lse=True, kv_block_scales=scales)
    torch.cuda.synchronize()
    check(s, tuple(t.cpu() for t in got), causal=True, **want)
    # the older entry point: its own cap and scale for a layer
    out = w.forward(s["q"].to(dev), s["cache"].to(dev), logits_soft_cap=10.0, sm_scale=0.125, kv_block_scales=scales)
    torch.cuda.synchronize()
    want.update(soft_cap=10.0, sm_scale=0.125)
    pa = pkg("paged_attention")
    direct = pa.paged_attention(
        s["q"].to(dev), s["cache"].to(dev), i32(s["qo"]).to(dev), i32(s["kvp"]).to(dev), s["table"].to(dev),
        i32(s["last"]).to(dev), max_q_len=1, max_kv_len=700, kv_block_scales=scales, kv_layout="HND", sm_scale=0.125,
        causal="window_left" in want, logits_soft_cap=10.0, window_left=want.get("window_left", -1),
        alibi_slopes=want["slopes"].to(dev) if "slopes" in want else None)
    assert torch.equal(out, direct)


def test_plans_between_the_two_kinds(dev):
    """One wrapper planned for plain, capped and again plain attention."""
    da = pkg("decode_attention")
    s = build(131, [1, 1], [200, 90], hq=8, hkv=2)
    w = da.BatchDecodeWithPagedKVCacheWrapper(workspace(dev), "NHD")
    args = (i32(s["kvp"]), s["table"], i32(s["last"]), 8, 2, 128, 16)
    q, kv = s["q"].to(dev), s["cache"].to(dev)
    for cap in (None, 30.0, 0.0, 5.0):
        w.plan(*args, q_data_type=torch.bfloat16, logits_soft_cap=cap)
        got = w.run(q, kv, return_lse=True)
        torch.cuda.synchronize()
        check(s, tuple(t.cpu() for t in got), causal=True, soft_cap=cap or 0.0)


def test_small_workspace(dev):
    """Split states that the wrapper's buffer does not hold come from the allocator."""
    da = pkg("decode_attention")
    s = build(141, [1], [5000], hq=8, hkv=2)
    w = da.BatchDecodeWithPagedKVCacheWrapper(torch.empty(64, dtype=torch.uint8, device=dev), "NHD")
    w.plan(i32(s["kvp"]), s["table"], i32(s["last"]), 8, 2, 128, 16, q_data_type=torch.bfloat16, logits_soft_cap=30.0)
    got = w.run(s["q"].to(dev), s["cache"].to(dev), return_lse=True)
    torch.cuda.synchronize()
    check(s, tuple(t.cpu() for t in got), causal=True, soft_cap=30.0)


def test_graph_over_run_follows_the_plan(dev):
    """A graph captured over run() reads the metadata of the newest plan."""
    da = pkg("decode_attention")
    w = da.BatchDecodeWithPagedKVCacheWrapper(workspace(dev), "NHD")
    a = build(151, [1, 1], [900, 40], hq=8, hkv=2)
    b = build(152, [1, 1], [33, 1500], hq=8, hkv=2)
    rows = max(a["cache"].shape[0], b["cache"].shape[0])
    kv = torch.zeros((rows, *a["cache"].shape[1:]), dtype=torch.bfloat16, device=dev)
    q = torch.zeros((2, 8, 128), dtype=torch.bfloat16, device=dev)
    out, lse = torch.zeros_like(q), torch.zeros((2, 8), device=dev)

    def put(s):
        w.plan(i32(s["kvp"]), s["table"], i32(s["last"]), 8, 2, 128, 16, q_data_type=torch.bfloat16, window_left=300,
               logits_soft_cap=30.0)
        kv[: s["cache"].shape[0]].copy_(s["cache"])
        q.copy_(s["q"])

    put(a)
    w.run(q, kv, out=out, lse=lse)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.run(q, kv, out=out, lse=lse)
    for s in (b, a, b):
        put(s)
        graph.replay()
        torch.cuda.synchronize()
        check(s, (out.cpu(), lse.cpu()), causal=True, window_left=300, soft_cap=30.0)


def test_refusals(dev):
    ta, da = pkg("tree_attention"), pkg("decode_attention")
    s = build(161, [3], [50], hq=8, hkv=2, cache=torch.int8)
    p = ta.BatchPrefillWithPagedKVCacheWrapper(workspace(dev, 8), "NHD")
    args = (i32(s["qo"]), i32(s["kvp"]), s["table"], i32(s["last"]), 8, 2, 128, 16)
    mask = torch.ones(150, dtype=torch.bool, device=dev)
    with pytest.raises(NotImplementedError):
        p.plan(*args, window_left=5)  # without causal
    with pytest.raises(NotImplementedError):
        p.plan(*args, pos_encoding_mode="ROPE_LLAMA")
    with pytest.raises(NotImplementedError):
        p.plan(*args, pos_encoding_mode="ALIBI", custom_mask=mask)
    with pytest.raises(ValueError):
        p.plan(*args, window_left=-2, causal=True)
    with pytest.raises(ValueError):
        p.plan(*args, logits_soft_cap=-1.0)
    with pytest.raises(ValueError):
        p.plan(*args, logits_soft_cap=math.inf)
    with pytest.raises(TypeError):
        p.plan(*args, q_data_type=torch.float32, kv_data_type=torch.int8)
    with pytest.raises(ValueError):
        p.plan(i32([1, 4]), *args[1:], kv_data_type=torch.int8)
    q, kv, sc = s["q"].to(dev), s["cache"].to(dev), s["scales"].to(dev)
    p.plan(*args, q_data_type=torch.bfloat16, kv_data_type=torch.int8)
    with pytest.raises(ValueError, match="kv_block_scales"):
        p.run(q, kv)
    with pytest.raises(TypeError):
        p.run(q.half(), kv, kv_block_scales=sc)
    with pytest.raises(TypeError):
        p.run(q, kv.to(torch.bfloat16), kv_block_scales=sc)
    with pytest.raises(ValueError):
        p.run(q, kv[:, :, :8], kv_block_scales=sc)
    with pytest.raises(ValueError):
        p.run(q[:2], kv, kv_block_scales=sc)
    with pytest.raises(NotImplementedError):
        p.run(q, kv, kv_block_scales=sc, append_key_states=q, append_value_states=q)
    p.plan(*args, q_data_type=torch.bfloat16)
    with pytest.raises(ValueError, match="kv_block_scales"):
        p.run(q, kv.to(torch.bfloat16), kv_block_scales=sc)
    d = da.BatchDecodeWithPagedKVCacheWrapper(workspace(dev, 8), "NHD")
    d.plan(*args[1:], q_data_type=torch.bfloat16, kv_data_type=torch.int8, logits_soft_cap=5.0)
    with pytest.raises(NotImplementedError):
        d.forward(q[:1], kv, window_left=3, kv_block_scales=sc)
    with pytest.raises(NotImplementedError):
        d.forward(q[:1], kv, pos_encoding_mode="ALIBI", kv_block_scales=sc)
    with pytest.raises(ValueError):
        d.forward(q[:1], kv, logits_soft_cap=-2.0, kv_block_scales=sc)
    with pytest.raises(NotImplementedError):
        d.run(q[:1], kv, k_scale=2.0, kv_block_scales=sc)
    with pytest.raises(NotImplementedError):
        d.plan(*args[1:], pos_encoding_mode="ROPE_LLAMA")

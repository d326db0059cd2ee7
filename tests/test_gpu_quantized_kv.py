"""8-bit caches: the quantising append and the route commit, bit for bit against
their definitions, and a run of append, verify, commit and decode together."""

import math

import pytest
import torch

from helpers import pkg
from oracle.quantized import Block8Cache
from oracle.scored_attention import scored_attention

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def tables(seed, kv_lens, ps, spare=2):
    pages = [-(-n // ps) for n in kv_lens]
    kvp = [0]
    for n in pages:
        kvp.append(kvp[-1] + n)
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(kvp[-1] + spare, generator=g)[:kvp[-1]].to(torch.int32)
    return kvp, table, [n - (p - 1) * ps if p else 0 for n, p in zip(kv_lens, pages)], kvp[-1] + spare


def random_layers(seed, count, pages, ps, hkv, d, dtype, layout):
    g = torch.Generator().manual_seed(seed)
    inner = (ps, hkv) if layout == "NHD" else (hkv, ps)
    layers, scales = [], []
    for _ in range(count):
        x = torch.randint(0, 256, (pages, 2, *inner, d), generator=g, dtype=torch.uint8)
        if dtype == INT8:
            x = torch.where(x == 128, torch.zeros_like(x), x)
        layers.append(x.view(dtype))
        scales.append(torch.exp2(torch.randint(-9, -5, (pages, 2, hkv), generator=g).float()))
    return layers, scales


def same_codes(got, want, dtype):
    """Equal values, NaN where NaN is."""
    a, b = got.cpu().float().double(), want
    return torch.equal(torch.isnan(a), torch.isnan(b)) and bool((torch.nan_to_num(a) == torch.nan_to_num(b)).all())


def i32(v, dev):
    return torch.as_tensor(v, dtype=torch.int32).to(dev)


@pytest.mark.parametrize("dtype", [E4M3, INT8], ids=str)
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ps,d,layout", [(16, 128, "HND"), (64, 64, "NHD"), (64, 128, "HND"), (1, 64, "NHD"),
                                         (5, 128, "NHD"), (200, 64, "HND")])
def test_append(dev, dtype, src, ps, d, layout):
    """Ragged appends: nothing, one row, rows that end and start inside pages,
    whole prompts; older rows kept, raised and left alone; several layers."""
    qk = pkg("quantized_kv")
    rows = [1, 0, 3, 17, 40, 64, 1, 130]
    lens = [1, 30, 16, 33, 40, 100, 64, 131]
    kvp, table, last, pages = tables(1, lens, ps)
    ap = [0]
    for n in rows:
        ap.append(ap[-1] + n)
    hkv = 3
    layers, scales = random_layers(2, 2, pages, ps, hkv, d, dtype, layout)
    g = torch.Generator().manual_seed(3)
    size = torch.exp2(torch.randint(-6, 7, (4, ap[-1], hkv, 1), generator=g).float())
    new = (torch.randn((4, ap[-1], hkv, d), generator=g) * size).to(src)
    new[:, 5:7] = 0
    new[1, 20] = -0.0
    oracles = [Block8Cache(l, s, layout) for l, s in zip(layers, scales)]
    for i, o in enumerate(oracles):
        o.append(new[i], new[2 + i], ap, kvp, table, lens)
    dl, ds = [t.to(dev) for t in layers], [t.to(dev) for t in scales]
    dn = new.to(dev)
    qk.append_quantized(dl, ds, [dn[0], dn[1]], [dn[2], dn[3]], i32(ap, dev), i32(kvp, dev), table.to(dev), i32(last, dev),
                        max_append=max(rows), kv_layout=layout)
    torch.cuda.synchronize()
    for l, s, o in zip(dl, ds, oracles):
        assert torch.equal(s.cpu().double(), o.scales)
        assert same_codes(l, o.layer(), dtype)


@pytest.mark.parametrize("dtype", [E4M3, INT8], ids=str)
def test_append_values_at_the_ends(dev, dtype):
    """Subnormal and huge rows, exact powers, values at the codes' top, ties, infinities and NaN."""
    qk = pkg("quantized_kv")
    ps, d, hkv = 16, 64, 2
    top = 448.0 if dtype == E4M3 else 127.0
    rows = [torch.full((d,), 1e-40), torch.full((d,), 3e38), torch.linspace(-top, top, d),
            torch.arange(d) + 0.5, torch.full((d,), top * 2.0 ** 5), torch.full((d,), top * 2.0 ** -5 * 1.01),
            torch.tensor([math.inf, -math.inf, math.nan, 1.0] * (d // 4)), torch.full((d,), math.inf),
            torch.full((d,), math.nan), torch.zeros(d), torch.full((d,), 2.0 ** -126),
            torch.tensor([1.0, 1.0625, 1.1875, -1.0625] * (d // 4))]
    new = torch.stack(rows).to(torch.bfloat16)[:, None, :].repeat(1, hkv, 1)
    n = new.shape[0]
    lens = [1] * n + [ps + 1] * n  # alone in a page, and behind an older row... one append each
    kvp, table, last, pages = tables(1, lens, ps)
    x = torch.cat((new, new))
    layers, scales = random_layers(4, 1, pages, ps, hkv, d, dtype, "HND")
    o = Block8Cache(layers[0], scales[0], "HND")
    ap = list(range(2 * n + 1))
    o.append(x, x.flip(0), ap, kvp, table, lens)
    dl, ds, dx = [layers[0].to(dev)], [scales[0].to(dev)], x.to(dev)
    args = (i32(ap, dev), i32(kvp, dev), table.to(dev), i32(last, dev))
    qk.append_quantized(dl, ds, [dx], [dx.flip(0)], *args, max_append=1, kv_layout="HND")
    torch.cuda.synchronize()
    assert torch.equal(ds[0].cpu().double(), o.scales)
    assert same_codes(dl[0], o.layer(), dtype)
    # behind an older row: the same rows once more, one position on
    lens2 = [v + 1 for v in lens]
    last2 = [v + 1 for v in last]
    o.append(x.roll(1, 0), x, ap, kvp, table, lens2)
    qk.append_quantized(dl, ds, [dx.roll(1, 0)], [dx], args[0], args[1], args[2], i32(last2, dev), kv_layout="HND")
    torch.cuda.synchronize()
    assert torch.equal(ds[0].cpu().double(), o.scales)
    assert same_codes(dl[0], o.layer(), dtype)


def test_append_sources_bounds_and_bad_pages(dev):
    """Row-strided sources; rows past max_append, at negative positions and on
    pages outside the pool are not written, and everything else is."""
    qk = pkg("quantized_kv")
    ps, d, hkv = 16, 64, 2
    lens = [40, 3, 20]
    rows = [10, 5, 4]
    kvp, table, last, pages = tables(5, lens, ps)
    layers, scales = random_layers(6, 1, pages, ps, hkv, d, INT8, "NHD")
    wide = torch.randn((19, 3, hkv, d)).to(torch.float16)
    src = wide[:, 1]
    o = Block8Cache(layers[0], scales[0], "NHD")
    # request 0: the first 6 of its 10 rows; request 1: its last 3 (the first two stand before 0); request 2: a bad page
    o.append(src, src, [0, 6], [0, 3], table, [36])
    o.append(src[12:15], src[12:15], [0, 3], [0, 1], table[3:], [3])
    bad = table.clone()
    bad[kvp[2] + 1] = pages
    dl, ds = [layers[0].to(dev)], [scales[0].to(dev)]
    dw = wide.to(dev)
    qk.append_quantized(dl, ds, [dw[:, 1]], [dw[:, 1]], i32([0, 10, 15, 19], dev), i32(kvp, dev), bad.to(dev),
                        i32(last, dev), max_append=6, kv_layout="NHD")
    torch.cuda.synchronize()
    assert torch.equal(ds[0].cpu().double(), o.scales)
    assert same_codes(dl[0], o.layer(), INT8)


@pytest.mark.parametrize("dtype", [E4M3, INT8], ids=str)
@pytest.mark.parametrize("ps,d,layout", [(16, 128, "HND"), (64, 64, "NHD"), (5, 128, "NHD")])
def test_commit(dev, dtype, ps, d, layout):
    """Routes that overlap their destinations, cross pages, move nothing or onto themselves; skipped items."""
    qk = pkg("quantized_kv")
    lens = [100, 77, 30, 200]
    kvp, table, last, pages = tables(7, lens, ps)
    hkv = 2
    layers, scales = random_layers(8, 3, pages, ps, hkv, d, dtype, layout)
    if dtype == E4M3:  # (a NaN code's value is NaN everywhere; keep the values comparable)
        layers = [torch.nan_to_num(t.float()).to(E4M3) for t in layers]
    src = [60, 62, 63, 70] + list(range(50, 70)) + [] + [150, 3, 4] + [10 ** 9, -1] + list(range(180, 200))
    dst = [60, 61, 62, 63] + list(range(45, 65)) + [] + [20, 150, 4] + [5, 6] + list(range(100, 120))
    items = [0, 4, 24, 24, 49]
    oracles = [Block8Cache(l, s, layout) for l, s in zip(layers, scales)]
    for o in oracles:
        o.commit(src, dst, items, kvp, table)
    dl, ds = [t.to(dev) for t in layers], [t.to(dev) for t in scales]
    qk.commit_quantized(dl, ds, torch.tensor(src, device=dev), torch.tensor(dst, device=dev), i32(items, dev), i32(kvp, dev),
                        table.to(dev), kv_layout=layout)
    torch.cuda.synchronize()
    for l, s, o in zip(dl, ds, oracles):
        assert torch.equal(s.cpu().double(), o.scales)
        assert same_codes(l, o.layer(), dtype)


@pytest.mark.parametrize("dtype", [E4M3, INT8], ids=str)
def test_append_verify_commit_decode(dev, dtype):
    """A request's life: prompt, draft tree, verify, commit of a route, decode; cache
    bit for bit, attention within its bounds, on one stream with no waits between."""
    qk, pa = pkg("quantized_kv"), pkg("paged_attention")
    ps, d, hkv, hq, layout = 16, 128, 2, 8, "HND"
    prompts, nodes, depth = [37, 70], 6, 3  # two routes of three nodes
    lens = [p + nodes for p in prompts]
    kvp, table, _, pages = tables(9, [n + 20 for n in lens], ps)
    layers, scales = qk.alloc_quantized_layers(1, pages, ps, hkv, d, dtype=dtype, device=dev, kv_layout=layout)
    o = Block8Cache(layers[0].cpu(), scales[0].cpu(), layout)
    g = torch.Generator().manual_seed(10)

    def meta(kv_lens):
        held = [-(-n // ps) for n in kv_lens]
        ptr = [0, held[0], sum(held)]
        t = torch.cat([table[kvp[b]:kvp[b] + held[b]] for b in range(2)])
        return ptr, t, [n - (h - 1) * ps for n, h in zip(kv_lens, held)]

    def append(counts, kv_lens):
        ptr, t, last = meta(kv_lens)
        ap = [0, counts[0], sum(counts)]
        k, v = (torch.randn((ap[-1], hkv, d), generator=g).to(torch.bfloat16) for _ in range(2))
        o.append(k, v, ap, ptr, t, kv_lens)
        qk.append_quantized(layers, scales, [k.to(dev)], [v.to(dev)], i32(ap, dev), i32(ptr, dev), t.to(dev), i32(last, dev),
                            max_append=max(counts), kv_layout=layout)

    def attend(n, kv_lens, visible=None, **kw):
        ptr, t, last = meta(kv_lens)
        q = torch.randn((2 * n, hq, d), generator=g).to(torch.bfloat16)
        qo = [0, n, 2 * n]
        got = pa.paged_attention(q.to(dev), layers[0], i32(qo, dev), i32(ptr, dev), t.to(dev), i32(last, dev), max_q_len=n,
                                 max_kv_len=max(kv_lens), kv_block_scales=scales[0], kv_layout=layout, return_lse=True,
                                 **kw)
        want = scored_attention(q, o.layer(), qo, ptr, t, kv_lens, page_size=ps, kv_layout=layout, scales=o.scales,
                                visible=visible, weight_eps=2.0 ** -11)
        return got, want

    results = []
    append(prompts, prompts)
    append([nodes, nodes], lens)
    words = torch.tensor([(1 << (i + 1)) - 1 if i < depth else ((1 << (i + 1)) - 1) & ~7 for i in range(nodes)] * 2)
    seen = torch.tensor([[(int(words[i]) >> j) & 1 for j in range(nodes)] for i in range(nodes)], dtype=torch.bool)
    masks = [torch.cat((torch.ones((nodes, p), dtype=torch.bool), seen), 1) for p in prompts]
    results.append(attend(nodes, lens, visible=masks, tree_mask=words.to(dev), mask_col_start=i32(prompts, dev)))
    src = [p + depth + i for p in prompts for i in range(depth)]
    dst = [p + i for p in prompts for i in range(depth)]
    ptr, t, _ = meta(lens)
    o.commit(src, dst, [0, depth, 2 * depth], ptr, t)
    qk.commit_quantized(layers, scales, torch.tensor(src, device=dev), torch.tensor(dst, device=dev),
                        i32([0, depth, 2 * depth], dev), i32(ptr, dev), t.to(dev), max_items=depth, kv_layout=layout)
    now = [p + depth for p in prompts]
    for _ in range(3):
        now = [n + 1 for n in now]
        append([1, 1], now)
        results.append(attend(1, now))
    torch.cuda.synchronize()
    assert torch.equal(scales[0].cpu().double(), o.scales)
    assert same_codes(layers[0], o.layer(), dtype)
    for (out, lse), (wo, wl, tol, ltol) in results:
        assert bool(((out.cpu().double() - wo).abs() <= tol).all())
        assert bool(((lse.cpu().double() - wl).abs() <= ltol).all())
    # the values that the cache stands for are within their codes' steps of what was appended
    back = qk.dequantize_layer(layers[0], scales[0], layout)
    assert back.shape == layers[0].shape and back.dtype == torch.float32

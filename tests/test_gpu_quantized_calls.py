"""Calls of the 8-bit writes and of attention over them that come with a serving
program: captured and replayed, many layers, two streams, odd head counts, the same
destination twice, pages far behind 2^31 bytes."""

import pytest
import torch

from helpers import pkg
from oracle.quantized import Block8Cache
from oracle.scored_attention import scored_attention
from test_gpu_quantized_kv import E4M3, INT8, i32, random_layers, same_codes, tables

pytestmark = pytest.mark.gpu


def on(dev, tensors):
    return [t.to(dev) for t in tensors]


@pytest.mark.parametrize("dtype", [E4M3, INT8], ids=str)
@pytest.mark.parametrize("ps,d,rows", [(300, 128, 290), (257, 64, 257)])
def test_append_to_long_pages(dev, dtype, ps, d, rows):
    """Pages of more rows than a workgroup's registers hold."""
    qk = pkg("quantized_kv")
    lens = [rows, ps + 3]
    kvp, table, last, pages = tables(21, lens, ps)
    layers, scales = random_layers(22, 1, pages, ps, 1, d, dtype, "NHD")
    k, v = (torch.randn((rows + ps, 1, d)).to(torch.bfloat16) for _ in range(2))
    o = Block8Cache(layers[0], scales[0], "NHD")
    ap = [0, rows, rows + ps]
    o.append(k, v, ap, kvp, table, lens)
    dl, ds = on(dev, layers), on(dev, scales)
    qk.append_quantized(dl, ds, [k.to(dev)], [v.to(dev)], i32(ap, dev), i32(kvp, dev), table.to(dev), i32(last, dev))
    torch.cuda.synchronize()
    assert torch.equal(ds[0].cpu().double(), o.scales) and same_codes(dl[0], o.layer(), dtype)


@pytest.mark.parametrize("hkv", [1, 3])
@pytest.mark.parametrize("d", [64, 128])
def test_commit_head_counts_and_full_requests(dev, hkv, d):
    """Heads that do not fill a workgroup's waves; 64 rows of a request; rows past max_items stay."""
    qk = pkg("quantized_kv")
    lens, ps = [200, 90], 16
    kvp, table, last, pages = tables(31, lens, ps)
    layers, scales = random_layers(32, 2, pages, ps, hkv, d, INT8, "HND")
    src = list(range(100, 164)) + list(range(50, 60))
    dst = list(range(90, 154)) + list(range(40, 50))
    oracles = [Block8Cache(l, s, "HND") for l, s in zip(layers, scales)]
    for o in oracles:
        o.commit(src, dst, [0, 64, 74], kvp, table)
    dl, ds = on(dev, layers), on(dev, scales)
    args = (i32(kvp, dev), table.to(dev))
    qk.commit_quantized(dl, ds, torch.tensor(src, device=dev), torch.tensor(dst, device=dev), i32([0, 64, 74], dev), *args,
                        max_items=64, kv_layout="HND")
    torch.cuda.synchronize()
    for l, s, o in zip(dl, ds, oracles):
        assert torch.equal(s.cpu().double(), o.scales) and same_codes(l, o.layer(), INT8)
    for o in oracles:  # (only the first three of each)
        o.commit(src[:3], dst[:3], [0, 3], kvp[:2], table)
        o.commit(src[64:67], dst[64:67], [0, 3], kvp[1:], table)
    qk.commit_quantized(dl, ds, torch.tensor(src, device=dev), torch.tensor(dst, device=dev), i32([0, 64, 74], dev), *args,
                        max_items=3, kv_layout="HND")
    torch.cuda.synchronize()
    for l, s, o in zip(dl, ds, oracles):
        assert torch.equal(s.cpu().double(), o.scales) and same_codes(l, o.layer(), INT8)


def test_commit_same_destination_twice(dev):
    """The last of the rows with one destination stays, whatever lies between them."""
    qk = pkg("quantized_kv")
    kvp, table, last, pages = tables(41, [120], 16)
    layers, scales = random_layers(42, 1, pages, 16, 2, 128, INT8, "NHD")
    src = [60, 61, 62, 63, 64, 65, 66, 67, 68, 69, 70]
    dst = [40, 41, 40, 42, 41, 43, 44, 45, 46, 47, 40]
    o = Block8Cache(layers[0], scales[0], "NHD")
    o.commit(src, dst, [0, 11], kvp, table)
    for _ in range(3):
        dl, ds = on(dev, layers), on(dev, scales)
        qk.commit_quantized(dl, ds, torch.tensor(src, device=dev), torch.tensor(dst, device=dev), i32([0, 11], dev),
                            i32(kvp, dev), table.to(dev))
        torch.cuda.synchronize()
        assert torch.equal(ds[0].cpu().double(), o.scales) and same_codes(dl[0], o.layer(), INT8)


def test_more_layers_than_a_launch(dev):
    qk = pkg("quantized_kv")
    n, ps, d, hkv = 70, 16, 64, 2
    kvp, table, last, pages = tables(51, [20, 9], ps)
    layers, scales = random_layers(52, n, pages, ps, hkv, d, INT8, "NHD")
    k = [torch.randn((5, hkv, d)).to(torch.float16) for _ in range(n)]
    v = [torch.randn((5, hkv, d)).to(torch.float16) for _ in range(n)]
    oracles = [Block8Cache(l, s, "NHD") for l, s in zip(layers, scales)]
    for o, kk, vv in zip(oracles, k, v):
        o.append(kk, vv, [0, 3, 5], kvp, table, [20, 9])
        o.commit([18, 7], [5, 0], [0, 1, 2], kvp, table)
    dl, ds = on(dev, layers), on(dev, scales)
    meta = (i32(kvp, dev), table.to(dev))
    qk.append_quantized(dl, ds, on(dev, k), on(dev, v), i32([0, 3, 5], dev), *meta, i32(last, dev), max_append=3)
    qk.commit_quantized(dl, ds, torch.tensor([18, 7], device=dev), torch.tensor([5, 0], device=dev), i32([0, 1, 2], dev),
                        *meta, max_items=1)
    torch.cuda.synchronize()
    for l, s, o in zip(dl, ds, oracles):
        assert torch.equal(s.cpu().double(), o.scales) and same_codes(l, o.layer(), INT8)


@pytest.mark.parametrize("dtype", [E4M3, INT8], ids=str)
def test_captured_writes(dev, dtype):
    """An append, a commit and the attention behind them in one graph, replayed with
    other rows and lengths; every replay against the eager calls on a copy."""
    qk, pa = pkg("quantized_kv"), pkg("paged_attention")
    ps, d, hkv, hq = 16, 64, 2, 8
    layers, scales = qk.alloc_quantized_layers(2, 12, ps, hkv, d, dtype=dtype, device=dev)
    other, other_scales = qk.alloc_quantized_layers(2, 12, ps, hkv, d, dtype=dtype, device=dev)
    new = torch.zeros((2, 2, 6, hkv, d), dtype=torch.bfloat16, device=dev)
    q = torch.zeros((2, hq, d), dtype=torch.bfloat16, device=dev)
    ap, kvp, table, last = i32([0, 3, 6], dev), i32([0, 6, 12], dev), torch.randperm(12).to(torch.int32).to(dev), i32([1, 1], dev)
    src, dst = torch.zeros(2, dtype=torch.int64, device=dev), torch.zeros(2, dtype=torch.int64, device=dev)
    items, qo = i32([0, 1, 2], dev), i32([0, 1, 2], dev)

    def step(lay, sca):
        qk.append_quantized(lay, sca, list(new[0].unbind(0)), list(new[1].unbind(0)), ap, kvp, table, last, max_append=3)
        qk.commit_quantized(lay, sca, src, dst, items, kvp, table, max_items=1)
        return [pa.paged_attention(q, l, qo, kvp, table, last, max_q_len=1, max_kv_len=96, kv_block_scales=s)
                for l, s in zip(lay, sca)]

    def put(turn):
        g = torch.Generator().manual_seed(turn)
        new.copy_((torch.randn(new.shape, generator=g) * 2.0 ** turn).to(torch.bfloat16))
        q.copy_(torch.randn(q.shape, generator=g).to(torch.bfloat16))
        lens = [10 * turn + 5, 6 * turn + 3]
        held = [-(-n // ps) for n in lens]
        kvp.copy_(i32([0, held[0], held[0] + held[1]], dev))
        last.copy_(i32([n - (h - 1) * ps for n, h in zip(lens, held)], dev))
        src.copy_(torch.tensor([n - 1 for n in lens]))
        dst.copy_(torch.tensor([n - 3 for n in lens]))

    put(0)
    step(layers, scales)
    step(other, other_scales)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(layers, scales)
    for turn in range(1, 6):
        put(turn)
        want = step(other, other_scales)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((*layers, *scales, *outs), (*other, *other_scales, *want)):
            assert torch.equal(a.view(torch.uint8) if a.dtype == dtype else a, b.view(torch.uint8) if b.dtype == dtype else b)


def test_writes_on_two_streams(dev):
    """Writes to two caches on two streams at once."""
    qk = pkg("quantized_kv")
    kvp, table, last, pages = tables(61, [1500, 700], 16)
    k = torch.randn((2200, 4, 128), device=dev).to(torch.bfloat16)
    meta = (i32([0, 1500, 2200], dev), i32(kvp, dev), table.to(dev), i32(last, dev))
    caches = [qk.alloc_quantized_layers(1, pages, 16, 4, 128, device=dev) for _ in range(3)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in (0, 1):
        with torch.cuda.stream(streams[i]):
            for _ in range(3):
                qk.append_quantized(*caches[i], [k], [k], *meta, max_append=1500)
    qk.append_quantized(*caches[2], [k], [k], *meta, max_append=1500)
    torch.cuda.synchronize()
    for i in (0, 1):
        assert torch.equal(caches[i][0][0].view(torch.uint8), caches[2][0][0].view(torch.uint8))
        assert torch.equal(caches[i][1][0], caches[2][1][0])


@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_pages_behind_two_gib(dev, layout):
    """A cache of more than 4 GiB: rows, scales and commits on pages at its end, and 16-bit pages there."""
    qk, pa = pkg("quantized_kv"), pkg("paged_attention")
    ps, d, hkv, hq, n = 16, 128, 8, 32, 90
    pages = (5 << 30) // (2 * ps * hkv * d)
    inner = (ps, hkv) if layout == "NHD" else (hkv, ps)
    codes = torch.empty((pages, 2, *inner, d), dtype=torch.uint8, device=dev).view(E4M3)
    scales = torch.empty((pages, 2, hkv), device=dev)
    held = -(-n // ps)
    table = torch.tensor([pages - 1 - 3 * j for j in range(held)], dtype=torch.int32)
    kvp, last = [0, held], [n - (held - 1) * ps]
    g = torch.Generator().manual_seed(71)
    k, v = (torch.randn((n, hkv, d), generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn((1, hq, d), generator=g).to(torch.bfloat16)
    o = Block8Cache(torch.zeros((held, 2, *inner, d)).to(E4M3), torch.ones((held, 2, hkv)), layout)
    near = torch.arange(held, dtype=torch.int32)
    o.append(k, v, [0, n], kvp, near, [n])
    o.commit([n - 1, n - 2], [3, 20], [0, 2], kvp, near)
    meta = (i32(kvp, dev), table.to(dev))
    qk.append_quantized([codes], [scales], [k.to(dev)], [v.to(dev)], i32([0, n], dev), *meta, i32(last, dev), max_append=n,
                        kv_layout=layout)
    qk.commit_quantized([codes], [scales], torch.tensor([n - 1, n - 2], device=dev), torch.tensor([3, 20], device=dev),
                        i32([0, 2], dev), *meta, max_items=2, kv_layout=layout)
    got = codes[table.long().to(dev)]
    torch.cuda.synchronize()
    assert torch.equal(scales[table.long().to(dev)].cpu().double(), o.scales)
    rows = torch.arange(ps)[None] < torch.tensor([ps] * (held - 1) + [last[0]])[:, None]  # the rows that are held
    at = rows[:, None, :, None, None] if layout == "NHD" else rows[:, None, None, :, None]
    assert bool((torch.where(at, got.cpu().double(), 0.0) == torch.where(at, o.layer(), 0.0)).all())

    def attend(cache, **kw):
        for tokens in (1, 40):  # the forms of few and of many rows
            qs = q.expand(tokens, hq, d).contiguous()
            out, lse = pa.paged_attention(qs.to(dev), cache, i32([0, tokens], dev), *meta, i32(last, dev),
                                          max_q_len=tokens, max_kv_len=n, kv_layout=layout, return_lse=True, **kw)
            torch.cuda.synchronize()
            yield tokens, qs, out.cpu().double(), lse.cpu().double()

    for tokens, qs, out, lse in attend(codes, kv_block_scales=scales):
        want, wl, tol, ltol = scored_attention(qs, o.layer(), [0, tokens], kvp, near, [n], page_size=ps, kv_layout=layout,
                                               scales=o.scales, weight_eps=2.0 ** -11)
        assert ((out - want).abs() <= tol).all() and ((lse - wl).abs() <= ltol).all()
    del codes
    wide = torch.empty((pages, 2, *inner, d), dtype=torch.bfloat16, device=dev)
    x = torch.randn((held, 2, *inner, d), generator=g).to(torch.bfloat16)
    wide[table.long().to(dev)] = x.to(dev)
    for tokens, qs, out, lse in attend(wide):
        want, wl, tol, ltol = scored_attention(qs, x, [0, tokens], kvp, near, [n], page_size=ps, kv_layout=layout)
        assert ((out - want).abs() <= tol).all() and ((lse - wl).abs() <= ltol).all()

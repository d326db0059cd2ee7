"""Paged attention from device-side metadata (16-bit and 8-bit caches; caps,
distance bias, windows, visible prefixes, draft trees) against 64 bits."""

import math

import pytest
import torch

from helpers import pkg
from oracle.scored_attention import scored_attention

pytestmark = pytest.mark.gpu


def build(seed, qo_lens, kv_lens, *, hq=8, hkv=2, d=128, ps=16, layout="NHD", cache="same", dtype=torch.bfloat16,
          spread=3, q_size=1.5):
    """Host tensors of a batch over scattered pages; slots that no request holds are NaN (of codes: every NaN / -128)."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // ps) for n in kv_lens]
    total = sum(pages) + 2
    kvp = [0]
    for n in pages:
        kvp.append(kvp[-1] + n)
    qo = [0]
    for n in qo_lens:
        qo.append(qo[-1] + n)
    table = torch.randperm(total, generator=g)[:kvp[-1]].to(torch.int32)
    x = torch.randn((total, 2, hkv, ps, d), generator=g)
    scales = None
    if cache == "same":
        x = x.to(dtype)
        bad = math.nan
    else:
        scales = torch.exp2(torch.randint(-spread, spread + 1, (total, 2, hkv), generator=g).float())
        top = 448.0 if cache == torch.float8_e4m3fn else 127.0
        codes = (x * top / 5).clamp(-top, top)
        scales = scales * (5 / top) * (1.0 + torch.rand(scales.shape, generator=g) * 0.5)  # any positive scale
        x = codes.to(cache) if cache == torch.float8_e4m3fn else codes.round().to(cache)
        bad = math.nan if cache == torch.float8_e4m3fn else -128
    held = torch.zeros((total, ps), dtype=torch.bool)
    for b, n in enumerate(kv_lens):
        for j in range(pages[b]):
            held[table[kvp[b] + j], :max(0, min(ps, n - j * ps))] = True
    xf = x.float()
    xf[~held[:, None, None, :, None].expand_as(xf)] = bad
    x = xf.to(x.dtype)
    if scales is not None:
        scales[~held.any(1)] = math.nan
    if layout == "NHD":
        x = x.transpose(-2, -3).contiguous()
    last = [n - (p - 1) * ps if p else 0 for n, p in zip(kv_lens, pages)]
    q = (torch.randn((qo[-1], hq, d), generator=g) * q_size).to(dtype)
    return dict(q=q, cache=x, scales=scales, qo=qo, kvp=kvp, table=table, kv_lens=kv_lens, last=last, ps=ps, layout=layout)


def call(dev, s, q=None, **kw):
    pa = pkg("paged_attention")
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).to(dev)  # noqa: E731
    kw.setdefault("max_q_len", max(b - a for a, b in zip(s["qo"], s["qo"][1:])))
    kw.setdefault("max_kv_len", max(s["kv_lens"]))
    out, lse = pa.paged_attention(
        (s["q"] if q is None else q).to(dev), s["cache"].to(dev), i32(s["qo"]), i32(s["kvp"]), i32(s["table"]), i32(s["last"]),
        kv_block_scales=None if s["scales"] is None else s["scales"].to(dev), kv_layout=s["layout"], return_lse=True, **kw)
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu()


def weight_eps(s):
    # weights are fp16 over 8-bit caches, q's type otherwise
    return 2.0 ** -8 if s["scales"] is None and s["q"].dtype == torch.bfloat16 else 2.0 ** -11


def check(s, got, **kw):
    out, lse, tol, ltol = scored_attention(s["q"], s["cache"], s["qo"], s["kvp"], s["table"], s["kv_lens"],
                                           page_size=s["ps"], kv_layout=s["layout"], scales=s["scales"],
                                           weight_eps=weight_eps(s), **kw)
    o, l = got[0].double(), got[1].double()
    assert not torch.isnan(o).any()
    worst = ((o - out).abs() / tol).max()
    assert worst <= 1, f"out off by {worst:.2f} of its bound"
    empty = lse == -math.inf
    assert torch.equal(l == -math.inf, empty) and bool((o[empty] == 0).all())
    worst = ((l - lse).abs()[~empty] / ltol[~empty]).max() if (~empty).any() else 0
    assert worst <= 1, f"lse off by {worst:.2f} of its bound"


CACHES = ["same", torch.float8_e4m3fn, torch.int8]


@pytest.mark.parametrize("cache", CACHES, ids=str)
@pytest.mark.parametrize("d,dtype", [(128, torch.bfloat16), (64, torch.float16), (64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("ps,layout", [(16, "NHD"), (64, "HND"), (48, "NHD"), (1, "NHD"), (5, "HND"), (8, "NHD")])
def test_decode(dev, cache, d, dtype, ps, layout):
    """One query per request; lengths of 0, 1, around pages and chunks, longer ones; GQA 1, 4 and 8."""
    for seed, (hq, hkv) in enumerate([(8, 2), (3, 3), (16, 2)]):
        lens = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 200, 517][seed::2] + [1000 + seed]
        s = build(seed, [1] * len(lens), lens, hq=hq, hkv=hkv, d=d, ps=ps, layout=layout, cache=cache, dtype=dtype)
        check(s, call(dev, s))


@pytest.mark.parametrize("cache", CACHES, ids=str)
@pytest.mark.parametrize("d,ps,layout", [(128, 16, "HND"), (64, 64, "NHD"), (128, 3, "NHD")])
@pytest.mark.parametrize("opts", [dict(), dict(soft_cap=30.0), dict(window_left=0), dict(window_left=37),
                                  dict(window_left=100, prefix=5), dict(prefix=64), dict(slopes=True),
                                  dict(soft_cap=5.0, slopes=True, window_left=70, prefix=1)], ids=str)
def test_causal_chunks(dev, cache, d, ps, layout, opts):
    """Ragged chunks under a causal mask with every kind of score and window,
    among them a chunk longer than its keys (its first rows see nothing) and an empty one."""
    qo, lens = [1, 7, 40, 0, 9, 33], [1, 130, 40, 50, 4, 300]
    s = build(5, qo, lens, hq=8, hkv=2, d=d, ps=ps, layout=layout, cache=cache,
              dtype=torch.float16 if d == 64 else torch.bfloat16, q_size=6.0 if "soft_cap" in opts else 1.5)
    opts = dict(opts)
    pre = opts.pop("prefix", None)
    slopes = pkg("paged_attention").default_alibi_slopes(8, torch.device("cpu")) if opts.pop("slopes", None) else None
    cap, win = opts.get("soft_cap", 0.0), opts.get("window_left", -1)
    pres = None if pre is None else [pre, 0, pre, pre, pre, 10 ** 6]
    got = call(dev, s, causal=True, logits_soft_cap=cap, window_left=win,
               prefix_lens=None if pres is None else torch.tensor(pres, dtype=torch.int32, device=dev),
               alibi_slopes=None if slopes is None else slopes.to(dev))
    check(s, got, causal=True, soft_cap=cap, window_left=win, prefix_lens=pres, slopes=slopes)


def tree_words(seen, before, wide):
    """Words of a request's [nodes, nodes] ancestor mask behind ``before`` keys."""
    n = seen.shape[0]
    if not wide:
        return [[sum(1 << j for j in range(n) if seen[i, j])] for i in range(n)]
    tiles = (before + n - 1) // 64 - before // 64 + 1
    rows = []
    for i in range(n):
        bits = [True] * (before % 64) + [bool(x) for x in seen[i]]
        bits += [False] * (tiles * 64 - len(bits))
        rows.append([sum(1 << j for j in range(64) if bits[64 * t + j]) for t in range(tiles)])
    return rows


@pytest.mark.parametrize("cache", CACHES, ids=str)
@pytest.mark.parametrize("nodes,befores", [([12, 3], [40, 0]), ([36, 64, 1], [700, 61, 129]), ([100, 70], [333, 64])])
@pytest.mark.parametrize("d,ps", [(128, 16), (64, 7)])
def test_draft_trees(dev, cache, nodes, befores, d, ps):
    """Verify of draft trees, narrow (one word a node) and wide (one per 64 keys), a cap among them."""
    g = torch.Generator().manual_seed(3)
    wide = max(nodes) > 64
    masks, words = [], []
    for n, p in zip(nodes, befores):
        seen = torch.eye(n, dtype=torch.bool)
        for i in range(1, n):
            up = int(torch.randint(-1, i, (1,), generator=g))
            if up >= 0:
                seen[i] |= seen[up]
        masks.append(torch.cat((torch.ones((n, p), dtype=torch.bool), seen), dim=1))
        words.append(tree_words(seen, p, wide))
    w = max(len(r[0]) for r in words)
    flat = [r + [0] * (w - len(r)) for rows in words for r in rows]
    flat = torch.tensor([[x - (1 << 64) if x >= 1 << 63 else x for x in r] for r in flat], dtype=torch.int64)
    if not wide:
        flat = flat[:, 0].contiguous()
    lens = [n + p for n, p in zip(nodes, befores)]
    s = build(9, nodes, lens, d=d, ps=ps, cache=cache)
    got = call(dev, s, tree_mask=flat.to(dev), mask_col_start=torch.tensor(befores, dtype=torch.int32, device=dev),
               logits_soft_cap=20.0)
    check(s, got, visible=masks, soft_cap=20.0)


@pytest.mark.parametrize("cache", ["same", torch.float8_e4m3fn], ids=str)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_hidden_keys_do_not_reach_a_row(dev, cache, bad):
    """Infinities and NaN in keys and values that a row does not see: a later
    token of the chunk, one behind the window.  Rows that see them are not finite there."""
    if cache != "same" and math.isinf(bad):
        pytest.skip("e4m3 has no infinities")
    n, length, win = 20, 90, 30
    s = build(11, [n], [length], cache=cache, ps=16, layout="HND")
    x = s["cache"].float()
    spots = [75, 42]  # a token of the chunk (position 70 + i), one that leaves the window on the way
    for p in spots:
        x[s["table"][p // 16].long(), :, :, p % 16, 3::2] = bad
    s["cache"] = x.to(s["cache"].dtype)
    out, lse = call(dev, s, causal=True, window_left=win)
    clean = dict(s)
    x = s["cache"].float()
    clean["cache"] = torch.nan_to_num(x, nan=1.0, posinf=1.0, neginf=1.0).to(s["cache"].dtype)
    want, want_lse = call(dev, clean, causal=True, window_left=win)
    for i in range(n):
        me = 70 + i
        if any(p <= me and p >= me - win for p in spots):
            assert not torch.isfinite(out[i, :, 3::2]).any(), i
        else:
            assert torch.equal(out[i], want[i]) and torch.equal(lse[i], want_lse[i]), i


def test_values_not_finite_without_keys(dev):
    """V alone holds an infinity: it reaches just its dim of the rows that see it."""
    s = build(12, [6], [40], ps=16, layout="HND")
    s["cache"][s["table"][2].long(), 1, :, 37 - 32, 9] = math.inf
    s["cache"][s["table"][2].long(), 1, :, 38 - 32, 10] = -math.inf
    out, _ = call(dev, s, causal=True)
    for i in range(6):
        assert bool((out[i, :, 9] == math.inf).all()) == (34 + i >= 37)
        assert bool((out[i, :, 10] == -math.inf).all()) == (34 + i >= 38)
        keep = [j for j in range(128) if j not in (9, 10)]
        assert torch.isfinite(out[i][:, keep]).all()


@pytest.mark.parametrize("cache", CACHES, ids=str)
def test_long_contexts_split(dev, cache):
    """Few requests with many keys: every key split is joined; with and without a
    window, and a launch sized for more or fewer keys than there are."""
    s = build(21, [1, 1, 3], [9001, 4096, 77], hq=4, hkv=1, cache=cache, layout="HND")
    for kw in (dict(), dict(causal=True, window_left=5000), dict(causal=True, window_left=700)):
        for longest in (9001, 20000, 300):
            check(s, call(dev, s, max_kv_len=longest, **kw), **kw)


def test_strides_and_given_buffers(dev):
    """q and out as slices of wider tensors, K and V as a pair, scales as a
    slice, given workspace; rows behind the last request stay as they were."""
    pa = pkg("paged_attention")
    s = build(31, [2, 5], [100, 300], hq=4, hkv=2, cache=torch.float8_e4m3fn, layout="NHD", ps=16)
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).to(dev)  # noqa: E731
    meta = [i32(s["qo"]), i32(s["kvp"]), i32(s["table"]), i32(s["last"])]
    wide_q = torch.randn((9, 6, 256)).to(torch.bfloat16).to(dev)
    wide_q[:7, 1:5, 64:192] = s["q"].to(dev)
    q = wide_q[:, 1:5, 64:192]
    codes = s["cache"].to(dev)
    big = torch.zeros((codes.shape[0], 2, 16, 4, 128), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    big[:, :, :, 1:3] = codes
    k, v = big[:, 0, :, 1:3], big[:, 1, :, 1:3]
    sc = torch.full((codes.shape[0], 2, 5), math.nan, device=dev)
    sc[:, :, 2:4] = s["scales"].to(dev)
    out = torch.full((9, 4, 256), 7.0, dtype=torch.bfloat16, device=dev)[:, :, :128]
    lse = torch.full((9, 4), 7.0, device=dev)
    shape = pa.launch_shape(2, 2, 2, 5, 300)
    ws = torch.empty(max(16, pa.workspace_bytes(2, 2, 128, shape)), dtype=torch.uint8, device=dev)
    got = pa.paged_attention(q, (k, v), *meta, max_q_len=5, max_kv_len=300, kv_block_scales=sc[:, :, 2:4], causal=True,
                             out=out, lse=lse, workspace=ws)
    torch.cuda.synchronize()
    assert got[0] is out and got[1] is lse
    check(s, (out[:7].cpu(), lse[:7].cpu()), causal=True)
    assert bool((out[7:] == 7).all()) and bool((lse[7:] == 7).all())
    # sizes read back from the metadata
    out2 = pa.paged_attention(q[:7], (k, v), *meta, kv_block_scales=sc[:, :, 2:4], causal=True)
    assert torch.equal(out2.cpu(), out[:7].cpu())


def test_bad_pages_stay_inside_the_pool(dev):
    """Page ids outside the pool are read as its nearest page: other requests' rows
    are right, and nothing faults."""
    s = build(41, [1, 1, 1], [40, 50, 60], cache=torch.int8)
    want = call(dev, s)
    s["table"] = s["table"].clone()
    s["table"][s["kvp"][1]] = -5
    s["table"][s["kvp"][1] + 1] = 1 << 30
    got = call(dev, s)
    for b in (0, 2):
        assert torch.equal(got[0][b], want[0][b])


def test_graph_replays_with_other_lengths(dev):
    """Two graphs captured over one call each, replayed in turn with other lengths,
    pages and queries in the same buffers, an eager call between."""
    pa = pkg("paged_attention")
    a = build(51, [1, 1], [900, 40], hq=8, hkv=2, cache=torch.float8_e4m3fn, ps=16)
    b = build(52, [1, 1], [17, 640], hq=8, hkv=2, cache=torch.float8_e4m3fn, ps=16)
    rows = max(a["cache"].shape[0], b["cache"].shape[0])
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32)  # noqa: E731
    idx = max(a["table"].numel(), b["table"].numel())
    buf = dict(q=torch.zeros((2, 8, 128), dtype=torch.bfloat16, device=dev),
               cache=torch.zeros((rows, *a["cache"].shape[1:]), dtype=torch.uint8, device=dev),
               scales=torch.ones((rows, 2, 2), device=dev), qo=i32([0, 1, 2]).to(dev), kvp=i32([0, 0, 0]).to(dev),
               table=torch.zeros(idx, dtype=torch.int32, device=dev), last=i32([0, 0]).to(dev))

    def put(s):
        buf["q"].copy_(s["q"])
        n = s["cache"].shape[0]
        buf["cache"][:n].copy_(s["cache"].view(torch.uint8))
        buf["scales"][:n].copy_(s["scales"])
        buf["kvp"].copy_(i32(s["kvp"]))
        buf["table"][:s["table"].numel()].copy_(s["table"])
        buf["last"].copy_(i32(s["last"]))

    def run():
        return pa.paged_attention(buf["q"], buf["cache"].view(torch.float8_e4m3fn), buf["qo"], buf["kvp"], buf["table"],
                                  buf["last"], max_q_len=1, max_kv_len=1024, kv_block_scales=buf["scales"],
                                  return_lse=True)

    put(a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(run())
        graphs.append(gr)
    for turn in range(4):
        s = (a, b)[turn % 2]
        put(s)
        eager = run()
        graphs[turn // 2].replay()
        torch.cuda.synchronize()
        for x, y in zip(outs[turn // 2], eager):
            assert torch.equal(x, y)
        check(s, tuple(t.cpu() for t in outs[turn // 2]))


def test_two_streams_at_once(dev):
    """Calls on two streams over one cache do not disturb each other."""
    s = build(61, [1] * 4, [700, 3000, 10, 1500], hq=8, hkv=2, cache=torch.int8)
    want = call(dev, s)
    streams = [torch.cuda.Stream() for _ in range(2)]
    pa = pkg("paged_attention")
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).to(dev)  # noqa: E731
    args = (s["q"].to(dev), s["cache"].to(dev), i32(s["qo"]), i32(s["kvp"]), i32(s["table"]), i32(s["last"]))
    scales = s["scales"].to(dev)
    torch.cuda.synchronize()
    outs = []
    for turn in range(6):
        with torch.cuda.stream(streams[turn % 2]):
            outs.append(pa.paged_attention(*args, max_q_len=1, max_kv_len=3000, kv_block_scales=scales, return_lse=True))
    torch.cuda.synchronize()
    for o, l in outs:
        assert torch.equal(o.cpu(), want[0]) and torch.equal(l.cpu(), want[1])


def test_extreme_scales_and_queries(dev):
    """Block scales far apart in one request, queries near the ends of bf16's range, a row of zeros."""
    s = build(71, [1, 1, 2], [100, 40, 64], cache=torch.float8_e4m3fn, spread=0)
    g = torch.Generator().manual_seed(1)
    k_scale = torch.exp2(torch.randint(-3, 1, s["scales"][:, 0].shape, generator=g).float()) / 90
    v_scale = torch.exp2(torch.randint(-40, 41, s["scales"][:, 1].shape, generator=g).float())
    s["scales"] = torch.stack((k_scale, v_scale), dim=1)
    q = s["q"].float()
    q[0] = 0
    q[2] *= 1e-30
    s["q"] = q.to(torch.bfloat16)
    got = call(dev, s)
    check(s, got)
    big = dict(s)
    big["scales"] = s["scales"].clone()
    big["scales"][:, 0] *= 2.0 ** -110
    big["q"] = (s["q"].float() * 2.0 ** 110).to(torch.bfloat16)
    check(big, call(dev, big))


@pytest.mark.parametrize("cache", CACHES, ids=str)
@pytest.mark.parametrize("scale", [-0.1, 0.0, 1e-30])
def test_other_score_scales(dev, cache, scale):
    """sm_scale negative, zero and tiny: hidden keys stay hidden, the rest is as defined."""
    s = build(81, [1, 30], [100, 90], cache=cache)
    check(s, call(dev, s, causal=True, sm_scale=scale), causal=True, sm_scale=scale)
    one = build(82, [1, 1], [100, 70], cache=cache)
    check(one, call(dev, one, causal=True, window_left=40, sm_scale=scale), causal=True, window_left=40, sm_scale=scale)


def test_nan_scores_reach_their_rows(dev):
    """A visible NaN key makes its row NaN (and no other), whichever wave or split holds it."""
    for length, spot in ((70, 3), (70, 69), (3000, 100), (3000, 2990)):
        s = build(91, [1, 1], [length, length], hq=8, hkv=2, layout="HND")
        s["cache"][s["table"][spot // 16].long(), 0, 1, spot % 16, 5] = math.nan
        out, lse = call(dev, s)
        assert torch.isnan(out[0, 4:]).all() and torch.isnan(lse[0, 4:]).all()
        assert torch.isfinite(out[0, :4]).all() and torch.isfinite(out[1]).all() and torch.isfinite(lse[1]).all()


@pytest.mark.parametrize("cache", ["same", torch.int8], ids=str)
@pytest.mark.parametrize("opts", [dict(causal=True), dict(causal=True, window_left=20), dict()])
def test_more_tokens_than_stated(dev, cache, opts):
    """max_q_len=1 over requests of several tokens: the first token of each is right
    (at its own position), the others stay as they were."""
    s = build(171, [3, 1, 2], [700, 1300, 5], cache=cache)
    out, lse = torch.full(s["q"].shape, 7.0, dtype=torch.bfloat16, device=dev), torch.full((6, 8), 7.0, device=dev)
    call(dev, s, max_q_len=1, out=out, lse=lse, **opts)
    want, wl, tol, ltol = scored_attention(s["q"], s["cache"], s["qo"], s["kvp"], s["table"], s["kv_lens"], page_size=16,
                                           kv_layout="NHD", scales=s["scales"], weight_eps=weight_eps(s), **opts)
    first = [0, 3, 4]
    assert ((out.cpu().double() - want).abs() <= tol)[first].all()
    assert ((lse.cpu().double() - wl).abs() <= ltol)[first].all()
    for row in (1, 2, 5):
        assert bool((out[row] == 7).all()) and bool((lse[row] == 7).all())


@pytest.mark.parametrize("cache", CACHES, ids=str)
@pytest.mark.parametrize("hq,hkv", [(40, 2), (17, 1), (6, 2), (71, 1)])
@pytest.mark.parametrize("n", [1, 2, 9])
def test_group_sizes(dev, cache, hq, hkv, n):
    """Groups of more query heads than a row tile, and odd ones."""
    s = build(181, [n, 1], [300, 2000], hq=hq, hkv=hkv, cache=cache, ps=32)
    check(s, call(dev, s, causal=True), causal=True)


@pytest.mark.parametrize("cache", ["same", torch.float8_e4m3fn], ids=str)
@pytest.mark.parametrize("prefix", [0, 5, 700])
def test_windows_behind_long_prefixes(dev, cache, prefix):
    """The splits are sized for the window; a prefix that is longer is still whole."""
    s = build(191, [1, 1, 4], [900, 3000, 1500], cache=cache)
    pre = torch.tensor([prefix] * 3, dtype=torch.int32)
    check(s, call(dev, s, causal=True, window_left=40, prefix_lens=pre.to(dev)), causal=True, window_left=40, prefix_lens=pre)


def test_extreme_caps(dev):
    """The smallest and the largest cap that are taken."""
    s = build(201, [1, 3], [300, 50])
    for cap in (1e-37, 1e-3, 1024.0):
        check(s, call(dev, s, causal=True, logits_soft_cap=cap), causal=True, soft_cap=cap)


def test_large_batches_and_lengths_stated(dev):
    """Many requests, and a max_kv_len far above any: few splits are left, and the rows are the same."""
    s = build(211, [1] * 80, [17 * i % 400 for i in range(80)], hq=8, hkv=2, cache=torch.int8)
    a, b = call(dev, s), call(dev, s, max_kv_len=1 << 40)
    check(s, a)
    check(s, b)

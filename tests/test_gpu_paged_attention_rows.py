"""The tests of paged attention again where the kernel of many rows takes every call
that it can (small calls stream otherwise), and batches of many rows with empty requests."""

import pytest
import torch

from helpers import pkg
from test_gpu_paged_attention import (  # noqa: F401  (collected here under the fixture below)
    CACHES, build, call, check,
    test_bad_pages_stay_inside_the_pool, test_causal_chunks, test_draft_trees, test_extreme_caps,
    test_extreme_scales_and_queries, test_group_sizes, test_hidden_keys_do_not_reach_a_row, test_long_contexts_split,
    test_nan_scores_reach_their_rows, test_other_score_scales, test_strides_and_given_buffers,
    test_values_not_finite_without_keys, test_windows_behind_long_prefixes)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def many_rows(monkeypatch):
    pa = pkg("paged_attention")
    for name in ("STREAM_KEYS_16BIT", "STREAM_KEYS_8BIT", "MAX_STREAM_ROWS"):
        monkeypatch.setattr(pa, name, 0)
    assert pa.launch_shape(1, 2, 4, 70, 300)[1] > pa.STREAM_ROWS_8BIT


@pytest.mark.parametrize("cache", CACHES, ids=str)
@pytest.mark.parametrize("ps,d", [(16, 128), (64, 64), (24, 128), (1, 64)])
def test_ragged_batches(dev, cache, ps, d):
    """Requests without queries, without keys, with fewer keys than queries, of one token, of more rows than a block."""
    s = build(301, [70, 0, 5, 40, 1, 130], [500, 300, 0, 17, 2000, 131], hq=8, hkv=2, d=d, ps=ps, cache=cache)
    check(s, call(dev, s, causal=True), causal=True)
    check(s, call(dev, s, causal=True, window_left=33, logits_soft_cap=30.0), causal=True, window_left=33, soft_cap=30.0)


@pytest.mark.parametrize("cache", CACHES, ids=str)
@pytest.mark.parametrize("tokens", [13, 64, 65, 257])
def test_row_counts(dev, cache, tokens):
    """Blocks with rows for some of the waves, and several blocks."""
    s = build(311, [tokens, tokens], [tokens + 3, 900], hq=4, hkv=1, cache=cache)
    check(s, call(dev, s, causal=True), causal=True)


@pytest.mark.parametrize("cache", CACHES, ids=str)
def test_rows_do_not_depend_on_the_batch(dev, cache):
    """A request's rows are the same bits beside other requests, and with its keys in the same parts."""
    s = build(321, [90, 33], [200, 250], cache=cache)
    a = call(dev, s, causal=True)
    one = dict(s, q=s["q"][:90], qo=s["qo"][:2], kvp=s["kvp"][:2], kv_lens=s["kv_lens"][:1], last=s["last"][:1])
    b = call(dev, one, causal=True, max_kv_len=250)
    assert torch.equal(a[0][:90], b[0]) and torch.equal(a[1][:90], b[1])


def test_graph_replays_with_other_lengths_of_many_rows(dev):
    """Chunks in a graph, replayed with other lengths and queries in the same buffers."""
    pa = pkg("paged_attention")
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32)  # noqa: E731
    states = [build(331, [100, 40], [900, 45], hq=8, hkv=2), build(332, [3, 137], [17, 640], hq=8, hkv=2)]
    rows = max(s["cache"].shape[0] for s in states)
    idx = max(s["table"].numel() for s in states)
    q = torch.zeros((140, 8, 128), dtype=torch.bfloat16, device=dev)
    cache = torch.zeros((rows, *states[0]["cache"].shape[1:]), dtype=torch.bfloat16, device=dev)
    qo, kvp, last = i32([0, 0, 0]).to(dev), i32([0, 0, 0]).to(dev), i32([0, 0]).to(dev)
    table = torch.zeros(idx, dtype=torch.int32, device=dev)

    def put(s):
        q.copy_(s["q"])
        cache[:s["cache"].shape[0]].copy_(s["cache"])
        qo.copy_(i32(s["qo"]))
        kvp.copy_(i32(s["kvp"]))
        table[:s["table"].numel()].copy_(s["table"])
        last.copy_(i32(s["last"]))

    def run():
        return pa.paged_attention(q, cache, qo, kvp, table, last, max_q_len=140, max_kv_len=1000, causal=True, return_lse=True)

    put(states[0])
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for turn in range(4):
        s = states[(turn + 1) % 2]
        put(s)
        eager = run()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, eager))
        check(s, tuple(t.cpu() for t in got), causal=True)

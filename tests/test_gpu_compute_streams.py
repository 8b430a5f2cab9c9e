"""Calls that keep partial sums (attention split over tokens, products split
over k) on several streams of one context, and captured into graphs beside
larger eager calls."""
import numpy as np
import pytest

import test_gpu_compute as G

pytestmark = pytest.mark.gpu


def attention_call(seed, tokens, heads=2):
    """A call of single rows over `tokens` tokens, split and joined; returns (call, its output buffer)."""
    t = G.T()
    n = (tokens + 15) // 16
    c = G.new_cache(n, 16, heads, 64, seed)[0]
    q = t.randn(1, 8 * heads, 64, generator=t.Generator("cuda").manual_seed(seed), device="cuda").bfloat16()
    table, start, lens = G.i32(np.random.default_rng(seed).permutation(n)[None]), G.i32([0, 1]), G.i32([tokens])
    out = t.empty_like(q)
    return (lambda: c.attention(q, table, start, lens, max_q=1, max_kv=tokens, out=out)), out


def linear_call(seed, m, n, k):
    """A product whose k is split."""
    t = G.T()
    g = t.Generator("cuda").manual_seed(seed)
    x = t.randn(m, k, generator=g, device="cuda").half()
    w = t.randn(n, k, generator=g, device="cuda").half()
    out = t.empty(m, n, dtype=t.half, device="cuda")
    return (lambda: G.K().linear(G.ctx(), x, w, out=out)), out


def test_two_streams_beside_each_other():
    t = G.T()
    calls = [[attention_call(s, 30000), linear_call(s, 80, 200, 4099), linear_call(s + 9, 70, 256, 8192)] for s in (1, 2)]
    want = [[call().clone() for call, _ in side] for side in calls]
    streams = [t.cuda.Stream(), t.cuda.Stream()]
    t.cuda.synchronize()
    for _ in range(20):
        for side in calls:
            for _, out in side:
                out.zero_()
        t.cuda.synchronize()
        for i in range(3):
            for s, side in zip(streams, calls):
                with t.cuda.stream(s):
                    side[i][0]()
        t.cuda.synchronize()
        for side, w in zip(calls, want):
            assert all(t.equal(out, x) for (_, out), x in zip(side, w))


def test_graphs_go_on_beside_larger_eager_calls():
    t = G.T()
    small = [attention_call(3, 5000), linear_call(3, 80, 200, 4099)]
    larger = [attention_call(4, 20000, heads=4), linear_call(4, 160, 400, 4099)]
    eager = [attention_call(5, 300000, heads=4), linear_call(5, 300, 900, 4099)]
    want = [[call().clone() for call, _ in side] for side in (small, larger)]
    graphs = []
    for side in (small, larger):            # the second's sums outgrow the first's
        g = t.cuda.CUDAGraph()
        with t.cuda.graph(g):
            for call, _ in side:
                call()
        graphs.append(g)
    for i in range(6):
        for call, _ in eager:
            call()
        # what was freed by now belongs to others
        others = [t.full((1 << 20,), float(i), device="cuda") for _ in range(20)]
        for g, side, w in zip(graphs, (small, larger), want):
            for _, out in side:
                out.zero_()
            g.replay()
            t.cuda.synchronize()
            assert all(t.equal(out, x) for (_, out), x in zip(side, w)), i
        assert all((o == i).all() for o in others)

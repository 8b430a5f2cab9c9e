"""hh_kv_append where a workgroup takes several rows' runs (calls of many rows
and heads): codes and scales compared exactly."""
import numpy as np
import pytest

import test_gpu_compute as G

pytestmark = pytest.mark.gpu


def span(rows, heads):
    return min(16, max(1, rows * 2 * heads // 2048))


def prompts(rng, bs, lengths, singles):
    """Runs of prompts of these lengths, from any token of a block on, with single rows of blocks of their own in between."""
    runs, block = [], 0
    for n in lengths:
        first = int(rng.integers(0, bs))
        held = (first + n + bs - 1) // bs
        runs.append((tuple(rng.permutation(held) + block), first, n))
        block += held
        for _ in range(int(rng.integers(0, singles + 1))):
            runs.append(((block,), int(rng.integers(0, bs)), 1))
            block += 1
    return runs, block


@pytest.mark.parametrize("dtype", G.DT)
@pytest.mark.parametrize("bs,dim,heads,least", [(16, 64, 8, 16), (32, 96, 8, 16), (64, 128, 4, 16), (128, 64, 16, 16),
                                                (128, 192, 2, 4), (64, 256, 2, 4)])
def test_prompts_and_single_rows(bs, dim, heads, least, dtype):
    rng = np.random.default_rng(bs + dim)
    lengths = [1, 2, 63, 64, 65, 127, 128, 129, 700] + list(rng.integers(1, 300, 30))
    runs, blocks = prompts(rng, bs, [int(n) for n in lengths], 3)
    assert span(sum(r[2] for r in runs), heads) >= least
    G.check_append(bs, heads, dim, dtype, runs, blocks=blocks + 1, seed=bs)


@pytest.mark.parametrize("bs,dim,heads,rows", [(16, 64, 4, 5000), (128, 64, 2, 2100), (32, 128, 8, 1500)])
def test_thousands_of_single_rows(bs, dim, heads, rows):
    rng = np.random.default_rng(rows)
    assert span(rows, heads) > 3
    runs = [((int(b),), int(rng.integers(0, bs)), 1) for b in rng.permutation(rows)]
    G.check_append(bs, heads, dim, "bf16", runs, blocks=rows, seed=1)


@pytest.mark.parametrize("bs", [16, 128])
def test_runs_at_every_place_of_a_span(bs):
    """Blocks filled from one row on, so that runs begin at every lane and cross the spans' ends and the 64 rows looked at."""
    firsts = [0 if b % 3 else 1 + b % (bs - 1) for b in range(1500 // bs * 4)]
    runs = [((b,), f, 1 + (b * 7) % min(bs // 2, bs - f)) for b, f in enumerate(firsts)]
    rows = sum(r[2] for r in runs)
    assert span(rows, 16) > 8
    G.check_append(bs, 16, 64, "f16", runs, blocks=len(runs) + 1)


def test_rows_left_out_within_a_span():
    """Slots of no block among and within runs: the rows after one begin a run of their own."""
    t = G.T()
    bs, heads, dim, n = 32, 16, 64, 3000
    rng = np.random.default_rng(4)
    slots = np.arange(n)                        # blocks in order, then some rows taken out of them
    out = rng.random(n) < 0.15
    for b in range(0, n, bs):                   # what is left of a block is its last tokens' run
        lost = np.flatnonzero(out[b:b + bs])
        if len(lost):
            out[b:b + lost[-1] + 1] = True
    slots = np.where(out, rng.choice([-1, -5, 10 ** 8, (n + bs) // bs * bs + 3], n), slots)
    assert span(n, heads) == 16 and 0.3 < out.mean() < 0.95
    c, kq, vq, ks, vs = G.new_cache((n + bs - 1) // bs, bs, heads, dim, 4)
    x, xv = G.dev(rng.normal(0, 1, (n, heads, dim)), "bf16")
    c.append(x, x.flip(0), G.i32(slots))
    for codes, scale, q0, s0, rows, last in ((c.k, c.k_scale, kq, ks, xv, False), (c.v, c.v_scale, vq, vs, xv[::-1], True)):
        q, s = G.R.append(q0, s0, rows, slots, bs)
        got = codes.cpu().numpy().astype(np.float64) - 128
        got = np.swapaxes(got, 2, 3) if last else got
        assert (G.f64(scale) == s).all() and (got == q).all()
    assert t.isfinite(c.k_scale).all()

"""Arguments of other ranks and sizes than the operators take raise the
package's error; tensors without rows are taken whatever their strides."""
import numpy as np
import pytest

import test_gpu_compute as G

pytestmark = pytest.mark.gpu


def test_other_ranks_and_sizes():
    t, k, H = G.T(), G.K(), __import__("haagenti_amd")
    half = lambda *s: t.zeros(*s, dtype=t.float16, device="cuda")  # noqa: E731
    one = G.i32(3).reshape(())
    c = G.new_cache(3, 16, 2, 64, 0)[0]
    plan = dict(lens=G.i32([1]), new=G.i32([1]), table=G.i32([[0]]), ring=G.i32([1, 2]), state=G.i32([0, 2]), block_size=16,
                tokens=3)
    att = dict(q=half(2, 4, 64), table=G.i32([[0, 1]]), start=G.i32([0, 2]), kv_len=G.i32([2]))
    bad = [
        lambda: k.linear(G.ctx(), half(4, 64), half(())),
        lambda: k.linear(G.ctx(), half(4, 64), half(64)),
        lambda: k.linear(G.ctx(), half(4, 64), half(1, 32, 64)),
        lambda: k.linear(G.ctx(), half(64), half(32, 64)),
        lambda: k.linear(G.ctx(), half(()), half(32, 64)),
        lambda: k.linear(G.ctx(), half(0, 1 << 33), half(0, 1 << 33)),
        lambda: k.linear(G.ctx(), half(4, 64), half(32, 64), bias=half(1, 32)),
        lambda: k.Int4Weight(t.zeros(64, dtype=t.uint8, device="cuda"), -1, 64),
        lambda: k.Int4Weight(t.zeros(64, dtype=t.uint8, device="cuda"), 1, -64),
        *[lambda a=a: k.kv_plan(G.ctx(), **{**plan, **a}) for a in (
            dict(lens=one, new=one), dict(new=one), dict(table=G.i32([0])), dict(state=one), dict(tokens=-1),
            dict(tokens=1 << 31), dict(tokens=1 << 40), dict(block_size=-16), dict(block_size=1 << 40))],
        lambda: k.KvCache(G.ctx(), c.k[0], c.v, c.k_scale, c.v_scale),
        lambda: k.KvCache(G.ctx(), c.k, c.v[0], c.k_scale, c.v_scale),
        lambda: c.append(half(()), half(()), one),
        lambda: c.append(half(2, 2, 64), half(2, 2, 64), one),
        lambda: c.append(half(2, 128), half(2, 128), G.i32([0, 1])),
        *[lambda a=a: c.attention(**{**att, **a}) for a in (
            dict(q=half(())), dict(kv_len=one), dict(start=one), dict(table=G.i32([0, 1])), dict(max_q=-1),
            dict(max_kv=1 << 40), dict(out=half(2, 256)))],
    ]
    for i, call in enumerate(bad):
        with pytest.raises(H.HaagentiError) as e:
            call()
        assert e.value.code == H.INVALID_ARGUMENT, i


def test_no_rows_from_numpy():
    t, k = G.T(), G.K()
    none = lambda *s: t.from_numpy(np.zeros(s, np.float16)).cuda()  # noqa: E731  (strides of 0)
    ints = lambda *s: t.from_numpy(np.zeros(s, np.int32)).cuda()  # noqa: E731
    w = t.zeros(32, 64, dtype=t.float16, device="cuda")
    assert k.linear(G.ctx(), none(0, 64), w, residual=none(0, 32)).shape == (0, 32)
    c = G.new_cache(3, 16, 2, 64, 0)[0]
    before = c.k.clone()
    c.append(none(0, 2, 64), none(0, 2, 64), ints(0))
    assert t.equal(c.k, before)
    assert c.attention(none(0, 4, 64), ints(0, 5), ints(1), ints(0)).shape == (0, 4, 64)
    assert [x.shape[0] for x in c.read(ints(0))] == [0, 0]
    p = k.kv_plan(G.ctx(), ints(0), ints(0), ints(0, 4), G.i32([3, 4]), G.i32([1, 1]), 16, 2)
    assert p.slots.cpu().tolist() == [-1, -1] and p.state.cpu().tolist() == [1, 1]

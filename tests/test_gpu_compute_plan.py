"""hh_kv_plan's lengths updated in place."""
import numpy as np
import pytest

import compute_ref as R
import test_gpu_compute as G

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 5, 1024, 5000])
def test_lengths_in_place(n):
    t, k = G.T(), G.K()
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 300, n)
    new = np.where(rng.random(n) < 0.1, -1, rng.integers(0, 40, n))
    bs, width = 16, 24
    held = (lens + bs - 1) // bs
    ids = rng.permutation(int(held.sum()) + 4 * n)
    table = np.full((n, width), -1, np.int64)
    at = 0
    for r in range(n):
        table[r, :held[r]] = ids[at:at + held[r]]
        at += held[r]
    ring, state = np.concatenate([ids[at:], ids[:at] * 0 - 5]), (0, len(ids) - at)
    tokens = int(np.maximum(new, 0).sum()) + 3
    want = R.plan(lens, new, table, ring, state, bs, tokens)
    d = dict(lens=G.i32(lens), new=G.i32(new), table=G.i32(table), ring=G.i32(ring), state=G.i32(state))
    out = {m: t.empty(size, dtype=t.int32, device="cuda") for m, size in (("start", n + 1), ("slots", tokens), ("after", 2))}
    # the lengths held take the old ones' place, the statuses the new rows'
    rc = k._plan(G.ctx().handle, k._PLAN.pack(
        d["lens"].data_ptr(), d["new"].data_ptr(), d["table"].data_ptr(), d["ring"].data_ptr(), d["state"].data_ptr(),
        out["start"].data_ptr(), d["lens"].data_ptr(), out["slots"].data_ptr(), d["new"].data_ptr(), out["after"].data_ptr(),
        width, n, width, len(ring), bs, tokens), t.cuda.current_stream().cuda_stream)
    assert rc == 0
    got = dict(start=out["start"], kv_len=d["lens"], slots=out["slots"], status=d["new"], table=d["table"], ring=d["ring"],
               state=out["after"])
    for key, v in got.items():
        assert (v.cpu().numpy() == np.asarray(want[key])).all(), key


@pytest.mark.parametrize("bs", [16, 32, 64, 128])
def test_ids_whose_slots_pass_31_bits(bs):
    k = G.K()
    last = (1 << 31) // bs - 1
    ids = [last, last + 1, (1 << 31) - 1, -1, -(1 << 31), (1 << 32) // bs]
    want = [last * bs + 3] + [-1] * 5
    # ids in the table, then from the ring
    table = np.full((6, 2), 7)
    table[:, 0] = ids
    p = k.kv_plan(G.ctx(), G.i32([3] * 6), G.i32([1] * 6), G.i32(table), G.i32([0]), G.i32([0, 0]), bs, 6)
    assert p.slots.cpu().tolist() == want
    p = k.kv_plan(G.ctx(), G.i32([bs] * 6), G.i32([1] * 6), G.i32(np.zeros((6, 2))), G.i32(ids), G.i32([0, 6]), bs, 6)
    assert p.slots.cpu().tolist() == [x - 3 if x >= 0 else x for x in want] and not p.status.any()

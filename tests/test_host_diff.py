"""hh_kv_diff_attention's C entry on a stand-in HIP runtime (no GPU): what it
refuses before anything is launched, and what it launches."""
from test_host_errors import host  # noqa: F401  (the fixture)

SETUP = """
import haagenti_amd.compute as K
buf = np.zeros(1 << 16, np.uint8)
at = (buf.ctypes.data + 255) & ~255
nan = float("nan")
def cache(blocks=4, block=16, heads=2, dim=64, k=at):
    return K._CACHE.pack(k, at, at, at, blocks, block, heads, dim)
def diff(c=None, requests=2, tokens=2, heads=4, width=4, max_q=1, max_kv=64, dtype=2, q=at, stride=None, lam=at, w=at, eps=1e-5,
         gain=1.0, ts=None):
    args = K._ATTENTION.pack(q, at, at, at, at, heads * 64, 64, heads * 64 if ts is None else ts, 64,
                             width if stride is None else stride, requests, tokens, heads, width, max_q, max_kv, 0.125, dtype)
    return K._diff_attention(ctx.handle, cache() if c is None else c, args, K._DIFF.pack(lam, w, eps, gain), None)
def nothing():
    assert not launches("launch"), calls()
hip.host_hip_fail(b"", 0)
"""

REFUSALS = [
    ("diff(heads=3)", 7), ("diff(dtype=0)", 5), ("diff(q=0)", 7), ("diff(q=at + 1)", 7), ("diff(stride=2)", 7),
    ("diff(requests=65537)", 7), ("diff(lam=0)", 7), ("diff(lam=at + 2)", 7), ("diff(w=at + 1)", 7), ("diff(eps=-1.0)", 7),
    ("diff(eps=nan)", 7), ("diff(ts=63)", 7), ("diff(cache(block=8))", 5), ("diff(cache(dim=80))", 5), ("diff(cache(k=at + 8))", 7),
    ("diff(max_kv=1 << 31, width=1 << 28)", 5), ("diff(tokens=0, lam=0)", 0),
]


def test_refused_before_any_launch(host):  # noqa: F811
    host(SETUP + "".join(f"assert {call} == {code}, {call!r}\nnothing()\n" for call, code in REFUSALS))


def test_launches(host):  # noqa: F811
    host(SETUP + """
import ctypes as C
grid = (C.c_uint * 6)()
assert diff(w=0) == 0 and [("diff_step" in x) for x in calls()] == [True], calls()
hip.host_hip_fail(b"", 0)
assert diff(requests=0) == 0 and launches("diff_zero") and len(launches("launch")) == 1
hip.host_hip_fail(b"", 0)          # two rows of 2 heads to a cache head: pairs of columns for the step kernel
assert diff(max_kv=60000, width=4000, max_q=2) == 0
assert launches("diff_step") and launches("diff_join") and not launches("diff_tile"), calls()
assert hip.host_hip_shape(b"diff_join", grid) and list(grid)[:2] == [2, 2 * 4]
hip.host_hip_fail(b"", 0)          # 300 rows: 600 pairs, 128 to a workgroup's 8 waves
assert diff(max_q=300, tokens=600) == 0 and launches("diff_tile")
assert hip.host_hip_shape(b"diff_tile", grid) and list(grid)[:2] == [2 * 5, 2], list(grid)
for kernel in (b"diff_step", b"diff_tile"):
    hip.host_hip_fail(kernel, 1)
    assert diff(max_q=300, tokens=600) == 10
    hip.host_hip_fail(b"", 0)
    assert diff(max_q=300, tokens=600) == 0
ctx = H.HipContext(0)
hip.host_hip_fail(b"malloc", 1)
assert diff(max_kv=60000, width=4000) == 8
nothing()
hip.host_hip_fail(b"", 0)
assert diff(max_kv=60000, width=4000) == 0
""")

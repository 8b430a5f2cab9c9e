"""The decoder-layer operators' C entries on a stand-in HIP runtime (no GPU):
what they refuse before anything is launched, what a failing launch or
allocation returns, and which kernels a shape launches."""
from test_host_errors import host  # noqa: F401  (the fixture)

SETUP = """
import haagenti_amd.compute as K
buf = np.zeros(1 << 20, np.uint8)
at = (buf.ctypes.data + 255) & ~255
def linear(m=4, n=32, k=64, dtype=2, w_dtype=2, y_dtype=2, act=0, x=at, w=at, b=0, c=0, d=0, y=at, xs=None, ws=None, cs=0,
           ds=0, ys=None, wb=0):
    args = K._LINEAR.pack(x, w, b, c, d, y, k if xs is None else xs, k if ws is None else ws, cs, ds, n if ys is None else ys,
                          wb, m, n, k, dtype, w_dtype, y_dtype, act)
    return K._linear(ctx.handle, args, None)
def plan(requests=2, width=4, cap=8, block=16, tokens=4, stride=None, state=at, after=at + 64, table=at):
    args = K._PLAN.pack(at, at, table, at, state, at, at, at, at, after, width if stride is None else stride, requests,
                        width, cap, block, tokens)
    return K._plan(ctx.handle, args, None)
def cache(blocks=4, block=16, heads=2, dim=64, k=at):
    return K._CACHE.pack(k, at, at, at, blocks, block, heads, dim)
def append(c, rows=3, dtype=2, k=at, slots=at):
    return K._append(ctx.handle, c, k, at, dtype, 128, 64, 128, 64, slots, rows, None)
def attention(c, requests=2, tokens=2, heads=4, width=4, max_q=1, max_kv=64, dtype=2, q=at, stride=None):
    args = K._ATTENTION.pack(q, at, at, at, at, heads * 64, 64, heads * 64, 64, width if stride is None else stride, requests,
                             tokens, heads, width, max_q, max_kv, 0.125, dtype)
    return K._attention(ctx.handle, c, args, None)
def nothing():
    assert not launches("launch"), calls()
hip.host_hip_fail(b"", 0)
"""


REFUSALS = [
    ("linear(dtype=0)", 5), ("linear(w_dtype=1)", 5), ("linear(y_dtype=1)", 5), ("linear(act=9)", 5),
    ("linear(x=0)", 7), ("linear(w=0)", 7), ("linear(y=0)", 7), ("linear(x=at + 1)", 7), ("linear(y=at + 2, y_dtype=0)", 7),
    ("linear(xs=63)", 7), ("linear(ws=63)", 7), ("linear(ys=31)", 7), ("linear(c=at, cs=31)", 7), ("linear(d=at, ds=31)", 7),
    ("linear(w_dtype=16, wb=1151)", 3), ("linear(m=1 << 21)", 7), ("linear(n=1 << 26)", 7),
    ("linear(m=0)", 0), ("linear(n=0)", 0),
    ("plan(block=48)", 5), ("plan(requests=65537)", 5), ("plan(stride=3)", 7), ("plan(after=at)", 7),
    ("plan(after=at + 4)", 7), ("plan(table=0)", 7), ("plan(state=0)", 7),
    ("append(cache(block=8))", 5), ("append(cache(dim=80))", 5), ("append(cache(blocks=0))", 7),
    ("append(cache(blocks=1 << 27))", 7), ("append(cache(k=at + 8))", 7), ("append(cache(), dtype=0)", 5),
    ("append(cache(), k=0)", 7), ("append(cache(), slots=0)", 7), ("append(cache(), rows=0)", 0),
    ("attention(cache(), heads=3)", 7), ("attention(cache(), dtype=0)", 5), ("attention(cache(), q=0)", 7),
    ("attention(cache(), stride=2)", 7), ("attention(cache(), requests=65537)", 7), ("attention(cache(), tokens=0)", 0),
]


def test_refused_before_any_launch(host):  # noqa: F811
    host(SETUP + "".join(f"assert {call} == {code}, {call!r}\nnothing()\n" for call, code in REFUSALS))


def test_a_failed_launch_is_reported_and_the_next_call_runs(host):  # noqa: F811
    host(SETUP + """
c = cache()
for call, kernel in ((lambda: linear(), b"linear_rows_kernel"), (lambda: linear(m=200), b"linear_large_kernel"),
                     (lambda: linear(m=200, k=63), b"linear_tile_kernel"), (plan, b"kv_plan_kernel"),
                     (lambda: append(c), b"kv_append_kernel"), (lambda: attention(c), b"attn_step_kernel")):
    hip.host_hip_fail(kernel, 1)
    assert call() == 10, kernel
    hip.host_hip_fail(b"", 0)
    assert call() == 0, kernel
""")


def test_a_failed_allocation_is_reported(host):  # noqa: F811
    host(SETUP + """
hip.host_hip_fail(b"malloc", 1)
assert attention(cache(), max_kv=60000, width=4000) == 8
hip.host_hip_fail(b"", 0)
assert attention(cache(), max_kv=60000, width=4000) == 0
assert len(launches("attn_step")) == 1 and len(launches("attn_join")) == 1
""")


KERNELS = [
    ("m=1", "linear_rows_kernel"), ("m=32", "linear_rows_kernel"), ("m=33", "linear_large_kernel"),
    ("m=33, k=60", "linear_rows_kernel"), ("m=65, k=60", "linear_tile_kernel"), ("m=33, xs=65", "linear_rows_kernel"),
    ("m=64, w_dtype=16, wb=4096", "linear_rows_kernel"), ("m=65, w_dtype=16, wb=4096", "linear_tile_kernel"),
    ("m=1, k=33, w_dtype=16, wb=4096", "linear_tile_kernel"),
]


def test_kernel_of_a_shape(host):  # noqa: F811
    host(SETUP + "".join(f"hip.host_hip_fail(b'', 0)\nassert linear({args}) == 0\nassert launches({kernel!r}), ({args!r}, calls())\n"
                         for args, kernel in KERNELS))


def test_short_requests_are_not_split(host):  # noqa: F811
    host(SETUP + """
assert attention(cache(), max_kv=500, width=40) == 0
assert len(launches("launch")) == 1, calls()
assert attention(cache(), max_kv=500, width=40, max_q=40, tokens=80) == 0
assert len(launches("attn_tile")) == 1
""")

"""The gated products' C entries on a stand-in HIP runtime (no GPU): what they
refuse before anything is launched, which kernels a shape launches, and what a
failing launch or allocation returns."""
from test_host_errors import host  # noqa: F401  (the fixture)

SETUP = """
import haagenti_amd.compute as K
buf = np.zeros(1 << 20, np.uint8)
at = (buf.ctypes.data + 255) & ~255
def args(m=4, n=32, k=64, dtype=2, w_dtype=None, y_dtype=None, act=4, x=at, gate=at, up=at, gb=0, ub=0, y=at, saved=0, xs=None,
         gs=None, us=None, ys=None, gbytes=1 << 40, ubytes=1 << 40):
    return K._GATED.pack(x, gate, up, gb, ub, y, saved, k if xs is None else xs, k if gs is None else gs, k if us is None else us,
                         n if ys is None else ys, gbytes, ubytes, m, n, k, dtype, dtype if w_dtype is None else w_dtype,
                         dtype if y_dtype is None else y_dtype, act)
def gated(**a):
    return K._gated(ctx.handle, args(**a), None)
def nothing():
    assert not launches("launch"), calls()
hip.host_hip_fail(b"", 0)
"""

REFUSALS = [
    ("gated(dtype=0)", 5), ("gated(w_dtype=1)", 5), ("gated(y_dtype=1)", 5), ("gated(act=5)", 5), ("gated(act=-1)", 5),
    ("gated(x=0)", 7), ("gated(gate=0)", 7), ("gated(up=0)", 7), ("gated(y=0)", 7), ("gated(x=at + 1)", 7),
    ("gated(gate=at + 1)", 7), ("gated(up=at + 1)", 7), ("gated(gb=at + 1)", 7), ("gated(ub=at + 1)", 7),
    ("gated(y=at + 1)", 7), ("gated(y=at + 2, y_dtype=0)", 7), ("gated(saved=at + 8)", 7), ("gated(xs=63)", 7),
    ("gated(gs=63)", 7), ("gated(us=63)", 7), ("gated(ys=31)", 7), ("gated(m=1 << 21)", 7), ("gated(n=1 << 25)", 7),
    ("gated(k=1 << 31)", 7), ("gated(w_dtype=16, gbytes=1151)", 3), ("gated(w_dtype=16, ubytes=1151)", 3),
    ("gated(m=0)", 0), ("gated(n=0)", 0),
]


def test_refused_before_any_launch(host):  # noqa: F811
    host(SETUP + "".join(f"assert {call} == {code}, {call!r}\nnothing()\n" for call, code in REFUSALS))


def test_kernels_and_splits_of_the_shapes(host):  # noqa: F811
    host(SETUP + """
import ctypes, gated_shapes
for m, n, k, weight, name, splits, dim in gated_shapes.cases():
    for y in (2, 0):
        kernel = (name % (2, y)).encode()
        hip.host_hip_fail(b"", 0)
        assert gated(m=m, n=n, k=k, w_dtype=16 if weight == "int4" else 2, y_dtype=y) == 0
        assert launches(kernel.decode()), (m, n, k, weight, kernel, calls())
        shape = (ctypes.c_uint * 6)()
        assert hip.host_hip_shape(kernel, shape)
        assert shape[dim] == splits or name.startswith("gated_rows"), (m, n, k, weight, list(shape), splits)
        assert len(launches("gated_join")) == (splits > 1), calls()
""")


def test_a_failed_launch_or_allocation_is_reported_and_the_next_call_runs(host):  # noqa: F811
    host(SETUP + """
for call, kernel in ((gated, b"gated_rows_kernel"), (lambda: gated(m=200), b"gated_large_kernel"),
                     (lambda: gated(m=200, k=63), b"gated_tile_kernel"), (lambda: gated(m=34, n=20, k=2240), b"gated_join_kernel")):
    hip.host_hip_fail(kernel, 1)
    assert call() == 10, kernel
    hip.host_hip_fail(b"", 0)
    assert call() == 0, kernel
ctx = H.HipContext(0)
hip.host_hip_fail(b"malloc", 1)
assert gated(m=34, n=20, k=2240) == 8
nothing()
hip.host_hip_fail(b"", 0)
assert gated(m=34, n=20, k=2240) == 0
""")

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
def back(dy=at, dx=at, dg=at, du=at, gb=at, ub=at, ds=None, dxs=None, dgs=None, dus=None, n=32, k=64, saved=at, **a):
    grads = K._GATED_GRADS.pack(dy, dx, dg, du, gb, ub, n if ds is None else ds, k if dxs is None else dxs,
                                k if dgs is None else dgs, k if dus is None else dus)
    return K._gated_backward(ctx.handle, args(n=n, k=k, saved=saved, **a), grads, None)
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
    ("back(dtype=0)", 5), ("back(w_dtype=16)", 5), ("back(act=7)", 5), ("back(x=0)", 7), ("back(gate=0)", 7), ("back(up=0)", 7),
    ("back(dy=0)", 7), ("back(saved=0)", 7), ("back(dy=at + 1)", 7), ("back(dx=at + 1)", 7), ("back(dg=at + 1)", 7),
    ("back(du=at + 1)", 7), ("back(gb=at + 2)", 7), ("back(ub=at + 2)", 7), ("back(saved=at + 8)", 7), ("back(dg=0)", 7),
    ("back(du=0)", 7), ("back(ds=31)", 7), ("back(dxs=63)", 7), ("back(dgs=63)", 7), ("back(dus=63)", 7), ("back(xs=63)", 7),
    ("back(gs=63)", 7), ("back(us=63)", 7), ("back(m=1 << 21)", 7), ("back(n=1 << 25)", 7),
    ("back(m=(1 << 21) - 1, n=(1 << 25) - 1)", 5), ("back(dx=0, dg=0, du=0, gb=0, ub=0)", 0), ("back(m=0, dg=0, du=0, gb=0, ub=0)", 0),
    ("back(n=0, dx=0)", 0), ("back(k=0, gb=0, ub=0)", 0),
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


def test_whole_rounds_and_the_rest(host):  # noqa: F811
    host(SETUP + """
import ctypes, gated_shapes
for m, n, k, (tn, tm), cols, (rn, rm) in gated_shapes.TWO:
    for y in (2, 0):
        hip.host_hip_fail(b"", 0)
        assert gated(m=m, n=n, k=k, y_dtype=y, saved=at) == 0
        c = launches("launch")
        assert len(c) == 2, c
        for line, (a, b), first, end in ((c[0], (tn, tm), 0, cols), (c[1], (rn, rm), cols, n)):
            kernel = f"gated_large_kernelILi2ELi{y}ELi{a}ELi{b}E"
            assert kernel in line, (m, n, k, c)
            shape = (ctypes.c_uint * 6)()
            assert hip.host_hip_shape(kernel.encode(), shape)
            assert list(shape[:2]) == [-(-2 * (end - first) // a) * -(-m // b), 1], (m, n, k, list(shape))
        hip.host_hip_fail(b"launch", 2)
        assert gated(m=m, n=n, k=k, y_dtype=y) != 0
""")


def test_kernels_of_the_gradients(host):  # noqa: F811
    host(SETUP + """
import gated_back_shapes as S
reached, split = set(), set()
for m, n, k in S.SHAPES:
    hip.host_hip_fail(b"", 0)
    assert back(m=m, n=n, k=k) == 0
    c = launches("launch")
    assert "gated_slope_kernel" in c[0] and "gated_bias_kernel" in c[1] and len(launches("back")) == len(c) - 2, c
    for i, name in enumerate(c):
        for kernel in S.KERNELS:
            if kernel in name:
                reached.add(kernel)
                if i + 1 < len(c) and "join" in c[i + 1]:
                    split.add(kernel)
                else:
                    split.add(kernel + " whole")
missing = [(k, e) for k in S.KERNELS for e in ("", " whole") if k + e not in split]
assert reached == set(S.KERNELS) and not missing, missing
hip.host_hip_fail(b"", 0)
assert back(gb=0, ub=0) == 0 and not launches("bias"), calls()
hip.host_hip_fail(b"", 0)
assert back(dx=0) == 0 and len(launches("gated_back")) == 1 and launches("ELb1E"), calls()
hip.host_hip_fail(b"", 0)
assert back(dg=0, du=0) == 0 and len(launches("gated_back")) == 1 and launches("ELb0E"), calls()
hip.host_hip_fail(b"", 0)
assert back(m=0) == 0 and len(launches("gated_zero")) == 4 == len(launches("launch")), calls()
hip.host_hip_fail(b"", 0)
assert back(x=at + 2) == 0 and launches("gated_back_any_kernelILi2ELb1E") and launches("gated_back_kernelILi2ELb0E"), calls()
hip.host_hip_fail(b"", 0)
assert back(us=65) == 0 and launches("gated_back_any_kernelILi2ELb0E") and launches("gated_back_kernelILi2ELb1E"), calls()
""")


def test_a_failed_launch_or_allocation_is_reported_and_the_next_call_runs(host):  # noqa: F811
    host(SETUP + """
for call, kernel in ((gated, b"gated_rows_kernel"), (lambda: gated(m=200), b"gated_large_kernel"),
                     (lambda: gated(m=200, k=63), b"gated_tile_kernel"), (lambda: gated(m=34, n=20, k=2240), b"gated_join_kernel")):
    hip.host_hip_fail(kernel, 1)
    assert call() == 10, kernel
    hip.host_hip_fail(b"", 0)
    assert call() == 0, kernel
for kernel in (b"gated_slope_kernel", b"gated_bias_kernel", b"gated_back_kernelILi2ELb0E", b"gated_back_kernelILi2ELb1E",
               b"gated_back_join_kernel"):
    hip.host_hip_fail(kernel, 1)
    assert back(m=645, n=321, k=16) == 10, kernel
    assert launches("failed") == launches("launch")[-1:], calls()
    hip.host_hip_fail(b"", 0)
    assert back(m=645, n=321, k=16) == 0, kernel
ctx = H.HipContext(0)
hip.host_hip_fail(b"malloc", 1)
assert gated(m=34, n=20, k=2240) == 8
nothing()
hip.host_hip_fail(b"malloc", 1)
assert back(m=645, n=3210, k=16) == 8
nothing()
hip.host_hip_fail(b"", 0)
assert gated(m=34, n=20, k=2240) == 0 and back(m=645, n=3210, k=16) == 0
""")

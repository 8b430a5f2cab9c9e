"""The norms' and rotary positions' C entries on a stand-in HIP runtime (no
GPU): what they refuse before anything is launched, what a failing launch or
allocation returns, and which kernels a shape launches."""
from test_host_errors import host  # noqa: F401  (the fixture)

SETUP = """
import haagenti_amd.compute as K
buf = np.zeros(1 << 16, np.uint8)
at = (buf.ctypes.data + 255) & ~255
nan = float("nan")
def norm_args(rows=4, n=32, dtype=2, wt=None, kind=0, x=at, y=at + 4096, w=at, b=at, xs=None, ys=None, eps=1e-5):
    return K._NORM.pack(x, w, b, y, n if xs is None else xs, n if ys is None else ys, rows, n, eps, dtype,
                        dtype if wt is None else wt, kind)
def norm(**a):
    return K._norm(ctx.handle, norm_args(**a), None)
def back(dy=at, add=0, dw=at, db=at, ds=None, adds=0, n=32, **a):
    grads = K._NORM_GRADS.pack(dy, add, dw, db, n if ds is None else ds, adds)
    return K._norm_backward(ctx.handle, norm_args(n=n, **a), grads, None)
def rotary(tokens=3, heads=2, dim=64, sections=(32,), x=at, y=at + 8192, pos=at, freq=at, xt=None, xh=None, yt=None, yh=None,
           ps=0, inter=0, inv=0, dtype=2):
    s = list(sections) + [0] * (4 - len(sections))
    return K._rotary(ctx.handle, K._ROTARY.pack(x, y, pos, freq, heads * dim if xt is None else xt, dim if xh is None else xh,
                                                heads * dim if yt is None else yt, dim if yh is None else yh, ps, tokens, heads,
                                                dim, min(len(sections), 9), *s[:4], inter, inv, dtype), None)
def nothing():
    assert not launches("launch"), calls()
hip.host_hip_fail(b"", 0)
"""

REFUSALS = [
    ("norm(dtype=3)", 5), ("norm(wt=1)", 5), ("norm(kind=2)", 5), ("norm(x=0)", 7), ("norm(y=0)", 7), ("norm(x=at + 1)", 7),
    ("norm(y=at + 1)", 7), ("norm(w=at + 1)", 7), ("norm(b=at + 2, wt=0)", 7), ("norm(xs=31)", 7), ("norm(ys=31)", 7),
    ("norm(eps=-1e-9)", 7), ("norm(eps=nan)", 7), ("norm(rows=1 << 31)", 7), ("norm(n=32769)", 5), ("norm(n=16385, dtype=0)", 5),
    ("norm(rows=0)", 0), ("norm(n=0)", 0), ("norm(rows=0, x=0, y=0)", 0),
    ("back(dtype=3)", 5), ("back(dy=0)", 7), ("back(dy=at + 1)", 7), ("back(add=at + 1, adds=32)", 7), ("back(dw=at + 2)", 7),
    ("back(db=at + 2)", 7), ("back(ds=31)", 7), ("back(add=at, adds=31)", 7), ("back(eps=-1.0)", 7), ("back(n=32769)", 5),
    ("back(rows=0, dw=0, db=0)", 0), ("back(n=0)", 0),
    ("rotary(dtype=3)", 5), ("rotary(sections=())", 5), ("rotary(sections=(1,) * 5)", 5), ("rotary(sections=(513,), dim=1200)", 5),
    ("rotary(sections=(33,))", 7), ("rotary(sections=(0xffffffff, 2))", 5), ("rotary(x=0)", 7), ("rotary(y=0)", 7),
    ("rotary(pos=0)", 7), ("rotary(freq=0)", 7), ("rotary(x=at + 1)", 7), ("rotary(y=at + 1)", 7), ("rotary(y=at + 2, dtype=0)", 7),
    ("rotary(pos=at + 2)", 7), ("rotary(freq=at + 2)", 7), ("rotary(heads=65536)", 7), ("rotary(tokens=1 << 31)", 7),
    ("rotary(yt=127)", 7), ("rotary(yh=63)", 7), ("rotary(y=at, yt=256)", 7), ("rotary(dim=65537)", 5),
    ("rotary(tokens=0)", 0), ("rotary(heads=0)", 0), ("rotary(dim=0, sections=(0,))", 0),
    ("rotary(sections=(0,), pos=0, freq=0, y=at)", 0),
]


def test_refused_before_any_launch(host):  # noqa: F811
    host(SETUP + "".join(f"assert {call} == {code}, {call!r}\nnothing()\n" for call, code in REFUSALS))


def test_a_failed_launch_or_allocation_is_reported_and_the_next_call_runs(host):  # noqa: F811
    host(SETUP + """
for call, kernel in ((norm, b"norm_kernel"), (back, b"norm_backward_kernel"), (back, b"norm_join_kernel"),
                     (lambda: back(rows=0), b"norm_zero_kernel"), (rotary, b"rotary_kernel")):
    hip.host_hip_fail(kernel, 1)
    assert call() == 10, kernel
    hip.host_hip_fail(b"", 0)
    assert call() == 0, kernel
ctx = H.HipContext(0)
hip.host_hip_fail(b"malloc", 1)
assert back() == 8
nothing()
hip.host_hip_fail(b"", 0)
assert back() == 0
hip.host_hip_fail(b"", 0)
assert back(dw=0, db=0) == 0 and len(launches("launch")) == 1, calls()
""")


# XT, W, G, C of the kernel's template: waves to a row, rows to a workgroup, pieces to a lane
KERNELS = [
    ("n=1", "norm_kernelILi2ELi1ELi4ELi1E"), ("n=512", "norm_kernelILi2ELi1ELi4ELi1E"), ("n=513", "norm_kernelILi2ELi1ELi4ELi2E"),
    ("n=1024", "norm_kernelILi2ELi1ELi4ELi2E"), ("n=1025", "norm_kernelILi2ELi4ELi1ELi1E"),
    ("n=2049", "norm_kernelILi2ELi4ELi1ELi2E"), ("n=4096", "norm_kernelILi2ELi4ELi1ELi2E"),
    ("n=4097", "norm_kernelILi2ELi8ELi1ELi2E"), ("n=8193", "norm_kernelILi2ELi16ELi1ELi2E"),
    ("n=16385", "norm_kernelILi2ELi16ELi1ELi4E"), ("n=512, dtype=0", "norm_kernelILi0ELi1ELi4ELi2E"),
]


def test_kernel_of_a_shape(host):  # noqa: F811
    host(SETUP + "".join(f"hip.host_hip_fail(b'', 0)\nassert norm({a}) == 0\nassert launches({k!r}), ({a!r}, calls())\n"
                         for a, k in KERNELS))

"""Which kernel and how many splits of k a product's shape takes, on a
stand-in HIP runtime (no GPU) of 256 CUs: the shapes that the GPU tests rely
on to reach every kernel, and that they do reach every one."""
import os
import re
import subprocess

from compute_shapes import cases
from test_host_compute import SETUP
from test_host_errors import host  # noqa: F401  (the fixture)


def test_kernels_of_shapes(host):  # noqa: F811
    host(SETUP + f"""
import ctypes as C
from compute_shapes import cases
grid = (C.c_uint * 6)()
for m, n, k, weight, kernel, splits, dim in cases():
    for dtype, y in ((2, 2), (1, 0)):
        hip.host_hip_fail(b"", 0)
        int4 = weight == "int4"
        assert linear(m=m, n=n, k=k, dtype=dtype, w_dtype=16 if int4 else dtype, y_dtype=y, wb=n * k if int4 else 0) == 0
        assert hip.host_hip_shape((kernel % (dtype, y)).encode(), grid), (m, n, k, weight, kernel, calls())
        assert grid[dim] == splits, (m, n, k, weight, list(grid))
        assert len(launches("linear_join")) == (splits > 1) and len(launches("launch")) == 1 + (splits > 1)
""")


def test_every_kernel_has_a_shape():
    lib = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "haagenti_amd", "libhaagenti_hip.so")
    names = subprocess.run(["nm", lib], capture_output=True, text=True, check=True).stdout
    built = set(re.findall(r"linear_(?:large|tile|rows)_kernelI(?:L[ib]\d+E)+", names))
    # of the types, the two that the shapes are run with
    built = {k for k in built if re.match(r"\w+I(Li2ELi2E|Li1ELi0E)", k)}
    want = {kernel % t for *_, kernel, _, _ in cases() for t in ((2, 2), (1, 0))}
    reached = {k for k in built if any(k.startswith(w) for w in want)}
    assert built and built == reached, sorted(built - reached)

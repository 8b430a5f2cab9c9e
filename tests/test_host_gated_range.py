"""What hh_gated_linear_backward launches for float16, whose dg and du are
scaled by their rows' and columns' largest, on a stand-in HIP runtime (no
GPU)."""
from test_host_errors import host  # noqa: F401  (the fixture)
from test_host_gated import SETUP


def test_launches(host):  # noqa: F811
    host(SETUP + """
def names(**a):
    hip.host_hip_fail(b"", 0)
    assert back(dtype=1, m=70, n=100, k=72, **a) == 0
    return ["tops" if "gated_slope_kernelILi1ELi1ELb1E" in c else "slope" if "gated_slope_kernelILi1ELi1ELb0E" in c else
            "bias" if "gated_bias_kernel" in c else "join" if "gated_tops_kernel" in c else
            "dx" if "ELb0E" in c and "back_kernel" in c else "dw" if "ELb1E" in c and "back_kernel" in c else c
            for c in launches("launch") if "back_join" not in c]
assert names() == ["tops", "join", "slope", "bias", "dx", "dw"], calls()
assert names(dx=0, gb=0, ub=0) == ["tops", "join", "slope", "dw"], calls()
assert names(dg=0, du=0, gb=0) == ["tops", "join", "slope", "bias", "dx"], calls()
assert names(dx=0, dg=0, du=0) == ["slope", "bias"], calls()
hip.host_hip_fail(b"", 0)
assert back(dtype=2, m=70, n=100, k=72) == 0 and not launches("gated_tops") and len(launches("slope")) == 1, calls()
""")


def test_a_failed_launch_is_reported_and_the_next_call_runs(host):  # noqa: F811
    host(SETUP + """
for kernel in (b"gated_tops_kernel", b"gated_slope_kernelILi1ELi1ELb1E", b"gated_slope_kernelILi1ELi1ELb0E"):
    hip.host_hip_fail(kernel, 1)
    assert back(dtype=1, m=70, n=100, k=72) == 10, kernel
    assert launches("failed") == launches("launch")[-1:], calls()
    hip.host_hip_fail(b"", 0)
    assert back(dtype=1, m=70, n=100, k=72) == 0, kernel
""")

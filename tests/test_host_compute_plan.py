"""hh_kv_plan with results laid over its inputs, which every part of the
launch reads: the inputs are set aside first.  On a stand-in HIP runtime (no
GPU)."""
from test_host_compute import SETUP
from test_host_errors import host  # noqa: F401  (the fixture)

MORE = SETUP + """
names = ["lens", "new", "table", "ring", "state", "start", "kv_len", "slots", "status", "after"]
size = dict(lens=3, new=3, table=12, ring=8, state=2, start=4, kv_len=3, slots=5, status=3, after=2)
apart = {n: at + 256 * i for i, n in enumerate(names)}
def call(**change):
    a = {**apart, **change}
    return K._plan(ctx.handle, K._PLAN.pack(*(a[n] for n in names), 4, 3, 4, 8, 16, 5), None)
"""


def test_inputs_under_results_are_set_aside(host):  # noqa: F811
    host(MORE + """
assert call() == 0 and len(launches("launch")) == 1
for i in ("lens", "new", "state"):
    for o in ("start", "kv_len", "slots", "status", "after"):
        for d in (0, 4 * size[i] - 4, 4 - 4 * size[o]):
            hip.host_hip_fail(b"", 0)
            if (i, o) == ("state", "after"):
                assert call(**{o: apart[i] + d}) == 7
                nothing()
                continue
            assert call(**{o: apart[i] + d}) == 0
            kernels = launches("launch")
            assert len(kernels) == 2 and "plan_inputs" in kernels[0] and "kv_plan" in kernels[1], (i, o, d, kernels)
        for d in (4 * size[i], -4 * size[o]):
            hip.host_hip_fail(b"", 0)
            assert call(**{o: apart[i] + d}) == 0 and len(launches("launch")) == 1, (i, o, d)
""")


def test_failures_of_setting_aside(host):  # noqa: F811
    host(MORE + """
for what, code in ((b"malloc", 8), (b"plan_inputs", 10)):
    hip.host_hip_fail(what, 1)
    assert call(kv_len=apart["lens"]) == code and not launches("kv_plan"), what
    hip.host_hip_fail(b"", 0)
    assert call(kv_len=apart["lens"]) == 0
""")


def test_no_requests_and_no_rows_overlap_nothing(host):  # noqa: F811
    host(SETUP + """
args = K._PLAN.pack(0, 0, 0, at, at, at + 64, 0, 0, 0, at + 128, 4, 0, 4, 8, 16, 0)
assert K._plan(ctx.handle, args, None) == 0
assert len(launches("launch")) == 1
""")

"""Where the decoder-layer operators keep their partial sums, on a stand-in
HIP runtime (no GPU): per stream, apart for captured calls, and what a
captured call has used is freed with the context only."""
from test_host_compute import SETUP
from test_host_errors import host  # noqa: F401  (the fixture)

MORE = SETUP + """
def on(stream, splits_of=60000, width=4000):
    args = K._ATTENTION.pack(at, at, at, at, at, 2048, 64, 2048, 64, width, 2, 2, 32, width, 1, splits_of, 0.125, 2)
    assert K._attention(ctx.handle, cache(), args, stream) == 0
def counts():
    out = tuple(len([c for c in calls() if c == w]) for w in ("malloc", "free"))
    hip.host_hip_fail(b"", 0)
    return out
"""


def test_each_stream_has_its_own(host):  # noqa: F811
    host(MORE + """
for stream in (None, 64, 128):
    on(stream)
    assert counts() == (1, 0)
for stream in (128, None, 64):
    on(stream)
    assert counts() == (0, 0)
ctx.close()
assert counts()[1] >= 3
""")


def test_what_a_captured_call_used_is_kept(host):  # noqa: F811
    host(MORE + """
on(64, 3000)
assert counts() == (1, 0)
hip.host_hip_capture(1)
on(64, 3000)                    # its own memory, though the stream's would do
assert calls().index("relaxed") < calls().index("malloc") < calls().index("global")
assert counts() == (1, 0)
hip.host_hip_capture(0)
for _ in range(2):
    on(64, 2000000, 1 << 17)    # more than before: the eager memory grows
assert counts() == (1, 1)
hip.host_hip_capture(1)
on(64, 3000)
assert counts() == (0, 0)
on(64, 2000000, 1 << 17)        # captured calls' memory grows: the old stays
assert counts() == (1, 0)
hip.host_hip_capture(0)
ctx.close()
assert counts()[1] >= 3
""")


def test_a_failed_allocation_leaves_the_next_call_working(host):  # noqa: F811
    host(MORE + """
on(64, 3000)
for captured in (0, 1):
    hip.host_hip_capture(captured)
    hip.host_hip_fail(b"malloc", 1)
    args = K._ATTENTION.pack(at, at, at, at, at, 2048, 64, 2048, 64, 1 << 17, 2, 2, 32, 1 << 17, 1, 2000000, 0.125, 2)
    assert K._attention(ctx.handle, cache(), args, 64) == 8
    assert not launches("launch") and len(launches("relaxed")) == len(launches("global")) == captured
    hip.host_hip_fail(b"", 0)
    on(64, 2000000, 1 << 17)
    assert len(launches("attn_step")) == 1
""")

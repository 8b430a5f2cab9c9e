"""hh_kv_attention's outputs whose rows would overlap, on a stand-in HIP
runtime (no GPU)."""
from test_host_compute import SETUP
from test_host_errors import host  # noqa: F401  (the fixture)


def test_overlapping_outputs_are_refused(host):  # noqa: F811
    host(SETUP + """
import itertools
def call(tokens, heads, ts, hs):
    args = K._ATTENTION.pack(at, at, at, at, at, 4096, 64, ts, hs, 4, 2, tokens, heads, 4, 1, 64, 0.125, 2)
    return K._attention(ctx.handle, cache(heads=1), args, None)
def meet(tokens, heads, ts, hs):
    starts = sorted(i * ts + j * hs for i in range(tokens) for j in range(heads))
    return any(b - a < 64 for a, b in zip(starts, starts[1:]))
strides = (0, 1, 63, 64, 65, 100, 127, 128, 129, 190, 191, 192, 193, 255, 256, 257, 320, 448, 511, 1000)
n = 0
for tokens, heads, ts, hs in itertools.product((1, 2, 3, 5, 17), (1, 2, 3, 7), strides, strides):
    want = 7 if meet(tokens, heads, ts, hs) else 0
    n += want == 7
    assert call(tokens, heads, ts, hs) == want, (tokens, heads, ts, hs)
assert 1000 < n < 7000, n
assert call(2, 2, 1 << 63, 64) == 0 and call(3, 2, 64, 1 << 63) == 0 and call(1 << 20, 32, 32 * 64, 64) == 0
assert call(1 << 20, 32, 64, 64 << 20) == 0 and call(1 << 20, 32, 64, (64 << 20) - 64) == 7
""")

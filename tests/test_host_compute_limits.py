"""The largest hh_kv_attention calls that one launch holds, on a stand-in HIP
runtime (no GPU)."""
import pytest

from test_host_compute import SETUP
from test_host_errors import host  # noqa: F401  (the fixture)


@pytest.mark.parametrize("dim,columns", [(64, 256), (128, 256), (192, 128), (256, 128)])
def test_launches_of_2_to_the_32_threads_are_refused(host, dim, columns):  # noqa: F811
    host(SETUP + f"""
def call(requests, rows, max_kv=64):
    args = K._ATTENTION.pack(at, at, at, at, at, {dim}, {dim}, {dim}, {dim}, 1 << 20, requests, 1 << 22, 1, 1 << 20, rows,
                             max_kv, 0.125, 2)
    return K._attention(ctx.handle, cache(heads=1, dim={dim}), args, None)
# a workgroup has 2 threads to a column: requests * tiles * 2 * columns < 2^32
for requests, tiles in ((65536, 65536 * 32768 // 65536 // {columns}), (4096, 16 * 32768 // {columns}), (8192, 8 * 32768 // {columns})):
    assert requests * tiles * 2 * {columns} == 1 << 32
    assert call(requests, tiles * {columns}) == 5 and call(requests, (tiles - 1) * {columns} + 1) == 5
    nothing()
    assert call(requests, (tiles - 1) * {columns}) == 0 and len(launches("attn_tile")) == 1
    hip.host_hip_fail(b"", 0)
# chunks of tokens never are that many
assert call(65536, 1, 1 << 30) == 0 and call(1, 1, 1 << 30) == 0
""")

"""The one-launch form of small calls of qraf_hip_group_attention_dev at its bounds: as many rows and groups as it
takes, prefixes and tails that begin and end inside tiles, and the first call beyond each bound."""
import numpy as np
import pytest

from tests import test_gpu_group_attention as calls

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [255, 256, 257])
@calls.KINDS
def test_rows_and_groups(hip, kv, n):
    """As many groups as rows: of one row, of two, of none, contexts up to 256."""
    rng = np.random.default_rng(n)
    groups = []
    for i in range(n // 3):
        p = int(rng.integers(0, 200))
        groups += [(p, [int(c) for c in rng.integers(0, 257, 2)]), (p, []), (int(rng.integers(0, 257)), [1 + i % 256])]
    groups += [(5, [9])] * (n - 3 * (n // 3))
    c = calls.Cache(rng, groups, 1, 64, 16, kv)
    assert c.n == n and len(c.prefix) == n
    q = calls.queries(rng, n, 2, 64)
    calls.check(c, calls.Call(hip, c, q, 2).run(), q, 2)


@pytest.mark.parametrize("longest", [511, 512, 513, 768, 769, 1024, 1025])
@calls.KINDS
def test_lengths(hip, kv, longest):
    rng = np.random.default_rng(longest)
    groups = [(longest - 7, [longest, longest - 7, longest - 8, 1, 0]), (0, [longest]), (33, [34, longest - 1])]
    c = calls.Cache(rng, groups, 2, 128, 16, kv)
    q = calls.queries(rng, c.n, 10, 128)
    call = calls.Call(hip, c, q, 10)
    first = call.run()
    calls.check(c, first, q, 10)
    assert np.array_equal(call.run(), first)


@pytest.mark.parametrize("H", [31, 32, 33, 64, 128])
@calls.KINDS
def test_query_heads_of_one_kv_head(hip, kv, H):
    rng = np.random.default_rng(H)
    c = calls.Cache(rng, [(50, [48, 49, 50]), (20, [77, 20])], 1, 64, 32, kv)
    q = calls.queries(rng, c.n, H, 64)
    calls.check(c, calls.Call(hip, c, q, H).run(), q, H)


@pytest.mark.parametrize("log2", [23, 25])
def test_pages_of_many_positions(hip, log2):
    """One page of 2^23 and of 2^25 positions (offsets inside it pass 2^31 bytes): keys of zero but for the last, which
    takes all the weight (2^25 e^-60 of it is left to the others), so each row's output is the V of its last position."""
    from qraf_amd.backend import DeviceBuffer
    hd, ps = 64, 1 << log2
    k, v = (DeviceBuffer(ps * hd * 2) for _ in range(2))
    k.zero()
    v.zero()
    rng = np.random.default_rng(log2)
    q = np.ones((3, 2, hd), np.float32)
    ctx = np.array([ps, ps - 1, 5], np.int32)
    want = rng.standard_normal((3, hd)).astype(np.float16)
    for r, c in enumerate(ctx):
        # scores 60, 120 and 180, the longest row's last one the largest
        k.upload(np.full(hd, 60.0 * (3 - r) / np.sqrt(hd), np.float16), int(c - 1) * hd * 2)
        for d in range(hd):
            v.upload(want[r, d:d + 1], (d * ps + int(c) - 1) * 2)
    up = DeviceBuffer.from_array
    bufs = [up(q), up(np.zeros((3, 1), np.int32)), up(ctx), up(np.array([0, 3], np.int32)), up(np.array([ps], np.int32))]
    size = hip.lib.qraf_hip_group_attention_workspace_bytes(3, 1, 2, 1, hd, ps)
    ws, out = DeviceBuffer(max(size, 16)), up(np.zeros((3, 2, hd), np.float32))
    hip._lib.call("qraf_hip_group_attention_dev", bufs[0].ptr, k.ptr, v.ptr, calls.F16, bufs[1].ptr, 1,
                  bufs[2].ptr, bufs[3].ptr, bufs[4].ptr, 3, 1, 2, 1, hd, ps, np.float32(1 / np.sqrt(hd)), ps, out.ptr,
                  ws.ptr, size, None)
    hip._lib.call("qraf_hip_stream_synchronize", None)
    got = out.download(np.float32, 6 * hd).reshape(3, 2, hd)
    assert np.all(np.abs(got - want[:, None]) <= 1e-5 * np.abs(want[:, None]) + 1e-6)

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

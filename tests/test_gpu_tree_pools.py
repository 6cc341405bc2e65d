"""Trees in caches of more than 2^32 bytes and 2^31 elements, on other streams, in graphs that share a workspace, and a
page that two sequences share."""
import numpy as np
import pytest

from tests.test_gpu_tree import Pool
from tests.test_gpu_tree_attention import F16, F32, I8, KINDS, Call, Trees, check, tree

pytestmark = pytest.mark.gpu


def block_bytes(kv, ps, hd):
    return ps * (hd + 4 if kv == I8 else hd * (4 if kv == F32 else 2))


@KINDS
@pytest.mark.parametrize("ps", [16, 8])  # the tiles, and the form of any page size
def test_attention_in_a_large_pool(hip, kv, ps):
    from qraf_amd.backend import DeviceBuffer
    rng = np.random.default_rng(21)
    c = Trees(rng, [(700, tree(rng, 20)), (90, tree(rng, 33)), (3, tree(rng, 7))], 2, 128, ps, kv, max_ctx=3000)
    q = rng.standard_normal((c.n, 8, 128)).astype(np.float32)
    call = Call(hip, c, q, 8)
    page = 2 * block_bytes(kv, ps, 128)
    far = (1 << 31) * (1 if kv == I8 else 4 if kv == F32 else 2) // page + (1 << 32) // page * (kv == I8) + 5  # pages
    k, v = c.device()
    for name, a in (("k", k), ("v", v)):
        b = DeviceBuffer(far * page + a.nbytes)
        b.upload(a, far * page)
        setattr(call, name, b)
    call.table.upload((c.table + far).astype(np.int32))
    call.launch()
    check(c, q, call.result())


@KINDS
def test_compaction_in_a_large_pool(hip, kv):
    """Layers 2^32 bytes apart and more, and in each a pool whose pages in use lie past 2^31 bytes."""
    from qraf_amd.backend import DeviceBuffer
    rng = np.random.default_rng(22)
    Hkv, ps, hd, base, nodes, path = 2, 16, 64, 37, 20, [0, 2, 3, 9, 10, 17]
    pool = Pool(rng, kv, 1, 5, Hkv, ps, hd)
    page = Hkv * pool.block
    far = (1 << 31) // page + 3
    layer = (1 << 32) + 256
    at = [far * page, layer + far * page]
    assert at[0] + pool.layer_bytes < layer
    table = rng.permutation(5).astype(np.int32)[None]
    up, dev = DeviceBuffer.from_array, []
    for a in (pool.k, pool.v):
        b = DeviceBuffer(at[1] + pool.layer_bytes)
        for o in at:
            b.upload(a, o)
        dev.append(b)
    args = [up(x) for x in ((table + far).astype(np.int32), np.array([base], np.int32), np.array([0, nodes], np.int32),
                            np.array(path + [-1] * (nodes - len(path)), np.int32))]
    hip._lib.call("qraf_hip_kv_compact_dev", dev[0].ptr, dev[1].ptr, kv, 2, layer, args[0].ptr, 5, args[1].ptr,
                  args[2].ptr, args[3].ptr, 1, nodes, Hkv, hd, ps, None)
    hip._lib.call("qraf_hip_device_synchronize")
    for v, (b, a) in enumerate(zip(dev, (pool.k, pool.v))):
        cell, want = pool.cells(bool(v)), a.copy()
        for j, node in enumerate(path):
            src, dst = base + node, base + j
            want[cell[:, table[0, dst // ps], :, dst % ps]] = a[cell[:, table[0, src // ps], :, src % ps]]
        for o in at:
            assert np.array_equal(b.download(np.uint8, want.size, o), want)


@KINDS
def test_calls_on_two_streams(hip, kv):
    """Each with a workspace of its own, neither waiting for the other."""
    from qraf_amd.backend import Stream
    rng = np.random.default_rng(23)
    calls = []
    for seqs in ([(1900, tree(rng, 40)), (500, tree(rng, 9))], [(60 * i, tree(rng, 5)) for i in range(20)]):
        c = Trees(rng, seqs, 2, 128, 16, kv)
        q = rng.standard_normal((c.n, 8, 128)).astype(np.float32)
        calls.append((c, q, Call(hip, c, q, 8), Stream()))
    for _ in range(20):
        for _, _, call, st in calls:
            call.launch(st.h)
    for c, q, call, st in calls:
        st.synchronize()
        check(c, q, call.result())
        st.destroy()


def test_graphs_that_share_a_workspace(hip):
    """Captured calls of several shapes and page types, one behind another, each replay with another behind it."""
    from qraf_amd.backend import DeviceBuffer, Graph, Stream
    rng, st, made = np.random.default_rng(24), Stream(), []
    for kv, seqs in ((F32, [(800, tree(rng, 30))]), (F16, [(100 * i, tree(rng, 6)) for i in range(9)]),
                     (I8, [(10, tree(rng, 2)) for _ in range(70)])):
        c = Trees(rng, seqs, 2, 64, 16, kv, max_ctx=2000)
        q = rng.standard_normal((c.n, 8, 64)).astype(np.float32)
        made.append((c, q, Call(hip, c, q, 8)))
    ws = DeviceBuffer.from_array(np.full(max(call.ws_bytes for _, _, call in made), 0xFF, np.uint8))
    graphs = []
    for _, _, call in made:
        call.ws = ws
        call.launch(st.h)
        st.synchronize()
        g = Graph(st)
        with g:
            call.launch(st.h)
        graphs.append(g)
    for order in ((0, 1, 2), (2, 0, 1), (1, 1, 0, 2)):
        for _, _, call in made:
            call.out.upload(np.full((call.c.n, 8, 64), np.float32(0x7F)))
        for i in order:
            graphs[i].launch()
        st.synchronize()
        for c, q, call in made:
            check(c, q, call.result())
    for g in graphs:
        g.destroy()
    st.destroy()


@KINDS
def test_sequences_that_share_pages(hip, kv):
    """Two sequences with the same first pages and one whose pages repeat."""
    rng = np.random.default_rng(25)
    c = Trees(rng, [(130, tree(rng, 12)), (200, tree(rng, 12)), (100, tree(rng, 5))], 2, 64, 16, kv, max_ctx=1500)
    c.table[1, :8] = c.table[0, :8]
    c.table[2, :6] = c.table[2, 0]
    q = rng.standard_normal((c.n, 8, 64)).astype(np.float32)
    call = Call(hip, c, q, 8)
    call.launch()
    check(c, q, call.result())

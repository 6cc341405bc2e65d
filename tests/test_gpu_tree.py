"""The walk along a tree of drafted tokens, the compaction of its cache and the store of its nodes: whole numbers and
copies, equal to their definitions bit for bit."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F32, F16, I8 = 0, 1, 102
KINDS = pytest.mark.parametrize("kv", [F32, F16, I8], ids=["f32", "f16", "i8"])


# ------------------------------------------------------------------ accept

def walk(parents, drafts, picks):
    at, path = 0, [0]
    while True:
        child = [i for i in range(at + 1, len(parents)) if parents[i] == at and drafts[i] == picks[at]]
        if not child:
            return path, [int(picks[i]) for i in path]
        at = child[0]
        path.append(at)


def accept(hip, parents, drafts, picks, starts, stream=None):
    from qraf_amd.backend import DeviceBuffer
    up, n = DeviceBuffer.from_array, len(parents)
    seqs = len(starts) - 1
    dev = [up(np.asarray(x, t)) for x, t in ((picks, np.uint32), (drafts, np.uint32), (parents, np.int32),
                                             (starts, np.int32))]
    out = [up(np.full(k, 77, np.int32)) for k in (seqs, n, n)]
    hip._lib.call("qraf_hip_tree_accept_dev", *(b.ptr for b in dev), seqs, n, *(b.ptr for b in out), stream)
    hip._lib.call("qraf_hip_device_synchronize")
    return (out[0].download(np.int32, seqs), out[1].download(np.int32, n), out[2].download(np.uint32, n), dev, out)


def random_tree(rng, n, likely=0.8, vocab=50):
    parents = [-1] + [int(rng.integers(max(0, i - 6), i)) for i in range(1, n)]
    drafts, picks = rng.integers(0, vocab, n), rng.integers(0, vocab, n)
    for i in rng.permutation(n):
        if parents[i] >= 0 and rng.random() < likely:
            picks[parents[i]] = drafts[i]
    return parents, list(drafts), list(picks)


def expect(trees, ahead=0, behind=0):
    acc, path, tokens = [], [77] * ahead, [77] * ahead
    for p, d, t in trees:
        if not p:
            acc.append(0)
            continue
        w, said = walk(p, d, t)
        acc.append(len(w) - 1)
        path += w + [-1] * (len(p) - len(w))
        tokens += said + [0xFFFFFFFF] * (len(p) - len(w))
    return acc, path + [77] * behind, tokens + [77] * behind


def run_accept(hip, trees, ahead=0, behind=0):
    cols = [sum((list(t[k]) for t in trees), []) for k in range(3)]
    cols = [[3] * ahead + c + [3] * behind for c in cols]
    starts = ahead + np.cumsum([0] + [len(t[0]) for t in trees])
    got = accept(hip, *cols, starts)
    for g, w in zip(got, expect(trees, ahead, behind)):
        assert list(g) == w


@pytest.mark.parametrize("n", [1, 2, 3, 8, 63, 64, 65, 127, 128, 129, 300])
def test_accept(hip, n):
    rng = np.random.default_rng(n)
    run_accept(hip, [random_tree(rng, n) for _ in range(9)])


def test_accept_ragged_with_rows_of_no_sequence(hip):
    rng = np.random.default_rng(0)
    trees = [random_tree(rng, int(n)) if n else ([], [], []) for n in (0, 5, 1, 0, 64, 17, 0, 2)]
    run_accept(hip, trees, ahead=3, behind=2)


def test_accept_deep_chain(hip):
    n = 200
    run_accept(hip, [([-1] + list(range(n - 1)), list(range(n)), list(range(1, n + 1)))])
    run_accept(hip, [([-1] + list(range(n - 1)), list(range(n)), list(range(1, 101)) + [5] * 100)])


def test_accept_takes_the_lowest_of_equal_children(hip):
    run_accept(hip, [([-1, 0, 0, 0, 1, 2], [0, 9, 9, 9, 4, 5], [9, 4, 5, 1, 8, 8])])


def test_accept_never_reaches_nodes_without_a_lower_parent(hip):
    """Parents that are the node itself, a later one, negative or past the tree; tokens of all ones."""
    run_accept(hip, [([7, 1, 3, 0, -5, 99, 3], [5] * 7, [5] * 7), ([0, 0], [5, 0xFFFFFFFF], [0xFFFFFFFF, 5])])


def test_accept_in_a_graph(hip):
    from qraf_amd.backend import Graph, Stream
    rng = np.random.default_rng(5)
    trees = [random_tree(rng, 40) for _ in range(3)]
    cols = [sum((list(t[k]) for t in trees), []) for k in range(3)]
    starts, st = np.arange(4) * 40, Stream()
    _, _, _, dev, out = accept(hip, *cols, starts, st.h)
    g = Graph(st)
    with g:
        hip._lib.call("qraf_hip_tree_accept_dev", *(b.ptr for b in dev), 3, 120, *(b.ptr for b in out), st.h)
    for k in range(4):
        trees = [random_tree(rng, 40, 0.5 + 0.1 * k) for _ in range(3)]
        for b, key, t in ((dev[0], 2, np.uint32), (dev[1], 1, np.uint32), (dev[2], 0, np.int32)):
            b.upload(np.array(sum((list(x[key]) for x in trees), []), t))
        g.launch()
        st.synchronize()
        want = expect(trees)
        assert list(out[0].download(np.int32, 3)) == want[0] and list(out[1].download(np.int32, 120)) == want[1]
        assert list(out[2].download(np.uint32, 120)) == want[2]
    g.destroy()
    st.destroy()


# ------------------------------------------------------------------ compact

ITEM = {F32: 4, F16: 2, I8: 1}


class Pool:
    """Random bytes as n_layers caches; their positions' bytes by (layer, page, head, offset)."""

    def __init__(self, rng, kv, layers, pages, Hkv, ps, hd, pad=0):
        self.kv, self.shape = kv, (layers, pages, Hkv, ps, hd)
        self.block = ps * (hd + 4 if kv == I8 else hd * ITEM[kv])
        self.layer_bytes = pages * Hkv * self.block + pad
        self.k, self.v = (rng.integers(0, 256, layers * self.layer_bytes).astype(np.uint8) for _ in range(2))

    def cells(self, v):
        """Index arrays of the bytes of every (layer, page, head, offset)."""
        L, P, H, ps, hd = self.shape
        at = (np.arange(L)[:, None, None] * self.layer_bytes + np.arange(P)[:, None] * H * self.block +
              np.arange(H) * self.block)[..., None, None]
        off, n = np.arange(ps)[:, None], ITEM[self.kv]
        if v and self.kv != F32:  # dimension-major
            inner = (np.arange(hd)[None, :, None] * ps + off[:, :, None]) * n + np.arange(n)
            inner = inner.reshape(ps, hd * n)
        else:
            inner = off * hd * n + np.arange(hd * n)
        if self.kv == I8:
            inner = np.concatenate([inner, ps * hd + off * 4 + np.arange(4)], 1)
        return at + inner


def run_compact(hip, kv, seqs, layers=2, Hkv=2, hd=64, ps=16, pad=0, wide=None, rng=None):
    """seqs: a list of (base, number of nodes, the path's entries)."""
    from qraf_amd.backend import DeviceBuffer
    rng = rng or np.random.default_rng(11)
    per = [-(-(b + n) // ps) for b, n, _ in seqs]
    wide = wide or max(per)
    pool = Pool(rng, kv, layers, sum(per) + 1, Hkv, ps, hd, pad)
    perm, at = rng.permutation(sum(per) + 1), 0
    table = np.full((len(seqs), wide), perm[-1], np.int32)
    for s, p in enumerate(per):
        table[s, :min(p, wide)] = perm[at:at + min(p, wide)]
        at += p
    starts = np.cumsum([0] + [n for _, n, _ in seqs]).astype(np.int32)
    path = np.concatenate([np.array(list(p) + [-1] * (n - len(p)), np.int32)[:n] for _, n, p in seqs])
    base = np.array([b for b, _, _ in seqs], np.int32)
    want = []
    for v, bytes_ in ((False, pool.k), (True, pool.v)):
        cell, w = pool.cells(v), bytes_.copy()
        for s, (b, n, p) in enumerate(seqs):
            last = -1
            for j, node in enumerate(p):
                if not last < node < n or b + node >= wide * ps:
                    break
                last = node
                src, dst = b + node, b + j
                w[cell[:, table[s, dst // ps], :, dst % ps]] = bytes_[cell[:, table[s, src // ps], :, src % ps]]
        want.append(w)
    up = DeviceBuffer.from_array
    k, v, t, bs, st, pt = (up(x) for x in (pool.k, pool.v, table, base, starts, path))
    hip._lib.call("qraf_hip_kv_compact_dev", k.ptr, v.ptr, kv, layers, pool.layer_bytes, t.ptr, wide, bs.ptr, st.ptr,
                  pt.ptr, len(seqs), path.size, Hkv, hd, ps, None)
    hip._lib.call("qraf_hip_device_synchronize")
    for b, w in ((k, want[0]), (v, want[1])):
        assert np.array_equal(b.download(np.uint8, w.size), w)


@KINDS
@pytest.mark.parametrize("Hkv,hd,ps", [(3, 64, 16), (2, 128, 16), (1, 128, 32), (4, 16, 16), (2, 32, 48), (1, 64, 1),
                                       (2, 64, 7), (8, 128, 64)])
def test_compact_shapes(hip, kv, Hkv, hd, ps):
    run_compact(hip, kv, [(37, 20, [0, 3, 4, 9, 19]), (16, 9, [0, 1, 2, 8]), (0, 5, [0, 4])], 3, Hkv, hd, ps)


@KINDS
def test_compact_paths(hip, kv):
    """Nothing to move, every node, nothing at all, the root moved, one node; entries that do not ascend, lie past the
    tree or are negative end a path."""
    run_compact(hip, kv, [(30, 6, [0]), (31, 6, [0, 1, 2, 3, 4, 5]), (5, 6, []), (90, 6, [2, 5]), (12, 1, [0]),
                          (40, 6, [0, 2, 2, 5]), (41, 6, [0, 3, 1, 5]), (42, 6, [0, 2, 6, 7]), (43, 6, [-3, 2]),
                          (0, 64, list(range(0, 64, 3)))])


@KINDS
def test_compact_more_nodes_than_a_wave(hip, kv):
    rng = np.random.default_rng(12)
    run_compact(hip, kv, [(77, 200, sorted(rng.choice(200, 150, replace=False))), (3, 129, list(range(129))),
                          (8, 300, list(range(1, 300))), (0, 130, list(range(0, 130, 2)))], 1)


@KINDS
def test_compact_ragged_sequences_without_nodes_and_padded_layers(hip, kv):
    run_compact(hip, kv, [(3, 0, []), (20, 7, [0, 5]), (9, 0, []), (300, 30, [0, 10, 20, 29]), (4, 0, [])], 5, pad=48)


@KINDS
def test_compact_past_the_table(hip, kv):
    run_compact(hip, kv, [(20, 30, [0, 5, 11, 13, 25])], wide=2)


@KINDS
@pytest.mark.parametrize("base", [5, 6, 100, 2 ** 30, 2 ** 31 - 64, 2 ** 31 - 63, 2 ** 31 - 1, -1, -2 ** 31])
def test_compact_bases_past_the_table(hip, kv, base):
    """Pages of one position: a base at the table's end or past it, up to int32's largest, moves nothing and names no
    page outside the table; a negative one is 0."""
    from qraf_amd.backend import DeviceBuffer
    rng, wide, nodes, up = np.random.default_rng(15), 5, 70, DeviceBuffer.from_array
    pool = Pool(rng, kv, 2, 3 * wide, 2, 1, 64)
    # the second sequence's table row; those beside it name other pages
    table = rng.permutation(3 * wide).astype(np.int32).reshape(3, wide)
    path = np.tile(np.concatenate([[1, 2, 4], np.arange(5, 5 + nodes - 3)]), 3).astype(np.int32)
    path[:nodes] = path[2 * nodes:] = -1
    d = [up(x) for x in (pool.k, pool.v, table, np.array([0, base, 0], np.int32),
                         (np.arange(4) * nodes).astype(np.int32), path)]
    hip._lib.call("qraf_hip_kv_compact_dev", d[0].ptr, d[1].ptr, kv, 2, pool.layer_bytes, d[2].ptr, wide, d[3].ptr,
                  d[4].ptr, d[5].ptr, 3, path.size, 2, 64, 1, None)
    hip._lib.call("qraf_hip_device_synchronize")
    for v, b, was in ((False, d[0], pool.k), (True, d[1], pool.v)):
        cell, want = pool.cells(v), was.copy()
        for to, at in ((0, 1), (1, 2), (2, 4)) if base < 0 else ():
            want[cell[:, table[1, to], :, 0]] = was[cell[:, table[1, at], :, 0]]
        assert np.array_equal(b.download(np.uint8, want.size), want)


@KINDS
@pytest.mark.parametrize("pad,shift", [(4, 0), (8, 0), (12, 0), (0, 4), (0, 8), (0, 12), (12, 4)])
@pytest.mark.parametrize("Hkv,hd,ps", [(3, 64, 16), (2, 128, 16), (5, 16, 6), (2, 32, 48)])
def test_compact_of_caches_that_four_bytes_align(hip, kv, Hkv, hd, ps, pad, shift):
    """Layers and pools whose alignment is 4 or 8 bytes: keys move in pieces of 4.  Paths of more than eight entries, of
    neighbours among them; the bytes ahead of a pool and behind a layer stay."""
    from qraf_amd.backend import DeviceBuffer
    rng, up, layers = np.random.default_rng(16), DeviceBuffer.from_array, 3
    seqs = [(37, 30, [0, 3, 4, 5, 6, 7, 9, 12, 13, 19, 28, 29]), (14, 12, [0, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11]),
            (0, 20, [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 16, 17, 18])]
    per = [-(-(b + n) // ps) for b, n, _ in seqs]
    pool = Pool(rng, kv, layers, sum(per), Hkv, ps, hd, pad)
    table, ids = np.zeros((3, max(per)), np.int32), np.split(rng.permutation(sum(per)), np.cumsum(per)[:-1])
    path = np.concatenate([p + [-1] * (n - len(p)) for _, n, p in seqs]).astype(np.int32)
    for t, i in zip(table, ids):
        t[:len(i)] = i
    base, starts = np.array([b for b, _, _ in seqs], np.int32), np.cumsum([0] + [n for _, n, _ in seqs]).astype(np.int32)
    ahead = rng.integers(0, 256, shift).astype(np.uint8)
    k, v, t, bs, st, pt = (up(x) for x in (np.concatenate([ahead, pool.k]), np.concatenate([ahead, pool.v]), table, base,
                                           starts, path))
    hip._lib.call("qraf_hip_kv_compact_dev", k.ptr + shift, v.ptr + shift, kv, layers, pool.layer_bytes, t.ptr,
                  table.shape[1], bs.ptr, st.ptr, pt.ptr, 3, path.size, Hkv, hd, ps, None)
    hip._lib.call("qraf_hip_device_synchronize")
    for b, was, by_dim in ((k, pool.k, False), (v, pool.v, True)):
        cell, want = pool.cells(by_dim), was.copy()
        for row, (at, _, nodes) in zip(table, seqs):
            for j, node in enumerate(nodes):
                src, dst = at + node, at + j
                want[cell[:, row[dst // ps], :, dst % ps]] = was[cell[:, row[src // ps], :, src % ps]]
        got = b.download(np.uint8, shift + want.size)
        assert np.array_equal(got[:shift], ahead) and np.array_equal(got[shift:], want)


def test_compact_many_layers_and_sequences(hip):
    rng = np.random.default_rng(13)
    seqs = [(int(rng.integers(0, 60)), 12, [0] + sorted(rng.choice(np.arange(1, 12), 4, replace=False)))
            for _ in range(40)]
    run_compact(hip, F16, seqs, 30, 2, 64, 16)


# ------------------------------------------------------------------ append

@KINDS
@pytest.mark.parametrize("H,Hkv,hd,bias", [(9, 3, 64, False), (16, 2, 128, True), (4, 4, 32, True)])
def test_append_is_rope_append_at_another_place(hip, kv, H, Hkv, hd, bias):
    """Row i's q, and its K and V at its slot, are those of qraf_hip_rope_append_dev at its position; nothing else
    changes."""
    from qraf_amd.backend import DeviceBuffer
    rng = np.random.default_rng(14)
    up, ps, n, seqs, wide = DeviceBuffer.from_array, 16, 11, 3, 6
    row = (H + 2 * Hkv) * hd
    qkv, b = rng.standard_normal((n, row)).astype(np.float32), rng.standard_normal(row).astype(np.float32)
    pos = rng.integers(0, 60, n).astype(np.int32)
    of = np.array([0] * 4 + [1] * 5 + [2] * 2, np.int32)
    slots = np.concatenate([30 + np.arange(4), 14 + np.arange(5), 60 + np.arange(2)]).astype(np.int32)
    table = rng.permutation(seqs * wide).astype(np.int32).reshape(seqs, wide)
    rope = np.zeros((96, hd), np.float32)
    hip._lib.call("qraf_hip_rope_table_host", 96, hd, 1e4, rope.ctypes.data_as(hip._lib.fp))
    pool = Pool(rng, kv, 1, seqs * wide, Hkv, ps, hd)
    d_qkv, d_b, d_pos, d_of, d_slots, d_table, d_rope = (up(x) for x in (qkv, b, pos, of, slots, table, rope))
    got = [up(pool.k), up(pool.v), up(np.zeros((n, H * hd), np.float32))]
    hip._lib.call("qraf_hip_tree_append_dev", d_qkv.ptr, d_b.ptr if bias else None, n, H, Hkv, hd, d_pos.ptr,
                  d_slots.ptr, d_of.ptr, d_rope.ptr, got[2].ptr, got[0].ptr, got[1].ptr, kv, d_table.ptr, wide, ps,
                  None)
    own = np.arange(n * wide, dtype=np.int32).reshape(n, wide)  # a cache for each row
    far = Pool(rng, kv, 1, n * wide, Hkv, ps, hd)
    ref = [up(far.k), up(far.v), up(np.zeros((n, H * hd), np.float32))]
    d_own = up(own)
    hip._lib.call("qraf_hip_rope_append_dev", d_qkv.ptr, d_b.ptr if bias else None, n, H, Hkv, hd, d_pos.ptr,
                  d_rope.ptr, ref[2].ptr, ref[0].ptr, ref[1].ptr, kv, d_own.ptr, wide, ps, None)
    hip._lib.call("qraf_hip_device_synchronize")
    assert np.array_equal(got[2].download(np.float32, n * H * hd), ref[2].download(np.float32, n * H * hd))
    for v in (False, True):
        g = got[v].download(np.uint8, pool.k.size)
        r = ref[v].download(np.uint8, far.k.size)
        cell, fcell = pool.cells(v), far.cells(v)
        want = (pool.v if v else pool.k).copy()
        for i in range(n):
            want[cell[0, table[of[i], slots[i] // ps], :, slots[i] % ps]] = r[fcell[0, own[i, pos[i] // ps], :,
                                                                                   pos[i] % ps]]
        assert np.array_equal(g, want)


# ------------------------------------------------------------------ a step of all of them

@KINDS
def test_a_captured_step_of_trees(hip, kv):
    """Append, attention, sampling, acceptance, compaction and log probabilities in one graph, replayed on new inputs
    with the same calls made eagerly between: equal bit for bit, the cache among them."""
    from qraf_amd._lib import SamplingParams, lib
    from qraf_amd.backend import DeviceBuffer, Graph, Stream
    rng = np.random.default_rng(21)
    H, Hkv, hd, ps, V, sizes, bases = 8, 2, 64, 16, 700, (9, 5), (45, 100)
    up, n, wide = DeviceBuffer.from_array, sum(sizes), 8
    starts = np.cumsum([0, *sizes]).astype(np.int32)
    of = np.repeat([0, 1], sizes).astype(np.int32)
    table = rng.permutation(2 * wide).astype(np.int32).reshape(2, wide)
    rope = np.zeros((128, hd), np.float32)
    hip._lib.call("qraf_hip_rope_table_host", 128, hd, 1e4, rope.ctypes.data_as(hip._lib.fp))
    if kv == I8:  # bytes with scales
        block = np.concatenate([rng.integers(0, 256, (2 * wide * Hkv, ps * hd)).astype(np.uint8),
                                np.full((2 * wide * Hkv, ps), 0.02, np.float32).view(np.uint8)], 1)
        cache = block.reshape(-1)
    else:
        cache = rng.standard_normal(2 * wide * Hkv * ps * hd).astype(np.float16 if kv == F16 else np.float32).view(np.uint8)
    d = {k: up(v) for k, v in dict(starts=starts, of=of, table=table, rope=rope, base=np.array(bases, np.int32),
                                   k=cache, v=cache).items()}
    for k, size in dict(qkv=n * (H + 2 * Hkv) * hd * 4, pos=n * 4, slots=n * 4, masks=n * 8, parents=n * 4, draft=n * 4,
                        logits=n * V * 4, q=n * H * hd * 4, out=n * H * hd * 4, picks=n * 4, acc=8, path=n * 4,
                        tokens=n * 4, lp=n * 4, rank=n * 4, ent=n * 4, tt=n * 16, tl=n * 16).items():
        d[k] = up(np.zeros(size, np.uint8))
    params = SamplingParams(0.0, 0, 1.0, 1.0)
    aw, lw = lib.qraf_hip_tree_attention_workspace_bytes(n, 2, H, Hkv, hd, 128), \
        lib.qraf_hip_token_logprobs_workspace_bytes(n, V, 4)
    d["aw"], d["lw"] = up(np.zeros(aw, np.uint8)), up(np.zeros(lw, np.uint8))
    p = {k: b.ptr for k, b in d.items()}

    def step(st):
        import ctypes
        call = hip._lib.call
        call("qraf_hip_tree_append_dev", p["qkv"], None, n, H, Hkv, hd, p["pos"], p["slots"], p["of"], p["rope"], p["q"],
             p["k"], p["v"], kv, p["table"], wide, ps, st)
        call("qraf_hip_tree_attention_dev", p["q"], p["k"], p["v"], kv, p["table"], wide, p["base"], p["starts"],
             p["masks"], n, 2, H, Hkv, hd, ps, 0.125, 128, p["out"], p["aw"], aw, st)
        call("qraf_hip_sample_dev", p["logits"], n, V, ctypes.byref(params), None, None, 0, None, p["picks"], st)
        call("qraf_hip_tree_accept_dev", p["picks"], p["draft"], p["parents"], p["starts"], 2, n, p["acc"], p["path"],
             p["tokens"], st)
        call("qraf_hip_kv_compact_dev", p["k"], p["v"], kv, 1, cache.size, p["table"], wide, p["base"], p["starts"],
             p["path"], 2, n, Hkv, hd, ps, st)
        call("qraf_hip_token_logprobs_dev", p["logits"], n, V, p["picks"], p["lp"], p["rank"], p["ent"], 4, p["tt"],
             p["tl"], p["lw"], lw, st)

    def inputs():
        trees = [random_tree(rng, k, 0.9, V) for k in sizes]
        masks, depth = [], []
        for parents, _, _ in trees:
            m, at = [], []
            for i, u in enumerate(parents):
                m.append((m[u] if i else 0) | 1 << i)
                at.append(at[u] + 1 if i else 0)
            masks += m
            depth += at
        x = rng.standard_normal((n, V)).astype(np.float32)
        for i, t in enumerate(sum((list(t[2]) for t in trees), [])):
            x[i, t] = 20.0
        d["logits"].upload(x)
        d["qkv"].upload(rng.standard_normal((n, (H + 2 * Hkv) * hd)).astype(np.float32))
        d["masks"].upload(np.array(masks, np.uint64))
        d["pos"].upload((np.array(bases)[of] + depth).astype(np.int32))
        d["slots"].upload((np.array(bases)[of] + np.arange(n) - starts[of]).astype(np.int32))
        d["parents"].upload(np.array(sum((t[0] for t in trees), []), np.int32))
        d["draft"].upload(np.array(sum((list(t[1]) for t in trees), []), np.uint32))
        return trees

    names = ("k", "v", "out", "acc", "path", "tokens", "lp", "rank", "ent", "tt", "tl")
    st = Stream()
    inputs()
    step(st.h)
    st.synchronize()
    g = Graph(st)
    with g:
        step(st.h)
    for _ in range(4):
        trees = inputs()
        results = []
        for way in (lambda: g.launch(), lambda: step(None)):
            d["k"].upload(cache)
            d["v"].upload(cache)
            way()
            st.synchronize()
            hip._lib.call("qraf_hip_device_synchronize")
            results.append({k: d[k].download(np.uint8, d[k].nbytes) for k in names})
        for k in names:
            assert np.array_equal(results[0][k], results[1][k]), k
        acc, path, toks = expect(trees)
        assert list(results[0]["acc"].view(np.int32)) == acc and list(results[0]["path"].view(np.int32)) == path
        assert list(results[0]["tokens"].view(np.uint32)) == toks
        assert list(results[0]["rank"].view(np.int32)) == [0] * n
    g.destroy()
    st.destroy()

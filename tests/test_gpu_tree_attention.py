"""Attention of trees of drafted tokens (qraf_hip_tree_attention_dev) against the softmax of its definition in 64
bits.

Tolerance, per output element: scores are sums of head_dim products whose operands keep at least 21 bits, so they
are off by at most
    d = scale * sum_d |q_d k_d| * (2^-20 + head_dim * 2^-24),
which moves every probability by a factor within exp(+-2 d); and the weighted sum and its divisor are chains of at
most ctx + 64 fp32 additions:
    |got - want| <= (2 max_t d + (ctx + 64) * 2^-24) * sum_t p_t |v_t| + ctx * 2^-37 * max_t |v_t| + 1e-30.
The last but one: a weight enters its product as two fp16 values, times 2^14 (the largest weight is at most 1, and
at least one is 1).  fp16 has steps of 2^-24 at its least, so a weight is off by up to 2^-38 however small it is;
int8 pages multiply it by the position's V scale over a power of two that may be twice the largest scale, which
makes that 2^-37 of the largest |v| for each of ctx positions.  (f32 V is held in steps of 2^-40 of the largest.)
ctx, max_t and sum_t: over the positions that the row attends to.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F32, F16, I8 = 0, 1, 102
KINDS = pytest.mark.parametrize("kv", [F32, F16, I8], ids=["f32", "f16", "i8"])


def tree(rng, n, width=8):
    """Masks of a random tree's nodes, node i at position i."""
    out = []
    for i in range(n):
        out.append((out[int(rng.integers(max(0, i - width), i))] if i else 0) | 1 << i)
    return out


class Trees:
    """seqs: a list of (base, [a mask of each row]); pages in logical form [page][kv head][position][dim] (int8: with a
    scale per position)."""

    def __init__(self, rng, seqs, Hkv, hd, ps, kv, max_ctx=None, ahead=0, behind=0):
        self.kv, self.ps, self.hd, self.Hkv = kv, ps, hd, Hkv
        self.base = np.array([b for b, _ in seqs], np.int32)
        self.masks = np.array([0] * ahead + [m for _, ms in seqs for m in ms] + [0] * behind, np.uint64)
        self.starts = (ahead + np.cumsum([0] + [len(ms) for _, ms in seqs])).astype(np.int32)
        self.n = self.masks.size
        ends = [b + max([int(m).bit_length() for m in ms] + [0]) for b, ms in seqs]
        self.max_ctx = max_ctx or max(1, max(ends))
        self.wide = -(-self.max_ctx // ps)
        per = [min(self.wide, -(-e // ps)) for e in ends]
        count = sum(per) + 2
        perm, at = rng.permutation(count), 0
        self.table = np.full((len(seqs), self.wide), perm[-1], np.int32)  # elsewhere: a page that nobody has
        for s, p in enumerate(per):
            self.table[s, :p] = perm[at:at + p]
            at += p
        shape = (count, Hkv, ps, hd)
        if kv == I8:
            self.K, self.V = (rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2))
            self.Ks, self.Vs = (rng.uniform(0.01, 0.04, shape[:3]).astype(np.float32) for _ in range(2))
        else:
            dt = np.float16 if kv == F16 else np.float32
            self.K, self.V = (rng.standard_normal(shape).astype(dt) for _ in range(2))
            self.Ks = self.Vs = None

    def at(self, s, t):
        return self.table[s, t // self.ps], t % self.ps

    def poison(self, s, t, what=np.nan, k=True, v=True):
        """Position t of sequence s no number (int8: its scales)."""
        p, o = self.at(s, t)
        for a, sc, on in ((self.K, self.Ks, k), (self.V, self.Vs, v)):
            if on:
                if sc is not None:
                    sc[p, :, o] = what
                else:
                    a[p, :, o] = what

    def rows(self):
        for s in range(len(self.base)):
            for r in range(self.starts[s], self.starts[s + 1]):
                yield s, r

    def sees(self, s, r):
        b, m = int(self.base[s]), int(self.masks[r])
        t = list(range(b)) + [b + j for j in range(64) if m >> j & 1]
        return np.array([x for x in t if x < self.max_ctx], np.int64)

    def device(self):
        def pool(a, s, v):
            x = np.ascontiguousarray(a.transpose(0, 1, 3, 2) if v and self.kv != F32 else a)
            if s is None:
                return x
            p = x.shape[0] * x.shape[1]
            return np.concatenate([x.reshape(p, -1).view(np.uint8),
                                   np.ascontiguousarray(s).reshape(p, -1).view(np.uint8)], 1)
        return pool(self.K, self.Ks, False), pool(self.V, self.Vs, True)


class Call:
    def __init__(self, hip, trees, q, H, fill=0x7F):
        from qraf_amd.backend import DeviceBuffer
        c, up = trees, DeviceBuffer.from_array
        self.c, self.hip, self.H = c, hip, H
        k, v = c.device()
        self.q, self.k, self.v, self.table, self.base = up(q), up(k), up(v), up(c.table), up(c.base)
        self.starts, self.masks, self.seqs = up(c.starts), up(c.masks), len(c.base)
        self.ws_bytes = hip.lib.qraf_hip_tree_attention_workspace_bytes(c.n, self.seqs, H, c.Hkv, c.hd, c.max_ctx)
        self.ws = up(np.full(self.ws_bytes, 0xFF, np.uint8))  # needs no initialisation: NaN in every float of it
        self.out = up(np.full((c.n, H, c.hd), np.float32(fill)))

    def launch(self, stream=None):
        c = self.c
        self.hip._lib.call("qraf_hip_tree_attention_dev", self.q.ptr, self.k.ptr, self.v.ptr, c.kv, self.table.ptr,
                           c.wide, self.base.ptr, self.starts.ptr, self.masks.ptr, c.n, self.seqs, self.H, c.Hkv, c.hd,
                           c.ps, 1.0 / np.sqrt(c.hd), c.max_ctx, self.out.ptr, self.ws.ptr, self.ws_bytes, stream)

    def result(self):
        self.hip._lib.call("qraf_hip_device_synchronize")
        return self.out.download(np.float32, self.c.n * self.H * self.c.hd).reshape(self.c.n, self.H, self.c.hd)


def check(c, q, got, rows=None, fill=0x7F):
    """Every row against its definition; rows of no sequence as they were."""
    H, scale = q.shape[1], float(np.float32(1.0 / np.sqrt(c.hd)))
    G = H // c.Hkv
    inside = np.zeros(c.n, bool)
    for s, r in c.rows():
        inside[r] = True
        if rows is not None and r not in rows:
            continue
        t = c.sees(s, r)
        if t.size == 0:
            assert np.all(got[r] == 0.0)
            continue
        page, off = c.table[s, t // c.ps], t % c.ps
        kv = []
        for a, sc in ((c.K, c.Ks), (c.V, c.Vs)):
            x = a[page, :, off].astype(np.float64)
            kv.append((x if sc is None else x * sc[page, :, off].astype(np.float64)[..., None]).transpose(1, 0, 2))
        K, V = kv
        for h in range(H):
            k, v, x = K[h // G], V[h // G], q[r, h].astype(np.float64)
            score = scale * (k @ x)
            p = np.exp(score - score.max())
            p /= p.sum()
            d = scale * (np.abs(k) @ np.abs(x)).max() * (2.0 ** -20 + c.hd * 2.0 ** -24)
            tol = (2 * d + (t.size + 64) * 2.0 ** -24) * (p @ np.abs(v)) + t.size * 2.0 ** -37 * np.abs(v).max(0) + 1e-30
            err = np.abs(got[r, h] - p @ v)
            assert np.all(err <= tol), (s, r, h, float((err / tol).max()))
    assert np.all(got[~inside] == fill)


def run(hip, c, H, rng, rows=None):
    q = rng.standard_normal((c.n, H, c.hd)).astype(np.float32)
    call = Call(hip, c, q, H)
    call.launch()
    got = call.result()
    check(c, q, got, rows)
    call.launch()
    assert np.array_equal(call.result(), got, equal_nan=True)  # the same from call to call
    return got


HEADS = [(9, 3, 64), (16, 2, 128), (4, 4, 64), (3, 1, 128), (12, 2, 64), (64, 1, 128)]


@KINDS
@pytest.mark.parametrize("H,Hkv,hd", HEADS)
def test_one_tree(hip, kv, H, Hkv, hd):
    rng = np.random.default_rng(hash((kv, H, hd)) & 0xFFFF)
    run(hip, Trees(rng, [(211, tree(rng, 13))], Hkv, hd, 16, kv), H, rng)


@KINDS
@pytest.mark.parametrize("base", [0, 1, 15, 16, 17, 31, 32, 33, 63, 255, 256, 257])
def test_bases(hip, kv, base):
    """The cache's end inside a page, inside a tile, and no cache at all."""
    rng = np.random.default_rng(base)
    run(hip, Trees(rng, [(base, tree(rng, 9)), (base + 3, tree(rng, 2))], 2, 64, 16, kv), 6, rng)


@KINDS
@pytest.mark.parametrize("nodes", [1, 2, 31, 32, 33, 63, 64])
def test_sizes(hip, kv, nodes):
    rng = np.random.default_rng(nodes)
    run(hip, Trees(rng, [(100, tree(rng, nodes)), (7, tree(rng, nodes, 64))], 1, 128, 16, kv), 8, rng)


@KINDS
@pytest.mark.parametrize("ps", [16, 32, 64, 128, 8, 4, 48, 1])
def test_page_sizes(hip, kv, ps):
    rng = np.random.default_rng(ps)
    run(hip, Trees(rng, [(75, tree(rng, 20)), (0, tree(rng, 5)), (130, tree(rng, 1))], 2, 64, ps, kv), 4, rng)


@KINDS
@pytest.mark.parametrize("hd", [16, 32])
def test_small_heads(hip, kv, hd):
    rng = np.random.default_rng(hd)
    run(hip, Trees(rng, [(90, tree(rng, 20)), (3, tree(rng, 5))], 2, hd, 16, kv), 4, rng)


@KINDS
def test_many_ragged(hip, kv):
    rng = np.random.default_rng(1)
    seqs = [(int(rng.integers(0, 700)), tree(rng, int(rng.integers(1, 24)))) for _ in range(20)]
    run(hip, Trees(rng, seqs, 2, 64, 16, kv), 8, rng)


@KINDS
@pytest.mark.parametrize("seqs", [63, 64, 65, 130])
@pytest.mark.parametrize("H,hd", [(6, 64), (32, 128)])
def test_many_sequences(hip, kv, seqs, H, hd):
    """Up to 64 sequences are planned by lane, more in LDS; bounds that choose the planned form; sequences without rows."""
    rng = np.random.default_rng(seqs)
    trees = [(int(rng.integers(0, 150)), tree(rng, int(rng.integers(0, 8)))) for _ in range(seqs)]
    trees[7] = (1200, tree(rng, 33))
    run(hip, Trees(rng, trees, 2, hd, 16, kv, max_ctx=3000, ahead=1, behind=2), H, rng)


@KINDS
def test_rows_of_two_blocks(hip, kv):
    """Rows whose query heads lie in two blocks of columns: 40 heads a KV head, and 128."""
    rng = np.random.default_rng(11)
    for H, n in ((40, 13), (128, 3), (100, 5)):
        run(hip, Trees(rng, [(700, tree(rng, n)), (33, tree(rng, 2))], 1, 64, 16, kv, max_ctx=2000), H, rng)


@KINDS
@pytest.mark.parametrize("max_ctx", [None, 9000])
def test_long(hip, kv, max_ctx):
    """Contexts that are split along their positions; bounds far above them."""
    rng = np.random.default_rng(2)
    c = Trees(rng, [(4999, tree(rng, 17)), (3000, tree(rng, 64)), (0, tree(rng, 3))], 2, 128, 16, kv, max_ctx=max_ctx)
    run(hip, c, 8, rng, rows={0, 5, 16, 17, 50, 80, 81, 83})


@KINDS
def test_bounds_above_the_lengths(hip, kv):
    rng = np.random.default_rng(3)
    run(hip, Trees(rng, [(40, tree(rng, 17)), (333, tree(rng, 40)), (0, tree(rng, 3))], 2, 64, 16, kv, max_ctx=4000), 6,
        rng)


@KINDS
@pytest.mark.parametrize("max_ctx", [None, 5000])
def test_any_masks(hip, kv, max_ctx):
    """Not only trees: random bits, none at all, the highest, holes."""
    rng = np.random.default_rng(4)
    ms = [int(m) for m in rng.integers(0, 1 << 64, 9, dtype=np.uint64)] + [0, 1 << 63, (1 << 64) - 1, 1, 0xAAAA << 30]
    run(hip, Trees(rng, [(50, ms), (0, ms), (0, [0, 0, 0]), (17, [0])], 2, 64, 16, kv, max_ctx=max_ctx), 4, rng)


@KINDS
@pytest.mark.parametrize("wide", [False, True])
def test_masks_past_the_bound(hip, kv, wide):
    """Bits at or past max_ctx name nothing, a base past it is it: also where nothing is left."""
    rng = np.random.default_rng(5)
    G = 8 if wide else 2
    ms = [(1 << 64) - 1, 1 << 40, (1 << 40) | 1, 0] * (5 if wide else 1)
    c = Trees(rng, [(60, ms), (0, [1 << 63, 1 << 62]), (70, [1, 1 << 3])], 2, 64, 16, kv, max_ctx=61)
    c.base[2] = 999
    run(hip, c, 2 * G, rng)


@KINDS
@pytest.mark.parametrize("max_ctx", [None, 5000])
def test_rows_of_no_sequence_and_empty_sequences(hip, kv, max_ctx):
    rng = np.random.default_rng(6)
    seqs = [(40, []), (33, tree(rng, 5)), (9, []), (20, tree(rng, 7)), (5, [])]
    run(hip, Trees(rng, seqs, 2, 64, 16, kv, max_ctx=max_ctx, ahead=2, behind=3), 6, rng)


@KINDS
@pytest.mark.parametrize("G", [1, 16])
@pytest.mark.parametrize("max_ctx", [None, 5000])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_values_not_attended_to(hip, kv, G, max_ctx, what):
    """No numbers at nodes of other paths, behind the tree and in pages of no sequence reach nobody; rows that attend
    to one show it."""
    rng = np.random.default_rng(7)
    seqs = [(45, tree(rng, 12)), (300, [m | 1 for m in tree(rng, 20)])]
    c = Trees(rng, seqs, 1, 128 if G == 16 else 64, 16, kv, max_ctx=max_ctx)
    bad = [(0, 45 + 7), (1, 300 + 3), (1, 300 + 11)]
    for s, t in bad:
        c.poison(s, t, what, k=True, v=True)
    for s in range(2):  # behind the tree's last node, in its last page
        end = int(c.base[s]) + len(seqs[s][1])
        for t in range(end, min(-(-end // 16) * 16, c.max_ctx)):
            c.poison(s, t, what)
    spare = c.table[0, -1] if max_ctx else None
    if spare is not None:
        (c.K if kv != I8 else c.Ks)[spare] = what
        (c.V if kv != I8 else c.Vs)[spare] = what
    q = rng.standard_normal((c.n, G, c.hd)).astype(np.float32)
    call = Call(hip, c, q, G)
    call.launch()
    got = call.result()
    clean = {r for s, r in c.rows() if not any(s == b and t in c.sees(s, r) for b, t in bad)}
    assert 0 < len(clean) < c.n
    check(c, q, got, clean)
    for s, r in c.rows():
        if r not in clean and (kv != I8 or np.isnan(what)):  # (int8: a score of -inf is a weight of 0)
            assert not np.isfinite(got[r]).any()


@KINDS
@pytest.mark.parametrize("G", [1, 16])
def test_value_alone_is_no_number(hip, kv, G):
    """V of a node is infinite in one dimension: that dimension of the rows that attend to it, nothing else."""
    if kv == I8:
        pytest.skip("an int8 position has one scale for all dimensions")
    rng = np.random.default_rng(8)
    c = Trees(rng, [(70, tree(rng, 24))], 1, 64, 16, kv)
    p, o = c.at(0, 70 + 5)
    c.V[p, 0, o, 9] = np.inf
    q = rng.standard_normal((c.n, G, 64)).astype(np.float32)
    call = Call(hip, c, q, G)
    call.launch()
    got = call.result()
    hit = np.array([int(m) >> 5 & 1 for m in c.masks], bool)
    assert 0 < hit.sum() < c.n
    assert not np.isfinite(got[hit, :, 9]).any()
    c.V[p, 0, o, 9] = 0.0
    check(c, q, got, {r for r in range(c.n) if not hit[r]})
    assert np.isfinite(np.delete(got, 9, axis=2)).all()


@KINDS
def test_graph_follows_the_lengths(hip, kv):
    """A captured call, replayed with other bases and masks, the program's own calls between."""
    from qraf_amd.backend import Graph, Stream
    rng = np.random.default_rng(9)
    c = Trees(rng, [(900, tree(rng, 30)), (200, tree(rng, 34))], 2, 64, 16, kv)
    q = rng.standard_normal((c.n, 8, 64)).astype(np.float32)
    call, st = Call(hip, c, q, 8), Stream()
    call.launch(st.h)
    st.synchronize()
    g = Graph(st)
    with g:
        call.launch(st.h)
    for k in range(4):
        c.base = np.array([900 - 211 * k, 200 - 3 * k], np.int32)
        c.masks = np.array([m for n in (30, 34) for m in tree(rng, n)], np.uint64)
        call.base.upload(c.base)
        call.masks.upload(c.masks)
        call.out.upload(np.full((c.n, 8, 64), np.float32(0x7F)))
        g.launch()
        st.synchronize()
        got = call.result()
        check(c, q, got)
        call.launch()
        assert np.array_equal(call.result(), got)
    g.destroy()
    st.destroy()


def test_chain_is_causal_attention(hip):
    """A chain of drafts on f16 pages against group attention of the same rows."""
    rng = np.random.default_rng(10)
    n, base = 7, 333
    c = Trees(rng, [(base, [(1 << (i + 1)) - 1 for i in range(n)])], 2, 64, 16, F16)
    q = rng.standard_normal((n, 8, 64)).astype(np.float32)
    call = Call(hip, c, q, 8)
    call.launch()
    got = call.result()
    from qraf_amd.backend import DeviceBuffer
    up = DeviceBuffer.from_array
    table, ctx = up(np.repeat(c.table, n, 0)), up((base + 1 + np.arange(n)).astype(np.int32))
    starts, prefix = up(np.array([0, n], np.int32)), up(np.array([base + n], np.int32))
    size = hip.lib.qraf_hip_group_attention_workspace_bytes(n, 1, 8, 2, 64, c.max_ctx)
    ws, out = DeviceBuffer(size), up(np.zeros_like(q))
    hip._lib.call("qraf_hip_group_attention_dev", call.q.ptr, call.k.ptr, call.v.ptr, F16, table.ptr, c.wide, ctx.ptr,
                  starts.ptr, prefix.ptr, n, 1, 8, 2, 64, 16, 0.125, c.max_ctx, out.ptr, ws.ptr, size, None)
    hip._lib.call("qraf_hip_device_synchronize")
    check(c, q, out.download(np.float32, q.size).reshape(q.shape))
    check(c, q, got)

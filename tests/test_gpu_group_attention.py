"""Attention of rows that share the first positions of their caches
(qraf_hip_group_attention_dev) against the softmax of its definition in 64 bits.

Tolerance, per output element: scores are sums of head_dim products whose
operands keep at least 21 bits, so they are off by at most
    d = scale * sum_d |q_d k_d| * (2^-20 + head_dim * 2^-24),
which moves every probability by a factor within exp(+-2 d); and the weighted sum
and its divisor are chains of at most ctx + 64 fp32 additions:
    |got - want| <= (2 max_t d + (ctx + 64) * 2^-24) * sum_t p_t |v_t| + ctx * 2^-37 * max_t |v_t| + 1e-30.
The last but one: a weight enters its product as two fp16 values, times 2^14 (the largest weight is at most 1, and
at least one is 1).  fp16 has steps of 2^-24 at its least, so a weight is off by up to 2^-38 however small it is;
int8 pages multiply it by the position's V scale over a power of two that may be twice the largest scale, which
makes that 2^-37 of the largest |v| for each of ctx positions.  (f32 V is held in steps of 2^-40 of the largest.)
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F32, F16, I8 = 0, 1, 102
KINDS = pytest.mark.parametrize("kv", [F32, F16, I8], ids=["f32", "f16", "i8"])


class Cache:
    """Pages in logical form [page][kv head][position][dim] (int8: with a scale per position), tables and layout.

    groups: a list of (prefix, [ctx of each row]); rows of a group have the pages of the first `prefix` positions
    in common, and where the prefix ends inside a page each row has a copy of it."""

    def __init__(self, rng, groups, Hkv, hd, ps, kv, spare=3, behind=0, only_first=False):
        self.kv, self.ps, self.hd, self.Hkv = kv, ps, hd, Hkv
        self.ctx = np.array([c for _, cs in groups for c in cs] + [1] * behind, np.int32)
        self.starts = np.cumsum([0] + [len(cs) for _, cs in groups]).astype(np.int32)
        self.prefix = np.array([p for p, _ in groups], np.int32)
        n = self.ctx.size
        longest = max(1, int(self.ctx.max()), int(self.prefix.max()))
        self.max_ctx = longest
        self.table = np.zeros((n, -(-longest // ps)), np.int32)
        plan, count = [], 0
        for g, (p, cs) in enumerate(groups):
            if not cs:
                continue
            rows = range(self.starts[g], self.starts[g + 1])
            most = max(cs)
            common = -(-min(p, most) // ps)
            shared = list(range(count, count + common))
            count += common
            for r in rows:
                first = r == self.starts[g]
                for j in range(-(-max(int(self.ctx[r]), min(p, most) if first else 0) // ps)):
                    if (j + 1) * ps <= p or (first and j < common) or self.ctx[r] <= p:
                        plan.append((r, j, shared[j], None))  # wholly inside the prefix
                    else:
                        copy = shared[j] if j * ps < p else None
                        plan.append((r, j, count, copy))
                        count += 1
        for r in range(n - behind, n):
            plan.append((r, 0, count, None))
            count += 1
        perm = rng.permutation(count + spare)
        shape = (count + spare, Hkv, ps, hd)
        if kv == I8:
            self.K, self.V = (rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2))
            self.Ks, self.Vs = (rng.uniform(0.01, 0.04, shape[:3]).astype(np.float32) for _ in range(2))
        else:
            dt = np.float16 if kv == F16 else np.float32
            self.K, self.V = (rng.standard_normal(shape).astype(dt) for _ in range(2))
            self.Ks = self.Vs = None
        for r, j, page, copy in plan:
            self.table[r, j] = perm[page]
            if copy is not None:
                keep = int(self.prefix[np.searchsorted(self.starts, r, side="right") - 1]) - j * ps
                for a in (self.K, self.V, self.Ks, self.Vs):
                    if a is not None:
                        a[perm[page], :, :keep] = a[perm[copy], :, :keep]
        if only_first:  # the other rows' tables name a page of NaN in the prefix
            decoy = perm[count]
            for a in ((self.K, self.V) if kv != I8 else (self.Ks, self.Vs)):
                a[decoy] = np.nan
            for g in range(len(groups)):
                for r in range(self.starts[g] + 1, self.starts[g + 1]):
                    self.table[r, :int(self.prefix[g]) // ps] = decoy
        self.n = n

    def table_row(self, r):
        """Row r's pages, those of the prefix taken from its group's first row."""
        g = int(np.searchsorted(self.starts, r, side="right") - 1)
        t = self.table[r].copy()
        if g < len(self.prefix) and r < self.starts[-1]:
            whole = int(self.prefix[g]) // self.ps
            t[:whole] = self.table[self.starts[g], :whole]
            if self.ctx[r] <= self.prefix[g]:
                t[:] = self.table[self.starts[g]]
        return t

    def values(self, r):
        """(K, V) [kv head][ctx][dim] of row r in 64 bits."""
        c = int(self.ctx[r])
        t = np.arange(c)
        pages, off = self.table_row(r)[t // self.ps], t % self.ps
        out = []
        for a, s in ((self.K, self.Ks), (self.V, self.Vs)):
            x = a[pages, :, off].astype(np.float64)
            if s is not None:
                x = x * s[pages, :, off].astype(np.float64)[..., None]
            out.append(x.transpose(1, 0, 2))
        return out

    def device(self):
        """The two pools as the library's pages."""
        def pool(a, s, v):
            x = a.transpose(0, 1, 3, 2) if v and self.kv != F32 else a
            x = np.ascontiguousarray(x)
            if s is None:
                return x
            p = x.shape[0] * x.shape[1]
            return np.concatenate([x.reshape(p, -1).view(np.uint8),
                                   np.ascontiguousarray(s).reshape(p, -1).view(np.uint8)], 1)
        return pool(self.K, self.Ks, False), pool(self.V, self.Vs, True)


class Call:
    """One call's device buffers."""

    def __init__(self, hip, cache, q, H, n_groups=None, fill=0x7F):
        from qraf_amd.backend import DeviceBuffer
        c = self.c = cache
        self.hip, self.H = hip, H
        k, v = c.device()
        up = DeviceBuffer.from_array
        self.q, self.k, self.v, self.table, self.ctx = up(q), up(k), up(v), up(c.table), up(c.ctx)
        self.starts, self.prefix = up(c.starts), up(c.prefix)
        self.groups = len(c.prefix)
        self.ws_bytes = hip.lib.qraf_hip_group_attention_workspace_bytes(c.n, self.groups, H, c.Hkv, c.hd, c.max_ctx)
        self.ws = up(np.full(self.ws_bytes, 0xFF, np.uint8))  # needs no initialisation: NaN in every float of it
        self.out = up(np.full((c.n, H, c.hd), np.float32(fill)))

    def launch(self, stream=None):
        c = self.c
        self.hip._lib.call("qraf_hip_group_attention_dev", self.q.ptr, self.k.ptr, self.v.ptr, c.kv, self.table.ptr,
                           c.table.shape[1], self.ctx.ptr, self.starts.ptr, self.prefix.ptr, c.n, self.groups, self.H,
                           c.Hkv, c.hd, c.ps, np.float32(1 / np.sqrt(c.hd)), c.max_ctx, self.out.ptr, self.ws.ptr,
                           self.ws_bytes, stream)

    def result(self, stream=None):
        self.hip._lib.call("qraf_hip_stream_synchronize", stream)
        return self.out.download(np.float32, self.c.n * self.H * self.c.hd).reshape(self.c.n, self.H, self.c.hd)

    def run(self):
        self.launch()
        return self.result()


def expected(c, q, H):
    """(output, tolerance) in 64 bits; NaN tolerance outside every group."""
    out, tol = np.zeros((c.n, H, c.hd)), np.full((c.n, H, c.hd), 1e-30)
    scale, per = float(np.float32(1 / np.sqrt(c.hd))), H // c.Hkv
    tol[c.starts[-1]:] = np.nan
    for r in range(c.starts[0], c.starts[-1]):
        n = int(c.ctx[r])
        if n == 0:
            continue
        K, V = c.values(r)
        for h in range(H):
            k, v, x = K[h // per], V[h // per], q[r, h].astype(np.float64)
            s = k @ x * scale
            d = scale * (np.abs(k) @ np.abs(x)) * (2.0 ** -20 + c.hd * 2.0 ** -24)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[r, h] = p @ v
            tol[r, h] += (2 * d.max() + (n + 64) * 2.0 ** -24) * (p @ np.abs(v)) + n * 2.0 ** -37 * np.abs(v).max()
    return out, tol


def check(c, got, q, H, fill=0x7F):
    want, tol = expected(c, q, H)
    outside = np.isnan(tol)
    assert np.all(got[outside] == fill), "a row outside every group was written"
    err = np.abs(got.astype(np.float64) - want)
    bad = ~outside & ~(err <= tol)
    assert not bad.any(), f"{bad.sum()} off, first {np.argwhere(bad)[0]}, worst {np.nanmax(err / tol):.2f} tolerances"


def queries(rng, n, H, hd):
    return (rng.standard_normal((n, H, hd)) * rng.choice([0.25, 1.0, 2.5], (n, H, 1))).astype(np.float32)


# (H, Hkv, hd)
HEADS = [(9, 3, 64), (16, 2, 128), (4, 4, 128), (14, 2, 64), (16, 1, 128), (5, 1, 64), (8, 8, 64), (20, 1, 64)]
# (prefix, ctx of each row) of each group
LAYOUTS = {
    "one row of one position": [(1, [1])],
    "no prefix": [(0, [1, 17, 300])],
    "drafts of one sequence": [(205, [201, 202, 203, 204, 205])],
    "drafts of several": [(33, [31, 32, 33]), (7, [7]), (512, [509, 510, 511, 512]), (64, [63, 64])],
    "prompt with tails": [(96, [97, 130, 96, 400, 111])],
    "prompt ends inside a page": [(77, [78, 200, 77, 81]), (5, [6, 40])],
    "rows shorter than the prefix": [(300, [1, 16, 0, 299, 300, 301, 40])],
    "empty rows and groups": [(0, [0, 0]), (50, []), (10, [0, 12]), (40, [])],
    "chunk": [(70, list(range(1, 71)))],
    "many rows": [(130, [130 + (7 * i) % 50 for i in range(90)])],
}


@pytest.mark.parametrize("layout", LAYOUTS.values(), ids=list(LAYOUTS))
@pytest.mark.parametrize("heads", HEADS, ids=["%dx%dx%d" % h for h in HEADS])
@KINDS
def test_layouts(hip, kv, heads, layout):
    H, Hkv, hd = heads
    rng = np.random.default_rng(H * 1000 + hd + kv)
    c = Cache(rng, layout, Hkv, hd, 16, kv)
    q = queries(rng, c.n, H, hd)
    check(c, Call(hip, c, q, H).run(), q, H)


@pytest.mark.parametrize("ps", [1, 3, 4, 8, 32, 64, 100, 256])
@KINDS
def test_page_sizes(hip, kv, ps):
    H, Hkv, hd = 6, 2, 64
    rng = np.random.default_rng(ps)
    c = Cache(rng, [(101, [102, 150, 90]), (300, [298, 299, 300]), (9, [10])], Hkv, hd, ps, kv)
    q = queries(rng, c.n, H, hd)
    check(c, Call(hip, c, q, H).run(), q, H)


@pytest.mark.parametrize("heads", [(4, 2, 16), (8, 1, 32), (3, 3, 32), (6, 2, 16)])
@KINDS
def test_small_heads(hip, kv, heads):
    H, Hkv, hd = heads
    rng = np.random.default_rng(hd)
    c = Cache(rng, [(40, [41, 100, 40, 0]), (270, [268, 269, 270])], Hkv, hd, 16, kv)
    q = queries(rng, c.n, H, hd)
    check(c, Call(hip, c, q, H).run(), q, H)


@KINDS
def test_long_ragged_groups(hip, kv):
    H, Hkv, hd = 16, 2, 128
    rng = np.random.default_rng(11)
    c = Cache(rng, [(4001, [4001 + int(x) for x in rng.integers(0, 300, 20)]), (1290, list(range(1281, 1291))),
                    (2048, [2048] * 3), (17, [3000])], Hkv, hd, 16, kv)
    q = queries(rng, c.n, H, hd)
    call = Call(hip, c, q, H)
    first = call.run()
    check(c, first, q, H)
    for _ in range(3):
        assert np.array_equal(call.run(), first), "results differ from call to call"


@KINDS
def test_most_rows(hip, kv):
    """1,024 rows: a group of many, groups of one row each, a chunk."""
    H, Hkv, hd = 3, 1, 64
    rng = np.random.default_rng(12)
    groups = [(64, [64 + i % 9 for i in range(500)])] + [(i % 40, [i % 40 + 1]) for i in range(268)]
    groups.append((256, list(range(1, 257))))
    c = Cache(rng, groups, Hkv, hd, 16, kv)
    assert c.n == 1024
    q = queries(rng, c.n, H, hd)
    check(c, Call(hip, c, q, H).run(), q, H)


@KINDS
def test_prefix_pages_come_from_the_first_row(hip, kv):
    H, Hkv, hd = 8, 2, 64
    rng = np.random.default_rng(13)
    c = Cache(rng, [(100, [100, 130, 101, 333]), (64, [64, 65])], Hkv, hd, 16, kv, only_first=True)
    q = queries(rng, c.n, H, hd)
    check(c, Call(hip, c, q, H).run(), q, H)


@KINDS
def test_rows_outside_the_groups_are_left(hip, kv):
    H, Hkv, hd = 4, 2, 64
    rng = np.random.default_rng(14)
    c = Cache(rng, [(30, [31, 35]), (8, [8])], Hkv, hd, 16, kv, behind=5)
    q = queries(rng, c.n, H, hd)
    check(c, Call(hip, c, q, H).run(), q, H)


@pytest.mark.parametrize("hd", [64, 128])
@KINDS
def test_contents_behind_a_context_never_matter(hip, kv, hd):
    """NaN in the positions behind each sequence's last, inside its last page."""
    H, Hkv, ps = 8, 2, 32
    rng = np.random.default_rng(15)
    c = Cache(rng, [(77, [78, 100, 77]), (50, [47, 48, 49, 50]), (3, [3])], Hkv, hd, ps, kv)
    q = queries(rng, c.n, H, hd)
    ends = {}
    for r in range(c.n):
        t = int(c.ctx[r]) - 1
        page = c.table[r, t // ps]
        ends[page] = max(ends.get(page, 0), t % ps + 1)
    for r in range(c.n):  # pages of a longer row are used up to its own end
        for t in range(int(c.ctx[r])):
            page = c.table_row(r)[t // ps]
            ends[page] = max(ends.get(page, 0), t % ps + 1)
    for page, e in ends.items():
        for a in ([c.Ks, c.Vs] if kv == I8 else [c.K, c.V]):
            a[page, :, e:] = np.nan
    check(c, Call(hip, c, q, H).run(), q, H)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("hd", [64, 128])
@KINDS
def test_what_a_row_does_not_attend_to_never_reaches_it(hip, kv, hd, bad):
    """A position of the prefix whose K or V is not a number reaches the rows that attend to it and no others."""
    H, Hkv, ps, at = 8, 2, 16, 70
    rng = np.random.default_rng(16)
    ctx = [60, 69, 70, 71, 72, 90, 10]
    for part in ("K", "V"):
        c = Cache(rng, [(90, ctx)], Hkv, hd, ps, kv)
        q = queries(rng, c.n, H, hd)
        want, tol = expected(c, q, H)
        a = getattr(c, part + "s") if kv == I8 else getattr(c, part)
        a[c.table[5, at // ps], :, at % ps] = bad
        got = Call(hip, c, q, H).run()
        for r, n in enumerate(ctx):
            if n <= at:
                assert np.all(np.abs(got[r] - want[r]) <= tol[r]), (part, r)
            elif part == "V" and not (kv == I8 and np.isinf(bad)):
                assert not np.isfinite(got[r]).any(), (part, r)


@KINDS
def test_extreme_scores(hip, kv):
    """Scores far apart and all equal: the running maximum carries the sums."""
    H, Hkv, hd = 4, 2, 64
    rng = np.random.default_rng(17)
    c = Cache(rng, [(130, [131, 260, 130])], Hkv, hd, 16, kv)
    for factor in (0.0, 40.0):
        q = (queries(rng, c.n, H, hd) * factor).astype(np.float32)
        check(c, Call(hip, c, q, H).run(), q, H)


def test_tiny_and_huge_values(hip):
    """f32 pages keep fp32's range: V of 1e-30 and 1e30 in one cache, K beyond fp16."""
    H, Hkv, hd = 4, 2, 64
    rng = np.random.default_rng(18)
    c = Cache(rng, [(50, [51, 90, 50])], Hkv, hd, 16, F32)
    c.K *= np.float32(1e6)
    q = (queries(rng, c.n, H, hd) * 1e-6).astype(np.float32)
    for f in (1e-30, 1e30):
        c.V = (rng.standard_normal(c.V.shape) * f).astype(np.float32)
        c2 = Cache(np.random.default_rng(18), [(50, [51, 90, 50])], Hkv, hd, 16, F32)
        c2.K, c2.V = c.K, c.V
        for r in range(c2.n):  # the copies of the page in which the prefix ends
            j = 50 // 16
            c2.V[c2.table[r, j], :, :50 % 16] = c2.V[c2.table[0, j], :, :50 % 16]
            c2.K[c2.table[r, j], :, :50 % 16] = c2.K[c2.table[0, j], :, :50 % 16]
        got = Call(hip, c2, q, H).run()
        want, tol = expected(c2, q, H)
        assert np.all(np.abs(got - want) <= tol + 1e-37)


@KINDS
def test_captured_and_replayed(hip, kv):
    """Lengths, groups and caches are read when the graph runs: replays on changed contents equal eager calls."""
    from qraf_amd.backend import Graph, Stream
    H, Hkv, hd = 8, 2, 128
    rng = np.random.default_rng(19)
    c = Cache(rng, [(300, [301, 390, 300]), (200, [197, 198, 199, 200])], Hkv, hd, 16, kv)
    q = queries(rng, c.n, H, hd)
    call, s = Call(hip, c, q, H), Stream()
    g = Graph(s)
    with g:
        call.launch(s.h)
    for step in range(4):
        q = queries(rng, c.n, H, hd)
        if step:
            c.ctx = np.maximum(0, c.ctx - rng.integers(0, 40, c.n)).astype(np.int32)
        call.q.upload(q)
        call.ctx.upload(c.ctx)
        call.out.zero()
        g.launch()
        replayed = call.result(s.h)
        call.out.zero()
        assert np.array_equal(call.run(), replayed)
        check(c, replayed, q, H)
    g.destroy()
    s.destroy()


@KINDS
def test_two_streams(hip, kv):
    """Calls with workspaces of their own on two streams at once."""
    from qraf_amd.backend import Stream
    rng = np.random.default_rng(20)
    calls = []
    for i in range(2):
        c = Cache(rng, [(500 + i, [501 + i, 700, 502]), (90, list(range(80, 91)))], 2, 64, 16, kv)
        q = queries(rng, c.n, 8, 64)
        calls.append((c, q, Call(hip, c, q, 8), Stream()))
    for _ in range(5):
        for _, _, call, s in calls:
            call.launch(s.h)
    for c, q, call, s in calls:
        check(c, call.result(s.h), q, 8)
        s.destroy()


def test_offsets_beyond_32_bits(hip):
    """Pages whose byte offsets pass 2^32 (fp16 pools of 4.5 GiB)."""
    from qraf_amd.backend import DeviceBuffer
    H, Hkv, hd, ps = 16, 8, 128, 16
    rng = np.random.default_rng(21)
    c = Cache(rng, [(40, [41, 60]), (20, [19, 20])], Hkv, hd, ps, F16)
    q = queries(rng, c.n, H, hd)
    call = Call(hip, c, q, H)
    k, v = c.device()
    page = k[0].nbytes
    pages = (9 << 29) // page
    far = pages - 1 - np.arange(k.shape[0])
    big = []
    for pool in (k, v):
        b = DeviceBuffer(pages * page)
        for i, at in enumerate(far):
            b.upload(pool[i], int(at) * page)
        big.append(b)
    assert far.min() * page > 1 << 32
    call.k, call.v = big
    call.table.upload(far[c.table].astype(np.int32))
    check(c, call.run(), q, H)


def test_agrees_with_paged_attention(hip):
    """The same rows through qraf_hip_paged_attention_dev."""
    from qraf_amd.backend import DeviceBuffer
    H, Hkv, hd = 16, 2, 128
    rng = np.random.default_rng(22)
    c = Cache(rng, [(600, [601, 900, 600, 755])], Hkv, hd, 16, F16)
    q = queries(rng, c.n, H, hd)
    call = Call(hip, c, q, H)
    got = call.run()
    need = hip.lib.qraf_hip_attention_workspace_bytes(c.n, H, Hkv, hd, c.max_ctx)
    ws, out = DeviceBuffer(need), DeviceBuffer(got.nbytes)
    hip._lib.call("qraf_hip_paged_attention_dev", call.q.ptr, call.k.ptr, call.v.ptr, F16, call.table.ptr,
                  c.table.shape[1], call.ctx.ptr, c.n, H, Hkv, hd, 16, np.float32(1 / np.sqrt(hd)), c.max_ctx, out.ptr,
                  ws.ptr, need, None)
    hip._lib.call("qraf_hip_stream_synchronize", None)
    other = out.download(np.float32, got.size).reshape(got.shape)
    _, tol = expected(c, q, H)
    assert np.all(np.abs(got - other) <= 2 * tol)

"""qraf_hip_group_attention_dev where the values of a cache lie far apart: positions that a row does not attend to, or
hardly attends to, change nothing in what it makes of the others.

Tolerance, per output element, p_t the softmax in 64 bits, kmax_t and vmax_t the largest magnitudes of position t's K
and V, w = max_t p_t vmax_t.  f32 and int8 operands enter fp16 products as two values, hi + lo, over a power of two:
22 bits of a value, in steps of 2^-24 at the least.
  K: the power of two brings the largest of 32 positions into [2^14, 2^15), or each position's where one of them lies
     2^-14 below it.  So a step is at most 2^-24 2^-14 2^14 kmax_t = 2^-24 kmax_t, and half of one is what is lost.
  q: over the query's own largest, 2^-39 of it.
  Powers of two end at 2^110: a q, K or V is off by 2^-25 2^-110 = 2^-135 at the least (values below 1e-33 have fewer
     bits: 3e-39 has 2^-7 of itself).
  scores: sums of hd products of two operands of at least 21 bits, in fp32:
     d_t = scale (sum_d |q k| (2^-20 + hd 2^-24) + (2^-24 kmax_t + 2^-135) sum_d |q| + (2^-38 qmax + 2^-135) sum_d |k|)
  weights: off by the factor exp(+-(d_t + D)), D = sum_t p_t d_t, and by 2^-22.
  V: as K, so 2^-22 of a value and 2^-25 vmax_t.  Its power of two is taken out of the weight, which enters over one of
     its own for each column: the largest weighted value of 32 positions, at most 2^14 over the true one, lies above
     2^11 2^14 there, and a step of the weight times V is at most 2^-24 2^15: n 2^-24 2^15 2^-25 2^14 w = n 2^-20 w.
  |got - want| <= sum_t p_t |v_t| (expm1(d_t + D) + (n + 64) 2^-24 + 2^-20) + 2^-24 sum_t p_t vmax_t + n 2^-20 w + 1e-37
(n: the fp32 sums of weights and outputs.)"""
import numpy as np
import pytest

from tests import test_gpu_group_attention as calls

pytestmark = pytest.mark.gpu
F32, F16, I8 = calls.F32, calls.F16, calls.I8
HEADS = pytest.mark.parametrize("heads", [(16, 2, 128), (9, 3, 64), (20, 1, 64)], ids=["16x2x128", "9x3x64", "20x1x64"])
FORMS = pytest.mark.parametrize("wide", [False, True], ids=["bound", "planned"])
WIDE = [(F32, 16), (F32, 32), (I8, 16)]  # page types that hold values this far apart, page sizes
PAGES = pytest.mark.parametrize("kv,ps", WIDE, ids=["f32-16", "f32-32", "i8-16"])


class Cache(calls.Cache):
    """Positions below the prefix are the first row's, whatever the row's own page holds there."""

    def __init__(self, rng, groups, Hkv, hd, ps, kv, wide):
        super().__init__(rng, groups, Hkv, hd, ps, kv)
        if wide:  # a long bound takes the planned form
            self.max_ctx = max(self.max_ctx, 2048)
            table = np.zeros((self.n, -(-self.max_ctx // ps)), np.int32)
            table[:, :self.table.shape[1]] = self.table
            self.table = table

    def place(self, r, t):
        """(page, offset) that row r reads position t from."""
        g = int(np.searchsorted(self.starts, r, side="right") - 1)
        row = np.where(t < self.prefix[g], self.starts[g], r)
        return self.table[row, t // self.ps], t % self.ps

    def values(self, r):
        page, off = self.place(r, np.arange(int(self.ctx[r])))
        out = []
        for a, s in ((self.K, self.Ks), (self.V, self.Vs)):
            x = a[page, :, off].astype(np.float64)
            if s is not None:
                x = x * s[page, :, off].astype(np.float64)[..., None]
            out.append(x.transpose(1, 0, 2))
        return out

    def scale(self, which, r, t, by):
        """Multiplies K or V (int8 pages: its scale) of position t of row r."""
        page, off = self.place(r, np.asarray(t))
        a = getattr(self, which + "s") if self.kv == I8 else getattr(self, which)
        a[page, :, off] *= np.float32(by)


def expected(c, q, H):
    out, tol = np.zeros((c.n, H, c.hd)), np.full((c.n, H, c.hd), 1e-37)
    scale, per = float(np.float32(1 / np.sqrt(c.hd))), H // c.Hkv
    for r in range(c.n):
        n = int(c.ctx[r])
        if n == 0:
            continue
        K, V = c.values(r)
        for h in range(H):
            k, v, x = K[h // per], V[h // per], q[r, h].astype(np.float64)
            s = k @ x * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            d = scale * ((np.abs(k) @ np.abs(x)) * (2.0 ** -20 + c.hd * 2.0 ** -24) +
                         (2.0 ** -24 * np.abs(k).max(1) + 2.0 ** -135) * np.abs(x).sum() +
                         (2.0 ** -38 * np.abs(x).max() + 2.0 ** -135) * np.abs(k).sum(1))
            D = (p * d).sum()
            assert D < 0.1, "the case leaves its own weights open"
            grow = np.where(p > 0, np.expm1(np.minimum(d + D, 600)), 0)
            vmax = np.abs(v).max(1)
            out[r, h] = p @ v
            tol[r, h] += ((p * (grow + (n + 64) * 2.0 ** -24 + 2.0 ** -20)) @ np.abs(v) +
                          2.0 ** -24 * (p @ vmax) + n * 2.0 ** -20 * (p * vmax).max())
    return out, tol


def check(hip, c, q, H, rows=None):
    got = calls.Call(hip, c, q, H).run().astype(np.float64)
    keep = slice(None) if rows is None else rows
    if rows is not None:  # the others are not looked at: their oracle need not be either
        c.ctx = np.where(np.isin(np.arange(c.n), rows), c.ctx, 0).astype(np.int32)
    want, tol = expected(c, q, H)
    err = np.abs(got - want)[keep]
    bad = ~(err <= tol[keep])
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, first {np.argwhere(bad)[0]}, worst {(err / tol[keep]).max():.2f} tolerances"


@FORMS
@pytest.mark.parametrize("word", [1e13, 3e37])
@pytest.mark.parametrize("kv,ps", WIDE + [(F16, 16)], ids=["f32-16", "f32-32", "i8-16", "f16-16"])
@HEADS
def test_words_of_an_own_page_below_the_prefix(hip, heads, kv, ps, word, wide):
    """Where a prefix ends inside a page, the first positions of a row's own page are never written by it."""
    H, Hkv, hd = heads
    rng = np.random.default_rng(H)
    c = Cache(rng, [(77, [78, 200, 77, 81, 80]), (5, [6, 40, 300])] + [(9, [12 + i for i in range(30)])] * wide, Hkv, hd,
              ps, kv, wide)
    q = calls.queries(rng, c.n, H, hd)
    for r in range(c.n):
        g = int(np.searchsorted(c.starts, r, side="right") - 1)
        p = int(c.prefix[g])
        if r != c.starts[g] and c.ctx[r] > p:
            for a in (c.K, c.V) if kv != I8 else (c.Ks, c.Vs):
                a[c.table[r, p // ps], :, :p % ps] = min(word, 6e4) if kv == F16 else word
    check(hip, c, q, H)


@FORMS
@pytest.mark.parametrize("which", ["K", "V"])
@PAGES
@HEADS
def test_values_of_positions_that_other_rows_attend_to(hip, heads, kv, ps, which, wide):
    """Chunks and drafts: one position's K or V is 1e13 times the others'.  (Rows that attend to such a K give it all
    their weight or none: only the rows that end ahead of it are looked at.)"""
    H, Hkv, hd = heads
    rng = np.random.default_rng(H + 1)
    chunk, at = list(range(101, 141)), (103, 119, 128, 139)
    for t in at:
        c = Cache(rng, [(140, chunk), (205, [201, 202, 203, 204, 205]), (33, [60, 40])], Hkv, hd, ps, kv, wide)
        q = calls.queries(rng, c.n, H, hd)
        c.scale(which, 0, t, 1e13)
        c.scale(which, 40, 203, 1e13)
        c.scale(which, 45, 50, 1e13)
        short = [r for r in range(40) if c.ctx[r] <= t] + [r for r in range(40, 45) if c.ctx[r] <= 203] + [46]
        check(hip, c, q, H, short if which == "K" else None)


def aim(c, q, H, r, t, score):
    """K of position t such that the row's scores there are about `score`: along a query that all heads share."""
    page, off = c.place(r, np.asarray(t))
    x = q[r, 0].astype(np.float64)
    k = score * np.sqrt(c.hd) * x / (x @ x)
    if c.kv == I8:
        s = np.abs(k).max() / 127
        c.K[page, :, off] = np.round(k / s).astype(np.int8) if s > 0 else 0
        c.Ks[page, :, off] = s
    else:
        c.K[page, :, off] = k.astype(np.float32)


@FORMS
@pytest.mark.parametrize("rows", [3, 40])
@pytest.mark.parametrize("places", [(0,), (31,), (40, 41), (0, 33, 70, 99)], ids=str)
@PAGES
@HEADS
def test_large_values_of_hardly_any_weight(hip, heads, kv, ps, places, rows, wide):
    """V of 1e20 where the score is 75 below the others' (a weight of e^-75: 3e-13 of the output), first, in the middle,
    in neighbouring positions: the sums go on in the others' range."""
    H, Hkv, hd = heads
    rng = np.random.default_rng(H + 2)
    c = Cache(rng, [(100, [100 + i % 3 for i in range(rows)])], Hkv, hd, ps, kv, wide)
    q = np.repeat(np.repeat(rng.standard_normal((1, 1, hd)), H, 1), rows, 0).astype(np.float32)
    for t in places:
        aim(c, q, H, 0, t, -75.0)
        c.scale("V", 0, t, 1e20)
    check(hip, c, q, H)


@FORMS
@pytest.mark.parametrize("rows", [3, 40])
@pytest.mark.parametrize("rise", [1, -1], ids=["rising", "falling"])
@PAGES
@HEADS
def test_scores_and_values_that_run_against_each_other(hip, heads, kv, ps, rise, rows, wide):
    """Tile by tile the scores rise by 12 to 20 and V falls by 1e6, and the other way round."""
    H, Hkv, hd = heads
    rng = np.random.default_rng(H + 3)
    n = 300
    c = Cache(rng, [(n, [n - i % 3 for i in range(rows)])], Hkv, hd, ps, kv, wide)
    q = np.repeat(np.repeat(rng.standard_normal((1, 1, hd)), H, 1), rows, 0).astype(np.float32)
    for t in range(n):
        tile = t // 32 if rise > 0 else 9 - t // 32
        aim(c, q, H, 0, t, 16.0 * tile - 80 + float(rng.uniform(-2, 2)))
        c.scale("V", 0, t, 10.0 ** (6 * (4 - tile)))
    check(hip, c, q, H)


@FORMS
@pytest.mark.parametrize("rows", [3, 40])
@HEADS
def test_every_position_in_a_range_of_its_own(hip, heads, rows, wide):
    H, Hkv, hd = heads
    rng = np.random.default_rng(H + 4)
    c = Cache(rng, [(150, [150 - i for i in range(rows)]), (64, [70] * rows)], Hkv, hd, 16, F32, wide)
    c.K *= np.exp2(rng.integers(-90, 2, c.K.shape[:3] + (1,))).astype(np.float32)
    c.V *= np.exp2(rng.integers(-100, 100, c.V.shape[:3] + (1,))).astype(np.float32)
    q = calls.queries(rng, c.n, H, hd)
    check(hip, c, q, H)


@FORMS
@pytest.mark.parametrize("rows", [3, 40])
@HEADS
def test_values_next_to_the_largest(hip, heads, rows, wide):
    """K, q and V whose largest values pass 2^126, products within fp32's range."""
    H, Hkv, hd = heads
    rng = np.random.default_rng(H + 5)
    layout = [(30, [30 - i % 5 for i in range(rows)]), (1, [1, 1]), (3, [1, 2])]
    c = Cache(rng, layout, Hkv, hd, 16, F32, wide)
    q = calls.queries(rng, c.n, H, hd)
    c.V = (rng.uniform(-1, 1, c.V.shape) * 1e36).astype(np.float32)
    c.V[c.place(rows, np.asarray(0))[0]] *= np.float32(340)  # one position, of two rows: the output is its V
    assert np.isfinite(c.V).all()
    check(hip, c, q, H)
    big, tiny = np.float32(3.3e38), np.float32(1e-38)
    for k, x in ((big, tiny), (tiny, big)):
        c = Cache(rng, layout, Hkv, hd, 16, F32, wide)
        c.K = np.clip(c.K / 5, -1, 1) * k
        q2 = np.clip(q / 10, -1, 1) * x
        check(hip, c, q2.astype(np.float32), H)

"""Log probabilities, ranks, entropies and top alternatives (qraf_hip_token_logprobs_dev) against their definitions in
64 bits.

Ranks and alternatives are equal.  Log probabilities and entropies are within 2^-19 (1 + |value|): an exponential is
off by 2^-22 of itself and by the rounding of its argument, |d| e^d 2^-24 < 2^-25 of the row's largest; terms are
summed in 32 bits in trees of at most 14 steps, 2^-24 each, and from there in 64.  So S and sum exp(d) |d| are off by
less than 19 * 2^-24 of themselves, ln S by less than 2^-19.7, and the entropy, the sum of ln S and their quotient, both
at least 0, by less than 2^-19.7 (1 + its size).  The last rounding is 2^-24 of the value, and takes one past fp32's range (logits 6e38 apart) to -inf: the nearest fp32 value of anything
below -(2 - 2^-24) 2^127.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def call(hip, x, tokens, top, want=(True, True, True), stream=None, offset=0):
    """offset: floats ahead of the logits in their buffer."""
    from qraf_amd.backend import DeviceBuffer
    rows, V = x.shape
    d_x = DeviceBuffer.from_array(np.concatenate([np.zeros(offset, np.float32), x.reshape(-1)]))
    d_t = DeviceBuffer.from_array(np.asarray(tokens, np.uint32)) if tokens is not None else None
    outs = [DeviceBuffer.from_array(np.full(rows, 77, t)) if w else None
            for w, t in zip(want, (np.float32, np.int32, np.float32))]
    tops = [DeviceBuffer.from_array(np.full(rows * top, 77, t)) if top else None for t in (np.uint32, np.float32)]
    size = hip.lib.qraf_hip_token_logprobs_workspace_bytes(rows, V, top)
    ws = DeviceBuffer.from_array(np.full(size, 0xFF, np.uint8))
    p = lambda b: b.ptr if b is not None else None  # noqa: E731

    def launch(stream=None):
        hip._lib.call("qraf_hip_token_logprobs_dev", d_x.ptr + 4 * offset, rows, V, p(d_t), *(p(b) for b in outs), top,
                      *(p(b) for b in tops), ws.ptr, size, stream)

    def read():
        hip._lib.call("qraf_hip_device_synchronize")
        got = [b.download(t, rows) if b is not None else None
               for b, t in zip(outs, (np.float32, np.int32, np.float32))]
        return got + [b.download(t, rows * top).reshape(rows, top) if b is not None else None
                      for b, t in zip(tops, (np.uint32, np.float32))]
    launch(stream)
    return read(), launch, read, (d_x, d_t)


def near(got, want):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    want = np.where(want <= -(2 - 2.0 ** -24) * 2.0 ** 127, -np.inf, want)
    inf = ~np.isfinite(want)
    assert np.array_equal(got[inf], want[inf]), (got[inf], want[inf])
    err, tol = np.abs(got[~inf] - want[~inf]), 2.0 ** -19 * (1 + np.abs(want[~inf]))
    assert np.all(err <= tol), float((err / tol).max())


def check(got, x, tokens, top):
    lp, rank, ent, tt, tl = got
    for r in range(x.shape[0]):
        l = np.where(np.isnan(x[r]), -np.inf, x[r]).astype(np.float64) + 0.0
        V, m = l.size, l.max()
        order = np.argsort(-l, kind="stable")
        if m == -np.inf:
            p_log, H = np.full(V, -np.inf), 0.0
        else:
            with np.errstate(invalid="ignore"):
                d = np.where(l == m, 0.0, l - m)
            w = np.exp(d)
            p_log = d - np.log(w.sum())
            H = np.log(w.sum()) - (w * np.where(w > 0, d, 0.0)).sum() / w.sum()
        if tokens is not None:
            t = int(tokens[r])
            if lp is not None:
                near([lp[r]], [p_log[t] if t < V else -np.inf])
            if rank is not None:
                assert rank[r] == (int(np.nonzero(order == t)[0][0]) if t < V else -1)
        if ent is not None:
            near([ent[r]], [H])
        if top:
            assert np.array_equal(tt[r], order[:top])
            near(tl[r], p_log[order[:top]])


def logits(rng, rows, V):
    x = rng.standard_normal((rows, V)) * 1.5 + 10 * rng.random((rows, V)) ** 400
    return x.astype(np.float32)


SIZES = [(1, 1), (3, 2), (2, 63), (2, 64), (3, 65), (1, 255), (2, 257), (2, 1000), (1, 1023), (2, 1025), (3, 4097),
         (2, 8191), (1, 32000), (5, 49152), (2, 50257), (2, 100003), (3, 151936), (1, 163843)]


@pytest.mark.parametrize("rows,V", SIZES)
@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
def test_sizes(hip, rows, V, top):
    if top > V:
        pytest.skip("more alternatives than tokens")
    rng = np.random.default_rng(V + top)
    x, tokens = logits(rng, rows, V), rng.integers(0, V, rows)
    check(call(hip, x, tokens, top)[0], x, tokens, top)


@pytest.mark.parametrize("V", [2047, 2048, 2049, 8191, 8192, 8193, 16385, 131072, 524288])
@pytest.mark.parametrize("top", [0, 3, 64])
def test_where_the_form_changes(hip, V, top):
    """The last row of a form and the first of the next, one row and several."""
    rng = np.random.default_rng(V)
    for rows in (1, 9):
        if rows * V > 1 << 21:
            continue
        x, tokens = logits(rng, rows, V), rng.integers(0, V, rows)
        check(call(hip, x, tokens, top)[0], x, tokens, top)


@pytest.mark.parametrize("V", [5000, 8192, 300000])
def test_flat_rows(hip, V):
    """More equal logits at the border than the lists hold, the ties behind a few larger ones, at the end, everywhere."""
    rng = np.random.default_rng(V)
    x = np.full((4, V), 1.5, np.float32)
    x[0, rng.choice(V, 7, replace=False)] = 2 + rng.random(7)
    x[1, :V // 2] = -3.0
    x[2] = np.round(rng.standard_normal(V))
    x[3, V - 3:] = 9.0
    tokens = np.array([5, V - 1, 0, V - 2])
    for top in (1, 20, 64):
        check(call(hip, x, tokens, top)[0], x, tokens, top)


@pytest.mark.parametrize("V", [1000, 49152, 151936])
@pytest.mark.parametrize("rows", [63, 300])
def test_many_rows(hip, rows, V):
    if rows * V > 64 * 151936:
        pytest.skip("time on the host")
    rng = np.random.default_rng(rows)
    x, tokens = logits(rng, rows, V), rng.integers(0, V, rows)
    check(call(hip, x, tokens, 8)[0], x, tokens, 8)


@pytest.mark.parametrize("V", [70, 1000, 1001, 49152, 151936])
@pytest.mark.parametrize("top", [0, 7, 64])
def test_values_of_every_kind(hip, V, top):
    """Rows of one value, of few values (ties over the whole row), one value above all, masked to a few tokens and to
    none, infinities of either sign, NaN, zeros of both signs, differences past fp32's range, the largest at either end."""
    rng = np.random.default_rng(V)
    x = logits(rng, 16, V)
    x[0] = 3.25
    x[1] = rng.integers(0, 3, V)
    x[2] = -1e30
    x[2, V // 2] = 0.0
    x[3] = -np.inf
    x[3, rng.choice(V, 9, replace=False)] = rng.standard_normal(9)
    x[4] = -np.inf
    x[5, [1, V - 1]] = np.inf
    x[6, ::2] = np.nan
    x[7] = np.nan
    x[8] = np.where(rng.random(V) < 0.5, 0.0, -0.0)
    x[9, 0], x[9, 1] = 3e38, -3e38
    x[10, V - 1] = 50.0
    x[11, 0] = 50.0
    x[12] = np.float32(-3.4028235e38)  # a mask of the type's lowest value everywhere but in one place
    x[12, 3] = 1.0
    x[13] = np.linspace(-40, 40, V)[::-1]
    x[14] = np.linspace(-40, 40, V)
    x[15] = np.float32(-3.4028235e38)
    tokens = np.array([V - 1, 5, 7, 11, 3, V - 1, 1, 2, V // 2, 1, V - 1, 0, 3, V - 1, 0, V - 1])
    check(call(hip, x, tokens, top)[0], x, tokens, top)
    tokens = np.array([0, V, 0xFFFFFFFF, 0, V - 1, 0, 0, V + 5] * 2)
    check(call(hip, x, tokens, top)[0], x, tokens, top)


@pytest.mark.parametrize("V", [1000, 49152, 151936])
def test_top_in_one_place(hip, V):
    """All of the largest logits side by side, at the start, in the middle and at the end; and spread evenly."""
    rng = np.random.default_rng(V)
    x = logits(rng, 4, V)
    for r, at in enumerate((0, V // 2 - 32, V - 64)):
        x[r, at:at + 64] = 20 + rng.standard_normal(64)
    x[3, ::V // 64][:64] = 20.0
    tokens = np.array([0, V // 2, V - 1, V // 64])
    check(call(hip, x, tokens, 64)[0], x, tokens, 64)


@pytest.mark.parametrize("rows,V", [(1, 524289), (2, 600001), (1, 2100000)])
def test_long_rows(hip, rows, V):
    """More splits than a row has: several chunks each, the largest in the first, in the last, rising maxima."""
    rng = np.random.default_rng(V)
    x, tokens = logits(rng, rows, V), rng.integers(0, V, rows)
    check(call(hip, x, tokens, 20)[0], x, tokens, 20)
    x[:, -5:] = 30.0
    check(call(hip, x, tokens, 20)[0], x, tokens, 20)
    x += np.linspace(-90, 0, V, dtype=np.float32)
    check(call(hip, x, tokens, 20)[0], x, tokens, 20)
    x[:, :V // 2] = -np.inf
    check(call(hip, x, tokens, 20)[0], x, tokens, 20)


@pytest.mark.parametrize("offset", [0, 1, 2, 3])
@pytest.mark.parametrize("V", [1003, 4096, 50257, 151936])
def test_alignments(hip, V, offset):
    rng = np.random.default_rng(offset)
    x, tokens = logits(rng, 3, V), rng.integers(0, V, 3)
    check(call(hip, x, tokens, 20, offset=offset)[0], x, tokens, 20)


@pytest.mark.parametrize("want", [(True, False, False), (False, True, False), (False, False, True),
                                  (False, False, False)])
def test_outputs_that_are_not_wanted(hip, want):
    rng = np.random.default_rng(1)
    x, tokens = logits(rng, 3, 5000), rng.integers(0, 5000, 3)
    for top in (0, 4):
        check(call(hip, x, tokens, top, want)[0], x, tokens, top)
    if not (want[0] or want[1]):
        check(call(hip, x, None, 4, want)[0], x, None, 4)


@pytest.mark.parametrize("rows,V,top", [(2, 3000, 5), (7, 49152, 4), (40, 151936, 20)])
def test_graph_replays(hip, rows, V, top):
    """A captured call, replayed on other logits, the program's own calls between; the same from call to call."""
    from qraf_amd.backend import Graph, Stream
    rng, st = np.random.default_rng(2), Stream()
    x, tokens = logits(rng, rows, V), rng.integers(0, V, rows)
    _, launch, read, (d_x, d_t) = call(hip, x, tokens, top, stream=st.h)
    g = Graph(st)
    with g:
        launch(st.h)
    for _ in range(4):
        x, tokens = logits(rng, rows, V), rng.integers(0, V, rows).astype(np.uint32)
        d_x.upload(x)
        d_t.upload(tokens)
        g.launch()
        st.synchronize()
        got = read()
        check(got, x, tokens, top)
        launch()
        assert all(np.array_equal(a, b) for a, b in zip(read(), got))
    g.destroy()
    st.destroy()


@pytest.mark.parametrize("V", [4, 5, 6, 7, 1022, 2050, 4099, 8191, 8194, 16387, 40001, 49155, 98301, 98305, 98306, 98307])
def test_ends_of_rows(hip, V):
    """Rows that end inside 16 bytes: the largest logits, NaN and -inf next to the end, behind which the next row begins."""
    rng = np.random.default_rng(V)
    x = logits(rng, 5, V)
    x[0, -3:] = 40.0, 41.0, 40.0
    x[1, -4:] = np.nan, 39.0, np.nan, -np.inf
    x[2, -1] = -np.inf
    x[3, :4] = 60.0
    x[4, -2:] = np.inf
    tokens = np.array([V - 1, V - 3, V - 1, V - 2, V - 1])
    for top in (0, 4):
        check(call(hip, x, tokens, top, offset=1)[0], x, tokens, top)


@pytest.mark.parametrize("rows,V", [(170, 49152), (171, 49152), (209, 40001), (210, 40001), (85, 98303), (86, 98303)])
def test_splits_of_either_size(hip, rows, V):
    """The last call whose splits are short and the first whose are long, in the workspace of the larger."""
    assert hip.lib.qraf_hip_token_logprobs_workspace_bytes(rows, V, 5) <= \
        hip.lib.qraf_hip_token_logprobs_workspace_bytes(rows + 1, V, 5)
    rng = np.random.default_rng(rows)
    x = np.tile(logits(rng, 5, V), (rows // 5 + 1, 1))[:rows]
    tokens = rng.integers(0, V, rows)
    got = call(hip, x, tokens, 5)[0]
    check([g[-9:] for g in got], x[-9:], tokens[-9:], 5)
    check([g[:3] for g in got], x[:3], tokens[:3], 5)
    for g in got[2:]:
        assert np.array_equal(g[:5], g[5:10])

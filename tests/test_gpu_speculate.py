"""Sampling probabilities (qraf_hip_sample_probs_dev) and draft verification (qraf_hip_verify_draft_dev) against
their definitions in 64 bits.

Probabilities: the kept set has to be the definition's, token by token.  A kept value is exp((l - max) / T) over the
kept sum: the exponent's argument, its product with log2 e and the hardware exponential are each within 2^-23 of
their values, the division and the last rounding within 2^-24, so values are within 8 * 2^-24 of the 64-bit ones
(and 2^-126 for those below fp32's normal range).

Tokens and counts of the verification are whole numbers and have to be equal; products and sums are 64-bit on both
sides, and the tests' draws lie further than 1e-9 of the total from a border."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def ref_probs(logits, T, top_k, top_p):
    out = np.zeros(logits.shape)
    T, top_p = float(np.float32(T)), float(np.float32(top_p))
    for r, row in enumerate(logits):
        l = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
        m = l.max()
        if m == -np.inf:
            continue
        if not T > 0:
            out[r, int(np.argmax(l))] = 1
            continue
        order = np.argsort(-l, kind="stable")
        if 0 < top_k < l.size:
            order = order[:top_k]
        x = l[order]
        with np.errstate(invalid="ignore", over="ignore"):
            w = np.where(x == m, 1.0, np.where(x == -np.inf, 0.0, np.exp((x - m) / T)))
        if 0 < top_p < 1:
            k = int(np.searchsorted(np.cumsum(w), top_p * w.sum()))
            order, w = order[:k + 1], w[:k + 1]
        out[r, order] = w / w.sum()
    return out


def device_probs(hip, logits, T, top_k, top_p, in_place=False, repeats=1, penalty=None, recent=None):
    from qraf_amd._lib import SamplingParams
    from qraf_amd.backend import DeviceBuffer
    rows, V = logits.shape
    d = DeviceBuffer.from_array(logits)
    need = hip.lib.qraf_hip_sample_probs_workspace_bytes(rows, V)
    ws = DeviceBuffer.from_array(np.full(need, 0xFF, np.uint8))
    out = d if in_place else DeviceBuffer.from_array(np.full((rows, V), np.float32(7)))
    rec = cnt = None
    stride = 0
    if recent is not None:
        stride = max(len(x) for x in recent)
        a = np.zeros((rows, stride), np.uint32)
        for i, x in enumerate(recent):
            a[i, :len(x)] = x
        rec, cnt = DeviceBuffer.from_array(a), DeviceBuffer.from_array(np.array([len(x) for x in recent], np.int32))
    p = SamplingParams(T, top_k, top_p, 1.0 if penalty is None else penalty)
    got = []
    for _ in range(repeats):
        hip._lib.call("qraf_hip_sample_probs_dev", d.ptr, rows, V, C.byref(p), rec.ptr if rec else None,
                      cnt.ptr if cnt else None, stride, out.ptr, ws.ptr, need, None)
        hip._lib.call("qraf_hip_stream_synchronize", None)
        got.append(out.download(np.float32, rows * V).reshape(rows, V))
    for g in got[1:]:
        assert np.array_equal(g, got[0]), "results differ from call to call"
    return got[0]


def check_probs(got, want):
    tiny = 2.0 ** -126
    differ = (got > 0) != (want > 0)
    assert not np.any(differ & (want > 2 * tiny)), f"another set: {np.argwhere(differ & (want > 2 * tiny))[:3]}"
    assert not np.any(differ & (got > 2 * tiny))
    err = np.abs(got.astype(np.float64) - want)
    tol = 8 * 2.0 ** -24 * want + 2 * tiny
    assert np.all(err <= tol), f"worst {np.max(err / tol):.2f} tolerances"


def model_logits(rng, rows, V):
    return (rng.standard_normal((rows, V)) * 1.5 + 10 * rng.random((rows, V)) ** 400).astype(np.float32)


PARAMS = [(1.0, 0, 1.0), (0.7, 0, 1.0), (0.0, 0, 1.0), (-1.0, 3, 0.5), (0.8, 40, 0.9), (1.3, 40, 1.0), (1.0, 0, 0.95),
          (0.5, 1, 1.0), (1.0, 400, 0.8), (2.0, 0, 0.3), (1.0, 5000, 0.999), (1.0, 0, 1e-6), (0.9, 7, 0.0)]


@pytest.mark.parametrize("T,k,p", PARAMS)
@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 65, 1000, 4099, 32000, 49152, 151936])
def test_probs(hip, V, T, k, p):
    rng = np.random.default_rng(V + k)
    x = model_logits(rng, 5, V)
    check_probs(device_probs(hip, x, T, k, p, repeats=2), ref_probs(x, T, k, p))


@pytest.mark.parametrize("rows", [1, 3, 130, 700])
def test_probs_rows(hip, rows):
    rng = np.random.default_rng(rows)
    x = model_logits(rng, rows, 8001)
    for T, k, p in ((1.0, 0, 1.0), (0.8, 40, 0.9), (1.0, 0, 0.95)):
        check_probs(device_probs(hip, x, T, k, p), ref_probs(x, T, k, p))


@pytest.mark.parametrize("V", [40, 5000, 151936])
def test_probs_of_equal_logits(hip, V):
    """Ties: the lowest indices first, in the whole row and at the border alone."""
    rng = np.random.default_rng(V)
    x = np.zeros((4, V), np.float32)
    x[1] = rng.integers(0, 3, V)
    x[2, ::2] = -0.0
    x[3] = np.round(rng.standard_normal(V) * 4) / 4
    for T, k, p in ((1.0, 0, 1.0), (1.0, 7, 1.0), (1.0, V // 2, 1.0), (1.0, 0, 0.5), (0.9, V - 1, 0.75), (0.0, 0, 1.0),
                    (1.0, 0, 0.3), (1.0, 17, 0.25)):
        check_probs(device_probs(hip, x, T, k, p), ref_probs(x, T, k, p))


def test_probs_of_masked_and_infinite_rows(hip):
    V = 3001
    rng = np.random.default_rng(5)
    x = model_logits(rng, 11, V)
    x[0] = -np.inf
    x[1, 5:] = -np.inf
    x[2] = -np.inf
    x[2, 2900] = -3.0
    x[3, 17] = np.inf
    x[4, [3, 99, 2000]] = np.inf
    x[5, ::3] = np.nan
    x[6] = np.nan
    x[7] = np.finfo(np.float32).min
    x[8] = np.finfo(np.float32).min
    x[8, 77] = 0
    x[9, 1::2] = -np.inf
    x[10] *= 1e30
    for T, k, p in ((1.0, 0, 1.0), (0.8, 40, 0.9), (1.0, 0, 0.95), (0.0, 0, 1.0), (1.0, 2, 1.0), (1e-30, 0, 1.0),
                    (1e30, 0, 0.5)):
        check_probs(device_probs(hip, x, T, k, p), ref_probs(x, T, k, p))


def test_probs_in_place_and_with_a_penalty(hip):
    rng = np.random.default_rng(6)
    x = model_logits(rng, 6, 9000)
    want = ref_probs(x, 0.8, 40, 0.9)
    check_probs(device_probs(hip, x, 0.8, 40, 0.9, in_place=True), want)
    from qraf_amd.engine import apply_repetition_penalty
    recent = [list(rng.integers(0, 9000, 5 + 3 * i)) + list(np.argsort(-x[i])[:3]) for i in range(6)]
    y = x.copy()
    for i in range(6):
        apply_repetition_penalty(y[i], recent[i], 1.3)
    check_probs(device_probs(hip, x, 0.8, 40, 0.9, penalty=1.3, recent=recent), ref_probs(y, 0.8, 40, 0.9))


def test_probs_unaligned_rows(hip):
    """Rows whose length is no multiple of 4, at a base that is 4-byte aligned only."""
    from qraf_amd._lib import SamplingParams
    from qraf_amd.backend import DeviceBuffer
    rng = np.random.default_rng(7)
    x = model_logits(rng, 3, 50001)
    pad = np.concatenate([np.zeros(1, np.float32), x.ravel()])
    d, out = DeviceBuffer.from_array(pad), DeviceBuffer.from_array(np.zeros_like(pad))
    need = hip.lib.qraf_hip_sample_probs_workspace_bytes(3, 50001)
    ws = DeviceBuffer(need)
    for T, k, p in ((1.0, 0, 1.0), (0.8, 40, 0.9), (1.0, 0, 0.9)):
        hip._lib.call("qraf_hip_sample_probs_dev", d.ptr + 4, 3, 50001, C.byref(SamplingParams(T, k, p, 1.0)), None,
                      None, 0, out.ptr + 4, ws.ptr, need, None)
        hip._lib.call("qraf_hip_stream_synchronize", None)
        check_probs(out.download(np.float32, x.size, 4).reshape(x.shape), ref_probs(x, T, k, p))


# ------------------------------------------------------------------ verification

def ref_verify(p, q, draft, starts, u, v):
    accepted, tokens = [], np.full(len(draft), 0xAAAAAAAA, np.uint32)
    V = p.shape[1]
    margin = 1.0
    for s in range(len(starts) - 1):
        r0, r1 = starts[s], starts[s + 1]
        if r0 == r1:
            accepted.append(0)
            continue
        r = r0
        while r < r1 - 1 and draft[r] < V and \
                float(u[r]) * (1.0 if q is None else float(q[r, draft[r]])) < float(p[r, draft[r]]):
            tokens[r] = draft[r]
            r += 1
        w = p[r].astype(np.float64)
        if r < r1 - 1:
            if q is not None:
                less = np.maximum(w - q[r], 0)
            else:
                less = w.copy()
                if draft[r] < V:
                    less[draft[r]] = 0
            w = less if less.sum() > 0 else w
        c = np.cumsum(w)
        t = c[-1] * float(v[s])
        k = int(np.searchsorted(c, t, side="right"))
        if c[-1] > 0:
            near = np.abs(c[max(0, k - 2):k + 2] - t).min() / c[-1]
            if float(v[s]) > 0:
                margin = min(margin, near)
        tokens[r] = k if k < V else 0
        tokens[r + 1:r1] = 0xFFFFFFFF
        accepted.append(r - r0)
    return np.array(accepted, np.int32), tokens, margin


def device_verify(hip, p, q, draft, starts, u, v, stream=None, repeats=2):
    from qraf_amd.backend import DeviceBuffer
    up = DeviceBuffer.from_array
    n, (rows, V) = len(starts) - 1, p.shape
    need = hip.lib.qraf_hip_verify_draft_workspace_bytes(n, V)
    b = [up(x) for x in (p, draft, np.asarray(starts, np.int32), u, v)]
    dq = up(q) if q is not None else None
    ws = up(np.full(need, 0xFF, np.uint8))
    acc, tok = up(np.full(n, -7, np.int32)), up(np.full(rows, 0xAAAAAAAA, np.uint32))
    res = []
    for _ in range(repeats):
        hip._lib.call("qraf_hip_verify_draft_dev", b[0].ptr, dq.ptr if dq else None, b[1].ptr, b[2].ptr, n, rows, V,
                      b[3].ptr, b[4].ptr, acc.ptr, tok.ptr, ws.ptr, need, stream)
        hip._lib.call("qraf_hip_stream_synchronize", stream)
        res.append((acc.download(np.int32, n), tok.download(np.uint32, rows)))
    for x in res[1:]:
        assert np.array_equal(x[0], res[0][0]) and np.array_equal(x[1], res[0][1])
    return res[0]


def drafted(rng, counts, V, T=1.0, closeness=0.5):
    starts = np.concatenate([[0], np.cumsum(counts)])
    x = model_logits(rng, max(1, int(starts[-1])), V)
    p = ref_probs(x, T, 0, 1.0).astype(np.float32)
    q = ref_probs((x + closeness * rng.standard_normal(x.shape)).astype(np.float32), T, 0, 1.0).astype(np.float32)
    cum = np.cumsum(q.astype(np.float64), 1)
    draft = np.minimum((cum < rng.random((len(q), 1)) * cum[:, -1:]).sum(1), V - 1).astype(np.uint32)
    u, v = rng.random(len(q), np.float32), rng.random(len(counts), np.float32)
    return p, q, draft, starts.astype(np.int32), u, v


def check_verify(hip, p, q, draft, starts, u, v):
    acc, tok, margin = ref_verify(p, q, draft, starts, u, v)
    assert margin > 1e-11, "the test's own draw lies on a border"
    got = device_verify(hip, p, q, draft, starts, u, v)
    assert np.array_equal(got[0], acc), (got[0], acc)
    assert np.array_equal(got[1], tok), (got[1], tok)
    return acc


@pytest.mark.parametrize("given", [True, False], ids=["model", "ngram"])
@pytest.mark.parametrize("V", [1, 2, 5, 64, 1000, 4099, 32000, 151936])
def test_verify(hip, V, given):
    rng = np.random.default_rng(V)
    counts = [5, 1, 3, 9, 2, 4]
    p, q, draft, starts, u, v = drafted(rng, counts, V)
    check_verify(hip, p, q if given else None, draft, starts, u, v)


def test_verify_many_sequences(hip):
    rng = np.random.default_rng(3)
    counts = rng.integers(1, 6, 300)
    p, q, draft, starts, u, v = drafted(rng, counts, 777, closeness=0.2)
    acc = check_verify(hip, p, q, draft, starts, u, v)
    assert 0.2 < np.mean(acc == counts - 1) < 0.999  # both outcomes are there


def test_verify_all_accepted_none_accepted(hip):
    rng = np.random.default_rng(4)
    p, q, draft, starts, u, v = drafted(rng, [6, 6, 4], 500)
    assert list(check_verify(hip, p, q, draft, starts, np.zeros_like(u), v)) == [5, 5, 3]
    for r in range(len(draft)):
        p[r, draft[r]] = 0
    assert list(check_verify(hip, p, q, draft, starts, u, v)) == [0, 0, 0]
    # a zero draw is not below a zero probability, and picks the first token of any weight
    p[0, :7] = 0
    v[:] = 0
    check_verify(hip, p, q, draft, starts, np.zeros_like(u), v)


def test_verify_greedy_rows(hip):
    """One-hot rows: drafts are accepted while they are the argmax, whatever the draws."""
    rng = np.random.default_rng(5)
    V, counts = 300, [5, 5, 5, 1]
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    best = rng.integers(0, V, 16)
    p = np.zeros((16, V), np.float32)
    p[np.arange(16), best] = 1
    draft = best.astype(np.uint32)
    draft[2] = (draft[2] + 1) % V
    draft[5] = (draft[5] + 1) % V
    u, v = rng.random(16, np.float32), rng.random(4, np.float32)
    for q in (None, ref_probs(model_logits(rng, 16, V), 1.0, 0, 1.0).astype(np.float32)):
        acc, tok = device_verify(hip, p, q, draft, starts, u, v)
        assert list(acc) == [2, 0, 4, 0]
        assert tok[2] == best[2] and tok[5] == best[5] and tok[14] == best[14] and tok[15] == best[15]


def test_verify_odd_sequences(hip):
    """Sequences without rows, drafts outside the vocabulary, p equal to q, rows behind the last sequence."""
    rng = np.random.default_rng(6)
    V = 129
    p, q, draft, starts, u, v = drafted(rng, [3, 0, 4, 2, 0], V)
    draft[0] = V
    draft[3] = 0xFFFFFFFF
    check_verify(hip, p, q, draft, starts, u, v)
    check_verify(hip, p, None, draft, starts, u, v)
    # p == q never rejects a draft that p holds; a draft outside it finds nothing left of p - q and draws from p
    check_verify(hip, p, p, draft, starts, u, v)
    short = np.array([0, 3, 3, 5, 5, 5], np.int32)  # the last rows belong to nobody
    acc, tok, _ = ref_verify(p, q, draft, short, u, v)
    got = device_verify(hip, p, q, draft, short, u, v)
    assert np.array_equal(got[0], acc) and np.array_equal(got[1], tok)
    assert np.all(got[1][5:] == 0xAAAAAAAA)


def test_verify_keeps_the_targets_distribution(hip):
    """Over many draws the first emitted token is distributed as the target's own sample.  20,000 sequences of one
    draft over 4 tokens: a frequency is off by more than 5 standard deviations with probability 6e-7."""
    rng = np.random.default_rng(7)
    n = 20000
    p1, q1 = np.array([0.5, 0.2, 0.25, 0.05], np.float32), np.array([0.1, 0.6, 0.2, 0.1], np.float32)
    starts = (2 * np.arange(n + 1)).astype(np.int32)
    p, q = np.tile(p1, (2 * n, 1)), np.tile(q1, (2 * n, 1))
    for qq in (q, None):
        draft = rng.choice(4, 2 * n, p=q1 / q1.astype(np.float64).sum() if qq is not None else None).astype(np.uint32)
        acc, tok = device_verify(hip, p, qq, draft, starts, rng.random(2 * n, np.float32), rng.random(n, np.float32))
        first = np.bincount(tok[::2], minlength=4) / n
        assert np.all(np.abs(first - p1) < 5 * np.sqrt(p1 * (1 - p1) / n)), first


@pytest.mark.parametrize("given", [True, False])
def test_captured_together_and_replayed(hip, given):
    """Probabilities of the draft and the target and their verification in one graph, on replaced inputs."""
    from qraf_amd._lib import SamplingParams
    from qraf_amd.backend import DeviceBuffer, Graph, Stream
    rng = np.random.default_rng(8)
    V, counts = 5003, [5, 3, 1, 7]
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    rows, n = int(starts[-1]), len(counts)
    up = DeviceBuffer.from_array
    x, y = DeviceBuffer(rows * V * 4), DeviceBuffer(rows * V * 4)
    p, q = DeviceBuffer(rows * V * 4), DeviceBuffer(rows * V * 4)
    need_p = hip.lib.qraf_hip_sample_probs_workspace_bytes(rows, V)
    need_v = hip.lib.qraf_hip_verify_draft_workspace_bytes(n, V)
    wp, wv, st = DeviceBuffer(need_p), DeviceBuffer(need_v), up(starts)
    draft, u, v = DeviceBuffer(rows * 4), DeviceBuffer(rows * 4), DeviceBuffer(n * 4)
    acc, tok = DeviceBuffer(n * 4), DeviceBuffer(rows * 4)
    params, s = SamplingParams(0.8, 40, 0.95, 1.0), Stream()

    def body(h):
        call = hip._lib.call
        call("qraf_hip_sample_probs_dev", x.ptr, rows, V, C.byref(params), None, None, 0, p.ptr, wp.ptr, need_p, h)
        call("qraf_hip_sample_probs_dev", y.ptr, rows, V, C.byref(params), None, None, 0, q.ptr, wp.ptr, need_p, h)
        call("qraf_hip_verify_draft_dev", p.ptr, q.ptr if given else None, draft.ptr, st.ptr, n, rows, V, u.ptr, v.ptr,
             acc.ptr, tok.ptr, wv.ptr, need_v, h)

    g = Graph(s)
    with g:
        body(s.h)
    for _ in range(4):
        lx = model_logits(rng, rows, V)
        ly = (lx + 0.3 * rng.standard_normal(lx.shape)).astype(np.float32)
        x.upload(lx), y.upload(ly)
        draft.upload(np.argmax(ly + rng.gumbel(size=ly.shape), 1).astype(np.uint32))
        u.upload(rng.random(rows, np.float32)), v.upload(rng.random(n, np.float32))
        out = []
        for launch in (g.launch, lambda: body(s.h)):
            for b in (p, q, acc, tok):
                b.zero()
            launch()
            s.synchronize()
            out.append((p.download(np.float32, rows * V), acc.download(np.int32, n), tok.download(np.uint32, rows)))
        for a, b in zip(*out):
            assert np.array_equal(a, b)
        check_probs(out[0][0].reshape(rows, V), ref_probs(lx, 0.8, 40, 0.95))
        pp, qq = out[0][0].reshape(rows, V), q.download(np.float32, rows * V).reshape(rows, V)
        want = ref_verify(pp, qq if given else None, draft.download(np.uint32, rows), starts,
                          u.download(np.float32, rows), v.download(np.float32, n))
        assert np.array_equal(out[0][1], want[0]) and np.array_equal(out[0][2], want[1])
    g.destroy()
    s.destroy()

"""Sampling probabilities and draft verification of many logits at once: the forms whose threads take 32 of them (from
2^21 logits a call; probabilities also from vocabularies of 65,536), both sides of those bounds, rows that the float4
loads do not take, and vocabularies beyond a short top-k's sub-ranges and beyond a split for each thread.  Tolerances
are those of test_gpu_speculate."""
import numpy as np
import pytest

from tests.test_gpu_speculate import check_probs, check_verify, device_probs, device_verify, drafted, model_logits, ref_probs

pytestmark = pytest.mark.gpu
PARAMS = [(0.7, 0, 1.0), (0.0, 0, 1.0), (0.8, 40, 0.9), (1.0, 0, 0.95), (1.0, 512, 0.8), (1.0, 700, 0.999), (2.0, 0, 0.3)]


@pytest.mark.parametrize("V", [131076, 151936, 151937])
def test_probs(hip, V):
    x = model_logits(np.random.default_rng(V), 16, V)
    for T, k, p in PARAMS:
        want = ref_probs(x, T, k, p)
        check_probs(device_probs(hip, x, T, k, p, repeats=2), want)
        if k in (0, 40):
            check_probs(device_probs(hip, x, T, k, p, in_place=True), want)


@pytest.mark.parametrize("rows,V", [(31, 65536), (32, 65536), (33, 65535), (32, 65540), (33, 65537), (13, 151936), (14, 151936)])
def test_probs_next_to_the_bounds(hip, rows, V):
    x = model_logits(np.random.default_rng(rows + V), rows, V)
    for T, k, p in ((0.7, 0, 1.0), (0.8, 40, 0.9), (1.0, 0, 0.95)):
        check_probs(device_probs(hip, x, T, k, p), ref_probs(x, T, k, p))


@pytest.mark.parametrize("rows,V", [(2, 163840), (2, 163841), (2, 262144), (9, 262147), (1, 700001)])
def test_probs_of_large_vocabularies(hip, rows, V):
    """A short top-k takes maxima of 20,480 sub-ranges: 163,840 logits by 8, 655,360 by 32; the radix select beyond."""
    x = model_logits(np.random.default_rng(V), rows, V)
    for T, k, p in ((0.7, 0, 1.0), (0.8, 40, 0.9), (1.0, 0, 0.95), (1.0, 512, 1.0)):
        check_probs(device_probs(hip, x, T, k, p), ref_probs(x, T, k, p))


def test_probs_of_equal_masked_and_infinite_rows(hip):
    V = 151937
    rng = np.random.default_rng(3)
    x = model_logits(rng, 16, V)
    x[0] = 0
    x[1] = rng.integers(0, 3, V)
    x[2] = -np.inf
    x[3, 7:] = -np.inf
    x[4, [5, 150000]] = np.inf
    x[5, ::3] = np.nan
    x[6] = np.finfo(np.float32).min
    x[7] = np.round(x[7] * 2) / 2
    for T, k, p in PARAMS:
        check_probs(device_probs(hip, x, T, k, p), ref_probs(x, T, k, p))


@pytest.mark.parametrize("V", [1000, 4099, 151936])
def test_probs_of_logits_further_apart_than_fp32(hip, V):
    """Differences past fp32's largest, over a temperature that brings them back: -6.6 at the most."""
    rng = np.random.default_rng(V)
    x = rng.uniform(-3.3e38, 3.3e38, (14, V)).astype(np.float32)
    for T, k, p in ((1e38, 0, 1.0), (1e38, 40, 1.0), (1e38, 0, 0.95), (2e38, 700, 0.9), (3e38, 0, 1.0)):
        check_probs(device_probs(hip, x, T, k, p), ref_probs(x, T, k, p))


@pytest.mark.parametrize("given", [True, False], ids=["model", "ngram"])
@pytest.mark.parametrize("n,V", [(13, 151936), (14, 151936), (16, 151937), (40, 52429), (4, 524289)])
def test_verify(hip, n, V, given):
    rng = np.random.default_rng(n + V)
    p, q, draft, starts, u, v = drafted(rng, rng.integers(1, 4, n), V)
    check_verify(hip, p, q if given else None, draft, starts, u, v)


@pytest.mark.parametrize("n,V", [(1, 524288), (1, 600000), (3, 600001)])
def test_verify_with_several_splits_a_thread(hip, n, V):
    """Past 524,288 tokens of few sequences a thread sums several splits; most of them hold nothing."""
    rng = np.random.default_rng(V)
    p = np.zeros((n, V), np.float32)
    for r in range(n):
        at = rng.choice(V, 200, replace=False)
        p[r, at] = rng.random(200) ** 8
    p /= p.sum(1, keepdims=True)
    starts = np.arange(n + 1).astype(np.int32)
    for v in (0.0, 1e-4, 0.3, 0.7, 0.9999999):
        check_verify(hip, p, None, np.zeros(n, np.uint32), starts, np.zeros(n, np.float32), np.full(n, v, np.float32))


# (seed, a tail's second value): the target lies within a rounding of the running sum behind a thread's first split, and
# its second split is empty (found with the device's order of sums, on the CPU)
BORDERS = [(9, "0x1.f04daep-45"), (31, "0x1.d30e94p-45"), (53, "0x1.d7c288p-45"), (85, "0x1.d7b0a2p-45"),
           (91, "0x1.d80e26p-45"), (92, "0x1.ef4c38p-45")]


def test_a_draw_next_to_a_split_of_nothing_takes_a_token_of_some_weight(hip):
    V, split = 600000, 2048
    v = np.float32(1 - 2.0 ** -24)
    for a in range(0, len(BORDERS), 3):
        p = np.zeros((3, V), np.float32)
        for row, (seed, last) in zip(p, BORDERS[a:a + 3]):
            rng = np.random.default_rng(seed)
            w = np.zeros(-(-V // split), np.float32)
            j = rng.integers(40, 120)
            w[0] = 0.9
            for t in range(1, j + 1):
                w[2 * t] = rng.random() * 1e-9
            tail = 2 * j + 2 + 2 * rng.integers(1, 6, 1)[0]
            w[tail] = float(np.sum(w.astype(np.float64))) / (2 ** 24 - 1) * (1 - 1e-6)
            w[tail + 2] = float.fromhex(last)
            row[np.arange(w.size) * split] = w
        _, tok = device_verify(hip, p, None, np.zeros(3, np.uint32), np.arange(4), np.zeros(3, np.float32), np.full(3, v))
        for row, t in zip(p, tok):
            assert row[t] > 0, t
            before = row[:t].astype(np.float64).sum()  # a border of the draw's, to a few roundings
            target = row.astype(np.float64).sum() * float(v)
            assert before - 1e-12 <= target <= before + float(row[t]) + 1e-12

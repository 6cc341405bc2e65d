"""Trees of few rows on f32 pages, which take a workgroup per row and query heads: every number of heads and positions that
it is built for, and the sizes where the next form begins.  Definition and tolerance: test_gpu_tree_attention.py."""
import numpy as np
import pytest

from tests.test_gpu_tree_attention import F32, Call, Trees, check, run, tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ctx", [65, 256, 257, 512, 513, 1024, 1025])
@pytest.mark.parametrize("H,Hkv,hd,nodes", [(9, 3, 64, 28), (9, 3, 64, 29), (16, 2, 128, 16), (16, 2, 128, 17), (2, 1, 64, 64),
                                            (4, 4, 64, 40), (8, 2, 64, 40), (6, 3, 64, 50), (12, 1, 64, 5), (16, 1, 128, 3)])
def test_contexts(hip, H, Hkv, hd, nodes, ctx):
    rng = np.random.default_rng(ctx + H)
    run(hip, Trees(rng, [(ctx - nodes, tree(rng, nodes))], Hkv, hd, 16, F32, max_ctx=ctx), H, rng)


@pytest.mark.parametrize("ps", [4, 8, 16, 64, 256])
@pytest.mark.parametrize("H,Hkv,hd", [(9, 3, 64), (4, 1, 128), (2, 2, 64)])
def test_several_sequences(hip, H, Hkv, hd, ps):
    """Rows of no sequence ahead and behind, sequences without rows between, caches of any length and none."""
    rng = np.random.default_rng(ps)
    seqs = [(0, []), (17, tree(rng, 3)), (0, tree(rng, 5)), (5, []), (5, []), (230, tree(rng, 1)), (101, tree(rng, 9)), (7, [])]
    run(hip, Trees(rng, seqs, Hkv, hd, ps, F32, ahead=2, behind=3), H, rng)


@pytest.mark.parametrize("seqs", [1, 2, 63, 64, 65, 128])
def test_as_many_sequences_as_a_wave_has_lanes(hip, seqs):
    rng = np.random.default_rng(seqs)
    run(hip, Trees(rng, [(int(rng.integers(0, 200)), tree(rng, 1 + i % 2)) for i in range(seqs)], 1, 64, 16, F32), 2, rng)


@pytest.mark.parametrize("max_ctx", [200, 210, 500, 1000])
def test_masks(hip, max_ctx):
    """Nothing at all (with and without a cache), the highest bit alone, every second, bits and caches past max_ctx."""
    rng = np.random.default_rng(max_ctx)
    masks = [0, 1 << 63, 0x5555555555555555, 1, (1 << 64) - 1, 3 << 40]
    seqs = [(0, masks), (150, masks), (max_ctx - 30, masks), (max_ctx, masks), (max_ctx + 9, masks[:2])]
    c = Trees(rng, seqs, 3, 64, 16, F32, max_ctx=max_ctx)
    c.base = np.minimum(c.base, max_ctx)
    q = rng.standard_normal((c.n, 6, 64)).astype(np.float32)
    call = Call(hip, c, q, 6)
    call.base.upload(np.array([b for b, _ in seqs], np.int32))
    call.launch()
    check(c, q, call.result())


@pytest.mark.parametrize("H,Hkv,hd,max_ctx", [(9, 3, 64, 250), (9, 3, 64, 500), (9, 3, 64, 1000), (8, 1, 128, 250), (8, 1, 128, 500),
                                              (4, 1, 64, 250)])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_no_numbers_that_nobody_attends_to(hip, H, Hkv, hd, max_ctx, what):
    rng = np.random.default_rng(7)
    masks = tree(rng, 20)
    masks[3:] = [m & ~(1 << 3 | 1 << 11) | 1 << i for i, m in enumerate(masks) if i >= 3]
    masks[3] &= ~(1 << 3)
    masks[11] &= ~(1 << 11)
    c = Trees(rng, [(max_ctx - 70, masks)], Hkv, hd, 16, F32, max_ctx=max_ctx)
    for j in (3, 11):
        c.poison(0, max_ctx - 70 + j, what)
    c.K[c.table[0, -1]], c.V[c.table[0, -1]] = what, what  # behind the tree
    q = rng.standard_normal((c.n, H, hd)).astype(np.float32)
    call = Call(hip, c, q, H)
    call.launch()
    got = call.result()
    assert np.isfinite(got).all()
    check(c, q, got)


@pytest.mark.parametrize("max_ctx", [250, 500, 1000])
def test_scores_and_values_that_are_no_numbers(hip, max_ctx):
    """Keys of -inf weigh nothing, of +inf and NaN and values that are attended to give no number, where they do."""
    rng = np.random.default_rng(8)
    masks = [1 << i for i in range(6)]
    c = Trees(rng, [(100, masks)], 1, 64, 16, F32, max_ctx=max_ctx)
    c.poison(0, 101, np.nan, v=False)
    c.poison(0, 103, np.inf, k=False)
    q = np.abs(rng.standard_normal((c.n, 4, 64))).astype(np.float32)
    p, o = c.at(0, 102)
    c.K[p, :, o] = -np.inf
    call = Call(hip, c, q, 4)
    call.launch()
    got = call.result()
    assert np.isnan(got[1]).all() and not np.isfinite(got[3]).any()
    check(c, q, got, {0, 2, 4, 5})

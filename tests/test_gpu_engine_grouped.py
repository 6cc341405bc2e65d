"""Engine steps whose attention reads the positions that a sequence's rows share once, with no least amount of them
(Engine.set_group_least), on models small enough for every row to be run alone as well.

Logits against those of attention by row: the engine's own bar, 1e-3 relative + 1e-4 absolute.  int8 pages of several
layers: 2e-3 of the largest logit, what a byte of a later layer that is stored a step apart may move (half a step of
rounding, reached from either side; the arithmetic is in test_gpu_engine_speculative.py); of one layer, whose bytes do
not depend on its attention, the engine's bar."""
import numpy as np
import pytest

from oracle import pyoracle as po
from tests.test_gpu_engine import SMALL, check_logits, engine_config, oracle_model
from tests.test_gpu_engine_speculative import reference_stream, tokens

pytestmark = pytest.mark.gpu
I8 = 102
KINDS = pytest.mark.parametrize("kv", [po.F32, po.F16, I8], ids=["f32", "f16", "i8"])
TILES = ["q4_gqa8_hd128", "q8_hd64_gqa3"]  # head_dim 64 and 128


def engine(name, kv, max_batch, page_size=16, flags=15, least=0, **change):
    from qraf_amd.engine import Transformer
    kw, seed = dict(SMALL[name][0], **change), SMALL[name][1]
    m = oracle_model(kw, seed)  # (its tensors are views)
    tf = Transformer.from_tensors(engine_config(kw), m.tensors(), kv_dtype=kv, max_batch=max_batch, page_size=page_size)
    tf.engine.set_fusion(flags)
    tf.engine.set_group_least(least)
    return tf


def run(e, toks, plan):
    """plan: steps of (sequence, first position, rows).  The logits of every step."""
    seqs = [e.seq_create() for _ in range(1 + max(s for step in plan for s, *_ in step))]
    out = []
    for step in plan:
        rows = [(s, p + i) for s, p, n in step for i in range(n)]
        out.append(e.step([seqs[s] for s, _ in rows], [toks[(17 * s + p) % len(toks)] for s, p in rows],
                          [p for _, p in rows], logits=True)[0])
    return out


def compare(a, b, kv, layers):
    for x, y in zip(a, b):
        if kv == I8 and layers > 1:
            assert np.abs(y.astype(np.float64) - x).max() <= 2e-3 * np.abs(x).max()
        else:
            check_logits(y, x)


# chunks that begin in one page and end in another, drafts, single rows, a sequence in two runs, the same step thrice
# (eager, captured, replayed) at sizes that are padded (13 rows: to 16)
PLAN = [[(0, 0, 40), (1, 0, 3)], [(0, 40, 21), (1, 3, 19)], [(0, 61, 1), (1, 22, 1)], [(0, 62, 5), (1, 23, 4), (0, 67, 4)],
        [(1, 27, 5)], [(0, 71, 4), (1, 32, 9)], [(0, 71, 4), (1, 32, 9)], [(0, 71, 4), (1, 32, 9)], [(0, 75, 50)]]


@KINDS
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("layers", [1, 3])
@pytest.mark.parametrize("name", TILES)
def test_steps_by_group(hip, name, layers, page, kv):
    toks = tokens(np.random.default_rng(1), SMALL[name][0], 300)
    got = []
    for flags in (7, 15):
        tf = engine(name, kv, 64, page, flags, layers=layers)
        got.append(run(tf.engine, toks, PLAN))
        assert tf.engine.group_steps() == (0 if flags == 7 else len(PLAN) - 1)  # all but the one of single rows
        assert flags == 7 or tf.engine.stats()["pad_rows"] > 0
        tf.engine.close()
    compare(*got, kv, layers)


@KINDS
def test_many_rows_by_group(hip, kv):
    """Steps of the batched layers, whose attention writes the next product's planes."""
    toks = tokens(np.random.default_rng(2), SMALL["q4_gqa8_hd128"][0], 300)
    plan = [[(s, at, 15) for s in range(8)] for at in (0, 15, 30)] + [[(0, 45, 100), (1, 45, 28)]]
    got = []
    for flags in (7, 15):
        tf = engine("q4_gqa8_hd128", kv, 128, 16, flags)
        got.append(run(tf.engine, toks, plan))
        assert tf.engine.group_steps() == (flags == 15) * len(plan)
        tf.engine.close()
    compare(*got, kv, 3)


@pytest.mark.parametrize("kv", [po.F32, po.F16], ids=["f32", "f16"])
@pytest.mark.parametrize("name", TILES)
def test_greedy_generation_by_group(hip, name, kv):
    """n-gram drafts and a model's drafts give the greedy tokens."""
    from qraf_amd.engine import InferenceEngine
    tf, other = engine(name, kv, 16), engine(name, kv, 8)
    prompt = tokens(np.random.default_rng(4), SMALL[name][0], 7) * 3
    want, sure = reference_stream(tf, prompt, 30)
    gen = InferenceEngine(tf, eos_token=None)
    for draft in (None, other):
        for drafts in (1, 4, 15):
            before = tf.engine.group_steps()
            got = gen.generate_speculative(prompt, max_tokens=30, drafts=drafts, draft=draft)
            assert len(got) == 30 and got[:sure] == want[:sure], (drafts, draft is not None)
            assert tf.engine.group_steps() > before
    other.engine.close()
    tf.engine.close()


@pytest.mark.parametrize("name,page,kv", [("q8_llama", 16, po.F32), ("q4_qwen2_tied_bias", 16, po.F16),
                                          ("q8_hd64_gqa3", 8, po.F16), ("q4_gqa8_hd128", 4, po.F32),
                                          ("q4_gqa8_hd128", 8, I8)])
def test_shapes_without_tiles_go_on_by_row(hip, name, page, kv):
    """head_dim 16 and 32 and pages of fewer than 16 positions: no step by group, and the same logits bit for bit."""
    toks = tokens(np.random.default_rng(3), SMALL[name][0], 300)
    got = []
    for flags in (7, 15):
        tf = engine(name, kv, 64, page, flags)
        got.append(run(tf.engine, toks, PLAN))
        assert tf.engine.group_steps() == 0
        tf.engine.close()
    for a, b in zip(*got):
        assert np.array_equal(a, b)


def test_the_least_amount(hip):
    """5 rows at positions 16 to 20 share the 17, 18, 19 and 20 that all but the last attend to, times 3 KV heads of 64."""
    from qraf_amd._lib import ERR_INVALID, HipError
    toks = tokens(np.random.default_rng(5), SMALL["q8_hd64_gqa3"][0], 300)
    share = (17 + 18 + 19 + 20) * 3 * 64
    for least, taken in ((share, 1), (share + 1, 0), (24000000, 0)):
        e = engine("q8_hd64_gqa3", po.F32, 8, least=least).engine
        run(e, toks, [[(0, at, 4)] for at in (0, 4, 8, 12)] + [[(0, 16, 5)]])  # (6, 18, 30 and 42 shared, then 74)
        assert e.group_steps() == taken
        with pytest.raises(HipError) as x:
            e.set_group_least(-1)
        assert x.value.code == ERR_INVALID
        e.close()

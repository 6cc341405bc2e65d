"""Engine steps of trees of drafted tokens, their acceptance, generation with them, and log probabilities, on models
small enough for every path to be run alone as well.

Logits of a tree's nodes against those of their paths fed as plain rows: the engine's own bar, 1e-3 relative + 1e-4
absolute (the same K and V, other orders of sums).  int8 pages: one layer, whose bytes do not depend on its attention.
Tokens are compared up to the first position whose two largest logits lie within 2e-3 of each other."""
import numpy as np
import pytest

from oracle import pyoracle as po
from tests.test_gpu_engine import SMALL, check_logits, oracle_model, upload
from tests.test_gpu_engine_speculative import reference_stream, tokens, transformer

pytestmark = pytest.mark.gpu
I8 = 102
MODELS = ["q8_llama", "q4_qwen2_tied_bias", "f32_llama", "q4_gqa8_hd128", "q8_hd64_gqa3"]
KINDS = pytest.mark.parametrize("kv", [po.F32, po.F16, I8], ids=["f32", "f16", "i8"])


def make(name, kv, **change):
    if kv == I8:
        if name in ("q8_llama", "q4_qwen2_tied_bias", "f32_llama"):
            pytest.skip("int8 pages need head_dim 64 or 128")
        change["layers"] = 1
    return transformer(name, kv, **change)


def random_tree(rng, n, width=5):
    return [-1] + [int(rng.integers(max(0, i - width), i)) for i in range(1, n)]


def paths_of(parents):
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [i])
    return out


def feed(e, seq, toks, at=0):
    for a in range(0, len(toks), e.max_batch):
        part = toks[a:a + e.max_batch]
        e.step([seq] * len(part), part, range(at + a, at + a + len(part)), want_logits=[0] * len(part), argmax=False)


def path_logits(e, seq, base, toks, parents):
    """Logits of every node, its path fed as plain rows at consecutive positions of a sequence with the same cache."""
    out = {}
    for path in sorted(paths_of(parents), key=len, reverse=True):
        if path[-1] not in out:
            lg = e.step([seq] * len(path), [toks[i] for i in path], range(base, base + len(path)), logits=True)[0]
            out.update({i: x for i, x in zip(path, lg) if i not in out})
    return np.stack([out[i] for i in range(len(parents))])


def flat(trees, seqs, bases):
    """The rows of a step_tree: trees of (tokens, parents)."""
    sid, tok, par, pos = [], [], [], []
    for (t, p), s, b in zip(trees, seqs, bases):
        par += [x if x < 0 else x + len(sid) for x in p]
        sid, tok, pos = sid + [s] * len(t), tok + list(t), pos + [b] * len(t)
    return sid, tok, par, pos


@KINDS
@pytest.mark.parametrize("name", MODELS)
@pytest.mark.parametrize("sizes", [(13, 5), (1, 1), (4, 3), (30, 0)])
def test_nodes_equal_their_paths(hip, name, kv, sizes):
    """Two sequences' trees in one step, three times: eager, captured and replayed; sizes with padding and without."""
    tf, kw = make(name, kv, max_batch=32)
    e, rng = tf.engine, np.random.default_rng(sum(sizes))
    prompts = [tokens(rng, kw, 19), tokens(rng, kw, 7)]
    seqs, alone = [e.seq_create() for _ in prompts], [e.seq_create() for _ in prompts]
    for p, s, r in zip(prompts, seqs, alone):
        feed(e, s, p)
        feed(e, r, p)
    for _ in range(3):
        trees = [(tokens(rng, kw, n), random_tree(rng, n)) for n in sizes if n]
        bases = [len(p) for p in prompts]
        got, best = e.step_tree(*flat(trees, seqs, bases), logits=True)
        assert np.array_equal(best, got.argmax(1))
        want = [path_logits(e, r, b, t, p) for (t, p), r, b in zip(trees, alone, bases)]
        check_logits(got, np.concatenate(want))
    e.close()


@pytest.mark.parametrize("graphs", [True, False])
def test_a_full_tree_of_long_sequences(hip, graphs):
    """64 nodes over 180 positions, many sequences: attention cut into pieces."""
    tf, kw = make("q4_gqa8_hd128", po.F16, max_batch=256)
    e, rng = tf.engine, np.random.default_rng(3)
    e.set_graphs(graphs)
    sizes, bases = [64, 64, 40, 1, 17], [180, 33, 100, 60, 128]
    prompts = [tokens(rng, kw, b) for b in bases]
    seqs, alone = [e.seq_create() for _ in prompts], [e.seq_create() for _ in prompts]
    for p, s, r in zip(prompts, seqs, alone):
        feed(e, s, p)
        feed(e, r, p)
    for _ in range(3):
        trees = [(tokens(rng, kw, n), random_tree(rng, n, 9)) for n in sizes]
        got = e.step_tree(*flat(trees, seqs, bases), logits=True)[0]
        want = [path_logits(e, r, b, t, p) for (t, p), r, b in zip(trees, alone, bases)]
        check_logits(got, np.concatenate(want))
    e.close()


def walk(toks, parents, picks):
    at, out = 0, []
    while True:
        out.append(int(picks[at]))
        child = [i for i in range(at + 1, len(toks)) if parents[i] == at and toks[i] == picks[at]]
        if not child:
            return out
        at = child[0]


@KINDS
@pytest.mark.parametrize("name", ["q8_llama", "q4_gqa8_hd128", "q8_hd64_gqa3"])
@pytest.mark.parametrize("sampling", [None, (0.8, 40, 0.9)])
def test_accepted_paths_go_on(hip, name, kv, sampling):
    """Trees whose drafts are mostly the tokens that will be sampled: the emitted tokens are the walk along them, and
    what follows sees the accepted path's keys and values as if it had been fed."""
    from qraf_amd._lib import SamplingParams
    tf, kw = make(name, kv, max_batch=32)
    e, rng = tf.engine, np.random.default_rng(4)
    params = SamplingParams(*(sampling or (0.0, 0, 1.0)), 1.0)
    prompts = [tokens(rng, kw, 21), tokens(rng, kw, 6), tokens(rng, kw, 33)]
    hist = [list(p) for p in prompts]
    seqs, alone = [e.seq_create() for _ in prompts], [e.seq_create() for _ in prompts]
    for p, s, r in zip(prompts, seqs, alone):
        feed(e, s, p[:-1])
        feed(e, r, p[:-1])
    lengths = []
    for turn in range(6):
        sizes = [int(rng.integers(1, 10)) for _ in hist]
        parents = [random_tree(rng, n, 3) for n in sizes]
        bases = [len(h) - 1 for h in hist]
        n = sum(sizes)
        uni = rng.random(n, np.float32)
        trees = [([h[-1], *tokens(rng, kw, k - 1)], p) for h, k, p in zip(hist, sizes, parents)]
        at = np.concatenate([[0], np.cumsum(sizes)])
        for _ in range(12):  # a node's children draft what is sampled behind it, from the root down
            e.step_tree(*flat(trees, seqs, bases))
            picks = e.sample(params, None, None if sampling is None else uni, rows=n)
            changed = False
            for k, (t, p) in enumerate(trees):
                for i in range(1, len(t)):
                    if i % 4 != 3 and t[i] != int(picks[at[k] + p[i]]):
                        t[i] = int(picks[at[k] + p[i]])
                        changed = True
            if not changed:
                break
        lg = e.step_tree(*flat(trees, seqs, bases), logits=True)[0]
        picks = e.sample(params, None, None if sampling is None else uni, rows=n)
        got = e.accept_tree(params, None, None if sampling is None else uni)
        assert got == [walk(t, p, picks[a:]) for (t, p), a in zip(trees, at)]
        lengths += [len(g) for g in got]
        for h, g, s, r, b in zip(hist, got, seqs, alone, bases):
            feed(e, r, [h[-1], *g[:-1]], b)
            h += g
            # the next token of both, over the cache that the path left
            x, y = (e.step([q], [h[-1]], [len(h) - 1], logits=True)[0] for q in (s, r))
            check_logits(x, y)
        assert lg.shape == (n, kw["vocab"])
    assert max(lengths) > 2 and min(lengths) >= 1
    e.close()


def test_acceptance_with_a_penalty(hip):
    from qraf_amd._lib import SamplingParams
    from qraf_amd.engine import apply_repetition_penalty
    tf, kw = make("q8_hd64_gqa3", po.F32)
    e, rng = tf.engine, np.random.default_rng(5)
    seq, hist = e.seq_create(), tokens(rng, kw, 12)
    feed(e, seq, hist[:-1])
    toks, parents = [hist[-1], *tokens(rng, kw, 8)], random_tree(rng, 9, 3)
    lg = e.step_tree([seq] * 9, toks, parents, [11] * 9, logits=True)[0]
    recent = [hist + [toks[i] for i in path[1:]] for path in paths_of(parents)]
    picks = []
    for x, r in zip(lg, recent):
        apply_repetition_penalty(x, r, 1.3)
        picks.append(int(np.argmax(x)))
    toks2 = [toks[0]] + [picks[parents[i]] if i % 3 else toks[i] for i in range(1, 9)]
    e.step_tree([seq] * 9, toks2, parents, [11] * 9)
    recent = [hist + [toks2[i] for i in path[1:]] for path in paths_of(parents)]
    lg = e.read_logits(0, 9)
    picks = []
    for x, r in zip(lg, recent):
        apply_repetition_penalty(x, r, 1.3)
        picks.append(int(np.argmax(x)))
    assert e.accept_tree(SamplingParams(0.0, 0, 1.0, 1.3), recent) == [walk(toks2, parents, picks)]
    e.close()


@pytest.mark.parametrize("name", ["q8_llama", "q4_qwen2_tied_bias", "q4_gqa8_hd128", "q8_hd64_gqa3"])
def test_greedy_generation_with_trees(hip, name):
    """Trees from the text, from the model itself and from another model all give the greedy tokens."""
    from qraf_amd.engine import InferenceEngine
    tf, kw = transformer(name)
    rng = np.random.default_rng(4)
    prompt = tokens(rng, kw, 7) * 3
    want, sure = reference_stream(tf, prompt, 30)
    eng = InferenceEngine(tf, eos_token=None)
    other = upload(oracle_model(SMALL[name][0], 99), SMALL[name][0], max_batch=16)
    for draft in (None, other, tf):
        for depth, width in ((0, 1), (1, 1), (3, 2), (3, 5), (15, 1), (1, 15)):
            got = eng.generate_tree(prompt, max_tokens=30, depth=depth, width=width, draft=draft)
            assert len(got) == 30 and got[:sure] == want[:sure], (depth, width, draft is not None)
    other.engine.close()
    tf.engine.close()


def test_trees_of_the_model_itself_are_accepted(hip):
    """Its own most likely tokens are the greedy ones: every depth is accepted, a step a depth + 1 tokens."""
    from qraf_amd.engine import InferenceEngine
    tf, kw = transformer("q8_hd64_gqa3")
    prompt = tokens(np.random.default_rng(5), kw, 9)
    eng = InferenceEngine(tf, eos_token=None)
    tf.engine.stats(reset=True)
    eng.generate_tree(prompt, 25, depth=4, width=2, draft=tf)
    # the prompt in a step, 5 times 4 drafting steps and the target's, and before each the draft's missing tokens
    assert tf.engine.stats()["steps"] <= 1 + 5 * 6 + 2
    tf.engine.close()


def test_generation_with_trees_stops_and_ends(hip):
    from qraf_amd.engine import InferenceEngine
    tf, kw = transformer("q8_llama", max_batch=32)
    short, _ = transformer("q8_llama", max_batch=16, max_seq=24)
    prompt = tokens(np.random.default_rng(5), kw, 5)
    want, sure = reference_stream(tf, prompt, 40)
    eng = InferenceEngine(tf, eos_token=None)
    stop = want[min(5, sure - 1)]
    free = tf.engine.free_pages(), short.engine.free_pages()
    assert eng.generate_tree(prompt, 12, stop_tokens=[stop]) == want[:want.index(stop)]
    assert eng.generate_tree(prompt, 0) == []
    assert len(eng.generate_tree(prompt, 1)) == 1
    got = eng.generate_tree(prompt, 40, depth=3, width=4, draft=short)  # past the draft model's last position
    assert len(got) == 40 and got[:sure] == want[:sure]
    for draft in (None, tf):
        assert len(eng.generate_tree(prompt, 128 - len(prompt), depth=5, width=2, draft=draft)) == 128 - len(prompt)
    assert (tf.engine.free_pages(), short.engine.free_pages()) == free
    for bad in (dict(depth=32, width=1), dict(depth=4, width=8), dict(depth=-1), dict(width=0)):
        with pytest.raises(ValueError):
            eng.generate_tree(prompt, 3, **bad)
    with pytest.raises(ValueError):
        eng.generate_tree([], 3)
    short.engine.close()
    tf.engine.close()


def test_sampled_generation_with_trees_runs(hip):
    from qraf_amd.engine import InferenceEngine, SamplingConfig
    tf, kw = transformer("q8_hd64_gqa3")
    other, _ = transformer("q8_hd64_gqa3", max_batch=16)
    prompt = tokens(np.random.default_rng(8), kw, 9)
    eng = InferenceEngine(tf, eos_token=None)
    for draft in (None, other):
        for penalty in (1.0, 1.1):
            s = SamplingConfig(0.9, 40, 0.95, penalty, seed=77)
            a = eng.generate_tree(prompt, 25, sampling=s, draft=draft, depth=3)
            assert len(a) == 25 and all(0 <= t < kw["vocab"] for t in a)
            assert eng.generate_tree(prompt, 25, sampling=s, draft=draft, depth=3) == a  # the seed's stream
    other.engine.close()
    tf.engine.close()


@pytest.mark.parametrize("name", ["q8_llama", "f32_llama"])
def test_scores_of_a_text(hip, name):
    """Engine.logprobs and InferenceEngine.score against the logits of the positions; the bar of logits, twice (a token's
    and the sum's), and ranks where no other logit is that near."""
    from qraf_amd.engine import InferenceEngine
    tf, kw = transformer(name, max_batch=8)
    text = tokens(np.random.default_rng(9), kw, 21)
    got = InferenceEngine(tf, eos_token=None).score(text, top=5)
    tf.reset()
    for i, t in enumerate(text[:-1]):
        lg = tf.forward(t, i).astype(np.float64)
        lp = lg - lg.max() - np.log(np.exp(lg - lg.max()).sum())
        bar = 2 * (1e-4 + 1e-3 * np.abs(lg).max())
        assert abs(got["logprobs"][i] - lp[text[i + 1]]) <= bar
        assert abs(got["entropies"][i] + (np.exp(lp) * lp).sum()) <= bar * (1 + np.abs(lp).max())
        order = np.argsort(-lg, kind="stable")
        assert np.abs(got["top_logprobs"][i] - lp[order[:5]]).max() <= bar
        if np.diff(-np.sort(-lg)[:6]).max() < -bar:
            assert list(got["top_tokens"][i]) == list(order[:5])
        near = np.abs(lg - lg[text[i + 1]]) <= bar
        low = int((lg > lg[text[i + 1]] + bar).sum())
        assert low <= got["ranks"][i] <= low + near.sum()
    assert all(len(v) == 20 for v in got.values())
    tf.engine.close()


def test_logprobs_of_a_step(hip):
    tf, kw = transformer("q8_hd64_gqa3")
    e, V = tf.engine, kw["vocab"]
    seq = e.seq_create()
    lg = e.step([seq] * 5, [3, 1, 4, 1, 5], range(5), logits=True)[0].astype(np.float64)
    lp = lg - lg.max(1, keepdims=True)
    lp -= np.log(np.exp(lp).sum(1, keepdims=True))
    got = e.logprobs([7, 0, V - 1], top=3, row0=1)
    order = np.argsort(-lg, axis=1, kind="stable")
    for i, t in enumerate([7, 0, V - 1]):
        assert abs(got["logprobs"][i] - lp[1 + i, t]) <= 2.0 ** -19 * (1 + abs(lp[1 + i, t]))
        assert got["ranks"][i] == int(np.nonzero(order[1 + i] == t)[0][0])
    assert np.array_equal(got["top_tokens"], order[1:4, :3])
    only = e.logprobs(rows=5)
    assert set(only) == {"entropies"} and np.abs(only["entropies"] + (np.exp(lp) * lp).sum(1)).max() <= 1e-4
    e.close()


def test_refusals(hip):
    from qraf_amd._lib import ERR_INVALID, ERR_STATE, HipError, SamplingParams
    tf, kw = transformer("q8_llama")
    e = tf.engine
    a, b = e.seq_create(), e.seq_create()
    greedy, hot = SamplingParams(0.0, 0, 1.0, 1.0), SamplingParams(1.0, 0, 1.0, 1.0)

    def refused(code, f):
        with pytest.raises(HipError) as x:
            f()
        assert x.value.code == code
    refused(ERR_STATE, lambda: e.accept_tree(greedy))  # no step yet
    refused(ERR_STATE, lambda: e.logprobs([1]))
    refused(ERR_INVALID, lambda: e.step_tree([a, a], [1, 2], [-1, 1], [0, 0]))  # its own parent
    refused(ERR_INVALID, lambda: e.step_tree([a, a, a], [1, 2, 3], [-1, 2, 0], [0] * 3))  # a later one
    refused(ERR_INVALID, lambda: e.step_tree([a, a], [1, 2], [-1, -1], [0, 0]))  # two roots
    refused(ERR_INVALID, lambda: e.step_tree([a, a], [1, 2], [0, 0], [0, 0]))
    refused(ERR_INVALID, lambda: e.step_tree([a, b], [1, 2], [-1, 0], [0, 0]))  # another sequence's
    refused(ERR_INVALID, lambda: e.step_tree([a, b, a], [1, 2, 3], [-1, -1, -1], [0] * 3))  # not side by side
    refused(ERR_INVALID, lambda: e.step_tree([a], [1], [-1], [1]))  # past its length
    refused(ERR_INVALID, lambda: e.step_tree([a], [1], [-1], [-1]))
    refused(ERR_INVALID, lambda: e.step_tree([a] * 2, [1, 2], [-1, 0], [2 ** 31 - 1] * 2))
    refused(ERR_INVALID, lambda: e.step_tree([a], [kw["vocab"]], [-1], [0]))
    refused(ERR_INVALID, lambda: e.step_tree([99], [1], [-1], [0]))
    refused(ERR_INVALID, lambda: e.step_tree([-1], [1], [-1], [0]))
    refused(ERR_INVALID, lambda: e.step_tree([a] * 17, [1] * 17, [-1] + [0] * 16, [0] * 17))
    assert e.seq_length(a) == 0 and e.seq_length(b) == 0
    e.step_tree([a, a], [1, 2], [-1, 0], [0, 0], want_logits=[1, 0])
    refused(ERR_STATE, lambda: e.accept_tree(greedy))  # a row without logits
    e.step_tree([a, a], [1, 2], [-1, 0], [0, 0])
    refused(ERR_INVALID, lambda: e.accept_tree(hot))  # needs uniforms
    with pytest.raises(ValueError):
        e.accept_tree(hot, uniforms=[0.5])
    assert e.accept_tree(greedy)
    refused(ERR_STATE, lambda: e.accept_tree(greedy))  # accepted before
    e.step_tree([a, a], [1, 2], [-1, 0], [0, 0])
    e.step([b], [1], [0])
    refused(ERR_STATE, lambda: e.accept_tree(greedy))  # another step between
    refused(ERR_STATE, lambda: e.logprobs([1, 2]))
    refused(ERR_INVALID, lambda: e.logprobs([1], top=65))
    refused(ERR_INVALID, lambda: e.logprobs([1], row0=-1))
    c = e.seq_create()
    e.set_repetition_penalty(c, 1.2)
    refused(ERR_STATE, lambda: e.step_tree([c], [1], [-1], [0]))
    e.step_async([b], [1], [1])
    refused(ERR_STATE, lambda: e.step_tree([a], [1], [-1], [0]))
    e.collect()
    e.seq_release(c)  # (steps keep their logits while some sequence has a penalty)
    e.set_keep_logits(False)
    e.step_tree([a], [1], [-1], [0])
    refused(ERR_STATE, lambda: e.accept_tree(greedy))
    refused(ERR_STATE, lambda: e.logprobs([1]))
    e.close()


@KINDS
def test_positions_of_drafts_are_not_read(hip, kv):
    """Whatever stands there, int32's ends among it: the same logits bit for bit, eager, captured and replayed, the same
    paths, and the same steps behind them."""
    from qraf_amd._lib import SamplingParams
    tf, kw = make("q8_hd64_gqa3", kv, max_batch=32)
    e, rng, greedy = tf.engine, np.random.default_rng(7), SamplingParams(0.0, 0, 1.0, 1.0)
    prompts, ends = [tokens(rng, kw, 19), tokens(rng, kw, 7)], [2 ** 31 - 1, -2 ** 31, -1, 10 ** 6]
    seqs = [[e.seq_create() for _ in prompts] for _ in range(2)]
    for p, s, r in zip(prompts, *seqs):
        feed(e, s, p)
        feed(e, r, p)
    bases = [len(p) for p in prompts]
    for turn in range(4):
        trees = [(tokens(rng, kw, n), random_tree(rng, n)) for n in (9, 4)]
        sid, tok, par, pos = flat(trees, seqs[0], bases)
        want = e.step_tree(sid, tok, par, pos, logits=True)[0]
        said = e.accept_tree(greedy)
        sid = flat(trees, seqs[1], bases)[0]
        pos = [p if up < 0 else ends[(i + turn) % 4] for i, (p, up) in enumerate(zip(pos, par))]
        assert np.array_equal(e.step_tree(sid, tok, par, pos, logits=True)[0], want)
        assert e.accept_tree(greedy) == said
        bases = [b + len(t) for b, t in zip(bases, said)]
    e.close()


def test_more_than_64_nodes_are_refused(hip):
    from qraf_amd._lib import ERR_INVALID, HipError
    tf, kw = transformer("q8_llama", max_batch=128)
    e = tf.engine
    a = e.seq_create()
    e.step_tree([a] * 64, [1] * 64, [-1] + [0] * 63, [0] * 64)
    with pytest.raises(HipError) as x:
        e.step_tree([a] * 65, [1] * 65, [-1] + [0] * 64, [0] * 65)
    assert x.value.code == ERR_INVALID
    e.close()


def test_a_pool_without_pages_for_a_tree(hip):
    """Nothing changes where the pool cannot hold the nodes."""
    from qraf_amd._lib import ERR_NOMEM, HipError
    kw, seed = SMALL["q8_llama"]
    tf = upload(oracle_model(kw, seed), kw, max_batch=64, num_pages=2)
    e = tf.engine
    a = e.seq_create()
    e.step([a] * 3, [1, 2, 3], range(3))
    with pytest.raises(HipError) as x:
        e.step_tree([a] * 40, [1] * 40, [-1] + [0] * 39, [3] * 40)
    assert x.value.code == ERR_NOMEM and e.seq_length(a) == 3 and e.free_pages() == 1
    e.step_tree([a] * 20, [1] * 20, [-1] + [0] * 19, [3] * 20)
    e.close()


def test_an_engine_of_one_row(hip):
    """A tree of its root alone: generate_tokens' steps."""
    from qraf_amd.engine import InferenceEngine
    tf, kw = transformer("q8_llama", max_batch=1)
    prompt = tokens(np.random.default_rng(2), kw, 5)
    want, sure = reference_stream(tf, prompt, 10)
    got = InferenceEngine(tf, eos_token=None).generate_tree(prompt, 10, depth=0, width=1)
    assert len(got) == 10 and got[:sure] == want[:sure]
    assert len(InferenceEngine(tf, eos_token=None).score(prompt)["logprobs"]) == 4
    tf.engine.close()


@KINDS
@pytest.mark.parametrize("rows", [1, 3])
def test_roots_alone_are_steps_as_any_other(hip, kv, rows):
    """The same logits bit for bit as qraf_engine_step's, eager, captured and replayed; their tokens, once."""
    from qraf_amd._lib import ERR_STATE, HipError, SamplingParams
    tf, kw = make("q4_gqa8_hd128", kv)
    e, rng = tf.engine, np.random.default_rng(4)
    params = SamplingParams(0.8, 10, 0.9, 1.0)
    seqs = [[e.seq_create() for _ in range(rows)] for _ in range(2)]
    for k in range(5):
        toks, uni = tokens(rng, kw, rows), rng.random(rows).astype(np.float32)
        want = e.step(seqs[0], toks, [k] * rows, logits=True)
        sampled = e.sample(params, uniforms=uni, rows=rows)
        with pytest.raises(HipError) as x:
            e.accept_tree(SamplingParams(0.0, 0, 1.0, 1.0))  # no trees
        assert x.value.code == ERR_STATE
        got = e.step_tree(seqs[1], toks, [-1] * rows, [k] * rows, logits=True)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        assert e.accept_tree(params, uniforms=uni) == [[int(t)] for t in sampled]
        with pytest.raises(HipError) as x:
            e.accept_tree(params, uniforms=uni)
        assert x.value.code == ERR_STATE
    e.close()


@pytest.mark.parametrize("kv", [po.F32, po.F16], ids=["f32", "f16"])
def test_a_sequence_released_ahead_of_its_acceptance(hip, kv):
    """The other's path goes on as if it were alone, and so does the sequence that takes the released pages."""
    from qraf_amd._lib import SamplingParams
    tf, kw = make("q4_gqa8_hd128", kv)
    e, rng, greedy = tf.engine, np.random.default_rng(6), SamplingParams(0.0, 0, 1.0, 1.0)
    prompt = tokens(rng, kw, 21)
    alone = e.seq_create()
    feed(e, alone, prompt[:-1])
    first = int(e.step([alone], [prompt[-1]], [20], argmax=True)[1][0])
    want = e.step([alone], [first], [21], logits=True)[0]
    a, b = e.seq_create(), e.seq_create()
    for s in (a, b):
        feed(e, s, prompt[:-1])
    rows = [prompt[-1], (first + 1) % kw["vocab"], first]
    e.step_tree([a] * 3 + [b] * 3, rows * 2, [-1, 0, 0, -1, 3, 3], [20] * 6)
    e.seq_release(a)
    got = e.accept_tree(greedy)
    assert [len(g) for g in got] == [2, 2] and got[1][0] == first
    c = e.seq_create()
    feed(e, c, prompt)
    check_logits(e.step([b], [first], [21], logits=True)[0], want)
    check_logits(e.step([c], [first], [21], logits=True)[0], want)
    e.close()

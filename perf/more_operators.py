"""Decoding with a tree of drafted tokens, and what a server says about a token beside it: four operators.

  attention  the nodes of each sequence's tree over its cache: all of the cache, and of the tree each node's own path
  accept     the walk along the tokens sampled behind the nodes: the accepted path and the token that follows it
  compact    the accepted path's keys and values to the positions where the sequence goes on, in every layer
  logprobs   log probabilities and ranks of given tokens, entropies and the top alternatives of rows of logits

listed() names the calls that are timed, draw() gives more of the same ranges, prepare() builds what a program
holds before the call, run() is one pass, work() what it cannot do without, exact() the same in 64 bits.  With
`own` false run() computes the operators from elementary products, sums, comparisons and indexing.
"""
import math

import numpy as np
import torch

own = False

PAGES = {"f32": 0, "f16": 1, "i8": 102}  # the library's page types
NODES = 64                               # positions behind its cache that a mask of a node speaks of


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one chat user of the small model, eight drafted nodes: the smallest call, pure latency
        dict(name="tree 1x8 at 300 f32", kind="attention", pages="f32", seqs=1, nodes=8, ragged=False, least=300,
             most=300, heads=9, kv_heads=3, head_dim=64, page=16),
        # one user with a long document and a wide tree
        dict(name="tree 1x64 at 8000 f16", kind="attention", pages="f16", seqs=1, nodes=64, ragged=False, least=8000,
             most=8000, heads=16, kv_heads=2, head_dim=128, page=16),
        # a batch that decodes with trees: contexts and trees of many sizes
        dict(name="tree 48x16 f16", kind="attention", pages="f16", seqs=48, nodes=16, ragged=True, least=128, most=4096,
             heads=16, kv_heads=2, head_dim=128, page=16),
        # long contexts on int8 pages
        dict(name="tree 24x26 at 8000 i8", kind="attention", pages="i8", seqs=24, nodes=26, ragged=True, least=3000,
             most=8000, heads=16, kv_heads=2, head_dim=128, page=16),
        # the reference's f32 cache, full trees
        dict(name="tree 8x64 at 2000 f32", kind="attention", pages="f32", seqs=8, nodes=64, ragged=False, least=777,
             most=2000, heads=16, kv_heads=2, head_dim=128, page=16),
        # one user's tree, and those of a batch
        dict(name="accept 1x8", kind="accept", seqs=1, nodes=8, vocab=49152),
        dict(name="accept 64x64", kind="accept", seqs=64, nodes=64, vocab=151936),
        # the small model's 30 layers for one user; a batch in 36 layers of fp16 pages
        dict(name="compact 1 of 30 f32", kind="compact", pages="f32", seqs=1, nodes=8, path=4, layers=30, kv_heads=3,
             head_dim=64, page=16, prefix=300),
        dict(name="compact 64 of 36 f16", kind="compact", pages="f16", seqs=64, nodes=32, path=6, layers=36, kv_heads=2,
             head_dim=128, page=16, prefix=500),
        # a drafter's rows: the alternatives that become the children of its nodes
        dict(name="logprobs 8x49152 top 4", kind="logprobs", rows=8, vocab=49152, top=4),
        # a batch's answers with their alternatives
        dict(name="logprobs 160x151936 top 20", kind="logprobs", rows=160, vocab=151936, top=20),
        # a text scored: every position's token, no alternatives
        dict(name="logprobs 512x151936", kind="logprobs", rows=512, vocab=151936, top=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "logprobs", "logprobs", "accept", "compact"])
    if kind == "logprobs":
        vocab = _log(rng, 1000, 151936)
        return dict(kind=kind, rows=min(_log(rng, 1, 512), 512 * 151936 // vocab), vocab=vocab,
                    top=min(vocab, rng.choice([0, 1, 4, 5, 8, 20, 64])))
    seqs, nodes = _log(rng, 1, 64), _log(rng, 1, NODES)
    if kind == "accept":
        return dict(kind=kind, seqs=seqs, nodes=nodes, vocab=_log(rng, 1000, 151936))
    hd, kv, page = rng.choice([64, 128]), rng.choice([1, 2, 3, 4, 8]), rng.choice([16, 16, 32])
    pages = rng.choice(["f32", "f16", "i8"])
    if kind == "compact":
        # at most the largest listed case's cache
        layers = _log(rng, 1, 36)
        seqs = max(1, min(seqs, (36 * 64 * 2 * 128 * 48 * 2) // (layers * kv * hd * (nodes + page) * 4)))
        return dict(kind=kind, pages=pages, seqs=seqs, nodes=nodes, path=rng.randint(1, min(nodes, 12)), layers=layers,
                    kv_heads=kv, head_dim=hd, page=page, prefix=_log(rng, 1, 4000))
    group, most = rng.choice([1, 2, 3, 4, 6, 8]), _log(rng, 24, 8000)
    # at most the largest listed case's query rows x positions, and its cache
    seqs = max(1, min(seqs, 1024 // nodes, (8 * 64 * 1400 * 16 * 128) // (nodes * most * kv * group * hd)))
    return dict(kind=kind, pages=pages, seqs=seqs, nodes=nodes, ragged=rng.random() < 0.5, least=rng.randint(0, most),
                most=most, heads=kv * group, kv_heads=kv, head_dim=hd, page=page)


# ------------------------------------------------------------------ inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, std=1.0):
    return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g)


def _counts(case, r):
    """Nodes of each sequence: as many in all for every seed."""
    n, s = case["nodes"], case["seqs"]
    return r.permutation(n - np.arange(s) % (n // 2 + 1) if case.get("ragged") else np.full(s, n))


def _trees(case, r):
    """(first row of each sequence, every row's parent within its sequence, every row's path as bits), on the host.
    A node's parent is one of the eight before it: wide and deep trees."""
    count = _counts(case, r)
    starts = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    parents, paths = [], []
    for n in count:
        bits = []
        for i in range(n):
            p = -1 if i == 0 else int(r.integers(max(0, i - 8), i))
            parents.append(p)
            bits.append((bits[p] if p >= 0 else 0) | 1 << i)
        paths += bits
    return starts, np.array(parents, np.int32), np.array(paths, np.uint64).view(np.int64)


def _tables(r, positions, page, shared=0):
    """Pages of sequences with so many positions each, the first `shared` whole pages the same for all: a table
    [sequences][pages], and how many pages there are."""
    per = -(-np.asarray(positions) // page)
    total = int(shared + (per - shared).sum())
    ids = r.permutation(total).astype(np.int32)
    table, at = np.zeros((len(per), int(per.max())), np.int32), shared
    for i, n in enumerate(per):
        table[i, :shared] = ids[:shared]
        table[i, shared:n] = ids[at:at + n - shared]
        at += n - shared
    return table, total


def _pools(g, case, *shape):
    """K and V in logical form [...][pages][kv heads][position][dim], int8 with a scale for each position."""
    kv = []
    for _ in range(2):
        if case["pages"] == "i8":
            b = (_normal(g, *shape) * 40).round().clamp(-127, 127)
            kv.append((b, torch.empty(shape[:-1], device="cuda").uniform_(0.01, 0.04, generator=g)))
        else:
            t = _normal(g, *shape)
            kv.append((t.half() if case["pages"] == "f16" else t, None))
    return kv


def _page_bytes(case, t, sc, v):
    """Such a pool as the library's pages: V of fp16 and int8 pages lies dimension-major, int8 pages end in a scale
    per position."""
    if case["pages"] == "f32":
        return t
    t = t.transpose(-2, -1) if v else t
    if case["pages"] == "f16":
        return t.contiguous()
    lead = t.shape[:-2]
    return torch.cat([t.to(torch.int8).reshape(*lead, -1).view(torch.uint8), sc.contiguous().view(torch.uint8)],
                     -1).contiguous()


def _attention_inputs(case, seed):
    c, r, g = case, np.random.default_rng(seed), _generator(seed)
    starts, _, paths = _trees(c, r)
    base = r.integers(c["least"], c["most"] + 1, c["seqs"]).astype(np.int32)
    table, pages = _tables(r, base + np.diff(starts), c["page"])
    q = _normal(g, int(starts[-1]), c["heads"], c["head_dim"])
    kv = _pools(g, c, pages, c["kv_heads"], c["page"], c["head_dim"])
    return starts, paths, base, table, q, kv


def _accept_inputs(case, seed):
    """Trees whose nodes' drafts are tokens, and a token sampled behind each node: mostly one of its children's."""
    c, r = case, np.random.default_rng(seed)
    starts, parents, _ = _trees(c, r)
    drafts = r.integers(0, c["vocab"], parents.size).astype(np.int32)
    picks = r.integers(0, c["vocab"], parents.size).astype(np.int32)
    first = np.repeat(starts[:-1], np.diff(starts))
    for i in r.permutation(parents.size):
        if parents[i] >= 0 and r.random() < 0.7:
            picks[first[i] + parents[i]] = drafts[i]
    return starts, parents, drafts, picks


def _compact_inputs(case, seed):
    """Caches whose first pages are one prompt's, and behind it the nodes of a tree; the accepted path of each
    sequence: its root and path - 1 nodes more."""
    c, r, g = case, np.random.default_rng(seed), _generator(seed)
    n = c["nodes"]
    starts = (np.arange(c["seqs"] + 1) * n).astype(np.int32)
    path = np.full((c["seqs"], n), -1, np.int32)
    path[:, 0] = 0
    for row in path:
        row[1:c["path"]] = np.sort(r.choice(n - 1, c["path"] - 1, replace=False) + 1) if c["path"] > 1 else 0
    base = (c["prefix"] + r.integers(0, c["page"], c["seqs"])).astype(np.int32)
    # (every sequence has the pages that the longest needs)
    table, pages = _tables(r, np.full(c["seqs"], c["prefix"] + c["page"] - 1 + n), c["page"], c["prefix"] // c["page"])
    kv = _pools(g, c, c["layers"], pages, c["kv_heads"], c["page"], c["head_dim"])
    return starts, path, base, table, kv


def _logprobs_inputs(case, seed):
    """A model's logits, one plausible token in five hundred above a broad rest, and tokens drawn from them."""
    c, g = case, _generator(seed)
    x = _normal(g, c["rows"], c["vocab"], std=1.5)
    x += 10.0 * torch.rand(x.shape, device="cuda", generator=g).pow_(400)
    gumbel = -torch.log(-torch.log(torch.rand(x.shape, device="cuda", generator=g).clamp_(1e-20, 0.9999999)))
    return x, torch.argmax(gumbel.add_(x), 1).to(torch.int32)


def prepare(case, seed):
    c = case
    if c["kind"] == "attention":
        starts, paths, base, table, q, kv = _attention_inputs(c, seed)
        s = dict(q=q, out=torch.empty_like(q), max_ctx=c["most"] + c["nodes"])
        s["table"] = np.zeros((c["seqs"], -(-s["max_ctx"] // c["page"])), np.int32)
        s["table"][:, :table.shape[1]] = table
        s.update(starts=starts, paths=paths, base=base)
    elif c["kind"] == "accept":
        starts, parents, drafts, picks = _accept_inputs(c, seed)
        s = dict(starts=starts, parents=parents, drafts=drafts, picks=picks)
        s["accepted"] = torch.empty(c["seqs"], dtype=torch.int32, device="cuda")
        s["path"], s["tokens"] = (torch.empty(parents.size, dtype=torch.int32, device="cuda") for _ in range(2))
    elif c["kind"] == "compact":
        starts, path, base, table, kv = _compact_inputs(c, seed)
        s = dict(starts=starts, path=path.reshape(-1), base=base, table=table)
    else:
        x, tokens = _logprobs_inputs(c, seed)
        s = dict(logits=x, tokens=tokens)
        s["logprobs"], s["entropies"] = (torch.empty(c["rows"], device="cuda") for _ in range(2))
        s["ranks"] = torch.empty(c["rows"], dtype=torch.int32, device="cuda")
        s["top_logprobs"] = torch.empty(c["rows"], c["top"], device="cuda")
        s["top_tokens"] = torch.empty(c["rows"], c["top"], dtype=torch.int32, device="cuda")
    if c["kind"] in ("attention", "compact"):
        s["k"], s["v"] = (_page_bytes(c, t, sc, i) for i, (t, sc) in enumerate(kv))
    s = {name: torch.from_numpy(a).cuda() if isinstance(a, np.ndarray) else a for name, a in s.items()}
    torch.cuda.synchronize()
    s["case"] = dict(case)
    return s


# ------------------------------------------------------------------ one pass, plain

def _plain_values(s, t, v):
    """A page pool [pages][kv heads][position][dim] in 32 bits from its bytes."""
    c = s["case"]
    if c["pages"] == "f32":
        return t
    if c["pages"] == "f16":
        return t.float().transpose(2, 3) if v else t.float()
    split = c["page"] * c["head_dim"]
    b, sc = t[..., :split].view(torch.int8).float(), t[..., split:].contiguous().view(torch.float32)
    shape = (-1, c["kv_heads"], c["page"], c["head_dim"])
    b = b.view(-1, c["kv_heads"], c["head_dim"], c["page"]).transpose(2, 3) if v else b.view(shape)
    return b * sc.unsqueeze(3)


def _sequences(s):
    """Every row's sequence, and its place there."""
    row = torch.arange(s["rows"] if "rows" in s else s["paths"].numel(), device="cuda")
    seq = torch.bucketize(row, s["starts"][1:].long(), right=True)
    return seq, row - s["starts"][seq].long()


def _plain_attention(s):
    c, table = s["case"], s["table"].long()
    n, hkv, hd, per = c["seqs"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    k, v = (_plain_values(s, s[name], name == "v")[table].transpose(1, 2).reshape(n, hkv, -1, hd) for name in "kv")
    seq, node = _sequences(s)
    q = torch.zeros(n, c["nodes"], c["heads"], hd, device="cuda")  # a sequence's rows side by side
    q[seq, node] = s["q"]
    q = q.view(n, c["nodes"], hkv, per, hd).transpose(1, 2).reshape(n, hkv, -1, hd)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(hd))
    behind = torch.arange(k.shape[2], device="cuda") - s["base"].unsqueeze(1)  # the tree's positions, from 0
    bits = torch.zeros(n, c["nodes"], dtype=torch.int64, device="cuda")
    bits[seq, node] = s["paths"]
    ahead = behind.unsqueeze(1)
    mine = (bits.unsqueeze(2) >> ahead.clamp(0, NODES - 1)) & 1
    sees = (ahead < 0) | ((ahead < NODES) & (mine == 1))
    sees = sees.view(n, 1, c["nodes"], 1, -1).expand(-1, -1, -1, per, -1).reshape(n, 1, c["nodes"] * per, -1)
    score.masked_fill_(~sees, -math.inf)
    p = torch.exp(score - score.amax(3, keepdim=True).clamp_(min=-3e38))  # (rows of no node see nothing)
    o = torch.matmul(p, v) / p.sum(3, keepdim=True)
    return o.view(n, hkv, c["nodes"], per, hd).transpose(1, 2).reshape(n, c["nodes"], c["heads"], hd)[seq, node]


def _plain_accept(s):
    c, n = s["case"], s["case"]["nodes"]
    shape = (c["seqs"], n)  # (as many nodes in every sequence)
    parents, drafts, picks = (s[name].long().view(shape) for name in ("parents", "drafts", "picks"))
    up = parents.clamp(min=0)
    good = (picks.gather(1, up) == drafts) & (parents >= 0)
    # of children with one draft the first
    same = (up.unsqueeze(2) == up.unsqueeze(1)) & good.unsqueeze(1)
    earlier = torch.tril(torch.ones(n, n, dtype=torch.bool, device="cuda"), -1)
    good &= ~(same & earlier).any(2)
    good[:, 0] = True
    # a node is reached over nodes that all are good: good steps, doubled until they span the deepest path
    step = torch.zeros(c["seqs"], n, n, device="cuda").scatter_(2, up.unsqueeze(2), 1.0) * good.unsqueeze(2)
    step[:, 0] = 0.0
    step[:, 0, 0] = 1.0
    twice = lambda x: torch.matmul(x, x)  # noqa: E731
    reached = twice(twice(twice(twice(twice(twice(step))))))[:, :, 0] > 0
    node = torch.arange(n, device="cuda").expand(shape)
    path = torch.where(reached, node, n).sort(1).values
    length = reached.sum(1, keepdim=True)
    last = path.gather(1, length - 1)
    tokens = torch.where(node + 1 < length, drafts.gather(1, path.roll(-1, 1).clamp(max=n - 1)),
                         torch.where(node + 1 == length, picks.gather(1, last), -1))
    path = torch.where(path < n, path, -1)
    return tuple(x.to(torch.int32) for x in (length[:, 0] - 1, path.reshape(-1), tokens.reshape(-1)))


def _plain_compact(s):
    c, ps, table = s["case"], s["case"]["page"], s["table"].long()
    to = torch.arange(c["nodes"], device="cuda").expand(c["seqs"], -1)
    path = s["path"].long().view(c["seqs"], -1)
    base = s["base"].long().unsqueeze(1)
    src, dst = base + torch.where(path < 0, to, path), base + to  # (behind the path: a position onto itself)
    ps_src, ps_dst = table.gather(1, src // ps), table.gather(1, dst // ps)
    views = [(s["k"], False), (s["v"], True)]
    if c["pages"] == "i8":
        split, shape = ps * c["head_dim"], (c["layers"], -1, c["kv_heads"])
        views = [(s["k"][..., :split].unflatten(-1, (ps, -1)), False), (s["v"][..., :split].unflatten(-1, (-1, ps)), True),
                 (s["k"][..., split:].unflatten(-1, (ps, 4)), False), (s["v"][..., split:].unflatten(-1, (ps, 4)), False)]
    elif c["pages"] == "f32":
        views = [(s["k"], False), (s["v"], False)]
    [_moved(t.transpose(-2, -1) if turned else t, ps_src, src % ps, ps_dst, dst % ps) for t, turned in views]
    return s["k"], s["v"]


def _moved(t, page_src, off_src, page_dst, off_dst):
    t[:, page_dst, :, off_dst] = t[:, page_src, :, off_src]


def _plain_logprobs(s):
    c, x, at = s["case"], s["logits"], s["tokens"].long().unsqueeze(1)
    d = x - x.amax(1, keepdim=True)
    w = torch.exp(d)
    total = w.sum(1, keepdim=True, dtype=torch.float64)
    log_total = torch.log(total)
    mine = x.gather(1, at)
    index = torch.arange(c["vocab"], device="cuda")
    ranks = ((x > mine) | ((x == mine) & (index < at))).sum(1)
    logprobs = d.gather(1, at).double() - log_total
    entropies = log_total - (w * d).sum(1, keepdim=True, dtype=torch.float64) / total
    out = [logprobs[:, 0].float(), ranks.to(torch.int32), entropies[:, 0].float()]
    if c["top"]:
        top, index = torch.sort(d, dim=1, descending=True, stable=True)  # ties: the lowest index first
        out += [index[:, :c["top"]].to(torch.int32), (top[:, :c["top"]].double() - log_total).float()]
    return tuple(out)


# ------------------------------------------------------------------ one pass

_library = []


def _lib():
    """The library and its call(), loaded on first use."""
    if not _library:
        from qraf_amd import _lib as library
        from qraf_amd.backend import backend_init
        backend_init(0)
        _library.extend([library.lib, library.call])
    return _library


def _workspace(s, size, *shape):
    if "workspace" not in s:  # kept with the state, as a program keeps it between calls
        s["workspace"] = torch.empty(max(int(size(*shape)), 16), dtype=torch.uint8, device="cuda")
    return s["workspace"].data_ptr(), s["workspace"].numel()


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"attention": _plain_attention, "accept": _plain_accept, "compact": _plain_compact,
                "logprobs": _plain_logprobs}[c["kind"]](s)
    lib, call = _lib()
    if c["kind"] == "attention":
        rows, h, hkv, hd, most = s["q"].shape[0], c["heads"], c["kv_heads"], c["head_dim"], s["max_ctx"]
        ws, size = _workspace(s, lib.qraf_hip_tree_attention_workspace_bytes, rows, c["seqs"], h, hkv, hd, most)
        call("qraf_hip_tree_attention_dev", s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), PAGES[c["pages"]],
             s["table"].data_ptr(), s["table"].shape[1], s["base"].data_ptr(), s["starts"].data_ptr(),
             s["paths"].data_ptr(), rows, c["seqs"], h, hkv, hd, c["page"], 1.0 / math.sqrt(hd), most,
             s["out"].data_ptr(), ws, size, None)
        return s["out"]
    if c["kind"] == "accept":
        call("qraf_hip_tree_accept_dev", s["picks"].data_ptr(), s["drafts"].data_ptr(), s["parents"].data_ptr(),
             s["starts"].data_ptr(), c["seqs"], s["picks"].numel(), s["accepted"].data_ptr(), s["path"].data_ptr(),
             s["tokens"].data_ptr(), None)
        return s["accepted"], s["path"], s["tokens"]
    if c["kind"] == "compact":
        call("qraf_hip_kv_compact_dev", s["k"].data_ptr(), s["v"].data_ptr(), PAGES[c["pages"]], c["layers"],
             s["k"].numel() * s["k"].element_size() // c["layers"], s["table"].data_ptr(), s["table"].shape[1],
             s["base"].data_ptr(), s["starts"].data_ptr(), s["path"].data_ptr(), c["seqs"], s["path"].numel(),
             c["kv_heads"], c["head_dim"], c["page"], None)
        return s["k"], s["v"]
    ws, size = _workspace(s, lib.qraf_hip_token_logprobs_workspace_bytes, c["rows"], c["vocab"], c["top"])
    top = [s[name].data_ptr() if c["top"] else None for name in ("top_tokens", "top_logprobs")]
    call("qraf_hip_token_logprobs_dev", s["logits"].data_ptr(), c["rows"], c["vocab"], s["tokens"].data_ptr(),
         s["logprobs"].data_ptr(), s["ranks"].data_ptr(), s["entropies"].data_ptr(), c["top"], *top, ws, size, None)
    out = (s["logprobs"], s["ranks"], s["entropies"])
    return out + (s["top_tokens"], s["top_logprobs"]) if c["top"] else out


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c = case
    if c["kind"] == "accept":
        rows = c["seqs"] * c["nodes"]
        return {"bytes": 20.0 * rows + 8.0 * c["seqs"], "flops": 2.0 * rows}
    if c["kind"] == "logprobs":
        return {"bytes": c["rows"] * (4.0 * c["vocab"] + 16 + 8 * c["top"]), "flops": 6.0 * c["rows"] * c["vocab"]}
    item = {"f32": 4, "f16": 2, "i8": 1}[c["pages"]] * c["head_dim"] + (4 if c["pages"] == "i8" else 0)
    if c["kind"] == "compact":
        # the root stays; of the rest, as many as are accepted move (a node that lies where it has to may stay too)
        moved = c["seqs"] * max(0, c["path"] - 1) * c["layers"] * c["kv_heads"]
        return {"bytes": 4.0 * moved * item + 4.0 * c["seqs"] * c["nodes"], "flops": float(moved)}
    rows = float(_counts(c, np.random.default_rng(0)).sum())
    positions = c["seqs"] * (c["least"] + c["most"]) / 2 + rows
    return {"bytes": 2 * positions * c["kv_heads"] * item + 2 * rows * c["heads"] * c["head_dim"] * 4,
            "flops": 4.0 * rows * ((c["least"] + c["most"]) / 2 + 1) * c["heads"] * c["head_dim"]}


# ------------------------------------------------------------------ 64 bits

def _exact_attention(case, seed):
    c = case
    starts, paths, base, table, q, kv = _attention_inputs(c, seed)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    per, scale = c["heads"] // c["kv_heads"], float(np.float32(1.0 / math.sqrt(c["head_dim"])))
    for i in range(c["seqs"]):
        a, b, n = int(starts[i]), int(starts[i + 1]), int(base[i])
        ids = torch.from_numpy(table[i].astype(np.int64)).cuda()
        most = n + b - a
        k, v = ((t[ids].double() if sc is None else t[ids].double() * sc[ids].double().unsqueeze(3))
                .transpose(0, 1).reshape(c["kv_heads"], -1, c["head_dim"])[:, :most] for t, sc in kv)
        sees = np.ones((b - a, most), bool)
        for j in range(b - a):
            for t in range(b - a):
                sees[j, n + t] = int(paths[a + j]) >> t & 1
        sees = torch.from_numpy(sees).cuda()
        for h in range(c["heads"]):
            w = q[a:b, h].double() @ k[h // per].T * scale
            w = torch.where(sees, w, -math.inf)
            w = torch.exp(w - w.amax(1, keepdim=True))
            out[a:b, h] = w @ v[h // per] / w.sum(1, keepdim=True)
    return out


def _exact_accept(case, seed):
    starts, parents, drafts, picks = _accept_inputs(case, seed)
    accepted, path, tokens = [], [], []
    for a, b in zip(starts[:-1], starts[1:]):
        at, way, said = 0, [0], []
        while True:
            token = picks[a + at]
            child = [i for i in range(b - a) if parents[a + i] == at and drafts[a + i] == token]
            said.append(token)
            if not child:
                break
            at = child[0]
            way.append(at)
        accepted.append(len(way) - 1)
        path += way + [-1] * (b - a - len(way))
        tokens += said + [-1] * (b - a - len(said))
    return tuple(torch.tensor(np.array(v, np.int32), device="cuda") for v in (accepted, path, tokens))


def _exact_compact(case, seed):
    c = case
    starts, path, base, table, kv = _compact_inputs(c, seed)
    for t in (x for pair in kv for x in pair if x is not None):
        before = t.clone()
        for i in range(c["seqs"]):
            for j in range(1, c["path"]):
                to, at = int(base[i]) + j, int(base[i]) + int(path[i, j])
                t[:, table[i, to // c["page"]], :, to % c["page"]] = before[:, table[i, at // c["page"]], :, at % c["page"]]
    return tuple(_page_bytes(c, t, sc, i) for i, (t, sc) in enumerate(kv))


def _exact_logprobs(case, seed):
    c = case
    x, tokens = _logprobs_inputs(c, seed)
    out = [[] for _ in range(5)]
    for i in range(c["rows"]):
        row, t = x[i].double(), int(tokens[i])
        order = torch.argsort(-x[i], stable=True)
        w = torch.exp(row - row[order[0]])
        p = w / w.sum()
        lp = (row - row[order[0]]) - torch.log(w.sum())
        out[0].append(lp[t])
        out[1].append((order == t).nonzero()[0, 0].to(torch.int32))
        out[2].append(-(p * lp).sum())
        out[3].append(order[:c["top"]].to(torch.int32))
        out[4].append(lp[order[:c["top"]]])
    return tuple(torch.stack(v) for v in (out if c["top"] else out[:3]))


def exact(case, seed):
    return {"attention": _exact_attention, "accept": _exact_accept, "compact": _exact_compact,
            "logprobs": _exact_logprobs}[case["kind"]](case, seed)

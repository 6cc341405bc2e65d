"""What decoding several tokens of a sequence at once, or many sequences with one prompt, needs: three operators.

  attention  rows of a group share the first positions of their caches (a system prompt, or, for the rows of one
             sequence - drafted tokens, a prompt chunk - the whole cache): those positions are read once for all
  probs      a Sampler's distribution (temperature, top-k, top-p) as probabilities over the vocabulary
  verify     drafted tokens accepted or rejected against the target's probabilities, and the token that follows

listed() names the calls that are timed, draw() gives more of the same ranges, prepare() builds what a program
holds before the call, run() is one pass, work() what it cannot do without, exact() the same in 64 bits.  With
`own` false run() computes the operators from elementary products, sums, comparisons and indexing.
"""
import ctypes
import math

import numpy as np
import torch

own = False

PAGES = {"f32": 0, "f16": 1, "i8": 102}  # the library's page types


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one chat user, four drafted tokens and the last accepted one: the smallest call, pure latency
        dict(name="draft rows 1x5 f32", kind="attention", pages="f32", groups=1, rows=5, causal=True, least=300,
             most=300, tail=0, heads=9, kv_heads=3, head_dim=64, page=16),
        # a batch that decodes speculatively: five rows of each sequence, ragged contexts
        dict(name="draft rows 48x5 f16", kind="attention", pages="f16", groups=48, rows=240, causal=True, least=128,
             most=4096, tail=0, heads=16, kv_heads=2, head_dim=128, page=16),
        # chat with one system prompt: every sequence has a tail of its own
        dict(name="shared 2048 + 512 f16", kind="attention", pages="f16", groups=1, rows=128, causal=False, least=2048,
             most=2048, tail=512, heads=16, kv_heads=2, head_dim=128, page=16),
        # several long shared documents, ragged, int8 pages
        dict(name="shared 5 of 8000 i8", kind="attention", pages="i8", groups=5, rows=96, causal=False, least=3000,
             most=8000, tail=256, heads=16, kv_heads=2, head_dim=128, page=16),
        # the reference's f32 cache, the small model, odd prefix
        dict(name="shared 1000 + 200 f32", kind="attention", pages="f32", groups=3, rows=61, causal=False, least=777,
             most=1000, tail=200, heads=9, kv_heads=3, head_dim=64, page=16),
        # prompt chunks: 128 rows of each of four sequences behind up to 2,000 positions
        dict(name="chunk 4x128 f32", kind="attention", pages="f32", groups=4, rows=512, causal=True, least=400,
             most=2000, tail=0, heads=16, kv_heads=2, head_dim=128, page=16),
        # the draft model's rows of one user: temperature alone, the small model's vocabulary
        dict(name="probs 4x49152", kind="probs", rows=4, vocab=49152, temperature=0.7, top_k=0, top_p=1.0),
        # the target's rows with the sampler's defaults
        dict(name="probs 160x151936 k40 p.9", kind="probs", rows=160, vocab=151936, temperature=0.8, top_k=40,
             top_p=0.9),
        # the nucleus of the whole vocabulary
        dict(name="probs 64x151936 p.95", kind="probs", rows=64, vocab=151936, temperature=1.0, top_k=0, top_p=0.95),
        # drafts from a prompt's own n-grams (no draft probabilities), one user
        dict(name="verify 1x4 49152", kind="verify", seqs=1, drafts=4, vocab=49152, temperature=0.8, given=False),
        # a batch with a draft model, ragged draft counts
        dict(name="verify 64x8 151936", kind="verify", seqs=64, drafts=8, vocab=151936, temperature=0.8, given=True),
    ]


def _single(x):
    """A parameter as the library takes it, in 32 bits."""
    return float(np.float32(x))


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "probs", "verify"])
    if kind == "attention":
        hd, kv, group = rng.choice([64, 128]), rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 6, 8])
        causal, most = rng.random() < 0.5, _log(rng, 24, 8000)
        tail = 0 if causal else rng.choice([0, _log(rng, 1, 512)])
        # at most the largest listed case's query rows x positions
        rows = max(1, min(_log(rng, 1, 512), (512 * 2000 * 16 * 128) // ((most + tail) * kv * group * hd)))
        groups = min(rows, _log(rng, 1, 48))
        return dict(kind=kind, pages=rng.choice(["f32", "f16", "i8"]), groups=groups, rows=rows, causal=causal,
                    least=rng.randint(1, most), most=most, tail=tail, heads=kv * group, kv_heads=kv, head_dim=hd,
                    page=rng.choice([16, 16, 32]))
    vocab = _log(rng, 1000, 151936)
    if kind == "probs":
        rows = max(1, min(_log(rng, 1, 256), 160 * 151936 // vocab))
        return dict(kind=kind, rows=rows, vocab=vocab, temperature=rng.choice([0.0, 0.5, 0.7, 1.0, 1.3]),
                    top_k=rng.choice([0, 0, 1, 20, 40, 400]), top_p=rng.choice([1.0, 0.8, 0.9, 0.95]))
    return dict(kind=kind, seqs=_log(rng, 1, 64), drafts=rng.randint(1, 8), vocab=vocab,
                temperature=rng.choice([0.6, 0.8, 1.0]), given=rng.random() < 0.6)


# ------------------------------------------------------------------ inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, std=1.0):
    return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g)


def _layout(case, seed):
    """(rows of each group, its shared positions, every row's positions, every row's pages), on the host.  A causal
    group is the rows of one sequence at consecutive positions, the last of them at the end of its cache."""
    c, r = case, np.random.default_rng(seed)
    cuts = np.sort(r.choice(c["rows"] - 1, c["groups"] - 1, replace=False) + 1) if c["groups"] > 1 else []
    if c["causal"] and c["rows"] % c["groups"] == 0:  # drafted rows and chunks: as many of each sequence
        cuts = np.arange(1, c["groups"]) * (c["rows"] // c["groups"])
    starts = np.concatenate([[0], cuts, [c["rows"]]]).astype(np.int32)
    count = np.diff(starts)
    prefix = r.integers(c["least"], c["most"] + 1, c["groups"]).astype(np.int32)
    if c["causal"]:
        prefix = np.maximum(prefix, count).astype(np.int32)
    group = np.repeat(np.arange(c["groups"]), count)
    if c["causal"]:
        ctx = prefix[group] - (starts[group + 1] - 1 - np.arange(c["rows"]))
    else:
        ctx = prefix[group] + r.integers(0, c["tail"] + 1, c["rows"])
    ctx, ps = ctx.astype(np.int32), c["page"]
    max_ctx = int(max(c["most"], int(count.max()))) + c["tail"]
    table = np.zeros((c["rows"], -(-max_ctx // ps)), np.int32)
    shared = prefix // ps  # whole pages; a row of a batch has the page that its own positions begin in to itself
    per = -(-ctx // ps)
    own_pages = np.zeros(c["rows"], np.int64) if c["causal"] else per - np.minimum(per, shared[group])
    group_pages = -(-prefix // ps) if c["causal"] else shared
    total = int(group_pages.sum() + own_pages.sum())
    ids = r.permutation(total).astype(np.int32)
    at = 0
    for j in range(c["groups"]):
        m = int(group_pages[j])
        table[starts[j]:starts[j + 1], :m] = ids[at:at + m]
        at += m
    for i in range(c["rows"]):
        m = int(own_pages[i])
        if m:
            table[i, shared[group[i]]:shared[group[i]] + m] = ids[at:at + m]
            at += m
    return starts, prefix, ctx, table, max_ctx, total


def _attention_inputs(case, seed):
    c, g = case, _generator(seed)
    starts, prefix, ctx, table, max_ctx, pages = _layout(c, seed)
    q = _normal(g, c["rows"], c["heads"], c["head_dim"])
    shape = (pages, c["kv_heads"], c["page"], c["head_dim"])
    kv = []
    for _ in range(2):
        if c["pages"] == "i8":  # a cached head's values: bytes with a scale for each position
            b = (_normal(g, *shape) * 40).round().clamp(-127, 127)
            kv.append((b, torch.empty(shape[:3], device="cuda").uniform_(0.01, 0.04, generator=g)))
        else:
            t = _normal(g, *shape)
            kv.append((t.half() if c["pages"] == "f16" else t, None))
    if not c["causal"] and c["page"] > 1:  # where a shared prefix ends inside a page, each row's page has a copy
        ps = c["page"]
        group = np.repeat(np.arange(c["groups"]), np.diff(starts))
        part = np.nonzero((prefix[group] % ps > 0) & (ctx > (prefix[group] // ps) * ps))[0]
        if part.size:
            j = prefix[group[part]] // ps
            dst = torch.from_numpy(table[part, j].astype(np.int64)).cuda()
            src = torch.from_numpy(table[starts[group[part]], j].astype(np.int64)).cuda()
            keep = torch.from_numpy(prefix[group[part]] % ps).cuda()
            inside = (torch.arange(ps, device="cuda") < keep.unsqueeze(1)).view(-1, 1, ps, 1)
            for k, (t, sc) in enumerate(kv):
                t[dst] = torch.where(inside, t[src], t[dst])
                if sc is not None:
                    sc[dst] = torch.where(inside.squeeze(3), sc[src], sc[dst])
    return starts, prefix, ctx, table, max_ctx, q, kv


def _page_bytes(c, t, sc, v):
    """Positions x dims [pages][kv heads][position][dim] as the library's pages: V of fp16 and int8 pages lies
    dimension-major, int8 pages end in a scale per position."""
    if c["pages"] == "f32":
        return t
    t = t.transpose(2, 3) if v else t
    if c["pages"] == "f16":
        return t.contiguous()
    p = t.shape[0] * t.shape[1]
    return torch.cat([t.to(torch.int8).reshape(p, -1).view(torch.uint8),
                      sc.reshape(p, -1).contiguous().view(torch.uint8)], 1).contiguous()


def _logits(case, seed, rows):
    """A model's logits: one plausible token in five hundred above a broad rest."""
    g = _generator(seed)
    x = _normal(g, rows, case["vocab"], std=1.5)
    x += 10.0 * torch.rand(x.shape, device="cuda", generator=g).pow_(400)
    return x


def _verify_inputs(case, seed):
    c, r = case, np.random.default_rng(seed)
    # drafted tokens, from none to all of them, and the row behind the last: as many rows for every seed
    count = r.permutation(c["drafts"] - np.arange(c["seqs"]) % (c["drafts"] + 1)) + 1
    starts = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    rows = int(starts[-1])
    x, g = _logits(c, seed, rows), _generator(seed + 1)
    probs = torch.softmax(x / c["temperature"], 1)
    x += _normal(g, rows, c["vocab"], std=0.5)  # what a draft model makes of them
    gumbel = -torch.log(-torch.log(torch.rand(x.shape, device="cuda", generator=g).clamp_(1e-20, 0.9999999)))
    tokens = torch.argmax(x / c["temperature"] + gumbel, 1).to(torch.int32)
    draft = torch.softmax(x / c["temperature"], 1) if c["given"] else None
    accept = torch.rand(rows, device="cuda", generator=g)
    pick = torch.rand(c["seqs"], device="cuda", generator=g)
    return torch.from_numpy(starts).cuda(), probs, draft, tokens, accept, pick


def prepare(case, seed):
    c = case
    if c["kind"] == "attention":
        starts, prefix, ctx, table, max_ctx, q, kv = _attention_inputs(c, seed)
        k, v = (_page_bytes(c, t, sc, i) for i, (t, sc) in enumerate(kv))
        s = dict(q=q, k=k, v=v, max_ctx=max_ctx, out=torch.empty_like(q))
        for name, a in (("starts", starts), ("prefix", prefix), ("ctx", ctx), ("table", table)):
            s[name] = torch.from_numpy(a).cuda()
    elif c["kind"] == "probs":
        s = dict(logits=_logits(c, seed, c["rows"]))
        s["out"] = torch.empty_like(s["logits"])
    else:
        starts, probs, draft, tokens, accept, pick = _verify_inputs(c, seed)
        s = dict(starts=starts, probs=probs, draft=draft, tokens=tokens, accept=accept, pick=pick,
                 accepted=torch.empty(c["seqs"], dtype=torch.int32, device="cuda"), out=torch.empty_like(tokens))
    torch.cuda.synchronize()
    s["case"] = dict(case)
    return s


# ------------------------------------------------------------------ one pass

_library = []


def _lib():
    """The library and its call(), loaded on first use."""
    if not _library:
        from qraf_amd import _lib as library
        from qraf_amd.backend import backend_init
        backend_init(0)
        _library.extend([library.lib, library.call, library.SamplingParams])
    return _library


def _workspace(s, size, *shape):
    if "workspace" not in s:  # kept with the state, as a program keeps it between calls
        s["workspace"] = torch.empty(max(int(size(*shape)), 16), dtype=torch.uint8, device="cuda")
    return s["workspace"].data_ptr(), s["workspace"].numel()


def _plain_values(s, t, v):
    """A page pool [pages][kv heads][position][dim] in 32 bits from its bytes."""
    c = s["case"]
    shape = (-1, c["kv_heads"], c["page"], c["head_dim"])
    if c["pages"] == "f32":
        return t
    if c["pages"] == "f16":
        return t.float().transpose(2, 3) if v else t.float()
    split = c["page"] * c["head_dim"]
    b, sc = t[:, :split].view(torch.int8).float(), t[:, split:].contiguous().view(torch.float32)
    b = b.view(-1, c["kv_heads"], c["head_dim"], c["page"]).transpose(2, 3) if v else b.view(shape)
    return b * sc.view(-1, c["kv_heads"], c["page"], 1)


def _plain_attention(s):
    c, table = s["case"], s["table"].long()
    n, hkv, hd = c["rows"], c["kv_heads"], c["head_dim"]
    k, v = (_plain_values(s, s[name], name == "v")[table].transpose(1, 2).reshape(n, hkv, -1, hd) for name in "kv")
    q = s["q"].view(n, hkv, c["heads"] // hkv, hd)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(hd))
    inside = torch.arange(k.shape[2], device="cuda") < s["ctx"].unsqueeze(1)
    score.masked_fill_(~inside.view(n, 1, 1, -1), -math.inf)
    p = torch.exp(score - score.amax(3, keepdim=True))
    return (torch.matmul(p, v) / p.sum(3, keepdim=True)).view(n, c["heads"], hd)


def _plain_probs(s):
    c, x = s["case"], s["logits"]
    if not c["temperature"] > 0:
        at = (x == x.amax(1, keepdim=True)).to(torch.int8).argmax(1)  # the lowest index of the largest
        return torch.zeros_like(x).scatter_(1, at.unsqueeze(1), 1.0)
    x, at = torch.sort(x, dim=1, descending=True, stable=True)  # ties: the lowest index first
    p = torch.exp((x.double() - x[:, :1].double()) / _single(c["temperature"]))  # 64 bits: the nucleus' border
    if 0 < c["top_k"] < c["vocab"]:
        p[:, c["top_k"]:] = 0
    p /= p.sum(1, keepdim=True)
    if 0 < c["top_p"] < 1:
        p[torch.cumsum(p, 1) - p >= _single(c["top_p"])] = 0  # behind the first whose sum with those before reaches it
        p /= p.sum(1, keepdim=True)
    return torch.zeros(p.shape, device="cuda").scatter_(1, at, p.float())


def _plain_verify(s):
    c, first = s["case"], s["starts"][:-1].long()
    drafts = s["starts"][1:].long() - first - 1
    j = torch.arange(c["drafts"], device="cuda")
    rows = torch.minimum(first.unsqueeze(1) + j, (first + drafts).unsqueeze(1))
    x = s["tokens"].long()[rows]
    p = s["probs"][rows, x].double()  # 64 bits: products next to their border
    q = s["draft"][rows, x].double() if c["given"] else torch.ones_like(p)
    good = (s["accept"].double()[rows] * q < p) & (j < drafts.unsqueeze(1))
    accepted = torch.cumprod(good.long(), 1).sum(1)
    at = first + accepted  # the row that gives the next token
    rest, out = s["probs"][at].double(), s["tokens"].long()
    missed = accepted < drafts
    if c["given"]:
        less = (rest - torch.where(missed.unsqueeze(1), s["draft"][at].double(), 0.0)).clamp_(min=0)
    else:
        drafted = out[at].unsqueeze(1)
        less = rest.scatter(1, drafted, torch.where(missed.unsqueeze(1), 0.0, rest.gather(1, drafted)))
    rest = torch.where(less.sum(1, keepdim=True) > 0, less, rest)
    total = torch.cumsum(rest, 1)
    token = (total > (s["pick"].double() * total[:, -1]).unsqueeze(1)).to(torch.int8).argmax(1)
    mine = torch.repeat_interleave(torch.arange(c["seqs"], device="cuda"), drafts + 1, output_size=out.numel())
    behind = torch.arange(out.numel(), device="cuda") - at[mine]
    out = torch.where(behind < 0, out, torch.where(behind == 0, token[mine], -1))
    return accepted.to(torch.int32), out.to(torch.int32)


def run(state):
    s, c = state, state["case"]
    if not own:
        if c["kind"] == "attention":
            return _plain_attention(s)
        return _plain_probs(s) if c["kind"] == "probs" else _plain_verify(s)
    lib, call, Params = _lib()
    if c["kind"] == "attention":
        n, groups, h, hkv, hd, most = c["rows"], c["groups"], c["heads"], c["kv_heads"], c["head_dim"], s["max_ctx"]
        ws, size = _workspace(s, lib.qraf_hip_group_attention_workspace_bytes, n, groups, h, hkv, hd, most)
        call("qraf_hip_group_attention_dev", s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(),
             PAGES[c["pages"]], s["table"].data_ptr(), s["table"].shape[1], s["ctx"].data_ptr(),
             s["starts"].data_ptr(), s["prefix"].data_ptr(), n, groups, h, hkv, hd, c["page"], 1.0 / math.sqrt(hd),
             most, s["out"].data_ptr(), ws, size, None)
        return s["out"]
    if c["kind"] == "probs":
        ws, size = _workspace(s, lib.qraf_hip_sample_probs_workspace_bytes, c["rows"], c["vocab"])
        params = Params(c["temperature"], c["top_k"], c["top_p"], 1.0)
        call("qraf_hip_sample_probs_dev", s["logits"].data_ptr(), c["rows"], c["vocab"], ctypes.byref(params), None,
             None, 0, s["out"].data_ptr(), ws, size, None)
        return s["out"]
    ws, size = _workspace(s, lib.qraf_hip_verify_draft_workspace_bytes, c["seqs"], c["vocab"])
    call("qraf_hip_verify_draft_dev", s["probs"].data_ptr(), s["draft"].data_ptr() if c["given"] else None,
         s["tokens"].data_ptr(), s["starts"].data_ptr(), c["seqs"], s["tokens"].numel(), c["vocab"],
         s["accept"].data_ptr(), s["pick"].data_ptr(), s["accepted"].data_ptr(), s["out"].data_ptr(), ws, size, None)
    return s["accepted"], s["out"]


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c = case
    if c["kind"] == "attention":
        shared = (c["least"] + c["most"]) / 2
        rows = c["rows"]
        own_positions = 0.0 if c["causal"] else c["tail"] / 2
        item = {"f32": 4, "f16": 2, "i8": 1}[c["pages"]] * c["head_dim"] + (4 if c["pages"] == "i8" else 0)
        positions = c["groups"] * shared + rows * own_positions
        attended = rows * (shared + own_positions) - (rows * (rows / c["groups"] - 1) / 2 if c["causal"] else 0)
        return {"bytes": 2 * positions * c["kv_heads"] * item + 2 * rows * c["heads"] * c["head_dim"] * 4,
                "flops": 4.0 * max(attended, rows) * c["heads"] * c["head_dim"]}
    if c["kind"] == "probs":
        return {"bytes": 8.0 * c["rows"] * c["vocab"], "flops": 4.0 * c["rows"] * c["vocab"]}
    # the row that gives each sequence's next token, and the draft's where there is one
    return {"bytes": (8.0 if c["given"] else 4.0) * c["seqs"] * c["vocab"], "flops": 3.0 * c["seqs"] * c["vocab"]}


# ------------------------------------------------------------------ 64 bits

def _exact_attention(case, seed):
    c = case
    starts, prefix, ctx, table, _, q, kv = _attention_inputs(c, seed)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    per, scale = c["heads"] // c["kv_heads"], _single(1.0 / math.sqrt(c["head_dim"]))
    for i in range(c["rows"]):
        n = int(ctx[i])
        ids = torch.from_numpy(table[i, :-(-n // c["page"])].astype(np.int64)).cuda()
        k, v = ((t[ids].double() if sc is None else t[ids].double() * sc[ids].double().unsqueeze(3))
                .transpose(0, 1).reshape(c["kv_heads"], -1, c["head_dim"])[:, :n] for t, sc in kv)
        for h in range(c["kv_heads"]):
            w = q[i, h * per:(h + 1) * per].double() @ k[h].T * scale
            w = torch.exp(w - w.amax(1, keepdim=True))
            out[i, h * per:(h + 1) * per] = w @ v[h] / w.sum(1, keepdim=True)
    return out


def _exact_probs(case, seed):
    c = case
    x = _logits(c, seed, c["rows"])
    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    for i in range(c["rows"]):
        order = torch.argsort(-x[i], stable=True)
        if not c["temperature"] > 0:
            out[i, order[0]] = 1.0
            continue
        if 0 < c["top_k"] < c["vocab"]:
            order = order[:c["top_k"]]
        w = x[i, order].double() / _single(c["temperature"])
        w = torch.exp(w - w[0])  # (a softmax of 64-bit values has come out only 5e-8 from them)
        w = w / w.sum()
        if 0 < c["top_p"] < 1:
            last = int(torch.searchsorted(torch.cumsum(w, 0), _single(c["top_p"])))  # the first sum that reaches it
            order, w = order[:last + 1], w[:last + 1]
        out[i, order] = w / w.sum()
    return out


def _exact_verify(case, seed):
    c = case
    starts, probs, draft, tokens, accept, pick = _verify_inputs(c, seed)
    starts, accept, pick, drafted = starts.tolist(), accept.tolist(), pick.tolist(), tokens.tolist()
    accepted, out = [], []
    for i in range(c["seqs"]):
        row, end, given = starts[i], starts[i + 1] - 1, []
        while row < end:
            x = drafted[row]
            if not accept[row] * (float(draft[row, x]) if c["given"] else 1.0) < float(probs[row, x]):
                break
            given.append(x)
            row += 1
        w = probs[row].double()
        if row < end:
            if c["given"]:
                less = (w - draft[row].double()).clamp(min=0)
            else:
                less = w.clone()
                less[drafted[row]] = 0
            w = less if float(less.sum()) > 0 else w
        total = torch.cumsum(w, 0)
        given.append(int(torch.searchsorted(total, total[-1] * pick[i], right=True)))
        accepted.append(len(given) - 1)
        out += given + [-1] * (starts[i + 1] - starts[i] - len(given))
    return tuple(torch.tensor(v, dtype=torch.int32, device="cuda") for v in (accepted, out))


def exact(case, seed):
    return {"attention": _exact_attention, "probs": _exact_probs, "verify": _exact_verify}[case["kind"]](case, seed)

"""What the operators of trees of drafted tokens and of log probabilities refuse, before anything reaches the device."""
import pytest

from qraf_amd._lib import ERR_DTYPE, ERR_INVALID, lib

P = 4096  # never read: every call here is refused on the host


def attention(**change):
    a = dict(q=P, k=P, v=P, kv=1, table=P, max_pages=8, base=P, starts=P, masks=P, n=4, seqs=2, H=8, Hkv=2, hd=64,
             ps=16, scale=0.125, max_ctx=128, out=P, ws=P, size=1 << 40, stream=None)
    a.update(change)
    return lib.qraf_hip_tree_attention_dev(*a.values()), lib.qraf_hip_last_error()


@pytest.mark.parametrize("change", [
    dict(q=None), dict(k=None), dict(v=None), dict(table=None), dict(base=None), dict(starts=None), dict(masks=None),
    dict(out=None), dict(ws=None), dict(n=0), dict(n=-1), dict(n=1025), dict(seqs=0), dict(seqs=5), dict(H=7),
    dict(H=0), dict(H=1 << 17), dict(Hkv=0), dict(Hkv=-2), dict(hd=48), dict(hd=256), dict(hd=0), dict(ps=0),
    dict(max_pages=0), dict(max_ctx=0), dict(max_ctx=129), dict(max_ctx=(1 << 30) + 1, max_pages=1 << 27),
    dict(max_pages=1 << 30, ps=1 << 30, max_ctx=-5), dict(q=P + 4), dict(k=P + 8), dict(v=P + 2), dict(out=P + 4),
    dict(ws=P + 8), dict(masks=P + 4), dict(size=0)])
def test_tree_attention_refuses(change):
    rc, msg = attention(**change)
    assert rc == ERR_INVALID and msg.startswith(b"tree attention"), msg


def test_tree_attention_refuses_other_pages():
    assert attention(kv=10)[0] == ERR_DTYPE


def append(**change):
    a = dict(qkv=P, bias=None, n=4, H=8, Hkv=2, hd=64, pos=P, slots=P, seqs=P, rope=P, q=P, k=P, v=P, kv=1, table=P,
             max_pages=8, ps=16, stream=None)
    a.update(change)
    return lib.qraf_hip_tree_append_dev(*a.values()), lib.qraf_hip_last_error()


@pytest.mark.parametrize("change", [
    dict(qkv=None), dict(n=0), dict(n=-2), dict(H=0), dict(Hkv=0), dict(Hkv=-1), dict(hd=0), dict(hd=63),
    dict(pos=None), dict(slots=None), dict(seqs=None), dict(rope=None), dict(q=None), dict(k=None), dict(v=None),
    dict(table=None), dict(max_pages=0), dict(ps=0), dict(kv=102, ps=6), dict(kv=102, hd=130)])
def test_tree_append_refuses(change):
    rc, msg = append(**change)
    assert rc == ERR_INVALID and msg, msg


def test_tree_append_refuses_other_pages():
    assert append(kv=10)[0] == ERR_DTYPE


def accept(**change):
    a = dict(picks=P, draft=P, parents=P, starts=P, seqs=2, n=6, accepted=P, path=P, tokens=P, stream=None)
    a.update(change)
    return lib.qraf_hip_tree_accept_dev(*a.values()), lib.qraf_hip_last_error()


@pytest.mark.parametrize("change", [
    dict(picks=None), dict(draft=None), dict(parents=None), dict(starts=None), dict(accepted=None), dict(path=None),
    dict(tokens=None), dict(seqs=0), dict(seqs=-1), dict(seqs=65536), dict(n=0), dict(n=-4)])
def test_tree_accept_refuses(change):
    rc, msg = accept(**change)
    assert rc == ERR_INVALID and msg.startswith(b"tree_accept"), msg


def compact(**change):
    a = dict(k=P, v=P, kv=1, layers=2, layer_bytes=1 << 20, table=P, max_pages=8, base=P, starts=P, path=P, seqs=2,
             n=6, Hkv=2, hd=64, ps=16, stream=None)
    a.update(change)
    return lib.qraf_hip_kv_compact_dev(*a.values()), lib.qraf_hip_last_error()


@pytest.mark.parametrize("change", [
    dict(k=None), dict(v=None), dict(table=None), dict(base=None), dict(starts=None), dict(path=None), dict(layers=0),
    dict(layers=-1), dict(layer_bytes=(1 << 20) + 2), dict(k=P + 2), dict(v=P + 1), dict(seqs=0), dict(seqs=65536),
    dict(n=0), dict(Hkv=0), dict(Hkv=1 << 20), dict(hd=48), dict(hd=0), dict(ps=0), dict(max_pages=0),
    dict(max_pages=1 << 20, ps=1 << 20)])
def test_kv_compact_refuses(change):
    rc, msg = compact(**change)
    assert rc == ERR_INVALID and msg.startswith(b"kv_compact"), msg


def test_kv_compact_refuses_other_pages():
    assert compact(kv=10)[0] == ERR_DTYPE


def logprobs(**change):
    a = dict(logits=P, rows=2, vocab=100, tokens=P, lp=P, ranks=P, ent=P, top=5, tt=P, tl=P, ws=P, size=1 << 40,
             stream=None)
    a.update(change)
    return lib.qraf_hip_token_logprobs_dev(*a.values()), lib.qraf_hip_last_error()


@pytest.mark.parametrize("change", [
    dict(logits=None), dict(ws=None), dict(rows=0), dict(rows=-1), dict(rows=65536), dict(vocab=0),
    dict(vocab=(1 << 30) + 1), dict(tokens=None), dict(tokens=None, lp=None), dict(tokens=None, ranks=None),
    dict(top=-1), dict(top=65), dict(top=5, vocab=4), dict(tt=None), dict(tl=None), dict(ws=P + 8), dict(size=0)])
def test_token_logprobs_refuses(change):
    rc, msg = logprobs(**change)
    assert rc == ERR_INVALID and msg.startswith(b"token_logprobs"), msg


def test_workspace_queries_of_bad_shapes_are_zero():
    assert lib.qraf_hip_tree_attention_workspace_bytes(0, 1, 8, 2, 64, 128) == 0
    assert lib.qraf_hip_tree_attention_workspace_bytes(4, 1, 8, -2, 64, 128) == 0
    assert lib.qraf_hip_token_logprobs_workspace_bytes(0, 100, 5) == 0
    assert lib.qraf_hip_token_logprobs_workspace_bytes(3, 100, -1) == 0


@pytest.mark.parametrize("vocab", [8192, 8193, 39999, 40000, 98303, 98304, 151936])
def test_logprobs_workspace_grows_with_rows_and_alternatives(vocab):
    size = lib.qraf_hip_token_logprobs_workspace_bytes
    rows = [1, 2, 84, 85, 86, 87, 208, 209, 210, 211, 1024, 65535]
    for top in (0, 1, 64):
        sizes = [size(r, vocab, top) for r in rows]
        assert sizes == sorted(sizes) and sizes[0] > 0
        assert top == 0 or all(size(r, vocab, 0) <= s for r, s in zip(rows, sizes))

"""What the operators over shared positions, probabilities and drafts refuse, before anything reaches the device."""
import ctypes as C

import pytest

from qraf_amd._lib import ERR_DTYPE, ERR_INVALID, SamplingParams, lib

P = 4096  # never read: every call here is refused on the host


def group(**change):
    a = dict(q=P, k=P, v=P, kv=1, table=P, max_pages=8, ctx=P, starts=P, prefix=P, n=4, groups=2, H=8, Hkv=2, hd=64,
             ps=16, scale=0.125, max_ctx=128, out=P, ws=P, size=1 << 40, stream=None)
    a.update(change)
    return lib.qraf_hip_group_attention_dev(*a.values()), lib.qraf_hip_last_error()


@pytest.mark.parametrize("change", [
    dict(q=None), dict(k=None), dict(v=None), dict(table=None), dict(ctx=None), dict(starts=None), dict(prefix=None),
    dict(out=None), dict(ws=None), dict(n=0), dict(n=-1), dict(n=1025), dict(groups=0), dict(groups=5), dict(H=7),
    dict(H=0), dict(Hkv=0), dict(Hkv=-2), dict(hd=48), dict(hd=256), dict(hd=0), dict(ps=0), dict(max_pages=0),
    dict(max_ctx=0), dict(max_ctx=129), dict(max_pages=1 << 30, ps=1 << 30, max_ctx=-5), dict(size=0)])
def test_group_attention_refuses(change):
    rc, msg = group(**change)
    assert rc == ERR_INVALID and msg.startswith(b"group attention"), msg


@pytest.mark.parametrize("change", [dict(q=P + 4), dict(k=P + 8), dict(v=P + 2), dict(out=P + 4), dict(ws=P + 8),
                                    dict(max_ctx=(1 << 30) + 1, max_pages=1 << 27)])
def test_group_attention_refuses_alignments_and_lengths(change):
    rc, msg = group(**change)
    assert rc == ERR_INVALID and msg.startswith(b"group attention"), msg


@pytest.mark.parametrize("change", [dict(ws=P + 4), dict(rows=65536), dict(vocab=(1 << 30) + 1)])
def test_sample_probs_refuses_alignments_and_sizes(change):
    rc, msg = probs(**change)
    assert rc == ERR_INVALID and msg.startswith(b"sample_probs"), msg


@pytest.mark.parametrize("change", [dict(ws=P + 8), dict(n=65536), dict(vocab=(1 << 30) + 1)])
def test_verify_draft_refuses_alignments_and_sizes(change):
    rc, msg = verify(**change)
    assert rc == ERR_INVALID and msg.startswith(b"verify_draft"), msg


def test_group_attention_refuses_other_pages():
    assert group(kv=10)[0] == ERR_DTYPE


def test_workspace_queries_of_bad_shapes_are_zero():
    assert lib.qraf_hip_group_attention_workspace_bytes(0, 1, 8, 2, 64, 128) == 0
    assert lib.qraf_hip_group_attention_workspace_bytes(4, 1, 8, -2, 64, 128) == 0
    assert lib.qraf_hip_sample_probs_workspace_bytes(0, 100) == 0
    assert lib.qraf_hip_verify_draft_workspace_bytes(3, 0) == 0


def probs(**change):
    a = dict(logits=P, rows=2, vocab=100, params=C.byref(SamplingParams(1.0, 0, 1.0, 1.0)), recent=None, count=None,
             stride=0, probs=P, ws=P, size=1 << 40, stream=None)
    a.update(change)
    return lib.qraf_hip_sample_probs_dev(*a.values()), lib.qraf_hip_last_error()


@pytest.mark.parametrize("change", [dict(logits=None), dict(rows=0), dict(vocab=0), dict(params=None),
                                    dict(probs=None), dict(ws=None), dict(size=0),
                                    dict(params=C.byref(SamplingParams(1.0, 0, 1.0, 1.1)), recent=P, stride=4),
                                    dict(params=C.byref(SamplingParams(1.0, 0, 1.0, 1.1)), recent=P, count=P)])
def test_sample_probs_refuses(change):
    rc, msg = probs(**change)
    assert rc == ERR_INVALID and msg, msg


def verify(**change):
    a = dict(p=P, q=None, draft=P, starts=P, n=2, rows=6, vocab=100, u=P, v=P, acc=P, tok=P, ws=P, size=1 << 40,
             stream=None)
    a.update(change)
    return lib.qraf_hip_verify_draft_dev(*a.values()), lib.qraf_hip_last_error()


@pytest.mark.parametrize("change", [dict(p=None), dict(draft=None), dict(starts=None), dict(u=None), dict(v=None),
                                    dict(acc=None), dict(tok=None), dict(ws=None), dict(n=0), dict(rows=0),
                                    dict(vocab=0), dict(n=-3), dict(size=0)])
def test_verify_draft_refuses(change):
    rc, msg = verify(**change)
    assert rc == ERR_INVALID and msg.startswith(b"verify_draft"), msg

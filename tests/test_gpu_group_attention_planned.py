"""The calls of test_gpu_group_attention with a longer bound on the contexts (max_ctx, the page tables' width): a short
bound takes the one-launch form of small calls where the batch is small, a long one the planned form, whose results
the same values and tolerances hold."""
import numpy as np
import pytest

from tests import test_gpu_group_attention as calls

pytestmark = pytest.mark.gpu

for _name in dir(calls):
    if _name.startswith("test_"):
        globals()[_name] = getattr(calls, _name)


@pytest.fixture(autouse=True)
def long_bound(monkeypatch):
    plain = calls.Cache.__init__

    def init(self, *args, **kw):
        plain(self, *args, **kw)
        self.max_ctx = max(self.max_ctx, 2048)
        wide = np.zeros((self.n, -(-self.max_ctx // self.ps)), np.int32)
        wide[:, :self.table.shape[1]] = self.table
        self.table = wide
    monkeypatch.setattr(calls.Cache, "__init__", init)


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("heads", [(16, 2, 128), (9, 3, 64), (20, 1, 64)], ids=["16x2x128", "9x3x64", "20x1x64"])
@calls.KINDS
def test_chunk_rows_that_do_not_attend_to_a_bad_position(hip, kv, heads, bad):
    """Chunks of 40 rows (blocks of many columns) with an infinity or NaN in K or V of one position: the rows that end
    ahead of it are what they were, the others no numbers (K: an infinite score may also be a weight of 0 or 1)."""
    H, Hkv, hd = heads
    rng = np.random.default_rng(21)
    c = calls.Cache(rng, [(140, list(range(101, 141))), (29, [29])], Hkv, hd, 16, kv)
    q = calls.queries(rng, c.n, H, hd)
    clean = calls.Call(hip, c, q, H).run()
    calls.check(c, clean, q, H)
    for which in "KV":
        for at in (100, 119, 128, 139):
            a = getattr(c, which if kv != calls.I8 else which + "s")
            page = c.table[0, at // 16]
            keep = a[page].copy()
            if kv == calls.I8:
                a[page, :, at % 16] = bad
            else:
                a[page, :, at % 16, 5] = bad
            got = calls.Call(hip, c, q, H).run()
            a[page] = keep
            before = np.nonzero(c.ctx <= at)[0]
            assert np.array_equal(got[before], clean[before]), (which, at)
            after = np.setdiff1d(np.arange(40), before)
            if which == "V":
                assert not np.isfinite(got[after] if kv == calls.I8 else got[after][:, :, 5]).any(), at
            elif np.isnan(bad):
                assert np.isnan(got[after]).all(), at


@pytest.mark.parametrize("rows", [22, 24, 31, 43, 44])
def test_blocks_with_waves_without_columns(hip, rows):
    """Three query heads a KV head: blocks of 66, 72, 93, 129 - 128 and 132 - 128 columns, whose last waves have few
    or none, values of very different sizes in neighbouring positions."""
    rng = np.random.default_rng(rows)
    c = calls.Cache(rng, [(500, [500 - i for i in range(rows)]), (64, [70] * rows)], 2, 64, 16, calls.F32)
    for a in (c.K, c.V):
        a *= np.exp2(rng.integers(-30, 3, a.shape[:3] + (1,))).astype(np.float32)
    q = calls.queries(rng, c.n, 6, 64)
    calls.check(c, calls.Call(hip, c, q, 6).run(), q, 6)

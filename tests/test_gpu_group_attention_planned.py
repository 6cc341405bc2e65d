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

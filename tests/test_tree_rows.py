"""Where the rows of trees of drafted tokens lie (qraf_amd/csrc/tree_rows.h), on the host: tests/cpp/tree_rows_check,
built with AddressSanitizer and UndefinedBehaviorSanitizer, over seeded random trees.  The positions of rows that are
not their sequence's first are not read."""
import os
import re
import subprocess

import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")


@pytest.mark.parametrize("seed", [1, 2])
def test_places(seed):
    r = subprocess.run(["make", "-s", "-C", CPP, "tree_rows_check"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([os.path.join(CPP, "tree_rows_check"), str(seed), "300"], capture_output=True, text=True)
    assert r.returncode == 0 and not r.stderr, r.stdout + r.stderr[-3000:]
    past, poisoned = map(int, re.search(r"(\d+) places past int32, (\d+) poisoned", r.stdout).groups())
    assert past > 100 and poisoned > 10000

"""How attention by group cuts its jobs into pieces (qraf_amd/csrc/group_pieces.h), on the host: tests/cpp/
group_pieces_check, built with AddressSanitizer and UndefinedBehaviorSanitizer, over seeded random jobs up to 1,024 rows
of 2^30 positions, whose tiles together pass 32 bits."""
import os
import re
import subprocess

import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")


@pytest.mark.parametrize("seed", [1, 2])
def test_pieces(seed):
    r = subprocess.run(["make", "-s", "-C", CPP, "group_pieces_check"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([os.path.join(CPP, "group_pieces_check"), str(seed), "400"], capture_output=True, text=True)
    assert r.returncode == 0 and not r.stderr, r.stdout + r.stderr[-3000:]
    assert int(re.search(r"(\d+) past 2\^31", r.stdout).group(1)) >= 40

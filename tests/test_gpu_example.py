"""The decoding example at a budget below what it would protect."""

import os
import subprocess
import sys

import pytest

from conftest import REPO

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("budget", [1, 3, 5])
def test_example_with_a_small_budget(budget):
    res = subprocess.run([sys.executable, os.path.join(REPO, "examples", "tree_decode.py"), "--steps", "4", "--batch",
                          "2", "--drafts", "6", "--budget", str(budget)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]
    assert "(cut)" in res.stdout and f"cached [{budget}, {budget}] (cut)" in res.stdout

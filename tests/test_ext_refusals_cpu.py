"""The extension's own checks, whose texts hold numbers: they raise and do not end the process.  No GPU is needed, the
checks come before anything is launched; a child process makes the calls."""
import subprocess
import sys
from pathlib import Path

import pytest

from shift_b200.ops._ext import available

CALLS = """
import torch
from shift_b200.ops._ext import ext
one = torch.ones(300)
plan = ext().adamw_many_plan([one], [], [one.clone()], [], [one.clone()], [])
codes = torch.zeros(4, 16, dtype=torch.uint8).view(torch.float8_e4m3fn)
scale = torch.zeros(1, 4, 4, dtype=torch.uint8).view(torch.float8_e8m0fnu)
word = torch.zeros(1, dtype=torch.int32)
def adamw(grads):
    ext().adamw_many(plan, grads, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, 1, None, None, None)
def product(cols, scale=scale):
    ext().fp8_matmul(codes, scale, cols, codes, scale, cols, None, None, 0, False, False, word)
for call, text in ((lambda: adamw([]), "0 gradients for 1 "), (lambda: adamw([torch.ones(3)]), "300 elements"),
                   (lambda: product(17), "16 columns of codes, 17 "), (lambda: product(-1), "-1 are said"),
                   (lambda: product(16, scale[:, :3]), "[1, 3, 4]")):
    try:
        call()
    except ValueError as e:
        assert text in str(e), e
    else:
        raise AssertionError(text)
print("refused")
"""


@pytest.mark.skipif(not available(), reason="the extension is not built")
def test_a_refusal_with_numbers_raises():
    got = subprocess.run([sys.executable, "-c", CALLS], cwd=Path(__file__).parents[1], capture_output=True, text=True)
    assert got.returncode == 0 and got.stdout.strip() == "refused", got.stderr[-2000:]

"""The status word where the first call of a process is captured into a graph."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CODE = """
import torch
from shift_b200.ops import packed, objectives
from shift_b200.ops import _ext
z = torch.randn(8, 64, device="cuda")
labels = torch.zeros(8, dtype=torch.int32, device="cuda")
row = torch.zeros(8, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    loss, _ = objectives.policy_loss_fwd_bwd(z, labels, row, row)
assert _ext.check_status() == 0                # before the graph ever ran
word = _ext.status_word(z.device)
word[3] = 5                                    # a replay leaves the word alone: it may hold what another kernel reported
graph.replay()
torch.cuda.synchronize()
assert int(word[3]) == 5 and _ext.check_status() == 0
del graph, loss
torch.cuda.empty_cache()
assert _ext.check_status() == 0
"""


def test_first_call_under_capture():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    got = subprocess.run([sys.executable, "-c", CODE], env={**os.environ, "PYTHONPATH": root}, capture_output=True, text=True,
                         timeout=300)
    assert got.returncode == 0, got.stderr[-2000:]

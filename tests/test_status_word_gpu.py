"""GPU: the status word of a process whose first call is captured into a graph."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

START = """
import sys; sys.path[:0] = [%r, %r]
import importlib
import torch, flaggems_sglang_b200 as F
from flaggems_sglang_b200.quant import quantize_fp8_block
fm = importlib.import_module("flaggems_sglang_b200.ops.fused_moe")
d = torch.device("cuda:0")
x = torch.randn(40, 512, device=d).to(torch.bfloat16)
w, s = quantize_fp8_block(torch.randn(1, 256, 512, device=d)); w, s = w[0], s[0]
garbage = torch.full((1 << 22,), 77, dtype=torch.int32, device=d)      # what a word without a value would hold
del garbage
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = F.fp8_block_linear(x, w, s)
word = fm._status_word(d)
""" % (str(ROOT), str(ROOT / "flaggems-sglang_b200"))


def _run(code):
    r = subprocess.run([sys.executable, "-c", START + code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stdout + r.stderr


def test_eager_calls_before_the_first_replay(cuda_device):
    """The word is zero before any replay, so no call takes it for a time-out and a time-out can be written into it."""
    _run("""
assert int(word.item()) == 0
want = F.fp8_block_linear(x, w, s)
for _ in range(2 * fm.STATUS_COPY_EVERY + 2):
    z = F.fp8_block_linear(x, w, s)
    torch.cuda.synchronize()
F.check_status()
g.replay(); torch.cuda.synchronize()
assert torch.equal(y, want) and torch.equal(z, want)
F.check_status(); print("done")
""")


def test_a_replay_keeps_what_others_reported(cuda_device):
    """A code that another call left in the word outlives the graph's replays, and is raised once."""
    _run("""
g.replay(); torch.cuda.synchronize()
word.fill_(103)
for _ in range(3):
    g.replay()
torch.cuda.synchronize()
try:
    F.check_status()
    raise SystemExit("the code is gone")
except RuntimeError as e:
    assert "code 103" in str(e), e
F.check_status(); print("done")
""")


def test_the_graph_may_go(cuda_device):
    """The word is not the graph's: calls go on when the graph and its memory are gone."""
    _run("""
g.replay(); torch.cuda.synchronize()
want = y.clone()
del y
g.reset(); del g
import gc; gc.collect(); torch.cuda.empty_cache()
for _ in range(20):
    assert torch.equal(F.fp8_block_linear(x, w, s), want)
assert int(word.item()) == 0
F.check_status(); print("done")
""")

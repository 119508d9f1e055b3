"""GPU: an operator's first call in a process is made in an unusual place: while a CUDA graph captures, or in inference mode.  In a
process of its own, which has called nothing before."""
import subprocess
import sys

import pytest

from conftest import PKG

pytestmark = pytest.mark.gpu

PROGRAM = r"""
import sys
sys.path.insert(0, sys.argv[1])
import torch
from b2g import _lib, ops

dev = torch.device("cuda", 0)
g = torch.Generator(device=dev).manual_seed(1)
logits = torch.randn(5, 9001, generator=g, device=dev)
target = torch.randint(0, 9001, (5,), generator=g, device=dev)
adv = torch.randn(5, generator=g, device=dev)
good, bad = target.clone(), target.clone()
bad[2] = 9001
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = ops.policy_loss(logits, target, adv)
ops.check_status()
graph.replay()
ops.check_status()
want = ops.policy_loss(logits, target, adv)
assert all(torch.equal(a, b) for a, b in zip(got, want))

def reported():
    try:
        ops.check_status()
    except _lib.B2GError as e:
        assert "902" in str(e)
        return True
    return False

# what one replay reports is still there after the next
target.copy_(bad)
graph.replay()
target.copy_(good)
graph.replay()
graph.replay()
assert reported() and not reported()
# and it is the word of every other call, also when the graph is gone
ops.policy_loss(logits, bad, adv)
graph.replay()
assert reported()
del graph
torch.cuda.synchronize()
ops.token_logprobs(logits, bad)
assert reported() and not reported()
print("fine")
"""


def test_first_call_in_a_capture(cuda):
    r = subprocess.run([sys.executable, "-c", PROGRAM, str(PKG)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


INFERENCE = r"""
import sys
sys.path.insert(0, sys.argv[1])
import torch
from b2g import _lib, ops

dev = torch.device("cuda", 0)
target = torch.tensor([1, 50, 3], device=dev)
with torch.inference_mode():
    logp, _ = ops.token_logprobs(torch.zeros(3, 40, device=dev), target)
for _ in range(2):
    try:
        ops.check_status()
    except _lib.B2GError as e:
        assert "902" in str(e)
        ops.token_logprobs(torch.zeros(3, 40, device=dev), target)
    else:
        raise AssertionError("nothing was reported")
try:
    ops.check_status()
except _lib.B2GError:
    ops.check_status()
print("fine")
"""


def test_first_call_in_inference_mode(cuda):
    r = subprocess.run([sys.executable, "-c", INFERENCE, str(PKG)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]

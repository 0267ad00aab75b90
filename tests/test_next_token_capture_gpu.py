"""Making and destroying handles of the next token while another thread captures a graph."""
import subprocess
import sys

import pytest

from tests.conftest import ROOT

pytestmark = pytest.mark.gpu

# In a process of its own, whose first use of these kernels it is: what loads them must not count as a call that a capture forbids.
PROGRAM = """
import threading
import numpy as np
import torch
from gpu_bpe_b200 import BPEEngine, TokenGrammar, TokenSampler

engine = BPEEngine(0).init()
a = torch.arange(5., device="cuda")
made, failed = [], []

def make():
    try:
        made.append(TokenSampler(engine, 100))
        made.append(TokenGrammar(engine, [b"a"] * 100, np.zeros((1, 256), int), [1]))
        TokenGrammar(engine, [b"a"] * 100, np.zeros((1, 256), int), [1]).destroy()
        TokenSampler(engine, 50).destroy()
    except BaseException as e:
        failed.append(e)

g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, capture_error_mode="global"):
    b = a + 1
    thread = threading.Thread(target=make)
    thread.start()
    thread.join()
    c = b * 2
assert not failed, failed
g.replay()
assert c.tolist() == [2., 4., 6., 8., 10.]
t = torch.randn(3, 100, device="cuda")
states = torch.zeros(3, dtype=torch.int32, device="cuda")
assert torch.equal(made[0].sample(t, mask=made[1].allowedTokens(states))[0], t.argmax(1).int())
print("made and captured")
"""


@pytest.mark.parametrize("loading", ["LAZY", "EAGER"])
def test_made_while_another_thread_captures(loading):
    import os
    out = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=300, env=dict(os.environ, CUDA_MODULE_LOADING=loading))
    assert out.returncode == 0 and "made and captured" in out.stdout, out.stderr[-3000:]

"""Dense feed-forward operators in fresh processes and in PyTorch's modes."""

import os
import subprocess
import sys

import pytest
import torch

from helpers import ROOT

pytestmark = pytest.mark.gpu


def _fresh(program):
    """Runs ``program`` in a process that has made no call yet."""
    done = subprocess.run([sys.executable, "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip().endswith("ok"), done.stdout + done.stderr


def test_a_first_call_in_inference_mode():
    """A serving warm-up, then more calls than lie between two looks at the status words, without a mode and training."""
    _fresh("""
import torch
from vllm_plugin_b200 import api
x, w13, w2 = (torch.randn(s, device="cuda").bfloat16() for s in ((5, 64), (64, 64), (64, 32)))
with torch.inference_mode():
    want = api.gated_feed_forward(x, w13, w2).clone()
for _ in range(80):
    y = api.gated_feed_forward(x, w13, w2)
    torch.cuda.synchronize()
assert torch.equal(y, want)
w13.requires_grad_(True)
for _ in range(80):
    api.gated_feed_forward(x, w13, w2).sum().backward()
    torch.cuda.synchronize()
with torch.inference_mode():
    for _ in range(80):
        api.gated_feed_forward(x, w13, w2)
        torch.cuda.synchronize()
api.read_dense_status()
print("ok")
""")

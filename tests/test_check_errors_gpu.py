"""The error check of a program that decodes only waits for its own streams. Attention's error word needs the whole
device, so this runs in a process that never calls attention."""
import subprocess
import sys

import pytest

from lik_testutil import ROOT

pytestmark = pytest.mark.gpu

PROGRAM = """
import sys
sys.path.insert(0, "llm-inference-kernels_b200")
import torch, llmik_cuda as L
q = torch.randn(1, 8, 128, device="cuda").half()
k = torch.randn(1, 2, 64, 128, device="cuda").half()
L.decode_attention(q, k, k, 0.1)
L.check_device_errors()
torch.cuda.synchronize()
other, done = torch.cuda.Stream(), torch.cuda.Event()
with torch.cuda.stream(other):
    torch.cuda._sleep(2_000_000_000)        # a second of somebody else's work
    done.record()
L.check_device_errors()
assert not done.query()
torch.cuda.synchronize()
print("ok")
"""


def test_decoding_alone_is_checked_without_the_device():
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr

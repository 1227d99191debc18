"""The host side of the language-model operators, without a GPU."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

FAKE = """
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
import pdefa_b200 as pb

with FakeTensorMode():
    f = lambda *s: torch.empty(s, device="cuda")                              # noqa: E731
    q = lambda *s: torch.empty(s, device="cuda", dtype=torch.float8_e4m3fn)     # noqa: E731
    i = lambda *s: torch.empty(s, device="cuda", dtype=torch.int32)           # noqa: E731
    for call in (lambda: pb.ops_rms_norm(f(2, 8), f(8)), lambda: pb.ops_rms_norm(f(2, 8), f(8), residual=f(2, 8)),
                 lambda: pb.ops_rms_norm_fp8(f(2, 8), f(8)), lambda: pb.ops_matmul_fp8(q(2, 8), f(2, 1), q(4, 8), f(1, 1)),
                 lambda: pb.ops_matmul_grouped_fp8(q(2, 8), f(2, 1), q(3, 4, 8), f(3, 1, 1), i(4)),
                 lambda: pb.ops_sample(f(2, 8), f(2, 8)), lambda: pb.ops_sample(f(2, 8), f(2, 8), temperature=f(2))):
        try:
            call()
        except RuntimeError as e:
            print("refused")
"""


def test_tensors_without_storage_are_refused():
    """Fake CUDA tensors, as tracing makes them: an exception, not the interpreter's end."""
    pytest.importorskip("torch")
    r = subprocess.run([sys.executable, "-c", FAKE], cwd=ROOT, capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTHONPATH": ROOT})
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.split() == ["refused"] * 7

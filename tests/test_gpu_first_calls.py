"""What a process pays when it starts: kernels of the paged cache are loaded by the first call that needs them."""
import json
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

CODE = """
import json, sys, time
sys.path[:0] = [%r, %r + "/tests"]
import torch
from __graft_entry__ import load_package
load_package()
from qwen30brust_b200 import engine as E
from _paged import Cache, ptr
E.lib()
cache = Cache("f16", 1, 64, 16, [5], cap=32)
row, pos = torch.zeros(1, 1, 64, device="cuda"), torch.full((1,), 7, dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
ms = []
for call in (lambda: E.Sampler(1, 0.5, 5, 0.9), lambda: cache.handle(E).append(ptr(row), ptr(row), 1, ptr(pos))):
    for _ in range(2):
        t = time.perf_counter()
        call()
        torch.cuda.synchronize()
        ms.append((time.perf_counter() - t) * 1e3)
print(json.dumps(ms))
"""


def test_only_users_of_pages_load_their_kernels(torch_cuda):
    """(24 ms for the paged cache's kernels, 10 for the others: whoever loads them is slower by far more than half.
    Three processes at most, as another's load may slow one down.)"""
    for _ in range(3):
        out = subprocess.run([sys.executable, "-c", CODE % (str(ROOT), str(ROOT))], capture_output=True, text=True, timeout=300)
        assert out.returncode == 0, out.stderr
        sampler, sampler2, append, append2 = json.loads(out.stdout)
        if append - append2 > 0.5 * (sampler - sampler2):
            return
    raise AssertionError((sampler, sampler2, append, append2))

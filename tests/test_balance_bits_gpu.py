"""The balance loss of a call does not depend on the calls before it: in a process of its own, after calls of more experts and after calls of
fewer that run the same kernel, it has the same bits."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import sys
import torch
import torch_ggml_ops_b200 as tgo

out = []
for experts in map(int, sys.argv[1].split(",")):
    g = torch.Generator(device="cuda").manual_seed(experts)
    x = torch.randn(20011, experts, device="cuda", generator=g)
    ids = torch.randint(0, experts, (20011, 2), device="cuda", generator=g).int()
    for scoring in ("softmax", "sigmoid"):
        for dtype in (torch.float32, torch.bfloat16):
            loss, _ = tgo.moe_balance_loss(x.to(dtype), ids, scoring=scoring)
            out.append(f"{experts}:{scoring}:{dtype}:{loss.view(torch.int32).item()}")
print(" ".join(out))
"""


def test_the_same_bits_whatever_came_before(cuda):
    found = {}
    for order in ("1024,513,512,257,33,64", "513,1024,257,512,64,33"):
        r = subprocess.run([sys.executable, "-c", PROGRAM, order], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]
        for entry in r.stdout.split():
            call, bits = entry.rsplit(":", 1)
            assert found.setdefault(call, bits) == bits, call
    assert len(found) == 24

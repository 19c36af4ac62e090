"""Where the projection with adapters reports a device-side wait that gave up: words that exist, and are zero, before anything can read them, also for a
process whose first call is captured; and that every replay reports to, not the first alone."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CAPTURED_FIRST = """
import torch
from turbodeberta_b200 import _cabi as cabi
from turbodeberta_b200.status import PENDING
from turbodeberta_b200.ops.flash_attention import check_pending_status
from turbodeberta_b200.ops.lora import lora_linear
g = torch.Generator("cuda").manual_seed(0)
r = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()
x, w, a, b = r(300, 128), r(192, 128), r(2, 8, 128), r(2, 192, 8)
ids = torch.randint(-1, 2, (300,), device="cuda", generator=g)
torch.cuda.synchronize()
# a pool whose freed blocks, large and small, hold sevens
pool = torch.cuda.graph_pool_handle()
first = torch.cuda.CUDAGraph()
with torch.cuda.graph(first, pool=pool):
    blocks = [torch.full((4,), 7, dtype=torch.int32, device="cuda") for _ in range(64)] + [torch.full((1 << 18,), 7, dtype=torch.int32, device="cuda")]
    del blocks
first.replay()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, pool=pool):
    y = lora_linear(x, w, None, a, b, 0.5, ids)
check_pending_status()                               # before the first replay: nothing has been reported
assert len(PENDING) == 0, len(PENDING)               # nothing of one graph's that a single check takes away
graph.replay()
check_pending_status()
want = lora_linear(x, w, None, a, b, 0.5, ids)
graph.replay()
check_pending_status()
assert torch.equal(y, want)
print("fine")
"""


def test_a_process_whose_first_call_is_captured():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CAPTURED_FIRST], cwd=root, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]

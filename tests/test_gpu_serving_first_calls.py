"""A process whose first calls are recorded into a graph."""
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

SCRIPT = """
import sys
sys.path.insert(0, sys.argv[1])
import torch, bgtq
fmt, dim, first = sys.argv[2], int(sys.argv[3]), sys.argv[4]
dt = torch.bfloat16 if fmt in ("bf16", "int8") else torch.float16
cache, n = bgtq.PagedCache(2, dim, 32, 16, fmt), 100
q, k, v = (torch.randn(n, h, dim, device="cuda").to(dt) for h in (8, 2, 2))
rotary, slots = torch.randn(n, dim, device="cuda"), torch.arange(n, device="cuda")
table = torch.arange(32, device="cuda", dtype=torch.int32)[None]
lengths, starts, two = (torch.tensor(x, device="cuda", dtype=torch.int32) for x in ([n], [0, n], [0, 2]))
logits, ids = torch.randn(2, 1000, device="cuda").to(dt), torch.randint(0, 1000, (2, 9), device="cuda")
half = torch.full((2,), 0.5, device="cuda")
calls = dict(append=lambda: cache.append(q, k, v, slots, rotary), many=lambda: cache.attend_chunk(q, starts, table, lengths),
             few=lambda: cache.attend_chunk(q[:2], two, table, lengths), window=lambda: cache.attend(q[:1], table, lengths, window=20),
             logits=lambda: bgtq.adjust_logits(logits, ids, repetition=half))
order = [first] + [name for name in calls if name != first]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = [calls[name]() for name in order]
graph.replay()
graph.replay()
torch.cuda.synchronize()
for name, x in zip(order, got):
    assert torch.equal(x, calls[name]()), name
assert bgtq.device_status(0) == 0
print("same")
"""


@pytest.mark.parametrize("fmt,dim,first", [("f16", 64, "append"), ("bf16", 128, "many"), ("int8", 64, "few"), ("int4", 128, "window"),
                                           ("int8", 128, "logits")])
def test_first_calls_in_a_graph(cuda, fmt, dim, first):
    done = subprocess.run([sys.executable, "-c", SCRIPT, str(ROOT / "block-gqt-webgpu_b200"), fmt, str(dim), first], capture_output=True,
                          text=True, timeout=120)
    assert done.returncode == 0 and "same" in done.stdout, done.stderr[-2000:]

"""What the operators of a serving step report in the device status word, each fault in a process of its own: the
word keeps its bits, so that what one call reports would hide what another does not."""
import itertools
import json
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

# Runs cases [name, code, bit], each in a child that is forked before the device is first used; prints those that fail.
PARENT = '''
import json, os, sys, traceback
sys.path.insert(0, sys.argv[1])
import torch
import bgtq
from bgtq import PagedCache, adjust_logits, device_status
bgtq.lib()
cases = json.load(sys.stdin)
i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
i64 = lambda *x: torch.tensor(x, device="cuda")

def child(code, bit):
    assert device_status(0) == 0
    exec(code, dict(globals()))
    assert device_status(0) == bit, device_status(0)

running, failed = {}, []
def collect():
    pid, status = os.wait()
    name = running.pop(pid)
    if status:
        failed.append(name)
for name, code, bit in cases:
    if len(running) == 6:
        collect()
    pid = os.fork()
    if pid == 0:
        status = 1
        try:
            child(code, bit)
            status = 0
        except BaseException:
            traceback.print_exc()
        finally:
            sys.stderr.flush()
            os._exit(status)
    running[pid] = name
while running:
    collect()
print("failed:", failed)
'''


def reported(cases):
    """Each case's code sets its bit and no other; what it does beside that it asserts itself."""
    done = subprocess.run([sys.executable, "-c", PARENT, str(ROOT / "block-gqt-webgpu_b200")], input=json.dumps(cases), capture_output=True,
                          text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip().endswith("failed: []"), done.stdout[-2000:] + done.stderr[-3000:]


APPEND = """
def appended(fmt, slots, positions, norm=None):
    cache = PagedCache(2, 64, 4, 16, fmt)
    n = len(slots)
    x, q = torch.randn(n, 2, 64, device="cuda"), torch.randn(n, 3, 64, device="cuda")
    cache.append(q, x, x, i64(*slots), torch.randn(10, 64, device="cuda"), i64(*positions), q_norm=norm, k_norm=norm)
"""

CHUNKS = """
import itertools
def made(fmt, dim, page, lens, heads=2):
    need = [-(-n // page) for n in lens]
    cache = PagedCache(heads, dim, sum(need), page, fmt)
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.randn((2, sum(need) * page, heads, dim), generator=g, device="cuda")
    cache.write(*rows, torch.arange(sum(need) * page, device="cuda"))
    table = torch.zeros((len(lens), max(need) + 2), dtype=torch.int32, device="cuda")
    order, at = torch.randperm(sum(need), generator=g, device="cuda").int(), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return cache, table, i32(*lens)
def queries(rows, heads, dim, fmt):
    g = torch.Generator(device="cuda").manual_seed(2)
    return torch.randn((rows, heads, dim), generator=g, device="cuda").to(torch.bfloat16 if fmt == "bf16" else torch.float16)
"""

LOGITS = """
x = torch.arange(66.0, device="cuda").view(2, 33)
"""


def test_append(cuda):
    faults = [((5, -1, 63), (0, 3, 9), 0), ((5, 64), (0, 1), 4), ((2**62,), (0,), 4), ((2**40, 1), (3, 3), 4), ((5, 6), (0, 10), 8),
              ((5,), (-1,), 8), ((5,), (2**62,), 8), ((-1,), (10,), 8)]
    reported([(f"{fmt} {slots} {positions} {norm}", APPEND + f"appended('{fmt}', {slots}, {positions}, {norm})", bit)
              for fmt, norm in (("int8", None), ("bf16", "torch.ones(64, device='cuda')"))
              for slots, positions, bit in faults])


@pytest.mark.parametrize("fmt", ["f16", "bf16", "int8", "int4"])
def test_chunks(cuda, fmt):
    """Both kernels, without a window and with one; n rows of each of three requests of 100, 300 and 17 tokens.  What the
    formats have in common is looked at in one of them."""
    faults = [("nothing", "", 0), ("page", "table[1, 18] = cache.pages", 4), ("negative page", "table[1, 18] = -1", 4),
              ("last page", "table[2, 1] = 2**31 - 1", 4), ("first page", "table[0, 0] = 2**31 - 1", 4),
              ("long", "lengths[1] = table.shape[1] * 16 + 1; table[1] = table[1, 0]", 8), ("negative length", "lengths[2] = -1", 8),
              ("starts fall", "starts[2] = n - 1", 8), ("starts pass", "starts[3] = 3 * n + 1", 8), ("starts below", "starts[0] = -1", 8)]
    cases = []
    calls = [(1, 30), (3, None), (40, None), (40, 30)] if fmt == "f16" else [(3, None), (40, None)]
    for (n, window), (name, change, bit) in itertools.product(calls, faults if fmt == "f16" else (faults[0], faults[1], faults[5], faults[7])):
        if name == "first page" and window is not None:
            bit = 0     # (no row sees it)
        cases.append((f"{n} {window} {name}", CHUNKS + f"""
n = {n}
cache, table, lengths = made("{fmt}", 64, 16, [100, 300, 17])
starts = [0, n, 2 * n, 3 * n]
{change}
q = queries(3 * n, 4, 64, "{fmt}")
cache.attend_chunk(q, i32(*starts), table, lengths, window={window})
""", bit))
        if n == 1 and window and "starts" not in name:
            cases.append((f"attend {name}", cases[-1][1].replace("cache.attend_chunk(q, i32(*starts),", "cache.attend(q,"), bit))
    reported(cases)


@pytest.mark.parametrize("dim", [64, 128])
def test_entries_that_no_row_sees_may_hold_anything(cuda, dim):
    """Between the first tokens and the window of a request's first row, and past its length, of which tiles hold a part."""
    reported([(f"{fmt} {page}", CHUNKS + f"""
fmt, page, dim, lens = "{fmt}", {page}, {dim}, [400, 7, 1000, 333, 64, 5000]
cache, table, lengths = made(fmt, dim, page, lens)
for n, (window, sinks) in itertools.product((1, 3, 6, 40), ((50, 4), (50, 0), (1, 0), (100, 40), (17, 65), (333, 1))):
    q = queries(n * len(lens), 8, dim, fmt)
    starts = i32(*range(0, n * len(lens) + 1, n))
    want = cache.attend_chunk(q, starts, table, lengths, window=window, sinks=sinks, lse=True)
    for wrong in (-1, 2**31 - 1, cache.pages):
        other = table.clone()
        for b, length in enumerate(lens):
            first = max(0, length - n - window + 1)
            hidden = [not any(t < sinks or t >= first for t in range(i * page, min(i * page + page, length))) for i in range(table.shape[1])]
            other[b, torch.tensor(hidden, device="cuda")] = wrong
        got = cache.attend_chunk(q, starts, other, lengths, window=window, sinks=sinks, lse=True)
        assert all(torch.equal(x, y) for x, y in zip(got, want)), (n, window, sinks, wrong)
""", 0) for fmt in ("f16", "bf16", "int8", "int4") for page in (16, 32, 64)])


def test_logits(cuda):
    faults = [
        ("tokens=i32(0, 32, -1, -7).view(2, 2), presence=1.0", 0), ("tokens=i64(0, 32, -1, -2**40).view(2, 2), presence=1.0", 0),
        ("tokens=i32(0, 33, -1, 3).view(2, 2), presence=1.0", 4), ("tokens=i64(0, 1, 2**31, 3).view(2, 2), frequency=1.0", 4),
        ("tokens=i64(0, 1, 2, 2**62).view(2, 2), repetition=2.0", 4), ("tokens=i32(0, 33, 1, 3).view(2, 2), lengths=i32(1, 2), presence=1.0", 0),
        ("tokens=i32(0, 3, 1, 3).view(2, 2), lengths=i32(1, 3), presence=1.0", 8), ("tokens=i32(0, 3, 1, 3).view(2, 2), lengths=i32(-1, 2), presence=1.0", 8),
        ("bias_ids=i32(0, 32, -1, -2**31).view(2, 2), bias=torch.ones(2, 2, device='cuda')", 0),
        ("bias_ids=i32(0, 33, -1, 3).view(2, 2), bias=torch.ones(2, 2, device='cuda')", 4),
        ("bias_ids=i32(2**31 - 1).view(1, 1), bias=torch.ones(1, 1, device='cuda')", 4),
        ("bias_ids=torch.arange(-300, 34, dtype=torch.int32, device='cuda')[None], bias=torch.ones(1, 334, device='cuda')", 4),
        ("mask=torch.zeros(2, 2, dtype=torch.int32, device='cuda')", 0)]
    cases = [(f"{dtype} {arguments}", LOGITS + f"adjust_logits(x.to(torch.{dtype}), {arguments})", bit)
             for dtype, some in (("float32", faults), ("bfloat16", faults[2::7])) for arguments, bit in some]
    for lengths, bit in (((0, 0), 0), ((1, 0), 8), ((0, -2), 8), ((0, 2**31 - 1), 8)):    # histories of no width
        cases.append((f"no width {lengths}", LOGITS + f"""
for ids in (torch.empty((2, 0), dtype=torch.int64, device="cuda"), torch.empty((2, 0), dtype=torch.int32, device="cuda")):
    assert torch.equal(adjust_logits(x, ids, i32(*{lengths}), presence=1.0), x)
""", bit))
    reported(cases)

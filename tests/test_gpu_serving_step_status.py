"""What the operators of a serving step report in the device status word, each fault in a process of its own: the
word keeps its bits, so that what one call reports would hide what another does not."""
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

START = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from bgtq import PagedCache, adjust_logits, device_status
i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
i64 = lambda *x: torch.tensor(x, device="cuda")
assert device_status(0) == 0
"""


def reported(code, bit):
    """The code's calls set this bit and no other; what they do beside that it asserts itself."""
    done = subprocess.run([sys.executable, "-c", START + code + f"\nassert device_status(0) == {bit}, device_status(0)\nprint('fine')",
                           str(ROOT / "block-gqt-webgpu_b200")], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and "fine" in done.stdout, done.stdout + done.stderr[-2000:]


LOGITS = """
x = torch.arange(66.0, device="cuda").view(2, 33)
"""


@pytest.mark.parametrize("lengths,bit", [((0, 0), 0), ((1, 0), 8), ((0, -2), 8), ((0, 2**31 - 1), 8)])
def test_lengths_of_histories_without_room(cuda, lengths, bit):
    reported(LOGITS + f"""
for ids in (torch.empty((2, 0), dtype=torch.int64, device="cuda"), torch.empty((2, 0), dtype=torch.int32, device="cuda")):
    assert torch.equal(adjust_logits(x, ids, i32({lengths[0]}, {lengths[1]}), presence=1.0), x)
""", bit)


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


@pytest.mark.parametrize("fmt", ["f16", "bf16", "int8", "int4"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dim", [64, 128])
def test_entries_that_no_row_sees_may_hold_anything(cuda, fmt, page, dim):
    """Between the first tokens and the window of a request's first row, and past its length, of which tiles hold a part."""
    reported(CHUNKS + f"""
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
            for i in range(table.shape[1]):
                tokens = range(i * page, min(i * page + page, length))
                if not any(t < sinks or t >= first for t in tokens):
                    other[b, i] = wrong
        got = cache.attend_chunk(q, starts, other, lengths, window=window, sinks=sinks, lse=True)
        assert all(torch.equal(x, y) for x, y in zip(got, want)), (n, window, sinks, wrong)
""", 0)

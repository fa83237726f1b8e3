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

"""`from bgtq import *` gives what the package has, and does without torch where that is not installed."""
import subprocess
import sys

from conftest import ROOT

WITHOUT = """
import importlib.abc, sys
class Hidden(importlib.abc.MetaPathFinder):
    def find_spec(self, name, path=None, target=None):
        if name.split(".")[0] == "torch":
            raise ModuleNotFoundError("no torch", name=name)
sys.meta_path.insert(0, Hidden())
"""


def star(before, after):
    r = subprocess.run([sys.executable, "-c", before + "from bgtq import *\n" + after], capture_output=True, text=True,
                       cwd=ROOT / "block-gqt-webgpu_b200")
    assert r.returncode == 0, r.stderr


def test_star_import_without_torch():
    star(WITHOUT, "PackedKeys, build_tables, AttentionEngine\nassert 'torch' not in sys.modules")


def test_star_import_with_torch():
    star("", "PagedCache, prompt_attention, PagedDecoder, PackedKeys")

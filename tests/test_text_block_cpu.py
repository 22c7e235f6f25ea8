"""Host-side logic of the text-conditioning blocks (no GPU)."""
import pathlib
import subprocess
import sys

ROOT = pathlib.Path(__file__).resolve().parents[1]


def test_the_package_brings_the_blocks():
    """``srdit.text_block`` after importing the package alone, as its documentation has it (in
    a process of its own: another test may have imported the submodule)."""
    code = ("import importlib; srdit = importlib.import_module('dreamx-creator_b200'); "
            "print(srdit.text_block.CrossStack.__name__, 'text_block' in srdit.__all__)")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-500:]
    assert r.stdout.split() == ["CrossStack", "True"]

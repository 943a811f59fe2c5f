"""The package's names that need no torch are there without it: importing them all
neither imports torch nor fails where there is none."""
import subprocess
import sys
from pathlib import Path

PROGRAM = """
import sys
if {missing}:
    sys.modules["torch"] = None
from leanstream_b200 import *
assert B200Backend and BatchMLP and union_plan and load_library and LIBRARY
assert sys.modules.get("torch") is None
"""


def run(program):
    return subprocess.run([sys.executable, "-c", program], cwd=Path(__file__).resolve().parents[1],
                          capture_output=True, text=True)


def test_star_import(native_lib):
    for missing in (False, True):
        got = run(PROGRAM.format(missing=missing))
        assert got.returncode == 0, got.stderr


def test_paged_cache_names(native_lib):
    got = run("import leanstream_b200 as l\nassert l.PagedAttention and l.evict_cache\n"
              "from leanstream_b200 import PagedAttention, evict_cache")
    assert got.returncode == 0, got.stderr

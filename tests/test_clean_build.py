"""The first build of a clean checkout, also on a machine with a GPU, where the package refuses to load without its extension."""
import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

from umdk_original_b200.ops import cam_ops

ROOT = Path(__file__).resolve().parent.parent
PKG = "umdk_original_b200"

# stands for the compilers: the objects that were built here are put where they belong
STUB = """
import shutil
from pathlib import Path

def build_all(force=False, debug=False, bindings=True):
    here, built = Path(__file__).resolve().parent, Path({built!r})
    (here / "lib").mkdir()
    for so in [*built.glob("_C*.so"), *built.glob("lib/*.so")]:
        shutil.copy(so, here / so.relative_to(built))
"""


@pytest.fixture
def checkout(tmp_path):
    """The sources alone"""
    shutil.copytree(ROOT / PKG, tmp_path / PKG, ignore=shutil.ignore_patterns("*.so", "build", "lib", "__pycache__", "csrc"))
    shutil.copy(ROOT / "__graft_entry__.py", tmp_path)
    return tmp_path


def run(checkout, gpu, *args):
    """A new interpreter in the checkout, one that believes in a GPU or one that does not"""
    site = checkout / "site"
    site.mkdir(exist_ok=True)
    (site / "sitecustomize.py").write_text(f"import torch\ntorch.cuda.is_available = lambda: {gpu}\n")
    env = dict(os.environ, PYTHONPATH=f"{site}{os.pathsep}{checkout}")
    return subprocess.run([sys.executable, *args], cwd=checkout, env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)


@pytest.mark.parametrize("gpu", [False, True])
def test_build_command_starts_without_the_extension(checkout, gpu):
    out = run(checkout, gpu, "-m", f"{PKG}._build", "--help")
    assert out.returncode == 0 and "--force" in out.stdout, out.stdout
    out = run(checkout, gpu, "-c", f"import {PKG}")
    if gpu:
        assert out.returncode != 0 and f"python -m {PKG}._build" in out.stdout, out.stdout
    else:
        assert out.returncode == 0, out.stdout


@pytest.mark.skipif(not cam_ops.native_loaded(), reason="native extension not built")
@pytest.mark.parametrize("gpu", [False, True])
def test_build_entry_point_loads_what_it_built(checkout, gpu):
    (checkout / PKG / "_build.py").write_text(STUB.format(built=str(ROOT / PKG)))
    out = run(checkout, gpu, "-c", "import __graft_entry__; __graft_entry__.build()")
    assert out.returncode == 0, out.stdout

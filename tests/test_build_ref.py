"""The reference build's recipe: nothing to build is skipped, half a checkout fails."""
import os
import subprocess
import sys

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
RECIPE = os.path.join(REPO, "oracle", "build_ref.py")


def run(*args):
    return subprocess.run([sys.executable, RECIPE, *args], capture_output=True, text=True)


def test_no_sources_are_skipped(tmp_path):
    for src in (tmp_path, tmp_path / "missing"):
        r = run("--src", str(src))
        assert r.returncode == 0 and "skipping" in r.stdout


def test_an_incomplete_checkout_fails(tmp_path):
    (tmp_path / "center_kernels.cu").write_text("")
    (tmp_path / "euclidean_cuda.cpp").write_text("")
    r = run("--src", str(tmp_path))
    assert r.returncode == 1 and "no euclidean_cuda_advanced.cpp" in r.stderr and "euclidean_kernels.cu" in r.stderr
    r = run("--src", str(tmp_path), "--only", "ref_euclidean_cuda")
    assert r.returncode == 1 and "no euclidean_kernels.cu" in r.stderr
    assert run("--src", str(tmp_path), "--only", "ref_euclidean_tiled").returncode == 0  # none of its sources

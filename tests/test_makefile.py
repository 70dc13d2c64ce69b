"""The Makefile on machines without torch: the C library and the front end need none of it."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def commands(*args):
    """What `make` would run for everything, nothing taken as built."""
    r = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "julia-cuda_b200"), *args], capture_output=True,
                       text=True, check=True)
    return r.stdout


def test_without_torch_the_library_builds_alone():
    for python in ("false", "/nowhere/python"):
        out = commands(f"PYTHON={python}")
        assert "libjulia_cuda.so" in out and "cli.cpp" in out and "torch_binding.cpp" not in out


def test_with_torch_the_binding_is_built_too():
    assert "torch_binding.cpp" in commands()

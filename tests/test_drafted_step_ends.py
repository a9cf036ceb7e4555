"""The ends of what a drafted step's operators accept, without a GPU: their tests on the CPU build, between guard pages."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HERE = os.path.join(ROOT, "tests")


@pytest.mark.parametrize("units", ["", "1"])
def test_the_ends_of_a_drafted_steps_operators_pass_on_the_cpu_build(units):
    """tests/test_drafted_step_ends_gpu.py over the kernels built for the CPU; with one compute unit the products of many matrix rows and
    the runs of many pages are chosen at its sizes."""
    from rust_inference_amd.errors import KernelError
    try:
        sys.path.insert(0, HERE)
        import emulated
        emulated.library()
    except KernelError as e:
        pytest.skip(f"no CPU build of the kernels here: {e}")
    env = dict(os.environ, RI_TEST_KERNELS="emulated")
    env.pop("RI_KERNEL_LIBRARY", None)
    env.pop("RI_EMU_COMPUTE_UNITS", None)
    if units:
        env["RI_EMU_COMPUTE_UNITS"] = units
    args = [sys.executable, "-m", "pytest", "-q", "-x", "-p", "no:cacheprovider", os.path.join(HERE, "test_drafted_step_ends_gpu.py")]
    try:
        import xdist  # noqa: F401
        args += ["-n", str(max(1, min(4, (os.cpu_count() or 2) // 2)))]
    except ImportError:
        pass
    run = subprocess.run(args, capture_output=True, text=True, env=env, cwd=ROOT, timeout=600)
    assert run.returncode == 0 and " passed" in run.stdout and "[emu]" not in run.stderr, run.stdout[-3000:] + run.stderr[-3000:]

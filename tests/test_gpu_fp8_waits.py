"""The waits that the 8-bit pair kernel has for itself: each gives up after its limit, which counts from the wait, or when another role has given up."""

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

pytestmark = pytest.mark.gpu
MS = 1_000_000


@pytest.fixture(scope="module")
def run_wait(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc is not installed")
    so = str(tmp_path_factory.mktemp("waits") / "fp8_waits.so")
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "-o", so,
                    os.path.join(os.path.dirname(__file__), "fp8_waits.cu")], check=True, capture_output=True)
    fn = ctypes.CDLL(so).run_fp8_wait
    fn.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]

    def run(polls, given_up, before, after, limit):
        status, out = torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        assert fn(polls, given_up, before, after, limit, status.data_ptr(), out.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        end.record()
        torch.cuda.synchronize()
        return out.tolist(), status.tolist(), start.elapsed_time(end)

    return run


@pytest.mark.parametrize("polls", [0, 1])
def test_a_wait_for_nothing_gives_up(run_wait, polls):
    """The whole warp at once, with a report, and tells the other roles."""
    out, status, ms = run_wait(polls, 0, 0, -1, 100 * MS)
    assert out == [1, 1] and status[:4] == [1, 34, 7 if polls else 0, 0]
    assert 90 < ms < 1000


@pytest.mark.parametrize("polls", [0, 1])
def test_the_limit_counts_from_the_wait_on(run_wait, polls):
    """A wait of 60 ms in a launch that has run for 250, with a limit of 150."""
    out, status, ms = run_wait(polls, 0, 250 * MS, 60 * MS, 150 * MS)
    assert out == [2, 0] and not any(status) and ms > 300


@pytest.mark.parametrize("polls", [0, 1])
def test_a_wait_ends_when_another_role_has_given_up(run_wait, polls):
    """Long before its limit, and without a report of its own."""
    out, status, ms = run_wait(polls, 1, 0, -1, 2000 * MS)
    assert out == [1, 1] and not any(status) and ms < 1000


@pytest.mark.parametrize("polls", [0, 1])
def test_a_barrier_that_has_completed(run_wait, polls):
    out, status, _ = run_wait(polls, 0, 20 * MS, 0, 100 * MS)
    assert out == [2, 0] and not any(status)

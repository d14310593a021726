"""The waits of the dense kernels: each gives up after its limit, and the limit is that of the wait, not of the launch."""

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
    so = str(tmp_path_factory.mktemp("waits") / "dense_waits.so")
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "-o", so,
                    os.path.join(os.path.dirname(__file__), "dense_waits.cu")], check=True, capture_output=True)
    fn = ctypes.CDLL(so).run_dense_wait
    fn.argtypes = [ctypes.c_int, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]

    def run(whole_warp, before, after, limit):
        status, out = torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        assert fn(whole_warp, before, after, limit, status.data_ptr(), out.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        end.record()
        torch.cuda.synchronize()
        return out.item(), status.tolist(), start.elapsed_time(end)

    return run


@pytest.mark.parametrize("whole_warp", [0, 1])
def test_a_wait_for_nothing_gives_up(run_wait, whole_warp):
    out, status, ms = run_wait(whole_warp, 0, -1, 100 * MS)
    assert out == 1 and status[:4] == [1, 31, 10 + whole_warp, 0]
    assert 90 < ms < 1000


@pytest.mark.parametrize("whole_warp", [0, 1])
def test_the_limit_counts_from_the_wait_on(run_wait, whole_warp):
    """A wait of 60 ms in a launch that has run for 250, with a limit of 150."""
    out, status, ms = run_wait(whole_warp, 250 * MS, 60 * MS, 150 * MS)
    assert out == 2 and not any(status) and ms > 300

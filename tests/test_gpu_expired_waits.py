"""GPU: a product whose wait for a slice runs out (after about two seconds: nothing loads that
slice) ends by itself, says so, and leaves unfinished sums unwritten."""
import ctypes as C
import os
import subprocess
import time

import pytest
import torch

import tbabi as tb

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def native(cuda, tmp_path_factory):
    import build
    out = str(tmp_path_factory.mktemp("native") / "libexpired_waits.so")
    tb.lib()
    lib_dir, lib_name = os.path.split(tb.LIB_PATH)
    cmd = [build.NVCC, *build.NVCC_FLAGS, *(f"-I{d}" for d in build.INCLUDES), "-shared", "-o", out, os.path.join(HERE, "native", "expired_waits.cu"),
           f"-L{lib_dir}", f"-l:{lib_name}", "-Xlinker", f"-rpath={lib_dir}"]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr
    return C.CDLL(out)


def product(native, clusters, left_out, n=512, slices=20):
    m = 128 if clusters else 256
    a = torch.ones(256, 64 * slices, device="cuda", dtype=torch.bfloat16)
    b = torch.ones(n, 64 * slices, device="cuda", dtype=torch.bfloat16)
    out = torch.full((m, n), -7.0, device="cuda")
    failed = torch.zeros(1, device="cuda", dtype=torch.int32)
    stream = torch.cuda.current_stream().cuda_stream
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    t0 = time.monotonic()
    tb.check(native.expired_product(p(a), p(b), p(out), p(failed), n, slices, int(clusters), left_out, C.c_void_p(stream)))
    torch.cuda.synchronize()
    took = time.monotonic() - t0
    error = C.c_int(-1)
    assert native.expired_error(C.byref(error)) == 0
    return out, int(failed), error.value, took


@pytest.mark.parametrize("clusters,left_out", [(False, 0), (False, 1), (True, 0), (True, 2)])
def test_a_slice_that_never_comes(native, clusters, left_out):
    out, failed, error, _ = product(native, clusters, -1)
    assert (out == 1280.0).all() and failed == 0 and error == 0
    out, failed, error, took = product(native, clusters, left_out)
    assert (out == -7.0).all(), "an unfinished sum was written"
    assert failed == 1 and error == 1 and took < 20
    out, failed, error, _ = product(native, clusters, -1)
    assert (out == 1280.0).all() and failed == 0 and error == 0

"""The drop-in fp32 GEMM file on the B200 against the in-tree oracle: bit-identical to AMP's CPU GEMM.

test_amp_check_gpu.py has AMP's own validator say so, where AMP's sources are; this needs only
nvcc and the oracle.  The kernel is launched as AMP's checker launches it (scripts/amp_check.sh:59-106):
16 x 16 threads a block, one block a 16 x 16 output tile, compiled by a bare `nvcc -shared`."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

import oracle

KERNEL = Path(__file__).resolve().parents[1] / "amp_b200" / "dropin" / "amp_b200_gemm_fp32.cu"
pytestmark = pytest.mark.gpu

HOST = """
#include <cuda_runtime.h>
#include "%s"
extern "C" int run(const float* A, const float* B, float* C, int M, int N, int K) {
    float *a = nullptr, *b = nullptr, *c = nullptr;
    const size_t na = 4 * (size_t)M * K, nb = 4 * (size_t)K * N, nc = 4 * (size_t)M * N;
    cudaMalloc(&a, na);
    cudaMalloc(&b, nb);
    cudaMalloc(&c, nc);
    if (a && b && c) {
        cudaMemcpy(a, A, na, cudaMemcpyHostToDevice);
        cudaMemcpy(b, B, nb, cudaMemcpyHostToDevice);
        amp_b200_gemm_fp32<<<dim3((N + 15) / 16, (M + 15) / 16), dim3(16, 16)>>>(a, b, c, M, N, K);
        cudaMemcpy(C, c, nc, cudaMemcpyDeviceToHost);
    }
    cudaFree(a);
    cudaFree(b);
    cudaFree(c);
    return (int)cudaGetLastError();
}
"""


@pytest.fixture(scope="module")
def dropin(tmp_path_factory, cuda):
    at = tmp_path_factory.mktemp("dropin")
    (at / "host.cu").write_text(HOST % KERNEL)
    subprocess.run(["nvcc", "-shared", "-Xcompiler", "-fPIC", "-o", str(at / "host.so"), str(at / "host.cu")],
                   check=True, capture_output=True)
    return C.CDLL(str(at / "host.so"))


@pytest.mark.parametrize("mnk", [(96, 96, 96), (512, 512, 512), (1024, 1024, 1024), (100, 70, 33),
                                 (257, 513, 1000), (1, 1, 1), (2048, 64, 4096)])
def test_dropin_is_bit_identical_to_the_cpu_gemm(mnk, dropin):
    M, N, K = mnk
    A, B = oracle.amp_harness_inputs(M, N, K, seed=42)
    got = np.full((M, N), np.nan, np.float32)
    args = [x.ctypes.data_as(C.c_void_p) for x in (A, B, got)]
    assert dropin.run(*args, M, N, K) == 0
    assert np.array_equal(got, oracle.gemm_fp32_amp(A, B))

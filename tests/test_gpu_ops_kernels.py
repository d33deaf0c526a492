"""Every kernel of the norm and of the 8-bit product runs here or in tests/test_gpu_ops.py, in every type (tests/test_ops_cpu.py checks
these lists against the kernels that are built)."""
import pytest
import torch

from tests import test_gpu_ops

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32

# columns for each number of threads a row gets, the longest rows being read twice; whole and partial groups of 128
NORM_KERNELS = [(t, h, dtype) for t, h in ((5, 300), (3, 700), (2, 2048), (3, 3000), (2, 8192), (2, 16384), (2, 20000)) for dtype in (BF16, F16, F32)]


@pytest.mark.parametrize("t,h,dtype", NORM_KERNELS)
@pytest.mark.parametrize("residual", [False, True])
def test_norm_kernels(t, h, dtype, residual):
    test_gpu_ops.test_norm(t, h, dtype, residual)


@pytest.mark.parametrize("m,n,k", test_gpu_ops.KERNEL_SIZES)
@pytest.mark.parametrize("out", [F16])
def test_matmul_kernels_in_float16(m, n, k, out):
    test_gpu_ops.test_matmul_kernels(m, n, k, out)

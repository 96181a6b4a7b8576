"""The 4-bit product over more columns than 2 GB of scale bytes a row of tiles hold (K past 2^29)."""
import ctypes as C

import pytest
import torch

import nemoasr_b200 as nb
import operators_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K", [(1 << 29) + 4096, 1 << 30])
def test_product_long_k(K):
    """One output, zero codes but for a few: those at the front, on both sides of column 2^29 and in the
    last block, each with a scale of its own, so that a tile of scales taken from elsewhere shows. The
    products are small integers: the sum is exact."""
    L = nb.api()
    n = L.nemo_mxfp4_scale_bytes(1, K)
    assert n == K // 128 * 512
    at = [0, 5, (1 << 29) - 32, 1 << 29, (1 << 29) + 256, K - 129, K - 1]
    want, ops = 0.0, []
    scale = [[127 + (i + 2 * w) % 5 for i in range(len(at))] for w in range(2)]
    for i in (0, 1):  # columns 0 and 5 share a block
        scale[i][1] = scale[i][0]
    for w in range(2):
        q = torch.zeros(K // 2, dtype=torch.uint8, device="cuda")
        s = torch.full((n,), 127, dtype=torch.uint8, device="cuda")
        for col, byte in zip(at, scale[w]):
            q[col // 2] |= 2 << 4 * (col % 2)  # 1.0
            b = col // 32
            s[b // 4 * 512 + b % 4] = byte  # row 0
        ops.append((q, s))
    want = sum(2.0 ** (a + b - 254) for a, b in zip(*scale))
    c = torch.zeros(1, 1, device="cuda")
    g = nb.GemmMxfp4Args(A=ops[0][0].data_ptr(), lda=K // 2, a_scales=ops[0][1].data_ptr(), W=ops[1][0].data_ptr(), ldw=K // 2, w_scales=ops[1][1].data_ptr(),
                         C=c.data_ptr(), ldc=1, M=1, N=1, K=K, alpha=1.0)
    nb.check(L.nemo_gemm_mxfp4(C.byref(g), R.stream_ptr()), "gemm")
    torch.cuda.synchronize()
    assert L.nemo_gpu_check_device_errors() == 0, L.nemo_gpu_last_error().decode()
    assert c.item() == want

"""A device wait that gave up is reported under the name of the kernel that recorded it, once."""
import ctypes as C

import pytest
import torch

import nemoasr_b200 as nb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code,name", [(1, "tensor-core GEMM"), (8, "tensor-core GEMM"), (9, "wait self-test"), (10, "wait self-test"), (11, "4-bit product"), (14, "4-bit product")])
def test_error_names(code, name):
    L = nb.api()
    L.nb_tc_error_ptr.restype = C.c_void_p
    torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    assert L.nemo_gpu_check_device_errors() == 0
    word = C.c_int(code)  # as a kernel's wait leaves it
    assert C.CDLL("libcuda.so.1").cuMemcpyHtoD_v2(C.c_uint64(L.nb_tc_error_ptr()), C.byref(word), C.c_size_t(4)) == 0
    assert L.nemo_gpu_check_device_errors() == -1
    assert L.nemo_gpu_last_error().decode() == f"{name}: a bounded device wait gave up (code {code})"
    assert L.nemo_gpu_check_device_errors() == 0

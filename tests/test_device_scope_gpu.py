"""A call leaves its caller's current device and context as they were."""

import ctypes
import threading

import numpy as np
import pytest
import torch

import llm_kernels
import oracle
from llm_kernels import _lib

pytestmark = pytest.mark.gpu


def test_a_thread_without_a_context():
    """Its calls run on the device picked, by default device 0, where CUDA has such a thread anyway."""
    x = torch.randn(40, 256, device="cuda:0", dtype=torch.float16)
    q, s = torch.zeros(40, 256, device="cuda:0", dtype=torch.int8), torch.zeros(40, device="cuda:0")
    torch.cuda.synchronize()
    cuda, seen = ctypes.CDLL("libcuda.so.1"), []

    def current():
        dev, ctx = ctypes.c_int(-1), ctypes.c_void_p(1)
        assert cuda.cuCtxGetCurrent(ctypes.byref(ctx)) == 0
        return None if ctx.value is None else (cuda.cuCtxGetDevice(ctypes.byref(dev)), dev.value)

    def work():
        seen.append(current())
        _lib.call("lk_set_device", 0)  # picks, and makes nothing current
        seen.append(current())
        _lib.call("lk_quantize_symmetric", x.data_ptr(), _lib.LK_F16, 40, 256, 256, q.data_ptr(), 256, s.data_ptr(), None)
        seen.append(current())
        seen.append(llm_kernels.device_status()[0])
        seen.append(torch.cuda.current_device())

    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert seen == [None, None, (0, 0), 0, 0]
    want, scale = oracle.quantize_symmetric(x.cpu())
    np.testing.assert_array_equal(q.cpu().numpy(), want)
    np.testing.assert_array_equal(s.cpu().numpy(), scale)


def test_backward_on_autograds_thread_finds_a_context(recwarn):
    """The library's backward is the first CUDA work of torch's autograd thread; a matrix product follows."""
    q = torch.randn(6, 4, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(64, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = llm_kernels.rotary_embed(q @ w, None, torch.arange(6, device="cuda"), llm_kernels.rotary_table(6, 64))
    y.backward(torch.ones_like(y))
    assert w.grad.isfinite().all() and not [r for r in recwarn if "context" in str(r.message)]


def test_the_callers_device_stays():
    before = torch.cuda.current_device()
    q = torch.randn(4, 2, 64, device="cuda", dtype=torch.float16)
    kc, vc = torch.zeros(2, 2, 16, 2, 64, device="cuda", dtype=torch.float16)
    table, lengths = torch.zeros(4, 1, dtype=torch.int32, device="cuda"), torch.ones(4, dtype=torch.int32, device="cuda")
    llm_kernels.rotary_embed(q, None, torch.arange(4, device="cuda"), llm_kernels.rotary_table(4, 64))
    llm_kernels.paged_kv_append(q, q, kc, vc, torch.arange(4, device="cuda"))
    llm_kernels.paged_attention(q, kc, vc, table, lengths)
    assert torch.cuda.current_device() == before and llm_kernels.device_status()[0] == 0


def test_a_device_that_is_not_there_is_refused():
    with pytest.raises(llm_kernels.LKError):
        _lib.set_device(torch.cuda.device_count())
    with pytest.raises(llm_kernels.LKError):
        _lib.set_device(-1)
    _lib.set_device(0)

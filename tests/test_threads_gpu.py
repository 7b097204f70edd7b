"""A thread whose first CUDA work is a kernel that encodes tensor maps (an autograd
worker served from cached memory is one)."""

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_gemm_is_the_first_work_of_a_thread():
    from vagus_b200.ops._core import gemm
    a, b = (torch.randn(256, 256, device="cuda").bfloat16() for _ in range(2))
    want, got = (torch.empty(256, 256, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    gemm(a, False, b, False, want)
    torch.cuda.synchronize()
    raised = []

    def work():
        try:
            gemm(a, False, b, False, got)
        except RuntimeError as e:
            raised.append(e)
    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert not raised and torch.equal(got, want)

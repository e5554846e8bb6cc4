"""GPU: the failure path of the waits in the paged attention's kernel for many
rows, without a GPU fault: moss_test_paged_wait runs them with a short limit on
phases that nothing completes."""

import time

import pytest
import torch

from test_gpu_paged import History, attention_reference, check_attention, take_device_error

pytestmark = pytest.mark.gpu


def test_waits_that_complete_record_nothing(moss, cuda_device):
    from fast_moss_b200 import _lib

    take_device_error()
    _lib.call("moss_test_paged_wait", 50_000_000, 1, torch.cuda.current_stream().cuda_stream)
    assert take_device_error() == _lib.OK


def test_the_first_wait_to_run_out_ends_the_others(moss, cuda_device):
    from fast_moss_b200 import _lib

    take_device_error()
    h = History([50, 1], [300, 40], 2, 64, 16, cuda_device)
    q = torch.randn(h.n, 4, 64, device=cuda_device, dtype=torch.bfloat16)
    want, size = attention_reference(h, q, 0, 1 / 8)
    torch.cuda.synchronize()
    t = time.perf_counter()
    _lib.call("moss_test_paged_wait", 3_000_000, 0, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert time.perf_counter() - t < 1.0  # the kernels' own limit is 2 s
    assert take_device_error() == _lib.ERR_TIMEOUT
    assert take_device_error() == _lib.OK  # read and cleared
    check_attention(moss.paged_attention(q, h.k, h.v, *h.index), want, size, 100)
    assert take_device_error() == _lib.OK

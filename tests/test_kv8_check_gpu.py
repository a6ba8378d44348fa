"""The attention kernels' error words, without a fault of the GPU: a self-test kernel waits, with the kernels' own bounded
wait at a limit of about a millisecond, on a barrier that nothing arrives on, and leaves its code in one of the words."""
import ctypes as C

import pytest
import torch

import qcom_htp_b200 as qhtp
from qcom_htp_b200 import _lib as L
from tests.test_kv8_gpu import BF, attend

pytestmark = pytest.mark.gpu

LIMIT, CODE = 2_000_000, 4


def give_up(kernel, stream=None):
    count = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    handle = (stream or torch.cuda.current_stream()).cuda_stream
    assert L.lib.qhtp_selftest_kv8_timeout(kernel, count.data_ptr(), LIMIT, handle) == L.OK
    return count


@pytest.mark.parametrize("kernel", [0, 1, 2])
def test_a_wait_that_gave_up_is_reported_once(kernel):
    qhtp.kv8_check()
    count = give_up(kernel)
    with pytest.raises(qhtp.QhtpError, match=f"device code {CODE}.*gave up") as e:
        qhtp.kv8_check()
    assert e.value.status == L.RUNTIME_ERROR
    assert int(count) == 4  # every warp stopped waiting and returned
    qhtp.kv8_check()  # cleared


def test_all_words_are_cleared_at_once():
    for kernel in range(3):
        give_up(kernel)
    code = C.c_int(0)
    stream = torch.cuda.current_stream().cuda_stream
    assert L.lib.qhtp_kv8_check(C.byref(code), stream) == L.RUNTIME_ERROR and code.value == CODE
    assert L.lib.qhtp_kv8_check(None, stream) == L.OK


def test_on_a_stream_and_a_device():
    s = torch.cuda.Stream()
    give_up(1, s)
    with pytest.raises(qhtp.QhtpError):
        qhtp.kv8_check(stream=s)
    give_up(0, s)
    s.synchronize()
    with pytest.raises(qhtp.QhtpError):
        qhtp.kv8_check("cuda:0")
    qhtp.kv8_check(torch.device("cuda", 0), s)


def test_each_kernel_runs_and_reports_nothing():
    """After a give-up the context is intact: few rows, one tile and two tiles, right and without an error."""
    for kernel in range(3):
        give_up(kernel)
    with pytest.raises(qhtp.QhtpError):
        qhtp.kv8_check()
    attend([300, 1200], [1, 1], 8, 2, 128, 16, BF)
    attend([300, 100], [100, 100], 8, 2, 256, 16, BF)
    attend([1500] * 6, [300] * 6, 32, 8, 64, 32, BF)
    qhtp.kv8_check()


def test_refusals():
    w = torch.zeros(1, dtype=torch.int32, device="cuda")
    for args in ((3, w.data_ptr(), 1000), (0, None, 1000), (0, w.data_ptr(), 0), (0, w.data_ptr(), (1 << 32) + 1)):
        assert L.lib.qhtp_selftest_kv8_timeout(*args, None) == L.INVALID_ARGUMENT
    with pytest.raises(ValueError):
        qhtp.kv8_check("cpu")
    qhtp.kv8_check()

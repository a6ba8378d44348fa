"""The softmax scale at the ends of float32."""
import ctypes as C

import pytest

from qcom_htp_b200 import _lib as L
from qcom_htp_b200 import kv8
from tests.test_kv8_cpu import attention
from tests.test_kv8_device_cpu import CACHE, COUNT, Rows, TABLE, library  # noqa: F401  (library is a fixture)


@pytest.mark.parametrize("scale,status", [(2.4e38, L.INVALID_ARGUMENT), (3.4e38, L.INVALID_ARGUMENT), (float("inf"), L.INVALID_ARGUMENT)])
def test_the_c_entry_refuses_a_scale_that_overflows(scale, status):
    """Exponents are taken with scale log2(e), which was infinite, and all outputs NaN, for a finite scale above 2.36e38."""
    run = attention(scale=scale)
    run.q.data = 8  # refused before any launch either way
    assert L.lib.qhtp_kv8_attention(C.byref(run)) == status
    assert b"scale" in L.lib.qhtp_last_error_string()


def test_python_refuses_the_same(library):  # noqa: F811
    attend = lambda scale: kv8.kv8_attention(Rows(3, 1, 4, 64), CACHE, TABLE, COUNT, scale=scale, out=Rows(3, 1, 4, 64))
    for scale in (2.0 ** -149, 1e-30, 1.0, 2.3e38):
        attend(scale)
    for scale in (0.0, -1.0, 1e-60, 2.4e38, 1e39, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            attend(scale)

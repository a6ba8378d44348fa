"""The host path without a GPU: everything that asks the library about a launch asks on the cache's device.  Tensors and
library are stand-ins that record the current device at each call."""
import contextlib

import pytest
import torch

from qcom_htp_b200 import kv8

DEV = torch.device("cuda", 1)


class Rows:
    """As much of a CUDA tensor as the host path looks at."""
    is_cuda, device = True, DEV

    def __init__(self, *shape, dtype=torch.bfloat16):
        self.shape, self.dtype = torch.Size(shape), dtype
        self.strides = torch.empty(shape, device="meta").stride()

    def stride(self):
        return self.strides

    def is_contiguous(self):
        return True

    def dim(self):
        return len(self.shape)

    def data_ptr(self):
        return 4096

    def new_empty(self, shape, dtype):
        return Rows(*shape, dtype=dtype)


class Library:
    def __init__(self, need):
        self.need, self.device, self.calls = need, 0, []

    def qhtp_kv8_attention_workspace_bytes(self, arg):
        self.calls.append(("size", self.device))
        return self.need

    def qhtp_kv8_attention(self, arg):
        fields = kv8._ATTENTION.unpack(arg)
        self.calls.append(("run", self.device, fields[-3:-1]))
        return 0

    def qhtp_kv8_write(self, arg):
        self.calls.append(("write", self.device))
        return 0

    qhtp_kv8_read = qhtp_kv8_write


@pytest.fixture(params=[0, 512])
def library(request, monkeypatch):
    lib = Library(request.param)

    @contextlib.contextmanager
    def device(dev):
        before, lib.device = lib.device, dev.index
        yield
        lib.device = before

    monkeypatch.setattr(kv8.L, "lib", lib)
    monkeypatch.setattr(kv8, "_device", lambda: lib.device)
    monkeypatch.setattr(kv8, "_current", lambda index: 7)
    monkeypatch.setattr(torch.cuda, "device", device)
    return lib


CACHE = (Rows(8, 2, 16, 64, dtype=torch.int8),) * 2 + (Rows(8, 2, dtype=torch.float32),) * 2
TABLE, COUNT = Rows(3, 4, dtype=torch.int32), Rows(3, dtype=torch.int32)


@pytest.mark.parametrize("current", [0, 1])
def test_attention_plans_and_runs_on_the_caches_device(library, current):
    """The plan, and so the workspace's size, depends on the device that is current."""
    library.device = current
    kv8.kv8_attention(Rows(3, 1, 4, 64), CACHE, TABLE, COUNT, out=Rows(3, 1, 4, 64))
    assert library.calls == [("size", 1), ("run", 1, (4096, 512) if library.need else (0, 0))]
    assert library.device == current


@pytest.mark.parametrize("current", [0, 1])
def test_write_runs_on_the_caches_device(library, current):
    library.device = current
    kv8.kv8_write(CACHE, Rows(3, 1, 2, 64), Rows(3, 1, 2, 64), TABLE, COUNT)
    assert library.calls == [("write", 1)]
    assert library.device == current

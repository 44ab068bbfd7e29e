"""What the Python binding takes for a device buffer: an object with data_ptr(), an address, or None."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from muyo_llm_b200 import nodes


class Buffer:
    def data_ptr(self):
        return 4096


def test_buffers_and_addresses():
    assert nodes._ptr(None) is None and nodes._ptr(8192) == 8192 and nodes._ptr(Buffer()) == 4096


@pytest.mark.parametrize("host", [b"host", bytearray(16), "text", (C.c_float * 4)(), C.c_void_p(4096), C.byref(C.c_int(1)), np.zeros(4, np.float32), [1.0], 1.5])
def test_host_memory_is_refused(host):
    """ctypes would pass the address of some of these to a kernel."""
    with pytest.raises(AttributeError):
        nodes._ptr(host)


def test_an_error_inside_data_ptr_is_not_hidden():
    class Broken:
        def data_ptr(self):
            return self.missing

    with pytest.raises(AttributeError, match="missing"):
        nodes._ptr(Broken())

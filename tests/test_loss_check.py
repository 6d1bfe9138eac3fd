"""A wait that ran out is an error where the user asks, not NaN alone."""
import ctypes as C
import types

import pytest


def test_a_result_says_whether_a_wait_ran_out(monkeypatch):
    import torch

    import culsh_b200 as culsh
    from culsh_b200 import _lib, loss
    status, asked = [0], []

    def product_check(handle, stream):
        asked.append((handle, stream))
        return status[0]

    handle = types.SimpleNamespace(ptr=C.c_void_p(7), lib=types.SimpleNamespace(culsh_mx_product_check=product_check))
    monkeypatch.setattr(loss, "get_handle", lambda device: handle)
    monkeypatch.setattr(loss, "_stream", lambda device: 11)
    r = culsh.CrossEntropy(torch.zeros(2), torch.zeros(2), torch.zeros(2))
    r.check()
    assert asked == [(handle.ptr, 11)] and len(r) == 3
    status[0] = _lib.load().culsh_i8_quantize(None, None, 0, 1, 1, 1, None, None, None, None)  # any status that is an error
    with pytest.raises(Exception, match="null"):
        r.check()

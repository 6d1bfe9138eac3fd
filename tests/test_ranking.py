"""The ranking entry points refuse bad arguments with a status and a message, before any work on a device."""
import ctypes as C

import pytest


def test_null_arguments_are_a_status():
    from culsh_b200 import _lib
    lib = _lib.load()
    need = C.c_uint64()
    for status in (
        lib.culsh_mx_quantize(None, None, 0, 1, 1, 1, None, None, None, None),
        lib.culsh_mx_dequantize(None, None, None, 1, 1, None, 0, None),
        lib.culsh_mx_product(None, None, None, None, 1, None, None, None, 1, 1, 0, None, 0, 1, None),
        lib.culsh_mx_product_dense(None, None, 0, 1, 1, None, None, None, 1, 1, 0, None, 0, 1, None, 0, None),
        lib.culsh_mx_product_check(None, None),
        lib.culsh_mx_score(None, None, 0, 1, 1, None, None, None, 1, 1, 0, None, None, 0, None, None, 0, None),
        lib.culsh_mx_score_workspace(None, 1, 1, 0, C.byref(need)),
        lib.culsh_candidates_after(None, None, None),
        lib.culsh_log_probs_workspace(None, 0, 1, 1, 0, 0, C.byref(need)),
        lib.culsh_log_probs(None, None, 0, 1, 1, 1, None, None, 0, 1.0, None, 0, None, None, None, None, None, None, 0, None),
        lib.culsh_log_probs_backward(None, None, 0, 1, 1, 1, None, None, 0, 1.0, None, None, None, None, None, None, 1, None),
    ):
        assert status == -1
        assert b"null" in lib.culsh_last_error()


def test_names_are_public():
    import culsh_b200
    for name in ("MXRows", "LogProbs", "log_probs", "log_probs_backward", "rank"):
        assert name in culsh_b200.__all__ and getattr(culsh_b200, name) is not None
    with pytest.raises(AttributeError):
        culsh_b200.no_such_name


def test_arguments_are_checked_before_a_device_is_needed():
    import torch

    import culsh_b200 as culsh
    with pytest.raises(ValueError):
        culsh.log_probs(torch.zeros(2, 2), top_k=1000)
    with pytest.raises(ValueError):
        culsh.log_probs(torch.zeros(2, 2), temperature=-1.0)
    with pytest.raises(ValueError):
        culsh.MXRows.from_parts(torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8), torch.zeros(2), 0)

"""Rows in 8 bits and the loss over every row refuse bad arguments with a status and a message, before any work on a device."""
import ctypes as C

import pytest


def test_null_arguments_are_a_status():
    from culsh_b200 import _lib
    lib = _lib.load()
    need = C.c_uint64()
    for status in (
        lib.culsh_i8_quantize(None, None, 0, 1, 1, 1, None, None, None, None),
        lib.culsh_i8_dequantize(None, None, None, 1, 1, None, 0, None),
        lib.culsh_i8_product(None, None, None, None, 1, None, None, None, 1, 1, 0, None, 0, 1, None),
        lib.culsh_i8_product_dense(None, None, 0, 1, 1, None, None, None, 1, 1, 0, None, 0, 1, None, 0, None),
        lib.culsh_i8_score(None, None, 0, 1, 1, None, None, None, 1, 1, 0, None, None, 0, None, None, 0, None),
        lib.culsh_cross_entropy_workspace(None, None, 1, None, 1, 0, 1, 1, 1, 0, 0, C.byref(need)),
        lib.culsh_cross_entropy(None, None, 1, None, 1, 0, 1, 1, 1, None, None, 1.0, None, None, None, None, 0, None),
        lib.culsh_cross_entropy_backward(None, None, 1, None, 1, 0, 1, 1, 1, None, None, 1.0, None, None, None, None, None, None, 1, None, 1, None, 0, None),
    ):
        assert status == -1
        assert b"null" in lib.culsh_last_error()


def test_names_are_public():
    import culsh_b200
    for name in ("Int8Rows", "CrossEntropy", "cross_entropy", "cross_entropy_backward"):
        assert name in culsh_b200.__all__ and getattr(culsh_b200, name) is not None


def test_arguments_are_checked_before_a_device_is_needed():
    import torch

    import culsh_b200 as culsh
    z = torch.zeros
    with pytest.raises(ValueError):
        culsh.cross_entropy(z(2, 2), z(2, 2), z(2).long(), temperature=0.0)
    with pytest.raises(ValueError):
        culsh.cross_entropy_backward(z(2, 2), z(2, 2), z(2).long(), culsh.CrossEntropy(z(2), z(2), z(2)), z(2), temperature=float("nan"))
    for codes, scales, squares, d in ((z(2, 16, dtype=torch.int8), z(2), z(2, dtype=torch.int32), 0), (z(2, 16, dtype=torch.int8), z(2), z(2, dtype=torch.int32), 17),
                                      (z(2, 16), z(2), z(2, dtype=torch.int32), 16), (z(2, 16, dtype=torch.int8), z(2), z(2), 16),
                                      (z(2, 16, dtype=torch.int8), z(2), z(2, dtype=torch.int32), 16)):
        with pytest.raises(ValueError):
            culsh.Int8Rows.from_parts(codes, scales, squares, d)

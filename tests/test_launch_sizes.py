"""Sizes whose launches would have 2^32 threads or more: of those the low 32 bits would run, without an error.  (Addresses are
looked at, never read: every call here is refused before its launch.)"""
import ctypes

import pytest

from test_training_refusals import _AT, _product, _status


@pytest.mark.parametrize("kw", [
    dict(M=2 ** 27, K=513, lda=513, N=16, ldb=16),                                   # rows of x that are copied
    dict(form=1, M=64, K=513, lda=513, N=2 ** 27, ldb=513),                          # ... of a transposed weight
    dict(form=2, M=513, lda=513, K=2 ** 27, N=16, ldb=16)])
def test_copies_of_operands(kw):
    from atomic_gdn2 import _lib
    p = _product(**kw)
    assert _status("gdn2_linear", ctypes.byref(p), ctypes.c_void_p(_AT), None) == 2
    assert b"too large" in _lib.lib().gdn2_last_error()
    assert _lib.lib().gdn2_linear_workspace_bytes(ctypes.byref(p)) == 0


def test_rows_that_are_not_copied_are_no_reason():
    from atomic_gdn2 import _lib
    L = _lib.lib()
    p = _product(M=2 ** 27, K=513 + 7, lda=520, N=16, ldb=16)
    assert L.gdn2_linear(ctypes.byref(_product(M=0)), ctypes.c_void_p(_AT), None) == 1      # (the error that is looked for below)
    L.gdn2_linear_workspace_bytes(ctypes.byref(p))
    assert b"too large" not in L.gdn2_last_error()


def test_a_tensor_of_adamw():
    from atomic_gdn2 import _lib
    a = dict(p=_AT, g=_AT, m=_AT, v=_AT, m_scale=_AT, v_scale=_AT, master=None, step=_AT, ordinal=0, dtype=0, lr=1e-3, beta1=0.9, beta2=0.99,
             eps=1e-8, weight_decay=0.0)
    t = _lib.Gdn2AdamwTensor(**a, numel=2 ** 34)
    for bits in (8, 32):
        assert _status("gdn2_adamw", ctypes.byref(t), 1, bits, 0.0, None, ctypes.c_void_p(_AT), None) == 1
        assert b"size" in _lib.lib().gdn2_last_error()

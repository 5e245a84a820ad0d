"""The dense products' argument checks, which run before anything is launched or copied (CPU)."""

import numpy as np
import pytest

from artlite_b200 import Error, ffn
from artlite_b200.linear import QuantLinear

W = np.zeros((16, 144), np.uint8)  # (16 Q4_K rows of 256 values)


def test_linear_refuses_types_it_does_not_read():
    for qt in ("Q8_0", "Q6_K", "F32", "BF16"):
        with pytest.raises(Error, match="Q4_0, Q4_1, Q4_K and IQ4_NL"):
            QuantLinear(W, n_in=256, n_out=16, qtype=qt)
    with pytest.raises(Error, match="type Q9"):
        QuantLinear(W, n_in=256, n_out=16, qtype="Q9")
    with pytest.raises(Error, match="activation type f64"):
        QuantLinear(W, n_in=256, n_out=16, qtype="Q4_K", act_dtype="f64")
    with pytest.raises(Error, match="activation relu"):
        QuantLinear(W, n_in=256, n_out=16, qtype="Q4_K", up=W, activation="relu")


@pytest.mark.parametrize("n_in,n_out,qt", [(0, 16, "Q4_0"), (33, 16, "Q4_0"), (128, 16, "Q4_K"), (256, 0, "Q4_K"),
                                           (-32, 16, "Q4_1")])
def test_linear_refuses_shapes(n_in, n_out, qt):
    with pytest.raises(Error, match="whole blocks"):
        QuantLinear(W, n_in=n_in, n_out=n_out, qtype=qt)


def test_linear_refuses_null():
    from artlite_b200._lib import lib
    with pytest.raises(Error, match="null weights"):
        QuantLinear(None, n_in=256, n_out=16, qtype="Q4_K")
    assert lib().artlite_linear_forward(None, None, 1, None, 1, 1, None) != 0
    assert b"null handle" in lib().artlite_moe_last_error()
    assert lib().artlite_linear_destroy(None) == 0


def test_ffn_refuses_shapes_types_and_nulls():
    ok = dict(T=4, n_in=64, n_ffn=32)
    for bad in (dict(n_in=60), dict(n_ffn=36), dict(n_in=0), dict(T=-1)):
        with pytest.raises(Error, match="multiples of 8"):
            ffn.gated_ffn(16, 16, 16, 16, **{**ok, **bad})
        with pytest.raises(Error, match="multiples of 8"):
            ffn.gated_ffn_backward(16, 16, 16, 16, 16, 16, 16, **{**ok, **bad})
    with pytest.raises(Error, match="type f32"):
        ffn.gated_ffn(16, 16, 16, 16, dtype="f32", **ok)
    with pytest.raises(Error, match="activation tanh"):
        ffn.gated_ffn(16, 16, 16, 16, activation="tanh", **ok)
    with pytest.raises(Error, match="null array"):
        ffn.gated_ffn(None, 16, 16, 16, **ok)
    with pytest.raises(Error, match="together or not at all"):
        ffn.gated_ffn(16, 16, 16, 16, gate=16, **ok)
    with pytest.raises(Error, match="together or not at all"):
        ffn.gated_ffn_backward(16, 16, 16, 16, 16, 16, 16, dw_gate=16, **ok)
    with pytest.raises(Error, match="dx needs the matrices"):
        ffn.gated_ffn_backward(16, 16, None, None, 16, 16, 16, dx=16, **ok)
    with pytest.raises(Error, match="need x"):
        ffn.gated_ffn_backward(16, None, None, None, 16, 16, 16, dw_gate=16, dw_up=16, **ok)


def test_ffn_refuses_alignment_strides_and_host_memory():
    a = np.zeros(4096, np.uint16)
    p = (a.ctypes.data + 15) // 16 * 16
    kw = dict(T=4, n_in=64, n_ffn=32)
    for bad, what in ((dict(ldx=66), "x is not"), (dict(ldx=56), "x is not"), (dict(ldh=36), "h is not")):
        with pytest.raises(Error, match="not device memory|" + what):
            ffn.gated_ffn(p, p, p, p, **{**kw, **bad})
    with pytest.raises(Error, match="x is not 16-byte aligned"):
        ffn.gated_ffn(p + 2, p, p, p, **kw)
    with pytest.raises(Error, match="x is not device memory"):
        ffn.gated_ffn(p, p, p, p, **kw)


def test_ffn_work_bytes():
    assert ffn.gated_ffn_work_bytes(5, 64) == 2 * 5 * 64 * 2
    assert ffn.gated_ffn_work_bytes(0, 64) == 0
    assert ffn.gated_ffn_work_bytes(1 << 20, 1 << 14) == 4 << 34  # (past 32 bits)


def test_linear_refuses_weights_of_another_size():
    for w in (W[:15], np.zeros((16, 143), np.uint8), np.zeros((17, 144), np.uint8)):
        with pytest.raises(Error, match="bytes of weights"):
            QuantLinear(w, n_in=256, n_out=16, qtype="Q4_K")
        with pytest.raises(Error, match="bytes of weights"):
            QuantLinear(W, up=w, n_in=256, n_out=16, qtype="Q4_K")

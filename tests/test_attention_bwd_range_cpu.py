"""Scales and caps for which the backward pass would divide or multiply past fp32's range are refused before any launch."""
import ctypes

import pytest

P = ctypes.c_void_p
OK, ARGUMENT = 0, 3


def call(lib, scale, softcap, batch=0):
    return lib.plb_attention_bwd(*[P(4096)] * 10, 1 << 20, batch, 128, 2, 1, scale, 0, softcap, None, None)


@pytest.mark.parametrize("scale,softcap", [(2.0 ** -97, 0.0), (1.2e-38, 0.0), (2.0 ** 97, 0.0), (3e38, 0.0), (0.0, 0.0), (-1.0, 0.0),
                                           (float("nan"), 0.0), (float("inf"), 0.0), (0.1, 2.0 ** 97), (0.1, 3e38), (0.1, -1.0),
                                           (0.1, float("nan")), (1.0, 1e-39)])
def test_refused(native_lib, scale, softcap):
    for batch in (0, 1):
        assert call(native_lib, scale, softcap, batch) == ARGUMENT


@pytest.mark.parametrize("scale,softcap", [(2.0 ** -96, 0.0), (2.0 ** 96, 0.0), (0.088, 2.0 ** 96), (0.088, 1e-30), (0.088, 30.0)])
def test_taken(native_lib, scale, softcap):
    assert call(native_lib, scale, softcap) == OK          # no batch: checked, and nothing to launch

"""Refusals of the 4-bit pools and of reading a pool back, and the tests' own quantiser: CPU only."""
import ctypes as C

import numpy as np
import pytest

import int4_ref as ref
from gollmgo_amd import _lib
from gollmgo_amd._lib import DType, ScaleMode, Status


def test_create_refuses_before_any_device_call():
    lib, h = _lib.lib(), C.c_void_p()
    for mode in (ScaleMode.NONE, ScaleMode.PER_HEAD, ScaleMode.PER_BLOCK):
        assert lib.gg_kv_create(1, 1, 16, 1, 128, int(DType.INT4), int(mode), C.byref(h)) == Status.ERR_INVALID
        assert "PER_TOKEN" in _lib.last_error()
    assert lib.gg_kv_create(1, 1, 16, 1, 127, int(DType.INT4), int(ScaleMode.PER_TOKEN), C.byref(h)) == Status.ERR_INVALID
    assert "even" in _lib.last_error()
    assert lib.gg_kv_create(1, 1, 16, 1, 128, int(DType.BF16), int(ScaleMode.PER_TOKEN), C.byref(h)) == Status.ERR_INVALID
    assert lib.gg_kv_create(1, 1, 16, 1, 128, int(DType.INT8), int(ScaleMode.PER_TOKEN), C.byref(h)) == Status.ERR_INVALID
    assert lib.gg_kv_create(1, 1, 16, 1, 128, 6, 0, C.byref(h)) == Status.ERR_INVALID
    assert not h.value


def test_read_refuses_no_handle():
    assert _lib.lib().gg_kv_read(None, 0, None, None, 0, None, 1, None) == Status.ERR_INVALID
    assert "kv is NULL" in _lib.last_error()


@pytest.mark.parametrize("seed", range(4))
def test_rule_holds_zero_and_half_steps(seed):
    """No value moves by more than half a step, zero stays zero, and the scale has five bits."""
    rng = np.random.default_rng(seed)
    x = (rng.normal(0, 1, (500, 64)) * np.exp2(rng.integers(-20, 21, (500, 1)))).astype(np.float32)
    x[:, 3] = 0
    if seed == 1:
        x = np.abs(x)
    n, s, z = ref.quantise(x)
    v = ref.values(n, s, z)
    assert (np.abs(v - x) <= s[:, None] * (0.5 + 2.0 ** -20)).all()
    assert (v[:, 3] == 0).all()
    assert ((s.view(np.uint32) & 0x7FFFF) == 0).all()
    assert (s <= (x.max(-1).clip(0) - x.min(-1).clip(None, 0)) / 15 * (1 + 1 / 16) * (1 + 2.0 ** -20)).all()

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


def rope_call(**kw):
    a = dict(q=1, qs=256, k=1, ks=128, dt=int(DType.F32), n=4, hq=4, hk=2, d=64, wq=None, wk=None, eps=1e-6, pos=1, axes=1,
             axis=None, freq=1, pairs=32, style=0, qo=1, ko=1, stream=None)
    a.update(kw)
    return _lib.lib().gg_qk_norm_rope(*a.values())


@pytest.mark.parametrize("bad,word", [
    (dict(dt=int(DType.INT4)), "dtype"), (dict(n=-1), "n_rows"), (dict(n=(1 << 24) + 1), "n_rows"), (dict(hq=0, hk=0), "head count"),
    (dict(hq=-1), "head count"), (dict(d=0), "head_dim"), (dict(d=1025, qs=9999, ks=9999), "head_dim"), (dict(pairs=33), "num_pairs"),
    (dict(pairs=-1), "num_pairs"), (dict(axes=0), "num_axes"), (dict(axes=9), "num_axes"), (dict(style=2), "style"),
    (dict(eps=float("nan")), "eps"), (dict(eps=-1e-9), "eps"), (dict(qs=255), "overlap"), (dict(ks=127), "overlap"),
    (dict(q=None), "NULL"), (dict(qo=None), "NULL"), (dict(k=None), "NULL"), (dict(ko=None), "NULL"), (dict(pos=None), "NULL"),
    (dict(freq=None), "NULL"), (dict(axis=bytes([1] * 32)), "pair_axis"),
])
def test_norm_rope_refuses_before_any_device_call(bad, word):
    assert rope_call(**bad) == Status.ERR_INVALID
    assert word in _lib.last_error()


def test_norm_rope_append_refuses_no_handle():
    lib = _lib.lib()
    assert lib.gg_qk_norm_rope_append(None, 0, 1, 256, 1, 128, 1, 128, 0, 4, 4, None, None, 1e-6, 1, 1, None, 1, 32, 0, 1, 1,
                                      None) == Status.ERR_INVALID
    assert "kv is NULL" in _lib.last_error()


# (4 rows of 4 query heads, 2 kv heads of 64 fp32 values: 1024 bytes a query row, 512 a key row.)
Q, K, QO, KO = 0x10000, 0x20000, 0x30000, 0x40000


@pytest.mark.parametrize("bad", [
    dict(qo=Q + 4), dict(qo=Q + 4095), dict(qo=Q - 4095), dict(qo=Q, qs=512), dict(ko=K, ks=256), dict(ko=K + 2047),
    dict(qo=K + 2047), dict(qo=K - 4095), dict(ko=Q), dict(ko=Q + 4092), dict(ko=QO + 4095), dict(qo=KO),
    dict(k=Q + 1024, qs=384, ks=384, qo=Q + 1536),
])
def test_norm_rope_refuses_overlaps(bad):
    a = dict(q=Q, k=K, qo=QO, ko=KO)
    a.update(bad)
    assert rope_call(**a) == Status.ERR_INVALID
    assert "overlaps" in _lib.last_error()

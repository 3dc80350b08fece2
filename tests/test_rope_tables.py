"""Values of rt_rope_tables' scalings against the formulas in 64 bits (CPU only): fp32 roundings of cos and sin, 2^-24 at most,
and the double arithmetic's own 2^-52 of angles up to some 1e5."""
import ctypes

import numpy as np
import pytest

from rustane_b200 import _lib


def tables(n_pos, rot, theta=10000.0, scaling=_lib.RT_ROPE_PLAIN, factor=1.0, low=1.0, high=32.0, trained=0):
    cos, sin = (np.full((n_pos, rot // 2), 9.0, np.float32) for _ in "cs")
    p = ctypes.POINTER(ctypes.c_float)
    rc = _lib.lib().rt_rope_tables(cos.ctypes.data_as(p), sin.ctypes.data_as(p), n_pos, rot, theta, scaling, factor, low, high, trained)
    return rc, cos, sin


def check(got, f):
    rc, cos, sin = got
    assert rc == _lib.RT_OK
    a = np.arange(cos.shape[0])[:, None] * f
    assert np.abs(cos - np.cos(a)).max() <= 2.0**-24 + 1e-10
    assert np.abs(sin - np.sin(a)).max() <= 2.0**-24 + 1e-10


@pytest.mark.parametrize("rot", [16, 64, 128])
@pytest.mark.parametrize("theta", [10000.0, 500000.0])
def test_plain_and_linear(rot, theta):
    f = theta ** (-2.0 * np.arange(rot // 2) / rot)
    check(tables(1000, rot, theta), f)
    check(tables(1000, rot, theta, _lib.RT_ROPE_LINEAR, 4.0), f / 4)
    check(tables(1000, rot, theta, _lib.RT_ROPE_LINEAR, 0.5), f * 2)


@pytest.mark.parametrize("factor,low,high,trained", [(8.0, 1.0, 4.0, 8192), (32.0, 1.0, 32.0, 4096), (2.0, 0.5, 0.75, 100)])
def test_bands(factor, low, high, trained):
    """Pairs that turn often over the trained positions keep their frequency, slow ones turn `factor` times slower, those between
    take a mean weighted by where their turns lie."""
    f = 500000.0 ** (-2.0 * np.arange(64) / 128)
    got = tables(3000, 128, 500000.0, _lib.RT_ROPE_BANDS, factor, low, high, trained)
    exp = []
    for x in f:
        turns = trained * x / (2 * np.pi)
        if turns > high:
            exp.append(x)
        elif turns < low:
            exp.append(x / factor)
        else:
            t = (turns - low) / (high - low)
            exp.append(x * t + x / factor * (1 - t))
    assert sum(abs(e - x) < 1e-15 for e, x in zip(exp, f)) and sum(abs(e - x / factor) < 1e-15 for e, x in zip(exp, f))
    check(got, np.array(exp))


@pytest.mark.parametrize("kw,rc", [(dict(scaling=3), _lib.RT_ERR_ARG), (dict(scaling=1, factor=0.0), _lib.RT_ERR_ARG),
                                   (dict(scaling=1, factor=float("nan")), _lib.RT_ERR_ARG),
                                   (dict(scaling=2, factor=8.0, low=4.0, high=4.0, trained=10), _lib.RT_ERR_ARG),
                                   (dict(scaling=2, factor=8.0, low=0.0, trained=10), _lib.RT_ERR_ARG),
                                   (dict(scaling=2, factor=8.0, trained=0), _lib.RT_ERR_ARG), (dict(theta=0.0), _lib.RT_ERR_SHAPE)])
def test_refusals_write_nothing(kw, rc):
    got, cos, sin = tables(4, 16, **kw)
    assert got == rc and (cos == 9).all() and (sin == 9).all()

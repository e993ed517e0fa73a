"""AdamW's argument checks (optimizers.AdamW, rst_adamw_*): refusals on the host, before any device work."""
import ctypes

import numpy as np
import pytest
import torch

from realtime_style_transfer_amd import _lib as L
from realtime_style_transfer_amd.optimizers import AdamW


def _lib():
    from realtime_style_transfer_amd import build
    build.build()
    return L.load()


def test_hyperparameters():
    for bad in (dict(state_bits=16), dict(global_clipnorm=0.0), dict(global_clipnorm=-1.0), dict(beta_1=1.0),
                dict(beta_2=-0.1), dict(epsilon=0.0), dict(epsilon=-1e-8), dict(global_clipnorm=float('inf')), dict(learning_rate=float('nan')),
                dict(weight_decay=float('inf'))):
        with pytest.raises(ValueError):
            AdamW(**bad)
    opt = AdamW(learning_rate=2e-4, global_clipnorm=1.0, state_bits=8)
    assert (opt.learning_rate, opt.beta_1, opt.beta_2, opt.global_clipnorm, opt.state_bits) == (2e-4, 0.9, 0.999, 1.0, 8)


def test_unbuilt_and_bad_variables():
    opt = AdamW()
    with pytest.raises(ValueError, match="no variables yet"):
        opt.apply_gradients(torch.zeros(4))
    for use in (lambda: opt.iterations, opt.slots, lambda: opt.set_slots([], [])):
        with pytest.raises(ValueError):
            use()
    with pytest.raises(ValueError):
        opt.build([])
    with pytest.raises(ValueError, match="CPU tensor"):
        opt.build([torch.zeros(4)])
    a = np.zeros(8, np.float32)
    with pytest.raises(ValueError, match="share memory"):      # the same variable twice, or overlapping ones
        opt._build([a.ctypes.data, a.ctypes.data], [4, 4], None, [True, True], 'cuda:0')
    with pytest.raises(ValueError, match="share memory"):
        opt._build([a.ctypes.data, a.ctypes.data + 12], [4, 4], None, [True, True], 'cuda:0')
    with pytest.raises(ValueError, match="decay"):
        opt._build([a.ctypes.data], [4], None, [True, False], 'cuda:0')


def test_create_refusals():
    lib = _lib()
    a = np.zeros(1024, np.float32)
    p = a.ctypes.data
    p += -p % 16
    h = ctypes.c_void_p()

    def create(param=p, count=8, n=1, bits=32, m=p, v=p, ms=p, vs=p, it=p, out=h, null=False):
        t = (L.RstAdamwTensor * 1)(L.RstAdamwTensor(param, count, 0, 1))
        s = L.RstAdamwState(m, v, ms, vs, it, None)
        return lib.rst_adamw_create(None if null else t, n, bits, ctypes.byref(s), ctypes.byref(out))
    for change, code in [(dict(null=True), 1), (dict(n=0), 1), (dict(bits=16), 2), (dict(it=None), 1),
                         (dict(param=None), 1), (dict(m=None), 1), (dict(v=None), 1), (dict(bits=8, ms=None), 1),
                         (dict(bits=8, vs=None), 1), (dict(bits=8, m=p + 4), 1), (dict(count=2 ** 37), 1),
                         (dict(count=2 ** 64 - 1), 1)]:
        assert create(**change) == code, (change, lib.rst_last_error())
        assert h.value is None and b"rst_adamw_create" in lib.rst_last_error()
    cfg = L.RstAdamwConfig(1e-3, 0, 0.9, 0.999, 1e-7, 0, 0)
    assert lib.rst_adamw_step(None, p, 0, ctypes.byref(cfg), None) == 1
    assert lib.rst_adamw_step_tensors(None, None, 1, 0, ctypes.byref(cfg), None) == 1
    assert lib.rst_adamw_num_blocks(None) == 0
    lib.rst_adamw_destroy(None)
    assert not lib.rst_trainer_weights(None) and not lib.rst_predictor_trainer_weights(None)
    assert lib.rst_trainer_weights_updated(None, None) == 1


def test_no_elements():
    lib = _lib()
    a = np.zeros(64, np.float32)
    p, h = a.ctypes.data, ctypes.c_void_p()
    t = (L.RstAdamwTensor * 2)(L.RstAdamwTensor(p, 0, 0, 1), L.RstAdamwTensor(None, 0, 0, 1))
    s = L.RstAdamwState(p, p, p, p, p, None)
    assert lib.rst_adamw_create(t, 2, 32, ctypes.byref(s), ctypes.byref(h)) == L.RST_ERR_INVALID and h.value is None
    with pytest.raises(ValueError, match="no variable has an element"):
        AdamW()._build([p, p], [0, 0], None, [True, True], 'cuda:0')


def test_hyperparameters_that_32_bits_do_not_hold():
    """The kernels divide by epsilon in 32 bits: below 2^-126 its reciprocal is none there, and 0 / epsilon a NaN."""
    for bad in (dict(epsilon=1e-50), dict(epsilon=2.0 ** -127), dict(epsilon=1e39), dict(learning_rate=1e39),
                dict(learning_rate=-1e39), dict(weight_decay=1e39)):
        with pytest.raises(ValueError, match="32 bits"):
            AdamW(**bad)
    opt = AdamW(epsilon=2.0 ** -126, learning_rate=1e38, weight_decay=-1e38)
    opt.epsilon = 1e-44
    with pytest.raises(ValueError, match="32 bits"):
        opt._check_config()


def test_more_workgroups_than_a_launch_takes_are_refused():
    """HIP launches fewer than 2^32 threads: 2^24 chunks of 256. A variable's chunk is 4096 elements at most."""
    lib = _lib()
    a = np.zeros(64, np.float32)
    p, h = a.ctypes.data, ctypes.c_void_p()
    s = L.RstAdamwState(p, p, p, p, p, None)
    half = (L.RstAdamwTensor * 2)(L.RstAdamwTensor(p, 2 ** 35, 0, 1), L.RstAdamwTensor(p, 2 ** 35, 2 ** 35, 1))
    for bits in (8, 32):
        assert lib.rst_adamw_create(half, 2, bits, ctypes.byref(s), ctypes.byref(h)) == L.RST_ERR_UNSUPPORTED
        assert h.value is None and b"one launch" in lib.rst_last_error()

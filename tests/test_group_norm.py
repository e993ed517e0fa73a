"""Group normalisation's argument checks (styleTransfer.group_norm, group_norm_gradients, rst_group_norm*): every refusal
happens on the host, before any device work."""
import numpy as np
import pytest
import torch

from realtime_style_transfer_amd import _lib as L
from realtime_style_transfer_amd.styleTransfer import group_norm, group_norm_gradients

F32, BF16 = L.DTYPES["float32"], L.DTYPES["bfloat16"]


def _lib():
    from realtime_style_transfer_amd import build
    build.build()
    return L.load()


def _buffer(n=64):
    a = np.zeros(n + 4, np.float32)
    at = a.ctypes.data
    return a, at + (-at % 16)


def _forward(lib, x, dtype=F32, batch=1, hw=4, channels=4, groups=2, act=0, eps=1e-5, y=None, ws=None, scale=None):
    return lib.rst_group_norm(x, dtype, batch, hw, channels, groups, x if scale is None else scale, x, 0, eps, act,
                              x if y is None else y, None, None, x if ws is None else ws, None)


@pytest.mark.parametrize("change, code", [
    (dict(groups=3), L.RST_ERR_INVALID), (dict(groups=0), L.RST_ERR_INVALID), (dict(channels=0), L.RST_ERR_INVALID),
    (dict(batch=-1), L.RST_ERR_INVALID), (dict(hw=-1), L.RST_ERR_INVALID), (dict(eps=-1.0), L.RST_ERR_INVALID),
    (dict(eps=float('nan')), L.RST_ERR_INVALID), (dict(y=0), L.RST_ERR_INVALID), (dict(scale=0), L.RST_ERR_INVALID),
    (dict(ws=0), L.RST_ERR_INVALID), (dict(dtype=2), L.RST_ERR_UNSUPPORTED), (dict(act=4), L.RST_ERR_UNSUPPORTED),
    (dict(act=-1), L.RST_ERR_UNSUPPORTED), (dict(batch=2 ** 31 - 1, hw=2 ** 31 - 1), L.RST_ERR_UNSUPPORTED)])
def test_forward_refusals(change, code):
    lib = _lib()
    keep, x = _buffer()
    if change.get('y') == 0:
        change = dict(change, y=None)
        rc = lib.rst_group_norm(x, F32, 1, 4, 4, 2, x, x, 0, 1e-5, 0, None, None, None, x, None)
    elif change.get('scale') == 0:
        rc = lib.rst_group_norm(x, F32, 1, 4, 4, 2, None, x, 0, 1e-5, 0, x, None, None, x, None)
    elif change.get('ws') == 0:
        rc = lib.rst_group_norm(x, F32, 1, 4, 4, 2, x, x, 0, 1e-5, 0, x, None, None, x + 4, None)
    else:
        rc = _forward(lib, x, **change)
    assert rc == code, lib.rst_last_error()
    assert b"rst_group_norm" in lib.rst_last_error()


def test_empty_forward_is_ok_and_touches_nothing():
    lib = _lib()
    assert lib.rst_group_norm(None, F32, 0, 4, 4, 2, None, None, 0, 1e-5, 0, None, None, None, None, None) == L.RST_OK
    assert lib.rst_group_norm(None, F32, 2, 0, 4, 2, None, None, 0, 1e-5, 0, None, None, None, None, None) == L.RST_OK


def test_backward_refusals():
    lib = _lib()
    keep, x = _buffer()
    ok = [x, x, F32, 1, 4, 4, 2, x, x, 0, x, x, 0, x, x, x, x, None]
    for at, bad, code in [(0, None, 1), (1, None, 1), (7, None, 1), (8, None, 1), (10, None, 1), (11, None, 1),
                          (13, None, 1), (14, None, 1), (15, None, 1), (16, x + 8, 1), (6, 3, 1),
                          (2, 7, 2), (12, 9, 2), (3, -1, 1)]:
        args = list(ok)
        args[at] = bad
        assert lib.rst_group_norm_backward(*args) == code, (at, bad)
        assert b"rst_group_norm_backward" in lib.rst_last_error()


def test_workspace_size():
    lib = _lib()
    for size in (lib.rst_group_norm_workspace_size, lib.rst_group_norm_backward_workspace_size):
        assert size(0, 4, 4, 2) == 0 and size(1, 4, 4, 3) == 0 and size(1, 4, 0, 1) == 0
        assert size(1, 450, 96, 8) == 0                              # one launch holds it in registers
        assert 0 < size(1, 28800, 128, 32) < 64 << 20
        assert 0 < size(4, 480 * 960, 32, 8) < 64 << 20              # partial sums, not another tensor
    assert lib.rst_group_norm_backward_workspace_size(3, 450, 96, 8) == 3 * 96 * 16     # a shared affine's sums


def test_a_workspace_that_is_needed_has_to_be_there():
    lib = _lib()
    keep, x = _buffer()
    assert lib.rst_group_norm(x, F32, 1, 28800, 128, 32, x, x, 0, 1e-5, 0, x, None, None, None, None) == L.RST_ERR_INVALID
    assert lib.rst_group_norm_backward(x, x, F32, 1, 28800, 128, 32, x, x, 0, x, x, 0, x, x, x, None, None) == \
        L.RST_ERR_INVALID


def test_python_refusals_without_a_device():
    x = torch.zeros(2, 3, 5, 8)
    s, st = torch.ones(8), torch.zeros(2, 4)
    for bad in [dict(x=x[0]), dict(x=x.double()), dict(x=x.half()), dict(groups=3), dict(groups=0),
                dict(activation="gelu"), dict(scale=torch.ones(2, 8)), dict(scale=torch.ones(4), bias=torch.ones(4)),
                dict()]:                                             # the last one: a CPU tensor
        a = dict(x=x, scale=s, bias=s, groups=4, activation="relu")
        a.update(bad)
        with pytest.raises(ValueError):
            group_norm(a['x'], a['scale'], a['bias'], a['groups'], activation=a['activation'])
    with pytest.raises(ValueError):
        group_norm_gradients(x, x, s, s, st, st, 4)


def test_sizes_past_the_interface_are_refused():
    """2^32 pixels are none in 32 bits, and a row of 2^28 channels is past 32 bits of offset."""
    lib = _lib()
    keep, x = _buffer()
    assert _forward(lib, x, channels=2 ** 27 + 8, groups=1, hw=1) == L.RST_ERR_UNSUPPORTED
    assert lib.rst_group_norm_backward(x, x, F32, 1, 1, 2 ** 28, 2, x, x, 0, x, x, 0, x, x, x, x, None) == \
        L.RST_ERR_UNSUPPORTED
    s = torch.ones(1)
    for shape in ((1, 2 ** 16, 2 ** 16, 1), (2 ** 31, 1, 1, 1)):
        with pytest.raises(ValueError, match="2\\^31"):
            group_norm(torch.empty(shape, dtype=torch.bfloat16, device='meta'), s, s, 1)


def test_numbers_of_other_kinds():
    """Groups as any whole number, eps as any real one; a group count of 2.0 is none."""
    x, s, st = torch.zeros(2, 3, 5, 14), torch.ones(14), torch.zeros(2, 7)
    for groups, eps in ((np.int64(7), np.float32(1e-5)), (torch.tensor(7), torch.tensor(1e-5))):
        with pytest.raises(ValueError, match="CPU tensor"):
            group_norm(x, s, s, groups, eps=eps)
        with pytest.raises(ValueError, match="CPU tensor"):
            group_norm_gradients(x, x, s, s, st, st, groups)
    for call in (lambda: group_norm(x, s, s, 7.0), lambda: group_norm_gradients(x, x, s, s, st, st, 7.0)):
        with pytest.raises(TypeError):
            call()

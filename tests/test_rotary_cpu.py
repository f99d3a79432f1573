"""The rotation ops without a GPU: frequency plans, schemas, fakes and the C
ABI's refusals, which are decided before any device is touched."""
import ctypes
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from kernels import rotary as rot
from tests import capi_rotary as capi


def test_plain_frequencies():
    f = rot.rotary_frequencies(64)
    assert f.dtype == torch.float64 and f.shape == (32,)
    for i in (0, 1, 31):
        assert math.isclose(float(f[i]), 10000.0 ** (-2 * i / 64), rel_tol=1e-15)


def test_linear_and_ntk_scaling():
    f = rot.rotary_frequencies(64)
    torch.testing.assert_close(rot.rotary_frequencies(64, scaling="linear", factor=4.0), f / 4)
    n = rot.rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert float(n[0]) == 1.0
    assert math.isclose(float(n[-1]), float(f[-1]) / 4, rel_tol=1e-12)
    assert ((n <= f) & (n >= f / 4 * (1 - 1e-12))).all()


def test_yarn_scaling():
    f = rot.rotary_frequencies(128, 10000.0)
    y = rot.rotary_frequencies(128, 10000.0, scaling="yarn", factor=16.0, original_length=4096)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(y[turns >= 32], f[turns >= 32])
    torch.testing.assert_close(y[turns <= 1], f[turns <= 1] / 16)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and ((y[mid] < f[mid]) & (y[mid] > f[mid] / 16)).all()
    assert (y[1:] < y[:-1]).all()
    assert rot.rotary_amplitude(1.0) == 1.0
    assert math.isclose(rot.rotary_amplitude(16.0), 1 + 0.1 * math.log(16.0))


@pytest.mark.parametrize("kw", [dict(rotary_dim=63), dict(rotary_dim=0), dict(scaling="x"),
                                dict(factor=2.0), dict(scaling="yarn", factor=2.0),
                                dict(scaling="yarn", factor=2.0, original_length=64, slow=9, fast=8),
                                dict(base=0.0), dict(scaling="linear", factor=0.0),
                                dict(rotary_dim=2, scaling="ntk", factor=2.0)])
def test_frequency_refusals(kw):
    with pytest.raises(ValueError):
        rot.rotary_frequencies(**{"rotary_dim": 64, **kw})


def test_ops_have_cuda_kernels_only():
    rot._ensure_registered()
    for name in ("rotary", "qk_norm_rotary", "qk_norm_rotary_bwd"):
        assert torch._C._dispatch_has_kernel_for_dispatch_key(f"vlak::{name}", "CUDA")
        assert not torch._C._dispatch_has_kernel_for_dispatch_key(f"vlak::{name}", "CPU")


def test_fakes_are_contiguous():
    rot._ensure_registered()
    with FakeTensorMode():
        x = torch.empty(2, 5, 9, 64, device="cuda", dtype=torch.bfloat16)
        pos = torch.empty(5, device="cuda", dtype=torch.int64)
        f = torch.empty(32, device="cuda", dtype=torch.float64)
        w = torch.empty(64, device="cuda")
        q, k = rot.rotary(x[:, :, :6], x[:, :, 6:], pos, f)
        assert q.shape == (2, 5, 6, 64) and k.shape == (2, 5, 3, 64)
        assert q.is_contiguous() and k.is_contiguous()
        assert rot.qk_norm_rotary(x[0], None, w, None, pos, f).shape == (5, 9, 64)
        d = torch.ops.vlak.qk_norm_rotary_bwd(q, k, q, k, w, w, pos, f)
        assert [t.shape for t in d] == [q.shape, k.shape, w.shape, w.shape]


def _args(**kw):
    a = capi.RotaryArgs()
    for t in a.t:
        t.x = t.grad = t.y = t.weight = t.grad_weight = 0x1000
        t.H = 3
        t.x_stride[:] = t.grad_stride[:] = (960, 192, 64)
    a.positions = a.inv_freq = 0x1000
    a.B, a.M, a.D, a.rotary_dim = 2, 5, 64, 64
    a.pos_stride[:] = (5, 1)
    a.amplitude, a.eps = 1.0, 1e-6
    a.n_tensors, a.dtype, a.pos_dtype, a.weight_dtype = 2, 2, 5, 0
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BAD = [dict(dtype=3), dict(dtype=9), dict(pos_dtype=0), dict(B=-1), dict(M=1 << 31), dict(D=0),
       dict(D=63), dict(D=1026), dict(rotary_dim=66), dict(rotary_dim=0), dict(rotary_dim=7),
       dict(n_tensors=0), dict(n_tensors=3), dict(amplitude=float("inf")), dict(eps=-1.0),
       dict(eps=float("nan")), dict(weight_dtype=1), dict(positions=None), dict(positions=0x1004),
       dict(inv_freq=None), dict(inv_freq=0x1004)]


@pytest.mark.parametrize("kw", BAD)
def test_c_abi_refuses(kw):
    L = capi.lib()
    a = _args(**kw)
    assert L.vlak_qk_norm_rotary_fwd(ctypes.byref(a), None) in (1, 2, 3)
    assert b"qk_norm_rotary" in L.vlak_last_error_message()
    assert L.vlak_qk_norm_rotary_bwd(ctypes.byref(a), 0x1000, 1 << 40, None) in (1, 2, 3)
    if not set(kw) & {"eps", "weight_dtype"}:
        assert L.vlak_rotary(ctypes.byref(a), None) in (1, 2, 3)


@pytest.mark.parametrize("field", ["x", "y", "weight", "grad", "grad_weight"])
def test_c_abi_refuses_null_and_misaligned_tensors(field):
    L = capi.lib()
    for value in (None, 0x1001):
        a = _args()
        setattr(a.t[1], field, value)
        assert L.vlak_qk_norm_rotary_bwd(ctypes.byref(a), 0x1000, 1 << 40, None) in (1, 2)
    a = _args()
    a.t[0].H = 0
    assert L.vlak_rotary(ctypes.byref(a), None) == 1
    assert L.vlak_rotary(None, None) == 1

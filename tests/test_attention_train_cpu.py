"""The training attention op without a GPU: schemas, fakes, the dispatcher keys
and the C ABI's refusals, which are decided before any device is touched."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from kernels import _native, attention
from tests import capi


class TrainArgs(ctypes.Structure):
    _fields_ = [("attn", capi.GqaArgs), ("lengths", ctypes.c_void_p), ("mask", ctypes.c_void_p),
                ("mask_stride_b", ctypes.c_int64), ("mask_stride_m", ctypes.c_int64),
                ("lse", ctypes.c_void_p), ("o_low", ctypes.c_void_p), ("grad_o", ctypes.c_void_p),
                ("grad_o_stride", ctypes.c_int64 * 3), ("dq", ctypes.c_void_p),
                ("dk", ctypes.c_void_p), ("dv", ctypes.c_void_p), ("lengths_dtype", ctypes.c_int)]


def lib():
    L = _native.capi()
    p, n = ctypes.POINTER(TrainArgs), ctypes.c_int64
    L.vlak_attn_gqa_train_fwd.argtypes = [p, ctypes.c_void_p, n, ctypes.c_void_p]
    L.vlak_attn_gqa_bwd.argtypes = [p, ctypes.c_void_p, n, ctypes.c_void_p]
    L.vlak_attn_gqa_bwd_workspace_size.argtypes = [p, ctypes.POINTER(n)]
    return L


def args(attn=(), **kw):
    t = TrainArgs()
    a = t.attn
    a.q = a.k = a.v = a.o = t.lse = t.grad_o = t.dq = t.dk = t.dv = 0x1000
    a.B, a.M, a.N, a.H, a.Hkv = 2, 50, 291, 15, 5
    a.q_stride[:] = a.o_stride[:] = t.grad_o_stride[:] = (48000, 960, 64)
    a.k_stride[:] = a.v_stride[:] = (93120, 320, 64)
    a.scale, a.prefix_len = -1.0, 241
    t.lengths_dtype = 5
    for k, v in dict(attn).items():
        setattr(a, k, v)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


BAD_ATTN = [dict(H=16), dict(Hkv=0), dict(B=-1), dict(prefix_len=292), dict(q=0x1008),
            dict(dead_start=5, dead_end=4), dict(dead_end=242), dict(H=645)]
BAD = [dict(lse=0x1002), dict(o_low=0x1008), dict(lengths=0x1000, mask=0x1000), dict(lengths=0x1004),
       dict(lengths=0x1000, lengths_dtype=2), dict(mask=0x1000, mask_stride_b=-1), dict(lse=None)]


@pytest.mark.parametrize("attn", BAD_ATTN)
def test_c_abi_refuses_attention(attn):
    L = lib()
    t, n = args(attn), ctypes.c_int64(0)
    assert L.vlak_attn_gqa_train_fwd(ctypes.byref(t), None, 0, None) in (1, 2)
    assert L.vlak_attn_gqa_bwd(ctypes.byref(t), 0x1000, 1 << 40, None) in (1, 2)
    if "q" not in attn:
        assert L.vlak_attn_gqa_bwd_workspace_size(ctypes.byref(t), ctypes.byref(n)) == 1


@pytest.mark.parametrize("kw", BAD)
def test_c_abi_refuses_masks_and_statistics(kw):
    L = lib()
    t = args(**kw)
    assert L.vlak_attn_gqa_train_fwd(ctypes.byref(t), None, 0, None) in (1, 2, 3)
    assert L.vlak_attn_gqa_bwd(ctypes.byref(t), 0x1000, 1 << 40, None) in (1, 2, 3)


@pytest.mark.parametrize("field", ["grad_o", "dq", "dk", "dv"])
def test_c_abi_refuses_gradient_pointers(field):
    L = lib()
    for value in (None, 0x1008):
        t = args(**{field: value})
        assert L.vlak_attn_gqa_bwd(ctypes.byref(t), 0x1000, 1 << 40, None) in (1, 2)
    t = args()
    t.grad_o_stride[1] = 961
    assert L.vlak_attn_gqa_bwd(ctypes.byref(t), 0x1000, 1 << 40, None) == 2


def test_c_abi_refuses_workspaces():
    L = lib()
    t, n = args(), ctypes.c_int64(0)
    assert L.vlak_attn_gqa_bwd_workspace_size(ctypes.byref(t), ctypes.byref(n)) == 0
    assert n.value > 0
    assert L.vlak_attn_gqa_bwd(ctypes.byref(t), None, 0, None) == 1
    assert L.vlak_attn_gqa_bwd(ctypes.byref(t), 0x1000, n.value - 1, None) == 1
    assert L.vlak_attn_gqa_bwd(ctypes.byref(t), 0x1010, n.value, None) == 2
    assert L.vlak_attn_gqa_bwd(None, 0x1000, n.value, None) == 1
    assert L.vlak_attn_gqa_train_fwd(None, None, 0, None) == 1
    t = args(dict(B=0))
    assert L.vlak_attn_gqa_bwd_workspace_size(ctypes.byref(t), ctypes.byref(n)) == 0
    assert n.value == 0


@pytest.mark.parametrize("attn", [dict(B=1 << 20, M=1 << 20), dict(B=1 << 30, N=1 << 30),
                                  dict(B=(1 << 31) - 1, M=(1 << 31) - 1, N=(1 << 31) - 1),
                                  dict(B=1 << 30, M=1, N=1)])
def test_c_abi_refuses_what_no_memory_holds(attn):
    L = lib()
    t, n = args(dict(attn, prefix_len=-1, dead_start=0, dead_end=0)), ctypes.c_int64(0)
    assert L.vlak_attn_gqa_train_workspace_size(ctypes.byref(t), ctypes.byref(n)) == 1
    assert L.vlak_attn_gqa_bwd_workspace_size(ctypes.byref(t), ctypes.byref(n)) == 1
    assert L.vlak_attn_gqa_train_fwd(ctypes.byref(t), 0x1000, 1 << 60, None) == 1
    assert L.vlak_attn_gqa_bwd(ctypes.byref(t), 0x1000, 1 << 60, None) == 1


def test_ops_have_cuda_kernels_only():
    attention._ensure_registered_train()
    for name in ("train", "fwd_lse", "bwd"):
        op = f"vlak::fused_attention_gqa_{name}"
        assert torch._C._dispatch_has_kernel_for_dispatch_key(op, "CUDA")
        assert not torch._C._dispatch_has_kernel_for_dispatch_key(op, "CPU")


def test_fakes():
    with FakeTensorMode():
        x = torch.empty(2, 50, 25, 64, device="cuda", dtype=torch.bfloat16)
        q, k, v = x[:, :, :15], x[:, :, 15:20], x[:, :, 20:]
        o = attention.fused_attention_gqa_train(q, k, v)
        assert o.shape == q.shape and o.is_contiguous()
        o, lse, low = torch.ops.vlak.fused_attention_gqa_fwd_lse(q, k, v)
        assert lse.shape == (2, 50, 15) and lse.dtype == torch.float32
        assert low.shape == q.shape and low.dtype == torch.int8
        d = torch.ops.vlak.fused_attention_gqa_bwd(o, q, k, v, o, lse, low)
        assert [t.shape for t in d] == [q.shape, k.shape, v.shape]
        assert all(t.is_contiguous() for t in d)
        assert len(torch.ops.vlak.fused_attention_gqa_bwd(o, q, k, v, o, lse, low, with_kv=False)) == 1

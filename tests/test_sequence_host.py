"""CPU: the sequence-model operators' argument checks, their FakeTensor kernels and the C entry points' refusals. No
kernel runs here."""

import ctypes
import math

import pytest
import torch

import torchsoftdtw_b200 as T
from torchsoftdtw_b200 import _ext

EINVAL, EDTYPE, EWORKSPACE = -1, -2, -3


def attend(**change):
    a = dict(q=torch.zeros(2, 3, 4, 8), k=torch.zeros(2, 5, 2, 8), v=torch.zeros(2, 5, 2, 8), lengths_x=None,
             lengths_y=None)
    a.update(change)
    return T.cross_attention(**a)


@pytest.mark.parametrize("change,message", [
    ({}, "CUDA devices only"),
    ({"q": torch.zeros(2, 3, 8)}, "must be 4D"),
    ({"v": torch.zeros(2, 6, 2, 8)}, "same shape"),
    ({"q": torch.zeros(3, 3, 4, 8)}, "Batch size"),
    ({"q": torch.zeros(2, 3, 4, 7)}, "same head dimension"),
    ({"q": torch.zeros(2, 3, 4, 129), "k": torch.zeros(2, 5, 2, 129), "v": torch.zeros(2, 5, 2, 129)}, r"\[1, 128\]"),
    ({"q": torch.zeros(2, 3, 4, 0), "k": torch.zeros(2, 5, 2, 0), "v": torch.zeros(2, 5, 2, 0)}, r"\[1, 128\]"),
    ({"q": torch.zeros(2, 3, 3, 8)}, "multiple of the key heads"),
    ({"q": torch.zeros(2, 3, 4, 8).double()}, "float16, bfloat16 or float32"),
    ({"q": torch.zeros(2, 3, 4, 8).half()}, "same dtype"),
    ({"scale": math.inf}, "scale"),
])
def test_attention_refusals(change, message):
    with pytest.raises(RuntimeError, match=message):
        attend(**change)


@pytest.mark.parametrize("change,message", [
    ({}, "CUDA devices only"),
    ({"x": torch.zeros(2, 3, 8)}, "must be 4D"),
    ({"x": torch.zeros(2, 3, 4, 257)}, r"\[1, 256\]"),
    ({"x": torch.zeros(2, 3, 4, 8).double()}, "float16, bfloat16 or float32"),
])
def test_rotate_refusals(change, message):
    with pytest.raises(RuntimeError, match=message):
        T.norm_rotate(**{"x": torch.zeros(2, 3, 4, 8), **change})


def test_clip_refusals():
    g = [torch.zeros(3)]
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        T.clip_grads(g, 1.0)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        T.global_norm(g)
    with pytest.raises(RuntimeError, match="norm_type"):
        T.clip_grads(g, 1.0, norm_type=1.0)
    with pytest.raises(RuntimeError, match="must not be negative"):
        T.clip_grads(g, -1.0)
    for bad in (math.nan, -math.inf):
        with pytest.raises(ValueError, match="max_norm"):
            T.clip_grads(g, bad)
    with pytest.raises(RuntimeError, match="one tensor for each"):
        T.clip_grads(g, 1.0, out=[])
    with pytest.raises(ValueError, match="one tensor for each"):
        T.clip_grads([], 1.0, out=g)
    with pytest.raises(RuntimeError, match="float16, bfloat16, float32 or float64"):
        T.global_norm([torch.zeros(3, dtype=torch.int32)])
    assert T.global_norm([]).item() == 0 and T.clip_grads([], 1.0) == ([], torch.tensor(0.0))


def test_structures_match_the_header():
    """The ctypes structures have the sizes the header's fields add up to on this ABI."""
    assert ctypes.sizeof(_ext.AttentionProblem) == 8 + 3 * 8 + 9 * 8 + 6 * 8 + 2 * 8 + 3 * 8
    assert ctypes.sizeof(_ext.RotateProblem) == 8 + 8 + 3 * 8 + 4 * 8 + 2 * 8 + 8 + 8 + 2 * 8 + 8 + 8 + 2 * 8 + 8
    assert ctypes.sizeof(_ext.TensorRef) == 32


def attention_problem(**change):
    p = _ext.AttentionProblem(dtype=0, lengths_int32=0, q=16, k=16, v=16, B=1, N=2, M=3, Hq=2, Hkv=1, d=8, bandwidth=-1,
                              scale=1.0, err_word=16)
    for name, value in change.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("change,status", [
    ({"dtype": 1}, EDTYPE), ({"dtype": 9}, EDTYPE), ({"d": 0}, EINVAL), ({"d": 129}, EINVAL), ({"Hq": 3, "Hkv": 2}, EINVAL),
    ({"Hkv": 0}, EINVAL), ({"N": -1}, EINVAL), ({"B": 1 << 40}, EINVAL), ({"q": None}, EINVAL), ({"v": None}, EINVAL),
    ({"scale": math.nan}, EINVAL), ({"err_word": None}, EINVAL), ({"N": 1 << 24, "B": 1 << 20}, EINVAL),
])
def test_c_attention_refuses(change, status):
    lib = _ext.capi()
    p = attention_problem(**change)
    assert lib.sdtw_cross_attention(ctypes.byref(p), 16, None, 16, None, 0, None) == status
    stride = (ctypes.c_int64 * 3)()
    assert lib.sdtw_cross_attention_backward(ctypes.byref(p), 16, None, 16, 16, stride, 16, 16, 16, None, 0, None) == status


def test_c_attention_refuses_missing_buffers():
    lib = _ext.capi()
    p = attention_problem()
    stride = (ctypes.c_int64 * 3)()
    assert lib.sdtw_cross_attention(None, 16, None, 16, None, 0, None) == EINVAL
    assert lib.sdtw_cross_attention(ctypes.byref(p), None, None, 16, None, 0, None) == EINVAL
    assert lib.sdtw_cross_attention_backward_workspace_bytes(ctypes.byref(p)) > 0
    assert lib.sdtw_cross_attention_backward(ctypes.byref(p), 16, None, 16, 16, stride, 16, 16, 16, None, 0, None) == EWORKSPACE
    assert lib.sdtw_cross_attention_backward(ctypes.byref(p), 16, None, 16, 16, None, 16, 16, 16, 16, 1 << 20, None) == EINVAL
    assert lib.sdtw_cross_attention(ctypes.byref(p), 24, None, 16, None, 0, None) == EINVAL  # outputs start on 16 bytes
    assert lib.sdtw_cross_attention(ctypes.byref(p), 16, 24, 16, None, 0, None) == EINVAL
    for bad in range(3):
        outs = [24 if n == bad else 16 for n in range(3)]
        assert lib.sdtw_cross_attention_backward(ctypes.byref(p), 16, None, 16, 16, stride, *outs, 16, 1 << 20, None) == EINVAL
    empty = attention_problem(B=0)
    assert lib.sdtw_cross_attention(ctypes.byref(empty), None, None, None, None, 0, None) == 0


@pytest.mark.parametrize("change,status", [
    ({"dtype": 1}, EDTYPE), ({"d": 0}, EINVAL), ({"d": 257}, EINVAL), ({"rotary": 3}, EINVAL), ({"rotary": 10}, EINVAL),
    ({"base": 0.0}, EINVAL), ({"eps": -1.0}, EINVAL), ({"position_kind": 3}, EINVAL), ({"x": None}, EINVAL), ({"err_word": None}, EINVAL),
])
def test_c_rotate_refuses(change, status):
    lib = _ext.capi()
    p = _ext.RotateProblem(dtype=0, x=16, B=1, N=2, H=1, d=8, rotary=8, base=1e4, eps=1e-6, err_word=16)
    for name, value in change.items():
        setattr(p, name, value)
    assert lib.sdtw_norm_rotate(ctypes.byref(p), 16, None) == status
    stride = (ctypes.c_int64 * 3)()
    assert lib.sdtw_norm_rotate_backward(ctypes.byref(p), 16, stride, 16, None, None, 0, None) == status


def test_c_clip_refuses():
    lib = _ext.capi()
    refs = (_ext.TensorRef * 1)(_ext.TensorRef(src=16, dst=16, numel=4, dtype=0))
    need = lib.sdtw_clip_workspace_bytes(1)
    assert lib.sdtw_clip_grads(refs, 1, 0, 1.0, 16, 0, None, 0, None) == EWORKSPACE
    assert lib.sdtw_clip_grads(refs, 1, 0, 1.0, 16, 0, 16, need - 1, None) == EWORKSPACE
    assert lib.sdtw_clip_grads(refs, 1, 2, 1.0, 16, 0, 16, need, None) == EINVAL
    assert lib.sdtw_clip_grads(refs, 1, 0, -1.0, 16, 0, 16, need, None) == EINVAL
    assert lib.sdtw_clip_grads(refs, 1, 0, 1.0, None, 0, 16, need, None) == EINVAL
    refs[0].dtype = 7
    assert lib.sdtw_global_norm(refs, 1, 0, 16, 0, 16, need, None) == EDTYPE
    refs[0].dtype, refs[0].src = 0, None
    assert lib.sdtw_global_norm(refs, 1, 0, 16, 0, 16, need, None) == EINVAL


def test_fake_kernels():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        q = torch.empty(2, 3, 4, 8, device="cuda", dtype=torch.bfloat16)
        k = torch.empty(2, 5, 2, 8, device="cuda", dtype=torch.bfloat16)
        out, lo, lse = torch.ops.torchsoftdtw_b200.attention(q, k, k, None, None, -1, 1.0)
        assert out.shape == q.shape and lo.shape == q.shape and lse.shape == (2, 4, 3) and lse.dtype == torch.float32
        f = q.float()
        assert torch.ops.torchsoftdtw_b200.attention(f, k.float(), k.float(), None, None, -1, 1.0)[1].numel() == 0
        assert T.cross_attention(q, k, k).shape == q.shape
        dq, dk, dv = torch.ops.torchsoftdtw_b200.attention_backward(out, q, k, k, out, lo, lse, None, None, -1, 1.0)
        assert dq.shape == q.shape and dk.shape == k.shape == dv.shape
        w = torch.empty(8, device="cuda")
        assert T.norm_rotate(q, w).shape == q.shape
        norm = torch.ops.torchsoftdtw_b200.global_norm([q, w.double()], 2.0)
        assert norm.dtype == torch.float64 and norm.dim() == 0


def test_forward_mode_is_refused():
    """A tangent would otherwise be dropped without a word."""
    import torch.autograd.forward_ad as fwad

    x = torch.randn(1, 2, 1, 8)
    with fwad.dual_level():
        d = fwad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            T.cross_attention(d, x, x)
        with pytest.raises(RuntimeError, match="forward-mode"):
            T.norm_rotate(d)
        with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
            T.norm_rotate(x, fwad.make_dual(torch.ones(8), torch.ones(8)))

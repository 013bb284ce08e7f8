"""CPU: what the training operators refuse (before anything reaches a device)."""
import ctypes as C

import pytest
import torch

import fish_diffusion_amd as fda
from fish_diffusion_amd import _lib


def qkv(B=1, H=4, Hkv=2, Tq=5, Tk=7, D=32, t=torch.float32):
    return torch.zeros(B, H, Tq, D, dtype=t), torch.zeros(B, Hkv, Tk, D, dtype=t), torch.zeros(B, Hkv, Tk, D, dtype=t)


def test_attention_needs_the_device():
    with pytest.raises(RuntimeError, match="MI355X"):
        fda.attention(*qkv())
    with pytest.raises(RuntimeError, match="MI355X"):
        fda.attention(*(x.requires_grad_() for x in qkv()))


@pytest.mark.parametrize("kw,exc", [
    (dict(q=torch.zeros(4, 5, 32)), ValueError), (dict(q=torch.zeros(1, 4, 5, 36)), ValueError), (dict(q=torch.zeros(2, 4, 5, 32)), ValueError),
    (dict(q=torch.zeros(1, 3, 5, 32)), ValueError), (dict(v=torch.zeros(1, 2, 8, 32)), ValueError), (dict(q=torch.zeros(1, 4, 5, 32).double()), TypeError),
    (dict(scale=0.0), ValueError), (dict(scale=-1.0), ValueError), (dict(scale=float("nan")), ValueError),
    (dict(key_mask=torch.zeros(1, 6, dtype=torch.bool)), ValueError), (dict(key_mask=torch.zeros(1, 7)), TypeError), (dict(k=None), ValueError)])
def test_attention_refusals(kw, exc):
    q, k, v = qkv()
    a = dict(q=q, k=k, v=v, **{})
    a.update(kw)
    with pytest.raises(exc):
        fda.attention_forward(**a)


def test_head_sizes_out_of_range():
    for D in (4, 12, 136, 256):
        with pytest.raises(ValueError, match="head size"):
            fda.attention_forward(*qkv(D=D))


def test_workspace_sizes_and_bad_descriptors(lib_built):
    lib, n = _lib.lib(), C.c_size_t()
    d = _lib.AttnDesc(1, 1, 32, 8, 1, 8192, 128, 0, 1.0)
    assert lib.fdx_attn_forward_workspace(C.byref(d), C.byref(n)) == 0 and n.value > 0          # one token: the keys are split
    assert lib.fdx_attn_backward_workspace(C.byref(d), C.byref(n)) == 0 and n.value > 0
    assert lib.fdx_attn_forward_workspace(C.byref(d), None) == -1
    for bad in (dict(dtype=3), dict(heads=0), dict(kv_heads=5), dict(head_dim=12), dict(head_dim=256), dict(q_len=-1), dict(scale=0.0),
                dict(scale=float("inf")), dict(heads=1 << 20, kv_heads=1, q_len=1 << 20)):
        d = _lib.AttnDesc(1, 1, 32, 8, 1, 8192, 128, 0, 1.0)
        for k, v in bad.items():
            setattr(d, k, v)
        assert lib.fdx_attn_forward_workspace(C.byref(d), C.byref(n)) == -1, bad
        assert lib.fdx_attn_backward_workspace(C.byref(d), C.byref(n)) == -1, bad
        assert lib.fdx_last_error(None)
    assert lib.fdx_attn_forward(None, C.byref(d), None, None, None, None, None, None, None, 0, None) == -1

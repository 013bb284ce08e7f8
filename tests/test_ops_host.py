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
                dict(scale=float("inf")), dict(heads=1 << 20, kv_heads=1, q_len=1 << 20),
                dict(batch=1 << 23, heads=1, kv_heads=1)):
        d = _lib.AttnDesc(1, 1, 32, 8, 1, 8192, 128, 0, 1.0)
        for k, v in bad.items():
            setattr(d, k, v)
        assert lib.fdx_attn_forward_workspace(C.byref(d), C.byref(n)) == -1, bad
        assert lib.fdx_attn_backward_workspace(C.byref(d), C.byref(n)) == -1, bad
        assert lib.fdx_last_error(None)
    assert lib.fdx_attn_forward(None, C.byref(d), None, None, None, None, None, None, None, 0, None) == -1


def test_norm_and_pack_need_the_device_and_refuse():
    x = torch.zeros(2, 5, 64)
    w = torch.ones(64)
    for call in (lambda: fda.residual_norm(x, x, pre_norm=(w, None)), lambda: fda.pack8(x), lambda: fda.gelu8(x), lambda: fda.linear8(x, torch.zeros(8, 64)),
                 lambda: fda.unpack8(fda.Packed8(torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2, 2, dtype=torch.uint8))),
                 lambda: fda.linear8_weight_grad(torch.zeros(2, 8), fda.Packed8(torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2, 2, dtype=torch.uint8)))):
        with pytest.raises(RuntimeError, match="MI355X"):
            call()


@pytest.mark.parametrize("kw", [
    dict(block=torch.zeros(2, 5, 32)), dict(pre_norm=(torch.ones(63), None)), dict(pre_norm=(torch.ones(64).half(), None)), dict(kind="group"),
    dict(pre_norm=(torch.ones(64), torch.ones(64).half())), dict(gate=torch.ones(5)), dict(gate=torch.ones(5, 64)), dict(gate=torch.ones(64).double()),
    dict(residual_scale=float("inf")), dict(eps=-1.0), dict(pre_norm=(None, torch.ones(64))), dict(need_h=False)])
def test_residual_norm_refusals(kw):
    a = dict(x=torch.zeros(2, 5, 64), block=torch.zeros(2, 5, 64))
    a.update(kw)
    with pytest.raises(ValueError):
        fda.residual_norm_forward(**a)


def test_other_refusals():
    with pytest.raises(ValueError):
        fda.residual_norm_forward(torch.zeros(2, 8200), torch.zeros(2, 8200))
    with pytest.raises(TypeError):
        fda.residual_norm_forward(torch.zeros(2, 8).double(), torch.zeros(2, 8).double())
    with pytest.raises(TypeError):
        fda.pack8(torch.zeros(2, 8).double())
    with pytest.raises(ValueError):
        fda.pack8(torch.zeros(()))
    with pytest.raises(ValueError):
        fda.linear8(torch.zeros(2, 8), torch.zeros(4, 9))


def test_c_entries_refuse_bad_sizes(lib_built):
    lib, n = _lib.lib(), C.c_size_t()
    good = dict(dtype=1, param_dtype=0, gate_dtype=1, rows=10, channels=64, gate_rows=5, rms=0, residual_scale=1.0, eps=1e-5)
    assert lib.fdx_resnorm_backward_workspace(C.byref(_lib.ResnormDesc(**good)), C.byref(n)) == 0 and n.value > 0
    for bad in (dict(dtype=5), dict(param_dtype=2), dict(channels=0), dict(channels=9000), dict(gate_rows=3), dict(rows=-1)):
        assert lib.fdx_resnorm_backward_workspace(C.byref(_lib.ResnormDesc(**{**good, **bad})), C.byref(n)) == -1, bad
    assert lib.fdx_linear8_weight_grad_workspace(1, 100, 16, 16, C.byref(n)) == 0
    assert n.value >= 4 * (16 * 16 + 16)
    for bad in ((3, 100, 16, 16), (1, -1, 16, 16), (1, 100, 0, 16), (1, 100, 16, 0)):
        assert lib.fdx_linear8_weight_grad_workspace(*bad, C.byref(n)) == -1, bad
    assert lib.fdx_pack8(None, 0, None, 1, 8, None, None, None) == -1


def test_training_forward_needs_the_device():
    net = fda.TransformerDecoderDenoiser(mel_channels=8, dim=128, mlp_factor=1, condition_dim=8, num_layers=1)
    with pytest.raises(RuntimeError, match="MI355X"):
        net.training_forward(torch.zeros(1, 8, 4), torch.zeros(1), torch.zeros(1, 8, 4))

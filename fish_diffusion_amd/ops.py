"""Operators for training on MI355X: what one decoder layer of `TransformerDecoderDenoiser` (nn.TransformerDecoderLayer under autograd in
fish_diffusion/modules/convnext.py:263-379) needs besides plain matrix products.

  attention / attention_forward / attention_backward
        softmax(scale q k^T) v with key masks, causal order and shared key / value heads; the backward pass recomputes the probabilities.

Each comes as a differentiable function and as the two calls it is made of (`*_forward`, `*_backward`); the latter build no autograd graph and
may be captured into a HIP graph as they are.  Device tensors only (fp32, bf16, fp16); work runs on the current stream of the tensors' device and
nothing is kept from one call for the next.  Every call gives the same bits for the same inputs.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import get_gradient_edge

from . import _lib

_EAGER = "fish_diffusion_amd.eager"


def _guard_capture(tensors):
    """Refuses to record an autograd graph during a capture while an eager graph of the same leaves is alive: the leaves' accumulation nodes then
    belong to the eager stream, and their part of a captured backward pass would run outside the capture, which ends the process.  Returns the
    leaves' nodes, to be held until the graph that is being built holds them."""
    if not torch.is_grad_enabled():
        return None
    tensors = [t for t in tensors if t.requires_grad and t.is_cuda]
    if not tensors:
        return None
    if not torch.cuda.is_current_stream_capturing():
        nodes = [get_gradient_edge(t).node for t in tensors if t.is_leaf]
        for n in nodes:
            n.metadata[_EAGER] = True
        return nodes
    todo, seen = [get_gradient_edge(t).node for t in tensors], set()
    while todo:
        n = todo.pop()
        if n in seen:
            continue
        seen.add(n)
        if n.metadata.get(_EAGER):
            raise RuntimeError("an autograd graph built outside this capture still holds the same leaf tensors: delete its outputs before the "
                               "capture, or capture the *_forward / *_backward calls, which build no graph")
        todo += [m for m, _ in n.next_functions if m is not None]
    return None


def _apply(fn, *args):
    held = _guard_capture([a for a in args if torch.is_tensor(a)])   # noqa: F841 (until apply() has linked them)
    return fn.apply(*args)


def _dtype(t: torch.Tensor, what: str) -> int:
    if t.dtype not in _lib.DTYPES:
        raise TypeError(f"{what}: {t.dtype} is not one of float32, bfloat16, float16")
    return _lib.DTYPES[t.dtype]


def _same(ref: torch.Tensor, what: str, **tensors):
    for name, t in tensors.items():
        if t is None:
            continue
        _lib.require_gpu(t, f"{what} {name}")
        if t.device != ref.device:
            raise ValueError(f"{what}: {name} is on {t.device}, expected {ref.device}")
        if t.dtype != ref.dtype:
            raise ValueError(f"{what}: {name} is {t.dtype}, expected {ref.dtype}")


def _handle(device: torch.device) -> _lib.Handle:
    with torch.cuda.device(device):   # creating a handle makes its device current
        return _lib.Handle.shared(device)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """The tensor itself where the kernels can read it in 16-byte pieces along its last dimension, else a contiguous copy."""
    es = t.element_size()
    if t.numel() == 0:
        return t
    ok = t.data_ptr() % 16 == 0 and (t.shape[-1] == 1 or t.stride(-1) == 1)
    ok = ok and all(n == 1 or s * es % 16 == 0 for n, s in zip(t.shape[:-1], t.stride()[:-1]))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _bht(t: Optional[torch.Tensor]):
    if t is None or t.numel() == 0:
        return _lib.Bht(None, 0, 0, 0)
    s = [0 if n == 1 else st for n, st in zip(t.shape[:3], t.stride()[:3])]
    return _lib.Bht(t.data_ptr(), *s)


def _workspace(fn, desc, device):
    n = C.c_size_t()
    _lib.check(fn(C.byref(desc), C.byref(n)))
    return (torch.empty(n.value, dtype=torch.uint8, device=device) if n.value else None), n.value


# ------------------------------------------------------------------------------------------------------------- attention
def _attn_desc(q, k, v, key_mask, causal, scale, what):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not torch.is_tensor(t) or t.dim() != 4:
            raise ValueError(f"{what}: {name} must be a [batch, heads, length, channels] tensor")
    dt = _dtype(q, what)
    B, H, Tq, D = q.shape
    Hkv, Tk = k.shape[1], k.shape[2]
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"{what}: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit together")
    if H == 0 or Hkv == 0 or H % Hkv:
        raise ValueError(f"{what}: {H} query heads cannot share {Hkv} key / value heads")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"{what}: head size {D} is not a multiple of 8 up to 128")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"{what}: scale must be positive and finite, got {scale}")
    if key_mask is not None:
        if key_mask.dtype not in (torch.bool, torch.uint8):
            raise TypeError(f"{what}: key_mask must be bool or uint8 (true = masked), got {key_mask.dtype}")
        if key_mask.shape != (B, Tk):
            raise ValueError(f"{what}: key_mask {tuple(key_mask.shape)} is not [batch, keys] = {(B, Tk)}")
        if key_mask.device != q.device:
            raise ValueError(f"{what}: key_mask is on {key_mask.device}, expected {q.device}")
        key_mask = key_mask.contiguous()
    _lib.require_gpu(q, f"{what} q")
    _same(q, what, k=k, v=v)
    return _lib.AttnDesc(dt, B, H, Hkv, Tq, Tk, D, int(bool(causal)), scale), key_mask


def _like_rows(t: torch.Tensor) -> torch.Tensor:
    """An uninitialised tensor of t's [B, H, T, D] shape that lies in memory as [B, T, H, D]: joining the heads afterwards is a view."""
    B, H, T, D = t.shape
    return torch.empty(B, T, H, D, dtype=t.dtype, device=t.device).transpose(1, 2)


@torch.no_grad()
def attention_forward(q, k, v, key_mask=None, causal=False, scale=None):
    """(out, lse): out [B, H, Tq, D] = softmax(scale q k^T) v, lse fp32 [B, H, Tq] = the natural logarithm of each row's sum of exponentials.

    q [B, H, Tq, D]; k, v [B, Hkv, Tk, D] with H a multiple of Hkv (query head h reads head h // (H // Hkv)); D a multiple of 8 up to 128.
    key_mask [B, Tk], true = masked (whatever masked keys and values hold, NaN included, is never used); causal: query i sees keys up to
    i + Tk - Tq; scale defaults to D ** -0.5.  A row that sees no key is 0 (lse -inf).  Any strides; channels that are not contiguous or not
    16-byte aligned are copied first."""
    desc, key_mask = _attn_desc(q, k, v, key_mask, causal, scale, "attention")
    q, k, v = _aligned(q), _aligned(k), _aligned(v)
    out = _like_rows(q)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
    h, lib = _handle(q.device), _lib.lib()
    ws, n = _workspace(lib.fdx_attn_forward_workspace, desc, q.device)
    with h.lock:
        _lib.check(lib.fdx_attn_forward(h.h, C.byref(desc), C.byref(_bht(q)), C.byref(_bht(k)), C.byref(_bht(v)), _lib.ptr(key_mask),
                                        C.byref(_bht(out)), _lib.ptr(lse), _lib.ptr(ws), n, _lib.stream_ptr(q.device)), h.h)
    return out, lse


@torch.no_grad()
def attention_backward(grad_out, q, k, v, out, lse, key_mask=None, causal=False, scale=None):
    """(dq, dk, dv) of `attention_forward` called with the same arguments, from grad_out and its results.  dk / dv are summed over the query
    heads that share a key / value head; masked keys get 0, rows that see no key give 0 whatever grad_out holds there."""
    desc, key_mask = _attn_desc(q, k, v, key_mask, causal, scale, "attention_backward")
    _same(q, "attention_backward", grad_out=grad_out, out=out)
    if grad_out.shape != q.shape or out.shape != q.shape:
        raise ValueError(f"attention_backward: grad_out {tuple(grad_out.shape)} and out {tuple(out.shape)} must have q's shape {tuple(q.shape)}")
    if lse.shape != q.shape[:3] or lse.dtype != torch.float32 or lse.device != q.device:
        raise ValueError(f"attention_backward: lse must be the forward's float32 {tuple(q.shape[:3])} on {q.device}")
    grad_out, q, k, v, out = (_aligned(t) for t in (grad_out, q, k, v, out))
    lse = lse.contiguous()
    dq, dk, dv = _like_rows(q), _like_rows(k), _like_rows(v)
    h, lib = _handle(q.device), _lib.lib()
    ws, n = _workspace(lib.fdx_attn_backward_workspace, desc, q.device)
    with h.lock:
        _lib.check(lib.fdx_attn_backward(h.h, C.byref(desc), *(C.byref(_bht(t)) for t in (grad_out, q, k, v, out)), _lib.ptr(lse),
                                         _lib.ptr(key_mask), *(C.byref(_bht(t)) for t in (dq, dk, dv)), _lib.ptr(ws), n,
                                         _lib.stream_ptr(q.device)), h.h)
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, key_mask, causal, scale):
        out, lse = attention_forward(q, k, v, key_mask, causal, scale)
        ctx.save_for_backward(q, k, v, out, lse, key_mask)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        q, k, v, out, lse, key_mask = ctx.saved_tensors
        return (*attention_backward(grad_out, q, k, v, out, lse, key_mask, ctx.causal, ctx.scale), None, None, None)


def attention(q, k, v, key_mask=None, causal=False, scale=None):
    """Differentiable `attention_forward`: returns out alone."""
    return _apply(_Attention, q, k, v, key_mask, causal, scale)

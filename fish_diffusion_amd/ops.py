"""Operators for training on MI355X: what one decoder layer of `TransformerDecoderDenoiser` (nn.TransformerDecoderLayer under autograd in
fish_diffusion/modules/convnext.py:263-379) needs besides plain matrix products.

  attention / attention_forward / attention_backward
        softmax(scale q k^T) v with key masks, causal order and shared key / value heads; the backward pass recomputes the probabilities.
  residual_norm / residual_norm_forward / residual_norm_backward
        h = a x + gate * post_norm(block), y = pre_norm(h): the step between two blocks, one launch each way.
  linear8, gelu8 (pack8, unpack8, linear8_weight_grad, gelu8_forward, gelu8_backward)
        a linear layer and a GELU that keep their input in 8 bits; the gradients are taken straight from the 8-bit form.

Each comes as a differentiable function and as the two calls it is made of (`*_forward`, `*_backward`); the latter build no autograd graph and
may be captured into a HIP graph as they are.  Device tensors only (fp32, bf16, fp16); work runs on the current stream of the tensors' device and
nothing is kept from one call for the next.  Every call gives the same bits for the same inputs.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
from typing import NamedTuple, Optional

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
    dt = _lib.DTYPES.get(t.dtype)
    if dt is None:
        raise TypeError(f"{what}: {t.dtype} is not one of float32, bfloat16, float16")
    return dt


def _same(ref: torch.Tensor, what: str, **tensors):
    device, dtype = ref.device, ref.dtype
    for name, t in tensors.items():
        if t is None:
            continue
        if t.device != device:
            _lib.require_gpu(t, f"{what} {name}")
            raise ValueError(f"{what}: {name} is on {t.device}, expected {device}")
        if t.dtype != dtype:
            raise ValueError(f"{what}: {name} is {t.dtype}, expected {dtype}")


_handles = {}


def _handle(device: torch.device) -> _lib.Handle:
    h = _handles.get(device.index)
    if h is None:
        with torch.cuda.device(device):   # creating a handle makes its device current
            h = _handles[device.index] = _lib.Handle.shared(device)
    return h


def _stream(h: _lib.Handle):
    return torch._C._cuda_getCurrentRawStream(h.device.index)   # torch.cuda.current_stream(device).cuda_stream without its objects: 2 us less a call


def _copy(t: torch.Tensor) -> torch.Tensor:
    return t.detach().clone(memory_format=torch.contiguous_format)


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _arg(t: torch.Tensor, vec: int):
    """(tensor, its description for the C call); a contiguous copy where the kernels cannot read it in 16-byte pieces of `vec` elements."""
    at, (b, h, n, _), (sb, sh, sn, sd) = t.data_ptr(), t.shape, t.stride()
    sb, sh, sn = (sb if b > 1 else 0), (sh if h > 1 else 0), (sn if n > 1 else 0)
    if (at & 15 or sd != 1 or (sb | sh | sn) & (vec - 1)) and t.numel():
        return _arg(_copy(t), vec)
    return t, _lib.Bht(at or None, sb, sh, sn)


def _workspace_bytes(fn, *args) -> int:
    n = C.c_size_t()
    _lib.check(fn(*args, C.byref(n)))
    return n.value


def _workspace(n: int, like):
    return like.new_empty((n,), dtype=torch.uint8) if n else None   # (new_empty: 1 us a call less than torch.empty with a device)


# ------------------------------------------------------------------------------------------------------------- attention
@functools.lru_cache(maxsize=1024)
def _attn_plan(dtype, qs, ks, vs, causal, scale):
    """What a call of these types and sizes needs (sizes only, no tensors): its C description, elements per 16 bytes, bytes of workspace each way, lse's
    shape, and the strides of out / dq and of dk / dv -- [B, H, T, D] that lies in memory as [B, T, H, D]: joining the heads afterwards is a view."""
    if len(qs) != 4 or len(ks) != 4 or len(vs) != 4:
        raise ValueError("attention: q, k and v must be [batch, heads, length, channels] tensors")
    dt = _lib.DTYPES.get(dtype)
    if dt is None:
        raise TypeError(f"attention: {dtype} is not one of float32, bfloat16, float16")
    (B, H, Tq, D), (Hkv, Tk) = qs, ks[1:3]
    if ks != vs or ks[0] != B or ks[3] != D:
        raise ValueError(f"attention: q {tuple(qs)}, k {tuple(ks)} and v {tuple(vs)} do not fit together")
    if H == 0 or Hkv == 0 or H % Hkv:
        raise ValueError(f"attention: {H} query heads cannot share {Hkv} key / value heads")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"attention: head size {D} is not a multiple of 8 up to 128")
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"attention: scale must be positive and finite, got {scale}")
    desc = _lib.AttnDesc(dt, B, H, Hkv, Tq, Tk, D, int(causal), scale)
    lib = _lib.lib()
    return (desc, 4 if dt == 0 else 8, _workspace_bytes(lib.fdx_attn_forward_workspace, desc), _workspace_bytes(lib.fdx_attn_backward_workspace, desc),
            (B, H, Tq), (Tq * H * D, D, H * D, 1), (Tk * Hkv * D, D, Hkv * D, 1))


def _attn_check(q, k, v, key_mask, causal, scale):
    for t in (q, k, v):
        if not isinstance(t, torch.Tensor):
            raise ValueError("attention: q, k and v must be [batch, heads, length, channels] tensors")
    plan = _attn_plan(q.dtype, q.shape, k.shape, v.shape, bool(causal), None if scale is None else float(scale))
    dev = q.get_device()
    if key_mask is not None:
        if key_mask.dtype not in (torch.bool, torch.uint8):
            raise TypeError(f"attention: key_mask must be bool or uint8 (true = masked), got {key_mask.dtype}")
        if key_mask.shape != (q.shape[0], k.shape[2]):
            raise ValueError(f"attention: key_mask {tuple(key_mask.shape)} is not [batch, keys] = {(q.shape[0], k.shape[2])}")
        if key_mask.get_device() != dev:
            raise ValueError(f"attention: key_mask is on {key_mask.device}, expected {q.device}")
        key_mask = key_mask.contiguous()
    if dev < 0:
        _lib.require_gpu(q, "attention q")
    if k.get_device() != dev or v.get_device() != dev or k.dtype is not q.dtype or v.dtype is not q.dtype:
        _same(q, "attention", k=k, v=v)
    return plan, key_mask


def _new_rows(t: torch.Tensor, strides):
    """An uninitialised tensor of t's shape and its description."""
    new = t.new_empty_strided(t.shape, strides)
    return new, _lib.Bht(new.data_ptr() or None, *strides[:3])


def attention_forward(q, k, v, key_mask=None, causal=False, scale=None):
    """(out, lse): out [B, H, Tq, D] = softmax(scale q k^T) v, lse fp32 [B, H, Tq] = the natural logarithm of each row's sum of exponentials.

    q [B, H, Tq, D]; k, v [B, Hkv, Tk, D] with H a multiple of Hkv (query head h reads head h // (H // Hkv)); D a multiple of 8 up to 128.
    key_mask [B, Tk], true = masked (whatever masked keys and values hold, NaN included, is never used); causal: query i sees keys up to
    i + Tk - Tq; scale defaults to D ** -0.5.  A row that sees no key is 0 (lse -inf).  Any strides; channels that are not contiguous or not
    16-byte aligned are copied first.  No autograd graph (`attention` builds one)."""
    (desc, vec, n, _, lse_shape, rows, _), key_mask = _attn_check(q, k, v, key_mask, causal, scale)
    (q, aq), (k, ak), (v, av) = _arg(q, vec), _arg(k, vec), _arg(v, vec)
    out, ao = _new_rows(q, rows)
    lse = q.new_empty(lse_shape, dtype=torch.float32)
    h, ws = _handle(q.device), _workspace(n, q)
    with h.lock:
        rc = _lib.lib().fdx_attn_forward(h.h, desc, aq, ak, av, _p(key_mask), ao, lse.data_ptr(), _p(ws), n, _stream(h))
        if rc:
            _lib.check(rc, h.h)
    return out, lse


def attention_backward(grad_out, q, k, v, out, lse, key_mask=None, causal=False, scale=None):
    """(dq, dk, dv) of `attention_forward` called with the same arguments, from grad_out and its results.  dk / dv are summed over the query
    heads that share a key / value head; masked keys get 0, rows that see no key give 0 whatever grad_out holds there."""
    (desc, vec, _, n, lse_shape, rows, keys), key_mask = _attn_check(q, k, v, key_mask, causal, scale)
    dev, dtype = q.get_device(), q.dtype
    if grad_out.get_device() != dev or out.get_device() != dev or grad_out.dtype is not dtype or out.dtype is not dtype:
        _same(q, "attention_backward", grad_out=grad_out, out=out)
    if grad_out.shape != q.shape or out.shape != q.shape:
        raise ValueError(f"attention_backward: grad_out {tuple(grad_out.shape)} and out {tuple(out.shape)} must have q's shape {tuple(q.shape)}")
    if lse.shape != lse_shape or lse.dtype is not torch.float32 or lse.get_device() != dev:
        raise ValueError(f"attention_backward: lse must be the forward's float32 {lse_shape} on {q.device}")
    (grad_out, ag), (q, aq), (k, ak), (v, av), (out, ao) = (_arg(t, vec) for t in (grad_out, q, k, v, out))
    lse = lse.contiguous()
    (dq, adq), (dk, adk), (dv, adv) = _new_rows(q, rows), _new_rows(k, keys), _new_rows(v, keys)
    h, ws = _handle(q.device), _workspace(n, q)
    with h.lock:
        rc = _lib.lib().fdx_attn_backward(h.h, desc, ag, aq, ak, av, ao, lse.data_ptr(), _p(key_mask), adq, adk, adv, _p(ws), n, _stream(h))
        if rc:
            _lib.check(rc, h.h)
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


# ------------------------------------------------------------------------------------------------------------- norm, gate, residual
class ResidualNormGrads(NamedTuple):
    """Gradients of `residual_norm_forward`'s arguments; None where the argument was None."""
    dx: torch.Tensor
    dblock: torch.Tensor
    dgate: Optional[torch.Tensor]
    dpost_weight: Optional[torch.Tensor]
    dpost_bias: Optional[torch.Tensor]
    dpre_weight: Optional[torch.Tensor]
    dpre_bias: Optional[torch.Tensor]


_KINDS = {"layer": 0, "rms": 1}
_NO_NORM = (None, None)


def _packed_rows(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """Contiguous and 16-byte aligned (a copy where it is not)."""
    if t is None or (t.is_contiguous() and not t.data_ptr() & 15):
        return t
    return _copy(t)


@functools.lru_cache(maxsize=1024)
def _norm_plan(dtype, shape, params, gate_dtype, gate_shape, residual_scale, kind, eps):   # params: (type, shape) or None each
    """The C description of a call of these types and sizes, and its backward pass's bytes of workspace."""
    dt = _lib.DTYPES.get(dtype)
    if dt is None:
        raise TypeError(f"residual_norm: {dtype} is not one of float32, bfloat16, float16")
    if len(shape) < 1 or not 1 <= shape[-1] <= 8192:
        raise ValueError(f"residual_norm: {tuple(shape)} does not end in 1 ... 8192 channels")
    C_, N = shape[-1], math.prod(shape[:-1])
    if kind not in _KINDS:
        raise ValueError(f"residual_norm: kind must be 'layer' or 'rms', got {kind!r}")
    if not (math.isfinite(residual_scale) and eps >= 0.0 and math.isfinite(eps)):
        raise ValueError("residual_norm: residual_scale must be finite and eps finite and not negative")
    pdt = set(p[0] for p in params if p is not None) or {dtype}
    if len(pdt) > 1 or not pdt <= {dtype, torch.float32}:
        raise ValueError(f"residual_norm: the norms' weights and biases must all be {dtype} or all float32, got {sorted(map(str, pdt))}")
    for p in params:
        if p is not None and p[1] != (C_,):
            raise ValueError(f"residual_norm: a norm's weight / bias has shape {tuple(p[1])}, expected {(C_,)}")
    rows = 0
    if gate_shape is not None:
        if gate_dtype not in (dtype, torch.float32):
            raise ValueError(f"residual_norm: gate must be {dtype} or float32, got {gate_dtype}")
        if gate_shape == shape and len(shape) > 1:
            rows = 1
        elif gate_shape == (C_,):
            rows = max(N, 1)
        elif len(shape) == 3 and tuple(gate_shape) in ((shape[0], C_), (shape[0], 1, C_)):
            rows = max(shape[1], 1)
        else:
            raise ValueError(f"residual_norm: gate {tuple(gate_shape)} is none of [channels], [batch, channels], [batch, 1, channels] and x's {tuple(shape)}")
    desc = _lib.ResnormDesc(dt, _lib.DTYPES[next(iter(pdt))], dt if gate_shape is None else _lib.DTYPES[gate_dtype], N, C_, rows, _KINDS[kind],
                            residual_scale, eps)
    return desc, _workspace_bytes(_lib.lib().fdx_resnorm_backward_workspace, desc)


def _norm_args(x, block, gate, residual_scale, post_norm, pre_norm, kind, eps):
    if not isinstance(x, torch.Tensor) or not isinstance(block, torch.Tensor) or x.shape != block.shape:
        raise ValueError("residual_norm: x and block must be tensors of one shape [..., channels]")
    pw, pb = post_norm or _NO_NORM
    nw, nb = pre_norm or _NO_NORM
    if (post_norm and pw is None) or (pre_norm and nw is None):
        raise ValueError("residual_norm: post_norm and pre_norm must be None or (weight, bias or None)")
    params = (pw, pb, nw, nb)
    plan = _norm_plan(x.dtype, x.shape, tuple([p if p is None else (p.dtype, p.shape) for p in params]), None if gate is None else gate.dtype,
                      None if gate is None else gate.shape, float(residual_scale), kind, float(eps))
    if block.dtype is not x.dtype:
        raise ValueError(f"residual_norm: block is {block.dtype}, x {x.dtype}")
    dev = x.get_device()
    if [True for t in (block, gate, *params) if t is not None and t.get_device() != dev]:
        raise ValueError("residual_norm: tensors on different devices")
    if dev < 0:
        _lib.require_gpu(x, "residual_norm x")
    return plan, [p if p is None else _packed_rows(p) for p in params]


def residual_norm_forward(x, block, gate=None, residual_scale=1.0, post_norm=None, pre_norm=None, kind="layer", eps=1e-5, need_h=True):
    """(h, y, stats): h = residual_scale * x + gate * post_norm(block), y = pre_norm(h) (None without one), stats for the backward pass.

    x, block [..., C], C up to 8192; post_norm / pre_norm = (weight, bias or None) of a LayerNorm (kind "layer") or RMSNorm ("rms") over the last
    dimension, or None; gate None, [C], x's own shape, or for x [B, T, C] one row per item: [B, C] or [B, 1, C].  Weights, biases and gate may be fp32
    beside 16-bit x.  y is computed from h before h is rounded.  A post-norm block's x = norm(x + block) is pre_norm alone with need_h=False: h is None and not
    written."""
    if not need_h and pre_norm is None:
        raise ValueError("residual_norm: need_h=False without a pre_norm leaves no result")
    (desc, _), (pw, pb, nw, nb) = _norm_args(x, block, gate, residual_scale, post_norm, pre_norm, kind, eps)
    x, block, gate = _packed_rows(x), _packed_rows(block), _packed_rows(gate)
    h_out = torch.empty_like(x) if need_h else None
    y = torch.empty_like(x) if nw is not None else None
    stats = x.new_empty((*x.shape[:-1], 4), dtype=torch.float32)
    if x.numel():
        h = _handle(x.device)
        with h.lock:
            rc = _lib.lib().fdx_resnorm_forward(h.h, desc, x.data_ptr(), block.data_ptr(), _p(gate), _p(pw), _p(pb), _p(nw), _p(nb), _p(h_out), _p(y),
                                                stats.data_ptr(), _stream(h))
            if rc:
                _lib.check(rc, h.h)
    return h_out, y, stats


def residual_norm_backward(grad_h, grad_y, x, block, stats, gate=None, residual_scale=1.0, post_norm=None, pre_norm=None, kind="layer", eps=1e-5):
    """`ResidualNormGrads` from the gradients of h and y (either may be None) and the forward's arguments and stats.  Where there is no gate, no post norm and
    residual_scale is 1, dx and dblock are equal and are ONE tensor.  The gate's gradient has the gate's shape."""
    (desc, n), (pw, pb, nw, nb) = _norm_args(x, block, gate, residual_scale, post_norm, pre_norm, kind, eps)
    for name, g in (("grad_h", grad_h), ("grad_y", grad_y)):
        if g is not None and (g.shape != x.shape or g.dtype is not x.dtype or g.get_device() != x.get_device()):
            raise ValueError(f"residual_norm_backward: {name} must be {x.dtype} {tuple(x.shape)} on {x.device}")
    if grad_y is not None and nw is None:
        raise ValueError("residual_norm_backward: grad_y without a pre_norm")
    if stats.shape != (*x.shape[:-1], 4) or stats.dtype != torch.float32 or stats.device != x.device:
        raise ValueError("residual_norm_backward: stats are not the forward's")
    x, block, gate_c, grad_h, grad_y, stats = (_packed_rows(t) for t in (x, block, gate, grad_h, grad_y, stats))
    dx = torch.empty_like(x)
    dblock = dx if gate is None and pw is None and residual_scale == 1.0 else torch.empty_like(x)
    dgate = None if gate is None else torch.empty_like(gate_c)
    grads = [None if p is None else torch.empty_like(p) for p in (pw, pb, nw, nb)]
    if x.numel() == 0:
        for t in (dgate, *grads):
            if t is not None:
                t.zero_()
    else:
        h, ws = _handle(x.device), _workspace(n, x)
        with h.lock:
            rc = _lib.lib().fdx_resnorm_backward(h.h, desc, *[_p(t) for t in (grad_h, grad_y, x, block, gate_c, pw, pb, nw, nb, stats, dx, dblock, dgate, *grads)],
                                                 _p(ws), n, _stream(h))
            if rc:
                _lib.check(rc, h.h)
    return ResidualNormGrads(dx, dblock, dgate, *grads)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, block, gate, post_w, post_b, pre_w, pre_b, residual_scale, kind, eps, need_h):
        post, pre = (None if w is None else (w, b) for w, b in ((post_w, post_b), (pre_w, pre_b)))
        h, y, stats = residual_norm_forward(x, block, gate, residual_scale, post, pre, kind, eps, need_h)
        ctx.save_for_backward(x, block, gate, post_w, post_b, pre_w, pre_b, stats)
        ctx.rest = (residual_scale, kind, eps)
        ctx.set_materialize_grads(False)
        return h, y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_h, grad_y):
        x, block, gate, post_w, post_b, pre_w, pre_b, stats = ctx.saved_tensors
        residual_scale, kind, eps = ctx.rest
        post, pre = (None if w is None else (w, b) for w, b in ((post_w, post_b), (pre_w, pre_b)))
        return (*residual_norm_backward(grad_h, grad_y, x, block, stats, gate, residual_scale, post, pre, kind, eps), None, None, None, None)


def residual_norm(x, block, gate=None, residual_scale=1.0, post_norm=None, pre_norm=None, kind="layer", eps=1e-5, need_h=True):
    """Differentiable `residual_norm_forward`: returns (h, y)."""
    return _apply(_ResidualNorm, x, block, gate, *(post_norm or (None, None)), *(pre_norm or (None, None)), residual_scale, kind, eps, need_h)


# ------------------------------------------------------------------------------------------------------------- activations in 8 bits
class Packed8(NamedTuple):
    """A tensor [..., C] in 8 bits: codes int8 [..., C] and exponents uint8 [..., ceil(C / 32)]; a group of 32 channels shares 2 ** (exponent - 127)."""
    codes: torch.Tensor
    exponents: torch.Tensor


def _rows_of(t: torch.Tensor, what: str, name: str):
    if not torch.is_tensor(t) or t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{what}: {name} must be a [..., channels] tensor")
    return t.numel() // t.shape[-1], t.shape[-1]


def _packed_ok(p: Packed8, what: str) -> Packed8:
    codes, exps = p
    if not torch.is_tensor(codes) or codes.dtype != torch.int8 or exps.dtype != torch.uint8 or codes.dim() < 1 or codes.shape[-1] < 1:
        raise ValueError(f"{what}: not a Packed8 of int8 codes and uint8 exponents")
    if exps.shape != (*codes.shape[:-1], (codes.shape[-1] + 31) // 32):
        raise ValueError(f"{what}: exponents {tuple(exps.shape)} do not belong to codes {tuple(codes.shape)}")
    _lib.require_gpu(codes, f"{what} codes")
    if exps.device != codes.device:
        raise ValueError(f"{what}: codes on {codes.device}, exponents on {exps.device}")
    return Packed8(_packed_rows(codes), exps.contiguous())


def _new_packed(x: torch.Tensor) -> Packed8:
    return Packed8(torch.empty_like(x, dtype=torch.int8), x.new_empty((*x.shape[:-1], (x.shape[-1] + 31) // 32), dtype=torch.uint8))


def pack8(x) -> Packed8:
    """x [..., C] in 8 bits.  Each group of 32 channels shares the smallest power of two 2^k, k >= -126, with max|x| <= 127 * 2^k; codes are x / 2^k rounded to
    nearest even, so the error is at most half of 2^k (at the very top of fp32's range, k = 122, codes end at 63 so that no finite value reads back
    infinite).  A group with an infinity or NaN reads back as NaN."""
    N, C_ = _rows_of(x, "pack8", "x")
    dt = _dtype(x, "pack8")
    if not x.is_cuda:
        _lib.require_gpu(x, "pack8 x")
    x = _packed_rows(x)
    p = _new_packed(x)
    h = _handle(x.device)
    with h.lock:
        rc = _lib.lib().fdx_pack8(h.h, dt, x.data_ptr(), N, C_, p.codes.data_ptr(), p.exponents.data_ptr(), _stream(h))
        if rc:
            _lib.check(rc, h.h)
    return p


def unpack8(packed: Packed8, dtype=torch.float32) -> torch.Tensor:
    """What the codes stand for (exact in float32 and bfloat16; in float16 at most 65504)."""
    p = _packed_ok(packed, "unpack8")
    if dtype not in _lib.DTYPES:
        raise TypeError(f"unpack8: {dtype} is not one of float32, bfloat16, float16")
    out = p.codes.new_empty(p.codes.shape, dtype=dtype)
    h = _handle(out.device)
    with h.lock:
        _lib.check(_lib.lib().fdx_unpack8(h.h, _lib.DTYPES[dtype], _p(p.codes), _p(p.exponents), *_rows_of(p.codes, "unpack8", "codes"), _p(out),
                                          _stream(h)), h.h)
    return out


@functools.lru_cache(maxsize=1024)
def _weight_grad_bytes(dt, N, O, I) -> int:
    return _workspace_bytes(_lib.lib().fdx_linear8_weight_grad_workspace, dt, N, O, I)


def linear8_weight_grad(dy, packed: Packed8, bias=True, dtype=None):
    """(dw, db) of y = x w^T + b from dy [..., out] and x kept as `pack8(x)` [..., in]: dw [out, in] = sum over rows of dy x8, db [out] = sum of dy (None if not
    `bias`).  Products are exact and summed in fp32; results in `dtype` (default dy's)."""
    N, O = _rows_of(dy, "linear8_weight_grad", "dy")
    dt = _dtype(dy, "linear8_weight_grad")
    dtype = dy.dtype if dtype is None else dtype
    if dtype not in _lib.DTYPES:
        raise TypeError(f"linear8_weight_grad: {dtype} is not one of float32, bfloat16, float16")
    if packed.codes.shape[:-1] != dy.shape[:-1]:
        raise ValueError(f"linear8_weight_grad: dy {tuple(dy.shape)} and the packed input {tuple(packed.codes.shape)} have different rows")
    _lib.require_gpu(dy, "linear8_weight_grad dy")
    p = _packed_ok(packed, "linear8_weight_grad")
    if p.codes.device != dy.device:
        raise ValueError(f"linear8_weight_grad: dy on {dy.device}, packed input on {p.codes.device}")
    I = p.codes.shape[-1]
    dy = _packed_rows(dy)
    dw = dy.new_empty((O, I), dtype=dtype)
    db = dy.new_empty((O,), dtype=dtype) if bias else None
    h, lib = _handle(dy.device), _lib.lib()
    n = _weight_grad_bytes(dt, N, O, I)
    ws = _workspace(n, dy)
    with h.lock:
        _lib.check(lib.fdx_linear8_weight_grad(h.h, dt, _p(dy), _p(p.codes), _p(p.exponents), N, O, I, _lib.DTYPES[dtype], _p(dw),
                                               _p(db), _p(ws), n, _stream(h)), h.h)
    return dw, db


def gelu8_forward(x):
    """(gelu(x), pack8(x)) in one pass; GELU in its erf form, from x itself."""
    N, C_ = _rows_of(x, "gelu8", "x")
    dt = _dtype(x, "gelu8")
    _lib.require_gpu(x, "gelu8 x")
    x = _packed_rows(x)
    y, p = torch.empty_like(x), _new_packed(x)
    h = _handle(x.device)
    with h.lock:
        _lib.check(_lib.lib().fdx_gelu8_forward(h.h, dt, _p(x), N, C_, _p(y), _p(p.codes), _p(p.exponents), _stream(h)), h.h)
    return y, p


def gelu8_backward(dy, packed: Packed8):
    """dy * gelu'(x8), x8 what `packed` stands for."""
    N, C_ = _rows_of(dy, "gelu8_backward", "dy")
    dt = _dtype(dy, "gelu8_backward")
    if packed.codes.shape != dy.shape:
        raise ValueError(f"gelu8_backward: dy {tuple(dy.shape)} and the packed input {tuple(packed.codes.shape)} differ")
    _lib.require_gpu(dy, "gelu8_backward dy")
    p = _packed_ok(packed, "gelu8_backward")
    if p.codes.device != dy.device:
        raise ValueError(f"gelu8_backward: dy on {dy.device}, packed input on {p.codes.device}")
    dy = _packed_rows(dy)
    dx = torch.empty_like(dy)
    h = _handle(dy.device)
    with h.lock:
        _lib.check(_lib.lib().fdx_gelu8_backward(h.h, dt, _p(dy), _p(p.codes), _p(p.exponents), N, C_, _p(dx), _stream(h)), h.h)
    return dx


class _Linear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        ctx.save_for_backward(*pack8(x), weight)
        ctx.has_bias = bias is not None
        with torch.autocast(x.device.type, enabled=False):   # the result has x's type, as the gradient that comes back
            return torch.nn.functional.linear(x, weight, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        codes, exps, weight = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad
        with torch.autocast(dy.device.type, enabled=False):
            dx = torch.matmul(dy, weight) if need_x else None
        dw, db = linear8_weight_grad(dy, Packed8(codes, exps), ctx.has_bias) if need_w or need_b else (None, None)
        return dx, dw, db


def linear8(x, weight, bias=None):
    """Differentiable x weight^T + bias that keeps x in 8 bits for the weight's gradient (x, weight and bias of one type); the result itself and x's gradient
    are those of torch.nn.functional.linear."""
    N, I = _rows_of(x, "linear8", "x")
    _dtype(x, "linear8")
    if weight.dim() != 2 or weight.shape[1] != I or (bias is not None and bias.shape != weight.shape[:1]):
        raise ValueError(f"linear8: x {tuple(x.shape)}, weight {tuple(weight.shape)} and bias do not fit together")
    _lib.require_gpu(x, "linear8 x")
    _same(x, "linear8", weight=weight, bias=bias)
    return _apply(_Linear8, x, weight, bias)


class _Gelu8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        y, p = gelu8_forward(x)
        ctx.save_for_backward(*p)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return gelu8_backward(dy, Packed8(*ctx.saved_tensors))


def gelu8(x):
    """Differentiable GELU (erf form) that keeps its input in 8 bits for the backward pass."""
    return _apply(_Gelu8, x)

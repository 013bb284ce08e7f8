"""`TransformerDecoderDenoiser` on MI355X: same constructor, call signature and state-dict keys as
fish_diffusion/modules/convnext.py:263-379 (12 x nn.TransformerDecoderLayer between 1x1-conv projections), computed by
libfishdx.so (csrc/tfdec.hip: convgemm GEMMs + an fp32 MFMA flash-attention kernel + LayerNorm).

`forward` is the inference path (no graph); `training_forward` is the same function under autograd, for fine-tuning: plain matrix products from
torch, everything between them -- attention, the residual + norm steps, GELU and the activations kept for the backward pass -- from `ops.py`.

Host plumbing only; there is no PyTorch fallback path.  The conditioner must have as many frames as the mel (how
`GaussianDiffusion` calls every denoiser, diffusion.py:217); at most 4096 frames (the positional table, convnext.py:317).
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F
from torch import nn

from . import _lib, ops
from .registry import DENOISERS
from .wavenet import HipDenoiser, _attach

N_POSITIONS = 4096


def positional_embedding(dim: int, n: int = N_POSITIONS) -> torch.Tensor:
    """convnext.py:317-329 (a registered buffer: checkpoints carry their own copy)."""
    half = dim // 2
    emb = math.log(10000) / (half - 1)
    emb = torch.exp(torch.arange(half, dtype=torch.float) * -emb)
    emb = torch.arange(n, dtype=torch.float).unsqueeze(1) * emb.unsqueeze(0)
    return torch.cat([torch.sin(emb), torch.cos(emb)], dim=1).view(n, -1)


def param_table(mel_channels, dim, mlp_factor, condition_dim, num_layers):
    """(state-dict key, shape, init) in state_dict order = the order fdx_tfdec_pack expects.  init: fan-in for the default
    nn.Conv1d / nn.Linear bound, 'xavier' (MultiheadAttention.in_proj_weight), 'zero', 'one', 'pos' (the buffer)."""
    h = dim * mlp_factor
    rows = [("position_scale_query", (1,), "one"), ("position_scale_key", (1,), "one"), ("positional_embedding", (N_POSITIONS, dim), "pos")]

    def wb(prefix, out_c, in_c, conv, bias_init=None):
        rows.append((prefix + ".weight", (out_c, in_c, 1) if conv else (out_c, in_c), in_c))
        rows.append((prefix + ".bias", (out_c,), bias_init if bias_init is not None else in_c))

    wb("input_projection.0", h, mel_channels, True)
    wb("input_projection.2", dim, h, True)
    wb("diffusion_embedding.1", h, dim, False)
    wb("diffusion_embedding.3", dim, h, False)
    wb("condition_projection.0", h, condition_dim, True)
    wb("condition_projection.2", dim, h, True)
    for i in range(num_layers):
        p = f"layers.{i}."
        for att in ("self_attn", "multihead_attn"):
            rows.append((p + att + ".in_proj_weight", (3 * dim, dim), "xavier"))
            rows.append((p + att + ".in_proj_bias", (3 * dim,), "zero"))
            wb(p + att + ".out_proj", dim, dim, False, bias_init="zero")
        wb(p + "linear1", h, dim, False)
        wb(p + "linear2", dim, h, False)
        for nrm in ("norm1", "norm2", "norm3"):
            rows.append((p + nrm + ".weight", (dim,), "one"))
            rows.append((p + nrm + ".bias", (dim,), "zero"))
    wb("output_projection.0", dim, dim, True)
    wb("output_projection.2", mel_channels, dim, True)
    return rows


class TransformerDecoderDenoiser(HipDenoiser):
    """Drop-in for the reference class of the same name (DENOISERS "TransformerDecoderDenoiser")."""

    _KIND = "tfdec"

    def __init__(self, mel_channels=128, dim=512, mlp_factor=4, condition_dim=256, num_layers=12, gradient_checkpointing=False):
        super().__init__()
        self.mel_channels, self.dim, self.mlp_factor = mel_channels, dim, mlp_factor
        self.condition_dim, self.n_layers = condition_dim, num_layers
        self.gradient_checkpointing = gradient_checkpointing   # inference: unused
        self._keys = []
        for key, shape, init in param_table(mel_channels, dim, mlp_factor, condition_dim, num_layers):
            if init == "pos":
                self.register_buffer(key, positional_embedding(dim))
                self._keys.append(key)
                continue
            t = torch.empty(shape)
            if init == "one":
                t.fill_(1.0)
            elif init == "zero":
                t.zero_()
            elif init == "xavier":
                nn.init.xavier_uniform_(t)
            else:
                bound = 1.0 / math.sqrt(init)
                nn.init.uniform_(t, -bound, bound)
            _attach(self, key, nn.Parameter(t))
            self._keys.append(key)
        self._desc = _lib.TfdecDesc(mel_channels, dim, mlp_factor, condition_dim, num_layers, N_POSITIONS)
        self._cond_channels = condition_dim
        self._init_engine()

    @torch.no_grad()
    def forward(self, x, diffusion_step, conditioner, x_masks=None, cond_masks=None):
        assert x.dim() == 3, f"mel must be 3 dim tensor, but got {x.dim()}"   # convnext.py:341 (no 4-D DiffSVC form here)
        if x.shape[-1] > N_POSITIONS:
            raise ValueError(f"{x.shape[-1]} frames exceed the positional table ({N_POSITIONS})")
        return super().forward(x, diffusion_step, conditioner, x_masks, cond_masks)

    def training_forward(self, x, diffusion_step, conditioner, x_masks=None, cond_masks=None, keep8=False):
        """`forward` under autograd (convnext.py:331-379; no dropout): x [B, mel, T], diffusion_step [B] or [1], conditioner [B, condition, T],
        masks [B, T] with true = padding; gradients for the parameters and for x and conditioner where they ask for them.  It runs in the parameters'
        type (fp32, or bf16 / fp16 after `.to()`) on the parameters themselves: nothing is packed.  keep8=True keeps the inputs of the linear layers and
        GELUs in 8 bits instead of the parameters' type (`ops.pack8`): the result is as exact (GELU is evaluated by `ops.gelu8`), weight gradients and GELU's
        derivative see inputs rounded to a step of at most 2/127 of the largest of their 32 neighbours.  Autocast is not applied: the parameters' type rules."""
        with torch.autocast(x.device.type, enabled=False):
            return self._training_forward(x, diffusion_step, conditioner, x_masks, cond_masks, keep8)

    def _training_forward(self, x, diffusion_step, conditioner, x_masks, cond_masks, keep8):
        assert x.dim() == 3, f"mel must be 3 dim tensor, but got {x.dim()}"
        sd = dict(self.named_parameters())
        w = sd["input_projection.0.weight"]
        _lib.require_gpu(x, "denoiser input")
        _lib.require_gpu(w, "denoiser parameters")
        B, M, T = x.shape
        if M != self.mel_channels or conditioner.dim() != 3 or conditioner.shape != (B, self.condition_dim, T):
            raise ValueError(f"x {tuple(x.shape)} does not match conditioner {tuple(conditioner.shape)}")
        if T > N_POSITIONS:
            raise ValueError(f"{T} frames exceed the positional table ({N_POSITIONS})")
        for name, m in (("x_masks", x_masks), ("cond_masks", cond_masks)):
            if m is not None and m.shape != (B, T):
                raise ValueError(f"{name} {tuple(m.shape)} is not [batch, frames] = {(B, T)}")
        held = ops._guard_capture([*sd.values(), x, conditioner])   # noqa: F841 (until the graph below holds the parameters' nodes)
        dim, dt = self.dim, w.dtype
        x_masks, cond_masks = (None if m is None else m.bool() for m in (x_masks, cond_masks))
        linear, gelu = (ops.linear8, ops.gelu8) if keep8 else (F.linear, F.gelu)

        def proj(t, name):                                  # Linear, or Conv1d with kernel 1 on [B, T, C]
            return linear(t, sd[name + ".weight"].flatten(1), sd[name + ".bias"])

        def mlp(t, a, b):
            return proj(gelu(proj(t, a)), b)

        def attend(q_in, kv_in, p, key_mask):
            wi, bi = sd[p + "in_proj_weight"], sd[p + "in_proj_bias"]
            if q_in is kv_in:
                q, k, v = linear(q_in, wi, bi).view(B, T, 3, 8, dim // 8).permute(2, 0, 3, 1, 4).unbind(0)
            else:
                q = linear(q_in, wi[:dim], bi[:dim]).view(B, T, 8, dim // 8).transpose(1, 2)
                k, v = linear(kv_in, wi[dim:], bi[dim:]).view(B, T, 2, 8, dim // 8).permute(2, 0, 3, 1, 4).unbind(0)
            return proj(ops.attention(q, k, v, key_mask).transpose(1, 2).reshape(B, T, dim), p + "out_proj")

        pos = self.positional_embedding[None, :T].to(dt)
        x = mlp(x.to(dt).transpose(1, 2).contiguous(), "input_projection.0", "input_projection.2") + pos * sd["position_scale_query"]
        t = diffusion_step.to(device=x.device, dtype=torch.float32).reshape(-1)
        half = dim // 2
        arg = t[:, None] * torch.exp(torch.arange(half, device=x.device) * -(math.log(10000) / (half - 1)))[None, :]
        step = mlp(torch.cat((arg.sin(), arg.cos()), dim=-1).to(dt), "diffusion_embedding.1", "diffusion_embedding.3")[:, None]
        mem = mlp(conditioner.to(dt).transpose(1, 2).contiguous(), "condition_projection.0", "condition_projection.2")
        mem = mem + pos * sd["position_scale_key"] + step
        if x_masks is not None:
            x = x.masked_fill(x_masks[..., None], 0.0)
        if cond_masks is not None:
            mem = mem.masked_fill(cond_masks[..., None], 0.0)
        for i in range(self.n_layers):
            p = f"layers.{i}."
            norm = lambda t, block, n: ops.residual_norm(t, block, pre_norm=(sd[p + n + ".weight"], sd[p + n + ".bias"]), need_h=False)[1]   # noqa: E731
            x = norm(x, attend(x, x, p + "self_attn.", x_masks), "norm1")
            x = norm(x, attend(x, mem, p + "multihead_attn.", cond_masks), "norm2")
            x = norm(x, mlp(x, p + "linear1", p + "linear2"), "norm3")
        x = mlp(x, "output_projection.0", "output_projection.2").transpose(1, 2)
        return x if x_masks is None else x.masked_fill(x_masks[:, None], 0.0)


DENOISERS.register_module(name="TransformerDecoderDenoiser", module=TransformerDecoderDenoiser, force=True)
DENOISERS.register_module(name="TransformerDecoderDenoiserMI355X", module=TransformerDecoderDenoiser, force=True)

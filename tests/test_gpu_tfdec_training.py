"""GPU: TransformerDecoderDenoiser.training_forward -- attention, residual + norm steps and 8-bit activations working together under autograd -- against the
oracle differentiated in 64 bits on the CPU."""
import pytest
import torch

from tests.helpers import TD_SMALL
from oracle import tfdec_ref

pytestmark = pytest.mark.gpu


def setup(dtype=torch.float32, B=2, T=70, masks=True):
    import fish_diffusion_amd as fda
    sd = tfdec_ref.seeded_state(11, **TD_SMALL)
    net = fda.TransformerDecoderDenoiser(**TD_SMALL)
    net.load_state_dict(sd, strict=True)
    net = net.cuda().to(dtype)
    g = torch.Generator().manual_seed(5)
    x, cond = torch.randn(B, 128, T, generator=g), torch.randn(B, 256, T, generator=g)
    step = torch.tensor([3.0, 700.0][:B])
    xm = cm = None
    if masks:
        xm = torch.arange(T)[None, :] >= torch.tensor([T, T - 23])[:, None]
        cm = torch.arange(T)[None, :] >= torch.tensor([T - 9, T - 23])[:, None]
    return net, sd, x, step, cond, xm, cm, torch.randn(B, 128, T, generator=g)


def oracle_grads(sd, x, step, cond, xm, cm, gy, dtype):
    """(output, {name: gradient}) of the oracle in `dtype` on the CPU (attention through torch's own elementary operations: the oracle's fused softmax has no
    64-bit gradient)."""
    leaf = {k: v.to(dtype, copy=True).requires_grad_(k != "positional_embedding") for k, v in sd.items()}
    x, cond = x.to(dtype, copy=True).requires_grad_(), cond.to(dtype, copy=True).requires_grad_()

    def mha(s, p, q_in, kv_in, kpm):
        D, H = q_in.shape[-1], 8
        w, b = s[p + "in_proj_weight"], s[p + "in_proj_bias"]
        heads = lambda t: t.view(*t.shape[:2], H, D // H).transpose(1, 2)      # noqa: E731
        q, k, v = (heads(torch.nn.functional.linear(t, w[i * D:(i + 1) * D], b[i * D:(i + 1) * D])) for i, t in enumerate((q_in, kv_in, kv_in)))
        z = q @ k.transpose(-1, -2) / (D // H) ** 0.5
        if kpm is not None:
            z = z.masked_fill(kpm[:, None, None, :], float("-inf"))
        o = (torch.softmax(z, -1) @ v).transpose(1, 2).reshape(q_in.shape)
        return torch.nn.functional.linear(o, s[p + "out_proj.weight"], s[p + "out_proj.bias"])
    keep = tfdec_ref.mha
    tfdec_ref.mha = mha
    try:
        y = tfdec_ref.tfdec_forward(leaf, x, step.to(dtype), cond, xm, cm, num_layers=TD_SMALL["num_layers"])
    finally:
        tfdec_ref.mha = keep
    names = [k for k in leaf if k != "positional_embedding"]
    grads = torch.autograd.grad((y * gy.to(dtype)).sum(), [leaf[k] for k in names] + [x, cond])
    return y.detach(), dict(zip(names + ["x", "cond"], grads))


def run(net, x, step, cond, xm, cm, gy, keep8):
    x, cond = x.cuda().requires_grad_(), cond.cuda().requires_grad_()
    net.zero_grad()
    on = lambda m: None if m is None else m.cuda()     # noqa: E731
    y = net.training_forward(x, step.cuda(), cond, on(xm), on(cm), keep8=keep8)
    y.backward(gy.cuda().to(y.dtype))
    return y.detach().cpu(), dict({k: p.grad.cpu() for k, p in net.named_parameters()}, x=x.grad.cpu(), cond=cond.grad.cpu())


def rel(a, b):
    return float((a.double() - b).norm() / b.norm().clamp_min(1e-30))


@pytest.mark.parametrize("masks", [False, True])
def test_fp32_gradients(masks):
    """Both sides evaluate the same fp32 operations in another order, so their distances from the 64-bit result are of one size: at most four times torch's own
    fp32 evaluation of the oracle, per tensor, or 1e-6 (where that happens to be near exact)."""
    net, sd, *a = setup(masks=masks)
    y64, g64 = oracle_grads(sd, *a, torch.float64)
    y32, g32 = oracle_grads(sd, *a, torch.float32)
    y, g = run(net, *a, keep8=False)
    assert set(g) == set(g64)
    assert rel(y, y64) <= max(4 * rel(y32, y64), 1e-6)
    for k in g64:
        # (a key bias shifts all scores of a row alike: its gradient is 0 and only noise is left; compared on the whole in_proj_bias)
        assert rel(g[k], g64[k]) <= max(4 * rel(g32[k], g64[k]), 1e-6), k
    # the inference path computes the same function
    on = lambda m: None if m is None else m.cuda()     # noqa: E731
    x, step, cond, xm, cm, _ = a
    assert rel(net(x.cuda(), step.cuda(), cond.cuda(), on(xm), on(cm)).cpu(), y64) < 2e-5


def test_activations_in_8_bits():
    """The result is fp32's (its GELU is another evaluation of the same function, so not the same bits: held to the bound of the fp32 test).  A code is off by at most half of 2/127 of its group's largest value, 1 % of a normal group's deviation (rms), so a weight's
    gradient is off by about 1 % for its own input and the same again, in quadrature, for each of the 9 GELUs behind which the gradient has passed: 4 %."""
    net, sd, *a = setup()
    y, g = run(net, *a, keep8=False)
    y8, g8 = run(net, *a, keep8=True)
    y64, y32 = (oracle_grads(sd, *a, d)[0] for d in (torch.float64, torch.float32))
    assert rel(y8, y64) <= max(4 * rel(y32, y64), 1e-6)
    for k in g:
        if k.endswith("in_proj_bias") or g[k].norm() == 0:
            continue
        assert rel(g8[k], g[k].double()) < 0.04, k


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_16_bit_parameters(dtype):
    """Every stored tensor is rounded (half a step u relative): some 30 roundings along the deepest path and as many back, in quadrature sqrt(60) u, and
    up to four times that where a layer norm amplifies."""
    net, sd, *a = setup(dtype)
    sd = {k: v.to(dtype).float() for k, v in sd.items()}
    a[0], a[2] = a[0].to(dtype).float(), a[2].to(dtype).float()
    y64, g64 = oracle_grads(sd, *a, torch.float64)
    u = torch.finfo(dtype).eps / 2
    for keep8 in (False, True):
        y, g = run(net, *a, keep8=keep8)
        assert rel(y, y64) < 4 * 60 ** 0.5 * u
        for k in g64:
            if not k.endswith("in_proj_bias"):
                assert rel(g[k], g64[k]) < 4 * 60 ** 0.5 * u + (0.04 if keep8 else 0.0), k


def test_memory_refusals_and_update():
    net, sd, x, step, cond, xm, cm, gy = setup(B=2, T=700, masks=False)
    x, step, cond = x.cuda(), step.cuda(), cond.cuda()

    def held(keep8):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = net.training_forward(x, step, cond, keep8=keep8)
        after = torch.cuda.memory_allocated()
        del y
        return after - before
    held(False)
    assert held(True) < 0.85 * held(False)
    with pytest.raises(ValueError):
        net.training_forward(x, step, cond[:, :, :-1])
    with pytest.raises(ValueError):
        net.training_forward(x, step, cond, x_masks=torch.zeros(2, 3, device="cuda"))
    with pytest.raises(RuntimeError, match="MI355X"):
        net.training_forward(x.cpu(), step, cond)
    # a step of gradient descent reaches the inference path (its packed weights follow the parameters)
    net.training_forward(x, step, cond).square().mean().backward()
    with torch.no_grad():
        for p in net.parameters():
            p -= 1e-2 * p.grad
        assert rel(net(x, step, cond).cpu(), net.training_forward(x, step, cond).cpu().double()) < 2e-5


def test_capture_beside_a_live_graph_is_refused():
    net, sd, x, step, cond, *_ = setup(masks=False)
    x, step, cond = x.cuda(), step.cuda(), cond.cuda()
    y = net.training_forward(x, step, cond)   # noqa: F841 (its graph holds the parameters)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="outside this capture"):
            net.training_forward(x, step, cond)


@pytest.mark.parametrize("keep8", [False, True])
def test_autocast_is_not_applied(keep8):
    net, _, x, step, cond, xm, cm, gy = setup()
    x, step, cond, xm, cm, gy = (t.cuda() for t in (x, step, cond, xm, cm, gy))
    got = []
    for on in (False, True):
        net.zero_grad()
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=on):
            y = net.training_forward(x, step, cond, xm, cm, keep8=keep8)
        y.backward(gy)
        got.append([y.detach()] + [p.grad.clone() for p in net.parameters()])
    assert all(a.dtype == torch.float32 and torch.equal(a, b) for a, b in zip(*got))

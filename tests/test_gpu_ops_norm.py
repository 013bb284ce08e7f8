"""GPU: the norm / gate / residual step and its backward pass against the formula in 64 bits.

Every quantity is carried with a bound on its error, e = 2^-24 per fp32 operation, u = eps / 2 of the result's type; a mean over a row is off by at most
K e times the mean of magnitudes (K = 64 > 32 terms in a thread + 6 + 8 steps over lanes and waves), a sum over N rows by (N + 64) e."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E, K = 2.0 ** -24, 64
T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def mean(x):
    return x.mean(-1, keepdim=True)


def norm(v, tv, wb, rms, eps):
    m = torch.zeros_like(mean(v)) if rms else mean(v)
    d = v - m
    td = tv + E * 2 * v.abs() + (0 if rms else mean(tv) + K * E * mean(v.abs()))
    r = (mean(d * d) + eps).rsqrt()
    hat = d * r
    rel = K * E + r * mean(hat.abs() * td)                      # of r
    that = r * td + hat.abs() * (rel + 2 * E)
    w, b = wb
    y = hat * w + (0 if b is None else b)
    return y, w.abs() * that + 2 * E * ((hat * w).abs() + (0 if b is None else b.abs())), hat, that, r, rel


def norm_grad(g, tg, hat, that, r, rel, w, rms):
    gw, tgw = g * w, tg * w.abs() + E * (g * w).abs()
    c2, tc2 = mean(gw * hat), mean(tgw * hat.abs() + gw.abs() * that) + K * E * mean((gw * hat).abs())
    c1, tc1 = (0.0, 0.0) if rms else (mean(gw), mean(tgw) + K * E * mean(gw.abs()))
    d = gw - c1 - hat * c2
    td = tgw + tc1 + that * c2.abs() + hat.abs() * tc2 + 4 * E * (gw.abs() + (0 if rms else c1.abs()) + (hat * c2).abs())
    return r * d, r * td + (r * d).abs() * (rel + 2 * E)


def reference(x, block, gate, a, post, pre, rms, eps, gh, gy):
    d = torch.float64
    t = x.dtype
    x, block = x.to(d), block.to(d)
    g = None if gate is None else gate.to(d)
    if g is not None and g.dim() == 2 and x.dim() == 3:
        g = g[:, None]
    post = None if post is None else [None if p is None else p.to(d) for p in post]
    pre = None if pre is None else [None if p is None else p.to(d) for p in pre]
    val, tol = {}, {}
    n, tn = block, torch.zeros_like(block)
    if post:
        n, tn, bhat, tbhat, br, brel = norm(block, tn, post, rms, eps)
    gn, tgn = (n, tn) if g is None else (g * n, g.abs() * tn)
    h = a * x + gn
    th = tgn + 3 * E * ((a * x).abs() + gn.abs())
    val["h"], tol["h"] = h, th
    if pre:
        y, ty, hhat, thhat, hr, hrel = norm(h, th, pre, rms, eps)
        val["y"], tol["y"] = y, ty
    dh, tdh = torch.zeros_like(x), torch.zeros_like(x)
    N = x.numel() // x.shape[-1]
    S = (N + 64) * E
    rows = lambda v: v.reshape(N, -1).sum(0)          # noqa: E731
    if gh is not None:
        dh = dh + gh.to(d)
    if gy is not None:
        gy = gy.to(d)
        k, tk = norm_grad(gy, torch.zeros_like(gy), hhat, thhat, hr, hrel, pre[0], rms)
        dh, tdh = dh + k, tdh + tk + 2 * E * (k.abs() + dh.abs())
        val["dpre_weight"], tol["dpre_weight"] = rows(gy * hhat), rows(gy.abs() * thhat) + S * rows((gy * hhat).abs())
        val["dpre_bias"], tol["dpre_bias"] = rows(gy), S * rows(gy.abs())
    elif pre:
        val["dpre_weight"] = val["dpre_bias"] = torch.zeros_like(pre[0])
        tol["dpre_weight"] = tol["dpre_bias"] = torch.zeros_like(pre[0])
    val["dx"], tol["dx"] = a * dh, abs(a) * (tdh + E * dh.abs())
    dn, tdn = dh, tdh
    if g is not None:
        dn, tdn = g * dh, g.abs() * tdh + E * (g * dh).abs()
        dg, tdg = dh * n, tdh * n.abs() + dh.abs() * tn + E * (dh * n).abs()
        if gate.shape == x.shape:
            val["dgate"], tol["dgate"] = dg, tdg
        elif gate.dim() == 1:
            val["dgate"], tol["dgate"] = rows(dg), rows(tdg) + S * rows(dg.abs())
        else:
            val["dgate"], tol["dgate"] = dg.sum(1).view(gate.shape), (tdg.sum(1) + S * dg.abs().sum(1)).view(gate.shape)
    val["dblock"], tol["dblock"] = dn, tdn
    if post:
        val["dpost_weight"], tol["dpost_weight"] = rows(dn * bhat), rows(tdn * bhat.abs() + dn.abs() * tbhat) + S * rows((dn * bhat).abs())
        val["dpost_bias"], tol["dpost_bias"] = rows(dn), rows(tdn) + S * rows(dn.abs())
        val["dblock"], tol["dblock"] = norm_grad(dn, tdn, bhat, tbhat, br, brel, post[0], rms)
    del t
    return val, tol


def make(t, shape, gate, post, pre, kind, pt=None, gt=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")      # noqa: E731
    C = shape[-1]
    x, block = (2 * rn(*shape)).to(t), (rn(*shape) + 0.5 * rn(C)).to(t)
    gs = {None: None, "channel": (C,), "item": (shape[0], C), "item1": (shape[0], 1, C), "full": shape}[gate]
    gate = None if gs is None else (0.5 + rn(*gs)).to(gt or t)
    wb = lambda: ((1 + 0.2 * rn(C)).to(pt or t), (0.1 * rn(C)).to(pt or t) if kind == "layer" else None)     # noqa: E731
    kw = dict(gate=gate, residual_scale=1.0 if gate is None else 0.8, post_norm=wb() if post else None, pre_norm=wb() if pre else None, kind=kind, eps=1e-5)
    return x, block, rn(*shape).to(t), rn(*shape).to(t) if pre else None, kw


def check(x, block, gh, gy, kw):
    import fish_diffusion_amd as fda
    h, y, stats = fda.residual_norm_forward(x, block, **kw)
    gr = fda.residual_norm_backward(gh, gy, x, block, stats, **kw)
    val, tol = reference(x, block, kw["gate"], kw["residual_scale"], kw["post_norm"], kw["pre_norm"], kw["kind"] == "rms", kw["eps"], gh, gy)
    got = dict(gr._asdict(), h=h, y=y)
    for n, v in got.items():
        if v is None:
            continue
        u = torch.finfo(v.dtype).eps / 2
        tiny = 2.0 ** -24 if v.dtype == torch.float16 else 2.0 ** -126
        assert v.shape == val[n].shape, n
        lim = tol[n] * (1 + u) + u * val[n].abs() + tiny
        err = (v.double() - val[n]).abs()
        assert (err <= lim).all(), f"{n}: worst {float((err / lim).max()):.3g} times its bound"
    assert (kw["pre_norm"] is None) == (y is None)
    return got


@pytest.mark.parametrize("t", list(T))
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 7), (1, 430, 512), (3, 37, 515), (2, 65, 1000), (2, 33, 1536), (1, 9, 2048), (2, 21, 3001), (1, 5, 8192)], ids=str)
@pytest.mark.parametrize("gate,post,pre,kind", [(None, False, True, "layer"), ("channel", False, True, "rms"), ("item", True, True, "layer"),
                                                ("full", True, False, "rms")])
def test_against_the_formula(t, shape, gate, post, pre, kind):
    check(*make(T[t], shape, gate, post, pre, kind))


@pytest.mark.parametrize("gate", [None, "channel", "item", "item1", "full"])
@pytest.mark.parametrize("shape", [(400, 2, 64), (2000, 3, 40), (40, 100, 48), (3, 5000, 72)], ids=str)
def test_gates_of_every_run_length(gate, shape):
    """Many short items (summed where they are read), few long ones (cut over workgroups), and between."""
    check(*make(torch.float32, shape, gate, True, True, "layer", seed=1))


@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_fp32_parameters_and_gate_beside_16_bits(t):
    for gate in ("channel", "item", "full"):
        got = check(*make(T[t], (4, 50, 256), gate, True, True, "layer", pt=torch.float32, gt=torch.float32))
        assert got["dpre_weight"].dtype == got["dgate"].dtype == torch.float32
    check(*make(T[t], (4, 50, 100), "item", True, True, "rms", pt=torch.float32))


def test_missing_gradients_views_and_no_rows():
    import fish_diffusion_amd as fda
    x, block, gh, gy, kw = make(torch.float32, (2, 31, 96), "item", True, True, "layer")
    check(x, block, None, gy, kw)
    check(x, block, gh, None, kw)
    check(x, block, None, None, kw)
    wide = torch.zeros(2, 31, 200, device="cuda")
    wide[..., 3:99] = x
    check(wide[..., 3:99], block.transpose(0, 1).contiguous().transpose(0, 1), gh, gy, kw)            # views that are copied
    flat = torch.zeros(2 * 31 * 96 + 1, device="cuda")
    flat[1:] = block.reshape(-1)
    check(x, flat[1:].view(2, 31, 96), gh, gy, kw)                                                    # 4 bytes off
    e = torch.zeros(0, 7, 96, device="cuda")
    h, y, stats = fda.residual_norm_forward(e, e, pre_norm=kw["pre_norm"], gate=torch.ones(96, device="cuda"))
    g = fda.residual_norm_backward(e, e, e, e, stats, pre_norm=kw["pre_norm"], gate=torch.ones(96, device="cuda"))
    assert h.shape == e.shape and (g.dpre_weight == 0).all() and (g.dgate == 0).all()
    h, y, _ = fda.residual_norm_forward(x[0, 0], block[0, 0])                                         # one vector
    assert y is None and torch.equal(h, x[0, 0] + block[0, 0])


def test_large_offset_keeps_the_variance():
    """A mean a thousand deviations off: the squares are summed after the mean is taken."""
    x = torch.randn(64, 512, device="cuda") + 1000.0
    z = torch.zeros_like(x)
    one = (torch.ones(512, device="cuda"), None)
    import fish_diffusion_amd as fda
    _, y, _ = fda.residual_norm_forward(x, z, pre_norm=one)
    d = x.double()
    d = d - d.mean(-1, keepdim=True)
    want = d * (d.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    # the mean is off by at most K e 1000 = 3.8e-3 in theory; its typical rounding, 2^-24 * 1000 * a few, is what (v - mean) r shows
    assert (y.double() - want).abs().max() < K * E * 1001


def test_same_bits_streams_and_capture():
    import fish_diffusion_amd as fda
    x, block, gh, gy, kw = make(torch.bfloat16, (8, 300, 512), "item", True, True, "layer")

    def both():
        h, y, stats = fda.residual_norm_forward(x, block, **kw)
        return (h, y, *fda.residual_norm_backward(gh, gy, x, block, stats, **kw))
    a = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(a, b) if p is not None)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = both()
    for s in range(3):
        x2, b2, gh2, gy2, _ = make(torch.bfloat16, (8, 300, 512), "item", True, True, "layer", seed=s + 9)
        for d, v in ((x, x2), (block, b2), (gh, gh2), (gy, gy2)):
            d.copy_(v)
        want = both()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(r, want) if p is not None), s


def test_autograd():
    import fish_diffusion_amd as fda
    x, block, gh, gy, kw = make(torch.float32, (2, 9, 48), "item", True, True, "layer")
    leaves = [t.clone().requires_grad_() for t in (x, block, kw["gate"], *kw["post_norm"], *kw["pre_norm"])]
    lx, lb, lg, pw, pb, nw, nb = leaves
    h, y = fda.residual_norm(lx, lb, lg, kw["residual_scale"], (pw, pb), (nw, nb))
    got = torch.autograd.grad((h * gh).sum() + (y * gy).sum(), leaves)
    d = [t.detach().double().requires_grad_() for t in leaves]

    def ln(v, w, b):
        return torch.nn.functional.layer_norm(v, (48,), w, b, 1e-5)
    hh = kw["residual_scale"] * d[0] + d[2][:, None] * ln(d[1], d[3], d[4])
    want = torch.autograd.grad((hh * gh.double()).sum() + (ln(hh, d[5], d[6]) * gy.double()).sum(), d)
    for a, b in zip(got, want):
        assert (a.double() - b).abs().max() <= 1e-5 * b.abs().max()
    # the post-norm step of a transformer layer: only y is used, x and block share one gradient
    lx, lb = x.clone().requires_grad_(), block.clone().requires_grad_()
    fda.residual_norm(lx, lb, pre_norm=kw["pre_norm"])[1].sum().backward()
    assert torch.equal(lx.grad, lb.grad) and lx.grad.data_ptr() != lb.grad.data_ptr()


def test_refusals_on_the_device():
    import fish_diffusion_amd as fda
    x, block, gh, gy, kw = make(torch.float32, (2, 9, 48), None, False, True, "layer")
    h, y, stats = fda.residual_norm_forward(x, block, **kw)
    for bad in (dict(gate=torch.ones(9, device="cuda")), dict(gate=torch.ones(48)), dict(pre_norm=(torch.ones(48), None)), dict(pre_norm=(None, None))):
        with pytest.raises((ValueError, RuntimeError)):
            fda.residual_norm_forward(x, block, **{**kw, **bad})
    for args in ((gh[:1], gy, x, block, stats), (gh, gy.half(), x, block, stats), (gh, gy, x, block, stats[:1])):
        with pytest.raises(ValueError):
            fda.residual_norm_backward(*args, **kw)
    with pytest.raises(ValueError):
        fda.residual_norm_backward(gh, gy, x, block, stats)


def test_only_the_normalised_result():
    import fish_diffusion_amd as fda
    x, block, gh, gy, kw = make(torch.float32, (2, 9, 48), "channel", False, True, "layer")
    h, y, stats = fda.residual_norm_forward(x, block, **kw)
    none, y2, stats2 = fda.residual_norm_forward(x, block, **kw, need_h=False)
    assert none is None and torch.equal(y, y2) and torch.equal(stats, stats2)
    lx = x.clone().requires_grad_()
    h, y = fda.residual_norm(lx, block, **kw, need_h=False)
    assert h is None
    y.backward(gy)
    assert torch.equal(lx.grad, fda.residual_norm_backward(None, gy, x, block, stats, **kw).dx)
    with pytest.raises(ValueError):
        fda.residual_norm(x, block, need_h=False)


def test_one_tensor_as_both_inputs():
    """x and block may be one tensor: their gradients, which are one tensor too where they are equal, add up."""
    import fish_diffusion_amd as fda
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(5, 7, 64, generator=g, device="cuda")
    w, gh, gy = (torch.randn(*s, generator=g, device="cuda") for s in ((64,), (5, 7, 64), (5, 7, 64)))
    for leaf in (True, False):
        t = x.clone().requires_grad_()
        u = t if leaf else t * 1.0
        h, y = fda.residual_norm(u, u, pre_norm=(w, None))
        got, = torch.autograd.grad((h, y), t, (gh, gy))
        t.grad = None
        h, y = fda.residual_norm(u if leaf else t * 1.0, u if leaf else t * 1.0, pre_norm=(w, None))
        torch.autograd.backward((h, y), (gh, gy))
        d = x.double().requires_grad_()
        z = 2 * d
        ref = torch.nn.functional.layer_norm(z, (64,), w.double())
        want, = torch.autograd.grad((z, ref), d, (gh.double(), gy.double()))
        # 64 products a sum, |grad| and |normalised| up to 4 each, three such terms, doubled: 2 * 3 * 66 * 16 * 2^-24
        assert (got.double() - want).abs().max() <= 4e-4 and torch.equal(t.grad, got)
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    h, y = fda.residual_norm(a, b, pre_norm=(w, None))
    torch.autograd.backward((h, y), (gh, gy))
    a.grad.zero_()                                       # (two parameters' gradients are two tensors)
    assert b.grad.any()

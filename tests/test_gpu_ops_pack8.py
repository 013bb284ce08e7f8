"""GPU: 8-bit activation checkpoints and the gradients taken from them."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def reference(x):
    """codes, exponents and values from the definition, in 64 bits: the smallest e >= 1 with max|x| <= 127 * 2^(e - 127); codes end at 63 at e = 249, where
    64 would stand for 2^128."""
    C = x.shape[-1]
    d = x.double().reshape(-1, C)
    G = (C + 31) // 32
    p = torch.nn.functional.pad(d, (0, G * 32 - C)).view(-1, G, 32)
    top = p.abs().amax(-1)
    bad = ~torch.isfinite(top)
    e = torch.ones_like(top)
    t = torch.where(bad, torch.zeros_like(top), top)
    for _ in range(256):
        e = torch.where(t > 127 * torch.exp2(e - 127), e + 1, e)
    s = torch.exp2(e - 127)[..., None]
    codes = torch.where(bad[..., None], torch.zeros_like(p), torch.round(torch.where(bad[..., None], torch.zeros_like(p), p) / s))
    codes = torch.where((e == 249)[..., None], codes.clamp(-63, 63), codes)
    val = torch.where(bad[..., None], torch.full_like(p, math.nan), codes * s)
    flat = lambda v: v.reshape(-1, G * 32)[:, :C].reshape(x.shape)      # noqa: E731
    return flat(codes).to(torch.int8), torch.where(bad, torch.full_like(e, 255), e).to(torch.uint8).view(*x.shape[:-1], G), flat(val)


def make(t, *shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * torch.exp(torch.randn(shape[-1], generator=g, device="cuda"))).to(t)


@pytest.mark.parametrize("t", list(T))
@pytest.mark.parametrize("shape", [(1, 1), (5, 31), (4, 32), (7, 33), (3, 40), (2, 9, 512), (861, 2048), (3, 1001)], ids=str)
def test_pack_and_unpack_bit_for_bit(t, shape):
    import fish_diffusion_amd as fda
    x = make(T[t], *shape)
    codes, exps, val = reference(x)
    p = fda.pack8(x)
    assert torch.equal(p.codes, codes) and torch.equal(p.exponents, exps)
    assert torch.equal(fda.unpack8(p).double(), val) and torch.equal(fda.unpack8(p, torch.bfloat16).double(), val)
    y, q = fda.gelu8_forward(x)
    assert torch.equal(q.codes, codes) and torch.equal(q.exponents, exps)


def test_borders_and_specials():
    import fish_diffusion_amd as fda
    rows = []
    for k in (-149, -140, -127, -126, -120, -7, 0, 1, 100, 120):
        for m in (1.0, 63.0, 63.5, 64.0, 126.5, 127.0, math.nextafter(127.0, 128.0), 127.5, 127.99999, 128.0, 2.5, 0.5):
            v = min(m * 2.0 ** k, 3.4e38)
            r = torch.zeros(32, dtype=torch.float64)
            r[0], r[1], r[2], r[3] = v, -v / 2, v / 3, -0.0
            rows.append(r.float())
    rows += [torch.zeros(32), torch.full((32,), 3.4028234e38), torch.full((32,), -1e-45)]
    x = torch.stack(rows).cuda()
    codes, exps, val = reference(x)
    p = fda.pack8(x)
    assert torch.equal(p.codes, codes) and torch.equal(p.exponents, exps) and torch.equal(fda.unpack8(p).double(), val)
    x = make(torch.float32, 4, 96)
    x[0, 5], x[1, 40], x[2, 95] = math.inf, -math.inf, math.nan
    codes, exps, val = reference(x)
    p = fda.pack8(x)
    assert torch.equal(p.codes, codes) and torch.equal(p.exponents, exps)
    assert torch.equal(torch.isnan(fda.unpack8(p)), torch.isnan(val)) and int(torch.isnan(val).sum()) == 96
    dw, _ = fda.linear8_weight_grad(torch.ones(4, 3, device="cuda"), p)
    assert torch.isnan(dw).all() and not torch.isnan(fda.linear8_weight_grad(torch.ones(1, 3, device="cuda"), fda.Packed8(p.codes[3:], p.exponents[3:]))[0]).any()


@pytest.mark.parametrize("t", list(T))
@pytest.mark.parametrize("N,O,I", [(1, 1, 1), (3, 8, 32), (31, 130, 40), (33, 7, 129), (861, 512, 256), (1000, 100, 333), (5000, 129, 257), (0, 16, 16)])
def test_weight_gradient(t, N, O, I):
    """Products are exact, so a sum of N of them is off by at most (N + 16) e sum|dy x8| (any order), and the result's own rounding."""
    import fish_diffusion_amd as fda
    x, dy = make(T[t], N, I), make(T[t], N, O, seed=1)
    p = fda.pack8(x)
    x8, d = fda.unpack8(p).double(), dy.double()
    for dtype in (None, torch.float32):
        dw, db = fda.linear8_weight_grad(dy, p, dtype=dtype)
        u = torch.finfo(dw.dtype).eps / 2
        for got, want, mag in ((dw, d.T @ x8, d.abs().T @ x8.abs()), (db, d.sum(0), d.abs().sum(0))):
            lim = (N + 16) * E * mag * (1 + u) + u * want.abs() + (2.0 ** -24 if got.dtype == torch.float16 else 2.0 ** -120)
            # (what rounds to fp16 from 65520 = 65504 + half a step on is infinity)
            past = (want.abs() - (N + 16) * E * mag >= 65520) & (got.double() == want.sign() * math.inf) & (got.dtype == torch.float16)
            assert got.shape == want.shape and (past | ((got.double() - want).abs() <= lim)).all()
    assert fda.linear8_weight_grad(dy, p, bias=False)[1] is None


def test_weight_gradient_of_every_bit_of_fp32():
    """One row: dw is dy x8 rounded once to fp32, to the last bit (the three parts of dy carry all 24 bits)."""
    import fish_diffusion_amd as fda
    dy, x = make(torch.float32, 1, 256), make(torch.float32, 1, 64, seed=3)
    p = fda.pack8(x)
    dw, _ = fda.linear8_weight_grad(dy, p)
    want = dy.double().T @ fda.unpack8(p).double()
    assert ((dw.double() - want).abs() <= 3 * E * want.abs()).all()      # three exact parts, two roundings of their sum and the last one
    dy16 = make(torch.float16, 1, 256)
    dw, _ = fda.linear8_weight_grad(dy16, p, dtype=torch.float32)
    want = dy16.double().T @ fda.unpack8(p).double()
    assert ((dw.double() - want).abs() <= 2 * E * want.abs()).all()


def gelu_parts(u):
    cdf = 0.5 * torch.erfc(-u / math.sqrt(2.0))
    return cdf, u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)


@pytest.mark.parametrize("t", list(T))
@pytest.mark.parametrize("shape", [(1, 1), (7, 33), (200, 2048)], ids=str)
def test_gelu_and_gradient(t, shape):
    """erfc's fit 3.3e-8 + 20 operations, the exponential's argument u^2 e: relative error q of the smaller tail; Phi, u phi and their sum follow."""
    import fish_diffusion_amd as fda
    x, dy = make(T[t], *shape), make(T[t], *shape, seed=5)
    if x.numel() > 1000:
        x.view(-1)[:400] = torch.linspace(-12, 12, 400, device="cuda").to(T[t])
    y, p = fda.gelu8_forward(x)
    u = torch.finfo(T[t]).eps / 2
    tiny = 2.0 ** -24 if t == "f16" else 2.0 ** -120

    def cdf_err(v):
        return torch.minimum(gelu_parts(v)[0], gelu_parts(-v)[0]) * (3.3e-8 + (24 + v * v) * E) + E * (v > 0)
    v = x.double()
    want = v * gelu_parts(v)[0]
    assert ((y.double() - want).abs() <= v.abs() * cdf_err(v) + (2 * E + u) * want.abs() + tiny).all()
    v = fda.unpack8(p).double()
    cdf, upd = gelu_parts(v)
    dx = fda.gelu8_backward(dy, p)
    d = dy.double()
    want = d * (cdf + upd)
    # the exponential instruction gives 0 for results below 2^-126, so exp(-v^2 / 2) is off by less than 2^-126 there and v phi(v) by 0.4 |v| times that
    lim = d.abs() * (0.4 * v.abs() * 2.0 ** -126 + cdf_err(v) + upd.abs() * (8 + v * v) * E + 2 * E * (cdf + upd.abs())) + u * want.abs() + tiny
    assert ((dx.double() - want).abs() <= lim).all()


def test_gelu_far_out():
    import fish_diffusion_amd as fda
    x = torch.tensor([[-1e30, -1e4, -40.0, -13.0, 13.0, 40.0, 1e4, 1e30, 0.0, -0.0, math.inf, math.nan]], device="cuda")
    y, _ = fda.gelu8_forward(x)
    assert torch.equal(y[0, :3], torch.zeros(3, device="cuda")) and torch.equal(y[0, 4:8], x[0, 4:8]) and (y[0, 8:10] == 0).all()
    assert y[0, 10] == math.inf and torch.isnan(y[0, 11])


def test_autograd_streams_and_capture():
    import fish_diffusion_amd as fda
    x, w, b = make(torch.float32, 3, 50, 96), make(torch.float32, 64, 96, seed=1), make(torch.float32, 64, seed=2)
    dy = make(torch.float32, 3, 50, 64, seed=4)
    lx, lw, lb = (t.clone().requires_grad_() for t in (x, w, b))
    y = fda.linear8(lx, lw, lb)
    assert torch.equal(y, torch.nn.functional.linear(x, w, b))
    y.backward(dy)
    dw, db = fda.linear8_weight_grad(dy, fda.pack8(x))
    assert torch.equal(lw.grad, dw) and torch.equal(lb.grad, db) and torch.equal(lx.grad, dy @ w)
    lx = x.clone().requires_grad_()
    fda.gelu8(lx).backward(x)
    assert torch.equal(lx.grad, fda.gelu8_backward(x, fda.pack8(x)))

    def all_of():
        p = fda.pack8(x)
        z, q = fda.gelu8_forward(x)
        return (*fda.linear8_weight_grad(dy, p), z, fda.gelu8_backward(x, q), fda.unpack8(p))
    want = all_of()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = all_of()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = all_of()
    for s in range(3):
        x.copy_(make(torch.float32, 3, 50, 96, seed=20 + s))
        want = all_of()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(r, want)), s


def test_refusals_on_the_device():
    import fish_diffusion_amd as fda
    x = make(torch.float32, 6, 64)
    p = fda.pack8(x)
    with pytest.raises(ValueError):
        fda.linear8_weight_grad(x[:5], p)
    with pytest.raises(ValueError):
        fda.gelu8_backward(x[:, :32], p)
    with pytest.raises(ValueError):
        fda.unpack8(fda.Packed8(p.codes, p.exponents[:, :1]))
    with pytest.raises(TypeError):
        fda.unpack8(p, torch.float64)
    with pytest.raises(ValueError):
        fda.linear8(x, make(torch.float32, 4, 63))
    with pytest.raises(ValueError):
        fda.linear8(x, make(torch.float16, 4, 64))


def test_finite_values_stay_finite():
    import fish_diffusion_amd as fda
    for t in T.values():
        x = torch.full((2, 40), torch.finfo(t).max, dtype=t, device="cuda")
        x[1] = -x[1]
        p = fda.pack8(x)
        for o in T.values():
            y = fda.unpack8(p, o)
            if torch.finfo(o).max >= torch.finfo(t).max or o == torch.float16:
                assert torch.isfinite(y).all() and (y[0] > 0).all() and (y[1] < 0).all()


def test_linear_under_autocast_keeps_its_type():
    import fish_diffusion_amd as fda
    x, w, b = (make(torch.float32, *s, seed=i).requires_grad_() for i, s in enumerate(((9, 64), (40, 64), (40,))))
    dy = make(torch.float32, 9, 40, seed=5)
    want = torch.autograd.grad(fda.linear8(x, w, b), (x, w, b), dy)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = fda.linear8(x, w, b)
        got = torch.autograd.grad(y, (x, w, b), dy)
    assert y.dtype == torch.float32 and torch.equal(y, fda.linear8(x, w, b))
    assert all(torch.equal(g, t) for g, t in zip(got, want))


@pytest.mark.parametrize("t", list(T))
@pytest.mark.parametrize("N,O,I", [(1, 256, 256), (17, 40, 384), (47, 256, 136), (65, 384, 128), (600, 200, 512), (2000, 504, 264), (6888, 512, 384), (9001, 136, 1000)], ids=str)
def test_weight_gradient_of_wide_tiles(t, N, O, I):
    test_weight_gradient(t, N, O, I)


@pytest.mark.parametrize("t", list(T))
def test_weight_gradient_from_misaligned_memory(t):
    """The C entry takes rows that cannot be read 16 bytes at a time; the workspace is sized without knowing."""
    import ctypes as C

    import fish_diffusion_amd as fda
    from fish_diffusion_amd import _lib
    N, O, I = 700, 256, 512
    x, dy = make(T[t], N, I), make(T[t], N, O, seed=1)
    p, want = fda.pack8(x), fda.linear8_weight_grad(dy, fda.pack8(x))
    dy1, codes1 = torch.empty(N * O + 8, dtype=T[t], device="cuda"), torch.empty(N * I + 8, dtype=torch.int8, device="cuda")
    dy1[1:N * O + 1] = dy.flatten()
    codes1[3:N * I + 3] = p.codes.flatten()
    lib, h, n = _lib.lib(), _lib.Handle.shared(x.device), C.c_size_t()
    dt = _lib.DTYPES[T[t]]
    assert lib.fdx_linear8_weight_grad_workspace(dt, N, O, I, C.byref(n)) == 0
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    for a, b in ((dy1[1:], p.codes), (dy, codes1[3:]), (dy1[1:], codes1[3:])):
        dw, db = torch.full((O, I), 7.0, dtype=T[t], device="cuda"), torch.full((O,), 7.0, dtype=T[t], device="cuda")
        rc = lib.fdx_linear8_weight_grad(h.h, dt, a.data_ptr(), b.data_ptr(), p.exponents.data_ptr(), N, O, I, dt, dw.data_ptr(), db.data_ptr(), ws.data_ptr(),
                                         n.value, _lib.stream_ptr(x.device))
        assert rc == 0
        x8, d = fda.unpack8(p).double(), dy.double()
        u = torch.finfo(T[t]).eps / 2
        for got, ref, mag in ((dw, d.T @ x8, d.abs().T @ x8.abs()), (db, d.sum(0), d.abs().sum(0))):
            lim = (N + 16) * E * mag * (1 + u) + u * ref.abs() + (2.0 ** -24 if t == "f16" else 2.0 ** -120)
            assert ((got.double() - ref).abs() <= lim).all()
    assert want[0].shape == (O, I)

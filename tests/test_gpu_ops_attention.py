"""GPU: attention and its backward pass against the formula in 64 bits.

Tolerances are elementwise bounds derived from the formula, u = eps / 2 of the type, e = 2^-24 (fp32 arithmetic inside every kernel):
  score error      |ds| <= (D + 4) e scale |q|.|k|  (D products and sums, scale, the two operations of the exponent)  =>  p off by 2 max|ds| relative
  out              u (P|v|)  [P rounded to the operand type; fp32: e]  + u |o|  [result]  + e (2 S + Tk + 16) (P|v|)      S = max (D + 4) scale |q|.|k|
  dv               the same with P^T|do|
  dS               P (dP - delta), delta from the out that the forward returned (off by its tolerance): P (|do|.tol(out) + e (D + 16) (|do||v|^T + |do|.|o|)) + (u + e (2 S + 16)) |dS|
  dq, dk           scale (tol(dS) |k|), plus the sum's own e (n + 16) scale |dS||k|, plus u |dq|
"""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def u_of(t):
    return torch.finfo(t).eps / 2


def reference(q, k, v, do, mask, causal, scale):
    """out, dq, dk, dv, lse and their tolerances, in float64 on the device."""
    t, u = q.dtype, u_of(q.dtype)
    B, H, Tq, D = q.shape
    Hkv, Tk = k.shape[1:3]
    G = H // Hkv
    hidden = torch.zeros(B, 1, Tq, Tk, dtype=torch.bool, device=q.device)
    if mask is not None:
        hidden = hidden | mask.bool()[:, None, None, :]
    if causal:
        hidden = hidden | (torch.arange(Tk, device=q.device)[None, :] > torch.arange(Tq, device=q.device)[:, None] + Tk - Tq)
    seen_key = (~hidden).any(2)[..., None]                      # [B, 1, Tk, 1]
    seen_row = (~hidden).any(3)[..., None]                      # [B, 1, Tq, 1]
    z = lambda x, keep: torch.where(keep, x.double(), torch.zeros((), dtype=torch.float64, device=q.device))   # noqa: E731
    q, k, v, do = z(q, seen_row), z(k, seen_key), z(v, seen_key), z(do, seen_row)
    kk, vv = (x.repeat_interleave(G, 1) for x in (k, v))
    s = (q @ kk.transpose(-1, -2).contiguous()) * scale
    s = s.masked_fill(hidden, -math.inf)
    lse = torch.logsumexp(s, -1, keepdim=True) if Tk else torch.full((B, H, Tq, 1), -math.inf, dtype=torch.float64, device=q.device)
    p = torch.where(seen_row & ~hidden, torch.exp(s - lse), torch.zeros_like(s))
    S = float((q.abs() @ kk.abs().transpose(-1, -2).contiguous()).max()) * scale * (D + 4) if s.numel() else 0.0
    o = p @ vv
    av, ado = p @ vv.abs(), do.abs()
    tol = {"out": (u + E * (2 * S + Tk + 16)) * av + u * o.abs(), "lse": E * (S + Tk + 16 + lse.abs().nan_to_num(posinf=0.0))}
    fold = lambda x: x.view(B, Hkv, G, Tk, D).sum(2)            # noqa: E731
    pt = p.transpose(-1, -2).contiguous()
    dv, adv = fold(pt @ do), fold(pt @ ado)
    R = G * Tq
    tol["dv"] = (u + E * (2 * S + R + 16)) * adv + u * dv.abs()
    dp = do @ vv.transpose(-1, -2).contiguous()
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    wob = (ado * tol["out"]).sum(-1, keepdim=True) + E * (D + 16) * (ado @ vv.abs().transpose(-1, -2).contiguous() + (ado * o.abs()).sum(-1, keepdim=True))
    tds = p * wob + (u + E * (2 * S + 16)) * ds.abs()
    dq, dk = scale * (ds @ kk), scale * fold(ds.transpose(-1, -2).contiguous() @ q)
    tol["dq"] = scale * ((tds + E * (Tk + 16) * ds.abs()) @ kk.abs()) + u * dq.abs()
    tol["dk"] = scale * fold((tds + E * (R + 16) * ds.abs()).transpose(-1, -2).contiguous() @ q.abs()) + u * dk.abs()
    tiny = 2.0 ** -24 if t == torch.float16 else 2.0 ** -126    # below the type's smallest normal number: half its step (fp16 2^-25)
    for n in ("out", "dq", "dk", "dv"):
        tol[n] = tol[n] + tiny
    return {"out": o, "lse": lse[..., 0], "dq": dq, "dk": dk, "dv": dv}, dict(tol, lse=tol["lse"][..., 0])


def inputs(t, B, H, Hkv, Tq, Tk, D, layout="bthd", seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * Tq + Tk)

    def one(heads, length):
        if layout == "bthd":
            return torch.randn(B, length, heads, D, generator=g, device="cuda").to(t).transpose(1, 2)
        if layout == "bhtd":
            return torch.randn(B, heads, length, D, generator=g, device="cuda").to(t)
        return torch.randn(B, heads, D, length, generator=g, device="cuda").to(t).transpose(2, 3)    # channels not contiguous
    return one(H, Tq), one(Hkv, Tk), one(Hkv, Tk), one(H, Tq)


def mask_of(kind, B, Tk):
    if kind == "none":
        return None
    g = torch.Generator().manual_seed(Tk)
    if kind == "pad":
        lens = torch.randint(1, Tk + 1, (B,), generator=g)
        m = torch.arange(Tk)[None, :] >= lens[:, None]
    elif kind == "holes":
        m = torch.rand(B, Tk, generator=g) < 0.5
    else:                                   # "empty": the first item has no key left
        m = torch.rand(B, Tk, generator=g) < 0.3
        m[0] = True
    return m.cuda()


def check(got, want, tol, names):
    for n in names:
        a, b = got[n].double(), want[n]
        assert a.shape == b.shape, n
        same_inf = torch.isinf(b) & (a == b)
        bad = ~same_inf & ~((a - b).abs() <= tol[n])
        assert not bad.any(), f"{n}: {int(bad.sum())} of {bad.numel()} off, worst {float(((a - b).abs() / tol[n])[bad].nan_to_num(nan=1e30).max()):.3g} times its bound"


def both(q, k, v, do, mask=None, causal=False, scale=None):
    import fish_diffusion_amd as fda
    out, lse = fda.attention_forward(q, k, v, mask, causal, scale)
    dq, dk, dv = fda.attention_backward(do, q, k, v, out, lse, mask, causal, scale)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


ALL = ("out", "lse", "dq", "dk", "dv")

SHAPES = [   # B, H, Hkv, Tq, Tk, D
    (1, 1, 1, 1, 1, 8), (2, 4, 2, 1, 300, 64), (1, 8, 1, 1, 1500, 128), (3, 2, 2, 37, 37, 32), (2, 6, 2, 33, 129, 80), (1, 4, 4, 130, 31, 16),
    (2, 4, 1, 50, 65, 128), (1, 2, 1, 700, 3, 64), (2, 8, 8, 86, 86, 64),
]


@pytest.mark.parametrize("t", list(T))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("causal,kind", [(False, "none"), (False, "holes"), (True, "none"), (True, "pad"), (False, "empty")])
def test_attention_and_gradients(t, shape, causal, kind):
    B, H, Hkv, Tq, Tk, D = shape
    q, k, v, do = inputs(T[t], *shape)
    mask = mask_of(kind, B, Tk)
    want, tol = reference(q, k, v, do, mask, causal, D ** -0.5)
    check(both(q, k, v, do, mask, causal), want, tol, ALL)


# the 128-row form (more than 1024 tiles of 32 rows), its split form, and both for the keys of dk / dv
@pytest.mark.parametrize("t,shape,causal", [
    ("f32", (8, 16, 16, 290, 300, 64), False), ("bf16", (8, 16, 16, 290, 300, 64), True), ("f16", (8, 16, 4, 290, 310, 128), True), ("f32", (9, 20, 4, 270, 270, 128), True),
    ("bf16", (1, 1, 1, 34000, 300, 32), False), ("f32", (1, 1, 1, 300, 34000, 32), False), ("bf16", (1, 4, 1, 8500, 260, 128), True), ("f16", (40, 16, 16, 60, 60, 40), True),
    ("f32", (8, 8, 8, 300, 300, 64), False), ("bf16", (8, 8, 8, 300, 300, 64), True), ("f16", (8, 8, 4, 290, 310, 128), True),
    ("f32", (2, 40, 8, 270, 333, 128), True), ("bf16", (1, 1, 1, 20000, 300, 32), False), ("f32", (1, 1, 1, 300, 20000, 32), False),
    ("f16", (1, 2, 2, 1100, 9000, 64), False), ("bf16", (1, 4, 1, 4400, 260, 128), True)], ids=str)
def test_wide_and_split_forms(t, shape, causal):
    q, k, v, do = inputs(T[t], *shape)
    mask = mask_of("pad", shape[0], shape[4])
    want, tol = reference(q, k, v, do, mask, causal, shape[5] ** -0.5)
    check(both(q, k, v, do, mask, causal), want, tol, ALL)


@pytest.mark.parametrize("t", list(T))
@pytest.mark.parametrize("layout", ["bhtd", "bhdt"])
def test_layouts_and_misaligned_views(t, layout):
    q, k, v, do = inputs(T[t], 2, 4, 2, 45, 70, 64, layout)
    want, tol = reference(q, k, v, do, None, False, 0.3)
    check(both(q, k, v, do, scale=0.3), want, tol, ALL)
    base = torch.zeros(2, 45, 4 * 64 + 3, dtype=T[t], device="cuda")      # rows that start at odd addresses
    odd = base[:, :, 1:257].view(2, 45, 4, 64).transpose(1, 2)
    odd.copy_(q)
    check(both(odd, k, v, do, scale=0.3), want, tol, ALL)
    one = v[:, :, :1].expand(-1, -1, 70, -1)                               # a broadcast value
    want, tol = reference(q, k, one, do, None, False, 0.3)
    check(both(q, k, one, do, scale=0.3), want, tol, ALL)


@pytest.mark.parametrize("t", list(T))
@pytest.mark.parametrize("shape", [(2, 4, 2, 40, 70, 64), (8, 8, 8, 300, 300, 64)], ids=str)
def test_what_masked_places_hold_never_matters(t, shape):
    B, H, Hkv, Tq, Tk, D = shape
    q, k, v, do = inputs(T[t], *shape)
    mask = mask_of("empty", B, Tk)
    clean = both(q, k, v, do, mask)
    for junk in (float("nan"), float("inf"), torch.finfo(T[t]).min):
        k2, v2, q2, do2 = (x.clone() for x in (k, v, q, do))
        k2.masked_fill_(mask[:, None, :, None], junk)
        v2.masked_fill_(mask[:, None, :, None], junk)
        q2[0], do2[0] = junk, junk                                         # every row of item 0 sees nothing
        got = both(q2, k2, v2, do2, mask)
        for n in ALL:
            assert torch.equal(got[n], clean[n]), n
    assert (clean["out"][0] == 0).all() and (clean["lse"][0] == -math.inf).all() and (clean["dq"][0] == 0).all()
    assert (clean["dk"].masked_select(mask[:, None, :, None]) == 0).all() and (clean["dv"].masked_select(mask[:, None, :, None]) == 0).all()


def test_causal_rows_before_the_first_key_are_empty():
    q, k, v, do = inputs(torch.float32, 1, 2, 2, 90, 40, 32)
    got = both(q, k, v, do, causal=True)
    want, tol = reference(q, k, v, do, None, True, 32 ** -0.5)
    check(got, want, tol, ALL)
    assert (got["out"][:, :, :50] == 0).all() and (got["lse"][:, :, :50] == -math.inf).all()


def test_lengths_of_zero():
    import fish_diffusion_amd as fda
    for B, Tq, Tk in ((0, 5, 5), (2, 0, 7), (2, 7, 0), (1, 0, 0)):
        q, k, v, do = inputs(torch.bfloat16, B, 4, 2, Tq, Tk, 32)
        r = both(q, k, v, do)
        assert r["out"].shape == q.shape and r["dk"].shape == k.shape
        for n in ("out", "dq", "dk", "dv"):
            assert (r[n] == 0).all(), n
        assert (r["lse"] == -math.inf).all()
    assert fda.attention(torch.zeros(1, 1, 0, 8, device="cuda"), *[torch.zeros(1, 1, 3, 8, device="cuda")] * 2).shape == (1, 1, 0, 8)


@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_small_gradients_keep_their_digits(t):
    """grad_out of 2^-12 makes dS far smaller than fp16's normal numbers; the result scales exactly (powers of two) with grad_out where it is itself
    a normal number, and stays within the bound."""
    q, k, v, do = inputs(T[t], 1, 2, 2, 200, 400, 64)
    s = 2.0 ** -12
    want, tol = reference(q, k, v, do * s, None, False, 0.125)
    check(both(q, k, v, do * s), want, tol, ALL)


def test_far_strides():
    """Rows more than 2^31 elements apart."""
    Tk, D, step = 40, 64, 1 << 26
    k = torch.empty((Tk - 1) * step + D, dtype=torch.bfloat16, device="cuda").as_strided((1, 1, Tk, D), (0, 0, step, 1))
    q, kc, v, do = inputs(torch.bfloat16, 1, 2, 1, 10, Tk, D)
    k.copy_(kc)
    want, tol = reference(q, kc, v, do, None, False, 0.125)
    check(both(q, k, v, do), want, tol, ALL)


def test_same_bits_every_time_and_on_another_stream():
    q, k, v, do = inputs(torch.bfloat16, 2, 8, 2, 300, 700, 64)
    a = both(q, k, v, do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = both(q, k, v, do)
    torch.cuda.current_stream().wait_stream(side)
    for n in ALL:
        assert torch.equal(a[n], b[n]), n


def test_captured_and_replayed():
    q, k, v, do = inputs(torch.float32, 1, 4, 2, 70, 900, 64)
    both(q, k, v, do)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = both(q, k, v, do)
    for seed in range(3):
        q2, k2, v2, do2 = inputs(torch.float32, 1, 4, 2, 70, 900, 64, seed=seed + 5)
        want = both(q2, k2, v2, do2)
        for dst, src in zip((q, k, v, do), (q2, k2, v2, do2)):
            dst.copy_(src)
        g.replay()
        torch.cuda.synchronize()
        for n in ALL:
            assert torch.equal(r[n], want[n]), (n, seed)


def test_autograd_matches_the_calls_and_differences():
    import fish_diffusion_amd as fda
    q, k, v, do = (x.detach().clone() for x in inputs(torch.float32, 1, 2, 1, 9, 13, 16))
    ref = both(q, k, v, do, causal=True)
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    out = fda.attention(q, k, v, causal=True)
    out.backward(do)
    for x, n in ((q, "dq"), (k, "dk"), (v, "dv")):
        assert torch.equal(x.grad, ref[n]), n
    # differences of the formula in 64 bits along random directions: (f(x + h d) - f(x - h d)) / 2h with h = 2^-10 is off by O(h^2) = 1e-6
    f = lambda a, b, c: float((reference(a, b, c, do, None, True, 0.25)[0]["out"] * do.double()).sum())   # noqa: E731
    g = torch.Generator(device="cuda").manual_seed(3)
    for i, n in enumerate(("dq", "dk", "dv")):
        x = [q.detach().double(), k.detach().double(), v.detach().double()]
        d = torch.randn(x[i].shape, generator=g, device="cuda", dtype=torch.float64)
        hi, lo = list(x), list(x)
        hi[i], lo[i] = x[i] + 2.0 ** -10 * d, x[i] - 2.0 ** -10 * d
        num = (f(*hi) - f(*lo)) * 2.0 ** 9
        assert abs(num - float((ref[n].double() * d).sum())) < 1e-4 * max(1.0, float(d.norm()))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(fda.attention(q, k, v).sum(), q, create_graph=True)[0].sum().backward()


def test_capture_with_a_live_eager_graph_is_refused():
    import fish_diffusion_amd as fda
    q, k, v, _ = (x.detach().clone().requires_grad_() for x in inputs(torch.float32, 1, 2, 2, 20, 20, 32))
    kept = fda.attention(q, k, v)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="outside this capture"):
            fda.attention(q, k, v)
        with pytest.raises(RuntimeError, match="outside this capture"):
            fda.attention(q * 2, k, v)
        r = fda.attention_forward(q, k, v)[0]
    g.replay()
    assert torch.equal(r, kept.detach())


def test_refusals_on_the_device():
    import fish_diffusion_amd as fda
    from fish_diffusion_amd import _lib
    q, k, v, do = inputs(torch.float32, 1, 2, 2, 8, 8, 32)
    with pytest.raises(ValueError):
        fda.attention_forward(q, k.half(), v)
    with pytest.raises((ValueError, RuntimeError)):
        fda.attention_forward(q, k.cpu(), v)
    with pytest.raises(ValueError):
        fda.attention_forward(q, k, v, key_mask=torch.zeros(1, 8, dtype=torch.bool))
    out, lse = fda.attention_forward(q, k, v)
    with pytest.raises(ValueError):
        fda.attention_backward(do[:, :, :4], q, k, v, out, lse)
    with pytest.raises(ValueError):
        fda.attention_backward(do, q, k, v, out, lse.double())
    # the C entry: a workspace that is too small, a misaligned pointer
    import ctypes as C
    desc = _lib.AttnDesc(0, 1, 2, 2, 8, 8, 32, 0, 1.0)
    h = _lib.Handle.shared(q.device)
    b = lambda t, shift=0: C.byref(_lib.Bht(t.data_ptr() + shift, t.stride(0), t.stride(1), t.stride(2)))   # noqa: E731
    lib, st = _lib.lib(), _lib.stream_ptr(q.device)
    assert lib.fdx_attn_forward(h.h, C.byref(desc), b(q, 4), b(k), b(v), None, b(out), _lib.ptr(lse), None, 0, st) == -1
    assert lib.fdx_attn_backward(h.h, C.byref(desc), b(do), b(q), b(k), b(v), b(out), _lib.ptr(lse), None, b(q), b(k), b(v), None, 0, st) == -1
    assert b"workspace" in lib.fdx_last_error(h.h)


def test_c_entries_refuse_strides_and_workspaces():
    import ctypes as C
    from fish_diffusion_amd import _lib
    q, k, v, do = inputs(torch.float32, 2, 2, 2, 8, 8, 32)
    out, lse, ws = torch.empty_like(q), torch.empty(2, 2, 8, device="cuda"), torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    desc, h, lib, st = _lib.AttnDesc(0, 2, 2, 2, 8, 8, 32, 0, 1.0), _lib.Handle.shared(q.device), _lib.lib(), _lib.stream_ptr(q.device)

    def bht(x, **strides):
        s = dict(b=x.stride(0), h=x.stride(1), t=x.stride(2))
        s.update(strides)
        return C.byref(_lib.Bht(x.data_ptr(), s["b"], s["h"], s["t"]))

    def forward(q=bht(q), out=bht(out), at=0):
        return lib.fdx_attn_forward(h.h, C.byref(desc), q, bht(k), bht(v), None, out, _lib.ptr(lse), ws.data_ptr() + at, ws.numel() - at, st)

    def backward(dk=bht(do), at=0):
        return lib.fdx_attn_backward(h.h, C.byref(desc), bht(do), bht(q), bht(k), bht(v), bht(out), _lib.ptr(lse), None, bht(do), dk, bht(do), ws.data_ptr() + at,
                                     ws.numel() - at, st)

    for bad in (dict(b=-512), dict(h=-256), dict(t=-32)):
        assert forward(q=bht(q, **bad)) == -1 and b"negative" in lib.fdx_last_error(h.h)
        assert backward(dk=bht(k, **bad)) == -1
    for bad in (dict(b=0), dict(h=0), dict(t=0)):
        assert forward(out=bht(out, **bad)) == -1 and b"overlap" in lib.fdx_last_error(h.h)
        assert backward(dk=bht(k, **bad)) == -1
    assert forward(at=4) == -1 and backward(at=4) == -1 and b"aligned" in lib.fdx_last_error(h.h)
    assert forward(q=bht(q, h=0)) == 0          # a repeated head is an input like any other
    torch.cuda.synchronize()
    want = torch.softmax((q[:, :1].double() @ k.double().transpose(-1, -2)), -1) @ v.double()
    assert (out.double() - want).abs().max() < 1e-3     # scores of up to 60 in sums of 32 products: 33 * 60 * 2^-24 = 1.2e-4 of P, |v| <= 4


@pytest.mark.parametrize("t", list(T))
@pytest.mark.parametrize("shape", [(2, 4, 2, 300, 1, 32), (1, 8, 8, 17, 1, 64), (2, 4, 4, 40, 700, 128), (16, 40, 40, 70, 5, 40)], ids=str)
def test_rows_of_one_key(t, shape):
    """One visible key: out is its value, dq and dk are exactly 0 (P = 1 whatever the score), dv the sum of grad_out."""
    import fish_diffusion_amd as fda
    q, k, v, do = inputs(T[t], *shape)
    B, H, Hkv, Tq, Tk, D = shape
    mask = torch.ones(B, Tk, dtype=torch.bool, device="cuda")
    only = [(5 * b + 1) % Tk for b in range(B)]
    for b, i in enumerate(only):
        mask[b, i] = False
    out, lse = fda.attention_forward(q, k, v, mask)
    dq, dk, dv = fda.attention_backward(do, q, k, v, out, lse, mask)
    at = torch.tensor(only, device="cuda")[:, None, None, None].expand(B, Hkv, 1, D)
    assert torch.equal(out, v.gather(2, at).repeat_interleave(H // Hkv, 1).expand_as(out))
    assert not dq.any() and not dk.any()
    assert not dv.masked_fill(~mask[:, None, :, None], 0).any()
    assert dv.any()

"""What the training operators of the framework are measured on: attention with its backward pass, the fused norm / gate / residual
step with its backward pass, and 8-bit activation checkpoints with the gradients that are taken from them.

`own` False computes them in plain torch operations in 32 bits; True makes the framework's own calls."""
import math

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# --------------------------------------------------------------------------------------------------------------- cases
def _attn(name, t, B, H, Hkv, Tq, Tk, D, causal, fill, train):
    # fill: the shortest item's share of valid keys (1.0: no padding mask); the items of a batch are spread between it and 1
    c = {"op": "attention", "dtype": t, "B": B, "H": H, "Hkv": Hkv, "Tq": Tq, "Tk": Tk, "D": D, "causal": causal, "fill": fill, "train": train}
    return dict(c, name=name) if name else c


def _norm(name, t, B, T, C, gate, post, pre, kind, train):
    # gate: "none" | "channel" ([C]) | "item" ([B, C]) | "full" ([B, T, C])
    c = {"op": "norm", "dtype": t, "B": B, "T": T, "C": C, "gate": gate, "post": post, "pre": pre, "kind": kind, "train": train}
    return dict(c, name=name) if name else c


def _pack(name, t, what, N, O, I):
    # what: "restore" (pack and read back), "linear" (a linear layer's checkpoint and the weight gradient from it), "gelu"
    c = {"op": "pack8", "dtype": t, "what": what, "N": N, "O": O, "I": I}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new token of eight long sequences against their caches, grouped heads: the serving form, bound by reading K and V
        _attn("attn_token_bf16", "bf16", 8, 32, 8, 1, 8192, 128, False, 0.6, False),
        # a short clip through one layer of the transformer denoiser (8 heads x 64): the call where latency counts
        _attn("attn_short_f32", "f32", 1, 8, 8, 86, 86, 64, False, 1.0, False),
        # 10 s of audio (861 frames), padded batch of eight, one layer of the transformer denoiser, forward and backward
        _attn("attn_train_f32", "f32", 8, 8, 8, 861, 861, 64, False, 0.6, True),
        # long sequences, causal, grouped heads, mixed precision: the largest
        _attn("attn_train_long_bf16", "bf16", 2, 16, 4, 4096, 4096, 128, True, 1.0, True),
        # cross attention from many frames to a short odd memory, narrow heads
        _attn("attn_cross_train_f16", "f16", 16, 8, 8, 861, 63, 32, False, 0.5, True),
        # the post-norm step x = norm(x + block) of one 5 s utterance: the smallest
        _norm("norm_short_f32", "f32", 1, 430, 512, "none", False, True, "layer", False),
        # the same step in training, batch of sixteen 10 s utterances, a learned scale per channel
        _norm("norm_train_f32", "f32", 16, 861, 512, "channel", False, True, "layer", True),
        # both norms around a wide block with a gate per item, mixed precision, forward and backward: the largest
        _norm("norm_train_wide_bf16", "bf16", 8, 2048, 2048, "item", True, True, "rms", True),
        # the input of one linear layer kept in 8 bits and read back
        _pack("pack8_restore_f32", "f32", "restore", 861, 1, 512),
        # weight and bias gradient of the MLP's first layer from the 8-bit input, batch of eight, fp32 gradients
        _pack("pack8_linear_f32", "f32", "linear", 8 * 861, 2048, 512),
        # the MLP's second layer in mixed precision, batch of 32
        _pack("pack8_linear_bf16", "bf16", "linear", 32 * 861, 512, 2048),
        # GELU kept in 8 bits: forward and backward, batch of eight
        _pack("pack8_gelu_bf16", "bf16", "gelu", 8 * 861, 1, 2048),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "norm", "pack8"])
    t = rng.choice(["f32", "bf16", "f16"])
    if op == "attention":
        while True:
            B, Hkv, G = _log(rng, 1, 16), rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4])
            D = rng.choice([16, 32, 64, 80, 128])
            mode = rng.choice(["token", "self", "cross"])
            Tk = _log(rng, 1, 8192)
            Tq = 1 if mode == "token" else Tk if mode == "self" else _log(rng, 1, 4096)
            causal = mode == "self" and rng.random() < 0.5
            train = mode != "token"
            fill = rng.choice([1.0, round(rng.uniform(0.2, 1.0), 2)])
            # no dearer than the listed cases: 14 flops per (query, key, channel) of the long one, and the token case's cache;
            # the products of fp32 cost the plain and the built form sixteen times those of 16 bits
            pairs = B * Hkv * G * Tq * Tk * D
            limit = 2 * 16 * 4096 * 4096 * 128 // (8 if t == "f32" else 2)
            if pairs <= limit and B * Hkv * Tk * D <= 8 * 8 * 8192 * 128 and B * Hkv * G * Tq * D <= 2 ** 25:
                return _attn(None, t, B, Hkv * G, Hkv, Tq, Tk, D, causal, fill, train)
    if op == "norm":
        while True:
            B, T = _log(rng, 1, 16), _log(rng, 1, 4096)
            C = rng.choice([_log(rng, 32, 4096), 8 * _log(rng, 4, 512), 512])
            if B * T * C <= 8 * 2048 * 2048:
                post, pre = rng.choice([(False, True), (True, True), (True, False)])
                return _norm(None, t, B, T, C, rng.choice(["none", "channel", "item", "full"]), post, pre, rng.choice(["layer", "rms"]), rng.random() < 0.7)
    what = rng.choice(["restore", "linear", "gelu"])
    while True:
        N = _log(rng, 1, 27552)
        O, I = (_log(rng, 8, 4096), _log(rng, 8, 4096)) if what == "linear" else (1, _log(rng, 8, 4096))
        if N * O * I <= 27552 * 512 * 2048 // (4 if t == "f32" else 1) and N * I <= 27552 * 2048:
            return _pack(None, t, what, N, O, I)


# --------------------------------------------------------------------------------------------------------------- inputs
def _lens(c):
    # valid keys of every item: spread evenly from fill * Tk to Tk, one at least
    B, Tk = c["B"], c["Tk"]
    return [max(1, int(round(Tk * (c["fill"] + (1.0 - c["fill"]) * (b + 1) / B)))) for b in range(B)]


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = DT[c["dtype"]]

    def rn(*shape, s=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * s).to(t)

    st = {"case": c}
    if c["op"] == "attention":
        B, H, Hkv, Tq, Tk, D = (c[n] for n in ("B", "H", "Hkv", "Tq", "Tk", "D"))
        # [B, T, H, D] as projections leave them, seen as [B, H, T, D]
        st["q"] = rn(B, Tq, H, D).transpose(1, 2)
        st["k"] = rn(B, Tk, Hkv, D).transpose(1, 2)
        st["v"] = rn(B, Tk, Hkv, D).transpose(1, 2)
        if c["train"]:
            st["do"] = rn(B, Tq, H, D).transpose(1, 2)
        st["mask"] = None
        if c["fill"] < 1.0:
            st["mask"] = torch.arange(Tk, device="cuda")[None, :] >= torch.tensor(_lens(c), device="cuda")[:, None]   # True = padding
    elif c["op"] == "norm":
        B, T, C = c["B"], c["T"], c["C"]
        st["x"], st["block"] = rn(B, T, C, s=2.0), rn(B, T, C) + torch.randn(C, generator=g, device="cuda").to(t) * 0.5
        shape = {"none": None, "channel": (C,), "item": (B, C), "full": (B, T, C)}[c["gate"]]
        st["gate"] = None if shape is None else (0.5 + 0.5 * torch.randn(*shape, generator=g, device="cuda")).to(t)
        st["scale"] = 1.0 if c["gate"] == "none" else 0.9

        def wb():
            w = (1.0 + 0.2 * torch.randn(C, generator=g, device="cuda")).to(t)
            return (w, (0.1 * torch.randn(C, generator=g, device="cuda")).to(t) if c["kind"] == "layer" else None)
        st["post"] = wb() if c["post"] else None
        st["pre"] = wb() if c["pre"] else None
        if c["train"]:
            st["gh"] = rn(B, T, C)
            st["gy"] = rn(B, T, C) if c["pre"] else None
    else:
        N, O, I = c["N"], c["O"], c["I"]
        # activations behind a norm: unit scale, channels of unlike magnitude
        st["x"] = (torch.randn(N, I, generator=g, device="cuda") * torch.exp(0.5 * torch.randn(I, generator=g, device="cuda"))).to(t)
        if c["what"] == "linear":
            st["dy"] = rn(N, O, s=0.1)
        if c["what"] == "gelu":
            st["dy"] = rn(N, I, s=0.1)
    return st


# --------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(st):
    import fish_diffusion_amd as fda
    c = st["case"]
    if c["op"] == "attention":
        kw = {"key_mask": st["mask"], "causal": c["causal"]}
        out, lse = fda.attention_forward(st["q"], st["k"], st["v"], **kw)
        if not c["train"]:
            return {"out": out}
        dq, dk, dv = fda.attention_backward(st["do"], st["q"], st["k"], st["v"], out, lse, **kw)
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    if c["op"] == "norm":
        kw = {"gate": st["gate"], "residual_scale": st["scale"], "post_norm": st["post"], "pre_norm": st["pre"], "kind": c["kind"]}
        h, y, stats = fda.residual_norm_forward(st["x"], st["block"], **kw)
        r = {"h": h, "y": y}
        if c["train"]:
            r.update(fda.residual_norm_backward(st["gh"], st["gy"], st["x"], st["block"], stats, **kw)._asdict())
        return {k: v for k, v in r.items() if v is not None}
    if c["what"] == "restore":
        return {"x8": fda.unpack8(fda.pack8(st["x"]), torch.float32)}
    if c["what"] == "linear":
        dw, db = fda.linear8_weight_grad(st["dy"], fda.pack8(st["x"]))
        return {"dw": dw, "db": db}
    y, kept = fda.gelu8_forward(st["x"])
    return {"y": y, "dx": fda.gelu8_backward(st["dy"], kept)}


def _plain_restore(x):
    # groups of 32 channels share a power of two: the smallest 2^k with max|x| <= 127 * 2^k, k >= -126
    N, C = x.shape
    x = x.float()
    G = (C + 31) // 32
    p = torch.zeros(N, G * 32, device=x.device)
    p[:, :C] = x
    p = p.view(N, G, 32)
    m, e = torch.frexp(p.abs().amax(-1, keepdim=True))      # amax = m * 2^e, m in [0.5, 1)
    k = (e - 7 + (m > 127.0 / 128.0)).clamp(min=-126)
    k = torch.where(m == 0, torch.full_like(k, -126), k)
    one = torch.ones((), device=x.device)
    return (torch.round(p * torch.ldexp(one, -k)) * torch.ldexp(one, k)).view(N, G * 32)[:, :C]


def _plain_norm(v, wb, kind, eps=1e-5):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else 0.0
    r = 1.0 / torch.sqrt(((v - mean) * (v - mean)).mean(-1, keepdim=True) + eps)
    hat = (v - mean) * r
    y = hat * wb[0].float()
    return (y + wb[1].float() if wb[1] is not None else y), hat, r


def _plain_norm_grad(g, hat, r, wb, kind):
    gw = g * wb[0].float()
    d = gw - hat * (gw * hat).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - gw.mean(-1, keepdim=True)
    return d * r


def _run_plain(st):
    c = st["case"]
    t = DT[c["dtype"]]
    if c["op"] == "attention":
        B, H, Hkv, Tq, Tk, D = (c[n] for n in ("B", "H", "Hkv", "Tq", "Tk", "D"))
        G, a = H // Hkv, 1.0 / math.sqrt(D)
        q = st["q"].float().reshape(B, Hkv, G * Tq, D)
        k, v = st["k"].float().contiguous(), st["v"].float().contiguous()
        s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * a
        if st["mask"] is not None:
            s = torch.where(st["mask"][:, None, None, :], float("-inf"), s)
        if c["causal"]:
            i = torch.arange(Tq, device=s.device)[:, None] + (Tk - Tq)
            s = torch.where((torch.arange(Tk, device=s.device)[None, :] > i).repeat(G, 1)[None, None], float("-inf"), s)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        del s
        out = torch.matmul(p, v)
        r = {"out": out.view(B, H, Tq, D).to(t)}
        if c["train"]:
            do = st["do"].float().reshape(B, Hkv, G * Tq, D)
            r["dv"] = torch.matmul(p.transpose(-1, -2).contiguous(), do).to(t)
            dp = torch.matmul(do, v.transpose(-1, -2).contiguous())
            ds = p * (dp - (do * out).sum(-1, keepdim=True)) * a
            del dp, p
            r["dq"] = torch.matmul(ds, k).view(B, H, Tq, D).to(t)
            r["dk"] = torch.matmul(ds.transpose(-1, -2).contiguous(), q).to(t)
        return {n: r[n] for n in ("out", "dq", "dk", "dv") if n in r}
    if c["op"] == "norm":
        x, block, a = st["x"].float(), st["block"].float(), st["scale"]
        gate = None if st["gate"] is None else st["gate"].float()
        if c["gate"] == "item":
            gate = gate[:, None]
        n, bhat, br = _plain_norm(block, st["post"], c["kind"]) if c["post"] else (block, None, None)
        h = a * x + (n if gate is None else gate * n)
        r = {"h": h.to(t)}
        if c["pre"]:
            y, hhat, hr = _plain_norm(h, st["pre"], c["kind"])
            r["y"] = y.to(t)
        if c["train"]:
            dh = st["gh"].float()
            if c["pre"]:
                gy = st["gy"].float()
                dh = dh + _plain_norm_grad(gy, hhat, hr, st["pre"], c["kind"])
            r["dx"] = (a * dh).to(t)
            dn = dh if gate is None else gate * dh
            r["dblock"] = (_plain_norm_grad(dn, bhat, br, st["post"], c["kind"]) if c["post"] else dn).to(t)
            if gate is not None:
                dg = dh * n
                r["dgate"] = {"channel": lambda: dg.sum((0, 1)), "item": lambda: dg.sum(1), "full": lambda: dg}[c["gate"]]().to(t)
            if c["post"]:
                r["dpost_weight"] = (dn * bhat).sum((0, 1)).to(t)
                if st["post"][1] is not None:
                    r["dpost_bias"] = dn.sum((0, 1)).to(t)
            if c["pre"]:
                r["dpre_weight"] = (gy * hhat).sum((0, 1)).to(t)
                if st["pre"][1] is not None:
                    r["dpre_bias"] = gy.sum((0, 1)).to(t)
        return r
    x8 = _plain_restore(st["x"])
    if c["what"] == "restore":
        return {"x8": x8}
    if c["what"] == "linear":
        dy = st["dy"].float()
        return {"dw": torch.matmul(dy.t(), x8).to(t), "db": dy.sum(0).to(t)}
    x = st["x"].float()
    y = x * 0.5 * (1.0 + torch.erf(x * math.sqrt(0.5)))
    d = 0.5 * (1.0 + torch.erf(x8 * math.sqrt(0.5))) + x8 * torch.exp(-0.5 * x8 * x8) * (1.0 / math.sqrt(2.0 * math.pi))
    return {"y": y.to(t), "dx": (st["dy"].float() * d).to(t)}


# --------------------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    es = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "attention":
        B, H, Hkv, Tq, Tk, D = (c[n] for n in ("B", "H", "Hkv", "Tq", "Tk", "D"))
        lens = _lens(c) if c["fill"] < 1.0 else [Tk] * B
        pairs = 0
        for n in lens:
            if c["causal"]:                     # query i sees keys 0 .. i + Tk - Tq, of them the first n
                off = Tk - Tq
                full = max(0, Tq - max(0, n - 1 - off))            # queries that see all n
                part = Tq - full
                pairs += full * n + sum(max(0, min(n, i + off + 1)) for i in range(part))
            else:
                pairs += Tq * n
        kv = sum(lens) * Hkv * D
        nb = (2 * B * H * Tq * D + 2 * kv) * es + (B * Tk if c["fill"] < 1.0 else 0)
        fl = 4 * H * pairs * D
        if c["train"]:                          # q, k, v, do, out, row sums in; three gradients out; five products (the scores again)
            nb += (4 * B * H * Tq * D + 2 * kv + 2 * B * Hkv * Tk * D) * es + 8 * B * H * Tq
            fl += 10 * H * pairs * D
        return {"bytes": nb, "flops": fl}
    if c["op"] == "norm":
        n = c["B"] * c["T"] * c["C"]
        gfull = 1 if c["gate"] == "full" else 0
        units = 2 + 1 + (1 if c["pre"] else 0) + gfull
        fl = 10 * n
        if c["train"]:
            units += 2 + 1 + (1 if c["pre"] else 0) + 2 + 2 * gfull
            if c["gate"] == "none" and not c["post"]:
                units -= 1                      # dx and dblock are one tensor (the residual scale is 1)
            fl += 25 * n
        return {"bytes": units * n * es, "flops": fl}
    N, O, I = c["N"], c["O"], c["I"]
    codes = N * I + N * ((I + 31) // 32)
    if c["what"] == "restore":
        return {"bytes": N * I * es + 2 * codes + 4 * N * I, "flops": 4 * N * I}
    if c["what"] == "linear":
        return {"bytes": N * I * es + 2 * codes + N * O * es + O * I * es + O * es, "flops": 2 * N * O * I}
    return {"bytes": 2 * N * I * es + 2 * codes + 2 * N * I * es, "flops": 30 * N * I}


# --------------------------------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    c = case
    st = prepare(c, seed)
    d = torch.float64
    if c["op"] == "attention":
        B, H, Hkv, Tq, Tk, D = (c[n] for n in ("B", "H", "Hkv", "Tq", "Tk", "D"))
        G = H // Hkv
        names = ("out", "dq", "dk", "dv") if c["train"] else ("out",)
        res = {n: torch.zeros(B, Hkv if n in ("dk", "dv") else H, Tk if n in ("dk", "dv") else Tq, D, dtype=d, device="cuda") for n in names}
        lens = _lens(c) if st["mask"] is not None else [Tk] * B
        pos = torch.arange(Tq, device="cuda")[:, None] + (Tk - Tq)
        for b in range(B):
            n = lens[b]                         # the padding lies behind the valid keys: they alone exist
            hidden = torch.arange(n, device="cuda")[None, :] > pos if c["causal"] else None
            for h in range(H):
                k, v, q = st["k"][b, h // G, :n].to(d), st["v"][b, h // G, :n].to(d), st["q"][b, h].to(d)
                z = (q @ k.T) / math.sqrt(D)
                if hidden is not None:
                    z = z.masked_fill(hidden, -math.inf)
                w = torch.exp(z - torch.logsumexp(z, -1, keepdim=True))
                o = w @ v
                res["out"][b, h] = o
                if c["train"]:
                    go = st["do"][b, h].to(d)
                    res["dv"][b, h // G, :n] += w.T @ go
                    gz = w * (go @ v.T - (go * o).sum(-1, keepdim=True)) / math.sqrt(D)
                    res["dq"][b, h] = gz @ k
                    res["dk"][b, h // G, :n] += gz.T @ q
        return res
    if c["op"] == "norm":
        # the gradients are torch's own differentiation of the definition, in 64 bits
        def leaf(v):
            return None if v is None else v.to(d).requires_grad_(c["train"])
        x, block, gate = leaf(st["x"]), leaf(st["block"]), leaf(st["gate"])
        post = [leaf(v) for v in st["post"]] if c["post"] else None
        pre = [leaf(v) for v in st["pre"]] if c["pre"] else None

        def norm(v, wb):
            if c["kind"] == "layer":
                v = v - v.mean(-1, keepdim=True)
            v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5) * wb[0]
            return v if wb[1] is None else v + wb[1]
        n = norm(block, post) if post else block
        h = st["scale"] * x + (n if gate is None else (gate[:, None] if c["gate"] == "item" else gate) * n)
        y = norm(h, pre) if pre else None
        r = {"h": h, "y": y}
        if c["train"]:
            loss = (h * st["gh"].to(d)).sum() + ((y * st["gy"].to(d)).sum() if pre else 0.0)
            want = {"dx": x, "dblock": block, "dgate": gate, "dpost_weight": post and post[0], "dpost_bias": post and post[1],
                    "dpre_weight": pre and pre[0], "dpre_bias": pre and pre[1]}
            want = {k: v for k, v in want.items() if v is not None}
            r.update(zip(want, torch.autograd.grad(loss, list(want.values()))))
        return {k: v.detach() for k, v in r.items() if v is not None}
    # 8 bits: bracket the scale by powers of two in 64 bits
    x = st["x"].to(d)
    x8 = torch.empty_like(x)
    for j in range(0, x.shape[1], 32):
        part = x[:, j:j + 32]
        top = part.abs().amax(1, keepdim=True)
        k = torch.ceil(torch.log2(torch.clamp(top, min=2.0 ** -140) / 127.0)).clamp(min=-126.0)
        s = torch.exp2(k)
        s = torch.where(top > 127.0 * s, 2.0 * s, s)                       # log2 next to a power of two may fall either way
        s = torch.where((top <= 63.5 * s) & (s > 2.0 ** -126), 0.5 * s, s)
        x8[:, j:j + 32] = torch.round(part / s) * s
    if c["what"] == "restore":
        return {"x8": x8}
    dy = st["dy"].to(d)
    if c["what"] == "linear":
        return {"dw": dy.T @ x8, "db": dy.sum(0)}
    cdf = 0.5 * torch.erfc(-x8 / math.sqrt(2.0))
    return {"y": 0.5 * x * torch.erfc(-x / math.sqrt(2.0)), "dx": dy * (cdf + x8 * torch.exp(-x8 * x8 / 2.0) / math.sqrt(2.0 * math.pi))}

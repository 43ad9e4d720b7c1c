"""The operators of a Transformer training step around the table products, over the range of their sizes.

``norm``    residual_norm: the norm after a block, its gate and residual scale, the sum, and the norm before the next block.
``rotary``  rotary positions of queries and keys.
``adamw``   one AdamW step over all tensors of a model, moments in 32 bits or in 8.
``quant``   a matrix in 4-bit floats with a scale per 32 elements, along both axes, and back.
``dense``   a dense layer whose product is taken in those 4-bit floats; with ``train`` both gradients too.

With ``own`` false everything is computed by elementary torch operations in 32 bits (64 for the angles of far positions).
Sizes are those of ``TransformerAM`` (512 wide, 8 heads of 64, 64 x 128 tokens, 8000 words) and LeNet-5, and generic larger ones.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one token through "LayerNorm(x + block)" of TransformerAM: what the call costs
        dict(name="norm_infer_1x512", op="norm", kind="layer", batch=1, seq=1, width=512, dtype="f32", post=False, gate="none", both=False, train=False),
        # the same of a training batch, 64 sentences of 128 tokens, with its gradients
        dict(name="norm_train_8192x512", op="norm", kind="layer", batch=64, seq=128, width=512, dtype="f32", post=False, gate="none", both=False, train=True),
        # a larger model's block: RMS norms on both sides, a gate for each sequence, bf16 activations
        dict(name="norm_gated_train_16384x2048", op="norm", kind="rms", batch=8, seq=2048, width=2048, dtype="bf16", post=True, gate="sequence", both=True, train=True),
        # one new token for each of 64 sequences
        dict(name="rotary_decode_b64", op="rotary", batch=64, seq=1, heads=8, kv_heads=8, dim=64, rot=64, layout="half", scaling="none", start=100, dtype="f32", heads_first=False, train=False),
        # a long document at far positions: scaled frequencies, half of each head rotated, shared key heads
        dict(name="rotary_long_32768", op="rotary", batch=1, seq=32768, heads=32, kv_heads=8, dim=128, rot=64, layout="interleaved", scaling="blend", start=900000, dtype="bf16", heads_first=False, train=True),
        # LeNet-5: ten tensors, 62 thousand parameters
        dict(name="adamw_lenet5", op="adamw", model="lenet5", count=0, total=0, bits=32, dtype="f32", shift=0),
        # TransformerAM: 56 million parameters in 244 tensors
        dict(name="adamw_transformer", op="adamw", model="transformer", count=0, total=0, bits=32, dtype="f32", shift=0),
        dict(name="adamw_transformer_8bit", op="adamw", model="transformer", count=0, total=0, bits=8, dtype="f32", shift=0),
        # activations of the feed-forward layer's training step, along both axes
        dict(name="quant_both_8192x2048", op="quant", rows=8192, cols=2048, dtype="f32"),
        # 16 tokens through the vocabulary layer of TransformerAM
        dict(name="dense_infer_16x512x8000", op="dense", rows=16, inner=512, cols=8000, dtype="f32", train=False),
        # its feed-forward layer, forward and backward
        dict(name="dense_train_8192x512x2048", op="dense", rows=8192, inner=512, cols=2048, dtype="f32", train=True),
        # a layer of a large model in bf16
        dict(name="dense_infer_8192x8192x8192", op="dense", rows=8192, inner=8192, cols=8192, dtype="bf16", train=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "rotary", "rotary", "adamw", "adamw", "quant", "dense", "dense"])
    if op == "norm":
        width = _log(rng, 16, 8192)
        batch = _log(rng, 1, 64)
        seq = max(1, min(_log(rng, 1, 16384), 16384 * 2048 // (width * batch)))
        gate = rng.choice(["none", "width", "sequence", "full"])
        return dict(op=op, kind=rng.choice(["layer", "rms"]), batch=batch, seq=seq, width=width, dtype=rng.choice(["f32", "bf16", "f16"]),
                    post=rng.random() < 0.5, gate=gate, both=rng.random() < 0.5, train=rng.random() < 0.7)
    if op == "rotary":
        dim = rng.choice([32, 64, 80, 96, 128, 192, 256, rng.randrange(8, 257)])
        rot = rng.choice([dim // 2 * 2, 2 * rng.randrange(1, dim // 2 + 1)])
        kv = _log(rng, 1, 16)
        heads = kv * rng.choice([1, 2, 4])
        batch = _log(rng, 1, 64)
        seq = max(1, min(_log(rng, 1, 32768), 32768 * 40 * 128 // (batch * (heads + kv) * dim)))
        return dict(op=op, batch=batch, seq=seq, heads=heads, kv_heads=kv, dim=dim, rot=rot, layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "base", "blend"]), start=_log(rng, 1, 1000000), dtype=rng.choice(["f32", "bf16", "f16"]),
                    heads_first=rng.random() < 0.5, train=rng.random() < 0.5)
    if op == "adamw":
        return dict(op=op, model="drawn", count=_log(rng, 1, 300), total=_log(rng, 1000, 40000000), bits=rng.choice([8, 32]),
                    dtype=rng.choice(["f32", "f32", "bf16"]), shift=rng.randrange(0, 4))
    if op == "quant":
        rows = _log(rng, 1, 16384)
        return dict(op=op, rows=rows, cols=min(_log(rng, 1, 16384), max(1, 8192 * 4096 // rows)), dtype=rng.choice(["f32", "bf16", "f16"]))
    train = rng.random() < 0.5
    return dict(op=op, rows=_log(rng, 1, 8192), inner=_log(rng, 32, 4096 if train else 8192), cols=_log(rng, 16, 4096 if train else 8192),
                dtype=rng.choice(["f32", "bf16"]), train=train)


# ---- inputs -------------------------------------------------------------------------------------------
def _transformer(layers=6, d=512, ff=2048, vocab=8000):
    att = [(d, d), (d,)] * 4
    norm, ffn = [(d,), (d,)], [(d, ff), (ff,), (ff, d), (d,)]
    return [(vocab, d)] * 2 + (att + norm + ffn + norm) * layers + (att + norm + att + ffn + norm) * layers + [(d, vocab), (vocab,)]


_LENET5 = [(5, 5, 1, 6), (6,), (5, 5, 6, 16), (16,), (400, 120), (120,), (120, 84), (84,), (84, 10), (10,)]


def _sizes(case):
    if case["model"] != "drawn":
        return [math.prod(s) for s in (_LENET5 if case["model"] == "lenet5" else _transformer())]
    n, total, sizes, x = case["count"], case["total"], [], 12345
    for i in range(n):
        x = (x * 1103515245 + 12345 + case["total"]) % (1 << 31)
        sizes.append(math.exp(6.0 * x / (1 << 31)))
    k = total / sum(sizes)
    return [max(1, int(s * k)) for s in sizes]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    s = dict(case=case, seed=seed)
    if case["op"] == "norm":
        t, b, n, d = _DT[case["dtype"]], case["batch"], case["seq"], case["width"]
        s["x"] = normal(b, n, d, dtype=t)
        s["block"] = normal(b, n, d, dtype=t, scale=0.7) + 0.1
        shape = {"none": None, "width": (d,), "sequence": (b, 1, d), "full": (b, n, d)}[case["gate"]]
        s["gate"] = normal(*shape, dtype=torch.float32 if case["gate"] == "width" else t, scale=0.5) if shape else None
        s["scale"] = 1.0 if case["gate"] == "none" else 0.5
        s["eps"] = 1e-3 if case["kind"] == "layer" else 1e-5
        s["pre_w"] = 1 + normal(d, scale=0.1)
        s["pre_b"] = normal(d, scale=0.1) if case["kind"] == "layer" else None
        s["post_w"] = 1 + normal(d, scale=0.1) if case["post"] else None
        s["post_b"] = normal(d, scale=0.1) if case["post"] and case["kind"] == "layer" else None
        s["dy"] = normal(b, n, d, dtype=t, scale=0.01) if case["train"] else None
        s["dr"] = normal(b, n, d, dtype=t, scale=0.01) if case["train"] and case["both"] else None
        for k in ("x", "block", "gate", "pre_w", "pre_b", "post_w", "post_b"):
            if case["train"] and s[k] is not None:
                s[k].requires_grad_()
    elif case["op"] == "rotary":
        t, b, n, d = _DT[case["dtype"]], case["batch"], case["seq"], case["dim"]

        def heads(h):
            return normal(b, h, n, d, dtype=t).transpose(1, 2) if case["heads_first"] else normal(b, n, h, d, dtype=t)
        s["q"], s["k"] = heads(case["heads"]), heads(case["kv_heads"])
        first = torch.randint(0, case["start"], (b, 1), generator=gen, device="cuda")
        s["positions"] = first + torch.arange(n, device="cuda")
        s["scaled"] = dict(none={}, linear=dict(scaling="linear", factor=8.0), base=dict(scaling="base", factor=4.0),
                           blend=dict(scaling="blend", factor=16.0, original_length=4096))[case["scaling"]]
        s["freqs"] = None
        if own:  # the handle that a program keeps beside its weights
            from approxtrain_b200 import ops
            s["freqs"] = ops.rotary_frequencies(case["rot"], base=10000.0, device="cuda", **s["scaled"])
        if case["train"]:
            s["dq"], s["dk"] = heads(case["heads"]), heads(case["kv_heads"])
            s["q"].requires_grad_()
            s["k"].requires_grad_()
    elif case["op"] == "adamw":
        sizes, t = _sizes(case), _DT[case["dtype"]]
        total = sum(sizes)
        # parameters and gradients are views of flat buffers, as in the trainer's buckets (shift: how far off their alignment)
        s["flat"] = normal(total + case["shift"], dtype=t, scale=0.05)[case["shift"]:]
        s["flat_grad"] = (normal(total + case["shift"]) * torch.exp(2.0 * normal(total + case["shift"])) * 1e-3).to(t)[case["shift"]:]
        s["params"], s["grads"] = list(s["flat"].split(sizes)), list(s["flat_grad"].split(sizes))
        s["sizes"], s["lr"], s["betas"], s["eps"], s["decay"], s["rseed"] = sizes, 1e-3, (0.9, 0.99), 1e-8, 0.01, seed % 65536
        if own:
            from approxtrain_b200 import ops
            s["state"] = ops.AdamWState(s["params"], bits=case["bits"])
        elif case["bits"] == 32:
            s["m"], s["v"] = (torch.zeros(total, device="cuda") for _ in range(2))
        else:
            # every tensor's codes start at a block of their own
            blocks = [(z + 255) // 256 for z in sizes]
            s["at"] = torch.cat([torch.arange(z, device="cuda") + 256 * f for z, f in zip(sizes, _starts(blocks))])
            s["m8"], s["v8"] = (torch.zeros(256 * sum(blocks), device="cuda", dtype=torch.float8_e4m3fn) for _ in range(2))
            s["ms"], s["vs"] = (torch.zeros(sum(blocks), device="cuda") for _ in range(2))
        s["step"] = 0
    elif case["op"] == "quant":
        # magnitudes spread from column to column, as in activations
        s["x"] = (normal(case["rows"], case["cols"]) * torch.exp(1.5 * normal(1, case["cols"]))).to(_DT[case["dtype"]])
    else:
        t, m, k, n = _DT[case["dtype"]], case["rows"], case["inner"], case["cols"]
        s["x"] = (normal(m, k) * torch.exp(0.5 * normal(1, k))).to(t)
        s["w"] = normal(k, n, scale=1 / math.sqrt(k)).to(t)
        s["bias"] = normal(n, scale=0.1)
        if case["train"]:
            s["dy"] = normal(m, n, dtype=t, scale=0.01)
            for name in ("x", "w", "bias"):
                s[name].requires_grad_()
        elif own:  # a served layer keeps its weights in 4 bits
            from approxtrain_b200 import ops
            s["wq"] = ops.mx_quantize(s["w"], axis=0)
        else:
            s["wq"] = _mx(s["w"].float().t()).t()
    return s


def _starts(lengths):
    at = torch.tensor([0] + lengths[:-1])
    return at.cumsum(0).tolist()


# ---- plain forms --------------------------------------------------------------------------------------
def _norm(z, kind, eps, w, b):
    if kind == "layer":
        z = z - z.mean(-1, keepdim=True)
    y = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + eps)
    y = y * w
    return y if b is None else y + b


def _plain_norm(s):
    c = s["case"]
    t = s["x"].dtype
    u = s["block"].float()
    if c["post"]:
        u = _norm(u, c["kind"], s["eps"], s["post_w"], s["post_b"])
    if s["gate"] is not None:
        u = u * s["gate"].float()
    r = s["x"].float() + s["scale"] * u
    y = _norm(r, c["kind"], s["eps"], s["pre_w"], s["pre_b"])
    return r.to(t), y.to(t)


def _frequencies(rot, scaling="none", factor=1.0, original_length=0, base=10000.0):
    """The angle of a position in 64 bits, and the factor on the rotated values."""
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    if scaling == "base" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2.0 * i / rot)
    if scaling == "linear":
        f = f / factor
    if scaling != "blend":
        return f, 1.0
    # frequencies that turn more than 32 times over the original length stay, those below one turn are interpolated
    turns = original_length * f / (2 * math.pi)
    keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
    return f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1.0


def _rotate(x, cos, sin, rot, layout):
    x = x.float()
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if layout == "half" else (x[..., :rot:2], x[..., 1:rot:2])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([ra, rb], -1) if layout == "half" else torch.stack([ra, rb], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_rotary(s):
    c = s["case"]
    f, mag = _frequencies(c["rot"], **s["scaled"])
    angle = s["positions"].double()[..., None, None] * f
    cos, sin = (mag * angle.cos()).float(), (mag * angle.sin()).float()
    t = s["q"].dtype
    out = [_rotate(s[x].detach(), cos, sin, c["rot"], c["layout"]).to(t) for x in ("q", "k")]
    if c["train"]:
        out += [_rotate(s[x], cos, -sin, c["rot"], c["layout"]).to(t) for x in ("dq", "dk")]
    return out


def _mix(h):
    """MurmurHash3's 32-bit finaliser on 64-bit integers."""
    h = h ^ (h >> 16)
    h = (h * 0x85EBCA6B) & 0xFFFFFFFF
    h = h ^ (h >> 13)
    h = (h * 0xC2B2AE35) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _random16(at, seed, step):
    """Two 16-bit random numbers for each place."""
    one = torch.ones((), dtype=torch.int64, device=at.device)
    key = _mix((seed * one) ^ _mix(step * one))
    h = _mix((((at & 0xFFFFFFFF) + (at >> 32) * 0x9E3779B1) & 0xFFFFFFFF) ^ key)
    return h & 0xFFFF, h >> 16


def _blocks8(a, random, at_least):
    """Blocks of 256 values in 8-bit floats (three fraction bits) with the largest at 448, rounded up with the probability of the rest."""
    top = a.abs().amax(1, keepdim=True)
    full = top >= 2.0 ** -100
    scale = torch.where(full, top / 448.0, torch.zeros_like(top))
    q = (a.abs() * torch.where(full, 448.0 / top, torch.zeros_like(top))).clamp(max=448.0)
    low = q < 2.0 ** -6
    z = torch.where(low, q + 2.0 ** -6, q)
    bits = (z.view(torch.int32) + ((random << 4) | 8).to(torch.int32)) & -0x100000
    z = bits.view(torch.float32)
    z = torch.where(low, z - 2.0 ** -6, z)
    if at_least:
        z = torch.where(q > 0, z.clamp(min=2.0 ** -9), z)
    return torch.copysign(z, a).to(torch.float8_e4m3fn), scale[:, 0]


def _plain_adamw(s):
    c, (b1, b2) = s["case"], s["betas"]
    s["step"] += 1
    t, lr = s["step"], s["lr"]
    g = s["flat_grad"].float()
    p = s["flat"].float() * (1 - lr * s["decay"])
    if c["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        at = s["at"]
        m = (s["m8"].float().view(-1, 256) * s["ms"][:, None]).view(-1)[at]
        v = (s["v8"].float().view(-1, 256) * s["vs"][:, None]).square().view(-1)[at]
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * (g * g)
    denom = torch.sqrt(v) / math.sqrt(1 - b2 ** t) + s["eps"]
    s["flat"].copy_(p - (lr / (1 - b1 ** t)) * (m / denom))
    if c["bits"] == 32:
        s["m"], s["v"] = m, v
        return s["flat"], m, v
    rm, rv = _random16(torch.arange(s["m8"].numel(), device="cuda"), s["rseed"], t)
    spread = torch.zeros(s["m8"].numel(), device="cuda")
    spread[at] = m
    m8, s["ms"] = _blocks8(spread.view(-1, 256), rm.view(-1, 256), False)
    spread = torch.zeros(s["m8"].numel(), device="cuda")
    spread[at] = torch.sqrt(v)
    v8, s["vs"] = _blocks8(spread.view(-1, 256), rv.view(-1, 256), True)
    s["m8"], s["v8"] = m8.view(-1), v8.view(-1)
    return s["flat"], s["m8"], s["ms"], s["v8"], s["vs"]


def _mx(x):
    """The values of x's rows in 4-bit floats (0, .5, 1, 1.5, 2, 3, 4, 6) with a power of two for each 32 elements."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -cols % 32)).view(rows, -1, 32)
    top = x.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top)[1] - 3).clamp(min=-127)  # the largest element's exponent less two
    scale = torch.ldexp(torch.ones_like(top), e)
    a = (x / scale).abs().clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return (torch.copysign(torch.round(a / step) * step, x) * scale).view(rows, -1)[:, :cols]


def _plain_dense(s):
    c, t = s["case"], s["x"].dtype
    if not c["train"]:
        return (_mx(s["x"]) @ s["wq"] + s["bias"]).to(t)
    x, w, g = s["x"].detach(), s["w"].detach(), s["dy"]
    y = _mx(x) @ _mx(w.t()).t() + s["bias"].detach()
    dx = _mx(g) @ _mx(w).t()
    dw = _mx(x.t()) @ _mx(g.t()).t()
    return y.to(t), dx.to(t), dw.to(t), g.float().sum(0)


# ---- one pass ------------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if c["op"] == "norm":
        if own:
            from approxtrain_b200 import layers
            r, y = layers.residual_norm(s["x"], s["block"], gate=s["gate"], scale=s["scale"], post=(s["post_w"], s["post_b"]) if c["post"] else None,
                                        pre=(s["pre_w"], s["pre_b"]), kind=c["kind"], eps=s["eps"], need_sum=c["both"])
        else:
            r, y = _plain_norm(s)
        outs = [y, r] if c["both"] else [y]
        if not c["train"]:
            return outs
        leaves = [s[k] for k in ("x", "block", "gate", "pre_w", "pre_b", "post_w", "post_b") if s[k] is not None]
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, [s["dy"], s["dr"]] if c["both"] else [s["dy"]]))
    if c["op"] == "rotary":
        if not own:
            return _plain_rotary(s)
        from approxtrain_b200 import layers
        q, k = layers.rotary(s["q"], s["positions"], s["freqs"], k=s["k"], layout=c["layout"])
        if not c["train"]:
            return q, k
        return [q.detach(), k.detach()] + list(torch.autograd.grad([q, k], [s["q"], s["k"]], [s["dq"], s["dk"]]))
    if c["op"] == "adamw":
        if not own:
            return _plain_adamw(s)
        from approxtrain_b200 import ops
        st = s["state"]
        ops.adamw_step(s["params"], s["grads"], st, lr=s["lr"], betas=s["betas"], eps=s["eps"], weight_decay=s["decay"], seed=s["rseed"])
        if c["bits"] == 32:
            return s["flat"], st.exp_avg, st.exp_avg_sq
        return s["flat"], st.exp_avg, st.exp_avg_scale, st.exp_avg_sq_root, st.exp_avg_sq_scale
    if c["op"] == "quant":
        if not own:
            return _mx(s["x"]), _mx(s["x"].t()).t()
        from approxtrain_b200 import ops
        along, across = ops.mx_quantize_both(s["x"])
        return along.dequantize(), across.dequantize()
    if not own:
        return _plain_dense(s)
    from approxtrain_b200 import layers, ops
    if not c["train"]:
        return ops.mx_matmul(ops.mx_quantize(s["x"]), s["wq"], bias=s["bias"], out_dtype=s["x"].dtype)
    y = layers.mxdense(s["x"], s["w"], s["bias"])
    return [y.detach()] + list(torch.autograd.grad([y], [s["x"], s["w"], s["bias"]], [s["dy"]]))


# ---- the definition in 64 bits ---------------------------------------------------------------------------
def _exact_norm(s):
    c = s["case"]
    d = c["width"]
    f = {k: v.detach().double().reshape(-1, d) for k, v in s.items() if isinstance(v, torch.Tensor)}
    rows, scale = f["x"].shape[0], s["scale"]

    def stats(z):
        mean = z.sum(1, keepdim=True) / d if c["kind"] == "layer" else torch.zeros_like(z[:, :1])
        return mean, ((z - mean).pow(2).sum(1, keepdim=True) / d + s["eps"]).pow(-0.5)

    def back(g, hat, rstd, w):  # gradient through hat * w + b to the norm's input
        a = g * w
        out = a - hat * ((a * hat).sum(1, keepdim=True) / d)
        return rstd * (out - a.sum(1, keepdim=True) / d if c["kind"] == "layer" else out)
    u, hat_b = f["block"], None
    if c["post"]:
        mean_b, rstd_b = stats(u)
        hat_b = (u - mean_b) * rstd_b
        u = hat_b * f["post_w"] + (f["post_b"] if s["post_b"] is not None else 0.0)
    gate = torch.ones(1, 1, d, dtype=torch.float64, device="cuda") if s["gate"] is None else f["gate"].reshape(-1, 1, d)
    groups = gate.shape[0]
    r = f["x"] + scale * (u.reshape(groups, -1, d) * gate).reshape(rows, d)
    mean, rstd = stats(r)
    hat = (r - mean) * rstd
    y = hat * f["pre_w"] + (f["pre_b"] if s["pre_b"] is not None else 0.0)
    shape = s["x"].shape
    outs = [y.reshape(shape)] + ([r.reshape(shape)] if c["both"] else [])
    if not c["train"]:
        return outs
    g = back(f["dy"], hat, rstd, f["pre_w"]) + (f["dr"] if c["both"] else 0.0)
    du = scale * (g.reshape(groups, -1, d) * gate).reshape(rows, d)
    outs += [g.reshape(shape), (back(du, hat_b, rstd_b, f["post_w"]) if c["post"] else du).reshape(shape)]
    if s["gate"] is not None:
        outs.append(scale * (g * u).reshape(groups, -1, d).sum(1).reshape(s["gate"].shape))
    outs.append((f["dy"] * hat).sum(0))
    if s["pre_b"] is not None:
        outs.append(f["dy"].sum(0))
    if c["post"]:
        outs.append((du * hat_b).sum(0))
        if s["post_b"] is not None:
            outs.append(du.sum(0))
    return outs


def _exact_rotary(s):
    c = s["case"]
    rot, half = c["rot"], c["rot"] // 2
    scaled = s["scaled"].get("scaling", "none")
    k = s["scaled"].get("factor", 1.0)
    table, mag = [], 1.0
    for i in range(half):
        f = math.exp(-(2.0 * i / rot) * math.log(10000.0 * (k ** (rot / (rot - 2.0)) if scaled == "base" and rot > 2 else 1.0)))
        if scaled == "linear":
            f /= k
        if scaled == "blend":
            keep = min(1.0, max(0.0, (4096 * f / (2 * math.pi) - 1.0) / 31.0))
            f = keep * f + (1.0 - keep) * f / k
            mag = 1.0 + 0.1 * math.log(k)
        table.append(f)
    turn = torch.polar(torch.full((half,), mag, dtype=torch.float64, device="cuda"), s["positions"].double()[:, :, None, None] * torch.tensor(table, dtype=torch.float64, device="cuda"))

    def apply(x, turn):
        x = x.detach().double()
        z = x[..., :rot].unflatten(-1, (2, half) if c["layout"] == "half" else (half, 2))
        z = z.transpose(-1, -2) if c["layout"] == "half" else z
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
        z = z.transpose(-1, -2) if c["layout"] == "half" else z
        return torch.cat([z.flatten(-2), x[..., rot:]], -1)
    outs = [apply(s["q"], turn), apply(s["k"], turn)]
    return outs + [apply(s["dq"], turn.conj()), apply(s["dk"], turn.conj())] if c["train"] else outs


def _exact_adamw(s):
    # the first step: both moments are zero before it
    (b1, b2), lr, eps = s["betas"], s["lr"], s["eps"]
    g = s["flat_grad"].double()
    m, v = g - b1 * g, g.square() - b2 * g.square()
    p = s["flat"].double()
    p = p - lr * s["decay"] * p - lr * (m / (1 - b1)) / ((v / (1 - b2)).sqrt() + eps)
    if s["case"]["bits"] == 32:
        return p, m, v
    lengths = [-(-n // 256) * 256 for n in s["sizes"]]
    pieces = list(zip(m.split(s["sizes"]), v.sqrt().split(s["sizes"]), lengths))
    place = torch.arange(sum(lengths), device="cuda")
    key = _mix(torch.tensor(s["rseed"], device="cuda") ^ _mix(torch.tensor(1, device="cuda")))
    h = _mix(place ^ key)
    found = [p]
    for which, rest in ((0, (h & 0xFFFF)), (1, h >> 16)):
        a = torch.cat([torch.nn.functional.pad(x[which], (0, x[2] - x[which].numel())) for x in pieces]).view(-1, 256)
        scale = a.abs().max(1).values / 448.0
        scale = torch.where(scale * 448.0 >= 2.0 ** -100, scale, 0.0)
        q = torch.where(scale[:, None] > 0, a.abs() / scale[:, None], 0.0)
        ulp = torch.exp2((torch.frexp(q)[1] - 1).clamp(min=-6).double() - 3)
        up = (rest.view(-1, 256).double() * 16 + 8) / 2 ** 20
        q = (torch.floor(q / ulp + up) * ulp).clamp(max=448.0)
        if which:
            q = torch.where(a > 0, q.clamp(min=2.0 ** -9), q)
        found += [(q * a.sign()).view(-1), scale]
    return found


_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_mx(x, axis):
    x = x.detach().double()
    x = x if axis == 1 else x.t()
    n, k = x.shape
    out = torch.zeros(n, -(-k // 32) * 32, dtype=torch.float64, device="cuda")
    out[:, :k] = x
    out = out.view(n, -1, 32)
    top = out.abs().max(2, keepdim=True).values
    unit = torch.where(top > 0, torch.ldexp(torch.ones_like(top), torch.frexp(top).exponent - 3).clamp(min=2.0 ** -127), 1.0)
    q = out / unit
    grid = torch.tensor(_GRID, dtype=torch.float64, device="cuda")
    border = (grid[1:] + grid[:-1]) / 2
    # borders belong to the neighbour with the even code
    lower, upper = torch.bucketize(q.abs(), border, right=False), torch.bucketize(q.abs(), border, right=True)
    code = torch.where(lower % 2 == 0, lower, upper)
    out = (grid[code] * q.sign() * unit).view(n, -1)[:, :k]
    return out if axis == 1 else out.t()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s)
    if case["op"] == "rotary":
        return _exact_rotary(s)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    if case["op"] == "quant":
        return _exact_mx(s["x"], 1), _exact_mx(s["x"], 0)
    x, w = s["x"], s["w"]
    y = _exact_mx(x, 1) @ _exact_mx(w, 0) + s["bias"].detach().double()
    if not case["train"]:
        return y
    g = s["dy"]
    return [y, _exact_mx(g, 1) @ _exact_mx(w, 1).t(), _exact_mx(x, 0).t() @ _exact_mx(g, 0), g.double().sum(0)]


def work(case):
    e = 4 if case.get("dtype") == "f32" else 2
    if case["op"] == "norm":
        n = case["batch"] * case["seq"] * case["width"]
        gate = {"none": 0, "width": 0, "sequence": n // case["seq"], "full": n}[case["gate"]]
        # forward: x, block in, y (and the sum) out; backward: the gradients, the sum and the block in, two gradients out
        reads = (2 + 1 + case["both"]) * n + gate
        if case["train"]:
            reads += (1 + case["both"]) * n + 2 * n + 2 * n + 2 * gate + (0 if case["both"] else n)
        return {"bytes": reads * e, "flops": n * (40 if case["train"] else 12)}
    if case["op"] == "rotary":
        n = case["batch"] * case["seq"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * n * e * (2 if case["train"] else 1) + 8 * case["batch"] * case["seq"], "flops": 3 * n * (2 if case["train"] else 1)}
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        return {"bytes": n * (3 * e + (16 if case["bits"] == 32 else 4 + 16 / 256)), "flops": 15 * n}
    if case["op"] == "quant":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (e + 4 * (0.5 + 1 / 32) + 8), "flops": 10 * n}
    m, k, n = case["rows"], case["inner"], case["cols"]
    four = 0.5 + 1 / 32
    if not case["train"]:
        return {"bytes": m * k * e + (k * n) * four + m * n * e + 4 * n, "flops": 2 * m * k * n}
    # x, w and the output's gradient are read and quantised both ways, three products written
    return {"bytes": (m * k + k * n + m * n) * 2 * e, "flops": 6 * m * k * n}

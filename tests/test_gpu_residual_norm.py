"""residual_norm and its gradient against the formulas in 64 bits."""
import itertools

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24      # half a step of FP32


def _half(t):
    return torch.finfo(t).eps / 2


def _norm64(z, kind, eps):
    mean = z.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(z[..., :1])
    rstd = ((z - mean).pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    return mean, rstd


def _plain(x, block, gate, scale, post, pre, kind, eps):
    """(r, y, everything the gradient needs) in 64 bits."""
    d = lambda t: None if t is None else t.detach().double()
    x, block, gate = d(x), d(block), d(gate)
    s = {}
    u = block
    if post is not None:
        s["pm"], s["pr"] = _norm64(block, kind, eps)
        s["ph"] = (block - s["pm"]) * s["pr"]
        u = s["ph"] * (d(post[0]) if post[0] is not None else 1.0) + (d(post[1]) if post[1] is not None else 0.0)
    s["u"] = u
    r = x
    if block is not None:
        r = x + scale * (u * gate if gate is not None else u)
    y = None
    if pre is not None:
        s["m"], s["r"] = _norm64(r, kind, eps)
        s["h"] = (r - s["m"]) * s["r"]
        y = s["h"] * (d(pre[0]) if pre[0] is not None else 1.0) + (d(pre[1]) if pre[1] is not None else 0.0)
    return r, y, s


def _plain_grad(s, block, gate, scale, post, pre, kind, dr, dy):
    """Gradients in 64 bits."""
    d = lambda t: None if t is None else t.detach().double()
    out = {}

    def back(g, hat, rstd, w):
        a = g * w if w is not None else g
        return rstd * ((a - a.mean(-1, keepdim=True) if kind == "layer" else a) - hat * (a * hat).mean(-1, keepdim=True))
    like = d(dr if dr is not None else dy)
    rows = tuple(range(like.dim() - 1))
    g = torch.zeros_like(like)
    if dy is not None:
        hat = s["h"]
        g = back(d(dy), hat, s["r"], d(pre[0]))
        out["pre_w"], out["pre_b"] = (d(dy) * hat).sum(rows), d(dy).sum(rows)
    if dr is not None:
        g = g + d(dr)
    out["x"] = g
    if block is not None:
        du = scale * g
        if gate is not None:
            full = s["u"] * du
            keep = [i for i in range(full.dim()) if gate.dim() < full.dim() or gate.shape[i] != 1 or full.shape[i] == 1]
            if gate.dim() == 1:
                out["gate"] = full.sum(rows)
            else:
                out["gate"] = full.sum([i for i in range(full.dim()) if i not in keep], keepdim=True) if len(keep) < full.dim() else full
            du = du * d(gate)
        if post is not None:
            out["post_w"], out["post_b"] = (du * s["ph"]).sum(rows), du.sum(rows)
            du = back(du, s["ph"], s["pr"], d(post[0]))
        out["block"] = du
    return out


def _close(got, want, t, size, what):
    """Half a step of the type for the one rounding, 64 FP32 roundings of the largest of the terms behind a value (`size`):
    a row's sum adds at most 16 per thread, 9 levels of threads and 3 of CTAs, twice, and the rest are a dozen products."""
    assert got.shape == want.shape and got.dtype == t, what
    tol = _half(t) * want.abs() + 64 * F32 * size + torch.finfo(t).tiny
    bad = (got.double() - want).abs() - tol
    assert bool((bad <= 0).all()), (what, float(bad.max()), float(want.abs().max()))


def _make(shape, t, kind, post, gate, pre, scale, affine, w_t, seed=0, strided=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = shape[-1]

    def rnd(*s, dt=t, k=1.0, at=0.0):
        return (torch.randn(*s, generator=g, device="cuda") * k + at).to(dt)
    if strided:
        x = rnd(*shape[:-1], 2 * width + 1)[..., 1:width + 1]
        block = rnd(*shape[:-1], width + 3)[..., 3:]
    else:
        x, block = rnd(*shape), rnd(*shape, k=0.7, at=0.3)
    gates = {None: None, "width": (width,), "sequence": (*shape[:1], *([1] * (len(shape) - 2)), width), "full": shape}[gate]
    pair = lambda: ((rnd(width, dt=w_t, k=0.2, at=1.0) if affine else None), (rnd(width, dt=w_t, k=0.2) if affine and kind == "layer" else None))
    return dict(x=x, block=block, gate=rnd(*gates, k=0.5) if gates else None, scale=scale, post=pair() if post else None,
                pre=pair() if pre else None, kind=kind, eps=1e-3), rnd


def _check(a, rnd, t, need_sum=True, which=("dr", "dy")):
    from approxtrain_b200 import layers, ops
    leaves = dict(x=a["x"], block=a["block"], gate=a["gate"])
    for n in ("post", "pre"):
        if a[n] is not None:
            leaves[n + "_w"], leaves[n + "_b"] = a[n]
    leaves = {k: v for k, v in leaves.items() if v is not None}
    r64, y64, s = _plain(**a)
    r, y = ops.residual_norm(**a)
    width = a["x"].shape[-1]
    size_r = a["x"].double().abs().amax(-1, keepdim=True) + (abs(a["scale"]) * (s["u"] * (a["gate"].double() if a["gate"] is not None else 1.0)).abs().amax(-1, keepdim=True) if a["block"] is not None else 0.0)
    if a["post"] is not None:  # the mean's error counts against the deviation
        size_r = size_r + abs(a["scale"]) * (a["block"].double().abs().amax(-1, keepdim=True) * s["pr"]) * 2
    _close(r, r64, t, size_r, "sum")
    if a["pre"] is not None:
        wmax = a["pre"][0].double().abs().max() if a["pre"][0] is not None else 1.0
        size_y = size_r * s["r"] * wmax + y64.abs().amax(-1, keepdim=True)
        _close(y, y64, t, size_y, "norm")
        if not need_sum:
            r2, y2 = ops.residual_norm(**a, need_sum=False)
            assert r2 is None and torch.equal(y2, y)
    for v in leaves.values():
        v.requires_grad_()
    r1, y1 = layers.residual_norm(**a, need_sum=need_sum)
    assert (r1 is None) == (not need_sum and a["pre"] is not None)
    if r1 is not None:
        assert torch.equal(r1, r)
    assert (y1 is None) == (y is None) and (y is None or torch.equal(y1, y))
    dr = rnd(*r.shape, k=0.1) if r1 is not None and "dr" in which else None
    dy = rnd(*r.shape, k=0.1) if y1 is not None and "dy" in which else None
    outs = [(o, g) for o, g in ((r1, dr), (y1, dy)) if g is not None]
    got = dict(zip(leaves, torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [g for _, g in outs], allow_unused=True)))
    want = _plain_grad(s, a["block"], a["gate"], a["scale"], a["post"], a["pre"], a["kind"], dr, dy)
    rows = r.numel() // width
    hat = s["h"].abs().amax() if "h" in s else 1.0
    top = (dr.double().abs().max() if dr is not None else 0.0) + (dy.double().abs().max() * (wmax * s["r"].max() * (1 + hat * hat) + 1) if dy is not None else 0.0)
    b_top = abs(a["scale"]) * top * (a["gate"].double().abs().max() if a["gate"] is not None else 1.0)
    if a["post"] is not None:
        ph = s["ph"].abs().max() + a["block"].double().abs().max() * s["pr"].max()
        b_top = b_top * (1 + (a["post"][0].double().abs().max() if a["post"][0] is not None else 1.0)) * (1 + s["pr"].max() * (1 + ph * ph))
    # a column's sum adds `rows` terms in pieces; each partial sum is rounded: the terms' root mean square times sqrt(rows) bounds
    # the typical partial sum, and 64 + rows / 64 roundings of the largest (terms x rows) bound all of them
    terms = {"x": top, "block": b_top, "pre_w": rows * (dy.double().abs().max() * (hat + size_r.max() * s["r"].max()) if dy is not None else 0.0) , "pre_b": rows * (dy.double().abs().max() if dy is not None else 0.0)}
    if a["post"] is not None:
        terms["post_w"] = rows * b_top * (ph + 1)
        terms["post_b"] = rows * b_top
    if a["gate"] is not None:
        terms["gate"] = (rows * a["gate"].numel() ** 0 if a["gate"].dim() == 1 else rows // (a["gate"].numel() // width)) * abs(a["scale"]) * top * (s["u"].abs().max() + size_r.max())
    for k, v in leaves.items():
        if k not in want:
            assert got[k] is None or not got[k].any(), k
            continue
        _close(got[k], want[k].reshape(v.shape), v.dtype, terms[k] * torch.ones((), device="cuda", dtype=torch.float64), k)
    return got


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("post,gate,pre", [(p, g, n) for p, g, n in itertools.product([False, True], [None, "width", "sequence", "full"], [False, True])])
def test_every_form(t, kind, post, gate, pre):
    for shape in ((3, 7, 96), (5, 4, 33)):
        a, rnd = _make(shape, t, kind, post, gate, pre, 0.5 if gate else 1.0, True, torch.float32 if gate != "full" else t)
        _check(a, rnd, t, need_sum=gate is None or not pre)
        a, rnd = _make(shape, t, kind, post, gate, pre, 1.0, False, t, seed=1)
        _check(a, rnd, t, need_sum=True, which=("dr",) if not pre or post else ("dy",))


@pytest.mark.parametrize("width", [1, 2, 5, 16, 17, 64, 100, 129, 256, 500, 512, 513, 1000, 1024, 2048, 2051, 4096, 4104, 8192, 8200, 12288, 16384, 20001, 32768])
@pytest.mark.parametrize("post", [False, True])
def test_widths(width, post):
    rows = 37 if width < 8000 else 9
    for t in (torch.float32, torch.bfloat16):
        a, rnd = _make((rows, width), t, "rms" if width < 3 else "layer", post, "width" if post else None, True, 0.75, True, torch.float32, seed=width)
        _check(a, rnd, t)


@pytest.mark.parametrize("rows,width", [(1, 512), (2, 40), (1000, 64), (8192, 24), (4099, 300), (2500, 1030)])
def test_rows_and_groups_of_the_gate(rows, width):
    for gate in ("width", "sequence", "full"):
        a, rnd = _make((rows, 1, width), torch.float32, "layer", True, gate, True, 1.5, True, torch.float32, seed=rows)
        _check(a, rnd, torch.float32)
    if rows % 4 == 0:
        for batch in (2, 4):  # groups that several workers share, and groups inside one worker
            a, rnd = _make((batch, rows // batch, width), torch.bfloat16, "rms", False, "sequence", True, 1.0, True, torch.float32, seed=rows + 1)
            _check(a, rnd, torch.bfloat16)


def test_unaligned_and_strided_tensors():
    for t in (torch.float32, torch.bfloat16):
        for width in (64, 65, 512):
            a, rnd = _make((6, 5, width), t, "layer", True, "width", True, 1.0, True, torch.float32, strided=True)
            _check(a, rnd, t)
            # contiguous, but one element after an aligned address
            off = lambda v: torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")[1:].view(v.shape).copy_(v.detach())
            a, rnd = _make((6, 5, width), t, "layer", True, "width", True, 1.0, True, torch.float32)
            a.update(x=off(a["x"]), block=off(a["block"]), gate=off(a["gate"]), pre=tuple(off(v) for v in a["pre"]))
            _check(a, rnd, t)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_of_four_byte_chunks_and_of_single_elements(t):
    """Even lengths that are no multiple of 16 bytes, odd ones, and tensors at half of a chunk's alignment."""
    for width in (6, 130, 3950, 1001):
        for gate, post in (("full", True), ("sequence", False), (None, True)):
            a, rnd = _make((5, 9, width), t, "layer", post, gate, True, 0.5, True, torch.float32, seed=width)
            _check(a, rnd, t)
    off = lambda v: torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")[1:].view(v.shape).copy_(v.detach())
    a, rnd = _make((6, 5, 66), t, "rms", True, "width", True, 1.0, True, torch.float32)
    a.update(x=off(a["x"]), pre=tuple(None if v is None else off(v) for v in a["pre"]))
    _check(a, rnd, t)


def test_the_formula_agrees_with_differences():
    """The 64-bit gradient above against central differences of the 64-bit forward pass."""
    g = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    a = dict(x=rnd(3, 2, 9), block=rnd(3, 2, 9), gate=rnd(3, 1, 9), scale=0.7, post=(rnd(9), rnd(9)), pre=(rnd(9), rnd(9)), kind="layer", eps=1e-3)
    dr, dy = rnd(3, 2, 9), rnd(3, 2, 9)

    def loss():
        r, y, _ = _plain(**a)
        return float((r * dr).sum() + (y * dy).sum())
    r, _, s = _plain(**a)
    want = _plain_grad(s, a["block"], a["gate"], a["scale"], a["post"], a["pre"], "layer", dr, dy)
    for k, v in dict(x=a["x"], block=a["block"], gate=a["gate"], post_w=a["post"][0], post_b=a["post"][1], pre_w=a["pre"][0], pre_b=a["pre"][1]).items():
        flat, grad = v.view(-1), want[k].reshape(-1)
        for i in range(0, flat.numel(), 5):
            was = float(flat[i])
            flat[i] = was + 1e-5
            hi = loss()
            flat[i] = was - 1e-5
            lo = loss()
            flat[i] = was
            assert abs((hi - lo) / 2e-5 - float(grad[i])) < 1e-6 * (1 + abs(float(grad[i]))), k


def test_empty_and_not_finite_rows():
    from approxtrain_b200 import layers, ops
    w = torch.ones(8, device="cuda", requires_grad=True)
    gate = torch.ones(8, device="cuda", requires_grad=True)
    x = torch.empty(0, 8, device="cuda", requires_grad=True)
    r, y = layers.residual_norm(x, x, gate=gate, pre=(w, None))
    gx, gw, gg = torch.autograd.grad([r, y], [x, w, gate], [torch.empty_like(r), torch.empty_like(y)])
    assert gx.shape == (0, 8) and not gw.any() and not gg.any()
    x = torch.randn(5, 40, device="cuda")
    b = torch.randn(5, 40, device="cuda")
    _, clean = ops.residual_norm(x, b, pre=(None, None))
    x[1, 3], x[3, 0] = float("nan"), float("inf")
    _, y = ops.residual_norm(x, b, pre=(None, None))
    assert y[1].isnan().all() and y[3].isnan().any()
    assert torch.equal(y[[0, 2, 4]], clean[[0, 2, 4]])


def test_same_bits_on_every_run_on_another_stream_and_in_a_graph():
    from approxtrain_b200 import layers
    a, rnd = _make((4, 700, 200), torch.bfloat16, "layer", True, "sequence", True, 0.5, True, torch.float32)
    dr, dy = rnd(4, 700, 200), rnd(4, 700, 200)

    def step():
        leaves = [a["x"], a["block"], a["gate"], *a["post"], *a["pre"]]
        for v in leaves:
            v.requires_grad_()
        r, y = layers.residual_norm(**a)
        return [r.detach(), y.detach(), *torch.autograd.grad([r, y], leaves, [dr, dy])]
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(u, v) for u, v in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    with torch.no_grad():
        a["x"].mul_(2.0)
    graph.replay()
    replayed = [t.clone() for t in captured]
    eager = step()
    assert all(torch.equal(u, v) for u, v in zip(replayed, eager))
    assert not torch.equal(eager[1], first[1])


def test_module_matches_torch_layer_norm():
    from approxtrain_b200 import layers
    m = layers.ResidualNorm(512).cuda()
    n = torch.nn.LayerNorm(512, eps=1e-3).cuda()
    x, b = (torch.randn(4, 9, 512, device="cuda") for _ in range(2))
    r, y = m(x, b)
    assert torch.equal(r, x + b)
    assert float((y - n(x + b)).detach().abs().max()) <= 1e-5      # both within a few FP32 roundings of values up to 5
    m = layers.ResidualNorm(64, kind="rms", post_norm=True, gate_init=0.5).cuda()
    r, y = m(x[..., :64], b[..., :64])
    (y.sum() + r.sum()).backward()
    assert all(p.grad is not None and p.grad.abs().sum() > 0 for p in m.parameters())
    assert m(x[..., :64])[1].shape == (4, 9, 64)          # the first norm of a network: nothing to add yet

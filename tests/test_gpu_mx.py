"""4-bit block-scaled matrices and their products against the definition in 64 bits."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _values(x, axis=1):
    """The quantised values in 64 bits: nearest grid value by comparison with the midpoints, ties to the even code."""
    x = x.detach().double()
    x = x if axis == 1 else x.t()
    n, k = x.shape
    p = torch.nn.functional.pad(x, (0, -k % 32)).reshape(n, -1, 32)
    top = p.abs().amax(2, keepdim=True)
    bad = ~top.isfinite()
    unit = torch.exp2((torch.frexp(torch.where(bad, 1.0, top)).exponent - 3).clamp(min=-127).double())
    q = p / unit
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    lo, hi = torch.bucketize(q.abs().contiguous(), mid, right=False), torch.bucketize(q.abs().contiguous(), mid, right=True)
    out = grid[torch.where(lo % 2 == 0, lo, hi)] * q.sign() * unit
    out = torch.where(bad, float("nan"), out)
    out = out.reshape(n, -1)[:, :k]
    return out if axis == 1 else out.t()


def _rand(*shape, t=torch.float32, seed=0, spread=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, generator=g, device="cuda")
    if spread:
        x = x * torch.exp(spread * torch.randn(*shape, generator=g, device="cuda"))
    return x.to(t)


def _same(a, b):
    return torch.equal(torch.nan_to_num(a.double(), nan=1e300), torch.nan_to_num(b.double(), nan=1e300))


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (32, 1), (3, 33), (128, 128), (129, 257), (200, 100), (1, 4096), (4096, 1), (256, 512), (300, 1000), (1025, 60)])
def test_quantise_and_back(t, shape):
    from approxtrain_b200 import ops
    for seed, spread in ((0, 0.0), (1, 3.0)):
        x = _rand(*shape, t=t, seed=seed, spread=spread)
        if t == torch.float16:
            x = x.clamp(-6e4, 6e4)
        along, across = ops.mx_quantize_both(x)
        for m, axis in ((along, 1), (across, 0), (ops.mx_quantize(x), 1), (ops.mx_quantize(x, axis=0), 0)):
            assert m.shape == shape and m.axis == axis
            want = _values(x, axis)
            assert _same(m.dequantize(), want), (axis, float((m.dequantize().double() - want).abs().max()))
            assert _same(m.dequantize(torch.bfloat16), want.float().to(torch.bfloat16))


def test_ties_borders_and_extreme_scales():
    from approxtrain_b200 import ops
    rows = []
    for e in (-149, -140, -130, -127, -126, -125, -124, -100, -3, 0, 1, 60, 125, 126, 127):
        row = torch.zeros(32, dtype=torch.float64)
        vals = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -5.0, 6.0, 7.999, 0.2500001, 0.7499999, 1e-3]
        for i, v in enumerate(vals):
            row[i] = v * 2.0 ** (e - 2)
        rows.append(row)
    x = torch.stack(rows).float().cuda()
    assert _same(ops.mx_quantize(x).dequantize(), _values(x))
    assert _same(ops.mx_quantize(x.t().contiguous(), axis=0).dequantize(), _values(x).t())
    x = _rand(40, 96)
    x[3, 5], x[7, 40], x[9, 95] = float("nan"), float("inf"), -float("inf")
    got = ops.mx_quantize(x).dequantize()
    assert _same(got, _values(x)) and got[3, :32].isnan().all() and got[7, 32:64].isnan().all() and got[9, 64:].isnan().all() and not got[3, 32:].isnan().any()
    assert not ops.mx_quantize(torch.zeros(5, 70, device="cuda")).dequantize().any()


def test_strided_and_unaligned_input():
    from approxtrain_b200 import ops
    x = _rand(70, 130)
    for v in (x.t(), x[:, 1:], x[::2], x.flatten()[1:1 + 60 * 128].view(60, 128)):
        a, b = ops.mx_quantize_both(v)
        assert _same(a.dequantize(), _values(v, 1)) and _same(b.dequantize(), _values(v, 0))


def _product(a, b, bias, relu, out_dtype):
    """Checks a product of the stored matrices a [m, k], b [n, k] given as floats."""
    from approxtrain_b200 import ops
    qa, qb = ops.mx_quantize(a), ops.mx_quantize(b)
    got = ops.mx_matmul(qa, qb, bias=bias, activation="relu" if relu else None, out_dtype=out_dtype)
    va, vb = _values(a), _values(b)
    want = va @ vb.t()
    # the accumulators hold at least FP32's 24 bits and truncate once per 64 elements: at most 2^-23 of the running sum each
    # time, which sum |products| bounds; a chunk's sums are added once each; bias, and the rounding to the type
    size = va.abs() @ vb.abs().t()
    k = a.shape[1]
    tol = ((k + 63) // 64 + (k + 2047) // 2048 + 2) * 2.0 ** -23 * size
    if bias is not None:
        want = want + bias.double()
        tol = tol + 2.0 ** -23 * (want.abs() + bias.double().abs())
    if relu:
        want = want.clamp(min=0.0)
    tol = tol + torch.finfo(out_dtype).eps / 2 * (want.abs() + tol) + torch.finfo(out_dtype).smallest_normal
    assert got.shape == want.shape and got.dtype == out_dtype
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), (tuple(a.shape), tuple(b.shape), float(off.max()), float((got.double() - want).norm() / want.norm()))
    return got, want


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 32), (3, 5, 64), (16, 100, 65), (17, 300, 256), (32, 129, 300), (33, 64, 512), (64, 1000, 100), (65, 128, 257), (100, 300, 700),
                                   (128, 128, 4096), (129, 257, 520), (200, 2000, 96), (1, 8000, 512), (16, 8000, 512),
                                   (16, 128, 8192), (5, 2048, 4200), (64, 300, 9000), (128, 200, 17000), (40, 128, 17000), (512, 2048, 8192), (100, 1000, 1500)])
def test_small_products(out_dtype, m, n, k):
    a, b = _rand(m, k, seed=m), _rand(n, k, seed=n + 1, spread=0.5)
    _product(a, b, None, False, out_dtype)
    _product(a, b, _rand(n, seed=9), True, out_dtype)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(2048, 2048, 512), (1500, 2300, 333), (4096, 1024, 2048), (1031, 3001, 2500), (1024, 1024, 8192), (5000, 600, 9000), (2049, 2047, 64), (256, 38000, 128)])
def test_large_products(out_dtype, m, n, k):
    a, b = _rand(m, k, seed=m), _rand(n, k, seed=n + 1, spread=0.5)
    got, want = _product(a, b, _rand(n, seed=9), False, out_dtype)
    if out_dtype == torch.float32:
        assert float((got.double() - want).norm() / want.norm()) <= 2e-6


def test_not_a_number_stays_in_its_row_and_column():
    from approxtrain_b200 import ops
    for m, n, k in ((40, 70, 96), (2048, 2048, 256)):
        a, b = _rand(m, k), _rand(n, k, seed=1)
        a[5, 33], b[60, 3] = float("inf"), float("nan")
        got = ops.mx_matmul(ops.mx_quantize(a), ops.mx_quantize(b))
        bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
        bad[5], bad[:, 60] = True, True
        assert torch.equal(got.isnan(), bad)


def test_empty_sizes():
    from approxtrain_b200 import ops
    q = lambda r, c, axis=1: ops.mx_quantize(torch.zeros(r, c, device="cuda"), axis=axis)
    assert ops.mx_matmul(q(0, 64), q(5, 64)).shape == (0, 5)
    assert ops.mx_matmul(q(5, 64), q(0, 64)).shape == (5, 0)
    bias = _rand(7)
    for n in (7, 2000):
        bias = _rand(n)
        assert torch.equal(ops.mx_matmul(q(3, 0), q(n, 0), bias=bias), bias.expand(3, n))
    a, b = ops.mx_quantize_both(torch.zeros(0, 9, device="cuda"))
    assert a.dequantize().shape == (0, 9) and b.dequantize().shape == (0, 9)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(0, 5), (1, 1), (3, 200), (128, 128), (129, 33), (5000, 300), (2049, 1000)])
def test_column_sums(t, shape):
    from approxtrain_b200 import ops
    x = _rand(*shape, t=t)
    sums = torch.full((shape[1],), float("nan"), device="cuda")
    a, b = ops.mx_quantize_both(x, sums=sums)
    # 8 terms a chain, then at most 2 + 2 + rows / 2048 + 16 partial sums
    tol = (8 + 4 + shape[0] / 2048 + 16) * 2.0 ** -24 * x.double().abs().sum(0)
    assert bool(((sums.double() - x.double().sum(0)).abs() <= tol).all())
    if shape[0]:
        assert _same(a.dequantize(), _values(x, 1)) and _same(b.dequantize(), _values(x, 0))


def test_transposed_operands_and_repeats():
    """The backward products' forms; the same bits on every run and on another stream."""
    from approxtrain_b200 import ops
    x, w = _rand(300, 500), _rand(500, 260, seed=1)
    xq, wq = ops.mx_quantize(x), ops.mx_quantize(w, axis=0)
    y = ops.mx_matmul(xq, wq)
    want = _values(x) @ _values(w, 0)
    assert float((y.double() - want).norm() / want.norm()) < 1e-6
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.mx_matmul(xq, wq)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, y)


def test_two_products_at_once():
    """Large products on two streams: their tensor memory is taken in turn."""
    from approxtrain_b200 import ops
    a, b, c = (ops.mx_quantize(_rand(2048, 1024, seed=i)) for i in range(3))
    want = [ops.mx_matmul(a, b), ops.mx_matmul(a, c)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    torch.cuda.synchronize()
    for _ in range(4):
        for i, (s, q) in enumerate(zip(streams, (b, c))):
            with torch.cuda.stream(s):
                got[i] = ops.mx_matmul(a, q)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lead,k,n", [((5,), 40, 24), ((3, 50), 96, 130), ((1100,), 512, 2048)])
def test_dense_layer_and_gradients(t, lead, k, n):
    from approxtrain_b200 import layers
    x, w, bias = _rand(*lead, k, t=t), _rand(k, n, t=t, seed=1), _rand(n, seed=2)
    dy = _rand(*lead, n, t=t, seed=3)
    for act in (None, "relu"):
        leaves = [v.clone().requires_grad_() for v in (x, w, bias)]
        y = layers.mxdense(*leaves, activation=act)
        dx, dw, db = torch.autograd.grad(y, leaves, dy)
        x2, g = x.reshape(-1, k), dy.reshape(-1, n)
        want = _values(x2) @ _values(w, 0) + bias.double()
        if act:
            g = torch.where(y.detach().reshape(-1, n) > 0, g, torch.zeros_like(g))
            want = want.clamp(min=0)
        # norms: sums to 2e-6 in FP32, and half a step of the type
        near = lambda got, want, tt: float((got.double().reshape(want.shape) - want).norm() / want.norm()) <= 2e-6 + torch.finfo(tt).eps / 2
        assert near(y.detach(), want, t)
        assert near(dx, _values(g) @ _values(w, 1).t(), t)
        assert near(dw, _values(x2, 0).t() @ _values(g, 0), t)
        assert near(db, g.double().sum(0), torch.float32)
        assert dx.dtype == t and dw.dtype == t and dx.shape == x.shape
        # without one of the gradients
        a = x.clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(layers.mxdense(a, w, bias, act), a, dy)[0], dx)
        b = w.clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(layers.mxdense(x, b, bias, act), b, dy)[0], dw)


def test_module_and_frozen_weights():
    from approxtrain_b200 import layers
    m = layers.densemx(64, 96, activation="tanh").cuda()
    x = _rand(4, 7, 64)
    y = m(x)
    with torch.no_grad():
        assert torch.equal(m.freeze()(x), y)
        m.kernel.mul_(2.0)
        assert torch.equal(m(x), y)
        m.train()
        assert not torch.equal(m(x), y)
    m(x).sum().backward()
    assert m.kernel.grad.abs().sum() > 0 and m.bias.grad.shape == (96,)


def test_captured():
    from approxtrain_b200 import layers
    x, w = _rand(300, 64).requires_grad_(), _rand(64, 48, seed=1).requires_grad_()
    dy = _rand(300, 48, seed=2)

    def step():
        y = layers.mxdense(x, w)
        return [y.detach(), *torch.autograd.grad(y, [x, w], dy)]
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.mul_(3.0)
    graph.replay()
    got = [t.clone() for t in out]
    assert all(torch.equal(u, v) for u, v in zip(got, step()))


def test_a_wait_that_runs_out_is_reported_by_the_next_call(monkeypatch):
    """With no tries at all every warp gives up at its first wait: the launch ends, and the next call says so, once."""
    from approxtrain_b200 import _lib, ops
    shapes = [(10, 300, 300), (16, 128, 8192), (200, 500, 300), (2048, 2048, 512)]     # one CTA a tile, shared by several, pairs
    cases = [(ops.mx_quantize(_rand(m, k)), ops.mx_quantize(_rand(n, k, seed=1))) for m, n, k in shapes]
    want = [ops.mx_matmul(a, b) for a, b in cases]
    for (a, b), w in zip(cases, want):
        monkeypatch.setenv("AMSIM_CODES_SPIN", "0")
        _lib.lib.amsim_debug_reload_env()
        try:
            ops.mx_matmul(a, b)
            torch.cuda.synchronize()
        finally:
            monkeypatch.delenv("AMSIM_CODES_SPIN")
            _lib.lib.amsim_debug_reload_env()
        with pytest.raises(ops.AmsimError, match="gave up waiting"):
            ops.mx_matmul(a, b)
        assert torch.equal(ops.mx_matmul(a, b), w)
    assert _lib.lib.amsim_async_status() == 0


def test_a_layer_in_bf16():
    from approxtrain_b200 import layers
    m = layers.densemx(64, 32, activation="relu").cuda().bfloat16()
    x = _rand(5, 64, t=torch.bfloat16)
    y = m(x)
    y.sum().backward()
    assert y.dtype == torch.bfloat16 and m.bias.grad.dtype == torch.bfloat16 and m.kernel.grad.dtype == torch.bfloat16
    with torch.no_grad():
        assert torch.equal(m.freeze()(x), y)


def test_refusals():
    from approxtrain_b200 import layers, ops
    with pytest.raises(ValueError):
        ops.MXTensor(torch.zeros(100, dtype=torch.uint8, device="cuda"), (4, 64), 1)
    with pytest.raises(ValueError):
        ops.MXTensor(torch.zeros(17408, dtype=torch.uint8, device="cuda"), (4, 64), 2)
    x = torch.zeros(4, 64, device="cuda")
    q = ops.mx_quantize(x)
    for bad in (lambda: ops.mx_quantize(x.double()), lambda: ops.mx_quantize(x[0]), lambda: ops.mx_quantize(x, axis=2), lambda: ops.mx_matmul(q, x),
                lambda: ops.mx_matmul(q, ops.mx_quantize(x[:, :32])), lambda: ops.mx_matmul(q, q, bias=torch.zeros(3, device="cuda")),
                lambda: ops.mx_matmul(q, q, bias=torch.zeros(4)), lambda: ops.mx_matmul(q, q, activation="tanh"), lambda: ops.mx_matmul(q, q, out_dtype=torch.float64),
                lambda: q.dequantize(torch.int32), lambda: layers.mxdense(x, torch.zeros(32, 4, device="cuda"))):
        with pytest.raises((ValueError, TypeError)):
            bad()


def test_frozen_weights_follow_loaded_moved_and_replaced_ones():
    from approxtrain_b200 import layers
    x = _rand(9, 64)
    other = layers.densemx(64, 96).cuda()
    with torch.no_grad():
        want = other(x)
        m = layers.densemx(64, 96).cuda().freeze()
        assert not torch.equal(m(x), want)
        m.load_state_dict(other.state_dict())
        assert torch.equal(m(x), want) and torch.equal(m.freeze()(x), want)
        for assign in (False, True):      # inside a larger module, too
            net = torch.nn.Sequential(layers.densemx(64, 96).cuda().freeze()).eval()
            net.load_state_dict({"0." + k: v.clone() for k, v in other.state_dict().items()}, assign=assign)
            assert torch.equal(net(x), want)
        m = layers.densemx(64, 96).cuda().freeze().cpu()
        m.load_state_dict(other.state_dict())
        assert torch.equal(m.cuda()(x), want)
        m = layers.densemx(64, 96).cuda().freeze()
        m.cpu()
        m.kernel.copy_(other.kernel.cpu())
        m.bias.copy_(other.bias.cpu())
        assert torch.equal(m.cuda()(x), want)
        m = layers.densemx(64, 96).cuda().freeze()
        m.kernel, m.bias = other.kernel, other.bias
        assert torch.equal(m(x), want)


def test_gradients_through_a_frozen_layer():
    from approxtrain_b200 import layers
    m = layers.densemx(64, 96, activation="relu").cuda()
    x, dy = _rand(9, 64), _rand(9, 96, seed=1)
    leaves = [x.clone().requires_grad_(), m.kernel, m.bias]
    y = m(leaves[0])
    want = torch.autograd.grad(y, leaves, dy)
    y2 = m.freeze()(leaves[0])
    assert torch.equal(y2, y)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y2, leaves, dy), want))
    # (with x's gradient unwanted the nine terms of a bias's gradient are added in another order: eight roundings in either)
    alone = torch.autograd.grad(m(x), m.bias, dy)[0]
    assert bool(((alone - want[2]).abs() <= 16 * 2.0 ** -24 * dy.abs().sum(0)).all())
    m.requires_grad_(False)
    assert torch.equal(torch.autograd.grad(m(leaves[0]), leaves[0], dy)[0], want[0])
    assert torch.equal(m(x), y) and not m(x).requires_grad

"""What lies beside the outputs and workspaces of the operators around the table products stays as it was: the C entry points on
buffers with guards on either side."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {0: torch.float32, 1: torch.bfloat16, 2: torch.float16}


class Guarded:
    """Buffers of so many bytes between two stretches of a pattern."""

    SIDE = 512

    def __init__(self):
        self.buffers = []

    def new(self, size, name, off=0):
        buf = torch.full((self.SIDE + off + size + self.SIDE,), 0xA5, dtype=torch.uint8, device="cuda")
        self.buffers.append((buf, self.SIDE + off, size, name))
        return buf.data_ptr() + self.SIDE + off

    def check(self):
        torch.cuda.synchronize()
        for buf, at, size, name in self.buffers:
            assert bool((buf[:at] == 0xA5).all()) and bool((buf[at + size:] == 0xA5).all()), name
        assert any(not bool((buf[at:at + size] == 0xA5).all()) for buf, at, size, _ in self.buffers)


def _lib():
    from approxtrain_b200 import _lib
    return _lib


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _rand(*shape, t=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(t)


def _tensor(buf, at, size, dtype):
    return buf[at:at + size].clone().view(dtype)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows,width", [(1, 1), (7, 33), (21, 96), (5, 130), (300, 512), (1000, 40), (45, 3950), (13, 8200), (6, 20001)])
def test_residual_norm(rows, width, dtype):
    L, t = _lib(), TYPES[dtype]
    e = torch.finfo(t).bits // 8
    x, block, dsum, dy = (_rand(rows, width, t=t, seed=i) for i in range(4))
    w = [_rand(width, seed=10 + i) for i in range(4)]
    for post, gate_rows, off in ((True, 1, 0), (True, rows, 0), (False, 1, e), (False, 0, 0), (True, 0, e)):
        gate = _rand(gate_rows, width, seed=20) if gate_rows else None
        ptr = lambda v: None if v is None else v.data_ptr()
        pw, pb = (w[0], w[1]) if post else (None, None)
        flags = L.NORM_PRE | (L.NORM_POST if post else 0)
        g, size = Guarded(), rows * width * e
        total, y, stats = g.new(size, "sum", off), g.new(size, "y", off), g.new(rows * 16, "stats")
        assert L.lib.amsim_residual_norm(_stream(), ptr(x), ptr(block), ptr(gate), ptr(pw), ptr(pb), ptr(w[2]), ptr(w[3]), total, y, stats, rows, width, gate_rows,
                                         0.5, 1e-3, dtype, 0, 0, flags) == 0
        need = L.lib.amsim_residual_norm_grad_workspace(rows, width, gate is not None, dtype, flags)
        dx, dblock, ws = g.new(size, "dx", off), g.new(size, "dblock", off), g.new(need, "workspace")
        dgate = g.new(gate_rows * width * 4, "dgate") if gate_rows else None
        dw = [g.new(width * 4, n) if on else None for n, on in (("dpost_w", post), ("dpost_b", post), ("dpre_w", True), ("dpre_b", True))]
        assert L.lib.amsim_residual_norm_grad(_stream(), ptr(dsum), ptr(dy), ptr(x), ptr(block), ptr(gate), ptr(pw), ptr(pb), ptr(w[2]), stats, dx, dblock, dgate, *dw,
                                              rows, width, gate_rows, 0.5, dtype, 0, 0, ws, need, flags) == 0
        g.check()


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 33), (33, 3), (128, 128), (129, 257), (200, 100), (1, 600), (600, 1), (300, 1000)])
def test_mx_quantize_and_back(rows, cols, dtype):
    L, t = _lib(), TYPES[dtype]
    e = torch.finfo(t).bits // 8
    x = _rand(rows, cols, t=t)
    for off in (0, e):
        g = Guarded()
        one, two = L.lib.amsim_mx_bytes(rows, cols), L.lib.amsim_mx_bytes(cols, rows)
        need = L.lib.amsim_mx_quantize_workspace(rows, cols)
        along, across, sums, ws = g.new(one, "along"), g.new(two, "across"), g.new(cols * 4, "sums", 4), g.new(need, "workspace")
        assert L.lib.amsim_mx_quantize(_stream(), x.data_ptr(), rows, cols, dtype, along, across, sums, ws, need) == 0
        for data, r, k, turned in ((along, rows, cols, 0), (across, cols, rows, 1), (along, rows, cols, 1)):
            out = g.new(rows * cols * e, "floats", off)
            assert L.lib.amsim_mx_dequantize(_stream(), data, r, k, turned, out, dtype) == 0
        for which in (0, 1):    # one axis alone
            only = g.new((one, two)[which], "one axis")
            assert L.lib.amsim_mx_quantize(_stream(), x.data_ptr(), rows, cols, dtype, None if which else only, only if which else None, None, None, 0) == 0
        g.check()


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (3, 5, 64), (17, 300, 256), (33, 64, 512), (64, 1000, 100), (65, 128, 257), (129, 257, 520), (16, 128, 8192), (40, 130, 9000), (2049, 2047, 64)])
def test_mx_matmul(m, n, k):
    from approxtrain_b200 import ops
    L = _lib()
    a, b, bias = ops.mx_quantize(_rand(m, k)), ops.mx_quantize(_rand(n, k, seed=1)), _rand(n, seed=2)
    for dtype in (0, 1):
        e = 4 if dtype == 0 else 2
        g = Guarded()
        for off in (0, e):
            out = g.new(m * n * e, "out", off)
            assert L.lib.amsim_mx_matmul(_stream(), a.data.data_ptr(), b.data.data_ptr(), m, n, k, bias.data_ptr(), 0, out, dtype) == 0
        g.check()
        want = ops.mx_matmul(a, b, bias=bias, out_dtype=TYPES[dtype])
        for buf, at, size, _ in g.buffers:
            assert torch.equal(_tensor(buf, at, size, TYPES[dtype]).view(m, n), want)

"""Refusals of the operators around the table products; no kernel is launched."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def L():
    from approxtrain_b200 import _build
    _build.build()
    from approxtrain_b200 import _lib
    return _lib


def test_residual_norm_refuses_cpu_tensors_and_other_types(L):
    from approxtrain_b200 import ops
    with pytest.raises(ValueError, match="CUDA"):
        ops.residual_norm(torch.zeros(2, 4), torch.zeros(2, 4), pre=(None, None))
    with pytest.raises(TypeError):
        ops.residual_norm([1.0], pre=(None, None))


def _norm(L, x=1 << 20, block=1 << 21, gate=None, w=(None,) * 4, r=1 << 22, y=1 << 23, stats=None, rows=4, width=8, gate_rows=0,
          scale=1.0, eps=1e-3, types=(0, 0, 0), flags=4):
    """The C entry point with made-up addresses: every call here is refused before anything is launched."""
    return L.lib.amsim_residual_norm(None, x, block, gate, *w, r, y, stats, rows, width, gate_rows, scale, eps, *types, flags)


def test_residual_norm_abi_refusals(L):
    p = 1 << 24
    assert _norm(L, flags=8) == L.ERR_INVALID and b"flag" in L.lib.amsim_last_error()
    assert _norm(L, rows=-1) == L.ERR_INVALID
    assert _norm(L, width=0) == L.ERR_INVALID
    assert _norm(L, width=L.NORM_MAX_WIDTH + 1) == L.ERR_UNSUPPORTED
    assert _norm(L, rows=1 << 40) == L.ERR_UNSUPPORTED
    assert _norm(L, types=(3, 0, 0)) == L.ERR_INVALID
    assert _norm(L, types=(0, 1, 0)) == L.ERR_INVALID
    assert _norm(L, types=(1, 1, 2)) == L.ERR_INVALID
    assert _norm(L, gate=p, gate_rows=3) == L.ERR_INVALID
    assert _norm(L, gate=p, gate_rows=0) == L.ERR_INVALID
    assert _norm(L, block=None, gate=p, gate_rows=1) == L.ERR_INVALID
    assert _norm(L, block=None, flags=6) == L.ERR_INVALID
    assert _norm(L, w=(None, None, None, p), flags=5) == L.ERR_INVALID       # an rms norm's bias
    assert _norm(L, eps=-1.0) == L.ERR_INVALID
    assert _norm(L, eps=float("nan")) == L.ERR_INVALID
    assert _norm(L, flags=0, r=None) == L.ERR_INVALID
    assert _norm(L, x=None) == L.ERR_INVALID
    assert _norm(L, y=None) == L.ERR_INVALID
    assert _norm(L, stats=p + 4) == L.ERR_INVALID
    assert _norm(L, rows=0) == 0


def test_residual_norm_grad_abi_refusals(L):
    p = 1 << 24

    def call(dsum=p, dy=p, r=p, block=p, gate=None, w=(None,) * 3, stats=p, dx=p, dblock=None, dgate=None, dw=(None,) * 4, rows=4,
             width=8, gate_rows=0, ws=p, ws_bytes=1 << 30, flags=4):
        return L.lib.amsim_residual_norm_grad(None, dsum, dy, r, block, gate, *w, stats, dx, dblock, dgate, *dw, rows, width, gate_rows,
                                              1.0, 0, 0, 0, ws, ws_bytes, flags)
    assert call(dsum=None, dy=None) == L.ERR_INVALID
    assert call(dx=None) == L.ERR_INVALID
    assert call(stats=None) == L.ERR_INVALID
    assert call(r=None) == L.ERR_INVALID
    assert call(flags=6, block=None) == L.ERR_INVALID
    assert call(dgate=p) == L.ERR_INVALID
    assert call(dw=(p, None, None, None)) == L.ERR_INVALID                   # no norm after the block
    assert call(flags=0) == L.ERR_INVALID                                    # a gradient of a norm that there is not
    assert call(flags=5, dw=(None, None, None, p)) == L.ERR_INVALID
    assert call(ws=None) == L.ERR_WORKSPACE
    assert call(ws_bytes=16) == L.ERR_WORKSPACE
    assert call(ws=p + 8) == L.ERR_WORKSPACE
    assert L.lib.amsim_residual_norm_grad_workspace(0, 8, 0, 0, 4) == 0
    assert L.lib.amsim_residual_norm_grad_workspace(1000, 8, 1, 0, 4) > L.lib.amsim_residual_norm_grad_workspace(1000, 8, 0, 0, 4) > 0


def test_gate_shapes():
    from approxtrain_b200.train_ops import _gate_rows
    x = torch.zeros(3, 5, 7, 4)
    assert _gate_rows(torch.zeros(4), x) == 1
    assert _gate_rows(torch.zeros(1, 1, 1, 4), x) == 1
    assert _gate_rows(torch.zeros(3, 1, 1, 4), x) == 3
    assert _gate_rows(torch.zeros(3, 5, 1, 4), x) == 15
    assert _gate_rows(x, x) == 105
    for bad in ((3,), (1, 5, 1, 4), (3, 1, 7, 4), (3, 5, 7, 1), (5, 4), (3, 2, 1, 4)):
        with pytest.raises(ValueError, match="gate"):
            _gate_rows(torch.zeros(bad), x)


def test_rotary_refusals(L):
    from approxtrain_b200 import ops
    with pytest.raises(ValueError, match="CUDA"):
        ops.rotary(torch.zeros(1, 2, 1, 8), torch.arange(2), None)
    for kw in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, scaling="other"),
               dict(rotary_dim=8, scaling="blend"), dict(rotary_dim=8, scaling="linear", factor=-1.0)):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(device="cpu", **kw)
    with pytest.raises(ValueError, match="CUDA"):
        ops.RotaryFrequencies(torch.ones(4, dtype=torch.float64))
    with pytest.raises(TypeError):
        ops.RotaryFrequencies(torch.ones(4))
    p = 1 << 20
    strides = (C.c_longlong * 14)(64, 16, 8, 64, 16, 8, 64, 16, 8, 64, 16, 8, 0, 1)

    def call(x=p, out=2 * p, heads=2, x2=None, out2=None, heads2=0, pos=p, freqs=p, batch=1, seq=4, dim=8, rot=8, st=strides, dtype=0, flags=0):
        return L.lib.amsim_rotary(None, x, out, heads, x2, out2, heads2, pos, freqs, batch, seq, dim, rot, st, 1.0, dtype, flags)
    assert call(flags=8) == L.ERR_INVALID
    assert call(dtype=3) == L.ERR_INVALID
    assert call(batch=-1) == L.ERR_INVALID
    assert call(rot=0) == L.ERR_INVALID and call(rot=7) == L.ERR_INVALID and call(rot=10) == L.ERR_INVALID
    assert call(dim=20000, rot=20000) == L.ERR_UNSUPPORTED
    assert call(batch=1 << 31) == L.ERR_UNSUPPORTED
    assert call(batch=1 << 21, seq=1 << 21) == L.ERR_UNSUPPORTED
    assert call(x=None) == L.ERR_INVALID and call(pos=None) == L.ERR_INVALID and call(freqs=None) == L.ERR_INVALID and call(st=None) == L.ERR_INVALID
    assert call(heads2=1) == L.ERR_INVALID
    other = (C.c_longlong * 14)(64, 16, 8, 64, 16, 4, 0, 0, 0, 0, 0, 0, 0, 1)
    assert call(out=p, st=other) == L.ERR_INVALID and b"in place" in L.lib.amsim_last_error()
    assert call(batch=0) == 0 and call(heads=0) == 0


def test_adamw_abi_refusals(L):
    import array
    p = 1 << 20
    one = array.array("Q", [p, p])
    n = array.array("q", [8, 3])
    dec = array.array("f", [0.0, 0.0])
    at = lambda a: a.buffer_info()[0]

    def call(tensors=2, params=at(one), grads=at(one), sizes=at(n), decay=at(dec), m=p, ms=None, v=p, vs=None, step=p, b1=0.9, b2=0.99, eps=1e-8,
             types=(0, 0), bits=32):
        return L.lib.amsim_adamw(None, tensors, params, grads, sizes, decay, m, ms, v, vs, step, 0.1, None, b1, b2, eps, 1.0, None, 0, *types, bits)
    assert call(tensors=-1) == L.ERR_INVALID
    assert call(bits=16) == L.ERR_INVALID
    assert call(types=(3, 0)) == L.ERR_INVALID and call(types=(1, 2)) == L.ERR_INVALID and call(types=(0, 1)) == L.ERR_INVALID
    assert call(b1=1.0) == L.ERR_INVALID and call(b2=-0.1) == L.ERR_INVALID and call(eps=float("nan")) == L.ERR_INVALID
    assert call(step=None) == L.ERR_INVALID and call(params=None) == L.ERR_INVALID and call(decay=None) == L.ERR_INVALID
    assert call(m=None) == L.ERR_INVALID and call(m=p + 4) == L.ERR_INVALID and call(bits=8) == L.ERR_INVALID
    bad = array.array("q", [8, -1])
    assert call(sizes=at(bad)) == L.ERR_INVALID
    null = array.array("Q", [p, 0])
    assert call(grads=at(null)) == L.ERR_INVALID


def test_adamw_refuses_cpu_tensors(L):
    from approxtrain_b200 import ops
    with pytest.raises(ValueError, match="CUDA"):
        ops.AdamWState([torch.zeros(3)])


def test_mx_refusals(L):
    from approxtrain_b200 import ops
    with pytest.raises(ValueError, match="CUDA"):
        ops.mx_quantize(torch.zeros(2, 4))
    p = 1 << 20
    from approxtrain_b200 import mx
    for rows in (0, 1, 127, 128, 129, 5000):
        for k in (0, 1, 255, 256, 257, 9000):
            assert mx._bytes(rows, k) == L.lib.amsim_mx_bytes(rows, k)
            assert -(-rows // 128) * k * 4 == L.lib.amsim_mx_quantize_workspace(rows, k)
    d, m = L.lib.amsim_mx_dequantize, L.lib.amsim_mx_matmul

    def q(stream, x, rows, cols, dtype, along, across, sums=None, ws=None, size=0):
        return L.lib.amsim_mx_quantize(stream, x, rows, cols, dtype, along, across, sums, ws, size)
    assert q(None, p, 4, 4, 0, p, None, sums=p, ws=p, size=1 << 20) == L.ERR_INVALID
    assert q(None, p, 4, 4, 0, p, p, sums=p) == L.ERR_WORKSPACE and q(None, p, 4, 4, 0, p, p, sums=p, ws=p, size=8) == L.ERR_WORKSPACE
    assert L.lib.amsim_mx_bytes(1, 1) == 17408 and L.lib.amsim_mx_bytes(129, 257) == 4 * 17408 and L.lib.amsim_mx_bytes(0, 5) == 0 and L.lib.amsim_mx_bytes(5, 0) == 17408
    assert q(None, p, -1, 4, 0, p, None) == L.ERR_INVALID and q(None, p, 4, 4, 3, p, None) == L.ERR_INVALID
    assert q(None, p, 4, 4, 0, None, None) == L.ERR_INVALID and q(None, None, 4, 4, 0, p, None) == L.ERR_INVALID
    assert q(None, p, 4, 4, 0, p + 8, None) == L.ERR_INVALID and q(None, p, 1 << 31, 4, 0, p, None) == L.ERR_UNSUPPORTED
    assert q(None, p, 1 << 21, 1 << 21, 0, p, None) == L.ERR_UNSUPPORTED
    assert q(None, None, 0, 4, 0, p, None) == 0
    assert d(None, p, 4, -1, 0, p, 0) == L.ERR_INVALID and d(None, None, 4, 4, 0, p, 0) == L.ERR_INVALID and d(None, p + 4, 4, 4, 0, p, 0) == L.ERR_INVALID
    assert d(None, p, 4, 4, 0, p, 5) == L.ERR_INVALID and d(None, None, 0, 4, 0, None, 0) == 0
    assert m(None, p, p, -1, 4, 4, None, 0, p, 0) == L.ERR_INVALID and m(None, p, p, 4, 4, 4, None, 2, p, 0) == L.ERR_INVALID
    assert m(None, p, p, 4, 4, 4, None, 0, p, 3) == L.ERR_INVALID and m(None, None, p, 4, 4, 4, None, 0, p, 0) == L.ERR_INVALID
    assert m(None, p + 8, p, 4, 4, 4, None, 0, p, 0) == L.ERR_INVALID and m(None, p, p, 1 << 30, 1 << 30, 4, None, 0, p, 0) == L.ERR_UNSUPPORTED
    assert m(None, p, p, 0, 4, 4, None, 0, p, 0) == 0


def test_tensors_that_overlap_are_told_from_those_that_do_not():
    import random
    from approxtrain_b200.train_ops import _repeats_elements, _share_elements
    buf = torch.zeros(4000)
    rng = random.Random(5)

    def places(t):
        at = torch.tensor(t.storage_offset())
        for n, st in zip(t.shape, t.stride()):
            at = at[..., None] + st * torch.arange(n)
        return at.flatten().tolist()

    def view():
        shape = [rng.randrange(1, 4) for _ in range(4)]
        strides = [rng.choice([0, 1, 2, 3, 5, 8, 12, 24, 40, 60]) for _ in range(4)]
        return buf.as_strided(shape, strides, rng.randrange(0, 120))
    shared = apart = 0
    for _ in range(3000):
        a, b = view(), view()
        both = bool(set(places(a)) & set(places(b)))
        assert _share_elements(a, b) == both == _share_elements(b, a)
        shared, apart = shared + both, apart + (not both)
        assert _repeats_elements(a) or len(set(places(a))) == a.numel()
    assert shared > 300 and apart > 300
    # what a model hands over: parts of one projection, by head or interleaved, and of one buffer
    joint = torch.zeros(2, 9, 3 * 4 * 48)
    q, k = joint[..., :192].unflatten(-1, (4, 48)), joint[..., 192:288].unflatten(-1, (2, 48))
    assert not _share_elements(q, k) and not _repeats_elements(q) and _share_elements(q, joint[..., 144:240].unflatten(-1, (2, 48)))
    three = joint.unflatten(-1, (4, 3, 48))
    assert not _share_elements(three[..., 0, :], three[..., 1, :]) and _share_elements(three[..., 1, :], three[..., 1, :])
    flat = torch.zeros(2 * 6 * 9 * 48)
    q, k = flat[:2 * 4 * 9 * 48].view(2, 4, 9, 48).transpose(1, 2), flat[2 * 4 * 9 * 48:].view(2, 2, 9, 48).transpose(1, 2)
    assert not _share_elements(q, k) and not _repeats_elements(q) and not _repeats_elements(k)
    assert not _share_elements(q[:0], q) and not _repeats_elements(q[:0])
    assert _repeats_elements(flat.as_strided((3, 5, 2, 8), (0, 8, 4, 1))) and _repeats_elements(flat[:48].expand(9, 4, 48))
    # (strides that make it a long search count as shared)
    wide = torch.zeros(1).as_strided((1, 1, 1, 1), (1, 1, 1, 1))
    assert not _share_elements(wide, torch.zeros(1, 1, 1, 1))


def test_rotary_of_one_output_twice_is_refused(L):
    p = 1 << 20
    strides = (C.c_longlong * 14)(64, 16, 8, 64, 16, 8, 64, 16, 8, 64, 16, 8, 0, 1)

    def call(x2, out2):
        return L.lib.amsim_rotary(None, p, p, 2, x2, out2, 2, p, p, 1, 4, 8, 8, strides, 1.0, 0, 0)
    assert call(p, p) == L.ERR_INVALID and b"same output" in L.lib.amsim_last_error()
    assert call(2 * p, p) == L.ERR_INVALID


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
def test_gradients_of_the_adamw_trainer_begin_at_16_bytes(t):
    from approxtrain_b200.dp import DataParallelAdamW, DataParallelSGD
    sizes = [1, 5, 12, 4, 7, 300]
    for cls in (DataParallelAdamW, DataParallelSGD):
        tr = object.__new__(cls)
        tr.buckets = []
        params = [torch.nn.Parameter(torch.zeros(n, dtype=t)) for n in sizes]
        tr._close_bucket(params)
        flat = tr.buckets[0]["flat"]
        at = [(p.grad.data_ptr() - flat.data_ptr()) for p in params]
        if cls is DataParallelAdamW:
            assert all(a % 16 == 0 for a in at)
        else:
            assert flat.numel() == sum(sizes)
        ends = [a + n * flat.element_size() for a, n in zip(at, sizes)]
        assert all(e <= a for e, a in zip(ends, at[1:])) and ends[-1] <= flat.numel() * flat.element_size()

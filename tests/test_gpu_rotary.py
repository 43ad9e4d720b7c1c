"""rotary against the rotation in 64 bits."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _plain(x, positions, inv_freq, scale, layout, inverse=False):
    """x [batch, positions, heads, dim] as complex products in 64 bits."""
    x = x.detach().double()
    half = inv_freq.numel()
    rot = 2 * half
    angle = positions.double().reshape(-1 if positions.dim() == 1 else positions.shape[0], positions.shape[-1])[..., None, None] * inv_freq if positions.dim() == 2 \
        else (positions.double()[:, None, None] * inv_freq)[None]
    turn = scale * torch.polar(torch.ones_like(angle), -angle if inverse else angle)
    a, b = (x[..., :half], x[..., half:rot]) if layout == "half" else (x[..., 0:rot:2], x[..., 1:rot:2])
    z = torch.complex(a, b) * turn
    out = x.clone()
    if layout == "half":
        out[..., :half], out[..., half:rot] = z.real, z.imag
    else:
        out[..., 0:rot:2], out[..., 1:rot:2] = z.real, z.imag
    return out


def _close(got, want, x, scale, rot):
    """One rounding to the type; the turn is rounded to FP32 (2^-25 of half a turn: 2^-25 pi), sincospif is good to two steps of FP32
    (2^-22), scale and three products and sums a half step each (2^-22 together), all times the pair's length, at most sqrt(2) times
    the larger of its elements.  Copied elements are equal."""
    t = got.dtype
    assert got.shape == want.shape
    size = 1.5 * abs(scale) * x.detach().double()[..., :rot].abs().amax(-1, keepdim=True)
    tol = torch.finfo(t).eps / 2 * want.abs() + (2.0 ** -23 + 2.0 ** -21) * size + torch.finfo(t).smallest_normal
    assert bool(((got.double() - want).abs() <= tol)[..., :rot].all()), float(((got.double() - want).abs() - tol)[..., :rot].max())
    assert torch.equal(got[..., rot:], x.detach()[..., rot:])


def _rand(*shape, t=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(t)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(64, 64), (128, 64), (128, 96), (80, 80), (2, 2), (7, 6), (33, 2), (256, 256), (96, 50), (257, 128), (1024, 1024)])
def test_layouts_and_sizes(t, layout, dim, rot):
    from approxtrain_b200 import layers, ops
    freqs = ops.rotary_frequencies(rot)
    for batch, seq, heads, kv in ((1, 1, 1, 1), (3, 17, 4, 2), (2, 130, 6, 1)):
        q, k = _rand(batch, seq, heads, dim, t=t), _rand(batch, seq, kv, dim, t=t, seed=1)
        for positions in (torch.arange(seq, device="cuda"), torch.randint(0, 5000, (batch, seq), device="cuda", dtype=torch.int32)):
            gq, gk = ops.rotary(q, positions, freqs, k=k, layout=layout)
            _close(gq, _plain(q, positions, freqs.inv_freq, 1.0, layout), q, 1.0, rot)
            _close(gk, _plain(k, positions, freqs.inv_freq, 1.0, layout), k, 1.0, rot)
            back = ops.rotary(q, positions, freqs, layout=layout, inverse=True)
            _close(back, _plain(q, positions, freqs.inv_freq, 1.0, layout, True), q, 1.0, rot)
            leaves = [q.clone().requires_grad_(), k.clone().requires_grad_()]
            outs = layers.rotary(leaves[0], positions, freqs, k=leaves[1], layout=layout)
            assert torch.equal(outs[0], gq) and torch.equal(outs[1], gk)
            dq, dk = torch.autograd.grad(outs, leaves, [q, k])
            assert torch.equal(dq, back)
            _close(dk, _plain(k, positions, freqs.inv_freq, 1.0, layout, True), k, 1.0, rot)
            only, = torch.autograd.grad(layers.rotary(leaves[0], positions, freqs, k=leaves[1], layout=layout)[1], leaves[1], k)
            assert torch.equal(only, dk)


@pytest.mark.parametrize("scaling", [dict(), dict(scaling="linear", factor=8.0), dict(scaling="base", factor=4.0),
                                     dict(scaling="blend", factor=16.0, original_length=4096)])
def test_far_positions_and_scaled_frequencies(scaling):
    from approxtrain_b200 import ops
    freqs = ops.rotary_frequencies(64, **scaling)
    for first in (0, 131071, 999999, 2 ** 31 - 64, -70, 2 ** 40):
        # 64-bit angles of such positions are good to first * 2^-53 turns
        positions = first + torch.arange(50, device="cuda")
        q = _rand(1, 50, 3, 64)
        got = ops.rotary(q, positions, freqs)
        if abs(first) < 2 ** 32:
            _close(got, _plain(q, positions, freqs.inv_freq, freqs.scale, "half"), q, freqs.scale, 64)
        assert bool(got.isfinite().all())


def test_frequencies():
    from approxtrain_b200 import ops
    f = ops.rotary_frequencies(64).inv_freq
    assert float(f[0]) == 1.0 and abs(float(f[-1]) - 10000 ** (-62 / 64)) < 1e-15
    assert torch.allclose(ops.rotary_frequencies(64, scaling="linear", factor=4.0).inv_freq, f / 4, rtol=1e-15)
    assert abs(float(ops.rotary_frequencies(64, scaling="base", factor=4.0).inv_freq[-1] / f[-1]) - 0.25) < 1e-12
    b = ops.rotary_frequencies(64, scaling="blend", factor=4.0, original_length=2048)
    assert float(b.inv_freq[0]) == 1.0 and abs(float(b.inv_freq[-1] / f[-1]) - 0.25) < 1e-12 and abs(b.scale - (0.1 * 1.3862943611198906 + 1)) < 1e-12


def test_strided_tensors_and_in_place():
    from approxtrain_b200 import ops
    freqs = ops.rotary_frequencies(32)
    positions = torch.arange(9, device="cuda")
    for t in (torch.float32, torch.bfloat16):
        joint = _rand(2, 9, 3 * 4 * 48 + 1, t=t)
        first = _rand(2, 4, 9, 48, t=t, seed=2).transpose(1, 2)                     # [batch, heads, positions, dim]
        odd = joint[..., 1:1 + 4 * 48].unflatten(-1, (4, 48))                        # not 16-byte aligned
        wide = joint[..., :8 * 48].unflatten(-1, (8, 48))[:, :, ::2]                  # every other head
        last = _rand(2, 9, 4, 96, t=t, seed=3)[..., ::2]                             # no dense last axis: copied
        packed = _rand(9, 4, 48, t=t, seed=4)                                        # no batch
        for x in (first, odd, wide, last):
            got = ops.rotary(x, positions, freqs)
            _close(got, _plain(x, positions, freqs.inv_freq, 1.0, "half"), x, 1.0, 32)
        _close(ops.rotary(packed, positions, freqs)[None], _plain(packed[None], positions, freqs.inv_freq, 1.0, "half"), packed[None], 1.0, 32)
        shared = positions.flip(0)[None].expand(2, 9)
        _close(ops.rotary(first, shared, freqs), _plain(first, shared, freqs.inv_freq, 1.0, "half"), first, 1.0, 32)
        _close(ops.rotary(first, torch.arange(18, device="cuda")[::2], freqs), _plain(first, 2 * positions, freqs.inv_freq, 1.0, "half"), first, 1.0, 32)
        for x in (first, odd, wide):
            was = joint.clone()
            want = ops.rotary(x, positions, freqs)
            keep = x.clone()
            assert ops.rotary(x, positions, freqs, inplace=True) is x
            assert torch.equal(x, want)
            x.copy_(keep)
            assert torch.equal(joint, was)                                           # nothing beside it was written
        with pytest.raises(ValueError):
            ops.rotary(last, positions, freqs, inplace=True)
        with pytest.raises(ValueError, match="gradient"):
            ops.rotary(packed.clone().requires_grad_(), positions, freqs, inplace=True)
        version = packed._version
        ops.rotary(packed, positions, freqs, inplace=True)
        assert packed._version == version + 1
        with pytest.raises(ValueError):
            ops.rotary(packed[:1].expand(9, 4, 48), positions, freqs, inplace=True)


def test_empty_and_refused():
    from approxtrain_b200 import ops
    freqs = ops.rotary_frequencies(16)
    pos = torch.arange(3, device="cuda")
    assert ops.rotary(torch.zeros(0, 3, 2, 16, device="cuda"), pos, freqs).shape == (0, 3, 2, 16)
    assert ops.rotary(torch.zeros(2, 0, 2, 16, device="cuda"), pos[:0], freqs).shape == (2, 0, 2, 16)
    assert ops.rotary(torch.zeros(2, 3, 0, 16, device="cuda"), pos, freqs).shape == (2, 3, 0, 16)
    q = torch.zeros(2, 3, 2, 16, device="cuda")
    for bad in (lambda: ops.rotary(q, pos[:2], freqs), lambda: ops.rotary(q, pos.float(), freqs), lambda: ops.rotary(q[..., :8], pos, freqs),
                lambda: ops.rotary(q, pos, freqs, layout="other"), lambda: ops.rotary(q, pos, freqs, k=q.half()), lambda: ops.rotary(q, pos, freqs, k=q[:, :2]),
                lambda: ops.rotary(q[0, 0], pos, freqs), lambda: ops.rotary(q, pos.cpu(), freqs), lambda: ops.rotary(q, pos, freqs.inv_freq),
                lambda: ops.rotary(q.int(), pos, freqs)):
        with pytest.raises((ValueError, TypeError)):
            bad()


def test_large_offsets():
    """Element offsets past 2^31: the last of many positions."""
    from approxtrain_b200 import ops
    freqs = ops.rotary_frequencies(64)
    seq = (2 ** 31) // (32 * 128) + 3
    q = torch.zeros(seq, 32, 128, dtype=torch.bfloat16, device="cuda")
    q[-2:] = _rand(2, 32, 128, t=torch.bfloat16)
    positions = torch.arange(seq, device="cuda")
    got = ops.rotary(q, positions, freqs)
    _close(got[None, -2:], _plain(q[None, -2:], positions[-2:], freqs.inv_freq, 1.0, "half"), q[None, -2:], 1.0, 64)
    assert not got[:-2].any()


def test_on_another_stream_and_in_a_graph():
    from approxtrain_b200 import ops
    freqs = ops.rotary_frequencies(64)
    q, positions = _rand(4, 100, 8, 64), torch.arange(100, device="cuda")
    want = ops.rotary(q, positions, freqs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.rotary(q, positions, freqs)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.rotary(q, positions, freqs)
    positions += 7
    graph.replay()
    assert torch.equal(out, ops.rotary(q, positions, freqs)) and not torch.equal(out, want)


def test_in_place_beside_each_other_and_overlapping():
    """Both tensors in place: parts of one projection are turned, tensors that share elements are refused as they are."""
    from approxtrain_b200 import ops
    freqs = ops.rotary_frequencies(32)
    positions = torch.arange(9, device="cuda")
    for t in (torch.float32, torch.bfloat16):
        joint = _rand(2, 9, 8 * 48, t=t)
        was = joint.clone()
        heads = joint.unflatten(-1, (8, 48))
        three = _rand(2, 9, 4 * 3 * 48, t=t, seed=1).unflatten(-1, (4, 3, 48))
        for q, k in ((heads[:, :, :5], heads[:, :, 5:7]), (three[..., 0, :], three[..., 1, :])):
            want = ops.rotary(q, positions, freqs, k=k)
            got = ops.rotary(q, positions, freqs, k=k, inplace=True)
            assert got[0] is q and got[1] is k and torch.equal(q, want[0]) and torch.equal(k, want[1])
        assert torch.equal(heads[:, :, 7], was.unflatten(-1, (8, 48))[:, :, 7])
        before = joint.clone()
        for q, k in ((heads, heads), (heads[:, :, :5], heads[:, :, 4:]), (heads[:, :, ::2], heads[:, :, 2:4])):
            with pytest.raises(ValueError, match="share"):
                ops.rotary(q, positions, freqs, k=k, inplace=True)
        with pytest.raises(ValueError, match="overlap"):
            ops.rotary(joint.as_strided((9, 4, 48), (48, 48, 1)), positions, freqs, inplace=True)
        assert torch.equal(joint, before)
        assert all(torch.equal(x, y) for x, y in zip(ops.rotary(heads, positions, freqs, k=heads), [ops.rotary(heads, positions, freqs)] * 2))

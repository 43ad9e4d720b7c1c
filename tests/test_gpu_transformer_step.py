"""The operators around the table products as they are used together: training steps of TransformerAM with fused norms, rotary
positions, 4-bit dense layers and AdamW, eager and replayed from a graph."""
import pytest

from conftest import lut_path

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

SMALL = dict(vocab=120, layers=2, d_model=64, heads=4, d_ff=96, d_k=64, d_v=64)


def _net(**kw):
    from approxtrain_b200 import nets
    torch.manual_seed(3)
    return nets.TransformerAM(lut_path("MIT_7"), **SMALL, **kw).cuda()


def _batch(seed=0, b=3, s=21, t=17):
    g = torch.Generator(device="cuda").manual_seed(seed)
    src, tgt = (torch.randint(1, 120, (b, n), generator=g, device="cuda") for n in (s, t))
    src[0, 15:], tgt[1, 9:] = 0, 0           # padding
    return src, tgt


def _loss(net, src, tgt):
    return torch.nn.functional.cross_entropy(net(src, tgt).flatten(0, 1), tgt.flatten())


def test_defaults_are_as_before():
    a, b = _net(), _net(fused_norms=False, positions="sinusoidal", dense="am")
    src, tgt = _batch()
    assert torch.equal(a(src, tgt), b(src, tgt))
    assert list(a.state_dict()) == list(_net(fused_norms=True, positions="rotary", dense="mx").state_dict())


def test_fused_norms_give_the_unfused_gradients():
    """Exact dense layers stand in for the table's, whose truncation turns a rounding into a step of 2^-7."""
    from approxtrain_b200 import nets

    class Exact(torch.nn.Module):
        def __init__(self, i, o, activation=None, **kw):
            super().__init__()
            self.kernel = torch.nn.Parameter(torch.randn(i, o) / i ** 0.5)
            self.act = activation

        def forward(self, x):
            y = x @ self.kernel
            return torch.relu(y) if self.act else y
    torch.manual_seed(0)
    ffn = nets._FFN(None, 96, 64, False, "mx")
    ffn.f1, ffn.f2 = Exact(64, 96, "relu"), Exact(96, 64)
    ffn = ffn.cuda()
    norms = [torch.nn.LayerNorm(64, eps=1e-3).cuda() for _ in range(2)]
    x0 = torch.randn(4, 9, 64, device="cuda")
    grads = []
    for fused in (False, True):
        x = x0.clone().requires_grad_()
        y = x
        for n in norms:
            y = nets._add_norm(n, y, ffn(y), fused)
        ps = [p for n in norms for p in n.parameters()] + list(ffn.parameters())
        grads.append([y.detach(), *torch.autograd.grad(y.square().sum() + y.sum(), [x, *ps])])
    # The gradient 2 y + 1 at the last norm's output lies in the directions that its backward pass takes out (weights 1, bias 0):
    # what comes out is a difference of terms of that size, |2 y + 1|.  Each of the two norms and two products behind it
    # rounds terms of that size about four times, in either chain: 2 x 4 x 4 roundings.  A weight's gradient is a product of that
    # error with the activations, which lengthens it by their spectral norm at most.
    y = grads[0][0].flatten(0, 1)
    left = 32 * 2.0 ** -24 * float((2 * y + 1).norm()) * (1 + float(torch.linalg.matrix_norm(y, 2)))
    for a, b in zip(*grads):
        assert float((a - b).norm()) <= 2e-5 * float(b.norm()) + left


def test_rotary_attention_depends_on_distance_only():
    """Scores of rotated queries and keys: the same for every shift of the positions."""
    from approxtrain_b200 import ops
    q, k = torch.randn(1, 6, 2, 16, device="cuda"), torch.randn(1, 6, 2, 16, device="cuda")
    freqs = ops.rotary_frequencies(16)
    scores = []
    for shift in (0, 1000):
        a, b = ops.rotary(q, shift + torch.arange(6, device="cuda"), freqs, k=k)
        scores.append(torch.einsum("bshd,bthd->bhst", a.double(), b.double()))
    # each rotated element carries about three roundings of FP32 of its size; 16 products a score
    assert float((scores[0] - scores[1]).abs().max()) <= 16 * 8 * 2.0 ** -24 * float(q.abs().max() * k.abs().max()) * 2


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dense", ["am", "mx"])
def test_training_steps_eager_and_replayed(dense, bits):
    from approxtrain_b200.dp import DataParallelAdamW
    src, tgt = _batch()
    seen, finals = [], []
    for captured in (False, True):
        net = _net(fused_norms=True, positions="rotary", dense=dense)
        tr = DataParallelAdamW(net, 1e-3, state_bits=bits, seed=1)
        loss_fn = lambda: _loss(net, src, tgt)
        if captured:
            replay = tr.capture(loss_fn, warmup=3)
            losses = [float(replay()) for _ in range(3)]
        else:
            losses = [float(tr.step(loss_fn)) for _ in range(6)][3:]
        assert int(tr.state.step) == 6
        assert all(torch.isfinite(torch.tensor(v)) for v in losses)
        assert all(p.grad.abs().sum() > 0 for n, p in net.named_parameters() if not n.endswith("wk.bias"))
        seen.append(losses)
        finals.append([p.detach().clone() for p in net.parameters()])
    if dense == "mx":   # (the table layers' small captured launches sum in another order than eager ones)
        assert seen[0] == seen[1]
        assert all(torch.equal(a, b) for a, b in zip(*finals))


def test_saved_and_resumed():
    from approxtrain_b200.dp import DataParallelAdamW
    src, tgt = _batch()
    net = _net(fused_norms=True, positions="rotary", dense="mx")
    tr = DataParallelAdamW(net, 1e-3, state_bits=8)
    for _ in range(2):
        tr.step(lambda: _loss(net, src, tgt))
    saved = {k: v.clone() for k, v in net.state_dict().items()}, tr.state_dict()
    want = float(tr.step(lambda: _loss(net, src, tgt)))
    want2 = float(tr.step(lambda: _loss(net, src, tgt)))
    again = _net(fused_norms=True, positions="rotary", dense="mx")
    again.load_state_dict(saved[0])
    tr2 = DataParallelAdamW(again, 5e-4, state_bits=8)
    tr2.load_state_dict(saved[1])
    assert float(tr2.step(lambda: _loss(again, src, tgt))) == want
    assert float(tr2.step(lambda: _loss(again, src, tgt))) == want2


def test_bad_options_are_refused():
    from approxtrain_b200 import nets
    for kw in (dict(positions="none"), dict(dense="fp4")):
        with pytest.raises(ValueError):
            nets.TransformerAM(lut_path("MIT_7"), **SMALL, **kw)

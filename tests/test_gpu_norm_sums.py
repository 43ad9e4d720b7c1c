"""The column sums of residual_norm's gradient (weights, biases, gate): each column against a bound made of its own terms, and all of
them by norm, so that a lost row, a swapped line or zeros cannot pass."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_residual_norm import F32, _make, _plain, _plain_grad

ROUNDINGS = 64    # of a row's values: 16 elements a thread, 9 levels of threads and 3 of CTAs, twice, and a dozen products
# A column's sum: the rows of a worker (4 at the cases below), the 64 workers of a CTA or 16 shares of up to 2048 workers' slots
# (128 each), and the 16 shares
DEPTH = 4 + 64 + 128 + 16


def _top(t):
    return t.abs().amax(-1, keepdim=True)


def _terms(a, dr, dy):
    """name -> (the rows' terms, how far each may be off for the roundings of its row), in 64 bits."""
    d = lambda t: t.detach().double()
    r, _, s = _plain(**a)
    unit = ROUNDINGS * F32
    gate = d(a["gate"]) if a["gate"] is not None else torch.ones((), dtype=torch.float64, device="cuda")
    k = abs(a["scale"])
    out = {}
    if a["post"] is not None:
        post_w = d(a["post"][0])
        e_ph = unit * (_top(d(a["block"])) * s["pr"] + _top(s["ph"]))
        e_u = post_w.abs().max() * e_ph + unit * _top(s["u"])
    else:
        e_u = torch.zeros_like(_top(s["u"]))
    size_r = _top(d(a["x"])) + k * _top(s["u"] * gate)
    pre_w = d(a["pre"][0])
    e_h = (unit * (size_r + _top(r)) + k * gate.abs().max() * e_u) * s["r"] + unit * _top(s["h"])
    out["pre_w"] = d(dy) * s["h"], d(dy).abs() * e_h
    out["pre_b"] = d(dy), torch.zeros_like(d(dy))
    # g = dr + rstd (a - mean a - hat mean(a hat)), a = dy w
    a_top = _top(d(dy) * pre_w)
    e_g = unit * (s["r"] * a_top * (2 + _top(s["h"]) ** 2) + _top(d(dr))) + 2 * s["r"] * a_top * _top(s["h"]) * e_h
    g = _plain_grad(s, a["block"], a["gate"], a["scale"], a["post"], a["pre"], a["kind"], dr, dy)["x"]
    if a["gate"] is not None:
        out["gate"] = a["scale"] * s["u"] * g, k * (s["u"].abs() * e_g + g.abs() * e_u)
    if a["post"] is not None:
        du, e_du = a["scale"] * gate * g, k * gate.abs() * e_g
        out["post_w"] = du * s["ph"], s["ph"].abs() * e_du + du.abs() * e_ph
        out["post_b"] = du, e_du.expand_as(du)
    return out


def _sum_like(rows, v):
    """The sum of the rows' terms in v's shape."""
    if v.dim() == 1:
        return rows.flatten(0, -2).sum(0)
    shared = [i for i in range(rows.dim()) if v.shape[i] == 1 and rows.shape[i] != 1]
    return rows.sum(shared, keepdim=True) if shared else rows


def _faults(got, v, terms, off):
    """What is wrong with a gradient: columns past their bound, or the norm of the error."""
    want = _sum_like(terms, v)
    half = torch.finfo(v.dtype).eps / 2 if v.dtype != torch.float32 else 0.0
    tol = _sum_like(off, v) + DEPTH * F32 * _sum_like(terms.abs(), v) + half * want.abs()
    err = (got.double() - want).abs()
    # roundings are as likely up as down: 64 of a row and the depth of a sum come to the root of their number, of terms that differ in
    # size by a factor of up to four
    by_norm = 4 * (ROUNDINGS + DEPTH) ** 0.5 * F32 * _sum_like(terms.square(), v).sqrt().norm() + half * want.norm()
    return int((err > tol).sum()), float(err.norm() / by_norm)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("shape", [(37, 1, 512), (3, 7, 96), (1000, 1, 64), (4, 250, 64), (8192, 1, 24), (2, 4096, 24), (5, 9, 3950), (4099, 1, 300), (5, 60, 8200), (3, 20, 32768)],
                         ids=lambda s: "x".join(map(str, s)))
def test_column_sums(shape, kind, t):
    from approxtrain_b200 import layers
    for post, gate in ((True, "width"), (True, "sequence"), (False, "width"), (False, "sequence"), (True, None), (False, None)):
        a, rnd = _make(shape, t, kind, post, gate, True, 0.75, True, torch.float32, seed=shape[-1])
        dr, dy = rnd(*shape, k=0.1), rnd(*shape, k=0.1)
        leaves = dict(gate=a["gate"], pre_w=a["pre"][0], pre_b=a["pre"][1])
        if post:
            leaves.update(post_w=a["post"][0], post_b=a["post"][1])
        leaves = {k: v for k, v in leaves.items() if v is not None}
        terms = _terms(a, dr, dy)
        for v in leaves.values():
            v.requires_grad_()
        got = torch.autograd.grad(layers.residual_norm(**a), list(leaves.values()), [dr, dy])
        for (name, v), g in zip(leaves.items(), got):
            rows, off = terms[name]
            assert g.shape == v.shape
            columns, norm = _faults(g, v, rows, off)
            assert columns == 0 and norm <= 1, (name, post, gate, columns, norm)
            # the check itself: zeros, and a sum without its last row (where rows are added at all), do not pass
            assert _faults(torch.zeros_like(g), v, rows, off)[1] > 1
            if v.dim() == 1 or shape[1] > 1:
                short = rows.clone()
                short[-1, -1] = 0
                columns, norm = _faults(_sum_like(short, v).to(v.dtype), v, rows, off)
                assert columns > 0 or norm > 1, (name, norm)

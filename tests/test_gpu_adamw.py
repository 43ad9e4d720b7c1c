"""adamw_step against the formula in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24


def _mix(h):
    m = 0xFFFFFFFF
    h = h ^ (h >> 16)
    h = (h * 0x85EBCA6B) & m
    h = h ^ (h >> 13)
    h = (h * 0xC2B2AE35) & m
    return h ^ (h >> 16)


def _codes(a, random, at_least):
    """Blocks of 256 in 64 bits: (values of the codes, scales).  `random`: 16 bits per place."""
    top = a.abs().amax(1)
    scale = torch.where(top >= 2.0 ** -100, top / 448, torch.zeros_like(top))
    q = torch.where(scale[:, None] > 0, a.abs() / scale[:, None].clamp(min=1e-300), torch.zeros_like(a)).clamp(max=448.0)
    step = torch.exp2((torch.frexp(q).exponent - 1).clamp(min=-6).double() - 3)
    code = torch.floor(q / step + (random.double() * 16 + 8) / 2 ** 20) * step
    code = code.clamp(max=448.0)
    if at_least:
        code = torch.where(q > 0, code.clamp(min=2.0 ** -9), code)
    return code * a.sign(), scale


def _spread(x, sizes):
    return torch.cat([torch.nn.functional.pad(p, (0, -n % 256)) for p, n in zip(x.split(sizes), sizes)]).view(-1, 256)


def _tensors(sizes, t, gt, shift=0, seed=0, device="cuda"):
    """Parameters and gradients as views of flat buffers that start `shift` elements after an aligned address."""
    g = torch.Generator(device=device).manual_seed(seed)
    total = sum(sizes)
    flat = (torch.randn(total + shift, generator=g, device=device) * 0.05).to(t)[shift:]
    grad = (torch.randn(total + shift, generator=g, device=device) * torch.exp(2 * torch.randn(total + shift, generator=g, device=device)) * 1e-3).to(gt)[shift:]
    return flat, grad, list(flat.split(sizes)), list(grad.split(sizes))


def _reference(p, g, m, v, t, lr, b1, b2, eps, decay, scale):
    g = g.double() * scale
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    p = p.double()
    return p - lr * decay * p - lr / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + eps), m, v


SIZES = [[1], [10], [256], [257, 3, 1, 4096, 4097, 0, 5], [4096 * 3 + 1, 12345, 64], [2] * 700, [100003, 1, 255, 256, 8191]]


@pytest.mark.parametrize("t,gt", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                  (torch.float16, torch.float16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{sum(s)}")
@pytest.mark.parametrize("shift", [0, 1, 2])
def test_steps(t, gt, bits, sizes, shift):
    from approxtrain_b200 import ops
    flat, grad, params, grads = _tensors(sizes, t, gt, shift)
    st = ops.AdamWState(params, bits=bits)
    lr, b1, b2, eps, decay, scale, seed = 1e-3, 0.9, 0.99, 1e-8, 0.1, 0.5, 77
    for step in (1, 2, 3):
        before = flat.clone()
        old = [st.moments(i) for i in range(len(sizes))]
        m0, v0 = (torch.cat([x[k].reshape(-1) for x in old]).double() for k in (0, 1))
        ops.adamw_step(params, grads, st, lr, betas=(b1, b2), eps=eps, weight_decay=decay, grad_scale=scale, seed=seed)
        assert int(st.step) == step and int(st._counter[1]) == 0
        p, m, v = _reference(before, grad, m0, v0, step, lr, b1, b2, eps, decay, scale)
        # the moments: three roundings of terms no larger than the sum of their sizes; the constants' own roundings as many
        size_m = (b1 * m0).abs() + ((1 - b1) * grad.double() * scale).abs()
        # the parameter: two roundings of p, and a dozen of an update whose own m and v carry those above
        up = lr / (1 - b1 ** step) * size_m / ((v / (1 - b2 ** step)).sqrt() + eps)
        tol = torch.finfo(t).eps / 2 * p.abs() + F32 * (3 * p.abs() + 16 * up) + torch.finfo(t).smallest_normal
        assert bool(((flat.double() - p).abs() <= tol).all()), float(((flat.double() - p).abs() - tol).max())
        if bits == 32:
            assert bool(((st.exp_avg.double() - m).abs() <= 6 * F32 * size_m + 1e-45).all())
            assert bool(((st.exp_avg_sq.double() - v).abs() <= 8 * F32 * v + 1e-45).all())
        else:
            place = torch.arange(st.exp_avg.numel(), device="cuda")
            key = _mix(torch.tensor(seed, device="cuda") ^ _mix(torch.tensor(step, device="cuda")))
            h = _mix(place ^ key).view(-1, 256)
            for code, sc, a, rest, least in ((st.exp_avg, st.exp_avg_scale, m, h & 0xFFFF, False), (st.exp_avg_sq_root, st.exp_avg_sq_scale, v.sqrt(), h >> 16, True)):
                want, scale64 = _codes(_spread(a, sizes), rest, least)
                assert bool(((sc.double() - scale64).abs() <= 16 * F32 * scale64).all())
                got = code.double().view(-1, 256)
                # the FP32 value may lie on the other side of the place where rounding turns: then the next code, for as many
                # of the values as its error is of a code's step (2^-20 at the least): a hundred in a million leaves room
                off = got != want
                assert float(off.double().mean()) <= 1e-4 or int(off.sum()) <= 1
                step_up = torch.exp2((torch.frexp(want.abs()).exponent - 1).clamp(min=-6).double() - 3)
                assert bool(((got - want).abs() <= step_up * 1.0001)[off].all())


def test_random_rounding_is_exact_on_average():
    """A second moment far below the next code still moves: the mean over seeds follows the exact moment."""
    from approxtrain_b200 import ops
    n = 256
    g = torch.linspace(0.1, 1.0, n, device="cuda")
    total = torch.zeros(2, n, dtype=torch.float64, device="cuda")
    seeds = 400
    for seed in range(seeds):
        p = torch.zeros(n, device="cuda")
        st = ops.AdamWState([p], bits=8)
        for _ in range(2):
            ops.adamw_step([p], [g], st, 1e-3, betas=(0.9, 0.999), seed=seed)
        total[0] += st.moments(0)[0].double()
        total[1] += st.moments(0)[1].sqrt().double()
    mean = total / seeds
    m, root = 0.19 * g.double(), (1 - 0.999 ** 2) ** 0.5 * g.double()
    # one rounding is off by at most a code's step, 1/8 of the value, with a variance of at most a quarter of its square; two steps
    # add two (the first's counted at most in full); 6 deviations of the mean over the seeds and 256 places; the square of the
    # first step's root adds its variance over twice the root: (1/16)^2 / 2
    tol = 6 * math.sqrt(2) / 16 / math.sqrt(seeds)
    assert bool(((mean[0] - m).abs() <= tol * m).all())
    assert bool(((mean[1] - root).abs() <= (tol + (1 / 16) ** 2) * root).all())


def test_rates_from_the_device_and_decay_per_tensor():
    from approxtrain_b200 import ops
    _, _, params, grads = _tensors([300, 7, 64], torch.float32, torch.float32)
    other = [p.clone() for p in params]
    a, b = ops.AdamWState(params), ops.AdamWState(other)
    ops.adamw_step(params, grads, a, 2e-3, weight_decay=[0.0, 0.1, 0.2], grad_scale=0.25)
    ops.adamw_step(other, grads, b, torch.full((1,), 2e-3, device="cuda"), weight_decay=[0.0, 0.1, 0.2], grad_scale=torch.full((1,), 0.25, device="cuda"))
    # lr = 2e-3 is rounded to FP32 in the tensor: each parameter's step by 2^-24 of itself
    for x, y in zip(params, other):
        assert float((x - y).abs().max()) <= 4 * F32 * (0.2 + 2e-3)


def test_zero_gradients_and_last_element_of_a_block():
    from approxtrain_b200 import ops
    for bits in (32, 8):
        p = torch.randn(513, device="cuda")
        st = ops.AdamWState([p], bits=bits)
        was = p.clone()
        ops.adamw_step([p], [torch.zeros_like(p)], st, 0.1, weight_decay=0.0)
        assert torch.equal(p, was) and not st.moments(0)[0].any() and not st.moments(0)[1].any()
        g = torch.zeros_like(p)
        g[512] = 1.0
        ops.adamw_step([p], [g], st, 0.1, weight_decay=0.0)
        assert torch.equal(p[:512], was[:512]) and abs(float(p[512] - was[512])) > 1e-3
        # tiny gradients: no infinite reciprocal, and the step is at most lr (|m| <= |g|, sqrt(v) = |g| at the first step)
        p = torch.zeros(300, device="cuda")
        st = ops.AdamWState([p], bits=bits)
        for _ in range(3):
            ops.adamw_step([p], [torch.full_like(p, 1e-36)], st, 0.1, weight_decay=0.0)
        assert bool(p.isfinite().all()) and float(p.abs().max()) < 0.35


def test_not_finite_gradients_stay_visible():
    from approxtrain_b200 import ops
    for bits in (32, 8):
        p = torch.zeros(1024, device="cuda")
        g = torch.ones(1024, device="cuda")
        g[300] = float("nan")
        st = ops.AdamWState([p], bits=bits)
        ops.adamw_step([p], [g], st, 0.1)
        assert bool(p[300].isnan()) and bool(p[:256].isfinite().all()) and bool(p[512:].isfinite().all())
        g[300] = float("inf")
        p.zero_()
        st = ops.AdamWState([p], bits=bits)
        ops.adamw_step([p], [g], st, 0.1)
        assert bool(p[300].isnan()) and bool(p[:256].isfinite().all())


def test_guards_and_neighbours_stay_as_they_are():
    """Nothing outside the parameters is written, whatever their alignment and length."""
    from approxtrain_b200 import ops
    for bits in (32, 8):
        for lead, n in ((1, 5), (3, 255), (4, 256), (2, 4097), (5, 9000)):
            buf = torch.full((lead + n + 9,), 7.0, device="cuda")
            p = buf[lead:lead + n]
            p.zero_()
            ops.adamw_step([p], [torch.ones(n, device="cuda")], ops.AdamWState([p], bits=bits), 0.1)
            assert bool((buf[:lead] == 7).all()) and bool((buf[lead + n:] == 7).all()) and bool((p < -0.09).all())


def test_captured_steps_count_on():
    from approxtrain_b200 import ops
    for bits in (32, 8):
        flat, grad, params, grads = _tensors([1000, 37], torch.float32, torch.float32)
        want, wp = flat.clone(), None
        wp = list(want.split([1000, 37]))
        a, b = ops.AdamWState(params, bits=bits), ops.AdamWState(wp, bits=bits)
        lr = torch.full((1,), 1e-2, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.adamw_step(params, grads, a, lr, seed=3)
        for i in range(4):
            lr.fill_(1e-2 / (i + 1))
            graph.replay()
            ops.adamw_step(wp, grads, b, lr, seed=3)
        assert int(a.step) == 4 and torch.equal(flat, want)
        for i in range(2):
            assert all(torch.equal(x, y) for x, y in zip(a.moments(i), b.moments(i)))


def test_saved_and_loaded():
    from approxtrain_b200 import ops
    for bits in (32, 8):
        _, _, params, grads = _tensors([70, 300], torch.float32, torch.float32)
        st = ops.AdamWState(params, bits=bits)
        ops.adamw_step(params, grads, st, 1e-2)
        saved, copy = st.state_dict(), [p.clone() for p in params]
        ops.adamw_step(params, grads, st, 1e-2)
        again = ops.AdamWState(copy, bits=bits)
        again.load_state_dict(saved)
        ops.adamw_step(copy, grads, again, 1e-2)
        assert all(torch.equal(x, y) for x, y in zip(params, copy)) and int(again.step) == 2
        with pytest.raises(ValueError):
            ops.AdamWState(params[:1], bits=bits).load_state_dict(saved)


def test_refusals():
    from approxtrain_b200 import ops
    p, g = [torch.zeros(8, device="cuda"), torch.zeros(3, device="cuda")], [torch.zeros(8, device="cuda"), torch.zeros(3, device="cuda")]
    st = ops.AdamWState(p)
    bad = [lambda: ops.adamw_step(p[:1], g, st, 0.1), lambda: ops.adamw_step(p, [g[1], g[0]], st, 0.1), lambda: ops.adamw_step(p, [g[0], g[1].half()], st, 0.1),
           lambda: ops.adamw_step([p[0].half(), p[1].half()], g, st, 0.1), lambda: ops.adamw_step(p, [g[0], g[1].cpu()], st, 0.1),
           lambda: ops.adamw_step(p, [torch.zeros(16, device="cuda")[::2], g[1]], st, 0.1), lambda: ops.adamw_step(p, g, st, 0.1, betas=(1.0, 0.9)),
           lambda: ops.adamw_step(p, g, st, 0.1, eps=-1.0), lambda: ops.adamw_step(p, g, st, 0.1, weight_decay=[0.1]),
           lambda: ops.adamw_step(p, g, st, torch.zeros(1)), lambda: ops.adamw_step(p, g, st, torch.zeros(2, device="cuda")), lambda: ops.adamw_step(p, g, None, 0.1),
           lambda: ops.AdamWState([]), lambda: ops.AdamWState(p, bits=16), lambda: ops.AdamWState([p[0], p[1].half()]), lambda: ops.AdamWState([torch.zeros(3)])]
    for f in bad:
        with pytest.raises((ValueError, TypeError)):
            f()
    assert int(st.step) == 0
    tied = torch.zeros(8, device="cuda")
    two = ops.AdamWState([tied, tied])
    with pytest.raises(ValueError, match="twice"):
        ops.adamw_step([tied, tied], [g[0], g[0]], two, 0.1)
    none = [torch.zeros(0, device="cuda"), torch.zeros(0, device="cuda"), tied]
    ops.adamw_step(none, [torch.zeros_like(t) for t in none], ops.AdamWState(none), 0.1)     # empty tensors share an address


def test_a_graph_that_saved_a_parameter_notices_the_step():
    from approxtrain_b200 import ops
    p = torch.ones(8, device="cuda", requires_grad=True)
    y = (p * p).sum()
    ops.adamw_step([p], [torch.ones(8, device="cuda")], ops.AdamWState([p]), 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_trainer():
    """LeNet-300-100 with AdamW, eager and replayed from a graph, against torch's own AdamW on the same gradients."""
    from conftest import lut_path
    from approxtrain_b200 import nets
    from approxtrain_b200.dp import DataParallelAdamW
    x, y = torch.rand(32, 784, device="cuda"), torch.randint(0, 10, (32,), device="cuda")
    torch.manual_seed(0)
    first = nets.LeNet300100(lut_path("MBM_7")).cuda()
    start = {k: v.clone() for k, v in first.state_dict().items()}
    for bits in (32, 8):
        losses = []
        for captured in (False, True):
            net = nets.LeNet300100(lut_path("MBM_7")).cuda()
            net.load_state_dict(start)
            tr = DataParallelAdamW(net, 1e-3, state_bits=bits)
            assert all(p.grad.data_ptr() % 16 == 0 for p in tr.params)
            loss_fn = lambda: torch.nn.functional.cross_entropy(net(x), y)
            if captured:
                replay = tr.capture(loss_fn, warmup=3)
                seen = [float(replay()) for _ in range(3)]
                assert int(tr.state.step) == 6
            else:
                seen = [float(tr.step(loss_fn)) for _ in range(6)][3:]
            losses.append(seen)
            if not captured and bits == 32:
                ref = nets.LeNet300100(lut_path("MBM_7")).cuda()
                ref.load_state_dict(start)
                opt = torch.optim.AdamW([dict(params=[p for p in ref.parameters() if p.dim() > 1], weight_decay=0.01),
                                         dict(params=[p for p in ref.parameters() if p.dim() == 1], weight_decay=0.0)], lr=1e-3)
                tr2 = DataParallelAdamW(ref, 1e-3)   # its gradients only
                tr2._update = opt.step
                for _ in range(1):
                    tr2.step(lambda: torch.nn.functional.cross_entropy(ref(x), y))
                one = nets.LeNet300100(lut_path("MBM_7")).cuda()
                one.load_state_dict(start)
                tr3 = DataParallelAdamW(one, 1e-3)
                tr3.step(lambda: torch.nn.functional.cross_entropy(one(x), y))
                for a, b in zip(one.parameters(), ref.parameters()):
                    # a first step is lr * g / (|g| + eps): at most lr, with a dozen roundings of it and one of p on either side
                    assert float((a - b).detach().abs().max()) <= 32 * F32 * (1e-3 + float(b.detach().abs().max()))
        assert losses[0] == losses[1]


def test_a_state_that_is_refused_changes_nothing():
    from approxtrain_b200 import ops
    from approxtrain_b200.dp import DataParallelAdamW
    for bits in (32, 8):
        net = torch.nn.Linear(30, 20).cuda()
        tr = DataParallelAdamW(net, 1e-3, state_bits=bits)
        x = torch.randn(4, 30, device="cuda")
        tr.step(lambda: net(x).square().sum())
        tr.step(lambda: net(x).square().sum())
        was = tr.state.state_dict()
        other = DataParallelAdamW(torch.nn.Linear(30, 20).cuda(), 5e-2, state_bits=bits).state_dict()
        for spoil in (lambda m: m.update(exp_avg=m["exp_avg"][1:]), lambda m: m.pop(tr.state._moments[-1]), lambda m: m.pop("step"),
                      lambda m: m.update({tr.state._moments[-1]: m[tr.state._moments[-1]].half()}), lambda m: m.update(bits=16), lambda m: m.update(shapes=[(1,)])):
            bad = dict(other, moments=dict(other["moments"]))
            spoil(bad["moments"])
            with pytest.raises((ValueError, KeyError)):
                tr.load_state_dict(bad)
            now = tr.state.state_dict()
            assert tr.lr == 1e-3 and float(tr._lr) == pytest.approx(1e-3) and int(tr.state.step) == 2
            assert all(torch.equal(now[k].float(), was[k].float()) for k in tr.state._moments)
        tr.load_state_dict(other)
        assert tr.lr == 5e-2 and int(tr.state.step) == 0 and not tr.state.moments(0)[0].any()


def test_the_rate_of_a_trainer_is_the_one_that_is_set():
    """``trainer.lr = x`` as with the other trainer, for eager and for captured steps."""
    from approxtrain_b200.dp import DataParallelAdamW
    x = torch.randn(16, 30, device="cuda")
    finals = []
    for captured in (False, True):
        torch.manual_seed(1)
        net = torch.nn.Linear(30, 20).cuda()
        tr = DataParallelAdamW(net, 1e-3, weight_decay=0.0)
        loss_fn = lambda: net(x).square().sum()
        step = tr.capture(loss_fn, warmup=3) if captured else lambda: tr.step(loss_fn)
        for _ in range(0 if captured else 3):
            step()
        tr.lr = 0.0
        before = net.weight.detach().clone()
        step()
        assert torch.equal(net.weight, before) and tr.lr == 0.0
        tr.lr = 0.25
        step()
        assert float((net.weight - before).detach().abs().max()) > 0.1 and tr.state_dict()["lr"] == 0.25
        tr.set_lr(0.5)
        assert tr.lr == 0.5
        step()
        finals.append(net.weight.detach().clone())
    assert torch.equal(*finals)

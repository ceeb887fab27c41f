"""FusedAdam(max_grad_norm=...): the norm of all gradients and the clipped update against both in 64 bits.

Tolerances (u = 2^-24).  norm: squares and sums are double, the root is rounded to float32: 2 u.  coefficient: the norm's
error, + 1e-6, a quotient: 6 u.  scaled and decayed gradient: 8 u of |coef g| + |wd p|; m: that times (1 - b1), plus 4 u of
its terms; v: twice the gradient's relative error (it is squared) plus 4 u, so with G the sum of the gradient's magnitudes
(1 - b2)(2 * 8 u + 4 u) G^2 + 4 u v.  sqrt and two quotients: the update's error is lr / bias1 times
dm / denom + m dv / (2 sqrt(v) denom^...) -- taken at its bound by moving m and v to the ends of their intervals."""
import copy
import math

import pytest
import torch

U = 2.0 ** -24


def reference(ps, gs, ms, vs, step, max_norm, lr, betas, eps, wd):
    """float64: (norm, [(p, m, v)], [(tol_p, tol_m, tol_v)])."""
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    coef = min(1.0, max_norm / (norm + 1e-6))
    b1, b2 = betas
    new, tol = [], []
    for p, g, m, v in zip(ps, gs, ms, vs):
        p, g, m, v = (t.double() for t in (p, g, m, v))
        grad, mag = coef * g + wd * p, (coef * g).abs() + (wd * p).abs()
        m1, v1 = m + (grad - m) * (1 - b1), b2 * v + (1 - b2) * grad * grad
        t_m = (1 - b1) * 9 * U * mag + 5 * U * (m.abs() + mag)
        t_v = (1 - b2) * 20 * U * mag * mag + 5 * U * v1 + 1e-44
        bias1, bias2 = 1 - b1 ** step, 1 - b2 ** step

        def update(mm, vv):
            return lr / bias1 * mm / ((vv / bias2).sqrt() + eps)

        far = torch.maximum(update(m1.abs() + t_m, (v1 - t_v).clamp_min(0.0)) - update(m1.abs(), v1), update(t_m, (v1 - t_v).clamp_min(0.0)))
        new.append((p - update(m1, v1), m1, v1))
        tol.append((far + 12 * U * update(m1.abs(), v1) + 2 * U * (p.abs() + update(m1.abs(), v1)), t_m, t_v))
    return norm, new, tol


def make(shapes, scale, seed, dev):
    gen = torch.Generator().manual_seed(seed)
    ps = [torch.randn(s, generator=gen) for s in shapes]
    gs = [torch.randn(s, generator=gen) * scale for s in shapes]
    return ps, gs


def close(got, want, tol):
    return float(((got.detach().double().cpu() - want).abs() - tol).max()) <= 0.0 if got.numel() else True


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-6, 1e-2, 30.0, 1e20])          # unclipped, and clipped by more and more
@pytest.mark.parametrize("wd,eps,capturable", [(0.0, 1e-8, False), (0.1, 1e-8, False), (0.0, 1e-15, True)])
def test_steps_against_64_bits(dev, scale, wd, eps, capturable):
    from nerf_amd.optim import FusedAdam
    shapes = [(256, 63), (256,), (1,), (4099, 2), (0, 5), (7, 13, 3), (65537,), (4096,), (3,)]
    ps, _ = make(shapes, scale, 1, dev)
    params = [torch.nn.Parameter(p.clone().to(dev)) for p in ps]
    opt = FusedAdam(params, lr=1e-3, eps=eps, weight_decay=wd, max_grad_norm=1.0, capturable=capturable)
    assert opt.grad_norm is None
    ms, vs = [torch.zeros_like(p) for p in ps], [torch.zeros_like(p) for p in ps]
    for step in range(1, 4):
        gs = make(shapes, scale, 10 + step, dev)[1]
        for p, g in zip(params, gs):
            p.grad = g.to(dev)
        norm, want, tol = reference([p.detach().cpu() for p in params], gs, ms, vs, step, 1.0, 1e-3, (0.9, 0.999), eps, wd)
        opt.step()
        assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm and opt.grad_norm.is_cuda and opt.grad_norm.dim() == 0
        for i, (p, w, t) in enumerate(zip(params, want, tol)):
            st = opt.state[p]
            assert float(st["step"]) == step and torch.equal(p.grad.cpu(), gs[i])          # gradients stay as they are
            for name, got, ww, tt in (("p", p, w[0], t[0]), ("m", st["exp_avg"], w[1], t[1]), ("v", st["exp_avg_sq"], w[2], t[2])):
                assert close(got, ww, tt), (step, i, name, shapes[i])
        ms, vs = [opt.state[p]["exp_avg"].cpu() for p in params], [opt.state[p]["exp_avg_sq"].cpu() for p in params]


@pytest.mark.gpu
def test_many_tensors_groups_and_missing_gradients(dev):
    """400 tensors (several launches of each kernel) in two groups with settings of their own: one norm over both."""
    from nerf_amd.optim import FusedAdam
    shapes = [(0,) if k % 50 == 3 else (1 + 37 * k,) for k in range(398)] + [(300000,), (1,)]
    ps, gs = make(shapes, 0.02, 2, dev)
    params = [torch.nn.Parameter(p.clone().to(dev)) for p in ps]
    opt = FusedAdam([{"params": params[:150], "lr": 1e-2}, {"params": params[150:], "lr": 1e-4, "betas": (0.8, 0.99), "weight_decay": 0.01}],
                    max_grad_norm=0.5)
    none = {5, 149, 200}
    for k, (p, g) in enumerate(zip(params, gs)):
        p.grad = None if k in none else g.to(dev)
    opt.step()
    have = [k for k in range(400) if k not in none]
    norm = math.sqrt(sum(float(gs[k].double().square().sum()) for k in have))
    assert norm > 0.5 and abs(float(opt.grad_norm) - norm) <= 2 * U * norm
    for part, lr, betas, wd in ((range(150), 1e-2, (0.9, 0.999), 0.0), (range(150, 400), 1e-4, (0.8, 0.99), 0.01)):
        keep = [k for k in part if k not in none]
        coef = 0.5 / (norm + 1e-6)
        zeros = [torch.zeros_like(ps[k]) for k in keep]
        # the group's own list has another norm: hand the reference gradients that are scaled already
        _, want, tol = reference([ps[k] for k in keep], [gs[k].double() * coef for k in keep], zeros, zeros, 1, math.inf, lr, betas, 1e-8, wd)
        for k, w, t in zip(keep, want, tol):
            assert close(params[k], w[0], t[0]) and close(opt.state[params[k]]["exp_avg_sq"], w[2], t[2]), k
    for k in none:
        assert torch.equal(params[k].detach().cpu(), ps[k]) and not opt.state[params[k]]
    for p in params:
        p.grad = None
    opt.step()
    assert float(opt.grad_norm) == 0.0


@pytest.mark.gpu
def test_same_as_clipping_first(dev):
    """Against the two calls it stands for, clip_grad_norm_ and then torch's Adam."""
    from nerf_amd.optim import FusedAdam
    shapes = [(64, 32), (64,), (524288, 2), (3, 64)]
    ps, gs = make(shapes, 0.01, 3, dev)
    a = [torch.nn.Parameter(p.clone().to(dev)) for p in ps]
    b = [torch.nn.Parameter(p.clone().to(dev)) for p in ps]
    mine, ref = FusedAdam(a, lr=1e-2, eps=1e-15, max_grad_norm=1.0), torch.optim.Adam(b, lr=1e-2, eps=1e-15)
    for step in range(3):
        for p, q, g in zip(a, b, gs):
            p.grad, q.grad = (g * (step + 1)).to(dev), (g * (step + 1)).to(dev)
        norm = torch.nn.utils.clip_grad_norm_(b, 1.0)
        ref.step()
        mine.step()
        assert abs(float(norm) - float(mine.grad_norm)) <= 2e-6 * float(norm)
        for p, q in zip(a, b):
            assert torch.allclose(p, q, rtol=2e-6, atol=1e-7 * (step + 1))      # the bound the unclipped step is held to
    ref.load_state_dict(mine.state_dict())
    again = FusedAdam([torch.nn.Parameter(p.detach().clone()) for p in a], lr=1e-2, eps=1e-15, max_grad_norm=1.0)
    again.load_state_dict(copy.deepcopy(mine.state_dict()))      # a state dict holds the optimiser's own moments, as torch's does
    for p, q, g in zip(a, again.param_groups[0]["params"], gs):
        p.grad, q.grad = g.to(dev), g.to(dev).t().contiguous().t() if g.dim() == 2 else g.to(dev)   # a gradient of other strides
    mine.step()
    again.step()
    assert all(torch.equal(p, q) for p, q in zip(a, again.param_groups[0]["params"]))


@pytest.mark.gpu
def test_step_counts_stay_apart(dev):
    """A parameter that misses a step, clipping switched off and on again, states loaded piecemeal: every parameter is
    stepped with its own count, as torch's Adam does it."""
    from nerf_amd.optim import FusedAdam
    shapes = [(40, 3), (17,), (4097,)]
    ps, _ = make(shapes, 1.0, 5, dev)
    a = [torch.nn.Parameter(p.clone().to(dev)) for p in ps]
    b = [torch.nn.Parameter(p.clone().to(dev)) for p in ps]
    mine, ref = FusedAdam(a, lr=1e-2, max_grad_norm=1e9), torch.optim.Adam(b, lr=1e-2)
    for step in range(7):
        gs = make(shapes, 1.0, 50 + step, dev)[1]
        for k, (p, q, g) in enumerate(zip(a, b, gs)):
            p.grad, q.grad = (None, None) if (step, k) in ((1, 0), (2, 2), (4, 1)) else (g.to(dev), g.to(dev))
        mine.max_grad_norm = None if step in (3, 4) else 1e9
        mine.step()
        ref.step()
        for k, (p, q) in enumerate(zip(a, b)):
            assert float(mine.state[p]["step"]) == float(ref.state[q]["step"]), (step, k)
            assert torch.allclose(p, q, rtol=2e-6, atol=1e-7 * (step + 1)), (step, k)


@pytest.mark.gpu
def test_infinite_and_nan_gradients(dev):
    from nerf_amd.optim import FusedAdam
    for bad in (float("inf"), float("nan")):
        a = [torch.nn.Parameter(torch.ones(5000, device=dev)), torch.nn.Parameter(torch.ones(7, device=dev))]
        b = [torch.nn.Parameter(p.detach().clone()) for p in a]
        mine, ref = FusedAdam(a, lr=0.1, max_grad_norm=1.0), torch.optim.Adam(b, lr=0.1)
        for ps in (a, b):
            for p in ps:
                p.grad = torch.full_like(p, 0.5)
            ps[0].grad[4999] = bad
        norm = torch.nn.utils.clip_grad_norm_(b, 1.0)
        ref.step()
        mine.step()
        assert torch.equal(norm.isnan(), mine.grad_norm.isnan()) and torch.equal(norm.isinf(), mine.grad_norm.isinf())
        for p, q in zip(a, b):
            assert torch.equal(p.isnan(), q.isnan()) and torch.allclose(p, q, rtol=2e-6, atol=1e-7, equal_nan=True)


@pytest.mark.gpu
def test_captured_step(dev):
    """Replayed from a HIP graph under a changing learning rate, step for step what an eager optimiser does."""
    from nerf_amd.graph import GraphedStep
    from nerf_amd.optim import FusedAdam
    gen = torch.Generator().manual_seed(4)
    first = [torch.randn(s, generator=gen) for s in ((70, 30), (5000,), (1,))]
    a, b = ([torch.nn.Parameter(p.clone().to(dev)) for p in first] for _ in range(2))
    x = torch.zeros((), device=dev)
    grads = [torch.randn(p.shape, generator=gen).to(dev) for p in first]
    opt_a, opt_b = (FusedAdam(ps, lr=1e-2, max_grad_norm=2.0, capturable=True) for ps in (a, b))
    for p, g in zip(a, grads):
        p.grad = g.clone()

    def step():
        for p, g in zip(a, grads):
            p.grad.copy_(g * x)
        opt_a.step()
        return opt_a.grad_norm

    def eager(k):
        for p, g in zip(b, grads):
            p.grad = g * float(k)
        opt_b.step()

    captured = GraphedStep(step, warmup=2, optimizers=[opt_a], prepare=lambda i: x.fill_(0.01 + i))
    for i in range(2):
        eager(torch.tensor(0.01 + i))
    for k in range(4):
        x.fill_(0.003 * (k + 1) ** 3)
        opt_a.param_groups[0]["lr"] = opt_b.param_groups[0]["lr"] = 1e-2 / (k + 1)
        norm = captured()
        torch.cuda.synchronize()
        eager(torch.tensor(0.003 * (k + 1) ** 3))
        assert torch.equal(norm, opt_b.grad_norm), k
        assert all(torch.equal(p, q) for p, q in zip(a, b)), k


@pytest.mark.gpu
def test_another_stream(dev):
    from nerf_amd.optim import FusedAdam
    got = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            torch.manual_seed(0)
            ps = [torch.nn.Parameter(torch.linspace(-1, 1, n, device=dev)) for n in (100000, 3)]
            opt = FusedAdam(ps, max_grad_norm=0.1)
            for _ in range(3):
                for p in ps:
                    p.grad = p.detach() * 3 + 1
                opt.step()
        stream.synchronize()
        got.append([p.detach().clone() for p in ps] + [opt.grad_norm.clone()])
    assert all(torch.equal(x, y) for x, y in zip(*got))


def test_copies_and_pickles_keep_the_clipping():
    """Without a step: no GPU needed."""
    import pickle
    from nerf_amd.optim import FusedAdam
    for limit in (None, 0.5):
        opt = FusedAdam([torch.nn.Parameter(torch.ones(3))], max_grad_norm=limit)
        for twin in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
            assert twin.max_grad_norm == limit and twin.grad_norm is None
            twin.load_state_dict(opt.state_dict())
            assert twin.max_grad_norm == limit


@pytest.mark.gpu
@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("limit", [None, 0.5])
def test_a_copy_goes_on_like_the_original(dev, limit, capturable):
    from nerf_amd.optim import FusedAdam
    params = [torch.nn.Parameter(torch.arange(1.0, n + 1, device=dev)) for n in (5, 300)]
    opt = FusedAdam(params, lr=1e-2, max_grad_norm=limit, capturable=capturable)
    model = {"opt": opt, "params": params}
    for step in range(4):
        if step == 2:
            twin = copy.deepcopy(model)
        for m in (model, twin) if step >= 2 else (model,):
            for p in m["params"]:
                p.grad = torch.full_like(p, 0.1 * step + 0.1)
            m["opt"].step()
    for a, b in zip(params, twin["params"]):
        assert a is not b and torch.equal(a, b)
        assert float(opt.state[a]["step"]) == 4 == float(twin["opt"].state[b]["step"])


def test_refusals():
    from nerf_amd._lib import NerfHipError
    from nerf_amd.optim import FusedAdam
    p = torch.nn.Parameter(torch.zeros(4))
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            FusedAdam([p], max_grad_norm=bad)
    opt = FusedAdam([p], max_grad_norm=1.0)
    opt.step()                                 # no gradients: nothing to do
    p.grad = torch.zeros(4)
    with pytest.raises(NerfHipError, match="GPU only"):
        opt.step()
    half = torch.nn.Parameter(torch.zeros(4, dtype=torch.float16))
    half.grad = torch.zeros(4, dtype=torch.float16)
    with pytest.raises(NerfHipError, match="float32"):
        FusedAdam([half], max_grad_norm=1.0).step()
    p.grad = None
    sparse = torch.nn.Parameter(torch.zeros(4, 2))
    sparse.grad = torch.sparse_coo_tensor([[1]], [[1.0, 2.0]], (4, 2))
    with pytest.raises(NerfHipError, match="sparse"):
        FusedAdam([sparse], max_grad_norm=1.0).step()


def test_entry_points_refuse():
    """Checked before anything is launched: no GPU needed."""
    import ctypes as C

    from nerf_amd import _lib as L
    lib = L.lib()
    ptrs, null, n = (C.c_void_p * 2)(4096, 8192), (C.c_void_p * 2)(4096, None), (C.c_int64 * 2)(5, 6)
    assert lib.nerf_grad_norm_workspace_doubles(2, n) == 2 and lib.nerf_grad_norm_workspace_doubles(0, None) == 0
    assert lib.nerf_grad_norm_workspace_doubles(1, (C.c_int64 * 1)(1 << 40)) == 2048
    for args in ((2, ptrs, n, 1.0, None, 4096), (2, ptrs, n, 1.0, 4096, None), (2, ptrs, n, -1.0, 4096, 4096), (2, ptrs, n, float("nan"), 4096, 4096),
                 (2, None, n, 1.0, 4096, 4096), (2, null, n, 1.0, 4096, 4096), (-1, ptrs, n, 1.0, 4096, 4096), (2, ptrs, (C.c_int64 * 2)(5, -6), 1.0, 4096, 4096)):
        assert lib.nerf_grad_norm(*args, None) == -22 and lib.nerf_last_error(), args
    step = lambda count=2, p=ptrs, step=1, b1=0.9, b2=0.999, scale=4096: lib.nerf_adam_step_scaled(  # noqa: E731
        count, p, ptrs, ptrs, ptrs, n, step, None, 0.1, b1, b2, 1e-8, 0.0, scale, None)
    for k in ({"count": -1}, {"p": None}, {"p": null}, {"step": 0}, {"b1": 1.0}, {"b2": -0.1}, {"scale": None}):
        assert step(**k) == -22 and lib.nerf_last_error(), k


@pytest.mark.gpu
@pytest.mark.parametrize("limit", [None, 1e9])
def test_every_parameter_keeps_its_own_step_tensor(dev, limit):
    """As with torch's Adam: a step count taken from the state goes on counting, and setting one leaves the others alone."""
    from nerf_amd.optim import FusedAdam
    ps, _ = make([(40, 3), (17,), (4097,)], 1.0, 5, dev)
    a = [torch.nn.Parameter(p.clone().to(dev)) for p in ps]
    b = [torch.nn.Parameter(p.clone().to(dev)) for p in ps]
    mine, ref = FusedAdam(a, lr=1e-2, max_grad_norm=limit), torch.optim.Adam(b, lr=1e-2)
    for step in range(6):
        gs = make([p.shape for p in ps], 1.0, 70 + step, dev)[1]
        for p, q, g in zip(a, b, gs):
            p.grad, q.grad = g.to(dev), g.to(dev)
        mine.step()
        ref.step()
        if step == 1:
            held = [mine.state[p]["step"] for p in a]
            assert len({t.data_ptr() for t in held}) == 3
        elif step == 2:
            held[1].zero_()
            ref.state[b[1]]["step"].zero_()
        for k, (p, q) in enumerate(zip(a, b)):
            assert float(mine.state[p]["step"]) == float(ref.state[q]["step"]), (step, k)
            assert step < 1 or mine.state[p]["step"] is held[k], (step, k)
            assert torch.allclose(p, q, rtol=2e-6, atol=1e-7 * (step + 1)), (step, k)      # the bound the unclipped step is held to


def test_shared_step_tensors_are_told_apart_on_loading():
    """A state whose parameters hold one step tensor between them (no GPU needed)."""
    import pickle
    from nerf_amd.optim import FusedAdam
    params = [torch.nn.Parameter(torch.ones(3)) for _ in range(3)]
    opt = FusedAdam(params, max_grad_norm=1.0)
    one = torch.tensor(4.0)
    for p in params:
        opt.state[p] = {"step": one, "exp_avg": torch.zeros(3), "exp_avg_sq": torch.zeros(3)}
    fresh = FusedAdam([torch.nn.Parameter(torch.ones(3)) for _ in range(3)], max_grad_norm=1.0)
    shared = torch.optim.Optimizer.state_dict(opt)
    assert len({st["step"].data_ptr() for st in shared["state"].values()}) == 1
    fresh.load_state_dict(shared)
    for twin in (fresh, copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        steps = [st["step"] for st in twin.state.values()]
        assert len(steps) == 3 and all(float(t) == 4.0 for t in steps) and len({t.data_ptr() for t in steps}) == 3


@pytest.mark.gpu
@pytest.mark.parametrize("limit", [None, 1e9])
@pytest.mark.parametrize("copied", [False, True])
def test_a_group_that_is_capturable_for_a_while(dev, limit, copied):
    """The parameters of a capturable group share their step count in device memory; before and after they count for themselves."""
    from nerf_amd.optim import FusedAdam
    ps, _ = make([(40, 3), (17,), (4097,)], 1.0, 6, dev)
    a = [torch.nn.Parameter(p.clone().to(dev)) for p in ps]
    b = [torch.nn.Parameter(p.clone().to(dev)) for p in ps]
    mine, ref = FusedAdam(a, lr=1e-2, max_grad_norm=limit), torch.optim.Adam(b, lr=1e-2)
    for step in range(8):
        gs = make([p.shape for p in ps], 1.0, 90 + step, dev)[1]
        if step == 4 and copied:
            a, mine = copy.deepcopy((a, mine))
        mine.param_groups[0]["capturable"] = step in (2, 3, 7)
        for k, (p, q, g) in enumerate(zip(a, b, gs)):
            p.grad, q.grad = (None, None) if (step, k) == (5, 1) else (g.to(dev), g.to(dev))
        if step == 7:                          # one count for the group again
            mine.state[a[1]]["step"] += 1
            ref.state[b[1]]["step"] += 1
        mine.step()
        ref.step()
        for k, (p, q) in enumerate(zip(a, b)):
            assert float(mine.state[p]["step"]) == float(ref.state[q]["step"]), (step, k)
            assert torch.allclose(p, q, rtol=2e-6, atol=1e-7 * (step + 1)), (step, k)

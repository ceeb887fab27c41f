"""ops.linear_scan against the recurrence in 64 bits, step by step.

Tolerances.  u = 2^-24.  Every value of h is a sum of x_s times gates; each of these terms meets at most two roundings a
step (one in the composed products, one in the replayed recurrence) and a handful when slices, waves, tiles and segments
are joined, so |error| <= (2 T + 64) u Hbar with Hbar the same recurrence over |gate|, |w x|, |state|.  The gradient that
arrives at a step obeys the same bound with Gbar; d_gate is a product of the two, summed over P channels:
(4 T + P + 128) u sum Gbar (Hbar + |x|).  1 - gate adds one rounding to the weight, which the constants hold.  An output
of a type of 16 bits is rounded once more: half a step, eps / 2 relative, or half the smallest step where it is subnormal.
"""
import pytest
import torch

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def ref_scan(a, x, state, reverse, blend, d_h=None, d_last=None):
    """float64 on the CPU: (h, last), and with d_h the gradients (d_gate [B,T,G], d_x, d_state) too."""
    B, T, C = x.shape
    G = a.shape[2]
    a = a.double().repeat_interleave(C // G, 2)
    x = x.double()
    wt = 1.0 - a if blend else torch.ones_like(a)
    order = list(range(T - 1, -1, -1)) if reverse else list(range(T))
    h = state.double().clone() if state is not None else torch.zeros(B, C, dtype=torch.float64)
    H, P = torch.empty_like(x), torch.empty_like(x)
    for t in order:
        P[:, t] = h
        h = a[:, t] * h + wt[:, t] * x[:, t]
        H[:, t] = h
    if d_h is None:
        return H, h
    r = d_last.double().clone() if d_last is not None else torch.zeros(B, C, dtype=torch.float64)
    d_a, d_x = torch.empty_like(x), torch.empty_like(x)
    for t in reversed(order):
        g = d_h[:, t].double() + r
        d_a[:, t] = g * (P[:, t] - x[:, t] if blend else P[:, t])
        d_x[:, t] = wt[:, t] * g
        r = a[:, t] * g
    return H, h, d_a.view(B, T, G, C // G).sum(3), d_x, r


def bounds(a, x, state, reverse, blend, d_h, d_last):
    """The tolerances of h, last, d_gate, d_x, d_state before the outputs' own rounding."""
    B, T, C = x.shape
    G = a.shape[2]
    aa, w = a.double().abs(), (1.0 - a.double()).abs() if blend else torch.ones_like(a.double())
    xw = x.double().abs() * w.repeat_interleave(C // G, 2)
    s = state.double().abs() if state is not None else None
    H, last, _, G_, r = ref_scan(aa, xw, s, reverse, False, d_h.double().abs(), d_last.double().abs() if d_last is not None else None)
    order = range(T - 1, -1, -1) if reverse else range(T)
    prev = torch.empty_like(H)
    before = s if s is not None else torch.zeros(B, C, dtype=torch.float64)
    for t in order:
        prev[:, t] = before
        before = H[:, t]
    d_a = (G_ * (prev + (x.double().abs() if blend else 0.0))).view(B, T, G, C // G).sum(3)
    k = (2 * T + 64) * U
    return k * H, k * last, (4 * T + C // G + 128) * U * d_a, k * G_ * w.repeat_interleave(C // G, 2), k * r


def assert_close(got, want, tol, what):
    half = 0.0 if got.dtype == F32 else torch.finfo(got.dtype).eps / 2
    tiny = 0.0 if got.dtype == F32 else torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    err = (got.detach().double().cpu() - want).abs()
    allow = tol + half * (want.abs() + tol) + tiny + 1e-37
    worst = (err - allow).max() if err.numel() else torch.tensor(-1.0)
    assert bool(torch.isfinite(got.float()).all()) and float(worst) <= 0.0, (what, float(worst), float(err.max()))


def make(B, T, C, G, tx, tg, state, seed, resets=0.05):
    gen = torch.Generator().manual_seed(seed)
    gate = torch.rand(B, T, G, generator=gen) * 1.5 - 0.5     # in [-0.5, 1)
    gate[torch.rand(B, T, G, generator=gen) < 0.5] = 0.99
    gate[torch.rand(B, T, 1, generator=gen).expand(B, T, G) < resets] = 0.0
    x = torch.randn(B, T, C, generator=gen)
    s = torch.randn(B, C, generator=gen) if state else None
    return gate.to(tg), x.to(tx), s, torch.randn(B, T, C, generator=gen).to(tx), torch.randn(B, C, generator=gen)


def check(dev, B, T, C, G, tx=F32, tg=None, reverse=False, blend=False, state=False, seed=0):
    from nerf_amd import ops
    tg = tg or tx
    gate, x, s, d_h, d_last = make(B, T, C, G, tx, tg, state, seed)
    leaves = [t.to(dev).requires_grad_(True) if t is not None else None for t in (gate, x, s)]
    h, last = ops.linear_scan(*leaves, reverse=reverse, blend=blend, return_state=True)
    assert h.dtype == tx and h.shape == x.shape and last.dtype == F32 and last.shape == (B, C)
    grads = torch.autograd.grad([h, last], [t for t in leaves if t is not None], [d_h.to(dev), d_last.to(dev)])
    want = ref_scan(gate, x, s, reverse, blend, d_h, d_last)
    tol = bounds(gate, x, s, reverse, blend, d_h, d_last)
    got = [h, last, grads[0], grads[1]] + ([grads[2]] if state else [])
    for name, g, w, t in zip(("h", "last", "d_gate", "d_x", "d_state"), got, want, tol):
        assert_close(g, w, t, (name, (B, T, C, G), tx, tg, reverse, blend, state))
    with torch.no_grad():                      # the inference form: the same bits
        h2 = ops.linear_scan(*leaves, reverse=reverse, blend=blend)
    assert torch.equal(h2, h)                  # (a chain's states do not depend on which tile waits for which)
    again = torch.autograd.grad(list(ops.linear_scan(*leaves, reverse=reverse, blend=blend, return_state=True)),
                                [t for t in leaves if t is not None], [d_h.to(dev), d_last.to(dev)])
    assert all(torch.equal(a, b) for a, b in zip(grads, again))   # sums in a fixed order


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 7, 8, 9, 63, 64, 65, 129, 1021, 3001])
@pytest.mark.parametrize("C,G", [(1, 1), (3, 1), (4, 4), (5, 5), (64, 1), (65, 65), (100, 10)])
def test_lengths_and_layouts(dev, T, C, G):
    check(dev, 2, T, C, G, state=True, reverse=T % 2 == 0, blend=T % 3 == 0, seed=T + C)


@pytest.mark.gpu
@pytest.mark.parametrize("tx,tg", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("blend", [False, True])
@pytest.mark.parametrize("B,T,C,G", [(3, 70, 132, 132), (2, 200, 96, 3), (4, 33, 7, 7), (1, 517, 30, 6), (5, 300, 3, 1), (2, 70, 6, 2), (3, 129, 4, 2), (9, 2500, 3, 1)])
def test_types(dev, tx, tg, reverse, blend, B, T, C, G):
    check(dev, B, T, C, G, tx, tg, reverse, blend, state=B % 2 == 0, seed=B)


@pytest.mark.gpu
@pytest.mark.parametrize("tx,tg", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("B,C,G", [(1, 1, 1), (3, 1, 1), (2, 7, 7), (5, 64, 64), (3, 65, 5), (2, 66, 3), (7, 129, 1), (300, 1023, 1023), (1000, 12, 4), (1, 2050, 2050)])
@pytest.mark.parametrize("blend,state", [(False, False), (True, True), (True, False)])
def test_one_step(dev, tx, tg, B, C, G, blend, state):
    check(dev, B, 1, C, G, tx, tg, reverse=C % 2 == 0, blend=blend, state=state, seed=C)


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,C,G", [(4099, 5, 3, 1), (700, 64, 1, 1), (300, 192, 3, 1), (9, 192, 3, 3), (130, 1, 260, 260), (1, 20000, 4, 4),
                                     (1, 9000, 68, 1), (2, 1500, 520, 2), (1, 4097, 300, 1), (17, 100, 600, 600), (2, 40, 1030, 1),
                                     # tiles in a chain: two, some, several groups of them; every way to lay out the lanes
                                     (3, 70, 132, 132), (3, 600, 132, 132), (9, 1021, 100, 100), (2, 3000, 520, 520), (8, 2500, 64, 1), (8, 2500, 5, 1), (600, 5000, 1, 1), (8, 40000, 4, 4),
                                     (4, 1021, 65, 65), (4, 700, 130, 2), (8, 9000, 12, 4), (3, 30000, 3, 1), (70, 9000, 6, 3)])
def test_sizes(dev, B, T, C, G):
    check(dev, B, T, C, G, reverse=True, blend=True, state=True, seed=5)


@pytest.mark.gpu
def test_is_the_compositing_loop(dev):
    """Back to front over the samples, the recurrence gives the colour, and its gradient, that ops.composite gives."""
    from nerf_amd import ops
    gen = torch.Generator().manual_seed(3)
    R, N = 37, 65
    rgb, sigma = torch.rand(R, N, 3, generator=gen).to(dev).requires_grad_(True), torch.rand(R, N, generator=gen).to(dev).requires_grad_(True)
    z = torch.sort(torch.rand(R, N, generator=gen) * 4 + 2)[0].to(dev)
    target = torch.randn(R, 3, generator=gen).to(dev)
    out, _, _ = ops.composite(rgb, sigma, z)
    want = torch.autograd.grad(out, [rgb, sigma], target)
    delta = torch.cat([z[:, 1:] - z[:, :-1], torch.full((R, 1), ops.TAIL_CAMERA, device=dev)], 1)
    h = ops.linear_scan(torch.exp(-sigma * delta)[..., None], rgb, reverse=True, blend=True)
    got = torch.autograd.grad(h[:, 0], [rgb, sigma], target)
    # a sum of N terms of at most 1 either way (N u each), exp and the distances a few roundings more; d_sigma is scaled by delta <= 4
    # (the tail's gate is 0 to all digits)
    assert float((h[:, 0] - out).detach().abs().max()) <= 4 * N * U * 3
    assert float((got[0] - want[0]).abs().max()) <= 4 * N * U * 4 * 4
    assert float((got[1] - want[1]).abs().max()) <= 4 * N * U * 4 * 4 * 4


@pytest.mark.gpu
def test_in_parts_and_step_by_step(dev):
    """A sequence in parts, the state handed on in float32, down to one step at a time."""
    from nerf_amd import ops
    gate, x, s, _, _ = make(3, 50, 20, 20, BF16, F32, True, 8)
    want_h, want_last = ref_scan(gate, x, s, False, False)
    tol_h, tol_last = bounds(gate, x, s, False, False, x, s)[:2]
    for size in (1, 13):
        state, parts = s.to(dev), []
        for t in range(0, 50, size):
            h, state = ops.linear_scan(gate[:, t:t + size].to(dev), x[:, t:t + size].to(dev), state, return_state=True)
            parts.append(h)
        assert_close(torch.cat(parts, 1), want_h, tol_h, size)
        assert_close(state, want_last, tol_last, size)


@pytest.mark.gpu
def test_gradient_by_differences(dev):
    """h is linear in x and state and, over two steps, of degree two in the gates: the central difference of <h, w> along a
    direction has no truncation error, only the bound of h at both ends over twice the step."""
    from nerf_amd import ops
    gen = torch.Generator().manual_seed(4)
    B, T, C = 2, 2, 6
    gate, x, s, w = (torch.randn(sh, generator=gen) for sh in ((B, T, C), (B, T, C), (B, C), (B, T, C)))
    leaves = [t.to(dev).requires_grad_(True) for t in (gate, x, s)]
    grads = torch.autograd.grad(ops.linear_scan(*leaves), leaves, w.to(dev))
    own = bounds(gate, x, s, False, False, w, None)[2:]
    step = 2.0 ** -4
    for k in range(3):
        d = torch.randn(leaves[k].shape, generator=gen)

        def value(sign):
            moved = [t.detach() for t in leaves]
            moved[k] = moved[k] + sign * step * d.to(dev)
            return float((ops.linear_scan(*moved).double().cpu() * w.double()).sum())

        slope = (value(1.0) - value(-1.0)) / (2 * step)
        want = float((grads[k].double().cpu() * d.double()).sum())
        far = [t.abs() + (step * d.abs() if i == k else 0.0) for i, t in enumerate((gate, x, s))]
        # the moved input is itself rounded: one more u, held in the constant of the bound
        at_ends = float((w.double().abs() * bounds(*far, False, False, w, None)[0]).sum()) / step
        assert abs(slope - want) <= at_ends + float((own[k] * d.double().abs()).sum()), (k, slope, want)


@pytest.mark.gpu
def test_strides_alignment_and_leading_axes(dev):
    from nerf_amd import ops
    gen = torch.Generator().manual_seed(6)
    big = torch.randn(2, 3, 40, 12, generator=gen).to(dev)
    gate = torch.rand(2, 3, 40, 1, generator=gen).to(dev)
    want = ops.linear_scan(gate.reshape(6, 40, 1), big.reshape(6, 40, 12)).view(2, 3, 40, 12)
    assert torch.equal(ops.linear_scan(gate, big), want)
    assert torch.equal(ops.linear_scan(gate[0, 0], big[0, 0]), want[0, 0])
    turned = big.transpose(2, 3).contiguous().transpose(2, 3)
    assert not turned.is_contiguous() and torch.equal(ops.linear_scan(gate, turned), want)
    flat = torch.empty(big.numel() + 1, device=dev)
    flat[1:] = big.reshape(-1)
    off = flat[1:].view(2, 3, 40, 12)      # 4 bytes past a 16-byte boundary
    assert off.data_ptr() % 16 == 4 and torch.equal(ops.linear_scan(gate, off), want)
    # an expanded gate: its gradient is the sum over what it was expanded to
    g1 = gate[:1, :1].clone().requires_grad_(True)
    h = ops.linear_scan(g1.expand(2, 3, 40, 1), big)
    d = torch.randn(h.shape, generator=gen).to(dev)
    (got,) = torch.autograd.grad(h, g1, d)
    _, _, per, _, _ = ref_scan(g1.detach().cpu().expand(2, 3, 40, 1).reshape(6, 40, 1), big.cpu().reshape(6, 40, 12), None, False, False, d.cpu().reshape(6, 40, 12))
    tol = bounds(g1.detach().cpu().expand(2, 3, 40, 1).reshape(6, 40, 1), big.cpu().reshape(6, 40, 12), None, False, False, d.cpu().reshape(6, 40, 12), None)[2]
    assert_close(got[0, 0], per.sum(0), tol.sum(0) + 8 * U * per.abs().sum(0), "expanded")
    # one gradient that is itself expanded (what .sum() sends back)
    x = big.clone().requires_grad_(True)
    (gx,) = torch.autograd.grad(ops.linear_scan(gate, x).sum(), x)
    ones = torch.ones(6, 40, 12)
    assert_close(gx.view(6, 40, 12), ref_scan(gate.cpu().reshape(6, 40, 1), big.cpu().reshape(6, 40, 12), None, False, False, ones)[3],
                 bounds(gate.cpu().reshape(6, 40, 1), big.cpu().reshape(6, 40, 12), None, False, False, ones, None)[3], "ones")


@pytest.mark.gpu
def test_empty_and_partial_gradients(dev):
    from nerf_amd import ops
    for B, T, C in ((0, 5, 4), (3, 0, 4), (3, 5, 0)):
        x = torch.zeros(B, T, C, device=dev, requires_grad=True)
        gate = torch.zeros(B, T, C if C else 1, device=dev, requires_grad=True)
        state = torch.ones(B, C, device=dev, requires_grad=True)
        h, last = ops.linear_scan(gate, x, state, return_state=True)
        assert h.shape == (B, T, C) and last.shape == (B, C) and (T > 0 or bool((last == 1).all()))
        (h.sum() + last.sum()).backward()
        assert x.grad.shape == x.shape and (T > 0 or bool((state.grad == 1).all()))
        with torch.no_grad():
            ops.linear_scan(gate, x, None, return_state=True)
        del h, last
        for lead in ((), (2, 0), (1, 2)):     # memory that held something, a gate with elements where there are no channels
            torch.full((4096,), 7.0, device=dev)
            leaves = [torch.ones(*lead, T, n, device=dev, requires_grad=True) for n in (C or 3, C)]
            y, end = ops.linear_scan(*leaves, return_state=True)
            assert y.shape == (*lead, T, C) and end.shape == (*lead, C) and (T > 0 or not bool(end.any()))
            if y.numel() == 0:
                grads = torch.autograd.grad([y, end], leaves, [torch.ones_like(y), torch.ones_like(end)])
                assert all(g.shape == t.shape and not bool(g.any()) for g, t in zip(grads, leaves))
    # only some of the inputs want gradients, only some of the outputs send any
    gate, x, s, d_h, d_last = make(2, 20, 8, 2, F32, F32, True, 9)
    want = ref_scan(gate, x, s, False, False, d_h, None)
    tol = bounds(gate, x, s, False, False, d_h, None)
    for k in range(3):
        leaves = [t.to(dev).requires_grad_(i == k) for i, t in enumerate((gate, x, s))]
        h, last = ops.linear_scan(*leaves, return_state=True)
        (g,) = torch.autograd.grad(h, [leaves[k]], d_h.to(dev))
        assert_close(g, want[2 + k], tol[2 + k], k)
    zero = torch.zeros_like(d_h)
    want = ref_scan(gate, x, s, False, False, zero, d_last)
    tol = bounds(gate, x, s, False, False, zero, d_last)
    leaves = [t.to(dev).requires_grad_(True) for t in (gate, x, s)]
    grads = torch.autograd.grad(ops.linear_scan(*leaves, return_state=True)[1], leaves, d_last.to(dev))
    for k in range(3):
        assert_close(grads[k], want[2 + k], tol[2 + k], k)
    # differentiable once: a graph of the gradients may be made, differentiating them raises -- also where the operator's
    # part would be one term of several
    leaves = [t.to(dev).requires_grad_(True) for t in (gate, x)]
    plain = torch.autograd.grad(ops.linear_scan(*leaves).sum(), leaves)
    tied = torch.autograd.grad(ops.linear_scan(*leaves).sum(), leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, tied))
    with pytest.raises(RuntimeError, match="differentiable once"):
        (tied[1].square().sum() + leaves[1].sum()).backward()


@pytest.mark.gpu
def test_large_gates_infinities_and_nan(dev):
    """A state of zero stays zero under gates whose products overflow; what is not finite spreads as in the formula and
    to no other column or sequence."""
    from nerf_amd import ops
    gate = torch.full((2, 300, 4), 1e30, device=dev)
    assert bool((ops.linear_scan(gate, torch.zeros(2, 300, 4, device=dev)) == 0).all())
    gate, x, _, _, _ = make(3, 300, 8, 8, F32, F32, False, 10, resets=0.0)
    clean = ops.linear_scan(gate.to(dev), x.to(dev)).cpu()
    for bad in (float("inf"), float("nan")):
        y = x.clone()
        y[1, 100, 3] = bad
        h = ops.linear_scan(gate.to(dev), y.to(dev)).cpu()
        assert torch.equal(h[0], clean[0]) and torch.equal(h[2], clean[2]) and torch.equal(h[1, :100], clean[1, :100])
        others = [c for c in range(8) if c != 3]
        assert torch.equal(h[1][:, others], clean[1][:, others]) and not bool(torch.isfinite(h[1, 100:, 3]).any())
    y = x.clone()
    y[:, 5] = 3e38                            # the largest values; the next gate lets nothing through
    g = gate.clone()
    g[:, 6] = 0.0
    h = ops.linear_scan(g.to(dev), y.to(dev)).cpu()
    assert torch.equal(h[:, 6], x[:, 6])


@pytest.mark.gpu
def test_streams_and_graph(dev):
    from nerf_amd import ops
    gate, x, s, d_h, d_last = (t.to(dev) for t in make(2, 2100, 24, 2, F32, F32, True, 11))

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (gate, x, s)]
        h, last = ops.linear_scan(*leaves, reverse=True, return_state=True)
        return [h.detach(), last.detach(), *torch.autograd.grad([h, last], leaves, [d_h, d_last])]

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        x.mul_(0.5)
        d_h.add_(0.25)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step(), out)), k
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_capture_refuses_a_live_eager_graph(dev):
    """Nothing of the refused call is captured; without the eager graph it is, and replays."""
    from nerf_amd import ops
    from nerf_amd._lib import NerfHipError
    gate, x, _, d_h, _ = (t.to(dev) if t is not None else None for t in make(3, 70, 8, 2, F32, F32, False, 3))
    table, ids = torch.randn(9, 8, device=dev, requires_grad=True), torch.arange(70, device=dev).expand(3, 70) % 9
    leaf = x.clone().requires_grad_(True)
    calls = {"scan": lambda: ops.linear_scan(gate, leaf), "lookup": lambda: ops.embedding(ids, table)}
    for name, of in (("scan", leaf), ("lookup", table)):
        call = calls[name]
        kept = call()
        want = torch.autograd.grad(kept, of, d_h, retain_graph=True)[0]
        torch.cuda.synchronize()
        with pytest.raises(NerfHipError, match="still alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        del kept
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(call(), of, d_h)[0]
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want), name


@pytest.mark.gpu
def test_two_streams_at_once(dev):
    """Calls that share the compute units, chained tiles and segments among them: each as if it were alone."""
    from nerf_amd import ops
    shapes = [(1, 9000, 640, 640), (2, 4000, 520, 520), (1, 20000, 4, 4), (700, 192, 3, 1)]
    data = [[t.to(dev) for t in make(*shape, F32, F32, True, k)[:4]] for k, shape in enumerate(shapes)]

    def step(gate, x, s, d_h):
        leaves = [t.detach().requires_grad_(True) for t in (gate, x, s)]
        h = ops.linear_scan(*leaves, blend=True)
        return [h.detach(), *torch.autograd.grad(h, leaves, d_h)]

    alone = [step(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    together = [None] * len(data)
    for _ in range(5):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                together[k] = step(*data[k])
    torch.cuda.synchronize()
    for one, other in zip(alone, together):
        assert all(torch.equal(a, b) for a, b in zip(one, other))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 900])
@pytest.mark.parametrize("G", [32768, 131072, 1])
def test_most_channels(dev, T, G):
    """The widest rows, with a gate for every few columns, a gate each and one for all: some columns in 64 bits."""
    from nerf_amd import ops
    B, C = 2, 131072
    gen = torch.Generator(device=dev).manual_seed(T)
    gate = torch.rand(B, T, G, device=dev, generator=gen).requires_grad_(True)
    x = torch.empty(B, T, C, device=dev).normal_(generator=gen).requires_grad_(True)
    h = ops.linear_scan(gate, x, reverse=True, blend=True)
    d_gate, d_x = torch.autograd.grad(h, [gate, x], x.detach())
    for c in (0, 65532, C - 8):
        cols = slice(c, c + 8)
        gates = slice(c * G // C, max((c + 8) * G // C, 1))
        g, v = gate.detach()[..., gates].cpu(), x.detach()[..., cols].cpu()
        want, tol = ref_scan(g, v, None, True, True, v, None), bounds(g, v, None, True, True, v, None)
        assert_close(h[..., cols], want[0], tol[0], ("h", c))
        assert_close(d_x[..., cols], want[3], tol[3], ("d_x", c))
        if G > 1:
            assert_close(d_gate[..., gates], want[2], tol[2], ("d_gate", c))


@pytest.mark.gpu
def test_more_than_two_to_the_31_elements(dev):
    """Offsets past 32 bits: the last rows of a large batch against the same rows alone."""
    from nerf_amd import ops
    B, T, C = 4200, 1024, 512                  # 2.2e9 elements of 2 bytes
    gen = torch.Generator(device=dev).manual_seed(12)
    x = torch.empty(B, T, C, device=dev, dtype=BF16).normal_(generator=gen).requires_grad_(True)
    gate = torch.rand(B, T, 1, device=dev, generator=gen).to(BF16)
    h = ops.linear_scan(gate, x)
    (d_x,) = torch.autograd.grad(h, x, x.detach())
    tail = x.detach()[-3:].clone().requires_grad_(True)
    # the number of rows has a part in how the time axis is cut, so the sums may differ by rounding: half a bf16 step and the float bound
    h2 = ops.linear_scan(gate[-3:], tail)
    (d2,) = torch.autograd.grad(h2, tail, tail.detach())
    tol = bounds(gate[-3:].cpu(), tail.detach().cpu(), None, False, False, tail.detach().cpu(), None)
    for got, want, t in ((h[-3:], h2, tol[0]), (d_x[-3:], d2, tol[3])):
        err = (got.detach().double().cpu() - want.detach().double().cpu()).abs()
        allow = 2 * t + torch.finfo(BF16).eps * (want.detach().double().cpu().abs() + t)
        assert float((err - allow).max()) <= 0.0


@pytest.mark.gpu
def test_entry_points_errors_reach_python(dev):
    from nerf_amd import ops
    from nerf_amd._lib import NerfHipError
    x = torch.zeros(1, 1, 131074, device=dev)
    for leaf in (x, x.clone().requires_grad_(True)):
        with pytest.raises(NerfHipError, match="131074 channels, at most 131072"):
            ops.linear_scan(leaf, leaf)


def test_refusals():
    from nerf_amd import ops
    from nerf_amd._lib import NerfHipError
    g, x = torch.zeros(2, 5, 4), torch.zeros(2, 5, 4)
    with pytest.raises(NerfHipError, match="GPU only"):
        ops.linear_scan(g, x)
    with pytest.raises(NerfHipError, match="float32, bfloat16 or float16"):
        ops.linear_scan(g, x.double())
    for bad in (lambda: ops.linear_scan(g[:, :, :3], x), lambda: ops.linear_scan(g[:, :4], x), lambda: ops.linear_scan(g[0], x),
                lambda: ops.linear_scan(g[:1], x), lambda: ops.linear_scan(g[..., :0], x), lambda: ops.linear_scan(g, x, torch.zeros(2, 3)),
                lambda: ops.linear_scan(g.int(), x), lambda: ops.linear_scan(g, x, torch.zeros(2, 4, dtype=torch.long)),
                lambda: ops.linear_scan(x[0, 0], x[0, 0])):
        with pytest.raises(ValueError):
            bad()


def test_entry_points_refuse():
    """Checked before anything is launched: no GPU needed."""
    from nerf_amd import _lib as L
    lib = L.lib()
    p, odd = 4096, 4100                        # never dereferenced
    ok = [p, 0, p, 0, None, 2, 5, 4, 2, 0, 0, p, None, None, None, None]
    def fwd(**k):
        a = list(ok)
        for i, v in k.items():
            a[int(i[1:])] = v
        return lib.nerf_linear_scan_fwd(*a)
    for k in ({"_0": None}, {"_2": None}, {"_11": None}, {"_1": 3}, {"_1": 1}, {"_3": 7}, {"_8": 3}, {"_8": 0}, {"_5": -1}, {"_6": 0}, {"_0": odd}, {"_2": odd},
              {"_11": odd}, {"_4": odd}, {"_12": odd}, {"_13": odd}, {"_5": 1 << 50}, {"_6": 1 << 39, "_5": 1}, {"_7": (1 << 17) + 2}):
        assert fwd(**k) == -22, k
        assert lib.nerf_last_error()
    assert fwd(_5=0) == 0 and fwd(_7=0) == 0   # nothing to do
    bwd = [p, 0, p, 0, None, None, p, None, 1, 5000, 4, 4, 0, 0, p, p, None, p, None]
    assert lib.nerf_linear_scan_carry_floats(1, 5000, 4, 4) > 0
    assert lib.nerf_linear_scan_bwd(*bwd) == -22 and b"null carry" in lib.nerf_last_error()
    bwd[5], bwd[17] = p, None
    assert lib.nerf_linear_scan_bwd(*bwd) == -22 and b"null workspace" in lib.nerf_last_error()
    assert lib.nerf_linear_scan_workspace_floats(1, 5000, 4, 3, 1) == 0


def test_entry_points_take_more_than_two_to_the_32_elements():
    """A gate for each channel has no sums over column tiles to hold, and the forward pass none at all: nothing about the
    number of elements is refused.  (Null outputs stop the calls before anything is launched: no GPU needed.)"""
    from nerf_amd import _lib as L
    lib = L.lib()
    p = 4096                                   # never dereferenced
    for B, T, C, G in ((1, (1 << 22) + 3, 1028, 1028), (2, 1 << 23, 1024, 1024), (16, 1 << 20, 640, 640), (3, 1 << 21, 1030, 1030)):
        assert B * T * G >= 1 << 32
        assert lib.nerf_linear_scan_fwd(p, 1, p, 1, None, B, T, C, G, 0, 0, None, None, None, None, None) == -22
        assert b"null pointer" in lib.nerf_last_error(), lib.nerf_last_error()
        assert lib.nerf_linear_scan_bwd(p, 1, None, 1, None, p, p, None, B, T, C, G, 0, 0, p, p, None, p, None) == -22
        assert b"null pointer" in lib.nerf_last_error(), lib.nerf_last_error()


@pytest.mark.gpu
def test_more_than_two_to_the_32_elements(dev):
    """One sequence with a gate for each channel: the steps behind the last reset, and behind the first of all, in 64 bits."""
    from nerf_amd import ops
    T, C, near = (1 << 22) + 3, 1028, 90       # 4.3e9 elements of 2 bytes
    gen = torch.Generator(device=dev).manual_seed(13)
    x = torch.empty(1, T, C, device=dev, dtype=BF16).normal_(generator=gen).requires_grad_(True)
    gate = torch.empty(1, T, C, device=dev, dtype=BF16).uniform_(generator=gen)
    for cut in (near, T - near):               # nothing passes from one side of it to the other, in either direction
        gate[:, cut] = 0.0
    gate.requires_grad_(True)
    h = ops.linear_scan(gate, x, blend=True)
    d_gate, d_x = torch.autograd.grad(h, [gate, x], x.detach())
    for steps in (slice(0, near), slice(T - near, T)):
        for cols in (slice(0, 8), slice(509, 519), slice(C - 8, C)):
            g, v = gate.detach()[:, steps, cols].cpu(), x.detach()[:, steps, cols].cpu()
            want, tol = ref_scan(g, v, None, False, True, v, None), bounds(g, v, None, False, True, v, None)
            if steps.start:                    # (what multiplies the gate of the cut comes from in front of it)
                d_first = d_gate[:, steps.start, cols].float()
                assert bool(torch.isfinite(d_first).all())
                d_gate[:, steps.start, cols] = want[2][:, 0].to(dev, BF16)
            for name, got, k in (("h", h, 0), ("d_gate", d_gate, 2), ("d_x", d_x, 3)):
                assert_close(got[:, steps, cols], want[k], tol[k], (name, steps, cols))


@pytest.mark.gpu
def test_capture_refuses_a_live_eager_graph_of_what_formed_the_operands(dev):
    """A leaf reached through other nodes, and a node that was made outside the capture, are refused like a leaf itself."""
    from nerf_amd import ops
    from nerf_amd._lib import NerfHipError
    _, x, s, d_h, _ = (t.to(dev) for t in make(3, 70, 8, 2, F32, F32, True, 3))
    sigma = torch.rand(3, 70, 2, device=dev, requires_grad=True)
    table, ids = torch.randn(9, 8, device=dev, requires_grad=True), torch.arange(70, device=dev).expand(3, 70) % 9
    start = s.clone().requires_grad_(True)
    calls = {"gate": (sigma, lambda: ops.linear_scan(torch.exp(-sigma * 0.5), x)), "state": (start, lambda: ops.linear_scan(sigma.detach(), x, start * 2)),
             "table": (table, lambda: ops.embedding(ids, (table * 0.5).reshape(9, 8)))}
    for name, (leaf, call) in calls.items():
        kept = call()
        want = torch.autograd.grad(kept, leaf, d_h, retain_graph=True)[0]
        torch.cuda.synchronize()
        with pytest.raises(NerfHipError, match="still alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        with torch.no_grad(), torch.cuda.graph(torch.cuda.CUDAGraph()):   # without a gradient there is nothing to refuse
            call()
        del kept
        formed = leaf * 1.0                    # this node's graph is alive; the leaf is not an operand by itself
        with pytest.raises(NerfHipError, match="still alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                ops.embedding(ids, formed) if name == "table" else ops.linear_scan(sigma.detach(), x, formed) if name == "state" else ops.linear_scan(formed, x)
        del formed
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(call(), leaf, d_h)[0]
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want), name


@pytest.mark.gpu
def test_capture_takes_a_graph_of_a_forked_stream(dev):
    """Nodes made on a stream that the capture has forked belong to it."""
    from nerf_amd import ops
    gate, x, _, _, _ = (t.to(dev) if t is not None else None for t in make(3, 70, 8, 2, F32, F32, False, 3))
    leaf = x.clone().requires_grad_(True)
    want = (ops.linear_scan(gate, leaf.detach()), ops.linear_scan(gate, leaf.detach() * 2))
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            first, twice = ops.linear_scan(gate, leaf), leaf * 2
        torch.cuda.current_stream().wait_stream(side)
        second = ops.linear_scan(gate, leaf)
        third = ops.linear_scan(gate, twice)
    for _ in range(3):
        for t in (first, second, third):
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, want[0]) and torch.equal(second, want[0]) and torch.equal(third, want[1])


@pytest.mark.gpu
def test_capture_takes_a_live_graph_of_another_stream(dev):
    """A graph that is alive on a stream other than the default one does not stand in the way: its accumulators' stream
    becomes part of the capture.  (What a warm-up on a side stream leaves behind.)"""
    from nerf_amd import ops
    gate, x, s, d_h, _ = (t.to(dev) for t in make(3, 70, 8, 2, F32, F32, True, 3))
    sigma, start = torch.rand(3, 70, 2, device=dev, requires_grad=True), s.clone().requires_grad_(True)
    table, ids = torch.randn(9, 8, device=dev, requires_grad=True), torch.arange(70, device=dev).expand(3, 70) % 9
    calls = {"gate": (sigma, lambda: ops.linear_scan(torch.exp(-sigma * 0.5), x)), "state": (start, lambda: ops.linear_scan(gate, x, start)),
             "table": (table, lambda: ops.embedding(ids, table))}
    side = torch.cuda.Stream()
    for name, (leaf, call) in calls.items():
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            kept = call()
            want = torch.autograd.grad(kept, leaf, d_h, retain_graph=True)[0]
        torch.cuda.synchronize()
        for whole in (False, True):            # the gradient handed back, and accumulated in the leaf
            leaf.grad = None
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                if whole:
                    call().backward(d_h)
                    got = leaf.grad
                else:
                    got = torch.autograd.grad(call(), leaf, d_h)[0]
            for _ in range(3):
                got.zero_()
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(got, want), (name, whole)
        leaf.grad = None
        del kept


# (type of x, of the gate, reverse, blend)
KINDS = [(F32, F32, False, False), (F32, F32, False, True), (BF16, BF16, False, False), (BF16, BF16, True, True), (BF16, F32, False, True), (BF16, F32, True, False),
         (F16, F16, True, False), (F16, F32, False, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("tx,tg,reverse,blend", KINDS)
@pytest.mark.parametrize("B,T,C,G", [
    # tiles in a chain, by columns a lane: four with a gate each (backward alone; both; sixteen steps a thread where all is of 16
    # bits), four, one and two of a shared gate, one with a gate each (sixteen steps a thread wherever x is of 16 bits)
    (3, 300, 132, 132), (3, 600, 132, 132), (3, 1100, 132, 132), (2, 1500, 520, 2), (4, 1100, 130, 2), (4, 600, 100, 2), (2, 1200, 252, 2), (4, 1021, 65, 65)])
def test_chains_by_type(dev, tx, tg, reverse, blend, B, T, C, G):
    check(dev, B, T, C, G, tx, tg, reverse, blend, state=not reverse, seed=T)


@pytest.mark.gpu
@pytest.mark.parametrize("tx,tg,reverse,blend", [(BF16, BF16, False, False), (F16, F32, True, True)])
@pytest.mark.parametrize("B,T,C,G", [(8, 4500, 6, 1), (8, 9000, 8, 1), (8, 17000, 12, 4), (8, 16500, 1, 1), (2, 17000, 520, 2), (2, 9000, 520, 520)])
def test_long_chains_by_type(dev, tx, tg, reverse, blend, B, T, C, G):
    """Few lanes side by side, so that a tile is thousands of steps; several groups of tiles."""
    check(dev, B, T, C, G, tx, tg, reverse, blend, state=True, seed=C)


@pytest.mark.gpu
@pytest.mark.parametrize("tx,tg", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("blend", [False, True])
@pytest.mark.parametrize("B,T", [(300, 192), (37, 196), (37, 197)])
@pytest.mark.parametrize("C", [1, 2, 3, 4])
def test_rays_of_few_channels(dev, tx, tg, reverse, blend, B, T, C):
    """One gate for one to four channels, whose steps are moved in whole pieces of 16 bytes: all of them whole, the last one
    partial, and none where a sequence does not start on a piece."""
    check(dev, B, T, C, 1, tx, tg, reverse, blend, state=C % 2 == 1, seed=C)


@pytest.mark.gpu
@pytest.mark.parametrize("tx,tg,reverse,blend", KINDS[2:])
@pytest.mark.parametrize("C", [2, 3, 4])
def test_rays_of_few_channels_in_segments(dev, tx, tg, reverse, blend, C):
    check(dev, 2, 2056, C, 1, tx, tg, reverse, blend, state=True, seed=C)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 40])
def test_gate_gradient_of_most_channels(dev, T):
    """One gate for 131072 channels: the sum over all of them, in 2048 column tiles.  A term passes the additions of its lane
    (3) and of 16 lanes (4) and up to 2048 over the tiles, in the place of the P that bounds() allows; all terms are positive, so
    that a tile left out or taken twice, 1/2048 of the sum, is beyond the bound (below 1/7000)."""
    from nerf_amd import ops
    B, C = 2, 131072
    gen = torch.Generator().manual_seed(T)
    gate, x, d_h = torch.rand(B, T, 1, generator=gen), torch.rand(B, T, C, generator=gen) + 0.5, torch.rand(B, T, C, generator=gen) + 0.5
    leaf = gate.to(dev).requires_grad_(True)
    (got,) = torch.autograd.grad(ops.linear_scan(leaf, x.to(dev), reverse=True), leaf, d_h.to(dev))
    want = ref_scan(gate, x, None, True, False, d_h)[2]
    tol = bounds(gate, x, None, True, False, d_h, None)[2] * ((4 * T + 2055 + 128) / (4 * T + C + 128))
    assert float(tol.max() / want.max()) < 1 / 7000
    assert_close(got, want, tol, T)

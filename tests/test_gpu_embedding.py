"""ops.embedding: rows bit for bit, the table's gradient against sums in 64 bits.

Gradients of whole numbers small enough that every partial sum is exact in float32 have to come out exactly, in any type
after one rounding; random ones within (n + 2) u of the sum of the magnitudes (u = 2^-24, n terms in a row, the product
with the scale among the roundings), plus half a step of a 16-bit type (eps / 2)."""
import pytest
import torch

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def make_ids(kind, N, V, gen):
    u = torch.rand(N, generator=gen, dtype=torch.float64)
    if kind == "one":
        return torch.full((N,), V // 2, dtype=torch.int64)
    if kind == "skewed":
        return (torch.pow(torch.tensor(V + 1.0, dtype=torch.float64), u).long() - 1).clamp_(0, V - 1)
    if kind == "borders":    # runs of 1 to 10 chunks of any power of two from 32 to 256 positions, ending at their borders and one past
        lengths = [(32 << (k % 4)) * (1 + k % 10) + (k % 3 == 2) - (k % 7 == 6) for k in range(V)]
        return torch.repeat_interleave(torch.arange(V), torch.tensor(lengths))[:N][torch.randperm(N, generator=gen)]
    if kind == "runs":       # long runs of one id, then another, some rows never
        return ((torch.arange(N) * 7) // max(1, N) * 3) % V
    return (u * V).long().clamp_(0, V - 1)


def want_grad(ids, d_out, V, scale, pad):
    d = d_out.double()
    if pad is not None:
        d = d * (ids != pad)[:, None]
    return scale * torch.zeros(V, d_out.shape[1], dtype=torch.float64).index_add_(0, ids, d)


@pytest.mark.gpu
@pytest.mark.parametrize("V,N,D,kind", [
    (1, 1, 1, "one"), (2, 63, 3, "uniform"), (40, 64, 32, "uniform"), (40, 65536, 32, "uniform"), (7, 127, 5, "runs"), (7, 128, 4, "one"), (9, 129, 8, "one"),
    (1023, 1000, 64, "skewed"), (1024, 8192, 16, "skewed"), (1025, 8193, 2, "uniform"), (70001, 20000, 100, "skewed"), (70001, 300, 520, "uniform"),
    (1100000, 100003, 2, "uniform"), (1100000, 9000, 1, "skewed"), (300, 30000, 65, "runs"), (3, 200000, 6, "one"), (524288, 262144, 2, "skewed"),
    (50, 5000, 1024, "skewed"), (100, 777, 2056, "uniform"), (2049, 16384, 24, "one"), (300000, 65, 7, "uniform"),
    (700, 1024, 12, "skewed"), (700, 1025, 12, "skewed"), (90, 4096, 40, "uniform"), (90, 4097, 40, "uniform"), (70001, 16385, 3, "skewed"), (8, 16385, 260, "runs"),
    (60, 28000, 2, "borders"), (60, 28000, 16, "borders"), (60, 28000, 48, "borders"), (30, 12000, 512, "borders"), (40, 16500, 1, "borders"),
    # rows of one vector: the smallest and the largest tables in buckets, one row more, buckets of no, one and many segments
    (1, 5000, 2, "one"), (2, 500000, 1, "one"), (33, 9000, 8, "uniform"), (5, 100003, 4, "skewed"), (1023, 70000, 4, "skewed"), (32768, 65536, 2, "uniform"),
    (32769, 66000, 8, "skewed"), (100000, 262145, 4, "runs"), (1048576, 20000, 4, "uniform"), (1048577, 20000, 4, "uniform"), (1048576, 400000, 2, "skewed")])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_and_exact_sums(dev, V, N, D, kind, dtype):
    from nerf_amd import ops
    gen = torch.Generator().manual_seed(N + D)
    ids = make_ids(kind, N, V, gen)
    table = torch.randn(V, D, generator=gen).to(dtype)
    d_out = torch.randint(-3, 4, (N, D), generator=gen).to(dtype)
    assert N * 3 < 2 ** 24
    t = table.to(dev).requires_grad_(True)
    for scale, pad in ((1.0, None), (0.5, V - 1)):
        out = ops.embedding(ids.to(dev), t, scale, pad)
        assert out.dtype == dtype and torch.equal(out.detach().cpu(), (table[ids].float() * scale).to(dtype))
        (g,) = torch.autograd.grad(out, t, d_out.to(dev))
        assert g.dtype == dtype and g.shape == t.shape
        assert torch.equal(g.cpu(), want_grad(ids, d_out, V, scale, pad).to(dtype)), (V, N, D, kind, dtype, scale)
    with torch.no_grad():
        assert torch.equal(ops.embedding(ids.to(dev).int(), t, 0.5), out)


@pytest.mark.gpu
@pytest.mark.parametrize("V,N,D,kind", [(40, 20000, 32, "uniform"), (5000, 9000, 96, "skewed"), (11, 5000, 7, "one"), (100, 100, 300, "uniform"), (3000, 50000, 4, "skewed"),
                                        (60, 9000, 2, "borders")])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_random_gradients(dev, V, N, D, kind, dtype):
    from nerf_amd import ops
    gen = torch.Generator().manual_seed(1)
    ids, scale = make_ids(kind, N, V, gen), 11.3137085
    d_out = torch.randn(N, D, generator=gen).to(dtype)
    t = torch.randn(V, D, generator=gen).to(dtype).to(dev).requires_grad_(True)
    out = ops.embedding(ids.to(dev), t, scale)
    want_out = t.detach().double().cpu()[ids] * scale
    half = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    # the scale itself is rounded to float32: 2 u in all
    assert float(((out.detach().double().cpu() - want_out).abs() - (2 * U + half) * 1.001 * want_out.abs()).max()) <= 1e-30
    (g,) = torch.autograd.grad(out, t, d_out.to(dev))
    want, mags = want_grad(ids, d_out, V, scale, None), want_grad(ids, d_out.abs(), V, scale, None)
    count = torch.bincount(ids, minlength=V).double()[:, None]
    tol = (count + 3) * U * mags
    tiny = 0.0 if dtype == F32 else torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert float(((g.double().cpu() - want).abs() - tol - half * (want.abs() + tol) - tiny).max()) <= 0.0
    (again,) = torch.autograd.grad(ops.embedding(ids.to(dev), t, scale), t, d_out.to(dev))
    assert torch.equal(again, g)


@pytest.mark.gpu
def test_gradient_by_differences(dev):
    """The lookup is linear in the table: a difference along any direction is the gradient's product with it, up to the
    roundings of the rows at both ends (u each of values below 8) and of the gradient."""
    from nerf_amd import ops
    gen = torch.Generator().manual_seed(2)
    ids = make_ids("uniform", 50, 6, gen).to(dev)
    t, w, d = (torch.randn(sh, generator=gen) for sh in ((6, 5), (50, 5), (6, 5)))
    leaf = t.to(dev).requires_grad_(True)
    (g,) = torch.autograd.grad(ops.embedding(ids, leaf, 1.5), leaf, w.to(dev))
    ends = [float((ops.embedding(ids, (t + s * d).to(dev), 1.5).double().cpu() * w.double()).sum()) for s in (1.0, -1.0)]
    want = float((g.double().cpu() * d.double()).sum())
    tol = (2 * 8 * U * 1.5 * 2 * w.abs().sum() + 55 * U * 1.5 * 50 * 5 * w.abs().max() * d.abs().max()).item()
    assert abs((ends[0] - ends[1]) / 2 - want) <= tol


@pytest.mark.gpu
def test_ids_out_of_range(dev):
    from nerf_amd import ops
    V, D = 10, 6
    ids = torch.tensor([3, -1, 10, 2 ** 40, -2 ** 40, 3, 9, 0] * 30)
    good = (ids >= 0) & (ids < V)
    table = torch.randn(V, D).to(dev).requires_grad_(True)
    out = ops.embedding(ids.to(dev), table)
    assert bool(out[~good.to(dev)].isnan().all()) and torch.equal(out[good.to(dev)].detach(), table.detach()[ids[good].to(dev)])
    d = torch.ones(len(ids), D, device=dev)
    d[~good.to(dev)] = float("nan")              # what arrives at a bad id goes nowhere
    (g,) = torch.autograd.grad(out, table, d)
    assert torch.equal(g.cpu(), torch.bincount(ids[good], minlength=V).float()[:, None].expand(V, D))
    out32 = ops.embedding(torch.tensor([-2147483648, 2147483647, 1], dtype=torch.int32, device=dev), table.detach())
    assert bool(out32[:2].isnan().all()) and torch.equal(out32[2], table.detach()[1])
    for n, width in ((500, D), (5000, D), (5000, 2)):     # none of them names a row
        table = torch.randn(V, width, device=dev, requires_grad=True)
        none = ops.embedding(torch.full((n,), -5, device=dev), table)
        (g,) = torch.autograd.grad(none, table, torch.full_like(none, float("nan")))
        assert bool((g == 0).all())
    table, many = torch.randn(V, 2, device=dev, requires_grad=True), ids.repeat(40)     # rows of one vector
    d = torch.ones(len(many), 2, device=dev)
    d[~good.repeat(40).to(dev)] = float("nan")
    (g,) = torch.autograd.grad(ops.embedding(many.to(dev), table), table, d)
    assert torch.equal(g.cpu(), 40 * torch.bincount(ids[good], minlength=V).float()[:, None].expand(V, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("N,V", [(1000, 5), (6000, 5), (6000, 2000)])
def test_infinities_and_nan_stay_in_their_rows(dev, N, V):
    from nerf_amd import ops
    ids = (torch.arange(N) % 5).to(dev)
    t = torch.randn(V, 4, device=dev).requires_grad_(True)
    d = torch.ones(N, 4, device=dev)
    d[2, 1], d[503, 2] = float("inf"), float("nan")
    (g,) = torch.autograd.grad(ops.embedding(ids, t, 1.0, padding_idx=3), t, d)
    want = torch.zeros(V, 4)
    want[:5] = N / 5.0
    want[3] = 0.0                                # the NaN arrived at the padding row
    want[2, 1] = float("inf")
    assert torch.equal(g.cpu(), want)


@pytest.mark.gpu
def test_shapes_strides_and_empty(dev):
    from nerf_amd import ops
    gen = torch.Generator().manual_seed(5)
    table = torch.randn(30, 12, generator=gen).to(dev)
    ids = torch.randint(0, 30, (3, 4, 5), generator=gen).to(dev)
    want = table[ids]
    assert torch.equal(ops.embedding(ids, table), want)
    assert torch.equal(ops.embedding(ids.transpose(0, 2), table), want.transpose(0, 2))
    assert torch.equal(ops.embedding(ids[..., 2], table), want[:, :, 2]) and torch.equal(ops.embedding(ids[0, 0, 0], table), want[0, 0, 0])
    for kind in (torch.uint8, torch.int16, torch.int32):
        assert torch.equal(ops.embedding(ids.to(kind), table), want)
    wide = torch.randn(30, 20, generator=gen).to(dev)
    leaf = wide.clone().requires_grad_(True)
    part = leaf[:, 3:15]                         # rows 20 apart, 12 bytes past a 16-byte boundary
    out = ops.embedding(ids, part)
    assert torch.equal(out.detach(), wide[:, 3:15][ids])
    (g,) = torch.autograd.grad(out.sum(), leaf)  # an expanded gradient
    full = torch.zeros(30, 20)
    full[:, 3:15] = torch.bincount(ids.cpu().reshape(-1), minlength=30).float()[:, None]
    assert torch.equal(g.cpu(), full)
    for shape in ((0,), (3, 0)):
        t = table.clone().requires_grad_(True)
        out = ops.embedding(torch.empty(shape, dtype=torch.long, device=dev), t)
        assert out.shape == (*shape, 12)
        (g,) = torch.autograd.grad(out.sum(), t)
        assert bool((g == 0).all()) and g.shape == t.shape
    t = torch.zeros(30, 0, device=dev, requires_grad=True)
    ops.embedding(ids, t).sum().backward()
    assert t.grad.shape == (30, 0)
    t = torch.zeros(0, 4, device=dev, requires_grad=True)
    assert ops.embedding(torch.zeros(0, dtype=torch.long, device=dev), t).shape == (0, 4)
    assert bool(ops.embedding(torch.zeros(2, dtype=torch.long, device=dev), t).isnan().all())
    ops.embedding(torch.zeros(2, dtype=torch.long, device=dev), t).sum().backward()
    leaf = table.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(ops.embedding(ids, leaf), leaf, torch.ones_like(want), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        (g.sum() + leaf.sum()).backward()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [20, 2])
@pytest.mark.parametrize("N", [3000, 20000])     # sorted by one workgroup, and by many
def test_streams_and_graph(dev, N, D):
    from nerf_amd import ops
    gen = torch.Generator().manual_seed(7)
    ids = make_ids("skewed", N, 3000, gen).to(dev)
    table, d_out = torch.randn(3000, D, generator=gen).to(dev), torch.randn(N, D, generator=gen).to(dev)

    def step():
        leaf = table.detach().requires_grad_(True)
        out = ops.embedding(ids, leaf, 2.0, 0)
        return [out.detach(), *torch.autograd.grad(out, leaf, d_out)]

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
        ids.copy_(torch.roll(ids, 17) if k else (ids + 1) % 3000)
        d_out.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step(), out)), k
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    from nerf_amd import ops
    V, D, N = 1 << 20, 2050, 70000               # 2.1e9 elements of 2 bytes in the table and in its gradient
    table = torch.zeros(V, D, device=dev, dtype=BF16)
    table[-1], table[0] = 3.0, 1.0
    ids = torch.full((N,), V - 1, device=dev)
    ids[::2] = 0
    t = table.requires_grad_(True)
    out = ops.embedding(ids, t)
    assert bool((out[1::2] == 3).all()) and bool((out[::2] == 1).all())
    (g,) = torch.autograd.grad(out, t, torch.ones_like(out))
    assert float(g[-1, 0]) == float(torch.tensor(35000.0).to(BF16)) and bool((g[-1] == g[-1, 0]).all()) and bool((g[0] == g[-1, 0]).all())
    assert not bool(g[1:-1].any())
    del t, table, g, out
    N = (1 << 20) + 77                           # and in the rows that come out
    ids = torch.zeros(N, dtype=torch.long, device=dev)
    ids[-1] = 1
    t = torch.arange(2, device=dev, dtype=F32)[:, None].expand(2, D).to(BF16).contiguous().requires_grad_(True)
    out = ops.embedding(ids, t)
    assert bool((out[-1] == 1).all()) and not bool(out[-1000:-1].any())
    d = torch.zeros_like(out)
    d[-2:] = 1
    (g,) = torch.autograd.grad(out, t, d)
    assert bool((g == 1).all())


def test_nodes_bind_to_the_library():
    """The C++ nodes call the entry points that the binding names: no GPU needed."""
    from nerf_amd import _lib as L
    native = L.native()
    assert native is L.native() and set(native.entries) <= set(L.SIGNATURES)
    assert {"nerf_embedding_bwd", "nerf_linear_scan_bwd", "nerf_last_error"} <= set(native.entries)


def test_refusals():
    from nerf_amd import ops
    from nerf_amd._lib import NerfHipError
    ids, table = torch.zeros(3, dtype=torch.long), torch.zeros(4, 2)
    with pytest.raises(NerfHipError, match="GPU only"):
        ops.embedding(ids, table)
    with pytest.raises(NerfHipError, match="float32, bfloat16 or float16"):
        ops.embedding(ids, table.double())
    for bad in (lambda: ops.embedding(ids.float(), table), lambda: ops.embedding(ids.bool(), table), lambda: ops.embedding(ids, table[0]),
                lambda: ops.embedding(ids, table, padding_idx=4), lambda: ops.embedding(ids, table, padding_idx=-5)):
        with pytest.raises(ValueError):
            bad()


def test_entry_points_refuse():
    """Checked before anything is launched: no GPU needed."""
    from nerf_amd import _lib as L
    lib = L.lib()
    p, odd = 4096, 4104                          # never dereferenced
    fwd = lambda table=p, type=0, V=9, D=4, ids=p, size=8, N=5, out=p: lib.nerf_embedding_fwd(table, type, V, D, ids, size, N, 1.0, out, None)  # noqa: E731
    for k in ({"table": None}, {"out": None}, {"ids": None}, {"type": 5}, {"size": 2}, {"V": -1}, {"D": -1}, {"N": -1}, {"table": odd}, {"out": odd}, {"ids": p + 4},
              {"V": 1 << 31}, {"N": 1 << 31}, {"D": 1 << 23}):
        assert fwd(**k) == -22 and lib.nerf_last_error(), k
    assert fwd(N=0) == 0 and fwd(D=0) == 0
    need = lib.nerf_embedding_bwd_workspace_bytes(5, 9, 4)
    bwd = lambda d_out=p, type=0, ids=p, size=8, N=5, V=9, D=4, grad=p, work=p, nbytes=need: lib.nerf_embedding_bwd(  # noqa: E731
        d_out, type, ids, size, N, V, D, 1.0, -1, grad, work, nbytes, None)
    for k in ({"d_out": None}, {"grad": None}, {"work": None}, {"nbytes": need - 1}, {"ids": None}, {"type": -1}, {"size": 1}, {"d_out": odd}, {"grad": odd}, {"work": odd}):
        assert bwd(**k) == -22 and lib.nerf_last_error(), k
    assert bwd(V=0) == 0 and bwd(D=0) == 0

"""Orthogonalisation and the Muon step against their formulas in 64 bits: sizes around the tiles, batches, matrices without
rank, far values, coefficients, copies, the optimizer.

Bounds.  What the documented roundings do is found by making them, in 64 bits: X to 32 bits, operands to fp16 (11 bits) for
bfloat16 and to two such parts for float32, and each product's sums off by as much as 32-bit sums may be, with random signs: 2^-24
times the magnitudes for each of the K / 16 steps (256 of K for float32, which are then added up) and six more.  The
error of a result against the formula is then of the same size: three times that, in the Frobenius norm, is the bound, and for
one value twelve times the root mean square (the error of some thousand values has no larger outliers unless a row or
column is far from the others: there the norm of that row and column counts)."""
import math

import pytest
import torch

from framewise_util import U, close

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
ABC = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module")
def fw():
    import i6_native_ops_b200.framewise as m

    return m


def formula(x, abc, steps, eps, rounded=None, gen=None):
    """``rounded``: float32 or bfloat16, with that type's roundings on the way."""
    x = x.double()
    if x.shape[-2] > x.shape[-1]:
        return formula(x.mT, abc, steps, eps, rounded, gen).mT
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp(min=eps)
    triples = abc if isinstance(abc[0], (tuple, list)) else [abc] * steps
    if rounded is None:
        for a, b, c in triples:
            g = x @ x.mT
            x = a * x + (b * g + c * g @ g) @ x
        return x
    parts = 2 if rounded == torch.float32 else 1

    def held(v):  # an operand: in the range of fp16 by a power of two
        s = 2.0 ** (14 - math.ceil(math.log2(max(float(v.abs().max()), 1e-30))))
        out, rest = torch.zeros_like(v), v * s
        for _ in range(parts):
            h = rest.half().double()
            out, rest = out + h, rest - h
        return out / s

    def times(p, q):
        K = p.shape[-1] if parts == 1 else min(p.shape[-1], 256)
        off = (K / 16 + 6) * parts * U * (p.abs() @ q.abs())
        return p @ q + off * (torch.rand(off.shape, dtype=torch.float64, device=off.device, generator=gen) * 2 - 1)

    x = x.float().double()
    for a, b, c in triples:
        o = held(x)
        g = held(times(o, o.mT))
        f = held(b * g + c * times(g, g))
        x = (a * x + times(f, o)).float().double()
    return x


def with_bound(x, abc=ABC, steps=5, eps=1e-7, dtype=None, out_type=None):
    """The result in 64 bits, and how far each value of it may be off."""
    dtype = dtype or x.dtype
    gen = torch.Generator(device="cuda").manual_seed(1)
    want = formula(x, abc, steps, eps)
    off = (formula(x, abc, steps, eps, dtype, gen) - want).square()
    m, n = x.shape[-2:]
    rms = torch.maximum(off.mean((-2, -1), keepdim=True), torch.maximum(off.mean(-1, keepdim=True), off.mean(-2, keepdim=True))).sqrt()
    r = torch.finfo(out_type or dtype).eps / 2
    norm = 3 * off.sum((-2, -1)).sqrt() + (r + 8 * U) * want.square().sum((-2, -1)).sqrt()
    return want, 12 * rms + (r + 8 * U) * want.abs(), norm


def check(got, bounds, name=""):
    want, each, norm = bounds
    close(got, (want, each), name)
    off = (got.double() - want).square().sum((-2, -1)).sqrt()
    assert bool((off <= norm + 1e-37).all()), (name, off, norm)


def matrices(cuda, shape, dtype=torch.float32, seed=0):
    """Some directions far stronger than the others, rows of their own sizes."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kw = dict(device=cuda, generator=gen)
    m, n = shape[-2:]
    rank = max(1, min(m, n) // 8)
    left = torch.randn(*shape[:-1], rank, **kw) * torch.logspace(0, -1.5, rank, device=cuda)
    x = left @ torch.randn(*shape[:-2], rank, n, **kw) / rank**0.5 + 0.3 * torch.randn(*shape, **kw)
    return (x * (0.7 * torch.randn(*shape[:-1], 1, **kw)).exp() * 1e-3).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (5, 1), (3, 64), (64, 3), (63, 65), (128, 128), (127, 129), (129, 300), (200, 65), (256, 64),
                                   (640, 257), (511, 513), (500, 2001), (1100, 1000), (2050, 700), (2, 3, 40, 50), (7, 130, 130), (0, 4, 5), (2, 0, 5)])
def test_sizes(fw, cuda, dtype, shape):
    x = matrices(cuda, shape, dtype, seed=sum(shape)) if 0 not in shape else torch.zeros(shape, device=cuda, dtype=dtype)
    before = x.clone()
    got = fw.orthogonalize(x)
    assert got.dtype == dtype and got.shape == x.shape and torch.equal(x, before)
    if x.numel():
        check(got, with_bound(x))
        assert torch.equal(fw.orthogonalize(x), got)


@pytest.mark.parametrize("dtype", TYPES)
def test_more_matrices_than_a_chain_takes(fw, cuda, dtype):
    x = matrices(cuda, (600, 9, 20), dtype, seed=4)
    got = fw.orthogonalize(x)
    check(got, with_bound(x))
    assert torch.equal(fw.orthogonalize(x[257:300]), got[257:300])


@pytest.mark.parametrize("dtype", TYPES)
def test_a_long_matrix_and_many_tiles(fw, cuda, dtype):
    for shape in ((130, 9000), (6000, 70)):
        x = matrices(cuda, shape, dtype, seed=8)
        check(fw.orthogonalize(x), with_bound(x))
    x = matrices(cuda, (24, 400, 900), dtype, seed=9)  # wide tiles
    check(fw.orthogonalize(x), with_bound(x))


@pytest.mark.parametrize("dtype", TYPES)
def test_rank_zeros_and_far_values(fw, cuda, dtype):
    x = matrices(cuda, (6, 150, 200), dtype, seed=2)
    x[0] = 0
    x[1, :, 1:] = 0  # one column
    x[2, 100:] = x[2, :50]  # equal rows
    x[3] = (x[3].double() * 1e30).to(dtype)
    x[4] = (x[4].double() * 1e-28).to(dtype)
    got = fw.orthogonalize(x, eps=1e-36)
    want = with_bound(x, eps=1e-36)
    check(got, want)
    assert not got[0].any()
    # below eps a matrix is not stretched
    tiny = (matrices(cuda, (40, 50), dtype, seed=3).double() * 1e-9).to(dtype)
    check(fw.orthogonalize(tiny, eps=1e-3), with_bound(tiny, eps=1e-3))


def test_nan_and_infinity_stay_in_their_matrix(fw, cuda):
    for dtype in TYPES:
        x = matrices(cuda, (5, 140, 70), dtype, seed=6)
        x[1, 3, 4] = float("nan")
        x[3, 139, 69] = float("inf")
        got = fw.orthogonalize(x)
        assert bool(got[[1, 3]].isnan().all())
        good = [0, 2, 4]
        check(got[good], with_bound(x[good]))


@pytest.mark.parametrize("dtype", TYPES)
def test_coefficients(fw, cuda, dtype):
    x = matrices(cuda, (90, 130), dtype, seed=12)
    cases = [((1.5, -0.5, 0.0), 8), ((2.0, -1.5, 0.5), 6), ([(4.0, -6.0, 2.5), (3.0, -3.0, 1.0), (1.875, -1.25, 0.375)], 3), ((1.0, 0.0, 0.0), 1), (ABC, 1)]
    for abc, steps in cases:
        check(fw.orthogonalize(x, steps=steps, coefficients=abc), with_bound(x, abc, steps), str(abc))


def test_strides(fw, cuda):
    x = matrices(cuda, (3, 60, 80), seed=14)
    want = fw.orthogonalize(x)
    assert torch.equal(fw.orthogonalize(x.mT.contiguous().mT), want)
    wide = torch.zeros(3, 60, 81, device=cuda)
    wide[..., 1:] = x
    assert torch.equal(fw.orthogonalize(wide[..., 1:]), want)
    check(fw.orthogonalize(x.mT), with_bound(x.mT))
    for shape in ((3, 60, 80), (2, 140, 272), (2, 272, 140)):
        for dtype in TYPES:
            x = matrices(cuda, shape, dtype, seed=15)
            want = fw.orthogonalize(x)
            for cut in (1, 2, 3, 4):  # values that begin anywhere
                flat = torch.zeros(x.numel() + cut, device=cuda, dtype=dtype)
                flat[cut:] = x.reshape(-1)
                assert torch.equal(fw.orthogonalize(flat[cut:].view(x.shape)), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(48, 96), (136, 264), (264, 136), (130, 257)])
def test_parameters_that_begin_anywhere(fw, cuda, dtype, shape):
    """Parameters, gradients, momentum and copies at any multiple of their type's size: the same bits."""
    n = shape[0] * shape[1]

    def cut(x, by):
        flat = torch.empty(n + by, device=cuda, dtype=x.dtype)
        flat[by:] = x.reshape(-1)
        return flat[by:].view(shape)

    gen = torch.Generator(device="cuda").manual_seed(5)
    p, g, v = torch.randn(shape, device=cuda, generator=gen).to(dtype), matrices(cuda, shape, dtype, seed=1), matrices(cuda, shape, seed=2)
    m = None if dtype == torch.float32 else [p.float()]
    first = [p.clone()], [v.clone()], None if m is None else [m[0].clone()]
    fw.muon_step(first[0], [g], first[1], lr=0.1, master=first[2])
    for by in ((1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (3, 2, 1, 5), (8, 4, 4, 4)):
        again = [cut(p, by[0])], [cut(v, by[2])], None if m is None else [cut(m[0], by[3])]
        fw.muon_step(again[0], [cut(g, by[1])], again[1], lr=0.1, master=again[2])
        assert torch.equal(again[0][0], first[0][0]) and torch.equal(again[1][0], first[1][0])
        assert m is None or torch.equal(again[2][0], first[2][0])


def reference_step(p, g, v, lr, beta, nesterov, decay, match, dtype, steps=5):
    """New momentum, parameter in 64 bits, each with a bound."""
    p, g, v = p.double(), g.double(), v.double()
    keep = 1 - beta
    new = v + (g - v) * keep
    dv = 6 * U * (v.abs() + g.abs())
    u = (g + (new - g) * beta) if nesterov else new
    want, each, _ = with_bound(u.float(), dtype=dtype, out_type=torch.float32, steps=steps)
    exact = formula(u, ABC, steps, 1e-7)  # the direction's own rounding is one more of X's
    s = 0.2 * math.sqrt(max(p.shape)) if match else math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
    out = p * (1 - lr * decay) - lr * s * exact
    return (new, dv), (out, lr * s * 2 * (each + (want - exact).abs()) + 4 * U * (p.abs() + lr * s * exact.abs()))


# up to 128 x 256 a CTA each, the others together; rows that begin at multiples of 16 bytes and elsewhere
SHAPES = [(64, 64), (40, 200), (200, 41), (1, 9), (300, 129), (128, 256), (256, 520), (520, 136), (131, 262)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nesterov,match", [(True, False), (False, True)])
def test_step(fw, cuda, dtype, nesterov, match):
    shapes = SHAPES * 7  # more than the arguments of a launch hold, of either kind
    gen = torch.Generator(device="cuda").manual_seed(5)
    p = [torch.randn(s, device=cuda, generator=gen).to(dtype) for s in shapes]
    g = [matrices(cuda, s, dtype, seed=i) for i, s in enumerate(shapes)]
    v = [matrices(cuda, s, seed=100 + i) for i, s in enumerate(shapes)]
    want = [reference_step(a, b, c, 0.05, 0.9, nesterov, 0.1, match, dtype) for a, b, c in zip(p, g, v)]
    before = [x._version for x in p + v]
    fw.muon_step(p, g, v, lr=0.05, beta=0.9, nesterov=nesterov, weight_decay=0.1, adjust_lr="match_rms_adamw" if match else "original")
    assert all(x._version > n for x, n in zip(p + v, before))
    r = torch.finfo(dtype).eps / 2
    for i, ((new, dv), (out, dout)) in enumerate(want):
        close(v[i], (new, dv), f"momentum {i}")
        close(p[i], (out, dout + r * out.abs()), f"parameter {i}")


@pytest.mark.parametrize("shapes", [SHAPES[:3], SHAPES[4:5], SHAPES[6:]])
def test_copies(fw, cuda, shapes):
    """With a copy in 32 bits the parameter is its rounded value; with ``follow`` a change of the parameter is taken over."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    master = [torch.randn(s, device=cuda, generator=gen) for s in shapes]
    p = [x.bfloat16() for x in master]
    g = [matrices(cuda, s, torch.bfloat16, seed=i) for i, s in enumerate(shapes)]
    v = [torch.zeros(s, device=cuda) for s in shapes]
    want = [reference_step(a, b, c, 0.05, 0.95, True, 0.1, False, torch.bfloat16) for a, b, c in zip(master, g, v)]
    fw.muon_step(p, g, v, lr=0.05, master=master)
    for i, (_, out) in enumerate(want):
        close(master[i], out, f"copy {i}")
        assert torch.equal(p[i], master[i].bfloat16())
    for follow in (False, True):
        held = [x.clone() for x in master]
        p[0][0].fill_(3.0)
        started = held[0].clone()
        if follow:
            started[0] = 3.0
        want = reference_step(started, g[0], v[0], 0.05, 0.95, True, 0.1, False, torch.bfloat16)[1]
        fw.muon_step(p, g, v, lr=0.05, master=master, follow=follow)
        close(master[0], want, "copy")


def test_a_zero_gradient_leaves_the_decay(fw, cuda):
    p = [torch.randn(30, 40, device=cuda)]
    want = p[0] * (1 - 0.1 * 0.5)
    fw.muon_step(p, [torch.zeros(30, 40, device=cuda)], [torch.zeros(30, 40, device=cuda)], lr=0.1, weight_decay=0.5)
    close(p[0], (want.double(), 2 * U * want.abs().double()))


@pytest.mark.parametrize("dtype", TYPES)
def test_optimizer(fw, cuda, dtype):
    gen = torch.Generator(device="cuda").manual_seed(0)
    params = [torch.nn.Parameter(torch.randn(s, device=cuda, generator=gen).to(dtype)) for s in SHAPES[2:7]]
    plain = [x.detach().clone() for x in params]
    momentum = [torch.zeros(x.shape, device=cuda) for x in plain]
    master = None if dtype == torch.float32 else [x.float() for x in plain]
    opt = fw.Muon(params, lr=0.03, weight_decay=0.2, adjust_lr="match_rms_adamw")
    for step in range(3):
        for i, x in enumerate(params):
            x.grad = matrices(cuda, x.shape, dtype, seed=10 * step + i)
        if step == 2:
            params[1].grad = None
            opt.param_groups[0]["lr"] = 0.01
        keep = [i for i, x in enumerate(params) if x.grad is not None]
        opt.step()
        pick = lambda xs: None if xs is None else [xs[i] for i in keep]  # noqa: E731
        fw.muon_step(pick(plain), [params[i].grad for i in keep], pick(momentum), lr=0.03 if step < 2 else 0.01, weight_decay=0.2,
                     adjust_lr="match_rms_adamw", master=pick(master))
        for a, b in zip(params, plain):
            assert torch.equal(a.detach(), b)
    # states keep their types when they are loaded, and go on alike
    other = [torch.nn.Parameter(x.detach().clone()) for x in params]
    again = fw.Muon(other, lr=0.01, weight_decay=0.2, adjust_lr="match_rms_adamw")
    again.load_state_dict(opt.state_dict())
    for a, b in zip(params, other):
        b.grad = a.grad = matrices(cuda, a.shape, dtype, seed=77)
        assert again.state[b]["momentum"].dtype == torch.float32
    opt.step(), again.step()
    for a, b in zip(params, other):
        assert torch.equal(a.detach(), b.detach())


def test_other_streams_and_graphs(fw, cuda):
    x = matrices(cuda, (2, 200, 300), seed=31)
    want = fw.orthogonalize(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fw.orthogonalize(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    p, g, v = [torch.randn(200, 300, device=cuda)], [x[0].clone()], [torch.zeros(200, 300, device=cuda)]
    start = p[0].clone()
    with torch.cuda.graph(first):
        got = fw.orthogonalize(x)
    with torch.cuda.graph(second, pool=first.pool()):
        fw.muon_step(p, g, v, lr=0.1)
    for _ in range(2):
        got.zero_()
        p[0].copy_(start), v[0].zero_()
        first.replay()
        second.replay()
        eager = [start.clone()], [torch.zeros(200, 300, device=cuda)]
        fw.muon_step(eager[0], g, eager[1], lr=0.1)
        assert torch.equal(got, want) and torch.equal(p[0], eager[0][0]) and torch.equal(v[0], eager[1][0])
        g[0].copy_(x[1])


def test_a_step_between_a_loss_and_its_gradients_is_an_error(fw, cuda):
    w = torch.nn.Parameter(torch.randn(20, 30, device=cuda))
    opt = fw.Muon([w])
    loss = (w * w).sum()
    w.grad = torch.ones_like(w)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_refusals(fw, cuda):
    x = torch.randn(4, 5, device=cuda)
    step = lambda *a, **k: fw.muon_step(*a, **k)  # noqa: E731
    bad = [
        (lambda: fw.orthogonalize(x.half()), "float32 or bfloat16"),
        (lambda: fw.orthogonalize(x.cpu()), "CUDA"),
        (lambda: fw.orthogonalize(x[0]), "rows, cols"),
        (lambda: fw.orthogonalize(x, steps=0), "steps"),
        (lambda: fw.orthogonalize(x, steps=101), "steps"),
        (lambda: fw.orthogonalize(x, eps=0.0), "eps"),
        (lambda: fw.orthogonalize(x, coefficients=(1.0, 2.0)), "coefficients"),
        (lambda: fw.orthogonalize(x, steps=2, coefficients=[ABC]), "coefficients"),
        (lambda: fw.orthogonalize(x, coefficients=(float("nan"), 0.0, 0.0)), "finite"),
        (lambda: fw.orthogonalize(x, coefficients=(100.0, 0.0, 0.0)), "coefficients"),
        (lambda: fw.orthogonalize(x.requires_grad_()), "no gradient"),
    ]
    y = x.detach().clone()
    g, v = torch.zeros_like(y), torch.zeros_like(y)
    bad += [
        (lambda: step([y], [g], []), "one entry per parameter"),
        (lambda: step([y[0]], [g[0]], [v[0]]), "matrices"),
        (lambda: step([y.T], [g.T], [v.T]), "contiguous"),
        (lambda: step([y], [g.double()], [v]), "gradient"),
        (lambda: step([y], [g[:2]], [v]), "gradient"),
        (lambda: step([y], [g], [v.bfloat16()]), "momentum"),
        (lambda: step([y], [g], [v], beta=1.0), "beta"),
        (lambda: step([y], [g], [v], lr=-1.0), "lr"),
        (lambda: step([y], [g], [v], master=[v]), "no copies"),
        (lambda: step([y, y.bfloat16()], [g, g.bfloat16()], [v, v]), "share"),
        (lambda: step([y], [g.cpu()], [v]), "gradient"),
        (lambda: step([y, y], [g, g], [v, v.clone()]), "twice"),
        (lambda: step([y, y.clone()], [g, g], [v, v]), "twice"),
        (lambda: step([y.bfloat16()], [g.bfloat16()], [v], master=[v]), "twice"),
    ]
    for f, what in bad:
        with pytest.raises(RuntimeError, match=what):
            f()
    with pytest.raises(ValueError, match="matrices"):
        fw.Muon([torch.nn.Parameter(torch.zeros(5, device=cuda))])
    with pytest.raises(ValueError, match="adjust_lr"):
        step([y], [g], [v], adjust_lr="other")
    assert not v.any()
    with torch.no_grad():
        fw.orthogonalize(x)

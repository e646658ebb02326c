"""AdamW against its formula in 64 bits, 8-bit states against their definition bit for bit, and the optimizer class."""
import pytest
import torch

from framewise_util import U, adamw_reference, close, codes_of, values_of

pytestmark = pytest.mark.gpu

SIZES = [(1,), (7,), (255,), (256,), (257,), (3, 5), (100, 33), (64, 64), (2049,), (0,), (31, 257)]
HYPER = dict(lr=3e-3, betas=(0.9, 0.98), eps=1e-8, weight_decay=0.1)


@pytest.fixture(scope="module")
def fw():
    import i6_native_ops_b200.framewise as m

    return m


def tensors(cuda, dtype, sizes=SIZES, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kw = dict(device=cuda, generator=gen)
    p = [torch.randn(s, **kw).to(dtype) for s in sizes]
    g = [(torch.randn(s, **kw) * 10.0 ** float(torch.randint(-6, 2, (), device=cuda, generator=gen))).to(dtype) for s in sizes]
    m = [torch.randn(s, **kw) * 0.1 * x.abs().float().mean().nan_to_num() for s, x in zip(sizes, g)]
    v = [torch.rand(s, **kw) * (x.float() ** 2).mean().nan_to_num() for s, x in zip(sizes, g)]
    return p, g, m, v


def bounds(p, g, m, v, step, lr, betas, eps, weight_decay, r):
    """Values in 64 bits and how far single operations in 32 bits may be: three roundings in m, four in v (each of a
    term's magnitude), and in the update ten of its own plus those of m and of the root (half of v's)."""
    new_p, new_m, new_v = adamw_reference(p, g, m, v, step, lr, betas, eps, weight_decay)
    mag = betas[0] * m.double().abs() + (1 - betas[0]) * g.double().abs()
    dm = 3 * U * mag
    dv = 5 * U * new_v
    den = (new_v / (1 - betas[1] ** step)).sqrt() + eps
    rate = lr / (1 - betas[0] ** step)
    update = rate * (new_m.abs() / den)
    dp = rate * dm / den + 14 * U * update + 4 * U * p.double().abs() + r * new_p.abs()
    return (new_p, dp), (new_m, dm), (new_v, dv)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("step", [1, 400])
def test_states_of_32_bits(fw, cuda, dtype, step):
    p, g, m, v = tensors(cuda, dtype)
    for master in (False, True) if dtype == torch.bfloat16 else (False,):
        x = [t.float() + 1e-3 for t in p] if master else p
        want = [bounds(*t, step, r=U, **{**HYPER}) for t in zip(x, g, m, v)]
        p2, m2, v2 = ([t.clone() for t in q] for q in (p, m, v))
        x2 = [t.clone() for t in x] if master else None
        fw.adamw_step(p2, g, m2, v2, step=step, master=x2, **HYPER)
        r = torch.finfo(dtype).eps / 2
        for i, (wp, wm, wv) in enumerate(want):
            close(m2[i], wm, "exp_avg")
            close(v2[i], wv, "exp_avg_sq")
            if master:
                close(x2[i], wp, "master")
                assert torch.equal(p2[i], x2[i].to(dtype))
            else:
                close(p2[i], (wp[0], wp[1] + r * wp[0].abs()), "param")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_states_of_8_bits(fw, cuda, dtype):
    """Three steps: the codes are those of the definition, bit for bit."""
    p, g, m, v = tensors(cuda, dtype)
    x = None if dtype == torch.float32 else [t.float() for t in p]
    em, ev = [codes_of(t, 127) for t in m], [codes_of(t.sqrt(), 255) for t in v]
    f32 = lambda y: torch.tensor(y, dtype=torch.float32, device=cuda)  # noqa: E731
    b1, b2 = HYPER["betas"]
    for step in (5, 6, 7):
        want = []
        for i in range(len(p)):
            # the step's single operations, each rounded
            mm, rr = values_of(*em[i]), values_of(*ev[i])
            gg = g[i].float()
            mm = mm * f32(b1) + gg * f32(1 - b1)
            vv = (rr * rr) * f32(b2) + (gg * gg) * f32(1 - b2)
            rr = vv.sqrt()
            y = p[i] if x is None else x[i]
            y = y * f32(1 - HYPER["lr"] * HYPER["weight_decay"]) - (mm * f32(HYPER["lr"] / (1 - b1**step))) / (
                rr * f32(1 / (1 - b2**step) ** 0.5) + f32(HYPER["eps"]))
            want.append((y, codes_of(mm, 127), codes_of(rr, 255)))
        fw.adamw_step(p, g, em, ev, step=step, master=x, **HYPER)
        values = fw.adamw_values(em, ev)
        for i, (y, cm, cv) in enumerate(want):
            assert torch.equal(em[i][0], cm[0]) and torch.equal(em[i][1], cm[1])
            assert torch.equal(ev[i][0], cv[0]) and torch.equal(ev[i][1], cv[1])
            assert torch.equal(p[i], y.to(dtype)) and (x is None or torch.equal(x[i], y))
            assert torch.equal(values[0][i], values_of(*cm)) and torch.equal(values[1][i], values_of(*cv).square())


def test_codes_keep_their_values(fw, cuda):
    """A moment is held to half a code: sqrt(x / k) to 1/2, so x to (c + 1/4) k."""
    p, g, m, v = tensors(cuda, torch.float32, [(5000,)])
    zero = [(torch.zeros(5000, dtype=t, device=cuda), torch.zeros(20, device=cuda)) for t in (torch.int8, torch.uint8)]
    m32, v32 = [torch.zeros(5000, device=cuda)], [torch.zeros(5000, device=cuda)]
    fw.adamw_step([p[0].clone()], g, m32, v32, step=1, **HYPER)
    em, ev = [zero[0]], [zero[1]]
    fw.adamw_step([p[0].clone()], g, em, ev, step=1, **HYPER)
    got = fw.adamw_values(em, ev)
    for have, codes, want in ((got[0][0], em[0], m32[0]), (got[1][0].sqrt(), ev[0], v32[0].sqrt())):
        k = codes[1].repeat_interleave(256)[:5000]
        c = codes[0].float().abs()
        assert bool(((have - want).abs() <= (c + 0.26) * k + 1e-6 * want.abs()).all())
    assert bool((ev[0][0][v32[0] > 0] > 0).all())


def test_blocks_with_an_infinity_or_a_nan(fw, cuda):
    p, g, m, v = tensors(cuda, torch.float32, [(1000,)])
    g[0][300] = float("nan")
    g[0][600] = float("inf")
    em, ev = [codes_of(m[0], 127)], [codes_of(v[0].sqrt(), 255)]
    fw.adamw_step(p, g, em, ev, step=3, **HYPER)
    a, b = fw.adamw_values(em, ev)
    assert bool(a[0][256:512].isnan().all()) and bool((a[0][512:768] == float("inf")).all()) and bool((b[0][512:768] == float("inf")).all())
    for x in (a[0], b[0]):
        assert bool(x[:256].isfinite().all()) and bool(x[768:].isfinite().all())
    assert int(p[0].isnan().sum()) == 2
    # 32 bits: the elements alone
    p, g, m, v = tensors(cuda, torch.float32, [(1000,)])
    g[0][300] = float("nan")
    fw.adamw_step(p, g, m, v, step=3, **HYPER)
    assert int(p[0].isnan().sum()) == int(m[0].isnan().sum()) == int(v[0].isnan().sum()) == 1


@pytest.mark.parametrize("bits", [8, 32])
def test_many_tensors_and_odd_addresses(fw, cuda, bits):
    """More tensors than a launch takes, parameters as views of one buffer at odd offsets: the same bits as one by one."""
    sizes = [(1 + 37 * i % 700,) for i in range(130)]
    p, g, m, v = tensors(cuda, torch.float32, sizes)
    states = lambda: ([codes_of(t, 127) for t in m], [codes_of(t.sqrt(), 255) for t in v]) if bits == 8 else (  # noqa: E731
        [t.clone() for t in m], [t.clone() for t in v])
    flat = torch.zeros(1 + sum(t.numel() for t in p), device=cuda)
    at, views = 1, []
    for t in p:
        views.append(flat[at : at + t.numel()])
        views[-1].copy_(t)
        at += t.numel()
    a, b = states()
    fw.adamw_step(views, g, a, b, step=9, **HYPER)
    c, d = states()
    for i in range(len(p)):
        fw.adamw_step([p[i]], [g[i]], [c[i]], [d[i]], step=9, **HYPER)
    assert all(torch.equal(x, y) for x, y in zip(views, p)) and float(flat[0]) == 0
    pick = (lambda s: s[0]) if bits == 8 else (lambda s: s)
    assert all(torch.equal(pick(x), pick(y)) for x, y in zip(a + b, c + d))


def test_optimizer(fw, cuda):
    """The class against torch's own AdamW over some steps, with a parameter that has no gradient and one whose gradient is
    strided.  Both round a few times a step: 20 steps of at most lr (1 + weight decay) each, 2^-20 of that."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    shapes = [(30, 40), (40,), (7, 9), (5,)]
    a = [torch.nn.Parameter(torch.randn(s, device=cuda, generator=gen)) for s in shapes]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    oa = fw.AdamW(a, **HYPER)
    ob = torch.optim.AdamW(b, **HYPER, foreach=False, fused=False)
    for i in range(20):
        for o in (oa, ob):
            o.param_groups[0]["lr"] = 1e-3 * (i + 1)
        for x, y in zip(a[:3], b[:3]):
            g = torch.randn(x.shape, device=cuda, generator=gen)
            x.grad = g.t().contiguous().t() if g.dim() == 2 else g
            y.grad = g.clone()
        oa.step()
        ob.step()
    for x, y in zip(a, b):
        assert float((x - y).detach().abs().max()) <= 20 * 0.02 * 2.0**-16 + 20 * U * 4
    assert not oa.state[a[3]]


@pytest.mark.parametrize("bits", [8, 32])
def test_state_dict(fw, cuda, bits):
    """A step after loading is the step that would have followed, whatever the parameters' type."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    a = [torch.nn.Parameter(torch.randn(50, 70, device=cuda, generator=gen).bfloat16())]
    grads = [torch.randn(50, 70, device=cuda, generator=gen).bfloat16() for _ in range(4)]
    o = fw.AdamW(a, state_bits=bits, **HYPER)
    for g in grads[:2]:
        a[0].grad = g
        o.step()
    b = [torch.nn.Parameter(a[0].detach().clone())]
    o2 = fw.AdamW(b, state_bits=bits, **HYPER)
    o2.load_state_dict(o.state_dict())
    for g in grads[2:]:
        a[0].grad, b[0].grad = g, g
        o.step()
        o2.step()
    assert torch.equal(a[0], b[0])
    for k, x in o.state[a[0]].items():
        y = o2.state[b[0]][k]
        assert torch.equal(x, y) and x.dtype == y.dtype if isinstance(x, torch.Tensor) else x == y


def test_closure_and_another_stream(fw, cuda):
    p = torch.nn.Parameter(torch.ones(300, device=cuda))
    o = fw.AdamW([p], lr=0.1)

    def closure():
        o.zero_grad()
        loss = (p * p).sum()
        loss.backward()
        return loss

    assert float(o.step(closure).detach()) == 300.0
    q = torch.nn.Parameter(torch.ones(300, device=cuda))
    o2 = fw.AdamW([q], lr=0.1)
    q.grad = 2 * torch.ones(300, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2.step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(p.detach(), q.detach())


def test_refusals(fw, cuda):
    p, g, m, v = tensors(cuda, torch.float32, [(8, 6)])
    ok = dict(step=1, **HYPER)
    em, ev = [codes_of(m[0], 127)], [codes_of(v[0].sqrt(), 255)]
    for args, kw in [
        (([p[0].cpu()], g, m, v), {}), (([p[0].half()], g, m, v), {}), (([p[0].T], [g[0].T], [m[0].T], [v[0].T]), {}),
        ((p, [g[0].bfloat16()], m, v), {}), ((p, [g[0][:3]], m, v), {}), ((p, g[:0], m, v), {}), ((p, g, m[:0], v), {}),
        ((p, g, [m[0].bfloat16()], v), {}), ((p, g, [m[0][:4]], v), {}), ((p, [g[0].to_sparse()], m, v), {}),
        ((p, g, [(em[0][0], em[0][1][:0])], ev), {}), ((p, g, [(em[0][0].float(), em[0][1])], ev), {}), ((p, g, em, v), {}),
        ((p, g, m, v), dict(step=0)), ((p, g, m, v), dict(lr=-1.0)), ((p, g, m, v), dict(betas=(1.0, 0.9))), ((p, g, m, v), dict(eps=-1.0)),
        ((p, g, m, v), dict(master=[p[0].bfloat16()])), ((p, g, m, v), dict(master=[p[0], p[0]])),
    ]:
        with pytest.raises(RuntimeError):
            fw.adamw_step(*args, **{**ok, **kw})
    with pytest.raises(ValueError):
        fw.AdamW([torch.nn.Parameter(p[0])], state_bits=16)

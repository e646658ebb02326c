"""8-bit states of AdamW with betas near one: codes by their definition bit for bit, and moments over thousands of steps."""
import pytest
import torch

from framewise_util import codes_of, values_of

pytestmark = pytest.mark.gpu

TURNS = 3242174889, 2447445413


@pytest.fixture(scope="module")
def fw():
    import i6_native_ops_b200.framewise as m

    return m


def offsets(shape, step, second, device):
    i = torch.arange(torch.Size(shape).numel(), device=device, dtype=torch.int64).view(shape)
    a, b = TURNS if second else TURNS[::-1]
    return (((i * a + step * b) % 2**32) >> 9).float() * 2.0**-23 - 0.5


def moved_codes(x, top, off, block=256):
    """8-bit codes and steps with offsets, by the definition."""
    n = x.numel()
    flat, off = (torch.nn.functional.pad(y.reshape(-1), (0, -n % block)).reshape(-1, block) for y in (x, off))
    k = flat.abs().amax(1, keepdim=True) * torch.tensor(1.0 / (top * top), device=x.device)
    k = torch.where(k < 2.0**-120, torch.zeros_like(k), k)
    c = ((flat.abs() * (torch.ones_like(k) / k)).sqrt() + off).round().clamp(0, top)
    if top == 255:
        c = torch.where(flat > 0, c.clamp(min=1), c)
    c = torch.where(k > 0, c, torch.zeros_like(c)) * flat.sign()
    return c.reshape(-1)[:n].reshape(x.shape).to(torch.int8 if top == 127 else torch.uint8), k.reshape(-1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.9, 0.9801), (0.99, 0.95)])
def test_codes_with_offsets(fw, cuda, dtype, betas):
    gen = torch.Generator(device="cuda").manual_seed(7)
    kw = dict(device=cuda, generator=gen)
    sizes = [(1,), (7,), (256,), (257,), (3, 5), (31, 257), (0,), (300, 1000)]
    p = [torch.randn(s, **kw).to(dtype) for s in sizes]
    g = [(torch.randn(s, **kw) * 10.0 ** (4 * torch.rand(s, **kw) - 4)).to(dtype) for s in sizes]
    g[5][3:9] = 0
    em = [codes_of(torch.randn(s, **kw) * 0.1, 127) for s in sizes]
    ev = [codes_of(torch.rand(s, **kw), 255) for s in sizes]
    x = None if dtype == torch.float32 else [t.float() for t in p]
    hyper = dict(lr=3e-3, betas=betas, eps=1e-8, weight_decay=0.1)
    f32 = lambda y: torch.tensor(y, dtype=torch.float32, device=cuda)  # noqa: E731
    b1, b2 = betas
    for step in (1, 2, 999, 123456789):
        want = []
        for i in range(len(p)):
            mm, rr, gg = values_of(*em[i]), values_of(*ev[i]), g[i].float()
            mm = mm * f32(b1) + gg * f32(1 - b1)
            rr = ((rr * rr) * f32(b2) + (gg * gg) * f32(1 - b2)).sqrt()
            want.append((moved_codes(mm, 127, offsets(sizes[i], step, False, cuda)), moved_codes(rr, 255, offsets(sizes[i], step, True, cuda))))
        fw.adamw_step(p, g, em, ev, step=step, master=x, **hyper)
        for i, (cm, cv) in enumerate(want):
            for have, c in ((em[i], cm), (ev[i], cv)):
                assert torch.equal(have[0], c[0]) and torch.equal(have[1], c[1]), (step, sizes[i])


def roots(fw, optimizer, p):
    s = optimizer.state[p]
    return fw.adamw_values([(s["exp_avg"], s["exp_avg_steps"])], [(s["exp_avg_sq"], s["exp_avg_sq_steps"])])[1][0].sqrt()


def test_moments_follow_gradients_over_thousands_of_steps(fw, cuda):
    """The class's own betas.  Half of each block's gradients fall to a tenth after 1000 steps, 3000 more follow; a
    quarter of the other half is a tenth and a hundredth throughout.  In 32 bits roots are right; in 8 bits a root with
    code c has a spread of about 1 / sqrt(2 c) and an upward bias below 1 / c, so the mean ratio of thousands of values is
    within 2 / c of one, with c from 25 (a hundredth of the block's largest; about 255 / 10) to 255."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    n = 256 * 64
    kind = torch.arange(n, device=cuda) % 4
    early = torch.ones(n, device=cuda)
    early[kind == 1], early[kind == 2] = 0.1, 0.01
    late = early.clone()
    falls = (kind == 0) & (torch.arange(n, device=cuda) % 8 == 0)
    late[falls] = 0.1
    p8, p32 = (torch.nn.Parameter(torch.zeros(n, device=cuda)) for _ in range(2))
    o8, o32 = fw.AdamW([p8], lr=1e-4, state_bits=8), fw.AdamW([p32], lr=1e-4)
    for step in range(4000):
        p8.grad = p32.grad = torch.randn(n, device=cuda, generator=gen) * (early if step < 1000 else late)
        o8.step()
        o32.step()
    ratio = roots(fw, o8, p8) / o32.state[p32]["exp_avg_sq"].sqrt()
    for name, at, code in (("falls", falls, 80), ("top", (kind == 3) | ((kind == 0) & ~falls), 220), ("tenth", kind == 1, 80), ("hundredth", kind == 2, 25)):
        r = ratio[at]
        assert abs(float(r.mean()) - 1) <= 2 / code, (name, float(r.mean()))
        assert float((r - 1).abs().quantile(0.99)) <= 4 / (2 * code) ** 0.5, (name, float(r.min()), float(r.max()))
    # the weights have gone as far: their steps are what the moments say
    move = (p8 - p32).detach().abs().mean() / p32.detach().abs().mean()
    assert float(move) <= 0.2

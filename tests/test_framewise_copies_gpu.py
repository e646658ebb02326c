"""The float32 copies that AdamW keeps of bfloat16 parameters, and changes of the parameters between steps."""
import pytest
import torch

from framewise_util import codes_of

pytestmark = pytest.mark.gpu

HYPER = dict(lr=3e-3, betas=(0.9, 0.98), eps=1e-8, weight_decay=0.1)


@pytest.fixture(scope="module")
def fw():
    import i6_native_ops_b200.framewise as m

    return m


def edits():
    """Ways in which programs change a parameter; each leaves some values as they were."""

    def clip(p):
        with torch.no_grad():
            p.clamp_(-0.5, 0.5)

    def data(p):
        p.data[3:40] = 0.25

    def whole(p):
        p.data = torch.where(torch.arange(p.numel(), device=p.device) % 3 == 0, 1.5, p.data).to(p.dtype)

    def nothing(p):
        pass

    return [clip, data, whole, nothing]


@pytest.mark.parametrize("bits,betas", [(32, (0.9, 0.98)), (8, (0.9, 0.98)), (8, (0.9, 0.999))])
@pytest.mark.parametrize("edit", edits(), ids=lambda f: f.__name__)
def test_changes_between_steps_are_kept(fw, cuda, bits, betas, edit):
    """A step after a change starts from the changed values, and where nothing changed from the copy's 32 bits: the same
    step as by hand, from a copy that was put right."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    p = torch.nn.Parameter(torch.randn(1000, device=cuda, generator=gen).bfloat16())
    o = fw.AdamW([p], state_bits=bits, **{**HYPER, "betas": betas})
    grads = [torch.randn(1000, device=cuda, generator=gen).bfloat16() for _ in range(4)]
    for g in grads[:3]:
        p.grad = g
        o.step()
    s = o.state[p]
    assert not torch.equal(s["master"], p.detach().float())  # the copy holds more bits
    edit(p)
    want = torch.where(s["master"].bfloat16() == p.detach(), s["master"], p.detach().float())
    x = p.detach().clone()
    m, v = s["exp_avg"].clone(), s["exp_avg_sq"].clone()
    if bits == 8:
        m, v = (m, s["exp_avg_steps"].clone()), (v, s["exp_avg_sq_steps"].clone())
    fw.adamw_step([x], grads[3:], [m], [v], step=4, master=[want], **{**HYPER, "betas": betas})
    p.grad = grads[3]
    o.step()
    assert torch.equal(s["master"], want) and torch.equal(p.detach(), x) and torch.equal(p.detach(), want.bfloat16())


def test_a_model_loaded_between_steps(fw, cuda):
    model = torch.nn.Linear(33, 20, device=cuda, dtype=torch.bfloat16)
    o = fw.AdamW(model.parameters(), lr=1e-3)
    other = {k: torch.ones_like(v) for k, v in model.state_dict().items()}
    for i in range(2):
        for p in model.parameters():
            p.grad = torch.ones_like(p)
        o.step()
        if i == 0:
            model.load_state_dict(other)
    for p in model.parameters():
        assert bool(((p.detach().float() - 1).abs() < 0.01).all())


@pytest.mark.parametrize("bits", [8, 32])
def test_the_step_itself_takes_either(fw, cuda, bits):
    """``follow``: odd addresses and lengths, NaN and zeros of either sign in a parameter; without it the copy alone counts."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    n = 777
    wide = torch.zeros(n + 1, device=cuda, dtype=torch.bfloat16)
    p = wide[1:]
    p.copy_(torch.randn(n, device=cuda, generator=gen))
    p[5], p[6], p[7] = float("nan"), -0.0, float("inf")
    master = p.float() + 1e-5 * torch.randn(n, device=cuda, generator=gen)
    master[6] = 0.0
    master[9:12] += 1.0
    g = torch.randn(n, device=cuda, generator=gen).bfloat16()
    fresh = lambda: [codes_of(torch.ones(n, device=cuda), t) if bits == 8 else torch.ones(n, device=cuda) for t in (127, 255)]  # noqa: E731
    changed = master.bfloat16().view(torch.int16) != p.view(torch.int16)
    assert 5 <= int(changed.sum()) < n // 2
    for follow in (False, True):
        start = torch.where(changed, p.float(), master) if follow else master
        out = []
        for copy, flag in ((master.clone(), follow), (start.clone(), False)):
            x = torch.zeros(n + 1, device=cuda, dtype=torch.bfloat16)[1:].copy_(p)
            m, v = fresh()
            fw.adamw_step([x], [g], [m], [v], step=3, master=[copy], follow=flag, **HYPER)
            out.append((x, copy))
        for a, b in zip(*out):
            assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())
        assert bool(out[0][1][5].isnan()) and bool((out[0][1][9:12] > p[9:12].float() + 0.5).all()) != follow


def test_a_refused_step_does_not_count(fw, cuda):
    """A gradient that the step cannot take: an error, and nothing has happened, the count of steps included."""
    p = [torch.nn.Parameter(torch.ones(6, 4, device=cuda)) for _ in range(2)]
    o = fw.AdamW(p, lr=1e-2)
    for x in p:
        x.grad = torch.ones_like(x)
    o.step()
    p[1].grad = torch.ones(6, 4, device=cuda).to_sparse()
    before = [x.detach().clone() for x in p]
    with pytest.raises(RuntimeError):
        o.step()
    assert [o.state[x]["step"] for x in p] == [1, 1] and all(torch.equal(a, b) for a, b in zip(p, before))
    p[1].grad = torch.ones(6, 4, device=cuda)
    o.step()
    q = [torch.nn.Parameter(torch.ones(6, 4, device=cuda)) for _ in range(2)]
    o2 = fw.AdamW(q, lr=1e-2)
    for _ in range(2):
        for x in q:
            x.grad = torch.ones_like(x)
        o2.step()
    assert all(torch.equal(a, b) for a, b in zip(p, q))


def trained(fw, cuda, dtype, bits, steps=3):
    gen = torch.Generator(device="cuda").manual_seed(9)
    p = torch.nn.Parameter(torch.randn(40, 30, device=cuda, generator=gen).to(dtype))
    o = fw.AdamW([p], state_bits=bits, **HYPER)
    for _ in range(steps):
        p.grad = torch.randn(40, 30, device=cuda, generator=gen).to(dtype)
        o.step()
    return p, o


@pytest.mark.parametrize("bits", [8, 32])
def test_states_that_hooks_change_on_the_way_in(fw, cuda, bits):
    """A hook before loading that gives another dict is heard; one after loading sees the states as they will be."""
    p, o = trained(fw, cuda, torch.bfloat16, bits)
    q = torch.nn.Parameter(p.detach().clone())
    o2 = fw.AdamW([q], state_bits=bits, **HYPER)

    def later(_, given):
        return {**given, "state": {i: {**s, "step": s["step"] + 100} for i, s in given["state"].items()}}

    types = []
    o2.register_load_state_dict_pre_hook(later)
    o2.register_load_state_dict_post_hook(lambda opt: types.append({k: v.dtype for k, v in opt.state[q].items() if k != "step"}))
    o2.load_state_dict(o.state_dict())
    assert o2.state[q]["step"] == 103
    assert types == [{k: v.dtype for k, v in o.state[p].items() if k != "step"}]
    assert all(torch.equal(v, o2.state[q][k]) for k, v in o.state[p].items() if k != "step")
    o2.load_state_dict(o.state_dict())  # the call's own hooks have gone, the program's stay
    assert o2.state[q]["step"] == 103 and len(types) == 2


@pytest.mark.parametrize("bits", [8, 32])
def test_states_of_float32_parameters_for_bfloat16_ones(fw, cuda, bits):
    p, o = trained(fw, cuda, torch.float32, bits)
    q = torch.nn.Parameter(p.detach().bfloat16())
    o2 = fw.AdamW([q], state_bits=bits, **HYPER)
    o2.load_state_dict(o.state_dict())
    before = q.detach().float()
    q.grad = torch.ones_like(q)
    o2.step()
    s = o2.state[q]
    assert s["step"] == 4 and torch.equal(s["master"].bfloat16(), q.detach())
    move = (s["master"] - before).abs()
    assert bool((move > 0).any()) and bool((move <= 0.1).all())

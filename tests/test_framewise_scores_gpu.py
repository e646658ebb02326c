"""Label scores (log probabilities, entropies, best classes) and their gradient against the formulas in 64 bits: class counts
around the steps of a warp, rows shared by warps and CTAs, ties, masks, infinities and NaN, strides, refusals."""
import pytest
import torch

from framewise_util import U, close, kept

pytestmark = pytest.mark.gpu

IGNORE = -100
TYPES = [torch.float32, torch.bfloat16]
INF = float("inf")


@pytest.fixture(scope="module")
def fw():
    import i6_native_ops_b200.framewise as m

    return m


def reference(logits, labels, lens, top, grads, best=None):
    """Results and gradient of positions in 64 bits, with a bound of each; best: the order of the alternatives, by their logits without it.

    A difference to the maximum, ``spread``, is off by its rounding, that of its product with log2 e and of that constant (3U of
    itself), an exponential by 4 times 2^-22 of itself more than that; a lane adds V / 32 terms, two chains side by side, and
    rescales its sums every 32 terms by a factor with such an error: V / 16 + 128 steps of U."""
    f64 = torch.float64
    V = logits.shape[-1]
    r = torch.finfo(logits.dtype).eps / 2
    ok = kept(labels, lens, IGNORE).reshape(-1)
    z = logits.detach().reshape(-1, V)[ok].to(f64)
    t = labels.reshape(-1)[ok].long()
    n = torch.arange(len(t), device=z.device)
    m = z.amax(1, keepdim=True)
    never = m == -INF  # no class is possible
    d = torch.where(never, -INF, z - torch.where(never, 0.0, m))
    e = d.exp()
    s = e.sum(1, keepdim=True)
    logs = torch.where(never, 0.0, s.log())
    p = torch.where(never, 0.0, e / s)
    lp = torch.where(never, -INF, d - logs)
    plp = torch.where(p > 0, p * lp, 0.0)
    H = -plp.sum(1, keepdim=True)
    spread = torch.where(p > 0, -d, 0.0)
    de = (4 * spread + 16) * U
    row = (p * de).sum(1, keepdim=True) + (V / 16 + 128) * U
    M = (p * spread).sum(1, keepdim=True)
    dlp = row + 6 * U * (torch.where(lp == -INF, 0.0, d.abs() + lp.abs()) + logs.abs())
    dH = row * (1 + M) + (p * spread * (de + 4 * U)).sum(1, keepdim=True) + (V / 16 + 128) * U * M + 8 * U * (logs.abs() + M)
    order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top]
    if best is not None and top:
        order = best.reshape(-1, top)[ok].long()
    g, h, gt = (None if x is None else x.reshape(len(ok), -1)[ok].to(f64) for x in grads)
    zero = torch.zeros(len(t), 1, dtype=f64, device=z.device)
    g, h = zero if g is None else g, zero if h is None else h
    gt = torch.zeros(len(t), top, dtype=f64, device=z.device) if gt is None else gt
    hot = torch.zeros_like(z)
    hot[n, t] += g[:, 0]
    hot.scatter_add_(1, order, gt)
    total = g + gt.sum(1, keepdim=True)
    size = g.abs() + gt.abs().sum(1, keepdim=True)
    fin = torch.where(p > 0, lp, 0.0)
    dz = torch.where(never, 0.0, hot - total * p - h * p * (fin + H))
    C = size + h.abs() * (H + fin.abs())
    ddz = p * ((de + row + 8 * U) * C + h.abs() * (dH + de + row) + (top + 12) * U * C) + 2 * U * (dz.abs() + hot.abs()) + r * dz.abs()

    def back(v, fill=0.0):
        full = torch.full((len(ok),) + tuple(v.shape[1:]), fill, dtype=v.dtype, device=v.device)
        full[ok] = v
        return full.reshape(labels.shape + tuple(v.shape[1:]))

    return {
        "log_probs": (back(lp[n, t]), back(dlp[n, t])),
        "entropy": (back(H[:, 0]), back(dH[:, 0])),
        "top_log_probs": (back(lp.gather(1, order)), back(dlp.gather(1, order))),
        "top_labels": back(order, IGNORE),
        "logits": (back(dz), back(ddz)),
    }


def inputs(cuda, dtype, B, T, V, seed=0, skip=0.1, short=True, scale=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kw = dict(device=cuda, generator=gen)
    t = torch.randint(0, V, (B, T), **kw).to(torch.int32)
    t = torch.where(torch.rand(B, T, **kw) < skip, IGNORE, t).to(torch.int32)
    lens = torch.randint(0, T + 1, (B,), **kw).to(torch.int32) if short else None
    return (torch.randn(B, T, V, **kw) * scale).to(dtype), t, lens


def incoming(shape, top, seed=0, which=(True, True, True)):
    gen = torch.Generator(device="cuda").manual_seed(seed + 77)
    full = [torch.randn(s, device="cuda", generator=gen) for s in (shape, shape, tuple(shape) + (top,))]
    return [g if w else None for g, w in zip(full, which)]


def check_order(z, best, log_probs):
    """The largest logits (equal ones by their class), each once, in falling order of their log probabilities, equal ones by their class."""
    assert bool((best.sort(1).values.diff(dim=1) > 0).all())
    of, equal = z.gather(1, best), log_probs[:, :-1] == log_probs[:, 1:]
    assert bool(torch.where(equal, best[:, :-1] < best[:, 1:], of[:, :-1] > of[:, 1:]).all())
    if best.shape[1] < z.shape[1]:
        rest, at = z.scatter(1, best, -INF).max(1)
        last = of.amin(1)
        assert bool(((rest < last) | ((rest == last) & ((at > best.where(of == last[:, None], -1).amax(1)) | (rest == -INF)))).all())


def check(fw, logits, labels, lens, top, grads=None):
    grads = incoming(tuple(labels.shape), top) if grads is None else grads
    z = logits.detach().requires_grad_()
    got = fw.label_scores(z, labels, top=top, seq_lens=lens, ignore_index=IGNORE)
    want = reference(logits, labels, lens, top, grads, got.top_labels)
    pairs = [(o, g) for o, g in zip(got, grads) if g is not None]
    torch.autograd.backward([o for o, _ in pairs], [g for _, g in pairs])
    for name in ("log_probs", "entropy", "top_log_probs"):
        close(getattr(got, name).detach(), want[name], name)
    best, ok = got.top_log_probs.detach(), kept(labels, lens, IGNORE)
    assert got.top_labels.dtype == labels.dtype and bool((got.top_labels[~ok] == IGNORE).all())
    if top:
        check_order(logits.detach()[ok].float(), got.top_labels[ok].long(), best[ok])
    # falling order to the last bit; equal logits have equal log probabilities, the label's among them
    assert bool((best[..., :-1] >= best[..., 1:]).all())
    same = (got.top_labels.long() == labels[..., None]) & ok[..., None]
    assert torch.equal(best[same], got.log_probs.detach()[..., None].expand_as(best)[same])
    close(z.grad, want["logits"], "logits")
    with torch.no_grad():
        again = fw.label_scores(logits, labels, top=top, seq_lens=lens, ignore_index=IGNORE)
    for a, b in zip(again, got):
        assert torch.equal(a.nan_to_num(7.0) if a.is_floating_point() else a, b.detach().nan_to_num(7.0) if b.is_floating_point() else b)
    return got, z.grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [(1, 1, 1), (1, 1, 2), (3, 5, 7), (2, 33, 8), (1, 9, 31), (4, 10, 33), (2, 17, 255), (3, 11, 257), (5, 7, 1000),
                                   (1, 1, 4099), (8, 1, 10025), (2, 3, 12001), (1, 1, 131071), (70, 3, 2047), (40, 125, 41), (17, 300, 1025)])
def test_sizes(fw, cuda, dtype, sizes):
    B, T, V = sizes
    for top in sorted({0, 1, min(V, 5), min(V, 32)}):
        check(fw, *inputs(cuda, dtype, B, T, V, seed=sum(sizes) + top, short=top % 2 == 0), top)


@pytest.mark.parametrize("rows", [1, 37, 74, 148, 296, 592, 1184, 2368, 2369, 9000])
def test_rows_shared_by_warps_and_ctas(fw, cuda, rows):
    """Row counts where another number of warps shares a row."""
    for dtype, V in ((torch.float32, 6001), (torch.bfloat16, 3003)):
        check(fw, *inputs(cuda, dtype, 1, rows, V, seed=rows, short=False), 7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 2, 6, 7, 8, 9, 15, 16, 17, 40])
def test_rows_that_begin_anywhere(fw, cuda, dtype, V):
    """Each row begins a value later than the one before, relative to the vectors that it is read in."""
    wide = torch.randn(1, 17, 2 * V + 17, device=cuda, generator=torch.Generator(cuda).manual_seed(V)).to(dtype)
    width = V + (V + 1) % 2  # odd, so that rows begin everywhere
    z = wide.flatten()[: 17 * width].view(1, 17, width)[..., :V]
    for first in range(3):
        t = torch.arange(17, device=cuda).view(1, 17).to(torch.int32) % V
        for top in sorted({0, 1, min(V, 5)}):
            check(fw, wide.flatten()[first:][: 17 * width].view(1, 17, width)[..., :V] if first else z, t, None, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [3, 13, 300, 2051])
def test_special_values_at_the_ends_of_rows(fw, cuda, dtype, V):
    z, t, _ = inputs(cuda, dtype, 1, 40, V, seed=V, short=False, skip=0.0)
    z[0, 0::5, 0] = -INF
    z[0, 1::5, V - 1] = -INF
    z[0, 2::5, 0] = torch.finfo(dtype).min
    z[0, 3::5, V - 1] = 30.0
    z[0, 4::5, : V - 1] = -INF
    check(fw, z, t, None, 3)
    for value in (float("nan"), INF):
        for at in (0, V - 1):
            bad = z.clone()
            bad[0, 8:24, at] = value
            got, fine = fw.label_scores(bad, t, top=3), fw.label_scores(z, t, top=3)
            assert bool(got.log_probs[0, 8:24].isnan().all()) and bool(got.entropy[0, 8:24].isnan().all())
            assert bool((got.top_labels[0, 8:24, 0] == at).all())
            for a, b in zip(got, fine):
                assert torch.equal(a[0, :8], b[0, :8]) and torch.equal(a[0, 24:], b[0, 24:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [16383, 16385, 33001, 70001])
def test_long_rows_by_several_ctas(fw, cuda, dtype, V):
    for rows in (1, 5):
        for top in (0, 9, 32):
            check(fw, *inputs(cuda, dtype, 1, rows, V, seed=V + top, short=False), top)
    z, t, _ = inputs(cuda, dtype, 1, 3, V, short=False, skip=0.0)
    z[0, 0] = 0.5  # all equal: the first ones are the best
    z[0, 1] = -INF
    z[0, 1, V - 3 :] = 1.0
    got, _ = check(fw, z, t, None, 4)
    assert got.top_labels[0, 0].tolist() == [0, 1, 2, 3] and got.top_labels[0, 1].tolist() == [V - 3, V - 2, V - 1, 0]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(3, 5000), (5000, 700)])
@pytest.mark.parametrize("order", ["equal", "few", "rising", "falling", "lowest", "zeros"])
def test_equal_and_ordered_logits(fw, cuda, dtype, rows, V, order):
    z, t, _ = inputs(cuda, dtype, 1, rows, V, short=False, skip=0.0)
    ramp = torch.arange(V, device=cuda)
    if order == "equal":
        z.fill_(1.25)
    elif order == "few":
        z = (z.float() / 3).round().to(dtype)
    elif order == "rising":
        z = (ramp.float() * (8.0 / V) - 4).to(dtype).expand(1, rows, V).contiguous()
    elif order == "falling":
        z = (4 - ramp.float() * (8.0 / V)).to(dtype).expand(1, rows, V).contiguous()
    elif order == "lowest":
        z.fill_(torch.finfo(dtype).min)
    else:
        z = torch.where(ramp % 3 == 0, -0.0, 0.0).to(dtype).expand(1, rows, V).contiguous()
    for top in (1, 9, 32):
        check(fw, z, t, None, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(4, 3001), (5000, 97)])
def test_masked_classes(fw, cuda, dtype, rows, V):
    z, t, _ = inputs(cuda, dtype, 1, rows, V, short=False, skip=0.0)
    z[0, :, ::2] = -INF  # every other class, labels among them
    z[0, 0] = -INF  # a row without a class
    z[0, 1] = -INF
    z[0, 1, V - 1] = -3.0  # one class
    z[0, 2] = -INF
    z[0, 2, 5:9] = torch.finfo(dtype).min
    for top in (0, 3, 32):
        grads = incoming((1, rows), top)
        # a class of -inf that is a label has no gradient of its own but the label's: as the formula has it
        got, dz = check(fw, z, t, None, top, grads)
        assert bool((got.log_probs[0, 0] == -INF) & (got.entropy[0, 0] == 0)) and not dz[0, 0].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_and_infinity_stay_in_their_rows(fw, cuda, dtype):
    z, t, _ = inputs(cuda, dtype, 1, 5000, 300, short=False, skip=0.0)
    z[0, 3, 17] = float("nan")
    z[0, 4, 200] = INF
    z[0, 5] = float("nan")
    good = torch.ones(5000, dtype=torch.bool, device=cuda)
    good[3:6] = False
    zz = z.detach().requires_grad_()
    got = fw.label_scores(zz, t, top=4)
    sum(x.sum() for x in got[:3]).backward()
    want = reference(z[:, good], t[:, good], None, 4, [torch.ones(1, 4997, device=cuda), torch.ones(1, 4997, device=cuda), torch.ones(1, 4997, 4, device=cuda)])
    for name in ("log_probs", "entropy", "top_log_probs"):
        close(getattr(got, name).detach()[:, good], want[name], name)
        assert bool(getattr(got, name)[:, ~good].isnan().all())
    close(zz.grad[:, good], want["logits"])
    assert bool(zz.grad[:, ~good].isnan().all())
    assert got.top_labels[0, 3, 0] == 17 and got.top_labels[0, 4, 0] == 200 and got.top_labels[0, 5].tolist() == [0, 1, 2, 3]


def test_equal_log_probabilities_go_by_class(fw, cuda):
    """Logits a rounding apart, far below the row's largest: what is left of them after it is taken off is equal."""
    z = torch.full((64, 500), -3.0, device=cuda)
    z[:, 400] = 18.0
    z[:, 7] = 5.0
    z[:, 300] = torch.nextafter(torch.tensor(5.0), torch.tensor(6.0)).to(cuda)  # 5 - 18 and this - 18 round alike: ulps of 2^-21, 2^-20
    z[:, 450] = 4.0
    t = torch.zeros(64, dtype=torch.int64, device=cuda)
    assert z[0, 7] != z[0, 300] and z[0, 7] - 18 == z[0, 300] - 18
    for top, want in ((2, [400, 300]), (3, [400, 7, 300]), (4, [400, 7, 300, 450]), (32, [400, 7, 300, 450, 0, 1, 2, 3, 4, 5, 6] + list(range(8, 29)))):
        got = fw.label_scores(z, t, top=top)
        assert bool((got.top_labels == torch.tensor(want, device=cuda)).all())
        assert bool((got.top_log_probs[:, 1] == got.top_log_probs[:, 2]).all()) if top > 2 else True


def test_nothing_is_read_of_positions_that_do_not_count(fw, cuda):
    z, t, lens = inputs(cuda, torch.float32, 6, 30, 500, seed=5, skip=0.3)
    ok = kept(t, lens, IGNORE)
    want = fw.label_scores(z, t, top=3, seq_lens=lens)
    z[~ok] = float("nan")
    zz = z.requires_grad_()
    got = fw.label_scores(zz, t, top=3, seq_lens=lens)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    g = incoming((6, 30), 3)
    for x in g:
        x[~ok] = float("nan")
    torch.autograd.backward(got[:3], g)
    assert not zz.grad[~ok].any() and bool(zz.grad.isfinite().all())
    mask = (torch.arange(30, device=cuda)[:, None] < lens[None, :]).to(torch.uint8)
    for a, b in zip(fw.label_scores(z.detach(), t, top=3, seq_lens=mask), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_offsets(fw, cuda, dtype):
    B, T, V = 3, 21, 1003
    z, t, lens = inputs(cuda, dtype, B, T, V + 9, seed=3)
    for cut in (0, 1, 2, 3, 5, 8):  # rows that begin anywhere
        check(fw, z[..., cut : cut + V].contiguous(), t.clamp(max=V - 1), lens, 4)
        check(fw, z[..., cut : cut + V], t.clamp(max=V - 1), lens, 4)
    time_major = z[..., :V].transpose(0, 1).contiguous().transpose(0, 1)
    check(fw, time_major, t.clamp(max=V - 1), lens, 4)
    check(fw, z[..., :V].transpose(1, 2).contiguous().transpose(1, 2), t.clamp(max=V - 1), lens, 4)
    check(fw, z[:1, :, :V].expand(B, T, V), t.clamp(max=V - 1), lens, 4)
    check(fw, z[..., :1], t.clamp(max=0), lens, 1)


def test_flat_and_wide_labels(fw, cuda):
    z, t, _ = inputs(cuda, torch.float32, 1, 40, 77, short=False)
    check(fw, z[0], t[0], None, 2)
    check(fw, z, t.long(), None, 2)
    for a, b in zip(fw.label_scores(z[0], t[0], top=2), fw.label_scores(z, t, top=2)):
        assert torch.equal(a, b[0])


@pytest.mark.parametrize("which", [(True, False, False), (False, True, False), (False, False, True), (True, False, True)])
def test_gradients_of_some_results(fw, cuda, which):
    for dtype in TYPES:
        z, t, lens = inputs(cuda, dtype, 4, 50, 611, seed=9)
        check(fw, z, t, lens, 6, incoming((4, 50), 6, which=which))


def test_broadcast_gradients(fw, cuda):
    z, t, lens = inputs(cuda, torch.float32, 4, 50, 611, seed=11)
    one = torch.tensor(0.37, device=cuda)
    grads = [one.expand(4, 50), one.expand(50).expand(4, 50), torch.randn(6, device=cuda).expand(4, 50, 6)]
    check(fw, z, t, lens, 6, grads)


def test_gradient_against_differences(fw, cuda):
    """Central differences of torch's own 64-bit functions: off by h^2 / 6 of a third derivative (at most some 40 here: cumulants
    of directions of 1 and logits of 6) and by 2^-52 * 20 / h, together below 1e-6 at h = 2^-12."""
    z, t, _ = inputs(cuda, torch.float32, 1, 6, 40, short=False, skip=0.0, scale=1.5)
    top = 3
    g = incoming((1, 6), top)
    zz = z.detach().requires_grad_()
    got = fw.label_scores(zz, t, top=top)
    torch.autograd.backward(got[:3], g)

    def f(x):
        lp = torch.log_softmax(x, -1)
        return ((lp.gather(-1, t.long()[..., None])[..., 0] * g[0]) + torch.special.entr(lp.exp()).sum(-1) * g[1]
                + (lp.gather(-1, got.top_labels.long()) * g[2]).sum(-1)).sum()

    gen = torch.Generator(device="cuda").manual_seed(0)
    h = 2.0**-12
    for _ in range(20):
        v = torch.randint(0, 2, z.shape, device=cuda, generator=gen).double() * 2 - 1
        slope = (f(z.double() + h * v) - f(z.double() - h * v)) / (2 * h)
        bound = 6e-6 * 6 + (reference(z, t, None, top, g)["logits"][1].sum())  # six rows; the gradient's own bound
        assert abs(float((zz.grad.double() * v).sum() - slope)) < float(bound)


def test_labels_outside_the_vocabulary(fw, cuda):
    z, t, _ = inputs(cuda, torch.float32, 1, 20, 50, short=False, skip=0.0)
    t[0, 3], t[0, 7] = 50, -1
    zz = z.requires_grad_()
    got = fw.label_scores(zz, t, top=2)
    bad = torch.zeros(20, dtype=torch.bool, device=cuda)
    bad[3] = bad[7] = True
    assert bool(got.log_probs[0].isnan().eq(bad).all()) and bool(got.entropy.isfinite().all()) and bool(got.top_log_probs.isfinite().all())
    got.log_probs.sum().backward()
    assert bool(zz.grad[0].isnan().all(1).eq(bad).all()) and bool(zz.grad[0].isnan().any(1).eq(bad).all())


def test_empty(fw, cuda):
    for B, T in ((0, 5), (3, 0)):
        z = torch.zeros(B, T, 9, device=cuda, requires_grad=True)
        got = fw.label_scores(z, torch.zeros(B, T, dtype=torch.int32, device=cuda), top=2)
        assert got.log_probs.shape == (B, T) and got.top_labels.shape == (B, T, 2)
        (got.log_probs.sum() + got.entropy.sum()).backward()
        assert z.grad.shape == z.shape


def test_other_streams_and_graphs(fw, cuda):
    z, t, lens = inputs(cuda, torch.bfloat16, 5, 60, 900, seed=21)
    g = incoming((5, 60), 4)
    want, grad = check(fw, z, t, lens, 4, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    zz = z.detach().requires_grad_()
    with torch.cuda.stream(side):
        for _ in range(2):
            got = fw.label_scores(zz, t, top=4, seq_lens=lens)
            (dz,) = torch.autograd.grad(got[:3], zz, g)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(dz, grad)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = fw.label_scores(zz, t, top=4, seq_lens=lens)
        (dz,) = torch.autograd.grad(got[:3], zz, g)
    with torch.no_grad():
        other = torch.randn_like(z)
        kept_z = z.clone()
        zz.copy_(other)
    graph.replay()
    eager, eager_grad = check(fw, other, t, lens, 4, g)
    for a, b in zip(got, eager):
        assert torch.equal(a.detach(), b.detach())
    assert torch.equal(dz, eager_grad)
    with torch.no_grad():
        zz.copy_(kept_z)
    graph.replay()
    assert torch.equal(dz, grad) and torch.equal(got.top_labels, want.top_labels)


def test_refusals(fw, cuda):
    z, t, lens = inputs(cuda, torch.float32, 2, 5, 20)
    bad = [
        (lambda: fw.label_scores(z.half(), t), "float32 or bfloat16"),
        (lambda: fw.label_scores(z.cpu(), t), "CUDA"),
        (lambda: fw.label_scores(z, t.cpu()), "device"),
        (lambda: fw.label_scores(z, t.float()), "int32 or int64"),
        (lambda: fw.label_scores(z, t[:, :4]), "shape"),
        (lambda: fw.label_scores(z[0], t), "one dimension more"),
        (lambda: fw.label_scores(z, t, top=33), "top"),
        (lambda: fw.label_scores(z[..., :3], t, top=4), "top"),
        (lambda: fw.label_scores(z, t, top=-1), "top"),
        (lambda: fw.label_scores(z[..., :0], t), "classes"),
        (lambda: fw.label_scores(z, t, seq_lens=lens[:1]), "seq_lens"),
        (lambda: fw.label_scores(z, t, seq_lens=lens.long()), "int32"),
        (lambda: fw.label_scores(z[0], t[0], seq_lens=lens), "seq_lens"),
    ]
    for f, what in bad:
        with pytest.raises(RuntimeError, match=what):
            f()
    zz = z.requires_grad_()
    got = fw.label_scores(zz, t, top=1)
    with torch.no_grad():
        zz.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        got.log_probs.sum().backward()
    got = fw.label_scores(zz, t, top=1)
    with pytest.raises(RuntimeError, match="no gradients of these gradients"):
        torch.autograd.grad(got.log_probs.sum(), zz, create_graph=True)
    import torch.autograd.forward_ad as fa

    with fa.dual_level():
        dual = fa.make_dual(z.detach(), torch.ones_like(z))
        with pytest.raises(RuntimeError, match="forward-mode"):
            fw.label_scores(dual, t)


def test_offsets_past_32_bits(fw, cuda):
    """More than 2^31 logits, of which a few rows count: first and last ones."""
    V, N = 12001, 180000
    z = torch.zeros(1, N, V, device=cuda, dtype=torch.bfloat16)
    t = torch.full((1, N), IGNORE, device=cuda, dtype=torch.int32)
    at = torch.tensor([0, 1, N // 2, N - 2, N - 1], device=cuda)
    gen = torch.Generator(device="cuda").manual_seed(1)
    z[0, at] = (torch.randn(5, V, device=cuda, generator=gen) * 3).bfloat16()
    t[0, at] = torch.randint(0, V, (5,), device=cuda, generator=gen, dtype=torch.int32)
    zz = z.requires_grad_()
    got = fw.label_scores(zz, t, top=3)
    torch.autograd.backward([got.log_probs, got.entropy], [torch.ones(1, N, device=cuda), torch.ones(1, N, device=cuda)])
    g = [torch.ones(1, 5, device=cuda), torch.ones(1, 5, device=cuda), None]
    want = reference(z.detach()[:, at], t[:, at], None, 3, g)
    for name in ("log_probs", "entropy", "top_log_probs"):
        close(getattr(got, name).detach()[:, at], want[name], name)
    assert torch.equal(got.top_labels[:, at].long(), want["top_labels"])
    close(zz.grad[:, at], want["logits"], "logits")
    zz.grad[:, at] = 0
    assert float(zz.grad.abs().amax()) == 0.0

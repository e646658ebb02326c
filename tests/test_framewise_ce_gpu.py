"""Output layer with softmax cross entropy against its formula in 64 bits: losses and gradients, both types, sizes
around the tiles' borders, masks, strides, values at positions that do not count, refusals."""
import pytest
import torch

from framewise_util import ce_reference, close

pytestmark = pytest.mark.gpu

IGNORE = -100
TYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def fw():
    import i6_native_ops_b200.framewise as m

    return m


def inputs(cuda, dtype, B, T, V, D, seed=0, bias=True, short=True, skip=0.1, spread=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kw = dict(device=cuda, generator=gen)
    w = (torch.randn(V, D, **kw) * spread / D**0.5).to(dtype)
    h = torch.randn(B, T, D, **kw).to(dtype)
    b = torch.randn(V, **kw).to(dtype) if bias else None
    t = torch.randint(0, V, (B, T), **kw).to(torch.int32)
    t = torch.where(torch.rand(B, T, **kw) < skip, IGNORE, t).to(torch.int32)
    lens = torch.randint(0, T + 1, (B,), **kw).to(torch.int32) if short else None
    g = torch.randn(B, T, **kw)
    return h, w, b, t, lens, g


def run(fw, h, w, b, t, lens, g):
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    b = None if b is None else b.detach().requires_grad_()
    loss = fw.linear_cross_entropy(h, w, t, bias=b, seq_lens=lens, ignore_index=IGNORE)
    loss.backward(g)
    got = {"loss": loss.detach(), "hidden": h.grad, "weight": w.grad}
    if b is not None:
        got["bias"] = b.grad
    return got


def check(fw, h, w, b, t, lens, g):
    want = ce_reference(h, w, b, t, lens, IGNORE, g)
    got = run(fw, h, w, b, t, lens, g)
    for n, v in got.items():
        close(v, want[n], n)
    with torch.no_grad():
        loss = fw.linear_cross_entropy(h, w, t, bias=b, seq_lens=lens, ignore_index=IGNORE)
    close(loss, want["loss"], "loss alone")
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [(1, 1, 1, 1), (1, 1, 2, 3), (3, 7, 41, 64), (2, 33, 63, 40), (1, 128, 64, 64), (1, 129, 65, 65),
                                   (2, 128, 256, 128), (5, 53, 257, 100), (2, 200, 511, 192), (3, 171, 1000, 257), (4, 64, 2050, 520)])
def test_sizes(fw, cuda, dtype, sizes):
    B, T, V, D = sizes
    for bias, short in ((True, True), (False, False)):
        check(fw, *inputs(cuda, dtype, B, T, V, D, seed=B + T + V + D, bias=bias, short=short))


@pytest.mark.parametrize("dtype", TYPES)
def test_one_position_and_a_large_vocabulary(fw, cuda, dtype):
    check(fw, *inputs(cuda, dtype, 1, 1, 30011, 96, short=False, skip=0.0))
    check(fw, *inputs(cuda, dtype, 16, 1, 10025, 512, short=False, skip=0.0))


@pytest.mark.parametrize("dtype,rows", [(torch.float32, 11500), (torch.bfloat16, 34000)])
def test_more_rows_than_a_chunk_holds(fw, cuda, dtype, rows):
    """q of 12001 classes is held for some ten thousand rows at a time."""
    check(fw, *inputs(cuda, dtype, 10, rows // 10, 12001, 24, skip=0.02, short=False))


@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_counts(fw, cuda, dtype):
    h, w, b, t, lens, g = inputs(cuda, dtype, 3, 40, 300, 72)
    for t_, lens_ in ((torch.full_like(t, IGNORE), None), (t, torch.zeros_like(lens)), (t[:, :0], None), (t[:0], None)):
        h_, g_ = h[: t_.shape[0], : t_.shape[1]], g[: t_.shape[0], : t_.shape[1]]
        got = run(fw, h_, w, b, t_, lens_, g_)
        assert got["loss"].shape == t_.shape and got["hidden"].shape == h_.shape
        for n, v in got.items():
            assert bool((v == 0).all()), n


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf"), "lowest"])
def test_values_at_positions_that_do_not_count(fw, cuda, dtype, junk):
    h, w, b, t, lens, g = inputs(cuda, dtype, 5, 90, 400, 136, skip=0.3)
    want = run(fw, h, w, b, t, lens, g)
    off = (t == IGNORE) | (torch.arange(t.shape[1], device=cuda) >= lens[:, None])
    fill = torch.finfo(dtype).min if junk == "lowest" else junk
    h2 = torch.where(off[..., None], torch.full_like(h, fill), h)
    g2 = torch.where(off, torch.full_like(g, float("nan")), g)
    t2 = torch.where(torch.arange(t.shape[1], device=cuda) >= lens[:, None], 12345678, t).to(torch.int32)
    got = run(fw, h2, w, b, t2, lens, g2)
    for n in want:
        assert torch.equal(got[n], want[n]), n
        assert bool(got[n].isfinite().all())


@pytest.mark.parametrize("dtype", TYPES)
def test_classes_without_probability(fw, cuda, dtype):
    """Biases of -inf and of the type's lowest value: probability 0, and no NaN, whole tiles of them among it."""
    h, w, b, t, lens, g = inputs(cuda, dtype, 3, 60, 1100, 80)
    for fill in (-float("inf"), torch.finfo(dtype).min):
        b2 = b.clone()
        b2[256:900] = fill
        b2[3::7] = fill
        alive = torch.nonzero(b2 > -1e30).reshape(-1)
        t2 = torch.where(t == IGNORE, t, alive[t.long().clamp(min=0) % len(alive)].to(torch.int32))
        got = check(fw, h, w, b2, t2, lens, g)
        assert bool((got["weight"][b2 < -1e30] == 0).all())
    # a label without probability: an infinite loss, finite gradients
    dead = torch.full_like(t, 300)
    b2 = b.clone()
    b2[300] = -float("inf")
    got = run(fw, h, w, b2, dead, None, g)
    assert bool((got["loss"] == float("inf")).all())
    assert all(bool(got[n].isfinite().all()) for n in ("hidden", "weight", "bias"))


@pytest.mark.parametrize("dtype", TYPES)
def test_large_logits(fw, cuda, dtype):
    """Logits of some thousands: the maximum is taken off before every exponential."""
    h, w, b, t, lens, g = inputs(cuda, dtype, 2, 70, 500, 64, spread=300.0)
    got = check(fw, h, w, b, t, lens, g)
    assert all(bool(v.isfinite().all()) for v in got.values())


@pytest.mark.parametrize("dtype", TYPES)
def test_labels_outside_the_vocabulary(fw, cuda, dtype):
    h, w, b, t, lens, g = inputs(cuda, dtype, 2, 140, 300, 64, skip=0.0, short=False)
    for wrong in (300, -1, 2**31 - 1, -(2**31)):
        t2 = t.clone()
        t2[1, 5] = wrong
        got = run(fw, h, w, b, t2, lens, g)
        nan = got["loss"].isnan()
        assert int(nan.sum()) == 1 and bool(nan[1, 5])
        assert bool(got["hidden"][1, 5].isnan().all()) and int(got["hidden"].isnan().any(-1).sum()) == 1
        assert bool(got["weight"].isnan().all()) and bool(got["bias"].isnan().all())
    t3 = t.long()
    t3[0, 3] = 2**40 + 7
    assert bool(run(fw, h, w, b, t3, lens, g)["loss"][0, 3].isnan())


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_types_and_masks_of_the_arguments(fw, cuda, dtype):
    h, w, b, t, lens, g = inputs(cuda, dtype, 6, 50, 333, 88)
    want = run(fw, h, w, b, t, lens, g)

    def same(*a):
        got = run(fw, *a)
        for n in want:
            assert torch.equal(got[n], want[n]), n

    same(h.transpose(0, 1).contiguous().transpose(0, 1), w, b, t, lens, g)  # an encoder's (T, B, D)
    same(h.transpose(1, 2).contiguous().transpose(1, 2), w, b, t, lens, g)  # last dimension not dense
    wide = torch.zeros(6, 50, 100, dtype=dtype, device=cuda)
    wide[..., 5:93] = h
    same(wide[..., 5:93], w, b, t, lens, g)  # rows at odd addresses
    off = torch.zeros(w.numel() + 1, dtype=dtype, device=cuda)
    off[1:] = w.reshape(-1)
    same(h, off[1:].reshape(w.shape), b, t, lens, g)  # a weight at an odd address
    same(h, w.T.contiguous().T, b, t, lens, g)
    same(h, w, torch.stack([b, b], 1)[:, 0], t, lens, g)
    same(h, w, b, t.long(), lens, g)
    same(h, w, b, t.T.contiguous().T, lens, g.T.contiguous().T)
    same(torch._neg_view(-h), w, b, t, lens, g)
    same(h, w, b, t, (torch.arange(50, device=cuda)[:, None] < lens[None]).float(), g)  # (T, B) index mask
    # gradients that one value was broadcast to
    a = run(fw, h, w, b, t, lens, torch.full_like(g, 0.5))
    c = run(fw, h, w, b, t, lens, torch.tensor(0.5, device=cuda).expand(6, 50))
    for n in a:
        assert torch.equal(a[n], c[n]), n
    # (N, D) activations are a batch of one
    flat = run(fw, h.reshape(-1, 88), w, b, t.reshape(-1), None, g.reshape(-1))
    batch = run(fw, h, w, b, t, None, g)
    for n in flat:
        assert torch.equal(flat[n].reshape(batch[n].shape), batch[n]), n


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_calls_give_equal_bits(fw, cuda, dtype):
    a = inputs(cuda, dtype, 8, 300, 3000, 200)
    first = run(fw, *a)
    for _ in range(3):
        again = run(fw, *a)
        for n in first:
            assert torch.equal(first[n], again[n]), n


def test_padding_changes_nothing(fw, cuda):
    """Positions past the lengths are as if they were not there."""
    h, w, b, t, lens, g = inputs(cuda, torch.float32, 4, 60, 500, 72)
    lens = lens.clamp(max=37)
    a = run(fw, h, w, b, t, lens, g)
    c = run(fw, h[:, :40], w, b, t[:, :40], lens, g[:, :40])
    assert torch.equal(a["loss"][:, :40], c["loss"]) and torch.equal(a["hidden"][:, :40], c["hidden"])
    close(a["weight"], (c["weight"].double(), 2.0**-18 * c["weight"].abs().double() + 1e-6), "weight")


def test_gradients_against_differences(fw, cuda):
    """Directional derivatives by central differences.  f = sum g loss; with |d| = 1 and step e the differences are off
    by e^2 / 6 f''' (below e^2 |w|^3 here) and by the losses' rounding, 2^-20 of each, over e."""
    h, w, b, t, lens, g = inputs(cuda, torch.float32, 3, 20, 90, 48)
    got = run(fw, h, w, b, t, lens, g)
    gen = torch.Generator(device="cuda").manual_seed(1)
    e = 2.0**-4
    for n, x in (("hidden", h), ("weight", w), ("bias", b)):
        for _ in range(4):
            d = torch.randn(x.shape, device=cuda, generator=gen)
            d /= d.norm()
            f = []
            for s in (e, -e):
                y = {"hidden": h, "weight": w, "bias": b}
                y[n] = x + s * d
                loss = fw.linear_cross_entropy(y["hidden"], y["weight"], t, bias=y["bias"], seq_lens=lens, ignore_index=IGNORE)
                f.append(float((loss.double() * g.double()).sum()))
            slope = (f[0] - f[1]) / (2 * e)
            want = float((got[n].double() * d.double()).sum())
            rounding = float((got["loss"].abs() * g.abs()).sum()) * 2.0**-20 / e
            assert abs(slope - want) <= rounding + e * e * (1 + float(w.norm(dim=1).max()) ** 3 * float(g.norm())), n


def test_parts_of_the_gradient(fw, cuda):
    h, w, b, t, lens, g = inputs(cuda, torch.bfloat16, 3, 50, 200, 64)
    want = run(fw, h, w, b, t, lens, g)
    for need in (("hidden",), ("weight",), ("bias",), ("hidden", "bias")):
        x = {"hidden": h.clone(), "weight": w.clone(), "bias": b.clone()}
        for n in need:
            x[n].requires_grad_()
        loss = fw.linear_cross_entropy(x["hidden"], x["weight"], t, bias=x["bias"], seq_lens=lens, ignore_index=IGNORE)
        loss.backward(g)
        for n in need:
            assert torch.equal(x[n].grad, want[n]), (need, n)


def test_another_stream_and_a_graph(fw, cuda):
    h, w, b, t, lens, g = inputs(cuda, torch.bfloat16, 4, 100, 700, 128)
    want = run(fw, h, w, b, t, lens, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(fw, h, w, b, t, lens, g)
    torch.cuda.current_stream().wait_stream(side)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    graph = torch.cuda.CUDAGraph()
    h2 = h.clone()
    with torch.no_grad():
        with torch.cuda.graph(graph):
            loss = fw.linear_cross_entropy(h2, w, t, bias=b, seq_lens=lens, ignore_index=IGNORE)
        h2.mul_(0.5)
        graph.replay()
        assert torch.equal(loss, fw.linear_cross_entropy(h * 0.5, w, t, bias=b, seq_lens=lens, ignore_index=IGNORE))


def test_a_training_step_in_a_graph(fw, cuda):
    h, w, b, t, lens, g = inputs(cuda, torch.bfloat16, 4, 100, 700, 128)
    x = [v.clone().requires_grad_() for v in (h, w, b)]

    def step():
        loss = fw.linear_cross_entropy(x[0], x[1], t, bias=x[2], seq_lens=lens, ignore_index=IGNORE)
        return [loss.detach(), *torch.autograd.grad(loss, x, g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x[0].mul_(0.5)
    graph.replay()
    want = run(fw, h * 0.5, w, b, t, lens, g)
    for a, c in zip(out, (want["loss"], want["hidden"], want["weight"], want["bias"])):
        assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", TYPES)
def test_one_large_row_leaves_the_others_alone(fw, cuda, dtype):
    """Rows meet only in the sums over rows: one with values of 1e20 changes nothing of the others' losses and gradients."""
    h, w, b, t, lens, g = inputs(cuda, dtype, 2, 90, 300, 80, skip=0.0, short=False)
    want = run(fw, h, w, b, t, lens, g)
    h2 = h.clone()
    h2[1, 40] *= 1e20
    got = run(fw, h2, w, b, t, lens, g)
    keep = torch.ones_like(t, dtype=torch.bool)
    keep[1, 40] = False
    assert torch.equal(got["loss"][keep], want["loss"][keep]) and torch.equal(got["hidden"][keep], want["hidden"][keep])


def test_large_offsets(fw, cuda):
    """Activations whose positions lie past 2^31 elements: rows of a buffer of 5 GB."""
    big = torch.empty(2, 5, 2**28, dtype=torch.bfloat16, device=cuda)[..., :64]
    h, w, b, t, lens, g = inputs(cuda, torch.bfloat16, 2, 5, 100, 64, short=False, skip=0.0)
    big.copy_(h)
    assert big.stride(0) * 1 + big.stride(1) * 4 > 2**31
    want, got = run(fw, h, w, b, t, None, g), run(fw, big, w, b, t, None, g)
    for n in want:
        assert torch.equal(got[n], want[n]), n


def test_refusals(fw, cuda):
    h, w, b, t, lens, g = inputs(cuda, torch.float32, 2, 5, 11, 8)
    f = fw.linear_cross_entropy
    bad = [
        (h.double(), w.double(), t, {}), (h.half(), w.half(), t, {}), (h, w.bfloat16(), t, {}), (h.cpu(), w, t, {}), (h, w.cpu(), t, {}),
        (h, w, t.cpu(), {}), (h, w, t.float(), {}), (h, w[:, :7], t, {}), (h[0], w, t, {}), (h, w, t[:, :4], {}), (h, w, t[0], {}),
        (h, w[0], t, {}), (h, w[:0], t, {}), (h[..., :0], w[:, :0], t, {}), (h, w, t, dict(bias=b[:-1])), (h, w, t, dict(bias=b.cpu())),
        (h, w, t, dict(bias=b.bfloat16())), (h, w, t, dict(seq_lens=lens.long())), (h, w, t, dict(seq_lens=lens[:1])),
        (h, w, t, dict(seq_lens=lens.cpu())), (h.reshape(-1, 8), w, t.reshape(-1), dict(seq_lens=lens)),
        (h, w, t, dict(seq_lens=torch.ones(4, 2, device=cuda))),
    ]
    for x, y, z, kw in bad:
        with pytest.raises(RuntimeError):
            f(x, y, z, **kw)
    # the weight must be what it was
    w2 = w.clone().requires_grad_()
    w3 = w2 * 1.0
    loss = f(h, w3, t, bias=b, seq_lens=lens)
    w3.data_ptr()
    with torch.no_grad():
        w3.add_(1.0)
    with pytest.raises(RuntimeError):
        loss.backward(g)
    # and there are no second derivatives
    h2 = h.clone().requires_grad_()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(f(h2, w, t).sum(), h2, create_graph=True)

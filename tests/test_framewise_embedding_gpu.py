"""Label embedding and its gradient against their formulas in 64 bits: label counts around the sort's borders, labels
that all positions share, masks, strides, refusals."""
import pytest
import torch

from framewise_util import U, close, kept

pytestmark = pytest.mark.gpu

IGNORE = -100
TYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def fw():
    import i6_native_ops_b200.framewise as m

    return m


def reference(labels, weight, lens, scale, g):
    f64 = torch.float64
    r = torch.finfo(weight.dtype).eps / 2
    scale = float(torch.tensor(scale, dtype=torch.float32))
    ok = kept(labels, lens, IGNORE)
    t = labels.long()[ok]
    out = torch.zeros(labels.shape + (weight.shape[1],), dtype=f64, device=weight.device)
    out[ok] = weight.detach().to(f64)[t] * scale
    dw = torch.zeros(weight.shape, dtype=f64, device=weight.device)
    mag = torch.zeros_like(dw)
    gg = g.to(f64)[ok] * scale
    dw.index_add_(0, t, gg)
    mag.index_add_(0, t, gg.abs())
    most = int(torch.bincount(t).max()) if len(t) else 0
    return (out, (r + U) * out.abs()), (dw, (most + 2) * 2 * U * mag + r * dw.abs())


def run(fw, labels, weight, lens, scale, g):
    w = weight.detach().requires_grad_()
    out = fw.label_embedding(labels, w, scale=scale, seq_lens=lens, ignore_index=IGNORE)
    out.backward(g)
    return out.detach(), w.grad


def inputs(cuda, dtype, B, T, V, D, seed=0, skip=0.1, short=True, few=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kw = dict(device=cuda, generator=gen)
    t = torch.randint(0, few or V, (B, T), **kw).to(torch.int32)
    t = torch.where(torch.rand(B, T, **kw) < skip, IGNORE, t).to(torch.int32)
    lens = torch.randint(0, T + 1, (B,), **kw).to(torch.int32) if short else None
    return t, torch.randn(V, D, **kw).to(dtype), lens, 1.7, torch.randn(B, T, D, **kw).to(dtype)


def check(fw, t, w, lens, scale, g):
    out, dw = reference(t, w, lens, scale, g)
    got = run(fw, t, w, lens, scale, g)
    close(got[0], out, "out")
    close(got[1], dw, "weight")
    with torch.no_grad():
        assert torch.equal(fw.label_embedding(t, w, scale=scale, seq_lens=lens, ignore_index=IGNORE), got[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [(1, 1, 1, 1), (1, 1, 5, 8), (3, 33, 41, 64), (2, 31, 7, 40), (1, 1025, 300, 72), (7, 300, 121, 256),
                                   (4, 500, 1000, 257), (9, 111, 2000, 513), (2, 700, 50, 1030)])
def test_sizes(fw, cuda, dtype, sizes):
    for short in (True, False):
        check(fw, *inputs(cuda, dtype, *sizes, seed=sum(sizes), short=short))


@pytest.mark.parametrize("V", [16382, 16383, 16384, 16385, 40000, 70001])
def test_label_counts_around_the_digits_of_the_sort(fw, cuda, V):
    t, w, lens, scale, g = inputs(cuda, torch.float32, 3, 900, V, 16, seed=V)
    t[0, :4] = torch.tensor([V - 1, 0, V - 1, V - 2], dtype=torch.int32)
    check(fw, t, w, lens, scale, g)


@pytest.mark.parametrize("V", [1, 3, 121, 12001, 16383])
def test_more_positions_than_one_pass_sorts(fw, cuda, V):
    check(fw, *inputs(cuda, torch.float32, 600, 1000, V, 4, seed=V))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("few", [1, 2, 5])
def test_labels_that_many_positions_share(fw, cuda, dtype, few):
    check(fw, *inputs(cuda, dtype, 20, 600, 30, 100, few=few))
    check(fw, *inputs(cuda, dtype, 1, 64, 30, 100, few=few, skip=0.0, short=False))


@pytest.mark.parametrize("dtype", TYPES)
def test_positions_that_do_not_count(fw, cuda, dtype):
    t, w, lens, scale, g = inputs(cuda, dtype, 5, 77, 60, 48, skip=0.4)
    off = ~kept(t, lens, IGNORE)
    want = run(fw, t, w, lens, scale, g)
    late = torch.arange(77, device=cuda) >= lens[:, None]
    t2 = torch.where(late, 2**30, t).to(torch.int32)
    got = run(fw, t2, w, lens, scale, torch.where(off[..., None], torch.full_like(g, float("nan")), g))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and bool((got[0][off] == 0).all())
    for t3, l3 in ((torch.full_like(t, IGNORE), None), (t, torch.zeros_like(lens)), (t[:, :0], None), (t[:0], None)):
        out, dw = run(fw, t3, w, l3, scale, g[: t3.shape[0], : t3.shape[1]])
        assert out.shape == t3.shape + (48,) and bool((out == 0).all()) and bool((dw == 0).all())


def test_labels_outside_the_vocabulary(fw, cuda):
    t, w, lens, scale, g = inputs(cuda, torch.float32, 2, 50, 30, 16, skip=0.0, short=False)
    for wrong in (30, -1, 2**31 - 1):
        t2 = t.clone()
        t2[0, 7] = wrong
        out, dw = run(fw, t2, w, None, scale, g)
        assert bool(out[0, 7].isnan().all()) and int(out.isnan().any(-1).sum()) == 1 and bool(dw.isnan().all())


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_types_of_the_arguments(fw, cuda, dtype):
    t, w, lens, scale, g = inputs(cuda, dtype, 4, 60, 90, 40)
    want = run(fw, t, w, lens, scale, g)

    def same(*a):
        got = run(fw, *a)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

    same(t.long(), w, lens, scale, g)
    same(t.T.contiguous().T, w, lens, scale, g.transpose(0, 1).contiguous().transpose(0, 1))
    same(t, w, lens, scale, g.transpose(1, 2).contiguous().transpose(1, 2))
    same(t, w.T.contiguous().T, lens, scale, g)
    off = torch.zeros(w.numel() + 1, dtype=dtype, device=cuda)
    off[1:] = w.reshape(-1)
    wide = torch.zeros(4, 60, 43, dtype=dtype, device=cuda)
    wide[..., 1:41] = g
    same(t, off[1:].reshape(w.shape), lens, scale, wide[..., 1:41])
    same(t, w, (torch.arange(60, device=cuda)[:, None] < lens[None]).int(), scale, g)
    one = torch.ones((), dtype=dtype, device=cuda)
    a, c = run(fw, t, w, lens, scale, one.expand(g.shape)), run(fw, t, w, lens, scale, torch.ones_like(g))
    assert torch.equal(a[1], c[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(fw, t, w, lens, scale, g)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_equal_calls_give_equal_bits(fw, cuda):
    a = inputs(cuda, torch.float32, 30, 800, 500, 128, few=20)
    first = run(fw, *a)
    for _ in range(3):
        assert torch.equal(run(fw, *a)[1], first[1])


def test_refusals(fw, cuda):
    t, w, lens, scale, g = inputs(cuda, torch.float32, 2, 5, 9, 8)
    for x, y, kw in [(t.cpu(), w, {}), (t, w.cpu(), {}), (t.float(), w, {}), (t, w.half(), {}), (t, w[0], {}), (t, w[:0], {}), (t, w[:, :0], {}),
                     (t[None], w, {}), (t, w, dict(seq_lens=lens.long())), (t, w, dict(seq_lens=lens[:1])), (t[0], w, dict(seq_lens=lens)),
                     (t, w, dict(seq_lens=torch.ones(4, 2, device=cuda)))]:
        for train in (False, True):
            with pytest.raises(RuntimeError):
                fw.label_embedding(x, y.detach().requires_grad_(train), **kw)

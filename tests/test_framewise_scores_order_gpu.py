"""The order of label_scores' alternatives: that of the logits, equal ones by their class, whatever is left of a difference
between them once the row's maximum and the logarithm of its sum are taken off, and however many warps share a row."""
import pytest
import torch

from test_framewise_scores_gpu import incoming, inputs, reference

from framewise_util import close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fw():
    import i6_native_ops_b200.framewise as m

    return m


def near_logits(cuda, rows, V, seed=0):
    """Rows of logits an ulp apart around 4.5 in an order of their own, under one that is far above them: log probabilities of
    some -13, whose ulp is two of the logits'."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    step = 2.0**-21
    z = 4.5 + step * torch.rand(rows, V, device=cuda, generator=gen).argsort(1).float()
    assert V < 2**19 and bool((z.sort(1).values.diff(dim=1) >= step).all())
    z.scatter_(1, torch.randint(0, V, (rows, 1), device=cuda, generator=gen), 18.0)
    return z


def by_logits(z, top):
    return torch.sort(z.double(), dim=-1, descending=True, stable=True).indices[..., :top]


@pytest.mark.parametrize("V", [41, 500, 3001, 6001, 33001])
@pytest.mark.parametrize("rows", [1, 40, 300, 1200, 2400, 5000])
def test_logits_an_ulp_apart(fw, cuda, rows, V):
    """Row counts and lengths at which one warp to eight CTAs have a row."""
    if rows * V > 40_000_000:
        pytest.skip("covered by the shorter rows")
    z = near_logits(cuda, rows, V, seed=rows + V)
    t = torch.zeros(rows, dtype=torch.int64, device=cuda)
    want = by_logits(z, 32)
    for top in (1, 2, 3, 8, 9, 31, 32):
        got = fw.label_scores(z, t, top=top)
        assert torch.equal(got.top_labels, want[:, :top]), top
        assert bool((got.top_log_probs[:, :-1] >= got.top_log_probs[:, 1:]).all())


def test_fewer_alternatives_are_the_first_of_more(fw, cuda):
    apart = torch.full((64, 500), -3.0, device=cuda)
    apart[:, 400] = 18.0
    apart[:, 7] = 5.0
    apart[:, 300] = torch.nextafter(torch.tensor(5.0), torch.tensor(6.0)).to(cuda)
    t = torch.zeros(64, dtype=torch.int32, device=cuda)
    for z in (near_logits(cuda, 64, 500), apart):
        lists = [fw.label_scores(z, t, top=top).top_labels for top in range(1, 33)]
        for fewer, more in zip(lists, lists[1:]):
            assert torch.equal(fewer, more[:, :-1])
    assert lists[2][0].tolist() == [400, 300, 7]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sizes", [(3, 5, 7), (2, 33, 8), (4, 10, 33), (3, 11, 257), (5, 7, 1000), (8, 1, 10025), (70, 3, 2047), (40, 125, 41), (17, 300, 1025)])
def test_sizes_by_the_order_of_64_bits(fw, cuda, dtype, sizes):
    B, T, V = sizes
    for top in sorted({1, min(V, 5), min(V, 32)}):
        z, t, lens = inputs(cuda, dtype, B, T, V, seed=sum(sizes) + top, short=top % 2 == 0)
        g = incoming((B, T), top)
        zz = z.detach().requires_grad_()
        got = fw.label_scores(zz, t, top=top, seq_lens=lens)
        torch.autograd.backward(got[:3], g)
        want = reference(z, t, lens, top, g)
        assert torch.equal(got.top_labels.long(), want["top_labels"])
        close(got.top_log_probs.detach(), want["top_log_probs"], "top_log_probs")
        close(zz.grad, want["logits"], "logits")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_go_to_the_labels_in_that_order(fw, cuda, dtype):
    z = near_logits(cuda, 50, 900, seed=5).to(dtype)[None]
    z[..., 3::7] = z[..., 5:6]  # and equal ones
    t = torch.arange(50, device=cuda)[None].to(torch.int32)
    top = 12
    g = incoming((1, 50), top, seed=3)
    zz = z.detach().requires_grad_()
    got = fw.label_scores(zz, t, top=top)
    torch.autograd.backward(got[:3], g)
    want = reference(z, t, None, top, g)  # its own order, by the logits in 64 bits
    assert torch.equal(got.top_labels.long(), want["top_labels"])
    close(got.top_log_probs.detach(), want["top_log_probs"], "top_log_probs")
    close(zz.grad, want["logits"], "logits")


def test_many_rows_of_a_batch(fw, cuda):
    """Some hundred thousand neighbours in the lists of normal logits, of which a few lie an ulp or two apart."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    for _ in range(4):
        z = 1.5 * torch.randn(20, 1000, 6001, device=cuda, generator=gen)
        z[..., 17] += 9.0
        got = fw.label_scores(z, torch.zeros(20, 1000, dtype=torch.int32, device=cuda), top=8)
        best = torch.topk(z, 9, dim=-1)
        label, value = best.indices, best.values
        order = label.argsort(-1)  # equal logits by their class
        label, value = label.gather(-1, order), value.gather(-1, order)
        order = torch.sort(value, dim=-1, descending=True, stable=True).indices
        assert bool((value.gather(-1, order)[..., 7] > value.gather(-1, order)[..., 8]).sum() > 19000)
        clear = value.gather(-1, order)[..., 7] > value.gather(-1, order)[..., 8]
        assert torch.equal(got.top_labels[clear].long(), label.gather(-1, order)[..., :8][clear])

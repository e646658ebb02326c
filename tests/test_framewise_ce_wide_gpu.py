"""Output layer with cross entropy at the widths and sizes of large models, against the formula in 64 bits."""
import pytest
import torch

from test_framewise_ce_gpu import check, inputs

pytestmark = pytest.mark.gpu

IGNORE = -100
TYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def fw():
    import i6_native_ops_b200.framewise as m

    return m


@pytest.mark.parametrize("dtype", TYPES)
def test_losses_do_not_drift_with_the_width(fw, cuda, dtype):
    """Tensor cores cut a sum off at 2^-24 of it each step of 16.  Over 512 of K that is 32 cuts (and those of the small
    parts of f32 values, 2^-8 of it: one more), so where sums of more come from segments of 512 a logit z, whose segments'
    magnitudes add up to no more than max(|z|, sqrt(segments) times its spread), loses less than 33 2^-24 of that whatever
    the width.  The largest logits, which make up the loss, are below 10 here, the spread of a logit 2.  One sum over
    all of 16384 would lose 1024 / 2 times 2^-24 of its mean magnitude, three times what is allowed."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    N, V, D = 600, 700, 16384
    x = torch.randn(N, D, device=cuda, generator=gen).to(dtype)
    w = (torch.randn(V, D, device=cuda, generator=gen) * 2 / D**0.5).to(dtype)
    t = torch.randint(0, V, (N,), device=cuda, generator=gen)
    want = torch.nn.functional.cross_entropy(x.double() @ w.double().T, t, reduction="none")
    got = fw.linear_cross_entropy(x, w, t).double()
    assert abs(float((got - want).mean())) <= 33 * 2.0**-24 * max(10.0, 2 * 32**0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [(1, 1025, 300, 257), (3, 700, 513, 500), (2, 1500, 1000, 1024), (5, 411, 70, 300), (1, 1100, 20000, 40),
                                   (2, 1300, 131, 24), (4, 700, 2049, 260)])
def test_tiles_of_two_ctas(fw, cuda, dtype, sizes):
    """More than 1024 positions: tiles of 256 rows on pairs of SMs, over one and several stages of K and tiles of D; with
    20000 classes whole rows of the weight's gradient as well as shared ones."""
    for bias, short in ((True, False), (False, True)):
        check(fw, *inputs(cuda, dtype, *sizes, seed=sum(sizes), bias=bias, short=short))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [(1, 20000, 300, 64), (3, 9000, 130, 300)])
def test_whole_rows_of_the_activations_gradient(fw, cuda, dtype, sizes):
    """More row tiles than teams of CTAs: some are one team's from the first stage to the last and leave in place."""
    check(fw, *inputs(cuda, dtype, *sizes, short=False))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1025, 2048, 2100, 4100])
@pytest.mark.parametrize("rows", [3, 200, 1100])
def test_widths_of_large_models(fw, cuda, dtype, D, rows):
    """Logits by segments; from 2049 on a row of dX or dW is shared by several teams, from 4097 on by three."""
    check(fw, *inputs(cuda, dtype, 1, rows, 300, D, short=False))


@pytest.mark.parametrize("dtype,rows,V,D,chunk", [(torch.float32, 15400, 10025, 512, 13312), (torch.float32, 27400, 10025, 300, 13312),
                                                   (torch.bfloat16, 34500, 12001, 1024, 33280), (torch.bfloat16, 11000, 40000, 600, 9984)])
def test_chunks_with_whole_rows(fw, cuda, dtype, rows, V, D, chunk):
    """Several chunks of q, of which all but the first are added to the weight's gradient by the copy engine (whole rows) and
    by joined pieces (shared ones)."""
    h, w, b, t, lens, g = inputs(cuda, dtype, 1, rows, V, D, skip=0.01, short=False)
    assert int((t != IGNORE).sum()) > rows // chunk * chunk + 256
    check(fw, h, w, b, t, lens, g)
    torch.cuda.empty_cache()

"""Output layer with cross entropy at the widths and sizes of large models, against the formula in 64 bits."""
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

"""Orthogonalisation of matrices whose norm is past the range of 32 bits."""
import pytest
import torch

from test_framewise_muon_gpu import check, matrices, with_bound

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fw():
    import i6_native_ops_b200.framewise as m

    return m


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 5), (64, 200), (128, 256), (500, 2001), (300, 140)])
@pytest.mark.parametrize("most", [3e38, 1e35, 1e31, 1e29])
def test_large_values(fw, cuda, dtype, shape, most):
    """1 / |U| is below the smallest normal number of 32 bits for the largest of these."""
    x = matrices(cuda, shape, dtype, seed=7).double()
    x = (x * (most / float(x.abs().max()))).to(dtype)
    assert bool(x.isfinite().all())
    check(fw.orthogonalize(x), with_bound(x))


@pytest.mark.parametrize("steps", [1, 5])
@pytest.mark.parametrize("shape", [(1, 5000), (128, 256), (500, 2001)])
def test_all_values_large(fw, cuda, shape, steps):
    """Norms of some 10^40 and 10^41: of their reciprocals 32 bits hold some 16 and 12."""
    for seed in range(4):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        x = 3.4e38 * (1 - 0.5 * torch.rand(shape, device=cuda, generator=gen))
        x *= torch.randint(0, 2, shape, device=cuda, generator=gen) * 2 - 1
        check(fw.orthogonalize(x, steps=steps), with_bound(x, steps=steps), str(seed))


@pytest.mark.parametrize("shape", [(60, 100), (150, 300)])
def test_a_step_on_large_gradients(fw, cuda, shape):
    x = matrices(cuda, shape, seed=3).double()
    g = (x * (3e38 / float(x.abs().max()))).float()
    p, v = torch.zeros(shape, device=cuda), torch.zeros(shape, device=cuda)
    fw.muon_step([p], [g], [v], lr=1.0, beta=0.5, nesterov=False, weight_decay=0.0)
    assert torch.equal(v, g * 0.5)
    check(-p / max(1.0, shape[0] / shape[1]) ** 0.5, with_bound(v))

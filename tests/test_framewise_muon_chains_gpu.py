"""More matrices than a chain of launches takes, by their number and by its scratch, of shapes that no CTA holds alone."""
import pytest
import torch

from test_framewise_muon_gpu import TYPES, check, matrices, reference_step, with_bound

from framewise_util import close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fw():
    import i6_native_ops_b200.framewise as m

    return m


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(300, 5, 260), (260, 130, 140), (530, 270, 2)])
def test_more_matrices_than_a_chain_takes(fw, cuda, dtype, shape):
    x = matrices(cuda, shape, dtype, seed=4)
    got = fw.orthogonalize(x)
    check(got, with_bound(x))
    assert torch.equal(fw.orthogonalize(x[250:260]), got[250:260])  # the last of a chain and the first of the next
    assert torch.equal(fw.orthogonalize(x), got)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_step_over_more_than_a_chain(fw, cuda, dtype):
    shapes = [(5, 260), (130, 140), (270, 3), (129, 129), (9, 20), (64, 300)] * 60  # 300 of a chain, and 60 that a CTA holds
    gen = torch.Generator(device="cuda").manual_seed(5)
    p = [torch.randn(s, device=cuda, generator=gen).to(dtype) for s in shapes]
    g = [matrices(cuda, s, dtype, seed=i) for i, s in enumerate(shapes)]
    v = [matrices(cuda, s, seed=1000 + i) for i, s in enumerate(shapes)]
    want = {i: reference_step(p[i], g[i], v[i], 0.05, 0.9, True, 0.1, False, dtype) for i in (*range(0, 12), *range(295, 330), *range(354, 360))}
    alone = [p[-6].clone()], [g[-6]], [v[-6].clone()]
    fw.muon_step(p, g, v, lr=0.05, beta=0.9)
    fw.muon_step(*alone, lr=0.05, beta=0.9)
    r = torch.finfo(dtype).eps / 2
    for i, ((new, dv), (out, dout)) in want.items():
        close(v[i], (new, dv), f"momentum {i}")
        close(p[i], (out, dout + r * out.abs()), f"parameter {i}")
    assert torch.equal(alone[2][0], v[-6])
    assert all(bool(x.isfinite().all()) for x in p + v)


@pytest.mark.parametrize("dtype,count", [(torch.float32, 30), (torch.bfloat16, 50)])
def test_more_scratch_than_a_chain_takes(fw, cuda, dtype, count):
    """Two gigabytes hold 25 float32 matrices of 2048 x 2048, 42 of bfloat16."""
    x = matrices(cuda, (count, 2048, 2048), dtype, seed=6)
    got = fw.orthogonalize(x)
    for i in (0, count - 7, count - 1):
        check(got[i], with_bound(x[i]))
    assert torch.equal(fw.orthogonalize(x[count - 10 :]), got[count - 10 :])

"""bfloat16 matrices of few rows and many columns.

Bound.  As a part of the result's norm: its own rounding has a root mean square of up to 2^-8 x 0.45 = 1.75e-3.  A step's factor B,
less a multiple of the identity, is at most 2.81 (the range of b q + c q^2 for q up to 1.3), and it and X are rounded to
11 bits, 2.0e-4 by root mean square each: 2.81 x 2.0e-4 x sqrt 2 = 8e-4 a step and sqrt 5 of that in five, 1.8e-3.  Together
sqrt(1.75^2 + 1.8^2) = 2.5e-3; three quarters of 2^-8, 2.93e-3, leave a sixth for matrices of so few values of B.  A in 11 bits
as well is what this excludes: b A and c A A, each larger than B, then no longer undo each other."""
import pytest
import torch

from test_framewise_muon_gpu import ABC, formula, matrices

pytestmark = pytest.mark.gpu

SHAPES = [(2, 257), (2, 300), (2, 4096), (3, 1024), (4, 600), (5, 260), (8, 700), (64, 512), (100, 300), (128, 300), (128, 257)]


@pytest.fixture(scope="module")
def fw():
    import i6_native_ops_b200.framewise as m

    return m


def off(got, x):
    want = formula(x, ABC, 5, 1e-7)
    return (got.double() - want).square().sum((-2, -1)).sqrt() / want.square().sum((-2, -1)).sqrt()


@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_few_rows(fw, cuda, shape, turned):
    for seed in range(4):
        x = matrices(cuda, (40,) + shape, torch.bfloat16, seed=seed)
        if turned:
            x = x.mT.contiguous()
        worst = float(off(fw.orthogonalize(x), x).max())
        assert worst <= 0.75 * 2.0**-8, (seed, worst)


def test_the_same_with_others_in_one_call(fw, cuda):
    """Few rows and many in one chain: each goes by its own number of rows."""
    shapes = [(2, 300), (300, 500), (3, 1024), (140, 260), (128, 600), (600, 2)] * 5
    x = [matrices(cuda, s, torch.bfloat16, seed=i) for i, s in enumerate(shapes)]
    p = [torch.zeros(s, device=cuda).bfloat16() for s in shapes]
    copy = [torch.zeros(s, device=cuda) for s in shapes]
    v = [torch.zeros(s, device=cuda) for s in shapes]
    fw.muon_step(p, x, v, lr=1.0, beta=0.0, nesterov=False, weight_decay=0.0, master=copy)
    for a, c, g in zip(p, copy, x):
        rate = max(1.0, a.shape[0] / a.shape[1]) ** 0.5
        assert torch.equal(a, c.bfloat16())
        assert float(off(-c / rate, g)) <= 0.75 * 2.0**-8

"""Orthogonalisation of matrices whose norm is past the range of 32 bits, and of any positive eps."""
import ctypes

import pytest
import torch

from test_framewise_muon_gpu import ABC, check, matrices, with_bound

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


@pytest.mark.parametrize("eps", [1e-46, 1e-60, 1e-300, 5e-324])
@pytest.mark.parametrize("shape", [(6, 10), (130, 260)])
def test_zeros_stay_zeros_at_any_eps(cuda, shape, eps):
    """Of the C ABI, which takes any positive eps in 64 bits."""
    from i6_native_ops_b200 import build

    lib = ctypes.CDLL(build.build_framewise_lib())
    lib.framewise_b200_orthogonalize_bytes.restype = ctypes.c_size_t
    i64, f64 = ctypes.c_int64, ctypes.c_double
    need = lib.framewise_b200_orthogonalize_bytes(i64(2), i64(shape[0]), i64(shape[1]), ctypes.c_int32(0))
    work = torch.empty(need, dtype=torch.uint8, device=cuda)
    tiny = 2.0**-149  # the smallest number
    x = torch.zeros(2, *shape, device=cuda)
    x[1] = tiny * torch.randint(0, 3, shape, device=cuda, generator=torch.Generator(cuda).manual_seed(1))
    out = torch.full_like(x, 7.0)
    co = (f64 * 15)(*ABC * 5)
    ptr = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.framewise_b200_orthogonalize(i64(2), i64(shape[0]), i64(shape[1]), ctypes.c_int32(0), ptr(x), ptr(out), co, ctypes.c_int32(5), f64(eps), ptr(work),
                                            ctypes.c_size_t(need), stream) == 0
    torch.cuda.synchronize()
    assert not out[0].any()
    check(out[1], with_bound(x[1].double(), eps=1e-300, dtype=torch.float32))  # larger than any of these eps by its norm

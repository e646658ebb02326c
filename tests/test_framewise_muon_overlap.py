"""A Muon step whose tensors overlap is refused: it would write what it has yet to read.  At the C ABI no device is needed: what is
refused is refused before any CUDA call."""
import ctypes

import pytest
import torch

i32, i64, f64, size_t = ctypes.c_int32, ctypes.c_int64, ctypes.c_double, ctypes.c_size_t
OVERLAP = 5


class Matrix(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "momentum", "master")] + [("rows", i64), ("cols", i64)]


@pytest.fixture(scope="module")
def status():
    from i6_native_ops_b200 import build

    lib = ctypes.CDLL(build.build_framewise_lib())
    lib.framewise_b200_status_string.restype = ctypes.c_char_p
    co = (f64 * 15)(*[3.4445, -4.775, 2.0315] * 5)
    assert b"overlap" in lib.framewise_b200_status_string(i32(OVERLAP))

    def run(matrices, dtype):
        # no coefficients: what does not overlap is refused for that, before any CUDA call
        return lib.framewise_b200_muon((Matrix * len(matrices))(*matrices), i64(len(matrices)), i32(dtype), f64(0.1), f64(0.9), i32(1), f64(0.1), i32(0),
                                       None if dtype < 2 else co, i32(5), f64(1e-7), i32(0), ctypes.c_void_p(1 << 40), size_t(1 << 30), None)

    return run


# 8 x 10 values: 320 bytes of float32, 160 of bfloat16
P, G, V, M = 1 << 20, 1 << 21, 1 << 22, 1 << 23


def of(param=P, grad=G, momentum=V, master=None, rows=8, cols=10):
    return Matrix(param, grad, momentum, master, rows, cols)


@pytest.mark.parametrize("size", [(8, 10), (200, 300)])
def test_what_is_written_meets_nothing_else(status, size):
    rows, cols = size
    one = lambda **k: of(rows=rows, cols=cols, **k)  # noqa: E731
    for dtype, each in ((0, 4), (1, 2)):
        values, held = rows * cols * each, rows * cols * 4
        far = dict(param=P * 16, grad=G * 16, momentum=V * 16)
        good = [
            [one()],
            [one(), one(**far)],
            [one(), one(**{**far, "grad": G})],  # a gradient of two parameters
            [one(), one(**{**far, "grad": G + 8 * each})],
            [one(), one(**{**far, "param": P + values})],  # one after another
            [one(grad=P + values)],
            [one(), one(**{**far, "momentum": V + held})],
            [one(), of(P, P, P, None, 0, 8)],  # nothing of it is met
        ]
        bad = [
            [one(grad=V)],  # a gradient that is its own momentum
            [one(grad=V + 4)],
            [one(grad=V - each)],
            [one(grad=P)],
            [one(momentum=P + 4)],
            [one(), one(**{**far, "param": P})],
            [one(), one(**{**far, "param": P + each})],
            [one(), one(**{**far, "param": P + values - each})],
            [one(), one(**{**far, "momentum": V + held - 4})],
            [one(), one(**{**far, "grad": V + held - each})],
            [one(), one(**{**far, "grad": P + values - each})],
            [one(**far), one(grad=far["param"])],
        ]
        if dtype == 1:
            good += [[one(master=M)], [one(master=P + values)]]
            bad += [[one(master=V)], [one(master=V + 8)], [one(master=G)], [one(master=P + 4)], [one(master=M), one(**far, master=M)]]
        for m in good:
            assert status(m, dtype) == 1
        for m in bad:
            assert status(m, dtype) == OVERLAP


@pytest.mark.gpu
def test_overlaps_are_refused(cuda):
    import i6_native_ops_b200.framewise as fw

    flat = torch.randn(4000, device=cuda)
    g, w = torch.randn(30, 40, device=cuda), torch.randn(30, 40, device=cuda)
    new = lambda: torch.zeros(30, 40, device=cuda)  # noqa: E731
    before = flat.clone()
    cut = lambda at: flat[at : at + 1200].view(30, 40)  # noqa: E731
    v = new()
    bad = [
        ([w], [v], [v]),
        ([w], [w], [v]),
        ([cut(0), cut(1000)], [g, g], [new(), new()]),
        ([w, new()], [g, g], [cut(0), cut(1199)]),
        ([w], [cut(4)], [cut(0)]),
        ([w, cut(0)], [cut(100), g], [new(), new()]),
    ]
    for params, grads, momentum in bad:
        with pytest.raises(RuntimeError, match="overlap"):
            fw.muon_step(params, grads, momentum)
    assert torch.equal(flat, before) and not v.any()
    # neighbours and shared gradients are no overlaps, nor is a gradient that has to be laid out anew
    fw.muon_step([cut(0), cut(1200)], [g, g], [new(), new()])
    fw.muon_step([w], [g.T.contiguous().T], [new()])
    assert torch.equal(flat[2400:], before[2400:]) and not torch.equal(flat[:2400], before[:2400])
    # nor a parameter's own gradient that changes sign in a view
    fw.muon_step([w], [torch._neg_view(g)], [new()])

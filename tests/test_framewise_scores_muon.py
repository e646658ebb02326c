"""CPU checks of the boundary of label scores and Muon: bad arguments are refused before any CUDA call, CPU tensors are refused.
No kernel is launched."""
import ctypes

import pytest
import torch

i32, i64, f64, size_t = ctypes.c_int32, ctypes.c_int64, ctypes.c_double, ctypes.c_size_t


class Shape(ctypes.Structure):
    _fields_ = [(n, i64) for n in ("B", "T", "V", "stride_b", "stride_t", "ignore")] + [(n, i32) for n in ("dtype", "labels64", "top")]


class Matrix(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "momentum", "master")] + [("rows", i64), ("cols", i64)]


@pytest.fixture(scope="module")
def lib():
    from i6_native_ops_b200 import build

    lib = ctypes.CDLL(build.build_framewise_lib())
    lib.framewise_b200_muon_bytes.restype = lib.framewise_b200_orthogonalize_bytes.restype = size_t
    return lib


def test_scores_arguments(lib):
    def forward(shape):
        return lib.framewise_b200_scores_forward(ctypes.byref(shape) if shape else None, None, None, None, None, None, None, None, None, None)

    def backward(shape):
        return lib.framewise_b200_scores_backward(ctypes.byref(shape) if shape else None, None, None, None, None, None, None, None, None)

    good = dict(B=2, T=3, V=10, stride_b=30, stride_t=10, ignore=-100, dtype=0, labels64=0, top=2)
    for f in (forward, backward):
        assert f(None) == 1 and f(Shape(**good)) == 1  # null pointers
        for bad in (dict(B=-1), dict(T=-1), dict(V=0), dict(V=1 << 27), dict(B=1 << 20, T=1 << 12), dict(top=-1), dict(top=33), dict(top=11), dict(dtype=2)):
            assert f(Shape(**{**good, **bad})) == 1, bad
        for none in (dict(B=0), dict(T=0)):
            assert f(Shape(**{**good, **none})) == 0


def test_orthogonalize_arguments(lib):
    size = lambda *a: lib.framewise_b200_orthogonalize_bytes(*(i64(x) for x in a[:3]), i32(a[3]))  # noqa: E731
    assert size(1, 4, 4, 2) == 0 and size(-1, 4, 4, 0) == 0 and size(1, -4, 4, 0) == 0 and size(1, 1 << 20, 1 << 20, 0) == 0
    assert size(0, 4, 4, 0) > 0 and size(1, 4, 0, 0) > 0 and size(1 << 40, 4, 4, 0) == size(1, 4, 4, 0)
    co = (f64 * 15)(*[3.4445, -4.775, 2.0315] * 5)

    def run(count=1, rows=4, cols=4, dtype=0, x=1 << 12, out=1 << 12, coefficients=co, steps=5, eps=1e-7, work=1 << 12, work_bytes=1 << 20):
        return lib.framewise_b200_orthogonalize(i64(count), i64(rows), i64(cols), i32(dtype), ctypes.c_void_p(x), ctypes.c_void_p(out), coefficients, i32(steps),
                                                f64(eps), ctypes.c_void_p(work), size_t(work_bytes), None)

    assert run(count=0) == 0 and run(rows=0) == 0  # nothing to do
    grows = (f64 * 15)(*[100.0, 0.0, 0.0] * 5)
    nan = (f64 * 15)(*[float("nan")] * 15)
    for bad in (dict(count=-1), dict(dtype=7), dict(x=None), dict(out=None), dict(coefficients=None), dict(coefficients=grows), dict(coefficients=nan), dict(steps=0),
                dict(steps=101), dict(eps=0.0), dict(eps=float("nan")), dict(work=None), dict(work=1 << 12 | 8), dict(rows=1 << 20, cols=1 << 20)):
        assert run(**bad) == 1, bad
    assert run(rows=200, cols=300, work_bytes=100) == 2


def test_muon_arguments(lib):
    one = (Matrix * 1)(Matrix(1 << 12, 1 << 13, 1 << 14, None, 8, 8))
    co = (f64 * 15)(*[3.4445, -4.775, 2.0315] * 5)

    def run(matrices=one, count=1, dtype=0, steps=5, eps=1e-7, work=1 << 12):
        return lib.framewise_b200_muon(matrices, i64(count), i32(dtype), f64(0.1), f64(0.9), i32(1), f64(0.1), i32(0), co, i32(steps), f64(eps), i32(0),
                                       ctypes.c_void_p(work), size_t(1 << 20), None)

    assert run(count=0) == 0
    for bad in (dict(matrices=None), dict(count=-1), dict(dtype=3), dict(steps=0), dict(eps=-1.0), dict(work=None)):
        assert run(**bad) == 1, bad
    for m in (Matrix(None, 1, 1, None, 8, 8), Matrix(1, None, 1, None, 8, 8), Matrix(1, 1, None, None, 8, 8), Matrix(1, 1, 1, 1, 8, 8), Matrix(1, 1, 1, None, -8, 8),
              Matrix(1, 1, 1, None, 1 << 31, 8)):
        assert run(matrices=(Matrix * 1)(m)) == 1
    bytes_of = lambda rows, cols, n=1: lib.framewise_b200_muon_bytes((Matrix * n)(*[Matrix(1, 1, 1, None, rows, cols)] * n), i64(n), i32(0))  # noqa: E731
    assert bytes_of(1 << 31, 8) == 0 and bytes_of(8, 8) > 0
    # scratch is bounded: more matrices than that go through it one after another
    assert bytes_of(500, 2001, 300) <= bytes_of(500, 2001, 150) < 3 << 30


def test_cpu_tensors_are_refused():
    import i6_native_ops_b200.framewise as fw

    x, t = torch.zeros(2, 3, 4), torch.zeros(2, 3, dtype=torch.int32)
    for f in (lambda: fw.label_scores(x, t), lambda: fw.orthogonalize(x), lambda: fw.muon_step([x[0]], [x[0]], [x[0]])):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()
    fw.muon_step([], [], [])  # nothing to do


def test_muon_options():
    import i6_native_ops_b200.framewise as fw

    w = torch.nn.Parameter(torch.zeros(3, 4))
    with pytest.raises(ValueError, match="matrices"):
        fw.Muon([w, torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(ValueError, match="adjust_lr"):
        fw.Muon([w], adjust_lr="none")
    for bad in ((1.0, 2.0), [], [(1.0, 2.0, 3.0)] * 4, 3.0):
        with pytest.raises(RuntimeError, match="coefficients"):
            fw.Muon([w], steps=5, coefficients=bad)
    opt = fw.Muon([w], steps=2, coefficients=[(1.0, 2.0, 3.0)] * 2)
    opt.step()  # no gradient: nothing to do
    assert not opt.state[w]

"""CPU checks of the framewise operators' boundary: the library exports what its header declares, bad arguments are
refused before any CUDA call, CPU tensors are refused.  No kernel is launched."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "framewise_b200.h")


@pytest.fixture(scope="module")
def lib():
    from i6_native_ops_b200 import build

    return ctypes.CDLL(build.build_framewise_lib())


def test_library_exports_every_declared_symbol(lib):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(framewise_b200_[a-z_0-9]+)\s*\(", text)))
    assert len(names) >= 10
    for n in names:
        assert hasattr(lib, n), n
    lib.framewise_b200_status_string.restype = ctypes.c_char_p
    assert lib.framewise_b200_status_string(0) == b"ok"
    for code in range(1, 5):
        assert lib.framewise_b200_status_string(code) not in (b"ok", b"unknown status")


def test_argument_checks_without_a_device(lib):
    i64, f64 = ctypes.c_int64, ctypes.c_double
    assert lib.framewise_b200_ce_bytes(None, None, None, None) == 1
    assert lib.framewise_b200_embed_forward(i64(-1), i64(1), i64(1), i64(1), 0, 0, i64(0), ctypes.c_float(1), None, None, None, None, None) == 1
    assert lib.framewise_b200_adamw(None, i64(1), 0, 32, f64(1), f64(0), f64(0), f64(0), f64(0), i64(1), None) == 1
    assert lib.framewise_b200_adamw(None, i64(0), 0, 16, f64(1), f64(0), f64(0), f64(0), f64(0), i64(1), None) == 1
    assert lib.framewise_b200_adamw_decode(None, i64(2), None) == 1


def test_cpu_tensors_are_refused():
    import i6_native_ops_b200.framewise as fw

    x, w, t = torch.zeros(2, 3, 4), torch.zeros(5, 4), torch.zeros(2, 3, dtype=torch.int32)
    for f in (lambda: fw.linear_cross_entropy(x, w, t), lambda: fw.label_embedding(t, w), lambda: fw.adamw_step([w], [w], [w], [w], step=1)):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()
    fw.adamw_step([], [], [], [], step=1)  # nothing to do

"""CPU: what the entry points of the linear softmax cross-entropy, the group norm and
the 8-bit activations refuse is refused before any device is touched."""
import pytest

import micrograd_b200
from micrograd_b200 import cabi as K

P = 4096  # stands for a device pointer; a refused call never follows it


@pytest.fixture(scope="module")
def lib():
    return micrograd_b200.load_abi()


def refused(lib, name, *args, text):
    with pytest.raises(K.MgError) as e:
        lib.call(name, *args)
    assert e.value.code == K.ERR_INVALID
    assert text in str(e.value), str(e.value)
    assert name in str(e.value), str(e.value)


def test_linear_xent(lib):
    fwd, both = "mg_linear_xent_fwd", "mg_linear_xent_fwd_bwd"
    refused(lib, fwd, P, P, P, P, None, 4, 8, 16, 4.0, text="null output")
    refused(lib, fwd, None, P, P, P, P, 4, 8, 16, 4.0, text="null input")
    refused(lib, fwd, P, None, P, P, P, 4, 8, 16, 4.0, text="null input")
    refused(lib, fwd, P, P, P, None, P, 4, 8, 16, 4.0, text="null input")
    for denom in (0.0, -1.0, float("nan")):
        refused(lib, fwd, P, P, P, P, P, 4, 8, 16, denom, text="denom must be positive")
    for sizes in ((1 << 30, 8, 16), (4, 1 << 30, 16), (4, 8, 1 << 30)):
        refused(lib, fwd, P, P, P, P, P, *sizes, 4.0, text="dimension too large")
    refused(lib, both, P, P, P, P, P, None, P, P, P, 4, 8, 16, 4.0, 0, text="null output")
    refused(lib, both, P, None, P, P, P, P, P, P, P, 4, 8, 16, 4.0, 0, text="null input")
    refused(lib, both, P, P, P, P, P, P, P, P, P, 4, 8, 16, 0.0, 0, text="denom must be positive")


def test_group_norm(lib):
    fwd, bwd = "mg_group_norm_fwd", "mg_group_norm_bwd"
    for c, g in ((10, 3), (10, 0), (0, 1), (4, 8)):
        refused(lib, fwd, P, P, P, P, P, P, 2, 3, c, g, 1e-5, K.ACT_NONE, text="groups of equal size")
    for act in (-1, 3):
        refused(lib, fwd, P, P, P, P, P, P, 2, 3, 8, 2, 1e-5, act, text="unknown activation")
        refused(lib, bwd, P, P, P, P, P, P, P, P, P, 2, 3, 8, 2, act, 0, text="unknown activation")
    for eps in (-1e-5, float("nan")):
        refused(lib, fwd, P, P, P, P, P, P, 2, 3, 8, 2, eps, K.ACT_NONE, text="eps must not be negative")
    refused(lib, fwd, P, P, P, P, P, P, 1 << 30, 3, 8, 2, 1e-5, K.ACT_NONE, text="dimension too large")
    refused(lib, fwd, P, P, P, P, P, P, 1 << 29, 1, 8, 8, 1e-5, K.ACT_NONE, text="too many groups")
    for hole in (0, 3, 4, 5):
        args = [P] * 6
        args[hole] = None
        refused(lib, fwd, *args, 2, 3, 8, 2, 1e-5, K.ACT_NONE, text="null pointer")
    for hole in (0, 3, 4, 5):
        args = [P] * 9
        args[hole] = None
        refused(lib, bwd, *args, 2, 3, 8, 2, K.ACT_NONE, 0, text="null pointer")


def test_q8(lib):
    for name in ("mg_q8_pack", "mg_q8_unpack"):
        for hole in range(3):
            args = [P] * 3
            args[hole] = None
            refused(lib, name, *args, 4, 65, text="null pointer")
        refused(lib, name, P, P, P, 1 << 40, 1, text="dimension too large")
        refused(lib, name, P, P, P, 1 << 35, 1 << 35, text="dimension too large")
    for hole in range(4):
        args = [P] * 4
        args[hole] = None
        refused(lib, "mg_gemm_tn_q8", *args, 4, 6, 8, 0, text="null pointer")
    for hole in range(3):
        args = [P] * 3
        args[hole] = None
        refused(lib, "mg_gemm_nt_q8", *args, 4, 6, 8, 0, P, text="null pointer")
    refused(lib, "mg_gemm_nt_q8", P, P, P, 4, 6, 8, 0, None, text="null pointer")
    for hole in range(3):
        args = [P] * 3
        args[hole] = None
        refused(lib, "mg_relu_bwd_q8", *args, 5, 0, text="null pointer")

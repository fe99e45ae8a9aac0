"""Argument checks of the 8-bit row operators, the INT8 product and the token
log probabilities: refused before any device work, with a message."""
import ctypes as C
import os

import pytest

from conftest import load_pkg_module

P = 4096  # an aligned pointer, never dereferenced: the arguments fail first


@pytest.fixture(scope="module")
def eng():
    e = load_pkg_module("engine")
    if not os.path.exists(e.LIB_PATH):
        pytest.skip("libengine_cuda.so not built")
    return e


def refused(eng, fn, good, changes, code):
    args = list(good)
    for i, v in changes.items():
        args[i] = v
    assert fn(*args) == code, changes
    assert eng.lib().ec_last_error()


NORM = [0, P, 64, P, 64, P, 64, P, 1e-5, 2, 64, P, 64, P, None]


@pytest.mark.parametrize("changes", [
    {0: 3}, {0: -1}, {1: None}, {2: 63}, {4: 63}, {6: 63}, {8: -1.0}, {8: float("nan")}, {9: 0},
    {9: -1}, {10: 0}, {11: None}, {12: 63}, {13: None}])
def test_norm_arguments(eng, changes):
    refused(eng, eng.lib().ec_op_add_rmsnorm_quant, NORM, changes, eng.EC_ERR_ARG)


@pytest.mark.parametrize("changes", [
    {1: P + 2}, {3: P + 1}, {5: P + 3}, {7: P + 1}, {13: P + 2}, {0: 1, 1: P + 1}, {0: 2, 5: P + 1}])
def test_norm_element_alignment(eng, changes):
    refused(eng, eng.lib().ec_op_add_rmsnorm_quant, NORM, changes, eng.EC_ERR_ARG)


def test_norm_width(eng):
    n = 57345
    refused(eng, eng.lib().ec_op_add_rmsnorm_quant, NORM,
            {2: n, 4: n, 6: n, 10: n, 12: n}, eng.EC_ERR_UNSUPPORTED)
    refused(eng, eng.lib().ec_op_add_rmsnorm_quant, NORM, {9: 2 ** 30 + 1}, eng.EC_ERR_UNSUPPORTED)


SILU = [0, P, P, 64, 2, 64, P, 64, P, None]


@pytest.mark.parametrize("changes", [
    {0: 3}, {1: None}, {2: None}, {3: 63}, {4: 0}, {5: 0}, {6: None}, {7: 63}, {8: None},
    {1: P + 2}, {2: P + 1}, {0: 1, 2: P + 1}, {8: P + 1}])
def test_silu_arguments(eng, changes):
    refused(eng, eng.lib().ec_op_silu_mul_quant, SILU, changes, eng.EC_ERR_ARG)


def test_silu_width(eng):
    n = 57345
    refused(eng, eng.lib().ec_op_silu_mul_quant, SILU, {3: n, 5: n, 7: n}, eng.EC_ERR_UNSUPPORTED)
    refused(eng, eng.lib().ec_op_silu_mul_quant, SILU, {4: 2 ** 30 + 1}, eng.EC_ERR_UNSUPPORTED)


# x ldx sx w ldw sw type y ldy m k nb status stream
GEMM = [P, 64, P, P, 64, P, 0, P, 32, 32, 64, 2, None, None]


@pytest.mark.parametrize("changes", [
    {0: None}, {2: None}, {3: None}, {5: None}, {7: None}, {6: 3}, {9: 0}, {10: 0}, {11: 0},
    {1: 48}, {4: 48}, {8: 31}, {1: 72}, {4: 72}, {0: P + 8}, {3: P + 1},
    {7: P + 2}, {6: 1, 7: P + 1}, {2: P + 2}, {5: P + 1}, {12: P + 2}])
def test_gemm_arguments(eng, changes):
    refused(eng, eng.lib().ec_op_gemm_w8a8, GEMM, changes, eng.EC_ERR_ARG)


def test_gemm_length(eng):
    fn, big = eng.lib().ec_op_gemm_w8a8, 2 ** 30 + 1
    refused(eng, fn, GEMM, {1: 131072, 4: 131072, 10: 131072}, eng.EC_ERR_UNSUPPORTED)
    refused(eng, fn, GEMM, {11: big}, eng.EC_ERR_UNSUPPORTED)
    refused(eng, fn, GEMM, {9: big, 8: big}, eng.EC_ERR_UNSUPPORTED)


# type logits ld n rows tokens temperature top_k logprob entropy ids tlp stream
LOGP = [0, P, 64, 64, 2, P, 1.0, 4, P, P, P, P, None]


@pytest.mark.parametrize("changes", [
    {0: 3}, {1: None}, {2: 63}, {3: 0}, {4: 0}, {5: None}, {8: None}, {6: 0.0}, {6: -1.0},
    {6: float("nan")}, {6: float("inf")}, {6: 1e-38}, {7: -1}, {7: 65}, {10: None}, {11: None},
    {1: P + 2}, {0: 2, 1: P + 1}, {5: P + 2}, {8: P + 1}, {9: P + 2}, {10: P + 2}, {11: P + 2}])
def test_logprob_arguments(eng, changes):
    refused(eng, eng.lib().ec_op_token_logprobs, LOGP, changes, eng.EC_ERR_ARG)


def test_logprob_top(eng):
    fn, big = eng.lib().ec_op_token_logprobs, 2 ** 30 + 1
    refused(eng, fn, LOGP, {7: 33}, eng.EC_ERR_UNSUPPORTED)
    refused(eng, fn, LOGP, {4: big}, eng.EC_ERR_UNSUPPORTED)
    refused(eng, fn, LOGP, {2: big, 3: big}, eng.EC_ERR_UNSUPPORTED)
    assert C.sizeof(C.c_int64) == 8

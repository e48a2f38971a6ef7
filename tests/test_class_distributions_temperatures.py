"""Temperatures that fp32 cannot divide by, or whose square it does not hold, are refused: no GPU needed, no pointer is followed."""
import pytest

from multimae_amd import _lib

P = 4096  # an address that is never read
# log2(e) / T has to be finite: from 1.4427 / 3.4028e38 = 4.24e-39 on
TOO_LOW = [1e-45, 1e-40, 4.2e-39]


def log_probs(temperature):
    return _lib.load().mmae_class_log_probs(P, 0, 4, 100, 1, 100, P, 5, temperature, P, P, P, P, P, P, None, 0, None)


def backward(temperature):
    return _lib.load().mmae_class_log_probs_bwd(P, 0, 4, 100, 1, 100, P, temperature, P, P, P, P, None, P, None)


def distill(temperature, mask=P):
    return _lib.load().mmae_distill(P, 0, 4, 100, 16, 1600, P, 8, P, 0, 5, 1, temperature, mask, 4, 2, None, 0, 0, P, P, P, 1 << 20, None)


@pytest.mark.parametrize("call", [log_probs, backward, distill], ids=lambda f: f.__name__)
@pytest.mark.parametrize("temperature", TOO_LOW)
def test_temperatures_without_a_reciprocal(call, temperature):
    assert call(temperature) == -1
    assert b"temperature" in _lib.load().mmae_last_error()


@pytest.mark.parametrize("mask", [P, None], ids=["mask", "no mask"])
# T^2 at most 3.4e38; T^2 / 64 positions, the smallest weight, at least 1.18e-38
@pytest.mark.parametrize("temperature", [1.9e19, 1e30, 3e38, 8e-19, 1e-19, 1e-30])
def test_temperatures_whose_square_is_no_weight(temperature, mask):
    assert distill(temperature, mask) == -1
    assert b"temperature" in _lib.load().mmae_last_error()

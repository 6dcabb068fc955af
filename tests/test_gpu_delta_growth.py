"""The gated delta rule with decays that grow: logarithms that are positive, up to sums of 80 over rows that are evaluated together."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from test_gpu_delta import delta_case
from test_gpu_ssm import GUARD


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("n", [1, 15, 60, 64, 150])
def test_logarithms_above_zero(n, dtype):
    """Little by little and back, at once and back, steps up and down, next to none"""
    def grow(x, rates, biases, S):
        g = x[3][GUARD:GUARD + n]
        rows = np.arange(n)
        g[:, 0] = np.where(rows % 128 < 64, 1.25, -1.25)
        g[:, 1] = np.where(rows % 64 == 10, 40, np.where(rows % 64 == 50, -45, 0.125))
        g[:, 2] = np.where(rows % 2 == 0, 35, -36)
        g[:, 3] = 0.01
    delta_case(4, 2, 64, 32, [n], dtype, softplus=0, A=False, bias=False, change=grow)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_single_tokens_above_zero(dtype):
    def grow(x, rates, biases, S):
        x[3][:] = np.array([0.01, 5, 40, 80])
    delta_case(4, 2, 64, 32, [1] * 3, dtype, one=True, softplus=0, A=False, bias=False, change=grow)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("n", [12, 100])
def test_rates_above_zero(n, dtype):
    def grow(x, rates, biases, S):
        rates[:] = np.abs(rates) * np.float32(0.05)
        biases[:] = -1
    delta_case(4, 2, 64, 32, [n], dtype, change=grow)

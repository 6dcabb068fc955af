"""The gated delta rule with values and states near the ends of fp32, and of both ends in one call."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from test_gpu_delta import delta_case
from test_gpu_ssm import GUARD


@pytest.mark.parametrize("log", [None, -np.inf, -85, -70])
@pytest.mark.parametrize("value,state", [(1e36, 1e36), (1e36, 1e-30), (1e-12, 1e30), (1e-30, 1e30), (1e-30, 1e36), (1e-30, 1e-30), (1, 1e36)])
@pytest.mark.parametrize("n", [3, 100])
def test_values_and_states(n, value, state, log):
    """A state that is kept, or (nearly) forgotten by the first row"""
    def far(x, rates, biases, S):
        x[3][:] = 0
        if log is not None:
            x[3][GUARD] = log
        x[2] *= np.float32(value)
        S *= np.float32(state)
    delta_case(2, 1, 64, 32, [n], "f32", softplus=0, A=False, bias=False, change=far)


@pytest.mark.parametrize("log", [-np.inf, -85, -70])
@pytest.mark.parametrize("n", [3, 100])
def test_a_large_state_that_small_values_of_binary16_replace(n, log):
    def far(x, rates, biases, S):
        x[3][:] = 0
        x[3][GUARD] = log
        x[2][:] = np.asarray(x[2], np.float64) * 2.0 ** -10
        S *= np.float32(1e36)
    delta_case(2, 2, 128, 32, [n], "f16", softplus=0, A=False, bias=False, change=far)

"""The gated delta rule where rows that are evaluated together are far apart: a value, a state or a growing decay many orders of magnitude above the
rows beside it, which forget it or stand ahead of it.  Each row is held to what its own terms allow (see delta64), whatever its neighbours are."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from test_gpu_delta import delta_case
from test_gpu_ssm import GUARD

AT = 20  # the row that is far from the others


def keep_all(x, but=()):
    """Logarithms of decays: nothing is forgotten but at the rows of `but`"""
    x[3][:] = 0
    for row, log in but:
        x[3][GUARD + row] = log


def values(x, size, dv, t):
    """Every third column has a value that is `size` times the others' at row AT; in binary16 the others are smaller instead"""
    if t == "f16":
        x[2][:] = np.asarray(x[2], np.float64) * 2.0 ** -8
        x[2][GUARD + AT, ::3] = min(size * 2.0 ** -8, 6e4)
    else:
        x[2][GUARD + AT, ::3] *= np.float32(size)


SHAPES = [(2, 2, 32, 32), (2, 1, 128, 48), (2, 1, 200, 33)]


@pytest.mark.parametrize("dtype,size", [("f16", 1e5), ("f16", 1e9), ("f32", 1e5), ("f32", 1e9), ("f32", 1e12), ("f32", 1e30)])
@pytest.mark.parametrize("log", [-np.inf, -40, -22, -12, 0])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_value_far_above_the_rows_around_it(shape, log, dtype, size):
    """Rows ahead of it and, as far as it is forgotten, behind it"""
    def far(x, rates, biases, S):
        keep_all(x, [(AT + 1, log)])
        values(x, size, shape[3], dtype)
    delta_case(*shape, [100], dtype, softplus=0, A=False, bias=False, change=far)


@pytest.mark.parametrize("dtype,size", [("f16", 1e9), ("f32", 1e12)])
@pytest.mark.parametrize("at", [0, 1, 3, 15, 16, 63])
def test_rows_of_every_place(at, dtype, size):
    """The far value in other rows of a chunk and in the last, short one, of two prompts; states in place"""
    shape = (2, 1, 64, 32)

    def far(x, rates, biases, S):
        keep_all(x, [(at + 1, -np.inf), (70, -25), (at + 101, -np.inf)])
        x[2][:] = np.asarray(x[2], np.float64) * 2.0 ** -8
        for row in (at, 69, 100 + at):
            x[2][GUARD + row, 1::4] = min(size * 2.0 ** -8, 6e4) if dtype == "f16" else size
    delta_case(*shape, [100, 150], dtype, softplus=0, A=False, bias=False, change=far, in_place=True)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("size", [1e6, 1e12, 1e25])
@pytest.mark.parametrize("row,log", [(0, -np.inf), (1, -np.inf), (37, -np.inf), (9, -30), (66, -np.inf)])
def test_a_state_far_above_the_rows_that_forget_it(row, log, size, dtype):
    def far(x, rates, biases, S):
        keep_all(x, [(row, log)])
        S[..., 1::3] *= np.float32(size)
    delta_case(2, 2, 64, 32, [100], dtype, softplus=0, A=False, bias=False, change=far)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_rows_of_nothing_behind_a_far_value(dtype):
    """What is left of it is all that they give"""
    def far(x, rates, biases, S):
        keep_all(x, [(AT + 1, -25), (AT + 9, -3)])
        x[2][GUARD + AT + 1:] = 0
        S[:] = 0
    delta_case(2, 2, 64, 32, [90], dtype, softplus=0, A=False, bias=False, change=far)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_a_prompt_from_nothing_whose_first_values_are_tiny(dtype):
    def far(x, rates, biases, S):
        S[:] = 0
        x[2][:GUARD + 3] = np.asarray(x[2][:GUARD + 3], np.float64) * 2.0 ** -12
        x[2][GUARD + 3:GUARD + 5] = 0
    delta_case(2, 1, 128, 64, [130], dtype, change=far)


@pytest.mark.parametrize("dtype,by", [("f16", 2.0 ** -10), ("f32", 2.0 ** -24)])
@pytest.mark.parametrize("turned", [False, True])
def test_keys_as_they_are_whose_lengths_are_far_apart(dtype, by, turned):
    """Every other one short; with values that are as much larger, too"""
    def far(x, rates, biases, S):
        x[1] *= np.asarray(0.08, x[1].dtype)
        x[1][::2] *= np.asarray(by, x[1].dtype)
        if turned:
            x[2][::2] *= np.asarray(1 / by, x[2].dtype)
    delta_case(2, 1, 64, 32, [100, 3], dtype, norm=False, change=far)


@pytest.mark.parametrize("name", ["dt", "k", "v", None])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("above", [25, 28])
def test_what_is_not_finite_in_a_chunk_whose_state_is_far_below_its_bound(above, dtype, name):
    """A value far above the others is forgotten: the next 64 rows' state is far below what it might have been.  One of them is not finite"""
    shape, row = (4, 2, 64, 32), 90  # the last head

    def far(x, rates, biases, S):
        keep_all(x, [(AT + 1, -np.inf)])
        size = 2.0 ** -14 if dtype == "f16" else 1.0
        x[2][:] = np.sign(np.asarray(x[2], np.float64) + 1e-30) * size
        x[2][GUARD + AT] *= np.float32(2.0 ** above)
        x[4][:] = 9
        S[:] = 0

    def spoil(x, rates, biases, S):
        far(x, rates, biases, S)
        if name == "dt":
            x[3][GUARD + row, 3] = np.nan
        elif name == "k":
            x[1][GUARD + row, 64 + 5] = np.inf  # of heads 2 and 3
        else:
            x[2][GUARD + row, 3 * 32 + 7] = np.nan
    run = dict(dtype=dtype, softplus=0, A=False, bias=False)
    if name is None:
        delta_case(*shape, [150], change=far, **run)
        return

    def look(y, left, starts, x, S0):
        return y[starts[0]:starts[1]].reshape(150, 4, 32).astype(np.float32), left[0]
    (clean, want), (y, S) = (delta_case(*shape, [150], change=c, check=look, **run) for c in (far, spoil))
    ybad, Sbad = np.zeros(y.shape, bool), np.zeros(S.shape, bool)
    if name == "dt":
        ybad[row:, 3] = Sbad[3] = True
    elif name == "k":
        ybad[row:, 2:] = Sbad[2:] = True
    else:
        ybad[row:, 3, 7] = Sbad[3, :, 7] = True
    assert np.isfinite(clean).all() and np.array_equal(y[~ybad], clean[~ybad]) and np.array_equal(S[~Sbad], want[~Sbad])
    assert not np.isfinite(y[ybad]).any() and not np.isfinite(S[Sbad]).any()


@pytest.mark.parametrize("log", [-np.inf, -22, -18, -15])
@pytest.mark.parametrize("dtype,above", [("f16", 26), ("f32", 24), ("f32", 28), ("f32", 40)])
def test_many_far_values_that_are_forgotten_together(dtype, above, log):
    """As many as there are ahead of the rows that forget them: each may show in those"""
    def far(x, rates, biases, S):
        keep_all(x, [(40, log)])
        x[2][:] = np.asarray(x[2], np.float64) * (2.0 ** -12 if dtype == "f16" else 1)
        x[2][GUARD:GUARD + 40] = np.clip(np.asarray(x[2][GUARD:GUARD + 40], np.float64) * 2.0 ** above, -6e4, 6e4) if dtype == "f16" else x[2][GUARD:GUARD + 40] * np.float32(2.0 ** above)
        S[:] = 0
    delta_case(2, 2, 64, 32, [100], dtype, softplus=0, A=False, bias=False, change=far)

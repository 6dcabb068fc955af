"""Calls of the gated delta rule some of whose prompts go token by token and others, beside them, 64 rows at once."""
import pytest

pytestmark = pytest.mark.gpu

from test_gpu_delta import delta_case

MIXED = [5, 300, 0, 17, 30, 64, 3, 41, 42]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("size", [(32, 16, 16, 128), (64, 64, 17, 70)])
def test_short_prompts_beside_long_ones(size, dtype, in_place):
    """Heads of 128 columns of 32: 256 workgroups a prompt by chunks, so that long prompts are more than the compute units take at once and short
    ones do not join them"""
    delta_case(*size, MIXED, dtype, in_place=in_place, pad=(0, 0, 1, 0, 1, 3))


@pytest.mark.parametrize("in_place", [False, True])
def test_more_of_them_than_a_launch_holds(in_place):
    lens = [(i * 7) % 90 if i % 3 == 0 else i % 6 for i in range(150)]
    delta_case(8, 8, 16, 16, lens, in_place=in_place)


def test_one_of_forty_rows_beside_longer_ones():
    delta_case(32, 32, 16, 128, [40, 130, 22, 64, 100])

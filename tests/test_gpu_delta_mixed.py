"""Calls of the gated delta rule some of whose prompts go token by token and others, beside them, 64 rows at once."""
import pytest

pytestmark = pytest.mark.gpu

from test_gpu_delta import delta_case

MIXED = [5, 300, 0, 17, 30, 64, 3, 41, 42]


@pytest.mark.parametrize("dtype,in_place", [("f16", False), ("f16", True), ("f32", True)])
@pytest.mark.parametrize("size", [(16, 16, 16, 112), (16, 8, 17, 100)])
def test_short_prompts_beside_long_ones(size, dtype, in_place):
    """112 workgroups a prompt by chunks: long prompts are more than the compute units take at once, and short ones do not join them"""
    delta_case(*size, MIXED, dtype, in_place=in_place, pad=(0, 0, 1, 0, 1, 3))


def test_more_of_them_than_a_launch_holds():
    delta_case(8, 8, 16, 16, [(i * 7) % 90 if i % 3 == 0 else i % 6 for i in range(150)], in_place=True)

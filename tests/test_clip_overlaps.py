"""What the gradients' norm and clipping refuse of memory that is shared, on the host and before any launch."""
from __future__ import annotations

import pytest

from tests.test_fp8_arguments import _clip, _lib, _refused

MB = 1 << 20
# 4 x 100 values of 4 bytes, and 3 x 50 of rows 80 apart
APART = ((1 * MB, 5 * MB, 4, 100, 100), (2 * MB, 6 * MB, 3, 50, 80))
IN_PLACE = ((1 * MB, 1 * MB, 4, 100, 100), (2 * MB, 2 * MB, 3, 50, 80))
NORM_ALONE = ((1 * MB, None, 4, 100, 100), (2 * MB, None, 3, 50, 80))


@pytest.mark.parametrize("tensors", [APART, IN_PLACE, NORM_ALONE], ids=["apart", "in_place", "norm_alone"])
@pytest.mark.parametrize("at", [1 * MB, 1 * MB + 1596, 2 * MB + 4 * 180])
def test_the_norm_on_a_gradient(tensors, at):
    _refused(_clip(*tensors, norm=at, ws=9 * MB), "the norm")
    _refused(_clip(*tensors, norm=8 * MB, ws=at & ~15), "the workspace")


@pytest.mark.parametrize("at", [5 * MB, 6 * MB + 196, 6 * MB + 4 * 160])
def test_the_norm_on_an_output(at):
    _refused(_clip(*APART, norm=at, ws=9 * MB), "the norm")
    _refused(_clip(*APART, norm=8 * MB, ws=at & ~15), "the workspace")


def test_the_norm_on_the_workspace():
    for tensors in (APART, IN_PLACE, NORM_ALONE):
        for norm in (9 * MB, 9 * MB + 4, 9 * MB + 12):  # two sums of 8 bytes
            _refused(_clip(*tensors, norm=norm, ws=9 * MB), "overlaps")
    _refused(_clip(*APART, norm=8 * MB + 2, ws=9 * MB), "misaligned norm")


@pytest.mark.parametrize("again", [1 * MB, 1 * MB + 4, 1 * MB + 1596, 1 * MB - 1596])
def test_a_gradient_given_twice(again):
    """With outputs of their own too: a value would count twice."""
    _refused(_clip((1 * MB, 5 * MB, 4, 100, 100), (again, 6 * MB, 4, 100, 100), norm=8 * MB, ws=9 * MB), "overlaps")
    _refused(_clip((1 * MB, 1 * MB, 4, 100, 100), (again, again, 4, 100, 100), norm=8 * MB, ws=9 * MB), "overlaps")


def test_rows_of_one_gradient_on_another_s():
    """Columns 0 .. 49 and 49 .. 98 of rows 200 apart."""
    a = (1 * MB, 5 * MB, 6, 50, 200)
    _refused(_clip(a, (1 * MB + 49 * 4, 6 * MB, 6, 50, 200), norm=8 * MB, ws=9 * MB), "gradient 0 overlaps gradient 1")

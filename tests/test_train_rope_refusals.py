"""Rotary positions of two tensors whose outputs stand where the other one does: blocks would read what others wrote.  They are
refused before anything is launched."""

import pytest

import n3d
from fake_tensor import FakeTensor


@pytest.mark.parametrize("y0,y1", [(2, 3), (3, 1), (2, 2), (2, 1), (5, 5)])
def test_outputs_in_the_place_of_the_other_tensor(y0, y1):
    at = lambda i: FakeTensor((2, 5, 4, 64), ptr=i << 20)
    x = [at(1), at(2)]
    with pytest.raises(n3d.DiarizationError) as e:
        n3d.rope(n3d.RopePlan(64), x, [at(y0), at(y1)])
    assert e.value.kind == "InvalidArgument" and "stands where" in str(e.value)

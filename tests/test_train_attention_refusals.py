"""Attention calls whose outputs stand where tensors do that are still read: dq in q's place would be read as q by the pass
that takes dk and dv, out in k's place by other blocks.  They are refused before anything is launched."""

import pytest

import n3d
from fake_tensor import FakeTensor

NAMES = ("q", "k", "v", "out", "dout", "dq", "dk", "dv")


def tensors(dtype="float32"):
    return {n: FakeTensor((2, 5, 4, 64), dtype=dtype, ptr=(i + 1) << 20) for i, n in enumerate(NAMES)}


def backward(t):
    lse, space = FakeTensor((2, 4, 5), ptr=20 << 20), FakeTensor((1 << 20,), dtype="uint8", ptr=21 << 20)
    n3d.attention_backward(t["q"], t["k"], t["v"], t["out"], lse, t["dout"], t["dq"], t["dk"], t["dv"], workspace=space)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("out,other", [("dq", "q"), ("dq", "k"), ("dq", "v"), ("dq", "dout"), ("dk", "q"), ("dk", "v"),
                                       ("dk", "out"), ("dk", "dout"), ("dv", "q"), ("dv", "k"), ("dv", "dout"),
                                       ("dq", "dk"), ("dk", "dv"), ("dq", "dv")])
def test_gradients_in_the_place_of_others(dtype, out, other):
    t = tensors(dtype)
    t[out] = t[other]
    with pytest.raises(n3d.DiarizationError) as e:
        backward(t)
    assert e.value.kind == "InvalidArgument" and "stands where" in str(e.value)


@pytest.mark.parametrize("other", ["k", "v"])
def test_the_output_in_the_place_of_keys_or_values(other):
    t = tensors()
    with pytest.raises(n3d.DiarizationError) as e:
        n3d.attention_forward(t["q"], t["k"], t["v"], t[other])
    assert e.value.kind == "InvalidArgument" and "stands where" in str(e.value)

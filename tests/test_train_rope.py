"""Rotary positions (n3d_rope): the plan's frequencies on the CPU, refusals, and on a
B200 the rotation and its transpose against 64-bit arithmetic.

Tolerance, derived: an output is m (a cos - b sin) with fp32 sines, cosines and products
of a phase rounded to 2^-32 of a turn and then to 24 bits.  The phase contributes at most
2 pi (2^-33 + 2^-26) < 1e-7, sincospi 2 ulp = 1.2e-7, the three roundings 3 * 2^-24 =
1.8e-7, each times |a| + |b| <= 2 max|x|: 8e-7 m max|x| for fp32, plus half an ulp of the
output's type."""

import math

import numpy as np
import pytest

import n3d
from fake_tensor import FakeTensor

ULP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}  # half an ulp, relative


def frequencies(n, theta=10000.0, scaling="none", factor=1.0, original=4096, fast=32.0, slow=1.0):
    if scaling == "ntk" and n > 2:
        theta = theta * factor ** (n / (n - 2))
    f = np.array([theta ** (-2.0 * i / n) for i in range(n // 2)])
    if scaling == "linear":
        return f / factor, 1.0
    if scaling != "yarn":
        return f, 1.0
    pair = lambda turns: n * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
    lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), n - 1)
    r = np.clip((np.arange(n // 2) - lo) / max(hi - lo, 1e-3), 0, 1)
    return f * (1 - r) + f / factor * r, 0.1 * math.log(factor) + 1.0


@pytest.mark.parametrize("n,scaling,factor", [(64, "none", 1.0), (64, "linear", 4.0), (128, "ntk", 8.0),
                                              (2, "ntk", 8.0), (64, "yarn", 8.0), (128, "yarn", 40.0), (34, "yarn", 2.0)])
def test_plan_frequencies(n, scaling, factor):
    plan = n3d.RopePlan(head_dim=128, rotary_dim=n, scaling=scaling, factor=factor)
    f, m = frequencies(n, scaling=scaling, factor=factor)
    got = np.array([t / 2.0 ** 64 for t in plan.turns]) * 2 * math.pi
    # 2^-62 of a turn of resolution, and pow's and exp's last bits
    np.testing.assert_allclose(got, f, rtol=1e-14, atol=2.0 ** -59)
    assert plan.attention_factor == np.float32(m)
    assert n3d.RopePlan(head_dim=128, rotary_dim=n, scaling=scaling, factor=factor,
                        attention_factor=0.5).attention_factor == 0.5


def test_yarn_keeps_fast_pairs_and_stretches_slow_ones():
    plain, yarn = n3d.RopePlan(64).turns, n3d.RopePlan(64, scaling="yarn", factor=16.0).turns
    assert yarn[0] == plain[0] and abs(yarn[-1] * 16 - plain[-1]) <= 64


@pytest.mark.parametrize("kw", [dict(head_dim=64, rotary_dim=63), dict(head_dim=64, rotary_dim=66),
                                dict(head_dim=64, rotary_dim=0), dict(head_dim=300), dict(head_dim=0),
                                dict(head_dim=64, theta=1.0), dict(head_dim=64, theta=math.nan),
                                dict(head_dim=64, scaling="linear", factor=0.5),
                                dict(head_dim=64, scaling="yarn", factor=math.inf),
                                dict(head_dim=64, scaling="yarn", factor=2.0, beta_fast=0.5),
                                dict(head_dim=64, scaling="yarn", factor=2.0, original_length=0),
                                dict(head_dim=64, attention_factor=math.inf), dict(head_dim=64, layout="other"),
                                dict(head_dim=64, scaling="other")])
def test_plan_refusals(kw):
    with pytest.raises(n3d.DiarizationError) as e:
        n3d.RopePlan(**kw)
    assert e.value.kind == "InvalidArgument"


@pytest.mark.parametrize("x,y", [
    (FakeTensor((2, 3, 4, 64)), FakeTensor((2, 3, 4, 64), (0, 256, 64, 1))),            # outputs of two sequences overlap
    (FakeTensor((2, 3, 4, 64)), FakeTensor((2, 3, 4, 64), (768, 256, 32, 1))),          # heads overlap
    (FakeTensor((2, 3, 4, 64), (768, 256, -64, 1)), FakeTensor((2, 3, 4, 64))),         # negative stride
    (FakeTensor((2, 3, 4, 64), (1 << 61, 256, 64, 1)), FakeTensor((2, 3, 4, 64))),      # offsets beyond 2^60
    (FakeTensor((2, 3, 4, 64)), FakeTensor((2, 3, 4, 64), (768, 64, 192, 1))),          # in place, other strides
    (FakeTensor((2, 3, 4, 64), ptr=(1 << 20) + 2), FakeTensor((2, 3, 4, 64))),          # not aligned to its type
    (FakeTensor((2, 3, 4, 64)), FakeTensor((2, 3, 2, 64))),                             # another shape
    (FakeTensor((2, 3, 4, 64)), FakeTensor((2, 3, 4, 64), dtype="float16")),            # another type
    (FakeTensor((2, 3, 4, 64), dtype="float64"), FakeTensor((2, 3, 4, 64), dtype="float64")),
    (FakeTensor((2, 3, 4, 32)), FakeTensor((2, 3, 4, 32))),                             # not the plan's head_dim
    (FakeTensor((2, 3, 4, 64), (1536, 512, 128, 2)), FakeTensor((2, 3, 4, 64))),        # elements not consecutive
])
def test_rope_refusals(x, y):
    with pytest.raises(n3d.DiarizationError) as e:
        n3d.rope(n3d.RopePlan(64), [x], [y])
    assert e.value.kind == "InvalidArgument"


def test_rope_refuses_null_and_counts():
    L = n3d.lib()
    assert n3d.STATUS[L.n3d_rope(0, None, 0, 1, 1, 1, None, None, None, 0, 0, None)] == "InvalidArgument"
    t = FakeTensor((1, 1, 1, 64))
    for xs in ([], [t, t, t]):
        with pytest.raises(n3d.DiarizationError):
            n3d.rope(n3d.RopePlan(64), xs, xs)
    with pytest.raises(n3d.DiarizationError):  # positions of another count
        n3d.rope(n3d.RopePlan(64), [t], [t], positions=FakeTensor((2,), dtype="int32"))


def reference(x, positions, n, layout, scaling, factor, transpose):
    f, m = frequencies(n, scaling=scaling, factor=factor)
    a = positions.astype(np.float64)[..., None] * f
    cos, sin = m * np.cos(a)[:, :, None], m * np.sin(a)[:, :, None] * (-1 if transpose else 1)
    y = x.astype(np.float64).copy()
    u, v = (slice(0, n // 2), slice(n // 2, n)) if layout == "half" else (slice(0, n, 2), slice(1, n, 2))
    p, q = y[..., u].copy(), y[..., v].copy()
    y[..., u], y[..., v] = p * cos - q * sin, q * cos + p * sin
    return y, m


CASES = [
    # seqs, rows, q heads, k heads, head_dim, rotary_dim, layout, scaling, dtype
    (1, 1, 1, 1, 64, 64, "half", "none", "float32"),
    (3, 37, 8, 8, 64, 64, "half", "none", "bfloat16"),
    (2, 5, 8, 2, 128, 64, "interleaved", "yarn", "float16"),
    (2, 19, 3, 1, 64, 34, "half", "ntk", "float16"),            # 17 pairs: no whole words
    (2, 19, 3, 1, 64, 18, "interleaved", "linear", "float32"),  # 18 elements: no whole words
    (1, 70, 4, 4, 128, 128, "interleaved", "none", "bfloat16"),
    (1, 33, 2, 2, 256, 256, "half", "none", "bfloat16"),
    (2, 9, 2, 1, 6, 2, "half", "ntk", "float32"),
    (40, 500, 8, 8, 64, 32, "half", "none", "bfloat16"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,rows,qh,kh,hd,n,layout,scaling,dtype", CASES)
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("packed", [False, True])
def test_rope_matches_64_bits(seqs, rows, qh, kh, hd, n, layout, scaling, dtype, transpose, packed):
    import torch

    dt = getattr(torch, dtype)
    g = torch.Generator().manual_seed(seqs * 1000 + rows)
    xs = [torch.randn(seqs, rows, h, hd, generator=g).to(dt).cuda() for h in (qh, kh)]
    pos = torch.randint(-1000, 1 << 24, (seqs, rows), generator=g, dtype=torch.int32)
    if packed:  # q and k in one buffer with values behind them, rotated in place
        buf = torch.cat(xs + [xs[1]], 2).contiguous()
        xs = list(buf.split([qh, kh, kh], 2)[:2])
        keep = buf[:, :, qh + kh:].clone()
    before = [x.float().cpu().numpy() for x in xs]
    ys = xs if packed else [torch.full_like(x, math.nan) for x in xs]
    plan = n3d.RopePlan(hd, n, layout, scaling=scaling, factor=4.0)
    n3d.rope(plan, xs, ys, positions=pos.cuda(), transpose=transpose, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    n3d.train_status(0)
    for x, y in zip(before, ys):
        want, m = reference(x, pos.numpy(), n, layout, scaling, 4.0, transpose)
        got = y.float().cpu().numpy()
        np.testing.assert_array_less(np.abs(got - want), 8e-7 * m * np.abs(x).max() + np.abs(want) * 1.001 * ULP[dtype]
                                     + (2.0 ** -25 if dtype == "float16" else 1e-37))
    if packed:
        assert torch.equal(buf[:, :, qh + kh:], keep)


@pytest.mark.gpu
def test_rope_rows_count_from_the_first_position_and_transpose_undoes_it():
    import torch

    x = torch.randn(2, 300, 4, 64, device="cuda")
    y, back, other = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    plan = n3d.RopePlan(64)
    n3d.rope(plan, [x], [y], first_position=(1 << 40) + 12)
    n3d.rope(plan, [y], [back], first_position=(1 << 40) + 12, transpose=True)
    torch.cuda.synchronize()
    # two rotations, each within 8e-7 max|x|; the second acts on values up to sqrt 2 larger
    assert (back - x).abs().max() <= 2 * 8e-7 * 1.5 * x.abs().max()
    pos = torch.arange(12, 312, dtype=torch.int32, device="cuda").repeat(2, 1)
    n3d.rope(plan, [x], [y], first_position=12)
    n3d.rope(plan, [x], [other], positions=pos)
    torch.cuda.synchronize()
    assert torch.equal(y, other)


@pytest.mark.gpu
def test_rope_unaligned_and_transposed_strides_agree_with_the_wide_path():
    import torch

    x = torch.randn(2, 21, 3, 64, device="cuda").to(torch.bfloat16)
    plan = n3d.RopePlan(64)
    want = torch.empty_like(x)
    n3d.rope(plan, [x], [want])
    odd = torch.empty(2 * 21 * 3 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 21, 3, 64)
    odd.copy_(x)
    heads_first = torch.empty(2, 3, 21, 64, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    n3d.rope(plan, [odd], [heads_first])
    broadcast = torch.empty_like(x)
    n3d.rope(plan, [x[:1].expand(2, -1, -1, -1)], [broadcast])
    torch.cuda.synchronize()
    # the same operations on the same values, whatever the width of the loads
    assert torch.equal(heads_first, want)
    assert torch.equal(broadcast[0], want[0]) and torch.equal(broadcast[1], want[0])


@pytest.mark.gpu
def test_rope_runs_on_the_callers_stream_and_in_a_graph():
    import torch

    x = torch.randn(1, 64, 8, 64, device="cuda")
    y, want = torch.empty_like(x), torch.empty_like(x)
    plan = n3d.RopePlan(64)
    n3d.rope(plan, [x], [want])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        n3d.rope(plan, [x], [y], stream=torch.cuda.current_stream().cuda_stream)
    y.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)


@pytest.mark.gpu
def test_rope_of_nothing():
    import torch

    x = torch.empty(0, 5, 2, 64, device="cuda")
    n3d.rope(n3d.RopePlan(64), [x], [x])
    x = torch.empty(3, 0, 2, 64, device="cuda")
    n3d.rope(n3d.RopePlan(64), [x], [x])
    torch.cuda.synchronize()

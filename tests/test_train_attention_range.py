"""Attention with its gradient on values far from 1 (n3d_attention_forward, n3d_attention_backward), against 64
bits within the bounds derived in test_train_attention.py."""

import numpy as np
import pytest

import n3d
from test_train_attention import E, TYPES, run, seen64


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("std", [1e-20, 1e-30])
def test_tiny_queries_and_keys_attend_evenly(dtype, hd, std):
    run(1, 130, 200, 2, 1, hd, dtype, std=std, seed=31)
    run(2, 130, 200, 1, 1, hd, dtype, -1, 0, 70, std=std, ragged=True, seed=32)
    run(1, 40, 50, 1, 1, hd, dtype, 5, 3, 0, std=std, seed=33)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_the_largest_limits_are_limits(dtype, hd):
    """left and right of 2^30 with an offset as far: causal attention, its mirror, and no key at all."""
    far = 1 << 30
    run(1, 90, 100, 1, 1, hd, dtype, -1, far, -far, seed=34)
    run(1, 90, 100, 1, 1, hd, dtype, far, -1, far, seed=35)
    run(1, 90, 100, 1, 1, hd, dtype, far, far, 0, seed=36)
    run(1, 90, 100, 1, 1, hd, dtype, far - 1, 0, far, seed=37)


# -------------------------------------------------- fp32: rows, heads and sequences of very different sizes
def head64_by_row(q, k, v, do, seen, scale):
    """One head in 64 bits, and a bound for each row of each output (largest element) that knows only what the row
    itself is made of.  With e = 2^-24, a_ij = scale sum_d |q_id k_jd| and x_j the largest |x| of row j: a score is off by
    16 e a_ij (operands of 22 bits, fp32 sums), its exponent is rounded with the row's statistics, so p_ij is off by
    d_ij = 16 e (a_ij + mean a_i + |lse_i| + 2), relatively.  The weights of a row keep 2^-31 of the largest, which
    16 e of the sum of magnitudes covers for the few hundred columns here."""
    s = np.where(seen, q @ k.T * scale, -np.inf)
    top = s.max(1, keepdims=True, initial=-np.inf)
    top = np.where(np.isfinite(top), top, 0.0)
    with np.errstate(divide="ignore"):
        lse = top + np.log(np.exp(s - top).sum(1, keepdims=True))
    base = np.where(np.isfinite(lse), lse, 0.0)
    p = np.where(seen, np.exp(s - base), 0.0)
    a = abs(scale) * (np.abs(q) @ np.abs(k).T)
    d = 16 * E * (a + (p * a).sum(1, keepdims=True) + np.abs(base) + 2)
    size = lambda t: np.abs(t).max(1)
    out = p @ v
    e_out = (p * (d + 16 * E)) @ size(v)
    dot, dp = (do * out).sum(1, keepdims=True), do @ v.T
    e_dot = np.abs(do).sum(1) * e_out + 16 * E * np.abs(do * out).sum(1)
    ds = p * (dp - dot)
    e_ds = p * ((d + 32 * E) * np.abs(dp - dot) + e_dot[:, None] + 16 * E * (np.abs(do) @ np.abs(v).T))
    val = dict(out=out, lse=lse[:, 0], dq=scale * (ds @ k), dk=scale * (ds.T @ q), dv=p.T @ do)
    err = dict(out=e_out, lse=16 * E * ((p * a).sum(1) + np.abs(base[:, 0]) + 2), dq=abs(scale) * (e_ds @ size(k)),
               dk=abs(scale) * (e_ds.T @ size(q)), dv=(p * (d + 16 * E)).T @ size(do))
    return val, err


def run_by_row(q, k, v, do, left=-1, right=-1, off=0):
    """Forward and backward on the GPU in fp32, every row within its own bound; returns the outputs."""
    import torch

    (b, nq, hq, hd), (_, nk, hk, _) = q.shape, k.shape
    t = [x.float().cuda().contiguous() for x in (q, k, v, do)]
    out, dq, dk, dv = (torch.full_like(x, np.nan) for x in (t[0], t[0], t[1], t[1]))
    lse = torch.full((b, hq, nq), np.nan, device="cuda")
    space = torch.full((n3d.attention_workspace(t[0], t[1]),), 255, dtype=torch.uint8, device="cuda")
    kw = dict(left=left, right=right, q_offset=off, workspace=space)
    n3d.attention_forward(*t[:3], out, lse, **kw)
    n3d.attention_backward(*t[:3], out, lse, t[3], dq, dk, dv, **kw)
    torch.cuda.synchronize()
    n3d.train_status(0)
    got = dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv)
    host = [x.double().cpu().numpy() for x in t]
    seen = seen64(nq, nk, nq, nk, left, right, off)
    for s in range(b):
        for g in range(hk):
            sums = {n: [np.zeros((nk, hd)), np.zeros(nk)] for n in ("dk", "dv")}
            for h in range(g * (hq // hk), (g + 1) * (hq // hk)):
                val, err = head64_by_row(host[0][s, :, h], host[1][s, :, g], host[2][s, :, g], host[3][s, :, h], seen,
                                         hd ** -0.5)
                for n in ("out", "dq", "lse"):
                    x = got[n][s, h] if n == "lse" else got[n][s, :, h]
                    within(x, val[n], err[n], (n, s, h))
                for n in ("dk", "dv"):
                    sums[n][0] += val[n]
                    sums[n][1] += err[n]
            for n in ("dk", "dv"):
                within(got[n][s, :, g], *sums[n], (n, s, g))
    return got


def within(x, want, err, what):
    x = x.double().cpu().numpy()
    assert np.array_equal(np.isneginf(x), np.isneginf(want)), what
    off = np.abs(np.where(np.isneginf(want), 0.0, x - np.where(np.isneginf(want), 0.0, want)))
    off = off.max(1) if off.ndim == 2 else off
    worst = (off / (err + 1e-37)).max()
    assert worst <= 1.0, (what, worst)


def normal(seed, *shape):
    import torch

    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


SIZES = [1.0, 1e-3, 1e-6, 1e-9, 1e6]


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("which", ["v", "dout", "q", "k", "v and dout"])
@pytest.mark.parametrize("by", ["sequence", "head", "row"])
def test_fp32_sizes_that_differ(hd, which, by):
    import torch

    b, n, h = len(SIZES), 130, len(SIZES)
    if by != "sequence":
        b = 1
    if by != "head":
        h = 2
    t = dict(q=normal(41, b, n, h, hd), k=normal(42, b, n, h, hd), v=normal(43, b, n, h, hd), dout=normal(44, b, n, h, hd))
    f = torch.tensor(SIZES, dtype=torch.float64)
    f = {"sequence": f.view(-1, 1, 1, 1), "head": f.view(1, 1, -1, 1), "row": f.repeat(n)[:n].view(1, n, 1, 1)}[by]
    for name in which.split(" and "):
        # (rows of q and k of 1e6 would make scores whose rounding leaves nothing to compare: 1e6 becomes 1)
        t[name] = t[name] * (f.clamp(max=1.0) if name in "qk" else f)
    run_by_row(*t.values())
    run_by_row(*t.values(), right=0)  # causal: rows that do not see the large ones


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("n", [150, 333])
def test_fp32_one_row_a_billion_times_the_others(hd, which, n):
    """Rows that a window keeps apart from it are as good as without it."""
    t = dict(q=normal(51, 2, n, 2, hd), k=normal(52, 2, n, 1, hd), v=normal(53, 2, n, 1, hd), dout=normal(54, 2, n, 2, hd))
    t[which][0, n // 2 + 7] *= 1e9
    run_by_row(*t.values(), right=0)
    run_by_row(*t.values(), left=20, right=5)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("q,k,v,dout", [(1e-12, 1e12, 1.0, 1.0), (1.0, 1.0, 1e-18, 1e-15), (1.0, 1.0, 1e18, 1e-30),
                                        (1e15, 1e-15, 1e-25, 1e25), (1.0, 1.0, 1.0, 1e-25)])
def test_fp32_sizes_far_from_one(hd, q, k, v, dout):
    run_by_row(normal(61, 1, 140, 2, hd) * q, normal(62, 1, 200, 1, hd) * k, normal(63, 1, 200, 1, hd) * v,
               normal(64, 1, 140, 2, hd) * dout)


@pytest.mark.gpu
def test_fp32_weights_that_grow_along_the_row():
    """Later blocks of columns that outweigh the earlier ones by any factor: the accumulators' units change."""
    n = 520
    grow = 10.0 ** (np.arange(n) // 40 * 2.0 - 14)  # 1e-14 .. 1e10, in steps inside blocks
    import torch

    g = torch.from_numpy(grow).view(1, n, 1, 1)
    t = [normal(71 + i, 1, n, 1, 64) for i in range(4)]
    run_by_row(t[0], t[1], t[2] * g, t[3])
    run_by_row(t[0], t[1], t[2], t[3] * g)
    run_by_row(t[0], t[1], t[2] * g.flip(1), t[3] * g.flip(1))
    run_by_row(t[0], t[1] * g.clamp(max=3.0), t[2], t[3])
    run_by_row(t[0] * g.clamp(max=3.0), t[1], t[2], t[3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [60, 200])
@pytest.mark.parametrize("size", [1.0, 1e2, 3e3])
def test_the_largest_of_huge_scores_takes_all(dtype, hd, n, size):
    """Every query is a large multiple of one key's row, the others are small beside it: scores of up to 1e8, of which the
    largest leads by far more than their rounding.  Then P is 1 there and 0 elsewhere, exactly, and out is v's row.  (In
    bf16 a row's weights keep a common factor that is no power of two, and are rounded with it.)"""
    import torch

    dt = getattr(torch, dtype)
    pick = torch.arange(n).flip(0)
    k = torch.sign(normal(91, 1, n, 1, hd))  # rows of the same norm, far from parallel
    q = (k[:, pick] * size).to(dt)
    k = (k * size).to(dt)
    if size == 1.0:  # scores of 8 and 11: scaled to 8e6 and more in the call
        scale = 1e6 * hd ** -0.5
    else:
        scale = hd ** -0.5
    v = normal(92, 1, n, 1, hd).to(dt)
    q, k, v = q.cuda(), k.cuda(), v.cuda()
    out, lse = torch.empty_like(q), torch.empty(1, 1, n, device="cuda")
    space = torch.empty(max(16, n3d.attention_workspace(q, k, False)), dtype=torch.uint8, device="cuda")
    n3d.attention_forward(q, k, v, out, lse, scale=scale, workspace=space)
    torch.cuda.synchronize()
    want = v[:, pick.cuda()].double()
    # fp32: v's row in 22 bits, divided by a sum of 1; 16 bits: one rounding of what the type holds
    assert ((out.double() - want).abs() <= 4 * E * want.abs().amax(3, keepdim=True)).all()
    top = (q.double() * k[:, pick.cuda()].double()).sum(3).transpose(1, 2) * scale
    assert ((lse.double() - top).abs() <= 16 * E * top).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("layout", ["rows", "odd"])
def test_gradients_of_huge_scores_stay_in_bounds(dtype, hd, layout):
    """One query and one key row with a score of about 1e9, whose row statistics are rounded by about 64.  P <= 1 bounds every
    gradient: |dS| <= 2 |dout row| |v row|; and rows of dq that do not see the pair are what they are without it."""
    import torch

    n = 200
    t = [normal(81 + i, 1, n, 1, hd).to(getattr(torch, dtype)) for i in range(4)]
    t[3] *= 0.1
    got = []
    for size in (1.0, 1e4):
        q, k, v, do = (x.clone() for x in t)
        q[0, 150] *= size
        k[0, 70] = q[0, 150]
        if layout == "odd":
            q, k, v, do = (torch.nn.functional.pad(x.cuda().reshape(-1), (1, 0))[1:].view(x.shape) for x in (q, k, v, do))
        q, k, v, do = (x.cuda() for x in (q, k, v, do))
        out, dq, dk, dv = (torch.empty_like(x) for x in (q, q, k, v))
        lse = torch.empty(1, 1, n, device="cuda")
        space = torch.empty(n3d.attention_workspace(q, k), dtype=torch.uint8, device="cuda")
        n3d.attention_forward(q, k, v, out, lse, right=0, workspace=space)
        n3d.attention_backward(q, k, v, out, lse, do, dq, dk, dv, right=0, workspace=space)
        torch.cuda.synchronize()
        got.append((dq, dk, dv))
    norm = lambda x: x.double().norm(dim=3).cpu()
    ds = 2.1 * norm(do).max() * norm(v).max() * hd ** -0.5
    assert norm(dq).max() <= ds * norm(k).sum() and norm(dk).max() <= ds * norm(q).sum()
    assert norm(dv).max() <= 1.1 * norm(do).sum()
    assert torch.equal(got[0][0][:, :70], got[1][0][:, :70])

"""The residual norm's gradient where a slot of threads takes many rows, in pairs, odd ones left over:
every pair of norms, gates in one slot and over several, 16-bit types, and each split of a row over threads.

The gradient kernel makes 148 to 2368 slots; these shapes give each 2 to 5 rows.  A pair of norms that takes one
sum over a row at a time (RMS norm or none before, none behind) must not write that sum's words again while another
warp of the row still reads them, so results are compared bit for bit over many calls.

Tolerances, derived: as in test_train_norm.py, with a column sum of ceil(rows / 148) additions in a thread, up to 8
slots, and 37 + 8 blocks."""

import math

import numpy as np
import pytest

import n3d
from test_train_norm import EPS, backward64, close, forward64, hat64, make

# rows, cols: 64, 128, 512 threads a row; 512 with one row at a time; single elements by 128 and 512 threads
SHAPES = [(3001, 264), (1501, 1024), (751, 4096), (451, 8192), (449, 8191), (450, 1030), (1601, 7)]
TYPES = [("float32", "float32"), ("float32", "bfloat16"), ("float16", "float16"), ("bfloat16", "bfloat16"),
         ("float32", "float16")]
NORMS = ["none", "layer", "rms"]


def gradient(d, post, pre, gate_rows, scale=0.5):
    """One call on the GPU: every output by name."""
    import torch

    rows, cols = d["x"].shape
    outs = {n: torch.full((cols,), math.nan, device="cuda") for n in
            (("dpost_w", "dpost_b") if post != "none" else ()) + (("dpre_w", "dpre_b") if pre != "none" else ())}
    kw = dict(post_w=d["post_w"], post_b=d["post_b"]) if post != "none" else {}
    if pre != "none":
        kw["pre_w"] = d["pre_w"]
    if gate_rows:
        outs["dgate"] = torch.full_like(d["gate"], math.nan)
    space = torch.full((n3d.residual_norm_workspace(rows, cols, gate_rows),), 255, dtype=torch.uint8, device="cuda")
    dx, dblock = torch.full_like(d["x"], math.nan), torch.full_like(d["block"], math.nan)
    n3d.residual_norm_grad(d["block"], d["r"] if pre != "none" else None, d["dy"] if pre != "none" else None, d["dr"], dx,
                           dblock, post=post, pre=pre, eps=EPS, scale=scale, gate=d.get("gate"), gate_rows=gate_rows,
                           workspace=space, **kw, **outs)
    return {"dx": dx, "dblock": dblock, **outs}


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("post", NORMS)
@pytest.mark.parametrize("pre", NORMS)
def test_many_rows_a_slot(rows, cols, post, pre):
    import torch

    n = SHAPES.index((rows, cols)) + 2 * NORMS.index(post) + 3 * NORMS.index(pre)
    rt, bt = TYPES[n % len(TYPES)]
    gate_rows = (0, rows, rows // 7 + 1, 3)[n % 4]
    t, p = make(rows, cols, rt, bt, gate_rows, 7 * rows + n)
    got = gradient({k: v.cuda() for k, v in t.items()}, post, pre, gate_rows)
    torch.cuda.synchronize()
    n3d.train_status(0)
    want, mag = backward64(p, p["r"], p["dy"], p["dr"], post, pre, 0.5, gate_rows)
    for name, v in got.items():
        count = {"dx": 150, "dblock": 300}.get(name, 500 + -(-rows // 148))
        close(v, want[name], mag[name], count, {"dx": rt, "dblock": bt}.get(name, "float32"), (name, rt, bt))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(20000, 512), (20000, 511), (6001, 4096), (3001, 8192)])
@pytest.mark.parametrize("rt,bt", [("float32", "float32"), ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("pre,gated", [("rms", False), ("rms", True), ("none", True)])
def test_one_sum_a_row_repeats_bit_for_bit(rows, cols, rt, bt, pre, gated):
    import torch

    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    d = {n: rnd(rows, cols).to(getattr(torch, rt if n in ("x", "r", "dr") else bt)) for n in ("x", "r", "dr", "block", "dy")}
    d["pre_w"] = 1 + 0.1 * rnd(cols)
    if gated:
        d["gate"] = rnd(1, cols)
    first = gradient(d, "none", pre, rows if gated else 0)
    for _ in range(12):
        for n, v in gradient(d, "none", pre, rows if gated else 0).items():
            assert torch.equal(v, first[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("post,pre", [("none", "rms"), ("rms", "none"), ("none", "none")])
@pytest.mark.parametrize("rows,cols", [(1, 3), (37, 512), (10, 2047), (5, 8192)])
@pytest.mark.parametrize("rt,bt", TYPES)
def test_forward_of_the_plain_pairs(rows, cols, rt, bt, post, pre):
    import torch

    t, p = make(rows, cols, rt, bt, 0, rows + cols)
    d = {n: v.cuda() for n, v in t.items()}
    r, y = torch.full_like(d["x"], math.nan), torch.full_like(d["block"], math.nan)
    kw = dict(post_w=d["post_w"], post_b=d["post_b"]) if post != "none" else {}
    n3d.residual_norm(d["x"], d["block"], r, y if pre != "none" else None, post=post, pre=pre, eps=EPS, scale=0.5,
                      pre_w=d["pre_w"] if pre != "none" else None, pre_b=d["pre_b"] if pre != "none" else None, **kw)
    torch.cuda.synchronize()
    r64, y64 = forward64(p, post, pre, 0.5, 0)
    row = lambda a: np.abs(a).max(1, keepdims=True)
    u = row(p["block"])
    if post != "none":
        u = u / hat64(p["block"], post)[1] * row(p["post_w"][None]) + row(p["post_b"][None])
    mag = row(p["x"]) + 0.5 * u
    close(r, r64, mag, 150, rt, "r")
    if pre != "none":
        h, s = hat64(r64, pre)
        close(y, y64, row(p["pre_w"][None]) * mag / s * (1 + row(h) ** 2) + row(p["pre_b"][None]), 150, bt, "y")


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [512, 7])
@pytest.mark.parametrize("post,pre", [("none", "rms"), ("none", "layer"), ("rms", "none"), ("layer", "none"), ("none", "none")])
def test_weights_of_a_norm_that_is_not_used_are_not_read(cols, post, pre):
    import torch

    t, _ = make(37, cols, "float32", "bfloat16", 0, cols)
    d = {n: v.cuda() for n, v in t.items()}
    bad = torch.full((cols,), math.nan, device="cuda")
    used = {n: d[n] for k, p in ((post, "post"), (pre, "pre")) if k != "none" for n in (p + "_w", p + "_b")}
    unused = {n: bad for k, p in ((post, "post"), (pre, "pre")) if k == "none" for n in (p + "_w", p + "_b")}
    space = torch.empty(n3d.residual_norm_workspace(37, cols), dtype=torch.uint8, device="cuda")
    with_pre = pre != "none"
    got = []
    for extra in ({}, unused):
        kw = dict(post=post, pre=pre, **used, **extra)
        r, y, dx, db = (torch.full_like(d[n], math.nan) for n in ("x", "block", "x", "block"))
        n3d.residual_norm(d["x"], d["block"], r, y if with_pre else None, **kw)
        n3d.residual_norm_grad(d["block"], d["r"] if with_pre else None, d["dy"] if with_pre else None, d["dr"], dx, db,
                               workspace=space, **kw)
        got.append([r, dx, db] + [y] * with_pre)
    for a, b in zip(*got):
        assert torch.equal(a, b) and not a.isnan().any()

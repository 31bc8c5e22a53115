"""The residual add with the norms before and after a block (n3d_residual_norm) and its
gradient: refusals on the CPU, and on a B200 both against the formulas in 64 bits, the
gradient also against differences of the 64-bit forward.

Tolerances, derived: e = 2^-24.  A sum over a row is a chain of at most 32 additions in a
thread and 10 levels of a tree, so each mean is within 42 e of the mean of magnitudes; a
normalised value, the residual and the row part of a gradient go through at most three such
sums and about 20 further roundings: 150 e times the row's largest magnitude of the terms.  A
column sum adds at most 128 rows in a thread, 8 slots, and 37 + 8 blocks, of terms that
are within 150 e: 350 e times the sum of the terms' magnitudes.  Outputs of 16 bits are
rounded once more: half an ulp (2^-8 of bf16, 2^-11 of fp16, whose subnormals end at
2^-24)."""

import math

import numpy as np
import pytest

import n3d
from fake_tensor import FakeTensor

E = 2.0 ** -24
HALF_ULP = {"float32": 0.0, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
EPS = 1e-5


# ------------------------------------------------------------------------- refusals
def _forward(rows=4, cols=64, x=None, block=None, r=None, y=None, **kw):
    t = FakeTensor((rows, cols))
    n3d.residual_norm(x or t, block or t, r or FakeTensor((rows, cols), ptr=1 << 21),
                      y or FakeTensor((rows, cols), ptr=1 << 22), **kw)


@pytest.mark.parametrize("kw", [
    dict(cols=8193), dict(cols=0), dict(eps=0.0), dict(eps=-1.0), dict(eps=math.nan), dict(post="other"),
    dict(x=FakeTensor((4, 64), dtype="bfloat16")),                                   # 16-bit stream, fp32 block
    dict(block=FakeTensor((4, 64), dtype="float64")), dict(block=FakeTensor((4, 65))),
    dict(r=FakeTensor((4, 64), (32, 1))), dict(r=FakeTensor((4, 64), (0, 1))),        # output rows overlap
    dict(r=FakeTensor((4, 64), (128, 2))), dict(x=FakeTensor((4, 64), (-64, 1))),
    dict(r=FakeTensor((4, 64), (128, 1))),                                            # in place, another stride
    dict(r=FakeTensor((4, 64), dtype="float16")),
    dict(gate=FakeTensor((1, 64))),                                                   # gate_rows is missing
    dict(gate=FakeTensor((3, 64)), gate_rows=2), dict(pre_w=FakeTensor((63,))),
    dict(pre_w=FakeTensor((64,), dtype="float16")), dict(x=FakeTensor((4, 64), ptr=(1 << 20) + 2)),
])
def test_forward_refusals(kw):
    with pytest.raises(n3d.DiarizationError) as e:
        _forward(**kw)
    assert e.value.kind == "InvalidArgument"


def _backward(rows=4, cols=64, space=1 << 30, **kw):
    at = iter(range(1 << 20, 1 << 28, 1 << 20))
    a = {n: FakeTensor((rows, cols), ptr=next(at)) for n in ("block", "r", "dy", "dr", "dx", "dblock")}
    a.update(kw)
    work = FakeTensor((space,), dtype="uint8", ptr=a.pop("work_ptr", next(at)))
    n3d.residual_norm_grad(workspace=work, **a)


@pytest.mark.parametrize("kw", [
    dict(space=64), dict(work_ptr=(1 << 20) + 8), dict(pre="none", dr=None), dict(dpost_w=FakeTensor((64,))),
    dict(pre="none", dpre_w=FakeTensor((64,))), dict(dx=FakeTensor((4, 64), (0, 1))),
    dict(gate=FakeTensor((4, 64)), gate_rows=1, dgate=FakeTensor((3, 64))), dict(cols=9000),
    dict(dy=None), dict(dblock=FakeTensor((4, 64), dtype="float16")),
])
def test_gradient_refusals(kw):
    with pytest.raises(n3d.DiarizationError) as e:
        _backward(**kw)
    assert e.value.kind == "InvalidArgument"


def test_null_configuration():
    L = n3d.lib()
    assert n3d.STATUS[L.n3d_residual_norm(0, None, *[None] * 9, None)] == "InvalidArgument"
    cfg = n3d._pack_residual(4, 64, 0, 0, 0, 1, 1e-5, 1e-5, 1.0, 0)
    assert n3d.STATUS[L.n3d_residual_norm(0, cfg, *[None] * 9, None)] == "InvalidArgument"


def test_workspace_sizes():
    assert n3d.residual_norm_workspace(1, 64, 0) > 0
    small, gated = n3d.residual_norm_workspace(100, 512, 0), n3d.residual_norm_workspace(100, 512, 100)
    assert gated > small
    # it stops growing once every slot has rows
    assert n3d.residual_norm_workspace(1 << 20, 512, 1) == n3d.residual_norm_workspace(1 << 30, 512, 1)
    assert n3d.residual_norm_workspace(5, 9000, 0) == 0


# ------------------------------------------------------------------------- 64 bits
def norm64(t, kind, w, b):
    if kind == "none":
        return t
    m = t.mean(1, keepdims=True) if kind == "layer" else 0.0
    h = (t - m) / np.sqrt(((t - m) ** 2).mean(1, keepdims=True) + EPS)
    return h * w + b


def forward64(p, post, pre, scale, gate_rows):
    u = norm64(p["block"], post, p["post_w"], p["post_b"])
    g = np.repeat(p["gate"], gate_rows, 0)[: len(u)] if gate_rows else 1.0
    r = p["x"] + scale * g * u
    return r, norm64(r, pre, p["pre_w"], p["pre_b"])


def hat64(t, kind):
    m = t.mean(1, keepdims=True) if kind == "layer" else 0.0
    s = np.sqrt(((t - m) ** 2).mean(1, keepdims=True) + EPS)
    return (t - m) / s, s


def backward64(p, r, dy, dr, post, pre, scale, gate_rows):
    """Gradients, and for each the magnitude its error bound is relative to."""
    row = lambda t: np.abs(t).max(1, keepdims=True)
    out, mag = {}, {}
    d, big = dr.copy(), row(dr)
    if pre != "none":
        h, s = hat64(r, pre)
        g = dy * p["pre_w"]
        mg = g.mean(1, keepdims=True) if pre == "layer" else 0.0
        d = d + (g - mg - h * (g * h).mean(1, keepdims=True)) / s
        # centring r cancels: its error is relative to r, not to r - mean
        grow = 1 + row(h) ** 2 + row(h) * row(r) / s
        big = big + row(g) / s * grow
        out["dpre_w"], mag["dpre_w"] = (dy * h).sum(0), (np.abs(dy) * (np.abs(h) + row(r) / s)).sum(0)
        out["dpre_b"], mag["dpre_b"] = dy.sum(0), np.abs(dy).sum(0)
    out["dx"], mag["dx"] = d, big
    gate = np.repeat(p["gate"], gate_rows, 0)[: len(d)] if gate_rows else np.ones_like(d)
    if post == "none":
        u, lift, base = p["block"], 1.0, np.abs(p["block"])
    else:
        k, s = hat64(p["block"], post)
        u = k * p["post_w"] + p["post_b"]
        lift = 1 + row(k) ** 2 + row(k) * row(p["block"]) / s
        base = (np.abs(k) + row(p["block"]) / s) * np.abs(p["post_w"]) + np.abs(p["post_b"])
    du = scale * gate * d
    if gate_rows:
        pad = -len(d) % gate_rows
        sums = lambda t: np.pad(t, ((0, pad), (0, 0))).reshape(-1, gate_rows, t.shape[1]).sum(1)
        out["dgate"], mag["dgate"] = sums(scale * d * u), sums(abs(scale) * big * base)
    if post != "none":
        out["dpost_w"], mag["dpost_w"] = (du * k).sum(0), (abs(scale) * np.abs(gate) * big * (np.abs(k) + row(p["block"]) / s)).sum(0)
        out["dpost_b"], mag["dpost_b"] = du.sum(0), (abs(scale) * np.abs(gate) * big).sum(0)
        e = du * p["post_w"]
        me = e.mean(1, keepdims=True) if post == "layer" else 0.0
        out["dblock"] = (e - me - k * (e * k).mean(1, keepdims=True)) / s
        mag["dblock"] = row(abs(scale) * gate * big * p["post_w"]) / s * lift
    else:
        out["dblock"], mag["dblock"] = du, abs(scale) * row(gate) * big
    return out, mag


def make(rows, cols, rt, bt, gate_rows, seed, offset=0.1):
    import torch

    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)
    t = {"x": rnd(rows, cols).to(getattr(torch, rt)), "block": (0.7 * rnd(rows, cols) + offset).to(getattr(torch, bt)),
         "r": rnd(rows, cols).to(getattr(torch, rt)), "dy": (0.1 * rnd(rows, cols)).to(getattr(torch, bt)),
         "dr": (0.1 * rnd(rows, cols)).to(getattr(torch, rt)), "post_w": 1 + 0.1 * rnd(cols), "post_b": 0.1 * rnd(cols),
         "pre_w": 1 + 0.1 * rnd(cols), "pre_b": 0.1 * rnd(cols)}
    if gate_rows:
        t["gate"] = 0.5 + 0.2 * rnd(-(-rows // gate_rows), cols)
    return t, {n: v.double().numpy() for n, v in t.items()}


def close(got, want, magnitude, count, dtype, what):
    got = got.double().cpu().numpy()
    tiny = 2.0 ** -25 if dtype == "float16" else 0.0
    limit = count * E * magnitude + HALF_ULP[dtype] * 1.01 * (np.abs(want) + count * E * magnitude) + tiny + 1e-37
    worst = (np.abs(got - want) / limit).max() if want.size else 0.0
    assert worst <= 1.0, (what, worst)


@pytest.mark.parametrize("post,pre,gate_rows", [("layer", "layer", 3), ("rms", "rms", 1), ("none", "layer", 0),
                                                ("layer", "none", 7), ("rms", "layer", 5)])
def test_the_gradient_formula_against_differences(post, pre, gate_rows):
    """The 64-bit formulas that the kernel is held to, against central differences of the forward."""
    rows, cols, scale = 7, 6, 0.5
    _, p = make(rows, cols, "float32", "float32", gate_rows, 3)
    r, _ = forward64(p, post, pre, scale, gate_rows)
    dy = p["dy"] if pre != "none" else np.zeros_like(r)
    loss = lambda q: sum((a * b).sum() for a, b in zip(forward64(q, post, pre, scale, gate_rows), (p["dr"], dy)))
    got, _ = backward64(p, r, dy, p["dr"], post, pre, scale, gate_rows)
    names = {"dx": "x", "dblock": "block", "dgate": "gate", "dpost_w": "post_w", "dpost_b": "post_b", "dpre_w": "pre_w",
             "dpre_b": "pre_b"}
    for name, grad in got.items():
        src = p[names[name]]
        for i in np.ndindex(src.shape):
            q = {**p, names[name]: src.copy()}
            q[names[name]][i] += 1e-5
            up = loss(q)
            q[names[name]][i] -= 2e-5
            # central differences: h^2 f''' / 6 and 1e-16 |f| / h, both below 1e-8 here
            assert abs((up - loss(q)) / 2e-5 - grad[i]) < 1e-7, (name, i)


SHAPES = [(1, 1), (1, 512), (5, 7), (33, 512), (130, 264), (64, 1024), (19, 1016), (17, 2048), (9, 4096), (3, 8192),
          (11, 8191), (2, 1030)]
KINDS = [("none", "layer", 0), ("layer", "layer", -1), ("rms", "rms", 4), ("layer", "none", 1), ("rms", "layer", 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("rt,bt", [("float32", "float32"), ("float32", "bfloat16"), ("float32", "float16"),
                                   ("bfloat16", "bfloat16"), ("float16", "float16")])
def test_residual_norm_and_its_gradient(rows, cols, rt, bt):
    import torch

    for i, (post, pre, gate_rows) in enumerate(KINDS):
        gate_rows = rows if gate_rows < 0 else gate_rows
        t, p = make(rows, cols, rt, bt, gate_rows, 100 * rows + cols + i)
        d = {n: v.cuda() for n, v in t.items()}
        kw = dict(post=post, pre=pre, eps=EPS, scale=0.5, gate=d.get("gate"), gate_rows=gate_rows, pre_w=d["pre_w"])
        if post != "none":
            kw.update(post_w=d["post_w"], post_b=d["post_b"])
        r, y = torch.full_like(d["x"], math.nan), torch.full_like(d["block"], math.nan)
        n3d.residual_norm(d["x"], d["block"], r, y if pre != "none" else None, pre_b=d["pre_b"], **kw)
        r64, y64 = forward64(p, post, pre, 0.5, gate_rows)
        row = lambda a: np.abs(a).max(1, keepdims=True)
        dev_b = hat64(p["block"], post)[1] if post != "none" else 1.0
        u = (row(p["block"]) / dev_b * row(p["post_w"][None]) + row(p["post_b"][None])) if post != "none" else row(p["block"])
        mag_r = row(p["x"]) + 0.5 * u * (np.abs(p["gate"]).max() if gate_rows else 1.0)
        close(r, r64, mag_r, 150, rt, "r")
        if pre != "none":
            h, s = hat64(r64, pre)
            close(y, y64, row(p["pre_w"][None]) * mag_r / s * (1 + row(h) ** 2) + row(p["pre_b"][None]), 150, bt, "y")

        outs = {n: torch.full((cols,), math.nan, device="cuda") for n in
                (("dpost_w", "dpost_b") if post != "none" else ()) + (("dpre_w", "dpre_b") if pre != "none" else ())}
        if gate_rows:
            outs["dgate"] = torch.full_like(d["gate"], math.nan)
        space = torch.empty(n3d.residual_norm_workspace(rows, cols, gate_rows), dtype=torch.uint8, device="cuda")
        dx, dblock = torch.full_like(d["x"], math.nan), torch.full_like(d["block"], math.nan)
        with_dy = pre != "none"
        n3d.residual_norm_grad(d["block"], d["r"] if with_dy else None, d["dy"] if with_dy else None, d["dr"], dx, dblock,
                               workspace=space, **outs, **kw)
        torch.cuda.synchronize()
        n3d.train_status(0)
        want, mag = backward64(p, p["r"], p["dy"], p["dr"], post, pre, 0.5, gate_rows)
        close(dx, want["dx"], mag["dx"], 150, rt, "dx")
        close(dblock, want["dblock"], mag["dblock"], 300, bt, "dblock")
        for n, v in outs.items():
            close(v, want[n], mag[n], 500, "float32", n)


@pytest.mark.gpu
@pytest.mark.parametrize("gate_rows", [1, 2, 100, 379, 1500, 1501, 5000])
def test_gate_rows_across_slots(gate_rows):
    """More rows than slots: gate rows that lie in one slot, end at a border, or span several."""
    import torch

    rows, cols = 3001, 512
    t, p = make(rows, cols, "float32", "float32", min(gate_rows, rows), 5)
    d = {n: v.cuda() for n, v in t.items()}
    got = []
    for _ in range(2):
        outs = {n: torch.full((cols,), math.nan, device="cuda") for n in ("dpost_w", "dpost_b", "dpre_w", "dpre_b")}
        outs["dgate"] = torch.full_like(d["gate"], math.nan)
        space = torch.full((n3d.residual_norm_workspace(rows, cols, gate_rows),), 255, dtype=torch.uint8, device="cuda")
        dx, dblock = torch.empty_like(d["x"]), torch.empty_like(d["block"])
        n3d.residual_norm_grad(d["block"], d["r"], d["dy"], d["dr"], dx, dblock, post="layer", pre="rms", scale=0.5,
                               gate=d["gate"], gate_rows=gate_rows, pre_w=d["pre_w"], post_w=d["post_w"],
                               post_b=d["post_b"], workspace=space, **outs)
        got.append({"dx": dx, "dblock": dblock, **outs})
    want, mag = backward64(p, p["r"], p["dy"], p["dr"], "layer", "rms", 0.5, min(gate_rows, rows))
    for n, v in got[0].items():
        close(v, want[n], mag[n], {"dx": 150, "dblock": 300}.get(n, 500), "float32", n)
        assert torch.equal(v, got[1][n])  # sums in a fixed order


@pytest.mark.gpu
def test_strides_in_place_and_null_weights():
    import torch

    t, p = make(37, 512, "float32", "bfloat16", 0, 8)
    d = {n: v.cuda() for n, v in t.items()}
    ones, zeros = torch.ones(512, device="cuda"), torch.zeros(512, device="cuda")
    r, y = torch.empty_like(d["x"]), torch.empty_like(d["block"])
    n3d.residual_norm(d["x"], d["block"], r, y, post="layer", post_w=ones, post_b=zeros, pre_w=ones, pre_b=zeros)
    # a view with wide rows that starts at an odd element: single elements, the same row sums up to their order
    wide = torch.empty(37, 1030, device="cuda")
    x2 = wide[:, 3:515]
    x2.copy_(d["x"])
    blk2 = d["block"].clone()
    n3d.residual_norm(x2, blk2, x2, blk2, post="layer")
    torch.cuda.synchronize()
    u = p["block"] - p["block"].mean(1, keepdims=True)
    mag = np.abs(p["x"]).max() + 6 * np.abs(u).max()
    assert (x2 - r).abs().max().item() <= 2 * 150 * E * mag
    assert (blk2.float() - y.float()).abs().max().item() <= 2.0 ** -7 * y.float().abs().max().item()
    # the gradient with dx in dr's place and dblock in dy's
    space = torch.empty(n3d.residual_norm_workspace(37, 512), dtype=torch.uint8, device="cuda")
    dx, dblock = torch.empty_like(r), torch.empty_like(y)
    n3d.residual_norm_grad(d["block"], r, d["dy"], d["dr"], dx, dblock, post="layer", workspace=space)
    n3d.residual_norm_grad(d["block"], r, d["dy"], d["dr"], d["dr"], d["dy"], post="layer", workspace=space)
    torch.cuda.synchronize()
    assert torch.equal(d["dr"], dx) and torch.equal(d["dy"], dblock)
    # no dr: zero
    n3d.residual_norm_grad(d["block"], r, y, None, dx, dblock, post="layer", workspace=space)
    other = torch.empty_like(dx)
    n3d.residual_norm_grad(d["block"], r, y, torch.zeros_like(dx), other, dblock.clone(), post="layer", workspace=space)
    torch.cuda.synchronize()
    assert torch.equal(dx, other)


@pytest.mark.gpu
def test_no_rows():
    import torch

    x = torch.empty(0, 512, device="cuda")
    n3d.residual_norm(x, x, x, x)
    space = torch.empty(n3d.residual_norm_workspace(0, 512), dtype=torch.uint8, device="cuda")
    dw, db = torch.full((512,), 3.0, device="cuda"), torch.full((512,), 3.0, device="cuda")
    n3d.residual_norm_grad(x, x, x, x, x, x, dpre_w=dw, dpre_b=db, workspace=space)
    torch.cuda.synchronize()
    assert not dw.any() and not db.any()


@pytest.mark.gpu
def test_a_row_of_nan_stays_in_its_row():
    import torch

    t, _ = make(40, 512, "float32", "float32", 0, 9)
    d = {n: v.cuda() for n, v in t.items()}
    r, y = torch.empty_like(d["x"]), torch.empty_like(d["x"])
    n3d.residual_norm(d["x"], d["block"], r, y, post="rms")
    d["block"][17] = math.nan
    d["x"][3, 5] = math.inf
    r2, y2 = torch.empty_like(r), torch.empty_like(y)
    n3d.residual_norm(d["x"], d["block"], r2, y2, post="rms")
    torch.cuda.synchronize()
    keep = [i for i in range(40) if i not in (3, 17)]
    assert torch.equal(r2[keep], r[keep]) and torch.equal(y2[keep], y[keep])
    assert y2[17].isnan().all() and r2[3, 5].isinf()

"""Attention with its gradient (n3d_attention_forward, n3d_attention_backward): refusals
and the formulas on the CPU, and on a B200 every output against 64-bit arithmetic.

Tolerances, derived (e = 2^-24, h = half an ulp of the type: 2^-8 bf16, 2^-11 fp16, 0 for
fp32).  A score is a sum of head_dim products: within 16 e A, A the largest sum of
|q_d k_d| times the scale (fp32 sums in chunks, or 22-bit operands); its exponent is rounded
with the scale and the maximum: 16 e max(1, A).  So p is off by d = 16 e (2 A + 2),
relatively, and so is the row sum.  Probabilities enter their products rounded (h p, and
for fp16 2^-25, the end of its subnormals), so out is off by (2 d + h) sum p |v|, plus its own
rounding.  D = dout.out is off by eD = sum |dout| err(out) + 16 e sum |dout out|, dP by 16 e
sum |dout v|, dS by P (2 d |dP - D| + eD + err(dP)) + h |dS| (fp16: + 2^-24 max|dout|), the
gradients by the sums of these against |k|, |q| and |dout|, plus 16 e of the sums of
magnitudes and their own rounding."""

import math

import numpy as np
import pytest

import n3d
from fake_tensor import FakeTensor

E = 2.0 ** -24
HALF_ULP = {"float32": 0.0, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


# ------------------------------------------------------------------------- 64 bits
def seen64(nq, nk, ql, kl, left, right, off):
    i, j = np.arange(nq)[:, None], np.arange(nk)[None]
    ok = (i < ql) & (j < kl)
    if right >= 0:
        ok &= j - i - off <= right
    if left >= 0:
        ok &= i + off - j <= left
    return ok


def head64(q, k, v, do, seen, scale, dtype):
    """One head: out, lse, dq, dk, dv, and their error bounds."""
    h, f16 = HALF_ULP[dtype], dtype == "float16"
    q, k, v, do = (np.where(np.isfinite(t), t, 0.0) for t in (q, k, v, do))
    s = np.where(seen, q @ k.T * scale, -np.inf)
    top = s.max(1, keepdims=True, initial=-np.inf)
    top = np.where(np.isfinite(top), top, 0.0)
    total = np.exp(s - top).sum(1, keepdims=True)
    with np.errstate(divide="ignore"):
        lse = top + np.log(total)
    p = np.where(seen, np.exp(s - np.where(np.isfinite(lse), lse, 0.0)), 0.0)
    a = abs(scale) * (np.abs(q) @ np.abs(k).T)
    A = np.where(seen, a, 0.0).max(initial=0.0)
    d = 16 * E * (2 * A + 2)
    out = p @ v
    pa = seen * 2.0 ** -25 if f16 else 0.0 * p  # absolute error of a rounded probability
    e_out = ((2 * d + h) * p + pa) @ np.abs(v)
    e_out = e_out + h * (np.abs(out) + e_out)
    dot, dp = (do * out).sum(1, keepdims=True), do @ v.T
    e_dot = (np.abs(do) * e_out).sum(1, keepdims=True) + 16 * E * np.abs(do * out).sum(1, keepdims=True)
    e_dp = 16 * E * (np.abs(do) @ np.abs(v).T)
    ds = p * (dp - dot)
    e_ds = p * (2 * d * np.abs(dp - dot) + e_dot + e_dp)
    e_ds = e_ds + h * (np.abs(ds) + e_ds) + (seen * 2.0 ** -24 * np.abs(do).max(initial=0.0) if f16 else 0.0)
    e_p = (2 * d + h) * p + pa
    grads = {"dq": scale * (ds @ k), "dk": scale * (ds.T @ q), "dv": p.T @ do}
    err = {"dq": abs(scale) * ((e_ds + 16 * E * np.abs(ds)) @ np.abs(k)),
           "dk": abs(scale) * ((e_ds + 16 * E * np.abs(ds)).T @ np.abs(q)),
           "dv": (e_p + 16 * E * p).T @ np.abs(do)}
    # lse: the scores' error and the logarithm's, in units of the sum
    return dict(out=out, lse=lse[:, 0], **grads), dict(out=e_out, lse=np.full(len(lse), 2 * d + 4 * E * (A + 8)), **err)


def attention64(q, k, v, do, ql, kl, scale, left, right, off, dtype):
    b, nq, hq, hd = q.shape
    nk, hk = k.shape[1:3]
    z = lambda t: np.zeros(t.shape)
    val = dict(out=z(q), lse=np.zeros((b, hq, nq)), dq=z(q), dk=z(k), dv=z(k))
    err = {n: np.zeros(t.shape) for n, t in val.items()}
    for s in range(b):
        seen = seen64(nq, nk, ql[s], kl[s], left, right, off)
        for h in range(hq):
            g = h // (hq // hk)
            one, off_by = head64(q[s, :, h], k[s, :, g], v[s, :, g], do[s, :, h], seen, scale, dtype)
            for src, dst in ((one, val), (off_by, err)):
                dst["out"][s, :, h], dst["dq"][s, :, h], dst["lse"][s, h] = src["out"], src["dq"], src["lse"]
                dst["dk"][s, :, g] += src["dk"]
                dst["dv"][s, :, g] += src["dv"]
    return val, err


def test_the_gradient_formula_against_differences():
    rng = np.random.default_rng(1)
    q, k, v, do = (rng.standard_normal(s) for s in ((5, 8), (7, 8), (7, 8), (5, 8)))
    for left, right, off in ((-1, -1, 0), (-1, 0, 2), (1, 1, 3)):
        seen = seen64(5, 7, 4, 6, left, right, off)
        loss = lambda q, k, v: (head64(q, k, v, do, seen, 0.35, "float32")[0]["out"] * do).sum()
        got, _ = head64(q, k, v, do, seen, 0.35, "float32")
        for n, name in enumerate(("dq", "dk", "dv")):
            for i in np.ndindex((q, k, v)[n].shape):
                up, down = [t.copy() for t in (q, k, v)], [t.copy() for t in (q, k, v)]
                up[n][i] += 1e-5
                down[n][i] -= 1e-5
                # central differences: h^2 f''' / 6 and 1e-16 |f| / h, both below 1e-9 here
                assert abs((loss(*up) - loss(*down)) / 2e-5 - got[name][i]) < 1e-8


# ------------------------------------------------------------------------- refusals
def _call(q=None, k=None, v=None, out=None, backward=False, space=1 << 20, **kw):
    f = lambda n, p: FakeTensor((2, n, 4, 64), ptr=p << 20)
    q, k = q or f(5, 1), k or f(7, 2)
    v, out = v or FakeTensor(k.shape, ptr=3 << 20), out or FakeTensor(q.shape, ptr=4 << 20)
    if not backward:
        return n3d.attention_forward(q, k, v, out, kw.pop("lse", None), **kw)
    work = FakeTensor((space,), dtype="uint8", ptr=10 << 20)
    g = {n: FakeTensor(t.shape, ptr=p << 20) for n, t, p in (("dout", q, 5), ("dq", q, 6), ("dk", k, 7), ("dv", k, 8))}
    g.update({n: kw.pop(n) for n in list(g) if n in kw})
    lse = kw.pop("lse", FakeTensor((2, 4, 5), ptr=9 << 20))
    return n3d.attention_backward(q, k, v, out, lse, g["dout"], g["dq"], g["dk"], g["dv"], workspace=work, **kw)


@pytest.mark.parametrize("kw", [
    dict(q=FakeTensor((2, 5, 3, 64))),                                    # 3 query heads over 4 key heads
    dict(q=FakeTensor((2, 5, 4, 96)), k=FakeTensor((2, 7, 4, 96))),       # head_dim
    dict(k=FakeTensor((2, 7, 4, 128))), dict(k=FakeTensor((3, 7, 4, 64))), dict(v=FakeTensor((2, 8, 4, 64))),
    dict(v=FakeTensor((2, 7, 4, 64), dtype="bfloat16")), dict(out=FakeTensor((2, 5, 4, 64), (0, 256, 64, 1))),
    dict(out=FakeTensor((2, 5, 4, 64), (1280, 256, 32, 1))), dict(q=FakeTensor((2, 5, 4, 64), (1280, -256, 64, 1))),
    dict(scale=math.inf), dict(scale=math.nan), dict(left=1 << 31), dict(right=1 << 40), dict(q_offset=-(1 << 31)),
    dict(q_len=FakeTensor((3,), dtype="int32")), dict(k_len=FakeTensor((2,), dtype="int64")),
    dict(lse=FakeTensor((2, 4, 6))), dict(lse=FakeTensor((2, 4, 5), dtype="bfloat16")),
    dict(q=FakeTensor((2, 5, 4, 64), dtype="float64"), k=FakeTensor((2, 7, 4, 64), dtype="float64")),
    dict(q=FakeTensor((2, 5, 4, 64), (2560, 512, 128, 2))), dict(q=FakeTensor((5, 4, 64))),
])
def test_forward_refusals(kw):
    with pytest.raises(n3d.DiarizationError) as e:
        _call(**kw)
    assert e.value.kind == "InvalidArgument"


@pytest.mark.parametrize("kw", [
    dict(space=16), dict(lse=None), dict(dout=FakeTensor((2, 5, 2, 64))), dict(dk=FakeTensor((2, 5, 4, 64))),
    dict(dv=FakeTensor((2, 7, 4, 64), (0, 256, 64, 1))), dict(dq=FakeTensor((2, 5, 4, 64), dtype="float16")),
])
def test_backward_refusals(kw):
    with pytest.raises(n3d.DiarizationError) as e:
        _call(backward=True, **kw)
    assert e.value.kind == "InvalidArgument"


def test_null_arguments():
    L = n3d.lib()
    assert n3d.STATUS[L.n3d_attention_forward(0, None, None, None, None, None, None, None, None, None, 0, None)] == \
        "InvalidArgument"
    cfg = n3d._pack_attn(1, 1, 1, 64, 0, 0.0, -1, -1, 0)
    assert n3d.STATUS[L.n3d_attention_forward(0, cfg, None, None, None, None, None, None, None, None, 0,
                                              None)] == "InvalidArgument"
    assert L.n3d_attention_workspace(None, 1, 1, 1) == 0


# ----------------------------------------------------------------------------- B200
def lengths(b, n, seed):
    rng = np.random.default_rng(seed)
    out = rng.integers(0, n + 1, b)
    out[0] = n
    return out.astype(np.int32)


def run(b, nq, nk, hq, hk, hd, dtype, left=-1, right=-1, off=0, ragged=False, layout="rows", scale=0.0, seed=0, std=1.0,
        do_std=0.1, v_std=1.0, check=True):
    """Forward and backward on the GPU, checked against 64 bits; returns the outputs."""
    import torch

    dt = getattr(torch, dtype)
    g = torch.Generator().manual_seed(seed)
    rnd = lambda n, h: torch.randn(b, n, h, hd, generator=g).to(dt)
    host = [(rnd(nq, hq) * std).to(dt), (rnd(nk, hk) * std).to(dt), (rnd(nk, hk) * v_std).to(dt),
            (rnd(nq, hq) * do_std).to(dt)]
    ql, kl = (lengths(b, nq, seed + 1), lengths(b, nk, seed + 2)) if ragged else ([nq] * b, [nk] * b)
    if ragged:  # what stands past the lengths is never read
        for s in range(b):
            for t, n in zip(host, (ql, kl, kl, ql)):
                t[s, n[s]:] = math.nan if s % 2 else math.inf
    place = {"rows": lambda t: t.cuda().contiguous(),
             "heads": lambda t: t.cuda().transpose(1, 2).contiguous().transpose(1, 2),
             "odd": lambda t: torch.nn.functional.pad(t.cuda().reshape(-1), (1, 0))[1:].view(t.shape),
             "wide": lambda t: torch.nn.functional.pad(t.cuda(), (0, 8))[..., : t.shape[3]]}[layout]
    q, k, v, do = (place(t) for t in host)
    fresh = lambda t: place(torch.full(t.shape, math.nan, dtype=dt))
    out, dq, dk, dv = fresh(host[0]), fresh(host[0]), fresh(host[1]), fresh(host[1])
    lse = torch.full((b, hq, nq), math.nan, device="cuda")
    space = torch.full((n3d.attention_workspace(q, k),), 255, dtype=torch.uint8, device="cuda")
    lens = dict(q_len=torch.tensor(ql, dtype=torch.int32, device="cuda"),
                k_len=torch.tensor(kl, dtype=torch.int32, device="cuda")) if ragged else {}
    kw = dict(scale=scale, left=left, right=right, q_offset=off, workspace=space,
              stream=torch.cuda.current_stream().cuda_stream, **lens)
    n3d.attention_forward(q, k, v, out, lse, **kw)
    n3d.attention_backward(q, k, v, out, lse, do, dq, dk, dv, **kw)
    torch.cuda.synchronize()
    n3d.train_status(0)
    got = dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv)
    if check:
        want, err = attention64(*(t.double().numpy() for t in host), ql, kl, scale or hd ** -0.5, left, right, off, dtype)
        for n, w in want.items():
            x = got[n].double().cpu().numpy()
            inf = np.isinf(w)
            assert np.array_equal(np.isneginf(x), inf), n
            h = 0.0 if n == "lse" else HALF_ULP[dtype]
            w = np.where(inf, 0.0, w)
            x = np.where(inf, 0.0, x)
            limit = err[n] + h * (np.abs(w) + err[n]) + (2.0 ** -25 if dtype == "float16" and n != "lse" else 1e-37)
            worst = (np.abs(x - w) / limit).max(initial=0.0)
            assert worst <= 1.0, (n, worst)
            assert not np.isnan(x).any(), n
    return got


TYPES = ["float32", "bfloat16", "float16"]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 300), (63, 64), (64, 65), (65, 63), (127, 129), (128, 128), (130, 257),
                                   (300, 1), (257, 512)])
def test_lengths(dtype, hd, nq, nk):
    run(2, nq, nk, 2, 2, hd, dtype, seed=nq + nk)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_ragged_sequences_with_nan_past_the_lengths(dtype, hd):
    run(7, 150, 210, 2, 1, hd, dtype, ragged=True, seed=3)
    run(9, 5, 70, 1, 1, hd, dtype, ragged=True, seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("left,right,off", [(-1, 0, 0), (-1, 0, 40), (-1, 0, -70), (0, 0, 0), (10, 3, 0), (130, -1, 5),
                                            (64, 64, 64), (-1, 200, -300), (5, 5, 1000), (5, 5, -1000), (300, 0, 190)])
def test_windows(dtype, left, right, off):
    """Causal, local, shifted windows; some leave rows, or everything, without keys."""
    run(2, 200, 240, 1, 1, 64, dtype, left, right, off, seed=left + right)
    run(2, 200, 240, 2, 1, 128, dtype, left, right, off, ragged=True, seed=abs(off))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hk", [(1, 1), (6, 2), (8, 1), (3, 3)])
def test_shared_key_heads(dtype, hq, hk):
    run(2, 100, 140, hq, hk, 64, dtype, -1, 0, 40, seed=hq)
    run(1, 140, 100, hq, hk, 128, dtype, seed=hk)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["heads", "odd", "wide"])
def test_layouts(dtype, layout):
    run(2, 77, 133, 4, 2, 64, dtype, ragged=True, layout=layout, seed=6)
    run(1, 133, 77, 2, 2, 128, dtype, -1, 0, 0, layout=layout, seed=7)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_peaked_and_flat_rows_and_small_gradients(dtype):
    run(1, 130, 200, 1, 1, 64, dtype, std=3.0, seed=8)                 # one key takes nearly all
    run(1, 130, 200, 1, 1, 64, dtype, scale=1e-3, seed=9)              # all keys alike
    run(1, 130, 200, 1, 1, 64, dtype, scale=-0.2, seed=10)             # a negative scale
    run(1, 130, 200, 1, 1, 128, dtype, do_std=2e-3, seed=11)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,v_std", [(64, 380.0), (128, 260.0)])
def test_large_values(dtype, hd, v_std):
    # rows of v of norms about 3000, inside the 4096 that fp16 gradients are held to; outputs stay far from its largest
    run(1, 130, 200, 2, 1, hd, dtype, -1, 0, 70, do_std=0.02, v_std=v_std, seed=15)


@pytest.mark.gpu
def test_longer_rows():
    run(1, 1030, 1500, 2, 1, 64, "bfloat16", -1, 0, 470, seed=12)
    run(1, 900, 1100, 1, 1, 128, "float16", 400, 100, 100, seed=13)
    run(1, 700, 700, 1, 1, 64, "float32", seed=14)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_repeatable_bit_for_bit(dtype):
    import torch

    a, b = (run(3, 333, 400, 4, 2, 64, dtype, ragged=True, seed=15, check=False) for _ in range(2))
    for n in a:
        assert torch.equal(a[n], b[n])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_offsets_past_32_bits(dtype):
    """Two sequences 2^32 elements apart give what they give side by side."""
    import torch

    dt = getattr(torch, dtype)
    n, h, hd, apart = 70, 2, 64, 1 << 32
    buf = torch.empty(apart + 4 * n * h * hd, dtype=dt, device="cuda")
    far = lambda i: torch.as_strided(buf, (2, n, h, hd), (apart, h * hd, hd, 1), i * n * h * hd)
    near = [torch.randn(2, n, h, hd, device="cuda").to(dt) for _ in range(3)]
    out, lse = torch.empty_like(near[0]), torch.empty(2, h, n, device="cuda")
    q, k, v = (far(i) for i in range(3))
    for f, t in zip((q, k, v), near):
        f.copy_(t)
    space = torch.empty(n3d.attention_workspace(q, k), dtype=torch.uint8, device="cuda")
    n3d.attention_forward(*near, out, lse, workspace=space)
    lse2 = torch.empty_like(lse)
    n3d.attention_forward(q, k, v, far(3), lse2, workspace=space)
    torch.cuda.synchronize()
    assert torch.equal(far(3), out) and torch.equal(lse, lse2)
    grads = [torch.empty_like(out) for _ in range(6)]
    n3d.attention_backward(*near, out, lse, near[0], *grads[:3], workspace=space)
    n3d.attention_backward(q, k, v, far(3), lse, q, *grads[3:], workspace=space)
    torch.cuda.synchronize()
    for a, b in zip(grads[:3], grads[3:]):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_broadcast_keys_lse_not_wanted_streams_and_graphs(dtype):
    import torch

    dt = getattr(torch, dtype)
    q = torch.randn(3, 90, 4, 64, device="cuda").to(dt)
    k, v = (torch.randn(1, 110, 1, 64, device="cuda").to(dt) for _ in range(2))
    want, got, other = torch.empty_like(q), torch.empty_like(q), torch.empty_like(q)
    full = [t.expand(3, -1, 4, -1).contiguous() for t in (k, v)]
    space = torch.empty(n3d.attention_workspace(q, full[0]), dtype=torch.uint8, device="cuda")
    n3d.attention_forward(q, *full, want, workspace=space)
    n3d.attention_forward(q, k.expand(3, -1, 4, -1), v.expand(3, -1, 4, -1), got, workspace=space)
    torch.cuda.synchronize()
    # the same keys through strides of zero, whichever path that takes
    tol = 2 * (HALF_ULP[dtype] + 16 * E * 30) * v.float().abs().max() * 2
    assert (want.float() - got.float()).abs().max() <= tol
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        n3d.attention_forward(q, *full, other, workspace=space, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(other, want)
    other.zero_()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        n3d.attention_forward(q, *full, other, workspace=space, stream=torch.cuda.current_stream().cuda_stream)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(other, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_to_attend(dtype):
    import torch

    dt = getattr(torch, dtype)
    e = lambda b, n, h: torch.full((b, n, h, 64), math.nan, dtype=dt, device="cuda")
    q, none, out, lse = torch.randn(2, 9, 2, 64, device="cuda").to(dt), e(2, 0, 2), e(2, 9, 2), torch.zeros(2, 2, 9, device="cuda")
    space = torch.empty(max(n3d.attention_workspace(q, q), 16), dtype=torch.uint8, device="cuda")
    n3d.attention_forward(q, none, none, out, lse, workspace=space)
    dq = e(2, 9, 2)
    n3d.attention_backward(q, none, none, out, lse, q, dq, none, none, workspace=space)
    torch.cuda.synchronize()
    assert not out.any() and lse.isneginf().all() and not dq.any()
    # no queries: the keys' gradients are zeros
    k, dk, dv, l0 = q, e(2, 9, 2), e(2, 9, 2), torch.empty(2, 2, 0, device="cuda")
    n3d.attention_forward(none, k, k, none, l0, workspace=space)
    n3d.attention_backward(none, k, k, none, l0, none, none, dk, dv, workspace=space)
    torch.cuda.synchronize()
    assert not dk.any() and not dv.any()
    zero = torch.empty(0, 9, 2, 64, dtype=dt, device="cuda")
    n3d.attention_forward(zero, zero, zero, zero, torch.empty(0, 2, 9, device="cuda"), workspace=space)

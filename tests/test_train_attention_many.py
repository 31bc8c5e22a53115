"""Attention with its gradient on more tiles than a GPU holds at a time, where blocks of threads take further tiles over
while they work: which block gets which tile depends on timing, the results must not.

Every case has 576 to 1728 tiles of 128 rows (148 or 296 are resident), of 1 to 7 column blocks by the sequences'
lengths, some of them none.  Results are compared with 64-bit arithmetic on the GPU, with further calls, and with calls
on single sequences, bit for bit.

Tolerances, derived: as in test_train_attention.py, by the norm of each output over a head of a sequence: rounding
errors h (half an ulp of the type) of the weights and of the outputs are independent, so a norm is off by at
most 2 h in out and dv and 4 h in dq and dk, in which dP - D cancels (both errors of P and of D enter).  fp32: 16 e (2 A + 2) as
there, with A = 40 above every score's sum of magnitudes, twice for the gradients."""

import math

import pytest

import n3d

pytestmark = pytest.mark.gpu
TYPES = ["float32", "bfloat16", "float16"]
E = 2.0 ** -24
LIMIT = {"float32": 16 * E * 82, "bfloat16": 2.0 ** -7, "float16": 2.0 ** -10}


def make(b, nq, nk, hq, hk, hd, dtype, seed):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda n, h, f: (f * torch.randn(b, n, h, hd, generator=g, device="cuda")).to(getattr(torch, dtype))
    t = [rnd(nq, hq, 1), rnd(nk, hk, 1), rnd(nk, hk, 1), rnd(nq, hq, 0.1)]
    lens = [torch.randint(0, n + 1, (b,), generator=g, device="cuda", dtype=torch.int32) for n in (nq, nk)]
    lens[0][::2] = nq
    lens[1][3] = 0
    return t, lens


def call(t, lens, **window):
    import torch

    q, k, v, do = t
    out, dq, dk, dv = (torch.full_like(x, math.nan) for x in (q, q, k, v))
    lse = torch.full((q.shape[0], q.shape[2], q.shape[1]), math.nan, device="cuda")
    kw = dict(q_len=lens[0], k_len=lens[1], workspace=torch.full((n3d.attention_workspace(q, k),), 255, dtype=torch.uint8,
                                                                 device="cuda"), **window)
    n3d.attention_forward(q, k, v, out, lse, **kw)
    n3d.attention_backward(q, k, v, out, lse, do, dq, dk, dv, **kw)
    torch.cuda.synchronize()
    n3d.train_status(0)
    return dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv)


def exact(t, lens, left=-1, right=-1, q_offset=0):
    """One sequence in 64 bits."""
    import torch

    q, k, v, do = (x.double().transpose(0, 1) for x in t)
    group = q.shape[0] // k.shape[0]
    k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
    i, j = torch.arange(q.shape[1], device="cuda")[:, None], torch.arange(k.shape[1], device="cuda")[None]
    seen = (i < lens[0]) & (j < lens[1])
    if right >= 0:
        seen &= j - i - q_offset <= right
    if left >= 0:
        seen &= i + q_offset - j <= left
    s = (q @ k.transpose(1, 2) * q.shape[2] ** -0.5).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, 2)
    p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[..., None])
    do = do * (i < lens[0])
    out = p @ v
    ds = p * (do @ v.transpose(1, 2) - (do * out).sum(2, keepdim=True)) * q.shape[2] ** -0.5
    shared = lambda x: x.view(-1, group, *x.shape[1:]).sum(1)
    got = dict(out=out, dq=ds @ k, dk=shared(ds.transpose(1, 2) @ q), dv=shared(p.transpose(1, 2) @ do))
    return {**{n: x.transpose(0, 1) for n, x in got.items()}, "lse": lse}


SHAPES = [(24, 330, 420, 8, 8, {}), (36, 383, 320, 16, 4, {}), (24, 330, 400, 8, 4, dict(right=0, q_offset=70)),
          (24, 384, 384, 8, 8, dict(left=90, right=30))]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_tiles_that_blocks_take_over(dtype, hd, case):
    import torch

    b, nq, nk, hq, hk, window = SHAPES[case]
    t, lens = make(b, nq, nk, hq, hk, hd, dtype, case)
    got = call(t, lens, **window)
    for s in range(b):
        want = exact([x[s] for x in t], [n[s] for n in lens], **window)
        for n, w in want.items():
            x = got[n][s].double()
            assert not x.isnan().any(), n
            if n == "lse":
                assert torch.equal(x.isinf(), w.isinf())
                assert (x - w).masked_fill(w.isinf(), 0.0).abs().max() <= 16 * E * 82
                continue
            off, size = ((y * y).sum((0, 2)).sqrt() for y in (x - w, w))
            limit = LIMIT[dtype] * (1 if n in ("out", "dv") else 2)
            assert (off <= limit * size + 1e-30).all(), (n, s, (off / size).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_results_do_not_depend_on_which_block_takes_a_tile(dtype, hd, case):
    import torch

    b, nq, nk, hq, hk, window = SHAPES[case]
    t, lens = make(b, nq, nk, hq, hk, hd, dtype, 10 + case)
    first = call(t, lens, **window)
    for _ in range(6):
        for n, x in call(t, lens, **window).items():
            assert torch.equal(x, first[n]), n
    for s in (0, 5, b - 2):  # alone: 24 to 48 tiles, none of them taken over
        one = call([x[s:s + 1] for x in t], [n[s:s + 1] for n in lens], **window)
        for n, x in one.items():
            assert torch.equal(x[0], first[n][s]), (n, s)

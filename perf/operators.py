"""The operators of an encoder block's fine-tuning step, as they are measured.

Three operators: rotary positions ("rope"), a block's residual add with the norms before
and after it ("norm"), and attention with its gradient ("attention").  A case names one
operator and its sizes; `run` makes one pass through it, in elementary torch operations
(`own` False) or through this repository's own entry points (`own` True).
"""

import functools
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
DEV = "cuda:0"


# ------------------------------------------------------------------------- cases
def _rope(name, seqs, rows, q_heads, k_heads, head_dim, rotary_dim, layout, scaling, dtype, packed, transpose):
    c = dict(op="rope", seqs=seqs, rows=rows, q_heads=q_heads, k_heads=k_heads, head_dim=head_dim,
             rotary_dim=rotary_dim, layout=layout, scaling=scaling, dtype=dtype, packed=packed, transpose=transpose)
    return dict(c, name=name) if name else c


def _norm(name, rows, cols, residual, block, post, pre, gate_rows, direction):
    c = dict(op="norm", rows=rows, cols=cols, residual=residual, block=block, post=post, pre=pre,
             gate_rows=gate_rows, direction=direction)
    return dict(c, name=name) if name else c


def _attn(name, seqs, q_rows, k_rows, q_heads, k_heads, head_dim, dtype, left, right, ragged, packed, train):
    c = dict(op="attention", seqs=seqs, q_rows=q_rows, k_rows=k_rows, q_heads=q_heads, k_heads=k_heads,
             head_dim=head_dim, dtype=dtype, left=left, right=right, ragged=ragged, packed=packed, train=train)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one ultra-low-latency step (3 encoder frames) of 32 streaming sessions, each at its own position
        _rope("rope_step", 32, 3, 8, 8, 64, 64, "half", "none", "bf16", True, False),
        # 128 offline windows, in 32 bits, as the encoder's own q and k
        _rope("rope_windows", 128, 376, 8, 8, 64, 64, "half", "none", "f32", True, False),
        # the gradient's rotation on a long recording: interleaved, half of the head, stretched context, shared key heads
        _rope("rope_long_grad", 1, 30001, 32, 8, 128, 64, "interleaved", "yarn", "f16", False, True),
        # residual add and LayerNorm of one step of 32 sessions: latency
        _norm("norm_step", 96, 512, "f32", "f32", "none", "layer", 0, "forward"),
        # the same of 128 windows in training: 32-bit residual stream, 16-bit blocks, one gate per channel
        _norm("norm_windows", 48128, 512, "f32", "bf16", "layer", "layer", 48128, "forward"),
        # the gradient at a wide block boundary: RMS norms on both sides, a gate for each sequence
        _norm("norm_wide_grad", 8191, 4096, "bf16", "bf16", "rms", "rms", 1024, "backward"),
        # new frames of 32 sessions over their windows: latency
        _attn("attn_step", 32, 3, 211, 8, 8, 64, "bf16", -1, -1, True, False, False),
        # 128 offline windows of uneven length, forward
        _attn("attn_windows", 128, 384, 384, 8, 8, 64, "bf16", -1, -1, True, True, False),
        # a training step on 64 windows of uneven length, odd row count
        _attn("attn_windows_train", 64, 377, 377, 8, 8, 64, "f16", -1, -1, True, True, True),
        # a causal training step on long sequences with shared key heads, the largest
        _attn("attn_causal_train", 2, 4096, 4096, 16, 4, 128, "bf16", -1, 0, False, True, True),
        # a long recording with a limited look-back and look-ahead
        _attn("attn_local_train", 1, 8191, 8191, 8, 8, 64, "bf16", 256, 64, False, False, True),
        # a training step in 32 bits, the type of the encoder's own activations
        _attn("attn_windows_train_f32", 8, 501, 501, 8, 8, 64, "f32", -1, -1, True, True, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rope", "norm", "attention"))
    if op == "rope":
        head_dim = rng.choice((64, 128))
        k_heads = rng.choice((1, 2, 4, 8))
        q_heads = k_heads * rng.choice((1, 2, 4))
        dtype = rng.choice(tuple(TYPES))
        seqs = _log(rng, 1, 128)
        most = 150_000_000 // (seqs * (q_heads + k_heads) * head_dim * BYTES[dtype] // 2)
        return _rope(None, seqs, _log(rng, 1, min(32768, most)), q_heads, k_heads, head_dim,
                     rng.choice((head_dim, head_dim // 2, head_dim // 4 + 2)), rng.choice(("half", "interleaved")),
                     rng.choice(("none", "linear", "ntk", "yarn")), dtype, rng.random() < 0.5, rng.random() < 0.5)
    if op == "norm":
        cols = rng.choice((512, 1024, 2048, 4096, rng.randrange(65, 4097)))
        residual, block = rng.choice((("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")))
        rows = _log(rng, 1, 30_000_000 // cols)
        return _norm(None, rows, cols, residual, block, rng.choice(("none", "layer", "rms")),
                     rng.choice(("layer", "rms")), rng.choice((0, rows, max(1, rows // 7), 1 + rows // 100)),
                     rng.choice(("forward", "backward")))
    dtype = rng.choice(("bf16", "bf16", "f16", "f16", "f32"))
    head_dim = rng.choice((64, 128))
    k_heads = rng.choice((1, 2, 4, 8))
    q_heads = k_heads * rng.choice((1, 1, 2, 4))
    rows = _log(rng, 1, 4096)
    most = max(1, min(128, (80_000_000 if dtype == "f32" else 400_000_000) // (rows * rows * q_heads * head_dim // 64)))
    seqs = _log(rng, 1, most)
    left, right = rng.choice(((-1, -1), (-1, -1), (-1, 0), (rng.randrange(16, 1024), rng.randrange(0, 256))))
    k_rows = rows if rng.random() < 0.7 else _log(rng, rows, max(rows, min(4096, 2 * rows + 64)))
    return _attn(None, seqs, rows, k_rows, q_heads, k_heads, head_dim, dtype, left, right, rng.random() < 0.6,
                 k_rows == rows and rng.random() < 0.5, rng.random() < 0.7)


def _lens(case):
    """(query lengths, key lengths) of the sequences: by the case alone.  Ragged batches of 8 and
    more hold one sequence without keys."""
    b, nq, nk = case["seqs"], case["q_rows"], case["k_rows"]
    if not case["ragged"]:
        return [nq] * b, [nk] * b
    r = random.Random(1009 * b + 31 * nq + nk)
    part = [r.uniform(0.4, 1.0) for _ in range(b)]
    part[0] = 1.0
    ql, kl = ([nq] * b if nq < 16 else [max(1, round(nq * p)) for p in part]), [max(1, round(nk * p)) for p in part]
    if b >= 8:
        kl[b // 2] = 0
    return ql, kl


def _offset(case):
    """Key position of query row 0: the queries are the last rows of the keys' range."""
    return case["k_rows"] - case["q_rows"]


# ------------------------------------------------------------------- rotary frequencies
def _rope_config(case):
    stretch = case["scaling"] != "none"
    return dict(head_dim=case["head_dim"], rotary_dim=case["rotary_dim"], layout=case["layout"], theta=10000.0,
                scaling=case["scaling"], factor=8.0 if stretch else 1.0, original_length=4096, beta_fast=32.0,
                beta_slow=1.0)


def _frequencies(cfg):
    """Angle per position of each pair, in radians, and the factor on the rotated values."""
    n, theta, factor = cfg["rotary_dim"], cfg["theta"], cfg["factor"]
    if cfg["scaling"] == "ntk" and n > 2:
        theta *= factor ** (n / (n - 2))
    f = [theta ** (-2.0 * i / n) for i in range(n // 2)]
    if cfg["scaling"] == "linear":
        return [x / factor for x in f], 1.0
    if cfg["scaling"] != "yarn":
        return f, 1.0

    def at(turns):  # the (fractional) pair that makes `turns` turns over the original length
        return n * math.log(cfg["original_length"] / (turns * 2 * math.pi)) / (2 * math.log(theta))

    lo, hi = max(math.floor(at(cfg["beta_fast"])), 0), min(math.ceil(at(cfg["beta_slow"])), n - 1)
    ramp = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3))) for i in range(n // 2)]
    return [x * (1 - r) + x / factor * r for x, r in zip(f, ramp)], 0.1 * math.log(factor) + 1.0


# ----------------------------------------------------------------------- inputs
def _heads(g, b, n, heads, d, dtype, packed, std=1.0):
    """Tensors [b, n, h, d] for each h of `heads`: slices of one buffer if `packed`."""
    if packed:
        x = (torch.randn(b, n, sum(heads), d, generator=g, device=DEV) * std).to(TYPES[dtype])
        return list(x.split(heads, dim=2))
    return [(torch.randn(b, n, h, d, generator=g, device=DEV) * std).to(TYPES[dtype]) for h in heads]


def _like(ts, packed):
    if packed:
        b, n, _, d = ts[0].shape
        heads = [t.shape[2] for t in ts]
        return list(torch.empty(b, n, sum(heads), d, dtype=ts[0].dtype, device=DEV).split(heads, dim=2))
    return [torch.empty_like(t) for t in ts]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "rope":
        b, n = case["seqs"], case["rows"]
        s["x"] = _heads(g, b, n, [case["q_heads"], case["k_heads"]], case["head_dim"], case["dtype"], case["packed"])
        s["y"] = _like(s["x"], case["packed"])
        first = torch.randint(0, 4096, (b, 1), generator=g, device=DEV, dtype=torch.int32)
        s["positions"] = (first + torch.arange(n, device=DEV, dtype=torch.int32)).contiguous()
        f, s["factor"] = _frequencies(_rope_config(case))
        # turns per position as 64-bit fractions of a turn: phases wrap exactly, at any position
        turns = [round(x / (2 * math.pi) * 2.0 ** 64) % 2 ** 64 for x in f]
        s["turns"] = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], device=DEV)
    elif case["op"] == "norm":
        n, c = case["rows"], case["cols"]
        rt, bt = TYPES[case["residual"]], TYPES[case["block"]]

        def randn(*shape):
            return torch.randn(*shape, generator=g, device=DEV)

        s["block"] = (0.7 * randn(n, c) + 0.1).to(bt)
        s["post_w"], s["post_b"] = 1 + 0.1 * randn(c), 0.1 * randn(c)
        s["pre_w"], s["pre_b"] = 1 + 0.1 * randn(c), 0.1 * randn(c)
        s["scale"] = 0.5
        s["gate"] = 0.5 + 0.2 * randn(-(-n // case["gate_rows"]), c) if case["gate_rows"] else None
        if case["direction"] == "forward":
            s["x"] = randn(n, c).to(rt)
            s["r"], s["y"] = torch.empty(n, c, dtype=rt, device=DEV), torch.empty(n, c, dtype=bt, device=DEV)
        else:
            s["r"], s["dy"], s["dr"] = randn(n, c).to(rt), (0.1 * randn(n, c)).to(bt), (0.1 * randn(n, c)).to(rt)
            s["dx"], s["dblock"] = torch.empty(n, c, dtype=rt, device=DEV), torch.empty(n, c, dtype=bt, device=DEV)
            s["dw"] = torch.empty(4, c, device=DEV)  # post weight and bias, pre weight and bias
            s["dgate"] = torch.empty_like(s["gate"]) if case["gate_rows"] else None
    else:
        b, nq, nk, d = case["seqs"], case["q_rows"], case["k_rows"], case["head_dim"]
        hq, hk, t = case["q_heads"], case["k_heads"], case["dtype"]
        if case["packed"]:
            s["qkv"] = _heads(g, b, nq, [hq, hk, hk], d, t, True)
        else:
            s["qkv"] = _heads(g, b, nq, [hq], d, t, False) + _heads(g, b, nk, [hk, hk], d, t, False)
        ql, kl = _lens(case)
        s["q_len"] = torch.tensor(ql, dtype=torch.int32, device=DEV)
        s["k_len"] = torch.tensor(kl, dtype=torch.int32, device=DEV)
        s["out"] = torch.empty(b, nq, hq, d, dtype=TYPES[t], device=DEV)
        s["lse"] = torch.empty(b, hq, nq, device=DEV)
        if case["train"]:
            s["dout"] = _heads(g, b, nq, [hq], d, t, False, 0.1)[0]
            s["grads"] = _like(s["qkv"], case["packed"])
    return s


# ------------------------------------------------------------------ the plain forms
def _rotate(x, cos, sin, layout):
    r = 2 * cos.shape[-1]
    if layout == "half":
        a, b = x[..., : r // 2], x[..., r // 2: r]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., r:]), -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), x[..., r:]), -1)


def _plain_rope(s):
    c = s["case"]
    phase = s["positions"].long()[..., None] * s["turns"]  # modulo 2^64
    angle = (phase >> 32).float() * (2 * math.pi / 2.0 ** 32)
    cos, sin = torch.cos(angle)[:, :, None] * s["factor"], torch.sin(angle)[:, :, None] * s["factor"]
    if c["transpose"]:
        sin = -sin
    return [_rotate(x.float(), cos, sin, c["layout"]).to(x.dtype) for x in s["x"]]


EPS = 1e-5


def _plain_hat(x, kind):
    """The normalised rows and 1 / their deviation."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * rstd, rstd


def _plain_norm_forward(s):
    c = s["case"]
    u = s["block"].float()
    if c["post"] != "none":
        u = _plain_hat(u, c["post"])[0] * s["post_w"] + (s["post_b"] if c["post"] == "layer" else 0.0)
    if c["gate_rows"]:
        u = u * s["gate"].repeat_interleave(c["gate_rows"], 0)[: c["rows"]]
    r = s["x"].float() + s["scale"] * u
    y = _plain_hat(r, c["pre"])[0] * s["pre_w"] + (s["pre_b"] if c["pre"] == "layer" else 0.0)
    return [r.to(s["x"].dtype), y.to(s["block"].dtype)]


def _plain_hat_grad(g, hat, rstd, kind):
    d = g - hat * (g * hat).mean(-1, keepdim=True)
    return rstd * (d - g.mean(-1, keepdim=True) if kind == "layer" else d)


def _plain_norm_backward(s):
    c = s["case"]
    dy, hat_r = s["dy"].float(), _plain_hat(s["r"].float(), c["pre"])
    dr = s["dr"].float() + _plain_hat_grad(dy * s["pre_w"], *hat_r, c["pre"])
    out = {"dx": dr.to(s["r"].dtype), "dpre_w": (dy * hat_r[0]).sum(0)}
    if c["pre"] == "layer":
        out["dpre_b"] = dy.sum(0)
    b = s["block"].float()
    u = b
    if c["post"] != "none":
        hat_b = _plain_hat(b, c["post"])
        u = hat_b[0] * s["post_w"] + (s["post_b"] if c["post"] == "layer" else 0.0)
    du = s["scale"] * dr
    if c["gate_rows"]:
        n = s["gate"].shape[0]
        t = torch.zeros(n * c["gate_rows"], c["cols"], device=DEV)
        t[: c["rows"]] = du * u
        out["dgate"] = t.view(n, c["gate_rows"], -1).sum(1)
        du = du * s["gate"].repeat_interleave(c["gate_rows"], 0)[: c["rows"]]
    if c["post"] != "none":
        out["dpost_w"] = (du * hat_b[0]).sum(0)
        if c["post"] == "layer":
            out["dpost_b"] = du.sum(0)
        du = _plain_hat_grad(du * s["post_w"], *hat_b, c["post"])
    out["dblock"] = du.to(s["block"].dtype)
    return out


def _allowed(s):
    """[seqs, 1, q_rows, k_rows]: which keys each query row sees."""
    c = s["case"]
    i = torch.arange(c["q_rows"], device=DEV)[:, None]
    j = torch.arange(c["k_rows"], device=DEV)[None, :]
    far = j - i - _offset(c)
    ok = (i < s["q_len"][:, None, None]) & (j < s["k_len"][:, None, None])
    if c["right"] >= 0:
        ok = ok & (far <= c["right"])
    if c["left"] >= 0:
        ok = ok & (-far <= c["left"])
    return ok[:, None]


def _plain_attention(s):
    c = s["case"]
    group, scale = c["q_heads"] // c["k_heads"], c["head_dim"] ** -0.5
    q, k, v = (t.float().transpose(1, 2) for t in s["qkv"])
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    scores = (q @ k.transpose(-1, -2) * scale).masked_fill(~_allowed(s), -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    del scores
    total = p.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(-1)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = p @ v
    out = {"out": o.transpose(1, 2).to(s["out"].dtype), "lse": lse}
    if c["train"]:
        do = s["dout"].float().transpose(1, 2)
        dv = p.transpose(-1, -2) @ do
        ds = (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True)) * p * scale
        dq, dk = ds @ k, ds.transpose(-1, -2) @ q
        b, _, n, d = dk.shape
        dk, dv = (t.view(b, -1, group, n, d).sum(2) for t in (dk, dv))
        out.update((name, t.transpose(1, 2).to(s["out"].dtype)) for name, t in (("dq", dq), ("dk", dk), ("dv", dv)))
    return out


# ------------------------------------------------------------- the repository's entry points
@functools.lru_cache(maxsize=None)
def _package():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                    "nemotron3-diarization-wgpu_b200"))
    import n3d

    return n3d


@functools.lru_cache(maxsize=None)
def _rope_plan(items):
    return _package().RopePlan(**dict(items))


def _own_rope(s):
    n3d, c = _package(), s["case"]
    n3d.rope(_rope_plan(tuple(_rope_config(c).items())), s["x"], s["y"], positions=s["positions"],
             transpose=c["transpose"], stream=torch.cuda.current_stream().cuda_stream)
    return s["y"]


def _own_norm(s):
    n3d, c = _package(), s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    layer_post, layer_pre = c["post"] == "layer", c["pre"] == "layer"
    common = dict(post=c["post"], pre=c["pre"], eps=EPS, scale=s["scale"], gate=s["gate"], gate_rows=c["gate_rows"],
                  post_w=s["post_w"] if c["post"] != "none" else None, post_b=s["post_b"] if layer_post else None,
                  pre_w=s["pre_w"], pre_b=s["pre_b"] if layer_pre else None, stream=stream)
    if c["direction"] == "forward":
        n3d.residual_norm(s["x"], s["block"], s["r"], s["y"], **common)
        return [s["r"], s["y"]]
    w = s["dw"]
    need = n3d.residual_norm_workspace(c["rows"], c["cols"], c["gate_rows"])
    space = torch.empty(need, dtype=torch.uint8, device=DEV)
    out = {"dx": s["dx"], "dblock": s["dblock"], "dpre_w": w[2]}
    if layer_pre:
        out["dpre_b"] = w[3]
    if c["post"] != "none":
        out["dpost_w"] = w[0]
    if layer_post:
        out["dpost_b"] = w[1]
    if c["gate_rows"]:
        out["dgate"] = s["dgate"]
    n3d.residual_norm_grad(s["block"], s["r"], s["dy"], s["dr"], out["dx"], out["dblock"], dgate=out.get("dgate"),
                           dpost_w=out.get("dpost_w"), dpost_b=out.get("dpost_b"), dpre_w=out["dpre_w"],
                           dpre_b=out.get("dpre_b"), workspace=space, **common)
    return out


def _own_attention(s):
    n3d, c = _package(), s["case"]
    kw = dict(q_len=s["q_len"], k_len=s["k_len"], left=c["left"], right=c["right"], q_offset=_offset(c),
              stream=torch.cuda.current_stream().cuda_stream)
    q, k, v = s["qkv"]
    kw["workspace"] = torch.empty(n3d.attention_workspace(q, k, c["train"]), dtype=torch.uint8, device=DEV)
    n3d.attention_forward(q, k, v, s["out"], s["lse"], **kw)
    out = {"out": s["out"], "lse": s["lse"]}
    if c["train"]:
        dq, dk, dv = s["grads"]
        n3d.attention_backward(q, k, v, s["out"], s["lse"], s["dout"], dq, dk, dv, **kw)
        out.update(dq=dq, dk=dk, dv=dv)
    return out


def run(state):
    c = state["case"]
    if c["op"] == "rope":
        return _own_rope(state) if own else _plain_rope(state)
    if c["op"] == "norm":
        if own:
            return _own_norm(state)
        return _plain_norm_forward(state) if c["direction"] == "forward" else _plain_norm_backward(state)
    return _own_attention(state) if own else _plain_attention(state)


# ------------------------------------------------------------------------------- work
def _pairs(case):
    """(query, key) pairs that the masks let through, in all sequences, per query head."""
    n, off = 0, _offset(case)
    for ql, kl in set(zip(*_lens(case))):
        count = list(zip(*_lens(case))).count((ql, kl))
        for i in range(ql):
            lo = max(0, i + off - case["left"]) if case["left"] >= 0 else 0
            hi = min(kl, i + off + case["right"] + 1) if case["right"] >= 0 else kl
            n += count * max(0, hi - lo)
    return n


def work(case):
    if case["op"] == "rope":
        n = case["seqs"] * case["rows"]
        heads = case["q_heads"] + case["k_heads"]
        return {"bytes": n * (2 * heads * case["head_dim"] * BYTES[case["dtype"]] + 4),
                "flops": n * heads * case["rotary_dim"] * 3}
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        r, b = BYTES[case["residual"]], BYTES[case["block"]]
        groups = -(-case["rows"] // case["gate_rows"]) if case["gate_rows"] else 0
        if case["direction"] == "forward":  # x, block -> r, y
            return {"bytes": n * (2 * r + 2 * b) + 4 * case["cols"] * (4 + groups), "flops": 16 * n}
        # r, dr, block, dy -> dx, dblock
        return {"bytes": n * (3 * r + 3 * b) + 4 * case["cols"] * (7 + 2 * groups), "flops": 40 * n}
    p, d, t = _pairs(case), case["head_dim"], BYTES[case["dtype"]]
    qn = case["seqs"] * case["q_rows"] * case["q_heads"]
    kn = case["seqs"] * case["k_rows"] * case["k_heads"]
    size = (2 * qn + 2 * kn) * d * t + 4 * qn  # q, out, k, v, lse
    if case["train"]:
        size += (2 * qn + 2 * kn) * d * t  # dout, dq, dk, dv
    return {"bytes": size, "flops": (14 if case["train"] else 4) * p * d * case["q_heads"]}


# ------------------------------------------------------------------------------ 64 bits
def _exact_rope(s):
    c = s["case"]
    f, factor = _frequencies(_rope_config(c))
    angle = s["positions"].double()[..., None] * torch.tensor(f, dtype=torch.float64, device=DEV)
    turn = torch.polar(torch.full_like(angle, factor), -angle if c["transpose"] else angle)[:, :, None]
    got, r = [], c["rotary_dim"]
    for x in s["x"]:
        y = x.double()
        if c["layout"] == "half":
            z = torch.complex(y[..., : r // 2].contiguous(), y[..., r // 2: r].contiguous()) * turn
            y[..., :r] = torch.cat((z.real, z.imag), -1)
        else:
            z = torch.view_as_complex(y[..., :r].unflatten(-1, (-1, 2)).contiguous()) * turn
            y[..., :r] = torch.view_as_real(z).flatten(-2)
        got.append(y)
    return got


def _exact_boundary(s, block, x, gate, w):
    """r and y in 64 bits, differentiable in every argument."""
    c = s["case"]

    def norm(t, kind, weight, bias):
        if kind == "none":
            return t
        if kind == "rms":
            return weight * t / torch.sqrt(t.pow(2).mean(1, keepdim=True) + EPS)
        return weight * (t - t.mean(1, keepdim=True)) / torch.sqrt(t.var(1, unbiased=False, keepdim=True) + EPS) + bias

    u = norm(block, c["post"], w[0], w[1])
    if gate is not None:
        u = u * gate[torch.arange(c["rows"], device=DEV) // c["gate_rows"]]
    r = x + s["scale"] * u
    return r, norm(r, c["pre"], w[2], w[3])


def _exact_norm(s):
    c = s["case"]
    w = [s[n].double().requires_grad_() for n in ("post_w", "post_b", "pre_w", "pre_b")]
    gate = s["gate"].double().requires_grad_() if c["gate_rows"] else None
    block = s["block"].double().requires_grad_()
    if c["direction"] == "forward":
        with torch.no_grad():
            return list(_exact_boundary(s, block, s["x"].double(), gate, w))
    # the residual stream that leads to the r at hand
    with torch.no_grad():
        x = s["r"].double() - _exact_boundary(s, block, torch.zeros_like(block), gate, w)[0]
    x.requires_grad_()
    r, y = _exact_boundary(s, block, x, gate, w)
    torch.autograd.backward([r, y], [s["dr"].double(), s["dy"].double()])
    out = {"dx": x.grad, "dblock": block.grad, "dpre_w": w[2].grad}
    if c["pre"] == "layer":
        out["dpre_b"] = w[3].grad
    if c["post"] != "none":
        out["dpost_w"] = w[0].grad
    if c["post"] == "layer":
        out["dpost_b"] = w[1].grad
    if c["gate_rows"]:
        out["dgate"] = gate.grad
    return out


def _exact_attention(s):
    c = s["case"]
    group, off = c["q_heads"] // c["k_heads"], _offset(c)
    qkv = [t.double() for t in s["qkv"]]
    b, nq, hq, d = qkv[0].shape
    out = {"out": torch.zeros_like(qkv[0]), "lse": torch.full((b, hq, nq), -math.inf, dtype=torch.float64, device=DEV)}
    if c["train"]:
        out.update(dq=torch.zeros_like(qkv[0]), dk=torch.zeros_like(qkv[1]), dv=torch.zeros_like(qkv[2]))
    for i, (ql, kl) in enumerate(zip(*_lens(c))):
        at = torch.arange(ql, device=DEV) + off
        lo = (at - c["left"]).clamp(min=0) if c["left"] >= 0 else torch.zeros_like(at)
        hi = (at + c["right"] + 1).clamp(max=kl) if c["right"] >= 0 else torch.full_like(at, kl)
        some = (hi > lo).nonzero()[:, 0]  # the rows that see a key
        if not len(some):
            continue
        j = torch.arange(kl, device=DEV)
        hide = (j < lo[some, None]) | (j >= hi[some, None])
        for h in range(hq):
            q = qkv[0][i, some, h].requires_grad_(c["train"])
            k, v = (t[i, :kl, h // group].clone().requires_grad_(c["train"]) for t in qkv[1:])
            score = (q @ k.T / math.sqrt(d)).masked_fill(hide, -math.inf)
            o = torch.softmax(score, 1) @ v
            out["out"][i, some, h] = o.detach()
            out["lse"][i, h, some] = torch.logsumexp(score.detach(), 1)
            if c["train"]:
                o.backward(s["dout"][i, some, h].double())
                out["dq"][i, some, h] = q.grad
                out["dk"][i, :kl, h // group] += k.grad
                out["dv"][i, :kl, h // group] += v.grad
            del score, o
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(s)
    return _exact_norm(s) if case["op"] == "norm" else _exact_attention(s)

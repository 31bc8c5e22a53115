"""examples/finetune_block.py: the training operators together.  Its gradients against automatic
differentiation of the same block in 64 bits, and a loss that falls.

Tolerance, derived: in bf16 the block's intermediate tensors (h, qkv, rotated q and k, ctx, o,
y, dy and the gradients between the operators, a dozen in a row) are each rounded by up to
2^-9 of an element's size (2^-8 of its leading bit); independent roundings of a dozen
tensors add up to sqrt(12) 2^-9 < 1 % of a gradient's norm, and the products mix them: 3 %
is asked for.  In fp32 each is good to 1e-6; 12 of them and torch's fp32 products: 2e-5."""

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load():
    spec = importlib.util.spec_from_file_location("finetune_block", os.path.join(ROOT, "examples", "finetune_block.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def reference(m, block, x, prev, target, lens):
    """Gradients of the parameters and of x in 64 bits."""
    import torch

    p = {n: v.double().requires_grad_() for n, v in block.p.items()}
    x = x.double().requires_grad_()
    b, s, w = block.b, block.s, m.WIDTH
    norm = lambda t, wt, bs: torch.nn.functional.layer_norm(t, (w,), wt, bs, 1e-5)
    r = x + p["gate"] * prev.double()
    qkv = (norm(r, p["w1"], p["b1"]) @ p["wqkv"].T).view(b, s, 3 * m.HEADS, m.HEAD_DIM)
    q, k, v = qkv.split(m.HEADS, 2)
    half = m.HEAD_DIM // 2
    angle = torch.arange(s, device=x.device)[:, None] * 10000.0 ** (-torch.arange(half, device=x.device).double() / half)
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    turn = lambda t: torch.cat((t[..., :half] * cos - t[..., half:] * sin, t[..., half:] * cos + t[..., :half] * sin), -1)
    seen = torch.arange(s, device=x.device) < lens[:, None]
    score = torch.einsum("bihd,bjhd->bhij", turn(q), turn(k)) * m.HEAD_DIM ** -0.5
    prob = torch.softmax(score.masked_fill(~seen[:, None, None], -torch.inf), -1) * seen[:, None, :, None]
    o = torch.einsum("bhij,bjhd->bihd", prob, v).reshape(b * s, w) @ p["wo"].T
    y = norm(r + p["gate2"] * o, p["w2"], p["b2"])
    live = seen.reshape(b * s, 1)
    (((y - target.double()) * live).square().sum() / (live.sum() * w)).backward()
    return {**{n: v.grad for n, v in p.items()}, "x": x.grad}


@pytest.mark.parametrize("dtype,limit", [("bfloat16", 0.03), ("float16", 0.03), ("float32", 2e-5)])
def test_gradients_of_the_block(dtype, limit):
    import torch

    import n3d

    m = load()
    block = m.Block(3, 150, getattr(torch, dtype), seed=4)
    data = m.batch(block, 5)
    block.step(*data)
    torch.cuda.synchronize()
    n3d.train_status(0)
    want = reference(m, block, *data)
    got = {**block.grads, "x": block.dx}
    for n, w in want.items():
        off = ((got[n].double() - w).norm() / w.norm()).item()
        assert off <= limit, (n, off)


def test_the_loss_falls():
    import torch

    m = load()
    block = m.Block(8, 100)
    data = m.batch(block, 2)
    losses = []
    for _ in range(15):
        losses.append(block.step(*data).item())
        block.update(100.0)
    torch.cuda.synchronize()
    assert losses[-1] < 0.9 * losses[0] and all(b < a for a, b in zip(losses, losses[1:]))

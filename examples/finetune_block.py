"""Fine-tunes one attention block of the encoder on synthetic windows.

The training operators of include/n3d.h as a training step uses them, on windows of uneven
length with the encoder's sizes (8 heads of 64, width 512):

    r = x + gate * prev,  h = LayerNorm(r)              residual_norm
    q, k, v = h Wqkv^T                                  (linear layer: torch)
    q, k = rotary(q, k)                                 rope, in place in the packed buffer
    c = attention(q, k, v)                              attention_forward
    o = c Wo^T                                          (linear layer: torch)
    r2 = r + gate2 * o,  y = LayerNorm(r2)              residual_norm
    loss = mean square of y - target over the windows' frames

and back through the same operators' gradients.  Weights, gates and the residual stream are
fp32, blocks are bf16 (or --dtype float32 / float16).

    python examples/finetune_block.py [--steps N] [--windows B] [--frames S] [--dtype T]
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "nemotron3-diarization-wgpu_b200"))
import n3d  # noqa: E402

HEADS, HEAD_DIM = 8, 64
WIDTH = HEADS * HEAD_DIM


class Block:
    """Parameters, buffers and one training step of the block."""

    def __init__(self, windows: int, frames: int, dtype=torch.bfloat16, seed: int = 0, device: str = "cuda:0"):
        g = torch.Generator(device=device).manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device=device)
        self.p = {"wqkv": rnd(3 * WIDTH, WIDTH) * 0.04, "wo": rnd(WIDTH, WIDTH) * 0.04, "gate": 0.5 + 0.1 * rnd(WIDTH),
                  "gate2": 0.5 + 0.1 * rnd(WIDTH), "w1": torch.ones(WIDTH, device=device),
                  "b1": torch.zeros(WIDTH, device=device), "w2": torch.ones(WIDTH, device=device),
                  "b2": torch.zeros(WIDTH, device=device)}
        self.b, self.s, self.dtype = windows, frames, dtype
        # a mean over many frames has gradients below fp16's normal range: they travel multiplied by this
        self.loss_scale = 2.0 ** 12 if dtype == torch.float16 else 1.0
        self.plan = n3d.RopePlan(HEAD_DIM)
        rows, e = windows * frames, lambda *sh, t=dtype: torch.empty(*sh, dtype=t, device=device)
        self.r, self.r2, self.dr, self.dx = (e(rows, WIDTH, t=torch.float32) for _ in range(4))
        self.h, self.y, self.do, self.dprev = (e(rows, WIDTH) for _ in range(4))
        self.ctx = e(windows, frames, HEADS, HEAD_DIM)
        self.lse = e(windows, HEADS, frames, t=torch.float32)
        self.dqkv = e(windows, frames, 3 * HEADS, HEAD_DIM)
        self.grads = {n: torch.empty_like(v) for n, v in self.p.items()}
        heads = self.dqkv.split(HEADS, 2)
        self.attn_space = e(max(16, n3d.attention_workspace(heads[0], heads[1])), t=torch.uint8)
        self.norm_space = e(n3d.residual_norm_workspace(rows, WIDTH, rows), t=torch.uint8)

    def step(self, x, prev, target, lens) -> torch.Tensor:
        """One forward and backward pass; the gradients are in self.grads and self.dx, and that of prev, still times
        self.loss_scale, in self.dprev.  x fp32 [rows, 512], prev and target [rows, 512] of the block's type, lens
        int32 [windows].  Returns the loss."""
        p, g, rows = self.p, self.grads, self.b * self.s
        st = torch.cuda.current_stream().cuda_stream
        norm1 = dict(gate=p["gate"], gate_rows=rows, pre_w=p["w1"], pre_b=p["b1"], stream=st)
        norm2 = dict(gate=p["gate2"], gate_rows=rows, pre_w=p["w2"], pre_b=p["b2"], stream=st)
        attn = dict(q_len=lens, k_len=lens, workspace=self.attn_space, stream=st)
        wqkv, wo = p["wqkv"].to(self.dtype), p["wo"].to(self.dtype)

        n3d.residual_norm(x, prev, self.r, self.h, **norm1)
        q, k, v = (self.h @ wqkv.T).view(self.b, self.s, 3 * HEADS, HEAD_DIM).split(HEADS, 2)
        n3d.rope(self.plan, [q, k], [q, k], stream=st)
        n3d.attention_forward(q, k, v, self.ctx, self.lse, **attn)
        ctx = self.ctx.view(rows, WIDTH)
        o = ctx @ wo.T
        n3d.residual_norm(self.r, o, self.r2, self.y, **norm2)

        live = (torch.arange(self.s, device=x.device) < lens[:, None]).view(rows, 1)
        off = (self.y.float() - target.float()) * live
        count = live.sum() * WIDTH
        loss = off.square().sum() / count
        dy = (off * (2.0 * self.loss_scale / count)).to(self.dtype)

        n3d.residual_norm_grad(o, self.r2, dy, None, self.dr, self.do, dgate=g["gate2"], dpre_w=g["w2"], dpre_b=g["b2"],
                               workspace=self.norm_space, **norm2)
        g["wo"].copy_(self.do.T @ ctx)
        dctx = (self.do @ wo).view_as(self.ctx)
        dq, dk, dv = self.dqkv.split(HEADS, 2)
        n3d.attention_backward(q, k, v, self.ctx, self.lse, dctx, dq, dk, dv, **attn)
        n3d.rope(self.plan, [dq, dk], [dq, dk], transpose=True, stream=st)
        dqkv = self.dqkv.view(rows, 3 * WIDTH)
        g["wqkv"].copy_(dqkv.T @ self.h)
        n3d.residual_norm_grad(prev, self.r, dqkv @ wqkv, self.dr, self.dx, self.dprev, dgate=g["gate"], dpre_w=g["w1"],
                               dpre_b=g["b1"], workspace=self.norm_space, **norm1)
        if self.loss_scale != 1.0:
            for t in (*g.values(), self.dx):
                t.mul_(1.0 / self.loss_scale)
        return loss

    def update(self, rate: float) -> None:
        """Gradient descent on every parameter."""
        for n, v in self.p.items():
            v.add_(self.grads[n], alpha=-rate)


def batch(block: Block, seed: int):
    """Synthetic windows: embeddings, the previous block's output, targets, lengths (40..100 % of the frames)."""
    dev = block.r.device
    g = torch.Generator(device=dev).manual_seed(seed)
    rows = block.b * block.s
    x = torch.randn(rows, WIDTH, generator=g, device=dev)
    prev, target = (torch.randn(rows, WIDTH, generator=g, device=dev).to(block.dtype) for _ in range(2))
    lens = (block.s * (0.4 + 0.6 * torch.rand(block.b, generator=g, device=dev))).round().clamp(min=1).to(torch.int32)
    return x, prev, target, lens


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--windows", type=int, default=64)
    ap.add_argument("--frames", type=int, default=376)
    ap.add_argument("--dtype", default="bfloat16", choices=("float32", "bfloat16", "float16"))
    ap.add_argument("--rate", type=float, default=200.0)
    a = ap.parse_args()
    block = Block(a.windows, a.frames, getattr(torch, a.dtype))
    data = batch(block, 1)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for i in range(a.steps):
        start.record()
        loss = block.step(*data)
        block.update(a.rate)
        end.record()
        end.synchronize()
        print(f"step {i}: loss {loss.item():.5f}  {start.elapsed_time(end):.3f} ms")
    n3d.train_status(0)


if __name__ == "__main__":
    main()

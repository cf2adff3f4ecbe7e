"""A transformer layer's feed-forward half on the library's operators: forward, backward, one token.

    h = layer_norm(x) * gamma + beta
    y = x + W2 act(W1 h + b1) + b2

Run it on a B200 (`python examples/feed_forward.py --steps 50`): it fits the layer to a fixed target
with plain gradient steps, prints the loss as it falls, then runs the trained layer on a single token,
as a streaming caller does.  Every number on the way is computed by the library; torch only holds the
tensors and applies the weight updates.
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "prime-tts_b200"))
import pt_b200  # noqa: E402


class FeedForward:
    """Weights [width] -> [inner] -> [width]; the text encoder's sizes are 192 and 768."""

    def __init__(self, ops, width=192, inner=768, act="gelu", dtype=torch.float32, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape, std):
            return (std * torch.randn(*shape, generator=gen, device="cuda")).to(dtype)

        self.ops, self.act = ops, act
        self.p = {"gamma": torch.ones(width, device="cuda", dtype=dtype),
                  "beta": torch.zeros(width, device="cuda", dtype=dtype),
                  "w1": normal(inner, width, std=1 / math.sqrt(width)),
                  "b1": torch.zeros(inner, device="cuda", dtype=dtype),
                  "w2": normal(width, inner, std=1 / math.sqrt(inner)),
                  "b2": torch.zeros(width, device="cuda", dtype=dtype)}

    def forward(self, x, keep=False):
        """y, and with `keep` what backward() needs."""
        p, ops = self.p, self.ops
        h, mean, rstd = ops.layer_norm(x, p["gamma"], p["beta"])
        if not keep:
            return ops.linear(ops.linear(h, p["w1"], p["b1"], act=self.act), p["w2"], p["b2"], residual=x)
        z, pre = ops.linear(h, p["w1"], p["b1"], act=self.act, save_pre=True)
        y = ops.linear(z, p["w2"], p["b2"], residual=x)
        return y, (x, mean, rstd, h, pre, z)

    def backward(self, dy, kept):
        """The gradients of the weights by name, and that of x."""
        p, ops = self.p, self.ops
        x, mean, rstd, h, pre, z = kept
        g = {}
        dz, g["w2"], g["b2"] = ops.linear_backward(dy, z, p["w2"])
        dh, g["w1"], g["b1"] = ops.linear_backward(dz, h, p["w1"], pre=pre, act=self.act)
        dx, g["gamma"], g["beta"] = ops.layer_norm_backward(dh, x, p["gamma"], mean, rstd)
        return g, dx + dy          # the residual path


def train(layer, x, target, steps, rate):
    """Plain gradient steps on the mean squared error; the losses."""
    losses = []
    for _ in range(steps):
        y, kept = layer.forward(x, keep=True)
        diff = y.float() - target.float()
        losses.append(diff.square().mean())
        grads, _ = layer.backward((diff * (2.0 / diff.numel())).to(y.dtype), kept)
        for name, g in grads.items():
            layer.p[name] -= rate * g
    return [v.item() for v in losses]


def main():
    a = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    a.add_argument("--rows", type=int, default=512)
    a.add_argument("--steps", type=int, default=50)
    a.add_argument("--dtype", choices=("float32", "bfloat16", "float16"), default="float32")
    a = a.parse_args()
    ops = pt_b200.Operators(device=0)
    dtype = getattr(torch, a.dtype)
    layer = FeedForward(ops, dtype=dtype)
    teacher = FeedForward(ops, dtype=dtype, seed=1)
    x = torch.randn(a.rows, 192, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(dtype)
    losses = train(layer, x, teacher.forward(x), a.steps, rate=2.0)
    ops.sync()
    for i in range(0, a.steps, max(1, a.steps // 10)):
        print(f"step {i:4d}  loss {losses[i]:.5f}")
    print(f"step {a.steps - 1:4d}  loss {losses[-1]:.5f}")
    whole, token = layer.forward(x), layer.forward(x[3:4])
    ops.sync()
    print(f"one token against its row of the batch: {(token[0] - whole[3]).abs().max().item():.2g}")


if __name__ == "__main__":
    main()

"""A residual attention layer over image or video tokens: LayerNorm, one
projection to q, k and v, rotary positions over the token's coordinates,
differential attention with a norm per head, and the output projection.

``DiffLayer.forward`` / ``backward`` train it (gradients accumulate in
``grads``, ``step`` is the framework's AdamW and Muon), ``extend`` answers new
tokens against a ``Cache`` of earlier ones.  Activations are float32 like the
framework's other layers; with ``dtype=torch.bfloat16`` q, k, v and the cache
are bfloat16.

    python -m rustnn_b200.diff [--steps 60] [--bf16]

trains one layer to predict the next token of synthetic clips (a pattern that
drifts over a grid), prints the loss, and checks that tokens answered one at a
time give what the whole clip gave.
"""
from __future__ import annotations

import argparse

import torch

from . import ops
from .ops import RnnError


def grid_positions(frames, height, width, device="cuda"):
    """[frames * height * width, 3] int32 coordinates (time, row, column)."""
    axes = (torch.arange(s, dtype=torch.int32, device=device) for s in (frames, height, width))
    return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(-1, 3).contiguous()


def axis_frequencies(pairs, base=100.0, device="cuda"):
    """inv_freq of rope for pairs[a] pairs on each axis: base ** (-j / pairs[a])."""
    return torch.tensor([base ** (-j / p) for p in pairs for j in range(p)], dtype=torch.float32, device=device)


class Cache:
    """Keys (rotated) and values of up to `size` tokens of n sequences."""

    def __init__(self, layer, n, size):
        shape = (n, size, layer.h, 2 * layer.dh)
        self.k = torch.empty(shape, device=layer.device, dtype=layer.dtype)
        self.v = torch.empty(shape, device=layer.device, dtype=layer.dtype)
        self.length = 0  # tokens held; the same for all sequences


class DiffLayer:
    """y = x + (norm(attention(norm(x))) Wo^T): h heads of 2 * dh columns over c = 2 * h * dh channels."""

    def __init__(self, h, dh, pairs, seed=0, lam=0.5, dtype=torch.float32, causal=True, device="cuda"):
        if 2 * sum(pairs) > dh:
            raise RnnError(f"{sum(pairs)} pairs do not fit halves of {dh} columns")
        self.h, self.dh, self.c, self.pairs, self.dtype = h, dh, 2 * h * dh, tuple(pairs), dtype
        self.causal, self.device = "end" if causal else None, device
        self.freq = axis_frequencies(pairs, device=device)
        c, g = self.c, torch.Generator(device=device).manual_seed(seed)

        def normal(*shape):
            return torch.randn(*shape, device=device, generator=g) * shape[-1] ** -0.5

        self.params = {
            "ln_g": torch.ones(c, device=device), "ln_b": torch.zeros(c, device=device),
            "wqkv": normal(3 * c, c), "bqkv": torch.zeros(3 * c, device=device),
            "lam": torch.full((h,), lam, device=device),
            "hn_g": torch.ones(2 * dh, device=device), "hn_b": torch.zeros(2 * dh, device=device),
            "wo": normal(c, c), "bo": torch.zeros(c, device=device),
        }
        self.grads = {k: torch.zeros_like(v) for k, v in self.params.items()}
        self.moments = {k: (torch.zeros_like(v), torch.zeros_like(v)) for k, v in self.params.items()}
        self.steps = 0

    def _project(self, x, n, t, pos):
        """LayerNorm, projection and rotation of n * t tokens; (q, k, v, saved)."""
        p, c = self.params, self.c
        y, xhat, inv = ops.layernorm_forward(x, n * t, c, p["ln_g"], p["ln_b"])
        qkv = ops.linear_forward(y, n * t, c, 3 * c, p["wqkv"], p["bqkv"]).to(self.dtype)
        # q and k: 4 * h halves of dh columns each, rotated in place
        halves = qkv.view(n * t, 6 * self.h, self.dh)[:, : 4 * self.h]
        ops.rope(halves, pos, self.freq, self.pairs, out=halves)
        parts = qkv.view(n, t, 3, self.h, 2 * self.dh)
        return parts[:, :, 0], parts[:, :, 1], parts[:, :, 2], (y, xhat, inv)

    def _answer(self, x, o, n, t):
        """Norm of each head, output projection and the residual."""
        p, c = self.params, self.c
        o = o.float().contiguous()
        z, zhat, zinv = ops.layernorm_forward(o, n * t * self.h, 2 * self.dh, p["hn_g"], p["hn_b"])
        y = ops.linear_forward(z.view(-1), n * t, c, c, p["wo"], p["bo"])
        return ops.add_(y, x), (z, zhat, zinv)

    def forward(self, x, n, t, pos, klen=None):
        """x [n * t * c] float32; pos [n * t, axes] int32; klen [n] int32 for ragged
        clips.  Returns y like x and keeps what backward needs."""
        q, k, v, head = self._project(x, n, t, pos)
        causal = "start" if self.causal else None
        o, o2, lse = ops.diffattn_forward(q, k, v, self.params["lam"], causal=causal, klen=klen, save=True)
        y, tail = self._answer(x, o, n, t)
        self.saved = (n, t, pos, klen, causal, q, k, v, o, o2, lse, head, tail)
        return y

    def backward(self, dy):
        """Accumulates the gradients of the last forward; returns dx."""
        n, t, pos, klen, causal, q, k, v, o, o2, lse, (y, xhat, inv), (z, zhat, zinv) = self.saved
        p, g, c = self.params, self.grads, self.c
        dz = ops.linear_backward(z.view(-1), dy, n * t, c, c, p["wo"], g["wo"], g["bo"])
        do = ops.layernorm_backward(dz, zhat, zinv, n * t * self.h, 2 * self.dh, p["hn_g"], g["hn_g"], g["hn_b"])
        dqkv = torch.empty((n, t, 3, self.h, 2 * self.dh), device=self.device, dtype=self.dtype)
        ops.diffattn_backward(do.view(o.shape).to(self.dtype), q, k, v, p["lam"], o, o2, lse, g["lam"], causal=causal,
                              klen=klen, dq=dqkv[:, :, 0], dk=dqkv[:, :, 1], dv=dqkv[:, :, 2])
        halves = dqkv.view(n * t, 6 * self.h, self.dh)[:, : 4 * self.h]
        ops.rope_backward(halves, pos, self.freq, self.pairs, out=halves)
        dln = ops.linear_backward(y, dqkv.float().view(-1), n * t, c, 3 * c, p["wqkv"], g["wqkv"], g["bqkv"])
        dx = ops.layernorm_backward(dln, xhat, inv, n * t, c, p["ln_g"], g["ln_g"], g["ln_b"])
        return ops.add_(dx, dy)

    def step(self, lr=1e-3, wd=0.0):
        """Muon for the two matrices, AdamW for the rest; gradients return to zero."""
        for name, v in self.params.items():
            g, (m, m2) = self.grads[name], self.moments[name]
            if v.dim() == 2:
                ops.muon_step_(v, g, m, v.shape[0], v.shape[1], 3, 10 * lr, wd=wd)
            else:
                ops.adamw_step_(v, g, m, m2, lr, wd, False, self.steps)
        self.steps += 1

    def extend(self, x, n, t, pos, cache):
        """Answers t new tokens of each of n sequences and adds them to the cache."""
        if cache.length + t > cache.k.shape[1]:
            raise RnnError(f"cache holds {cache.k.shape[1]} tokens, {cache.length + t} needed")
        q, k, v, _ = self._project(x, n, t, pos)
        end = cache.length + t
        cache.k[:, cache.length:end].copy_(k)
        cache.v[:, cache.length:end].copy_(v)
        cache.length = end
        o = ops.diffattn_forward(q, cache.k[:, :end], cache.v[:, :end], self.params["lam"], causal=self.causal)
        return self._answer(x, o, n, t)[0]


def clips(n, frames, side, c, seed, device="cuda"):
    """Tokens [n, frames * side * side, c] of waves that drift over the grid, one drift a clip."""
    g = torch.Generator(device=device).manual_seed(seed)
    pos = grid_positions(frames, side, side, device).float()
    speed = torch.rand(n, 1, 2, device=device, generator=g) * 2 - 1
    where = pos[None, :, 1:] + speed * pos[None, :, :1]
    wave = torch.rand(2, c, device=device, generator=torch.Generator(device=device).manual_seed(1)) * 2
    return torch.sin(where @ wave + torch.arange(c, device=device))


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--frames", type=int, default=4)
    ap.add_argument("--side", type=int, default=8)
    ap.add_argument("--bf16", action="store_true", help="q, k, v and the cache in bfloat16")
    args = ap.parse_args()
    n, t = args.batch, args.frames * args.side * args.side
    layer = DiffLayer(h=4, dh=32, pairs=(4, 6, 6), dtype=torch.bfloat16 if args.bf16 else torch.float32)
    pos = grid_positions(args.frames, args.side, args.side)
    all_pos = pos.repeat(n, 1)
    for i in range(args.steps):
        x = clips(n, args.frames, args.side, layer.c, i)
        target = torch.cat([x[:, 1:], x[:, :1] * 0], 1).contiguous().view(-1)
        y = layer.forward(x.view(-1), n, t, all_pos)
        dy = torch.zeros_like(y)
        loss = ops.hint_mse(y, target, n * t, layer.c, 1.0, dy)
        layer.backward(dy)
        layer.step()
        if i % 10 == 0 or i + 1 == args.steps:
            print(f"step {i}: loss {float(loss):.5f}")
    x = clips(2, args.frames, args.side, layer.c, 12345)
    whole = layer.forward(x.reshape(-1), 2, t, pos.repeat(2, 1)).view(2, t, layer.c)
    cache, worst = Cache(layer, 2, t), 0.0
    for i in range(t):
        one = layer.extend(x[:, i].reshape(-1).contiguous(), 2, 1, pos[i:i + 1].repeat(2, 1), cache)
        worst = max(worst, float((one.view(2, layer.c) - whole[:, i]).abs().max()))
    print(f"{t} tokens one at a time: largest difference {worst:.2e} from the whole clip")
    ops.default_context().synchronize()


if __name__ == "__main__":
    main()

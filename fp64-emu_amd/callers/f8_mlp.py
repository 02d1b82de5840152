"""A gated MLP, y = (silu(x Wg^T) * (x Wu^T)) Wd^T, trained and served by the 8-bit
operators together (fp64_emu.quant_f8, quant_f8_tiles, mm_f8, swiglu_f8,
swiglu_f8_backward): every product on e4m3 operands with a scale per block
of 128, every tensor that waits for the backward pass in 8 bits, weights and
their gradients in float32.

One training step:

  forward    x -> (rows, columns);  h = x W1^T (rows x tiles), bfloat16
             h -> y's rows and columns, and h's checkpoint, one pass
             out = y W2^T
  backward   dout -> (rows, columns);  dy = dout W2 (rows x tiles transposed)
             dW2 += dout^T y (columns x columns, into float32)
             dy and h's checkpoint -> dh's rows and columns, one pass
             dx = dh W1;  dW1 += dh^T x

Serving a token: x's rows, h, y's rows, out; nothing kept.

    python fp64-emu_amd/callers/f8_mlp.py [d=4096] [f=4096] [tokens=8192]
"""
import argparse
import os
import statistics
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import fp64_emu as emu  # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32


class GatedMlp:
    """Weights w1 [2 f, d] (gate rows, then up rows) and w2 [d, f] in float32, their 8-bit
    forms laid out by `quantise` once per update."""

    def __init__(self, d, f, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.w1 = (torch.randn(2 * f, d, generator=g) * d ** -0.5).to(device)
        self.w2 = (torch.randn(d, f, generator=g) * f ** -0.5).to(device)
        self.g1, self.g2 = torch.zeros_like(self.w1), torch.zeros_like(self.w2)
        self.quantise()

    def quantise(self):
        self.q1 = emu.quant_f8_tiles(self.w1, transposed=True)
        self.q2 = emu.quant_f8_tiles(self.w2, transposed=True)

    def forward(self, x):
        """(out, what backward takes): x [tokens, d] in bfloat16."""
        q, s, *x_cols = emu.quant_f8(x, cols=True)
        h = emu.mm_f8(q, s, *self.q1[:2])
        yq, ys, yqt, yst, hq, hs = emu.swiglu_f8(h, quant="both")
        return emu.mm_f8(yq, ys, *self.q2[:2]), (x_cols, (yqt, yst), (hq, hs))

    def backward(self, dout, kept):
        """dx; the weights' gradients are added to g1 and g2."""
        x_cols, y_cols, h_kept = kept
        q, s, qt, st = emu.quant_f8(dout, cols=True)
        dy = emu.mm_f8(q, s, *self.q2[2:])
        emu.mm_f8(qt, st, *y_cols, out=self.g2, accumulate=True)
        q, s, qt, st = emu.swiglu_f8_backward(dy, *h_kept, quant="both")
        emu.mm_f8(qt, st, *x_cols, out=self.g1, accumulate=True)
        return emu.mm_f8(q, s, *self.q1[2:])

    def serve(self, x):
        """out for tokens that nothing is kept of."""
        h = emu.mm_f8(*emu.quant_f8(x), *self.q1[:2])
        return emu.mm_f8(*emu.swiglu_f8(h, quant="rows", keep=False), *self.q2[:2])

    def sgd(self, rate):
        self.w1.sub_(self.g1, alpha=rate)
        self.w2.sub_(self.g2, alpha=rate)
        self.g1.zero_()
        self.g2.zero_()
        self.quantise()


class PlainMlp:
    """The same from float32 torch operations and autograd."""

    def __init__(self, like):
        self.w1, self.w2 = (w.clone().requires_grad_() for w in (like.w1, like.w2))

    def forward(self, x):
        gate, up = (x.float() @ self.w1.t()).chunk(2, dim=-1)
        return (torch.nn.functional.silu(gate) * up) @ self.w2.t()


def train(d=256, f=384, tokens=1024, steps=60, rate=0.5, seed=0, device="cuda"):
    """Both fit a teacher of the same form from the same start and the same batches.
    Returns the losses: {"start", "f8", "plain"}."""
    teacher, f8 = GatedMlp(d, f, seed + 1, device), GatedMlp(d, f, seed, device)
    plain = PlainMlp(f8)
    losses = {}
    g = torch.Generator().manual_seed(seed + 2)
    for step in range(steps):
        x = torch.randn(tokens, d, generator=g).to(device, BF16)
        with torch.no_grad():
            target = PlainMlp(teacher).forward(x)
        out, kept = f8.forward(x)
        diff = out.float() - target
        losses["f8"] = diff.square().mean().item()
        losses.setdefault("start", losses["f8"])
        f8.backward((2 * diff / tokens).to(BF16), kept)
        f8.sgd(rate)
        loss = (plain.forward(x) - target).square().sum() / tokens
        g1, g2 = torch.autograd.grad(loss, (plain.w1, plain.w2))
        losses["plain"] = loss.item() / d
        with torch.no_grad():
            plain.w1 -= rate * g1
            plain.w2 -= rate * g2
    return losses


def _time(fn, reps=20):
    for _ in range(3):
        fn()
    out = []
    for _ in range(3):
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        for _ in range(reps):
            fn()
        torch.cuda.synchronize()
        out.append((time.perf_counter() - t0) / reps)
    return statistics.median(out)


def run(d, f, tokens, device="cuda"):
    net = GatedMlp(d, f, device=device)
    x = torch.randn(tokens, d, device=device).to(BF16)
    dout = (torch.randn(tokens, d, device=device) * 1e-3).to(BF16)

    def step():
        _, kept = net.forward(x)
        net.backward(dout, kept)

    _, kept = net.forward(x)
    held = sum(t.numel() * t.element_size() for pair in kept for t in pair)
    train_s, token_s = _time(step), _time(lambda: net.serve(x[:1]))
    return {"step_ms": train_s * 1e3, "step_tflops": 18 * tokens * d * f / train_s / 1e12,
            "token_us": token_s * 1e6, "held_mb": held / 1e6,
            "held_bf16_mb": 2 * tokens * (d + 3 * f) / 1e6}


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("d", nargs="?", type=int, default=4096)
    ap.add_argument("f", nargs="?", type=int, default=4096)
    ap.add_argument("tokens", nargs="?", type=int, default=8192)
    a = ap.parse_args()
    r = run(a.d, a.f, a.tokens)
    print(f"{torch.cuda.get_device_name(0)} | d={a.d} f={a.f} tokens={a.tokens}", flush=True)
    print(f"forward and backward {r['step_ms']:.3f} ms, {r['step_tflops']:.0f} TFLOP/s | held for the backward pass "
          f"{r['held_mb']:.1f} MB ({r['held_bf16_mb']:.1f} MB in bfloat16) | one token {r['token_us']:.1f} us",
          flush=True)
    print("losses after 60 steps:", {k: round(v, 5) for k, v in train().items()}, flush=True)


if __name__ == "__main__":
    main()

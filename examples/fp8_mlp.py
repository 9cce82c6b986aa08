"""A language model's MLP block on FP8 weights kept tANS-coded on disk:

    h = x + residual
    out = h + down(silu(gate(norm(h))) * up(norm(h)))

    python examples/fp8_mlp.py [--hidden 5120] [--inner 17408] [--tokens 1 97 2048]

The weights (random, one scale per row) are encoded on the GPU and written to a
container; load() decodes them to FP8 bytes in device memory, once.  forward()
is four calls, all on 8-bit rows with one scale each: fp8_rmsnorm (the
residual's addition, the norm, 8 bits), fp8_linear with the gate in its
epilogue, fp8_quantize_rows, fp8_linear with the residual in its epilogue.
"""
from __future__ import annotations

import argparse
import os
import sys
import tempfile
import time

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tans-vectoradd_amd"))

import rans_vectoradd as R  # noqa: E402
from rans_vectoradd import container, tans_codec  # noqa: E402


def random_fp8_rows(rows: int, cols: int, seed: int, device="cuda"):
    """E4M3FN bytes [rows, cols] of N(0, 0.02) and a float32 scale per row."""
    g = torch.Generator(device=device).manual_seed(seed)
    w = torch.randn(rows, cols, generator=g, device=device).mul_(0.02)
    return R.fp8_quantize_rows(w.to(torch.bfloat16))


def encode_rows(w: torch.Tensor) -> tans_codec.TansTensor:
    """A weight matrix as lanes of one row each, with a table of its own
    exponents (every exponent counted once more, so that none is without a code)."""
    hist = torch.bincount(((w.view(-1) >> 3) & 15).to(torch.int32), minlength=16).double() + 1
    return tans_codec.TansTensor.from_tuple(tans_codec.encode_gpu(w, hist.cpu()), *w.shape)


def decode_rows(t: tans_codec.TansTensor) -> torch.Tensor:
    """The bytes [rows, cols] again."""
    cols_rows = R.gpu_tans_decode(t.comp, t.offsets, t.states, t.partial, t.sm, t.spread, t.freqs,
                                  t.N)
    return cols_rows.t().contiguous()


class Fp8Mlp:
    """The block's weights on a GPU: gate and up [2 inner, hidden] in one
    matrix, down [hidden, inner], their row scales and the norm's weight."""

    def __init__(self, norm, gate_up, gate_up_scale, down, down_scale, eps: float = 1e-6):
        self.norm, self.eps = norm, eps
        self.gate_up, self.gate_up_scale = gate_up, gate_up_scale
        self.down, self.down_scale = down, down_scale

    def save(self, path: str) -> None:
        container.save(path, {"gate_up": encode_rows(self.gate_up), "down": encode_rows(self.down),
                              "gate_up_scale": self.gate_up_scale, "down_scale": self.down_scale,
                              "norm": self.norm})

    @classmethod
    def load(cls, path: str, device="cuda") -> "Fp8Mlp":
        e = container.load(path, device=device)
        return cls(e["norm"], decode_rows(e["gate_up"]), e["gate_up_scale"],
                   decode_rows(e["down"]), e["down_scale"])

    def forward(self, x: torch.Tensor, residual: torch.Tensor) -> torch.Tensor:
        """x, residual bf16 [hidden] or [tokens, hidden] -> the block's output,
        the residual of what follows."""
        q, scale, h = R.fp8_rmsnorm(x, self.norm, residual, eps=self.eps)
        inner = R.fp8_linear(q, scale, self.gate_up, self.gate_up_scale, activation="silu",
                             gated=True)
        q, scale = R.fp8_quantize_rows(inner)
        return R.fp8_linear(q, scale, self.down, self.down_scale, residual=h)


def reference(m: Fp8Mlp, x: torch.Tensor, residual: torch.Tensor) -> torch.Tensor:
    """The block in 64 bits on the same weights, nothing rounded between."""
    def weights(b, s):
        return b.view(torch.float8_e4m3fn).to(torch.float32).double() * s.double()[:, None]
    h = x.double() + residual.double()
    y = h * torch.rsqrt(h.square().mean(dim=-1, keepdim=True) + m.eps) * m.norm.double()
    gate, up = (y @ weights(m.gate_up, m.gate_up_scale).t().contiguous()).chunk(2, dim=-1)
    inner = torch.nn.functional.silu(gate) * up
    return h + inner @ weights(m.down, m.down_scale).t().contiguous()


def random_block(hidden: int, inner: int, seed: int = 0) -> Fp8Mlp:
    g = torch.Generator(device="cuda").manual_seed(seed)
    norm = (torch.randn(hidden, generator=g, device="cuda") * 0.1 + 1).to(torch.bfloat16)
    return Fp8Mlp(norm, *random_fp8_rows(2 * inner, hidden, seed + 1),
                  *random_fp8_rows(hidden, inner, seed + 2))


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--hidden", type=int, default=5120)
    p.add_argument("--inner", type=int, default=17408)
    p.add_argument("--tokens", type=int, nargs="+", default=[1, 97, 2048])
    a = p.parse_args()
    block = random_block(a.hidden, a.inner)
    raw = block.gate_up.numel() + block.down.numel()
    with tempfile.TemporaryDirectory() as d:
        path = os.path.join(d, "mlp.tans.safetensors")
        block.save(path)
        loaded = Fp8Mlp.load(path)
        print(f"{raw / 1e6:.1f} MB of FP8 weights, {os.path.getsize(path) / 1e6:.1f} MB in the "
              f"container", flush=True)
    assert torch.equal(loaded.gate_up, block.gate_up) and torch.equal(loaded.down, block.down)
    for n in a.tokens:
        g = torch.Generator(device="cuda").manual_seed(n)
        x, res = (torch.randn(n, a.hidden, generator=g, device="cuda").to(torch.bfloat16)
                  for _ in range(2))
        for _ in range(3):
            out = loaded.forward(x, res)
        torch.cuda.synchronize()
        began, k = time.perf_counter(), 20
        for _ in range(k):
            out = loaded.forward(x, res)
        torch.cuda.synchronize()
        us = (time.perf_counter() - began) / k * 1e6
        want = reference(loaded, x, res)
        off = ((out.double() - want).norm() / want.norm()).item()
        print(f"{n} tokens: {us:.1f} us, {6 * a.hidden * a.inner * n / us / 1e6:.1f} TFLOP/s, "
              f"{off:.2e} from 64 bits", flush=True)


if __name__ == "__main__":
    main()

"""One bidirectional encoder layer whose weights are held in 8 bits, on the layer operators of ``ops``:

    x -> RMS norm -> q | k | v (8-bit product) -> per-head norm -> rotary positions -> attention
      -> output projection (8-bit) -> + x -> RMS norm -> gate | up (8-bit) -> GELU -> down (8-bit) -> + x

Several documents are packed into one buffer and kept apart by a document mask; scores are capped and a sliding
window may bound them; positions may be stretched past the length the layer was made for. Compares with the same
layer in 32 bits and prints the time of a pass.

    python examples/encoder_layer_int8.py [--tokens 35328] [--document 2208] [--window 512]
"""
import argparse
import importlib
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
ops = importlib.import_module("embeddinggemma2-rust_b200.ops")

EPS = 1e-6


def rms(x, eps=EPS):
    y = x.float()
    return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)).to(x.dtype)


class Linear8:
    """A weight as whole numbers of -127 .. 127 with a scale per output channel; rows of the input are quantised as they come."""

    def __init__(self, weight):
        self.w, self.scale = ops.quantize_rows(weight)

    def __call__(self, x):
        q, s = ops.quantize_rows(x)
        return ops.gemm_i8(q, s, self.w, self.scale)


class EncoderLayer8:
    """Heads and widths of the text tower's sliding layers by default."""

    def __init__(self, seed=0, hidden=512, ff=2048, nh=4, nkv=2, hd=256, window=512, softcap=50.0, theta=10000.0,
                 scaling="none", factor=1.0, original_len=0, device="cuda"):
        g = torch.Generator(device).manual_seed(seed)
        self.nh, self.nkv, self.hd, self.ff, self.window, self.softcap = nh, nkv, hd, ff, window, softcap
        mk = lambda n, k: torch.randn(n, k, device=device, generator=g) * k ** -0.5
        self.plain = {"qkv": mk((nh + 2 * nkv) * hd, hidden), "o": mk(hidden, nh * hd), "gu": mk(2 * ff, hidden), "down": mk(hidden, ff)}
        self.w = {k: Linear8(v) for k, v in self.plain.items()}
        steps, self.magnitude = ops.rotary_steps(hd, theta, scaling, factor, original_len)
        self.steps = torch.from_numpy(steps.view(np.int64)).to(device)

    def __call__(self, x, pos, doc, offsets, longest):
        """``x [rows, hidden]`` bf16, ``pos`` / ``doc`` int32 per row, ``offsets`` of the packed buffers (int32)."""
        nh, nkv, hd = self.nh, self.nkv, self.hd
        qkv = self.w["qkv"](rms(x))
        q, k, v = (t.unflatten(1, (-1, hd)) for t in qkv.split([nh * hd, nkv * hd, nkv * hd], 1))
        q, k = ops.rotary(rms(q), rms(k), pos, self.steps, magnitude=self.magnitude)
        a = ops.attention_masked(q, k, v, offsets, offsets, longest, longest, scale=hd ** -0.5 * 4, softcap=self.softcap,
                                 window=self.window, q_doc=doc, k_doc=doc)
        x = x + self.w["o"](a.flatten(1))
        gate, up = self.w["gu"](rms(x)).chunk(2, 1)
        return x + self.w["down"](torch.nn.functional.gelu(gate.float(), approximate="tanh").to(x.dtype) * up)

    def in_32_bits(self, x, pos, doc):
        """The same layer by plain operations on the unquantised weights, one buffer."""
        nh, nkv, hd = self.nh, self.nkv, self.hd
        x = x.float()
        qkv = rms(x) @ self.plain["qkv"].T
        q, k, v = (t.unflatten(1, (-1, hd)) for t in qkv.split([nh * hd, nkv * hd, nkv * hd], 1))
        turns = (pos.long()[:, None] * self.steps >> 32).float() * 2.0**-32
        c, s = (m * self.magnitude for m in (torch.cos(2 * torch.pi * turns)[:, None], torch.sin(2 * torch.pi * turns)[:, None]))

        def turn(t):
            u, w = rms(t).chunk(2, -1)
            return torch.cat([u * c - w * s, w * c + u * s], -1)

        q, k = turn(q), turn(k)
        k, v = (t.repeat_interleave(nh // nkv, 1) for t in (k, v))
        i = torch.arange(len(x), device=x.device)
        seen = (doc[:, None] == doc[None]) & ((i[:, None] - i[None]).abs() <= self.window)
        z = torch.einsum("ihd,jhd->hij", q, k) * (hd ** -0.5 * 4)
        z = (self.softcap * torch.tanh(z / self.softcap)).masked_fill(~seen, -torch.inf)
        a = torch.einsum("hij,jhd->ihd", z.softmax(-1), v)
        x = x + a.flatten(1) @ self.plain["o"].T
        gate, up = (rms(x) @ self.plain["gu"].T).chunk(2, 1)
        return x + (torch.nn.functional.gelu(gate, approximate="tanh") * up) @ self.plain["down"].T


def packed(tokens, document, device="cuda"):
    """Positions, document numbers and offsets of `tokens` rows of documents of up to `document` tokens."""
    lens, left = [], tokens
    while left:
        lens.append(min(left, max(1, int(document * (1.0 - (len(lens) * 0.618) % 1.0)))))
        left -= lens[-1]
    lens = torch.tensor(lens)
    doc = torch.repeat_interleave(torch.arange(len(lens)), lens)
    start = (torch.cumsum(lens, 0) - lens)[doc]
    pos = torch.arange(tokens) - start
    to = lambda t: t.to(torch.int32).to(device)
    return to(pos), to(doc), to(torch.tensor([0, tokens]))


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--tokens", type=int, default=35328)
    ap.add_argument("--document", type=int, default=2208)
    ap.add_argument("--window", type=int, default=512)
    a = ap.parse_args()
    layer = EncoderLayer8(window=a.window)
    small = min(a.tokens, 2048)
    x = torch.randn(a.tokens, 512, device="cuda").bfloat16()
    pos, doc, off = packed(small, a.document)
    got, want = layer(x[:small], pos, doc, off, small).float(), layer.in_32_bits(x[:small], pos, doc)
    cos = torch.nn.functional.cosine_similarity(got, want, 1)
    print(f"{small} tokens against 32 bits: relative error {float((got - want).norm() / want.norm()):.4f}, "
          f"cosine of the rows at least {float(cos.min()):.5f}")
    pos, doc, off = packed(a.tokens, a.document)
    for _ in range(3):
        layer(x, pos, doc, off, a.tokens)
    t0, t1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    t0.record()
    for _ in range(10):
        layer(x, pos, doc, off, a.tokens)
    t1.record()
    torch.cuda.synchronize()
    ms = t0.elapsed_time(t1) / 10
    print(f"{a.tokens} tokens: {ms:.3f} ms a layer, {a.tokens / ms * 1e3:.3g} tokens/s")


if __name__ == "__main__":
    main()

"""Generates tokens with a small random mixture-of-experts language model, whose step is the
engine's operators one after the other: the norm with the residual's addition and an 8-bit
output, the experts' products over ragged groups, the norm again, the head's 8-bit
product, and the choice of a token.

    python examples/lm_step.py [--batch 16] [--steps 32] [--layers 4]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import pdefa_b200 as pb  # noqa: E402

BLOCK, E4M3_MAX = 128, 448.0


def quantize_weight(w):
    """w [..., N, K] -> e4m3 values and one float32 scale per 128 x 128 block."""
    *lead, n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    pad = torch.nn.functional.pad(w.float(), (0, kb * BLOCK - k, 0, nb * BLOCK - n))
    blocks = pad.view(*lead, nb, BLOCK, kb, BLOCK)
    scales = blocks.abs().amax((-3, -1)).clamp(min=1e-10) / E4M3_MAX
    q = (blocks / scales[..., :, None, :, None]).view(*lead, nb * BLOCK, kb * BLOCK)[..., :n, :k]
    return q.to(torch.float8_e4m3fn).contiguous(), scales


class Model:
    """An embedding, layers of (norm, router, one expert product per token), a norm and a head."""

    def __init__(self, hidden=1024, experts=8, layers=4, vocab=32000, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        randn = lambda *s: torch.randn(s, generator=g, device="cuda")   # noqa: E731
        self.embedding = randn(vocab, hidden).to(torch.bfloat16)
        self.layers = []
        for _ in range(layers):
            w, s = quantize_weight(randn(experts, hidden, hidden) / hidden ** 0.5)
            self.layers.append({"norm": 1 + 0.1 * randn(hidden), "router": randn(hidden, experts) / hidden ** 0.5,
                                "w": w, "s": s})
        self.norm = 1 + 0.1 * randn(hidden)
        self.head, self.head_scales = quantize_weight(randn(vocab, hidden) / hidden ** 0.5)

    def logits(self, tokens):
        """Float32 logits [batch, vocab] for one token per sequence."""
        h = torch.zeros(len(tokens), self.embedding.shape[1], dtype=torch.bfloat16, device="cuda")
        x = self.embedding[tokens]
        for layer in self.layers:
            q, s, h = pb.ops_rms_norm_fp8(x, layer["norm"], residual=h)
            values = q.float() * s.repeat_interleave(BLOCK, -1)[:, :q.shape[1]]
            expert = (values @ layer["router"]).argmax(-1)
            # rows sorted by expert; the experts' ranges stay on the GPU
            order = torch.argsort(expert, stable=True)
            counts = torch.bincount(expert, minlength=layer["w"].shape[0])
            offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
            rows = q.view(torch.uint8)[order].view(torch.float8_e4m3fn)
            out = pb.ops_matmul_grouped_fp8(rows, s[order], layer["w"], layer["s"], offsets)
            x = torch.empty_like(out)
            x[order] = out
        q, s, h = pb.ops_rms_norm_fp8(x, self.norm, residual=h)
        return pb.ops_matmul_fp8(q, s, self.head, self.head_scales, out_dtype=torch.float32)


def generate(model, tokens, steps, seed=0, temperature=0.8, top_k=50, top_p=0.95):
    """[batch, steps] sampled tokens and their probabilities, from one start token each."""
    n = len(tokens)
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.full((n,), temperature, device="cuda")
    k = torch.full((n,), top_k, dtype=torch.int32, device="cuda")
    p = torch.full((n,), top_p, device="cuda")
    chosen, probs = [], []
    for _ in range(steps):
        logits = model.logits(tokens)
        noise = torch.empty_like(logits).exponential_(generator=g)
        tokens, prob = pb.ops_sample(logits, noise, temperature=t, top_k=k, top_p=p)
        chosen.append(tokens)
        probs.append(prob)
    return torch.stack(chosen, 1), torch.stack(probs, 1)


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--layers", type=int, default=4)
    a = ap.parse_args()
    model = Model(layers=a.layers)
    start = torch.arange(a.batch, device="cuda")
    generate(model, start, 2)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    tokens, probs = generate(model, start, a.steps)
    end.record()
    torch.cuda.synchronize()
    print(f"{a.steps} steps of {a.batch} sequences: {begin.elapsed_time(end) / a.steps * 1e3:.0f} us a step")
    print("first sequence:", tokens[0].tolist()[:12], "probabilities", [round(v, 3) for v in probs[0].tolist()[:6]])


if __name__ == "__main__":
    main()

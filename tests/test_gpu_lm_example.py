"""The language-model operators together, as examples/lm_step.py runs them, against the
same step in 64-bit torch operations on the same quantised weights."""
import os
import sys

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def _quantized_norm(x, w, h):
    """The norm's 8-bit output as the values it stands for, and the rounded residual stream."""
    h = x.float() + h.float()
    y = (h.double() / (h.double().square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()).float()
    b = y.view(y.shape[0], -1, 128)
    s = b.abs().amax(-1, keepdim=True).clamp(min=1e-10) / 448
    return ((b / s).to(torch.float8_e4m3fn).double() * s.double()).view_as(y), h.to(torch.bfloat16)


def _weights(q, s):
    return q.double() * s.double().repeat_interleave(128, -2)[..., :q.shape[-2], :].repeat_interleave(128, -1)[..., :q.shape[-1]]


@pytest.mark.parametrize("batch", [1, 24, 200])
def test_step_matches_plain_operations(batch):
    import lm_step
    model = lm_step.Model(hidden=512, experts=6, layers=2, vocab=3001, seed=3)
    tokens = torch.arange(batch, device="cuda") * 7 % 3001
    got = model.logits(tokens)

    h = torch.zeros(batch, 512, dtype=torch.bfloat16, device="cuda")
    x = model.embedding[tokens]
    for layer in model.layers:
        v, h = _quantized_norm(x, layer["norm"], h)
        expert = (v.float() @ layer["router"]).argmax(-1)
        w = _weights(layer["w"], layer["s"])
        x = torch.einsum("tk,tnk->tn", v, w[expert]).to(torch.bfloat16)
    v, h = _quantized_norm(x, model.norm, h)
    want = v @ _weights(model.head, model.head_scales).t()
    # A value on the boundary between two 8-bit or bfloat16 neighbours may round the other way
    # (one part in 16 or 256 of that value); a row in which a router's top two are that close
    # may take another expert. Rows are compared as a whole.
    far = (got.double() - want).norm(dim=1) / want.norm(dim=1)
    assert (far < 2e-2).float().mean() >= 0.95 and far.median() < 2e-3, far.sort().values[-5:]


def test_generation_is_repeatable_and_valid():
    import lm_step
    model = lm_step.Model(hidden=256, experts=4, layers=2, vocab=1000, seed=4)
    start = torch.arange(9, device="cuda")
    a, pa = lm_step.generate(model, start, 6, seed=1)
    b, pb_ = lm_step.generate(model, start, 6, seed=1)
    c, _ = lm_step.generate(model, start, 6, seed=2)
    assert a.shape == (9, 6) and torch.equal(a, b) and torch.equal(pa, pb_) and not torch.equal(a, c)
    assert ((a >= 0) & (a < 1000)).all() and ((pa > 0) & (pa <= 1)).all()

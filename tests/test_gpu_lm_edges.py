"""The language-model operators where their contracts are exact: what has to be equal to the
last bit, and special values in settings and variates."""
import numpy as np
import pytest

import pdefa_b200 as pb
from test_gpu_lm import SETTINGS, check_sample, logits_of, noise_of

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ids = lambda v: str(v).replace("torch.", "")   # noqa: E731


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def quantised(y):
    """scale = max(largest |y| of 128, 1e-10) / 448 and e4m3(y / scale), both divisions rounded
    to 32 bits, from the 32-bit y (on the CPU, where a division is one)."""
    y = y.cpu().numpy()
    rows, cols = y.shape
    nb = -(-cols // 128)
    pad = np.zeros((rows, nb * 128), np.float32)
    pad[:, :cols] = y
    pad = pad.reshape(rows, nb, 128)
    scale = np.maximum(np.abs(pad).max(-1), np.float32(1e-10)) / np.float32(448)
    q = (pad / scale[..., None]).reshape(rows, -1)[:, :cols]
    return torch.from_numpy(q.copy()).clamp(-448, 448).to(torch.float8_e4m3fn), torch.from_numpy(scale)


def on_boundaries(g, rows, cols, dtype):
    """Rows of +-1 and weights that make y / scale a whole number (of 1.25 for some blocks): half
    of the odd ones above 16 lie between two 8-bit values."""
    x = torch.where(torch.rand((rows, cols), generator=g, device="cuda") < 0.5, -1.0, 1.0).to(dtype)
    w = torch.randint(1, 240, (cols,), generator=g, device="cuda").float()
    w[::128] = 448.0 if dtype != torch.bfloat16 else 224.0
    return x, w


# whole pieces; rows of every offset with one to four pieces a thread; rows too long for the registers
@pytest.mark.parametrize("rows,cols", [(5, 512), (3000, 4096), (5, 1033), (1100, 1153), (1300, 2051), (1300, 1537), (5, 8191),
                                       (3, 13001), (2, 20001)])
def test_norm_8bit_values_are_quotients_by_their_scale(rows, cols):
    g = gen(rows + cols)
    x, w = on_boundaries(g, rows, cols, torch.float32)
    x *= 1 + torch.rand((rows, 1), generator=g, device="cuda")
    y = pb.ops_rms_norm(x, w, eps=1e-3)
    q, scales = pb.ops_rms_norm_fp8(x, w, eps=1e-3)
    want_q, want_s = quantised(y)
    assert torch.equal(scales.cpu(), want_s)
    assert torch.equal(q.cpu().float(), want_q.float())


@pytest.mark.parametrize("cols", [513, 4100])
def test_norm_8bit_quotients_of_unlike_rows(cols):
    """A residual whose rows start elsewhere than x's."""
    rows = 7
    g = gen(cols)
    x, w = on_boundaries(g, rows, cols, torch.float32)
    res = torch.zeros(rows, cols + 2, device="cuda")[:, :cols]
    res[:] = x * 0.5
    y, _ = pb.ops_rms_norm(x, w, residual=res, eps=1e-3)
    q, scales, _ = pb.ops_rms_norm_fp8(x, w, residual=res, eps=1e-3)
    want_q, want_s = quantised(y)
    assert torch.equal(scales.cpu(), want_s)
    assert torch.equal(q.cpu().float(), want_q.float())


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("rows", [3, 2000])
def test_norm_8bit_quotients_of_known_values(dtype, rows):
    """4096 values of +-1 without eps: the root is 1 and y the weight, exactly."""
    x, w = on_boundaries(gen(rows), rows, 4096, dtype)
    q, scales = pb.ops_rms_norm_fp8(x, w.to(dtype), eps=0.0)
    want_q, want_s = quantised(x.float() * w)
    assert torch.equal(scales.cpu(), want_s)
    assert torch.equal(q.cpu().float(), want_q.float())


@pytest.mark.parametrize("rows,cols", [(5, 512), (5, 1033), (3, 13001), (2, 20001)])
def test_norm_8bit_of_infinite_products(rows, cols):
    """A weight that makes one y infinite: its group's scale is, it is NaN and the group's others are 0."""
    x, w = on_boundaries(gen(cols), rows, cols, torch.float32)
    w[130] = float("inf")
    w[300] = 3e38
    y = pb.ops_rms_norm(x, w, eps=0.0)
    q, scales = pb.ops_rms_norm_fp8(x, w, eps=0.0)
    with np.errstate(invalid="ignore"):
        want_q, want_s = quantised(y)
    assert torch.equal(scales.cpu(), want_s) and scales[:, 1].isinf().all() and scales[:, 2].isfinite().all()
    got, want = q.cpu().float(), want_q.float()
    assert torch.equal(got.isnan(), want.isnan()) and got[:, 130].isnan().all()
    assert torch.equal(got.nan_to_num(), want.nan_to_num())


# rows that a cluster holds, and longer ones
@pytest.mark.parametrize("vocab", [3001, 409701])
@pytest.mark.parametrize("t", [1.5e-45, 1e-39, 4.2e-39, 1.1e-38, 1.2e-38, 3e38])
def test_sample_extreme_temperatures(vocab, t):
    """Temperatures whose inverse no 32-bit number holds: the largest logits share the mass, or all do."""
    g = gen(vocab)
    rows = len(SETTINGS)
    x, e = logits_of(g, rows, vocab, torch.float32), noise_of(g, rows, vocab)
    x[1::2] = torch.round(x[1::2])                # several largest
    x[2::4, ::2] = -float("inf")
    tok, prob = check_sample(x, e, t=[t] * rows, k=[s.get("k", 0) for s in SETTINGS], p=[s.get("p", 1.0) for s in SETTINGS],
                             m=[s.get("m", 0.0) for s in SETTINGS])
    assert prob.isfinite().all() and (prob > 0).all()
    if t < 1:
        assert torch.equal(x.gather(1, tok[:, None].long())[:, 0], x.amax(1))


@pytest.mark.parametrize("vocab", [3001, 409701])
def test_sample_infinite_temperature(vocab):
    g = gen(vocab)
    x, e = logits_of(g, 3, vocab, torch.float32), noise_of(g, 3, vocab)
    x[1, ::3] = -float("inf")                     # ruled out at any temperature
    x[2, [70, 1000, 2900]] = float("inf")         # these alone share the mass
    tok, prob = pb.ops_sample(x, e, temperature=torch.full((3,), float("inf"), device="cuda"))
    left = torch.stack([torch.ones(vocab, dtype=torch.bool, device="cuda"), x[1] > -float("inf"), x[2] == float("inf")])
    assert torch.equal(tok.long(), torch.where(left, e, torch.inf).argmin(1))
    assert torch.allclose(prob, 1 / left.sum(1).float(), rtol=1e-5)


@pytest.mark.parametrize("vocab", [3001, 409701])
def test_sample_negative_zero_noise(vocab):
    """w / -0 is -inf: the token loses, in every kind of row; against +0 too."""
    g = gen(vocab)
    n = len(SETTINGS)
    x, e = logits_of(g, 4 * n, vocab, torch.float32), noise_of(g, 4 * n, vocab)
    at = torch.arange(n, device="cuda")
    e[at, x[:n].argmax(1)] = -0.0
    e[n:2 * n, 100::2] = -0.0
    e[2 * n:3 * n] = -0.0                         # no usable variate: the first token
    top = x[3 * n:].topk(2, dim=1).indices
    e[3 * n + at, top[:, 0]] = -0.0
    e[3 * n + at, top[:, 1]] = 0.0
    every = 4 * SETTINGS
    tok, _ = check_sample(x, e, t=[s.get("t", 1.0) for s in every], k=[s.get("k", 0) for s in every],
                          p=[s.get("p", 1.0) for s in every], m=[s.get("m", 0.0) for s in every])
    assert torch.equal(tok[2 * n:3 * n].long(), x[2 * n:3 * n].argmax(1))
    assert tok[3 * n] == top[0, 1]                # no filter: the one with +0

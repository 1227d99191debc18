"""The language-model operators where their contracts are exact: what has to be equal to the
last bit, and special values in settings and variates."""
import numpy as np
import pytest

import pdefa_b200 as pb

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

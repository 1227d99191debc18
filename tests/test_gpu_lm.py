"""The language-model operators (norm with residual and 8-bit output, 8-bit products,
sampling) against their definitions in 64 bits, on inputs of every type, odd sizes,
spaced rows and the values where they can go wrong.

Error bounds, with u the unit roundoff of 32 bits (2^-24) and v that of the output type:
  * norm: a thread adds at most cols / 128 squares in turn and the threads are joined
    in a tree, the root, two products and the quotient add a few: (cols / 128 + 32) u,
    plus v for the rounding of the output;
  * 8-bit values: half a step, 2^-4 of the value or 2^-10 for the smallest, on top of
    the norm's bound;
  * products: (128 + blocks + 4) u times the sum of absolute products (any order of
    32-bit addition inside a block of 128, then the blocks one after the other), plus v.
"""
import math

import numpy as np
import pytest

import pdefa_b200 as pb

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
V = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ids = lambda v: str(v).replace("torch.", "")   # noqa: E731


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def spaced(t, gap):
    """t with `gap` unused elements after each row (NaN, so that a stray read shows)."""
    if not gap:
        return t
    wide = torch.full((*t.shape[:-1], t.shape[-1] + gap), float("nan"), device=t.device)
    wide = wide.to(t.dtype)
    wide[..., :t.shape[-1]] = t
    return wide[..., :t.shape[-1]]


# ----------------------------------------------------------------------------
# norm
# ----------------------------------------------------------------------------
def norm_ref(x, w, res, eps):
    h = x.double() if res is None else x.double() + res.double()
    return h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w.double(), h


NORM_SIZES = [(1, 1), (1, 2), (3, 7), (2, 128), (5, 129), (4, 255), (33, 256), (1, 1000), (7, 1024), (2, 2050),
              (3, 4096), (2, 5120), (1, 8192), (2, 8200), (1, 16384), (1, 20000), (1, 33001), (1, 70000), (300, 64)]


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("rows,cols", NORM_SIZES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("gap", [0, 3, 8])
def test_norm(rows, cols, dtype, residual, gap):
    g = gen(rows * 100003 + cols)
    x = spaced((randn(g, rows, cols) * 3).to(dtype), gap)
    res = spaced(randn(g, rows, cols).to(dtype), gap) if residual else None
    w = (1 + 0.3 * randn(g, cols)).to(torch.float32 if cols % 2 else dtype)
    y64, h64 = norm_ref(x, w, res, 1e-5)
    got = pb.ops_rms_norm(x, w, residual=res, eps=1e-5)
    y, h = got if residual else (got, None)
    assert y.dtype == dtype and y.shape == x.shape
    tol = (cols / 128 + 32) * U
    err = (y.double() - y64).abs()
    assert (err <= (tol + V[dtype]) * y64.abs() * 1.0001 + LEAST[dtype]).all(), float(err.max())
    if residual:
        assert torch.equal(h, (x.float() + res.float()).to(dtype))

    got = pb.ops_rms_norm_fp8(x, w, residual=res, eps=1e-5)
    q, scales = got[:2]
    nb = -(-cols // 128)
    assert q.dtype == torch.float8_e4m3fn and scales.shape == (rows, nb)
    pad = torch.nn.functional.pad(y64, (0, nb * 128 - cols)).view(rows, nb, 128)
    s64 = pad.abs().amax(-1).clamp(min=1e-10) / 448
    assert ((scales.double() - s64).abs() <= (tol + 4 * U) * s64).all()
    unit = torch.nn.functional.pad(y64, (0, nb * 128 - cols)).view(rows, nb, 128) / s64[..., None]
    unit = unit.view(rows, -1)[:, :cols]
    far = (q.double() - unit).abs()
    assert (far <= torch.maximum(unit.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10, device="cuda")) * 1.001 + 448 * (tol + 8 * U)).all()
    if residual:
        assert torch.equal(got[2], h)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("rows,cols", [(9, 17), (40, 131), (13, 1031), (1100, 1153), (700, 3001), (1100, 2051), (1300, 1537), (9, 8191), (11, 13001),
                                       (7, 16383), (3, 32761)])
def test_norm_rows_of_every_offset(rows, cols, dtype):
    """Contiguous rows of odd lengths start at every offset within 16 bytes; what lies beside a row stays out of it."""
    g = gen(rows + cols)
    x, res = (randn(g, rows, cols) * 3).to(dtype), randn(g, rows, cols).to(dtype)
    x[1::3] = float("nan")
    w = (1 + 0.3 * randn(g, cols)).to(dtype)
    fine = [i for i in range(rows) if i % 3 != 1]
    tol = (cols / 128 + 32) * U
    nb = -(-cols // 128)
    for r in (None, res):
        y64, h64 = norm_ref(x[fine], w, None if r is None else r[fine], 1e-5)
        got = pb.ops_rms_norm(x, w, residual=r, eps=1e-5)
        y, h = got if r is not None else (got, None)
        assert ((y[fine].double() - y64).abs() <= (tol + V[dtype]) * y64.abs() * 1.0001 + LEAST[dtype]).all()
        assert y[1::3].isnan().all()
        got = pb.ops_rms_norm_fp8(x, w, residual=r, eps=1e-5)
        pad = torch.nn.functional.pad(y64, (0, nb * 128 - cols)).view(len(fine), nb, 128)
        s64 = pad.abs().amax(-1).clamp(min=1e-10) / 448
        assert ((got[1][fine].double() - s64).abs() <= (tol + 4 * U) * s64).all()
        assert got[1][1::3].isnan().all()
        unit = (pad / s64[..., None]).view(len(fine), -1)[:, :cols]
        far = (got[0][fine].double() - unit).abs()
        assert (far <= torch.clamp(unit.abs() * 2.0 ** -4, min=2.0 ** -10) * 1.001 + 448 * (tol + 8 * U)).all()
        if r is not None:
            want = (x.float() + res.float()).to(dtype)
            assert torch.equal(h[fine], want[fine]) and h[1::3].isnan().all()
            assert torch.equal(got[2][fine], want[fine])
    one = pb.ops_rms_norm(x[:1], w)
    assert torch.equal(pb.ops_rms_norm(x[:1].expand(5, cols), w), one.expand(5, cols))


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_norm_special_rows(dtype):
    g = gen(5)
    cols = 384
    x = randn(g, 8, cols).to(dtype)
    x[1] = 0                                   # eps alone under the root
    x[2, 200] = float("nan")
    x[3, 5] = float("inf")
    x[4, 5], x[4, 6] = float("inf"), -float("inf")
    x[5] *= 1e-4
    x[6, 128:256] = 0                          # one block of zeros
    w = torch.ones(cols, device="cuda", dtype=dtype)
    y = pb.ops_rms_norm(x, w, eps=1e-6)
    q, s = pb.ops_rms_norm_fp8(x, w, eps=1e-6)
    y64, _ = norm_ref(x, w, None, 1e-6)
    assert (y[1] == 0).all() and (q[1].float() == 0).all() and torch.allclose(s[1], torch.full_like(s[1], 1e-10 / 448))
    assert y[2].isnan().all() and q[2].float().isnan().all() and s[2].isnan().all()
    for r in (3, 4):                           # inf * 0 is NaN, the others of the row are 0
        assert torch.equal(y[r].isnan(), y64[r].isnan())
        assert q[r].float().isnan()[5] and s[r, 0].isnan()
    assert (q[6, 128:256].float() == 0).all()
    ok = [0, 5, 6, 7]
    assert ((y[ok].double() - y64[ok]).abs() <= (V[dtype] + 40 * U) * y64[ok].abs() + LEAST[dtype]).all()


def test_norm_leading_dimensions_broadcast_and_empty():
    g = gen(6)
    x = randn(g, 2, 3, 5, 96).to(torch.bfloat16)
    w = randn(g, 96).to(torch.bfloat16)
    y = pb.ops_rms_norm(x, w)
    assert torch.equal(y, pb.ops_rms_norm(x.view(30, 96), w).view(2, 3, 5, 96))
    assert torch.equal(pb.ops_rms_norm(x[0, 0, 0], w), y[0, 0, 0])
    q, s = pb.ops_rms_norm_fp8(x, w)
    assert q.shape == x.shape and s.shape == (2, 3, 5, 1)
    same = x[0, 0, :1].expand(4, 96)           # one row four times
    assert torch.equal(pb.ops_rms_norm(same, w), y[0, 0, :1].expand(4, 96))
    for shape in ((0, 96), (2, 0, 96)):
        q, s, h = pb.ops_rms_norm_fp8(x.new_zeros(shape), w, residual=x.new_zeros(shape))
        assert q.shape == h.shape == shape and s.shape == (*shape[:-1], 1)
    y = pb.ops_rms_norm(x.new_zeros(3, 0), w[:0])
    assert y.shape == (3, 0)


def test_norm_in_place_residual():
    """h may be the residual's (or x's) own memory through the C entry point."""
    from pdefa_b200 import _native as N
    for cols in (640, 641, 4096):
        for into in ("x", "residual"):
            g = gen(cols)
            x, r = (randn(g, 9, cols).to(torch.bfloat16) for _ in range(2))
            w = randn(g, cols).to(torch.bfloat16)
            y, h = pb.ops_rms_norm(x, w, residual=r)
            y2 = torch.empty_like(y)
            dst = x if into == "x" else r
            rc = N.lib().engine_rms_norm_device(
                x.data_ptr(), cols, r.data_ptr(), cols, w.data_ptr(), dst.data_ptr(), cols, y2.data_ptr(), cols, None,
                0, 9, cols, 2, 2, 1e-6, 0, torch.cuda.current_stream().cuda_stream)
            assert rc == 0
            assert torch.equal(dst, h) and torch.equal(y2, y)


# ----------------------------------------------------------------------------
# products
# ----------------------------------------------------------------------------
def e4m3(g, *shape):
    return (randn(g, *shape) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)


def widen(s, n):
    return s.double().repeat_interleave(128, -1)[..., :n]


def operands(g, m, n, k, experts=0):
    nb, kb = -(-n // 128), -(-k // 128)
    lead = (experts,) if experts else ()
    return (e4m3(g, m, k), 0.01 * (0.1 + torch.rand((m, kb), generator=g, device="cuda")), e4m3(g, *lead, n, k),
            0.01 * (0.1 + torch.rand((*lead, nb, kb), generator=g, device="cuda")))


def product_ref(a, sa, b, sb):
    k, n = a.shape[1], b.shape[0]
    wa = a.double() * widen(sa, k)
    wb = b.double() * widen(sb, k) if sb.shape[0] == n and n == 1 else b.double() * widen(
        sb.repeat_interleave(128, 0)[:n], k)
    return wa @ wb.t(), wa.abs() @ wb.abs().t()


def check_product(out, a, sa, b, sb):
    ref, size = product_ref(a, sa, b, sb)
    kb = -(-a.shape[1] // 128)
    tol = (128 + kb + 4) * U * size + V[out.dtype] * ref.abs() + LEAST[out.dtype]
    err = (out.double() - ref).abs()
    assert out.shape == ref.shape
    assert (err <= tol).all(), (float(err.max()), float((err / tol).max()))


PRODUCT_SIZES = [(1, 1, 1), (1, 128, 128), (1, 256, 512), (3, 5, 16), (7, 130, 144), (8, 4096, 1024), (15, 200, 4096),
                 (16, 128, 2048), (17, 129, 129), (31, 1000, 272), (33, 384, 640), (64, 300, 1024), (65, 257, 1040),
                 (100, 1111, 400), (127, 640, 127), (128, 128, 128), (129, 256, 384), (200, 96, 100), (256, 512, 896),
                 (257, 513, 1025), (300, 1024, 256), (513, 768, 512), (1000, 72, 333), (700, 2000, 2048)]


@pytest.mark.parametrize("m,n,k", PRODUCT_SIZES)
@pytest.mark.parametrize("out", DTYPES, ids=ids)
def test_matmul(m, n, k, out):
    a, sa, b, sb = operands(gen(m * 7 + n * 3 + k), m, n, k)
    check_product(pb.ops_matmul_fp8(a, sa, b, sb, out_dtype=out), a, sa, b, sb)


@pytest.mark.parametrize("gap_a,gap_b", [(16, 32), (8, 0), (0, 1), (3, 5)])
@pytest.mark.parametrize("m,n,k", [(5, 300, 512), (140, 260, 400)])
def test_matmul_strides(m, n, k, gap_a, gap_b):
    a, sa, b, sb = operands(gen(gap_a * 10 + gap_b), m, n, k)
    got = pb.ops_matmul_fp8(spaced(a, gap_a), spaced(sa, 1), spaced(b, gap_b), spaced(sb, 2), out_dtype=torch.float32)
    assert torch.equal(got, pb.ops_matmul_fp8(a, sa, b, sb, out_dtype=torch.float32))
    check_product(got, a, sa, b, sb)
    # a base that is not a multiple of 16 bytes
    wide = torch.zeros(m * k + 16, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    off = wide[5:5 + m * k].view(m, k)
    off.copy_(a)
    assert torch.equal(pb.ops_matmul_fp8(off, sa, b, sb, out_dtype=torch.float32), got)
    # one row of a for all rows
    one = a[:1].expand(m, k)
    check_product(pb.ops_matmul_fp8(one, sa, b, sb, out_dtype=torch.float32), one.contiguous(), sa, b, sb)


@pytest.mark.parametrize("m", [4, 40, 300])
def test_matmul_special_values(m):
    n, k = 256, 384
    a, sa, b, sb = operands(gen(m), m, n, k)
    nan = torch.tensor(float("nan"), device="cuda").to(torch.float8_e4m3fn)
    a[1, 130] = nan
    sa[2, 1] = 0                                # a block that counts for nothing
    sa[3, 0] = float("inf")
    out = pb.ops_matmul_fp8(a, sa, b, sb, out_dtype=torch.float32)
    assert out[1].isnan().all() and out[0].isfinite().all() and out[2].isfinite().all()
    assert (~out[3].isfinite()).all()
    b[7, 3] = nan
    out = pb.ops_matmul_fp8(a, sa, b, sb, out_dtype=torch.float32)
    assert out[:, 7].isnan().all() and out[0, torch.arange(n, device="cuda") != 7].isfinite().all()
    # the largest values and scales that still fit, exactly
    a = torch.full((m, k), 448.0, device="cuda").to(torch.float8_e4m3fn)
    b = torch.full((n, k), -448.0, device="cuda").to(torch.float8_e4m3fn)
    out = pb.ops_matmul_fp8(a, torch.ones_like(sa), b, torch.ones_like(sb), out_dtype=torch.float32)
    assert (out == -448.0 * 448.0 * k).all()


def test_matmul_empty():
    z = lambda *s: torch.zeros(s, device="cuda")                          # noqa: E731
    q = lambda *s: torch.zeros(s, device="cuda").to(torch.float8_e4m3fn)   # noqa: E731
    assert pb.ops_matmul_fp8(q(0, 64), z(0, 1), q(32, 64), z(1, 1)).shape == (0, 32)
    assert pb.ops_matmul_fp8(q(4, 64), z(4, 1), q(0, 64), z(0, 1)).shape == (4, 0)
    out = pb.ops_matmul_fp8(q(4, 0), z(4, 0), q(8, 0), z(1, 0))
    assert out.shape == (4, 8) and (out == 0).all()


GROUPS = [(1, [1]), (1, [0, 0, 1]), (4, [0, 4, 0]), (64, None), (200, [200]), (200, [0, 130, 0, 0, 70]), (300, None),
          (1000, None), (129, [1, 127, 1]), (2000, None)]


@pytest.mark.parametrize("rows,counts", GROUPS)
@pytest.mark.parametrize("n,k", [(128, 128), (200, 272), (513, 1024), (48, 100)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16], ids=ids)
def test_grouped(rows, counts, n, k, out):
    g = gen(rows + n + k)
    if counts is None:
        rng = np.random.default_rng(rows)
        e = 12
        p = rng.random(e) ** 3
        counts = rng.multinomial(rows, p / p.sum()).tolist()
    a, sa, b, sb = operands(g, rows, n, k, experts=len(counts))
    off = torch.tensor([0] + np.cumsum(counts).tolist(), dtype=torch.int32, device="cuda")
    got = pb.ops_matmul_grouped_fp8(a, sa, b, sb, off, out_dtype=out)
    for e, (lo, hi) in enumerate(zip(off.tolist(), off.tolist()[1:])):
        if hi > lo:
            check_product(got[lo:hi], a[lo:hi], sa[lo:hi], b[e], sb[e])


def test_grouped_rows_of_no_expert_and_odd_offsets():
    rows, n, k = 150, 160, 256
    a, sa, b, sb = operands(gen(1), rows, n, k, experts=3)
    off = torch.tensor([10, 60, 60, 140], dtype=torch.int32, device="cuda")
    out = pb.ops_matmul_grouped_fp8(a, sa, b, sb, off, out_dtype=torch.float32)
    assert (out[:10] == 0).all() and (out[140:] == 0).all()
    check_product(out[10:60], a[10:60], sa[10:60], b[0], sb[0])
    check_product(out[60:140], a[60:140], sa[60:140], b[2], sb[2])
    # outside 0 .. rows: cut there
    off = torch.tensor([-5, 20, 20, 1 << 30], dtype=torch.int32, device="cuda")
    out = pb.ops_matmul_grouped_fp8(a, sa, b, sb, off, out_dtype=torch.float32)
    check_product(out[:20], a[:20], sa[:20], b[0], sb[0])
    check_product(out[20:], a[20:], sa[20:], b[2], sb[2])
    # falling offsets: nothing but the named rows is touched, and nothing is out of bounds
    off = torch.tensor([0, 100, 50, 150], dtype=torch.int32, device="cuda")
    out = pb.ops_matmul_grouped_fp8(a, sa, b, sb, off, out_dtype=torch.float32)
    check_product(out[:50], a[:50], sa[:50], b[0], sb[0])
    check_product(out[100:], a[100:], sa[100:], b[2], sb[2])
    none = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert (pb.ops_matmul_grouped_fp8(a, sa, b, sb, none) == 0).all()


def test_grouped_strides():
    rows, n, k = 90, 130, 400
    a, sa, b, sb = operands(gen(2), rows, n, k, experts=4)
    off = torch.tensor([0, 20, 21, 21, 90], dtype=torch.int32, device="cuda")
    want = pb.ops_matmul_grouped_fp8(a, sa, b, sb, off, out_dtype=torch.float32)
    for ga, gb in ((16, 16), (1, 3)):
        got = pb.ops_matmul_grouped_fp8(spaced(a, ga), spaced(sa, 2), spaced(b, gb), spaced(sb, 1), off,
                                        out_dtype=torch.float32)
        assert torch.equal(got, want)
    # every other expert of a larger weight
    big, bsc = b.repeat_interleave(2, 0), sb.repeat_interleave(2, 0)
    assert torch.equal(pb.ops_matmul_grouped_fp8(a, sa, big[::2], bsc[::2], off, out_dtype=torch.float32), want)


# ----------------------------------------------------------------------------
# sampling
# ----------------------------------------------------------------------------
def acceptable(x, e, t, k, p, m, slack=2e-5):
    """Tokens that a 32-bit evaluation may return for one row, and their shares: those
    kept when every bound is `slack` looser whose race is within `slack` of the best
    among those kept when every bound is as much tighter."""
    x = np.nan_to_num(x.astype(np.float64), nan=-np.inf, posinf=np.inf, neginf=-np.inf)
    mx = x.max()
    if mx == -np.inf:
        return {-1}, {-1: 0.0}
    if not t > 0:
        t, k = 1.0, 1
    with np.errstate(invalid="ignore"):
        w = np.where(x == mx, 1.0, np.exp((x - mx) / t))
    z = w.sum()
    order = np.lexsort((np.arange(len(x)), -x))
    sw = w[order]
    before = np.concatenate([[0.0], np.cumsum(sw)[:-1]])
    rank = np.arange(len(x))

    def keep(s):
        ok = sw > 0
        if k > 0:
            ok &= rank < k
        if not p >= 1:
            ok &= before < p * z * (1 + s)
        ok &= sw >= m * (1 - s)
        ok[0] = True
        return ok

    with np.errstate(divide="ignore", invalid="ignore"):
        race = sw / e[order].astype(np.float64)
    race = np.where(e[order] >= 0, race, -1.0)
    tight = np.where(keep(-slack), race, -1.0)
    best = tight.max()
    if best < 0:
        return {int(order[0])}, {int(order[0]): sw[0] / z}
    ok = keep(slack) & (race >= best * (1 - slack)) if np.isfinite(best) else keep(slack) & (race == best)
    return {int(i) for i in order[ok]}, {int(i): w[i] / z for i in order[ok]}


def check_sample(logits, noise, t=None, k=None, p=None, m=None):
    rows = logits.shape[0]
    put = lambda v, d: None if v is None else torch.tensor(v, dtype=d, device="cuda")   # noqa: E731
    tok, prob = pb.ops_sample(logits, noise, temperature=put(t, torch.float32), top_k=put(k, torch.int32),
                              top_p=put(p, torch.float32), min_p=put(m, torch.float32))
    assert tok.dtype == torch.int32 and tok.shape == prob.shape == (rows,)
    x, e = logits.float().cpu().numpy(), noise.cpu().numpy()
    f32 = lambda v, i, d: d if v is None else float(np.float32(v[i]))   # noqa: E731
    for i in range(rows):
        ok, share = acceptable(x[i], e[i], f32(t, i, 1.0), 0 if k is None else k[i], f32(p, i, 1.0), f32(m, i, 0.0))
        got = int(tok[i])
        assert got in ok, (i, got, sorted(ok)[:5])
        assert abs(float(prob[i]) - share[got]) <= 1e-5 * share[got] + 1e-38
    return tok, prob


def logits_of(g, rows, vocab, dtype, spikes=True):
    x = randn(g, rows, vocab) * 2.5
    if spikes:
        x += 6.0 * (torch.rand((rows, vocab), generator=g, device="cuda") < 20.0 / vocab)
    return x.to(dtype)


def noise_of(g, rows, vocab):
    return torch.empty(rows, vocab, device="cuda").exponential_(generator=g)


SETTINGS = [dict(), dict(t=0.0), dict(t=0.7, k=50, p=0.9, m=0.02), dict(k=1), dict(k=7), dict(k=1000), dict(p=0.95),
            dict(p=0.3), dict(m=0.1), dict(t=3.0, p=0.999), dict(t=0.05, k=20), dict(p=0.0), dict(m=2.0),
            dict(t=5.0, k=100000), dict(p=0.99999), dict(t=1.5, p=0.8, m=0.001)]


@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 1025, 8191, 32000, 50257, 131072, 262147])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_sample_settings(vocab, dtype):
    g = gen(vocab)
    rows = len(SETTINGS)
    x, e = logits_of(g, rows, vocab, dtype), noise_of(g, rows, vocab)
    check_sample(x, e, t=[s.get("t", 1.0) for s in SETTINGS], k=[s.get("k", 0) for s in SETTINGS],
                 p=[s.get("p", 1.0) for s in SETTINGS], m=[s.get("m", 0.0) for s in SETTINGS])


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 409600), (torch.float32, 409701), (torch.bfloat16, 900001)])
def test_sample_long_rows(dtype, vocab):
    """Rows that do not fit the shared memory of a cluster."""
    g = gen(vocab)
    x, e = logits_of(g, 4, vocab, dtype), noise_of(g, 4, vocab)
    x[3] = -float("inf")
    tok, _ = check_sample(x, e, t=[0.8, 0.0, 1.5, 1.0], k=[60, 0, 0, 0], p=[0.9, 1.0, 0.97, 1.0])
    assert tok[1] == x[1].argmax() and tok[3] == -1


@pytest.mark.parametrize("rows", [1, 2, 5, 40, 147, 300])
@pytest.mark.parametrize("vocab", [640, 20011])
def test_sample_row_counts(rows, vocab):
    g = gen(rows)
    x, e = logits_of(g, rows, vocab, torch.bfloat16), noise_of(g, rows, vocab)
    check_sample(x, e, t=[0.9] * rows, k=[30 + i % 9 for i in range(rows)], p=[0.5 + 0.4 * i / rows for i in range(rows)])
    check_sample(x, e)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("vocab", [3000, 33001])
def test_sample_many_rows(vocab, dtype):
    """More rows than run at once, with every setting and special rows among them."""
    g = gen(vocab + 1)
    rows = 20 * len(SETTINGS)
    x, e = logits_of(g, rows, vocab, dtype), noise_of(g, rows, vocab)
    inf = float("inf")
    n = len(SETTINGS)
    for i in range(n):                            # a special row of each kind under every setting
        x[i] = -inf
        x[n + i, 100:] = -inf
        x[2 * n + i, [5, 2900]] = inf
        x[3 * n + i, ::3] = float("nan")
        x[4 * n + i] = torch.round(x[4 * n + i])
        x[5 * n + i] = 2.5
        e[6 * n + i] = float("nan")
        x[7 * n + i] = torch.finfo(dtype).min
        x[8 * n + i, 1500:] = torch.finfo(dtype).min
        x[9 * n + i] *= 0.01                      # nearly even: long lists
    cycle = [SETTINGS[i % n] for i in range(rows)]
    tok, _ = check_sample(x, e, t=[s.get("t", 1.0) for s in cycle], k=[s.get("k", 0) for s in cycle],
                          p=[s.get("p", 1.0) for s in cycle], m=[s.get("m", 0.0) for s in cycle])
    assert (tok[:n] == -1).all()
    again = pb.ops_sample(spaced(x, 3), spaced(e, 1))
    want = pb.ops_sample(x, e)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("k,p", [(0, 1.0), (1, 1.0), (5, 1.0), (0, 0.5), (100, 0.3)])
def test_sample_ties(dtype, k, p):
    """Equal logits are ordered by index: the filters cut inside a run of equals."""
    g = gen(9)
    rows, vocab = 6, 5000
    x = torch.round(randn(g, rows, vocab)).to(dtype)
    x[0] = 1.5
    x[1, 1000:] = -float("inf")
    x[2] = torch.where(x[2] > 0, torch.zeros_like(x[2]), -torch.zeros_like(x[2]))   # +0 and -0 are equal
    check_sample(x, noise_of(g, rows, vocab), k=[k] * rows, p=[p] * rows)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_sample_masks_and_special_values(dtype):
    g = gen(10)
    rows, vocab = 12, 3001
    x, e = logits_of(g, rows, vocab, dtype), noise_of(g, rows, vocab)
    inf, low = float("inf"), torch.finfo(dtype).min
    x[0] = -inf                                   # nothing left
    x[1] = low                                    # the type's lowest value everywhere
    x[2, :3000] = -inf                            # one token left
    x[3, 1::2] = low
    x[4, 17] = inf
    x[5, [17, 40, 2999]] = inf
    x[6, 5] = float("nan")
    x[7] = float("nan")
    x[8] = torch.finfo(dtype).max
    x[9, :] = low
    x[9, 12] = torch.finfo(dtype).max
    for k, p, m, t in ((0, 1.0, 0.0, 1.0), (3, 0.9, 0.0, 0.6), (0, 0.9, 0.1, 2.0), (0, 0.5, 0.0, 1e30), (0, 1.0, 0.0, 0.0)):
        tok, prob = check_sample(x, e, t=[t] * rows, k=[k] * rows, p=[p] * rows, m=[m] * rows)
        assert tok[0] == -1 and prob[0] == 0 and tok[7] == -1 and tok[2] == 3000 and prob[2] == 1
        assert tok[4] == 17 and tok[5] in (17, 40, 2999)
        # 2 * 65504 / 1e30 is nothing: at that temperature the half-precision row 9 is even
        assert tok[9] == 12 or (dtype == torch.float16 and t == 1e30)


def test_sample_odd_settings_and_noise():
    g = gen(11)
    rows, vocab = 10, 2000
    x, e = logits_of(g, rows, vocab, torch.float32), noise_of(g, rows, vocab)
    nan = float("nan")
    tok, _ = check_sample(x, e, t=[-1.0, nan, 1, 1, 1, 1, 1, 1, 1, 1], k=[0, 0, -7, 1 << 30, 0, 0, 0, 0, 0, 0],
                          p=[1, 1, 1, 1, -0.5, 7.0, 1, 1, 1, 1], m=[0, 0, 0, 0, 0, 0, -1.0, 5.0, 0, 0])
    assert tok[0] == x[0].argmax() and tok[1] == x[1].argmax() and tok[4] == x[4].argmax() and tok[7] == x[7].argmax()
    e[0] = nan                                    # no usable variate: the first token
    e[1] = -1.0
    e[2] = 0.0                                    # all equal at infinity: the lowest index of the kept
    e[3] = float("inf")
    e[4, x[4].argmax()] = 0.0
    tok, _ = check_sample(x, e, k=[50] * rows)
    assert tok[0] == x[0].argmax() and tok[1] == x[1].argmax() and tok[4] == x[4].argmax()
    assert tok[2] == x[2].topk(50).indices.min()


def test_sample_adversarial_noise():
    """Variates that make the race run against the order: every round's winner is the last
    token still in, so the filters cut only through the bisection."""
    rows, vocab = 4, 4096
    x = torch.linspace(4, -4, vocab, device="cuda").repeat(rows, 1)
    w = torch.exp((x - 4).double())
    e = (w / (1 + torch.arange(vocab, device="cuda"))).float()     # w / e rises along the order
    check_sample(x, e, k=[1, 10, 0, 0], p=[1, 1, 0.25, 1.0], m=[0, 0, 0, 0.5])


def test_sample_draws_with_the_given_probabilities():
    n, vocab = 20000, 12
    x = torch.tensor([2.0, 1.0, 1.5, -1.0, 0.0, 0.5, -2.0, 1.9, -0.5, 0.1, -3.0, 1.2], device="cuda")
    tok, prob = pb.ops_sample(x.expand(n, vocab), noise_of(gen(12), n, vocab), top_k=torch.full((n,), 5, dtype=torch.int32,
                                                                                           device="cuda"))
    w = torch.exp(x.double()).cpu()
    kept = torch.topk(w, 5).indices
    share = torch.zeros(vocab, dtype=torch.float64)
    share[kept] = w[kept] / w[kept].sum()
    seen = torch.bincount(tok.long().cpu(), minlength=vocab).double() / n
    assert ((seen - share).abs() <= 6 * (share * (1 - share) / n).sqrt()).all()    # six standard deviations
    assert torch.allclose(prob.cpu().double(), (w / w.sum())[tok.long().cpu()], rtol=1e-5)


def test_sample_strides_and_empty():
    g = gen(13)
    x, e = logits_of(g, 7, 1003, torch.bfloat16), noise_of(g, 7, 1003)
    want = pb.ops_sample(x, e)
    for gx, ge in ((1, 0), (5, 3), (8, 4)):
        got = pb.ops_sample(spaced(x, gx), spaced(e, ge))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    wide = torch.zeros(8, 1003, dtype=torch.bfloat16, device="cuda").view(-1)
    off = wide[1:1 + 7 * 1003].view(7, 1003)
    off.copy_(x)
    assert torch.equal(pb.ops_sample(off, e)[0], want[0])
    tok, prob = pb.ops_sample(x[:0], e[:0])
    assert tok.shape == prob.shape == (0,)


# ----------------------------------------------------------------------------
# all
# ----------------------------------------------------------------------------
def test_repeatable_and_on_other_streams():
    g = gen(14)
    x = randn(g, 70, 640).to(torch.bfloat16)
    w = randn(g, 640).to(torch.bfloat16)
    a, sa, b, sb = operands(g, 70, 1000, 640)
    lg, e = logits_of(g, 70, 30000, torch.float32), noise_of(g, 70, 30000)
    p = torch.full((70,), 0.9, device="cuda")

    def all_of():
        return (*pb.ops_rms_norm_fp8(x, w, residual=x), pb.ops_matmul_fp8(a, sa, b, sb), *pb.ops_sample(lg, e, top_p=p))

    want = all_of()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            got = all_of()
        side.synchronize()
        for u, v in zip(got, want):
            assert torch.equal(u.view(torch.uint8), v.view(torch.uint8))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = all_of()
    x.mul_(2)
    lg.add_(1.0)
    graph.replay()
    torch.cuda.synchronize()
    for u, v in zip(got, all_of()):
        assert torch.equal(u.view(torch.uint8), v.view(torch.uint8))


def test_refusals():
    f = lambda *s, d=torch.float32: torch.zeros(s, device="cuda", dtype=d)   # noqa: E731
    q = lambda *s: torch.zeros(s, device="cuda").to(torch.float8_e4m3fn)       # noqa: E731
    i = lambda *s: torch.zeros(s, device="cuda", dtype=torch.int32)          # noqa: E731
    err = pytest.raises(pb.PdefaError)
    typ = pytest.raises(TypeError)
    for what, call in [
        (typ, lambda: pb.ops_rms_norm(torch.zeros(2, 8), f(8))), (typ, lambda: pb.ops_rms_norm(f(2, 8), f(8).cpu())),
        (typ, lambda: pb.ops_rms_norm(f(2, 8, d=torch.float64), f(8))), (typ, lambda: pb.ops_rms_norm([[1.0]], f(1))),
        (typ, lambda: pb.ops_rms_norm(f(2, 8), f(8, d=torch.float16))), (err, lambda: pb.ops_rms_norm(f(2, 8), f(9))),
        (err, lambda: pb.ops_rms_norm(f(2, 8), f(8), residual=f(2, 9))), (err, lambda: pb.ops_rms_norm(f(8, 2).t(), f(8))),
        (typ, lambda: pb.ops_rms_norm(f(2, 8), f(8), residual=f(2, 8, d=torch.float16))),
        (err, lambda: pb.ops_rms_norm(f(2, 8), f(8), eps=-1.0)), (err, lambda: pb.ops_rms_norm(f(2, 8), f(8), eps=float("nan"))),
        (err, lambda: pb.ops_rms_norm(f(4, 6, 8)[:, ::4].transpose(0, 1), f(8))),
        (typ, lambda: pb.ops_matmul_fp8(f(2, 8), f(2, 1), q(4, 8), f(1, 1))),
        (typ, lambda: pb.ops_matmul_fp8(q(2, 8), f(2, 1, d=torch.float16), q(4, 8), f(1, 1))),
        (err, lambda: pb.ops_matmul_fp8(q(2, 8), f(2, 1), q(4, 9), f(1, 1))),
        (err, lambda: pb.ops_matmul_fp8(q(2, 8), f(2, 2), q(4, 8), f(1, 1))),
        (err, lambda: pb.ops_matmul_fp8(q(2, 8), f(2, 1), q(4, 8), f(4, 1))),
        (err, lambda: pb.ops_matmul_fp8(q(8, 2).t(), f(2, 1), q(4, 8), f(1, 1))),
        (typ, lambda: pb.ops_matmul_fp8(q(2, 8), f(2, 1), q(4, 8), f(1, 1), out_dtype=torch.int8)),
        (err, lambda: pb.ops_matmul_grouped_fp8(q(2, 8), f(2, 1), q(3, 4, 8), f(3, 1, 1), i(3))),
        (typ, lambda: pb.ops_matmul_grouped_fp8(q(2, 8), f(2, 1), q(3, 4, 8), f(3, 1, 1), i(4).long())),
        (err, lambda: pb.ops_matmul_grouped_fp8(q(2, 8), f(2, 1), q(4, 8), f(1, 1), i(4))),
        (err, lambda: pb.ops_sample(f(2, 8), f(2, 9))), (typ, lambda: pb.ops_sample(f(2, 8), f(2, 8, d=torch.float16))),
        (typ, lambda: pb.ops_sample(f(2, 8), f(2, 8), top_k=f(2))), (err, lambda: pb.ops_sample(f(2, 8), f(2, 8), top_p=f(3))),
        (err, lambda: pb.ops_sample(f(8), f(8))), (err, lambda: pb.ops_sample(f(2, 0), f(2, 0))),
        (typ, lambda: pb.ops_sample(i(2, 8), f(2, 8))),
    ]:
        with what:
            call()
    torch.cuda.synchronize()

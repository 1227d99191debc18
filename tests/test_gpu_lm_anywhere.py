"""The C entry points of the language-model operators on arrays that lie anywhere: every element
offset, rows apart by any distance, repeated rows, inside buffers of NaN (inputs) or of a mark
(outputs), so that a stray access shows. Bounds as in test_gpu_lm.py."""
import numpy as np
import pytest

from pdefa_b200 import _native as N
from test_gpu_lm import DTYPES, LEAST, U, V, acceptable, check_product, gen, ids, norm_ref, operands, randn

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def stream():
    return torch.cuda.current_stream().cuda_stream


class Array:
    """rows x cols of a larger buffer, `off` elements into it and `gap` after each row (the last one too)."""

    def __init__(self, rows, cols, dtype, off=0, gap=0, fill=float("nan"), data=None):
        wide = dtype if dtype != torch.float8_e4m3fn else torch.uint8
        self.mark = 0x7F if wide == torch.uint8 and dtype != wide else fill      # 0x7F: e4m3's NaN
        self.buf = torch.full((off + rows * (cols + gap) + 16,), self.mark, dtype=wide, device="cuda")
        self.stride = cols + gap
        self.raw = self.buf[off:off + rows * self.stride].view(rows, self.stride)
        self.rows = self.raw[:, :cols]
        if data is not None:
            self.rows.copy_(data if wide == dtype else data.view(torch.uint8))
        self.dtype, self.off = dtype, off
        self.ptr = self.buf.data_ptr() + off * self.buf.element_size()

    def value(self):
        return self.rows.contiguous() if self.rows.dtype == self.dtype else self.rows.contiguous().view(self.dtype)

    def untouched_around(self):
        seen = self.buf.clone()
        seen[self.off:self.off + self.raw.numel()].view(self.raw.shape)[:, :self.rows.shape[1]] = self.mark
        return bool((seen == self.mark).all())


def pick(rng, *options):
    return options[rng.integers(len(options))]


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("seed", range(24))
def test_norm_anywhere(seed, dtype):
    rng = np.random.default_rng(seed)
    g = gen(seed)
    rows, cols = int(pick(rng, 1, 2, 7, 40, 700)), int(pick(rng, 1, 5, 16, 127, 130, 513, 1024, 2047, 4097, 8200))
    per = 16 // dtype.itemsize
    alike = seed % 3 == 0                          # all arrays start and step alike, as dense ones do
    off, gap = int(rng.integers(0, per)), int(pick(rng, 0, 0, 1, per, 5))
    place = lambda: (off, gap) if alike else (int(rng.integers(0, per)), int(pick(rng, 0, 1, per, 3)))   # noqa: E731
    x = Array(rows, cols, dtype, *place(), data=(randn(g, rows, cols) * 3).to(dtype))
    res = Array(rows, cols, dtype, *place(), data=randn(g, rows, cols).to(dtype)) if seed % 2 else None
    wd = pick(rng, dtype, torch.float32)
    w = Array(1, cols, wd, int(rng.integers(0, 4)), data=(1 + 0.3 * randn(g, 1, cols)).to(wd))
    h = Array(rows, cols, dtype, *place(), fill=7.0) if res else None
    nb = -(-cols // 128)
    y64, _ = norm_ref(x.value(), w.value()[0], res.value() if res else None, 1e-5)
    tol = (cols / 128 + 32) * U
    for fp8 in (False, True):
        y = Array(rows, cols, torch.float8_e4m3fn if fp8 else dtype, *place(), fill=7.0)
        s = Array(rows, nb, torch.float32, int(rng.integers(0, 4)), int(rng.integers(0, 3)), fill=7.0)
        rc = N.lib().engine_rms_norm_device(
            x.ptr, x.stride, res.ptr if res else None, res.stride if res else 0, w.ptr, h.ptr if h else None, h.stride if h else 0,
            y.ptr, y.stride, s.ptr if fp8 else None, s.stride, rows, cols, CODE[dtype], CODE[wd], 1e-5, 0, stream())
        assert rc == 0
        assert y.untouched_around() and s.untouched_around() and (h is None or h.untouched_around())
        if h:
            assert torch.equal(h.value(), (x.value().float() + res.value().float()).to(dtype))
        if not fp8:
            assert ((y.value().double() - y64).abs() <= (tol + V[dtype]) * y64.abs() * 1.0001 + LEAST[dtype]).all()
            continue
        pad = torch.nn.functional.pad(y64, (0, nb * 128 - cols)).view(rows, nb, 128)
        s64 = pad.abs().amax(-1).clamp(min=1e-10) / 448
        assert ((s.value().double() - s64).abs() <= (tol + 4 * U) * s64).all()
        unit = (pad / s64[..., None]).view(rows, -1)[:, :cols]
        far = (y.value().double() - unit).abs()
        assert (far <= torch.clamp(unit.abs() * 2.0 ** -4, min=2.0 ** -10) * 1.001 + 448 * (tol + 8 * U)).all()


SHAPES = [(1, 1, 5), (3, 130, 100), (8, 1000, 512), (40, 257, 1040), (100, 700, 272), (129, 203, 1040), (257, 640, 2064),
          (300, 6000, 200), (700, 4001, 256), (2600, 1500, 400)]


@pytest.mark.parametrize("out", DTYPES, ids=ids)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("turn", range(3))
def test_matmul_anywhere(shape, turn, out):
    m, n, k = shape
    rng = np.random.default_rng(turn * 1000 + n)
    a, sa, b, sb = operands(gen(n + turn), m, n, k)
    tma = [(0, -k % 16), (16, 16 - k % 16), (int(rng.integers(1, 16)), int(rng.integers(0, 9)))]     # read in place, or not
    pa = Array(m, k, torch.float8_e4m3fn, *tma[turn], data=a)
    pb = Array(n, k, torch.float8_e4m3fn, *tma[(turn + int(rng.integers(3))) % 3], data=b)
    psa, psb = (Array(*s.shape, torch.float32, int(rng.integers(0, 4)), int(rng.integers(0, 3)), data=s) for s in (sa, sb))
    per = 16 // out.itemsize
    po = Array(m, n, out, *((0, -n % per), (per, 2 * per - n % per), (int(rng.integers(0, per)), int(rng.integers(0, per))))[turn], fill=7.0)
    rc = N.lib().engine_matmul_fp8_device(pa.ptr, pa.stride, psa.ptr, psa.stride, pb.ptr, pb.stride, psb.ptr, psb.stride, po.ptr,
                                          po.stride, CODE[out], m, n, k, 0, stream())
    assert rc == 0
    assert po.untouched_around()
    check_product(po.value(), a, sa, b, sb)


@pytest.mark.parametrize("out", DTYPES, ids=ids)
@pytest.mark.parametrize("rows,experts,n,k", [(5, 3, 130, 100), (300, 40, 257, 144), (900, 17, 1041, 400), (5000, 20, 699, 272)])
@pytest.mark.parametrize("turn", range(3))
def test_grouped_anywhere(rows, experts, n, k, turn, out):
    rng = np.random.default_rng(turn * 1000 + n)
    a, sa, b, sb = operands(gen(n + turn), rows, n, k, experts=experts)
    gap = (-k % 16, 16 - k % 16, int(rng.integers(0, 9)))[turn]
    pa = Array(rows, k, torch.float8_e4m3fn, 16 * turn, gap, data=a)
    pb = Array(experts * n, k, torch.float8_e4m3fn, 16 * turn, gap, data=b.reshape(-1, k))
    psb = Array(experts * sb.shape[1], sb.shape[2], torch.float32, turn, turn, data=sb.reshape(-1, sb.shape[2]))
    psa = Array(rows, sa.shape[1], torch.float32, turn, turn, data=sa)
    off = np.sort(rng.integers(0, rows + 1, experts + 1))
    where = torch.from_numpy(off.astype(np.int32)).cuda()
    per = 16 // out.itemsize
    po = Array(rows, n, out, (0, per, 1)[turn], (-n % per, per - n % per, 1)[turn], fill=7.0)
    rc = N.lib().engine_matmul_grouped_fp8_device(
        pa.ptr, pa.stride, psa.ptr, psa.stride, pb.ptr, pb.stride, n * pb.stride, psb.ptr, psb.stride, sb.shape[1] * psb.stride,
        where.data_ptr(), experts, po.ptr, po.stride, CODE[out], rows, n, k, 0, stream())
    assert rc == 0
    assert po.untouched_around()
    got = po.value()
    assert (got[:off[0]] == 0).all() and (got[off[-1]:] == 0).all()
    for e, (lo, hi) in enumerate(zip(off, off[1:])):
        if hi > lo:
            check_product(got[lo:hi], a[lo:hi], sa[lo:hi], b[e], sb[e])


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("seed", range(12))
def test_sample_anywhere(seed, dtype):
    rng = np.random.default_rng(seed)
    g = gen(seed)
    rows, vocab = int(pick(rng, 1, 6, 35, 90, 160)), int(pick(rng, 1, 3, 9, 700, 5003, 20001))
    x = Array(rows, vocab, dtype, int(rng.integers(0, 16 // dtype.itemsize)), int(rng.integers(0, 9)),
              data=(randn(g, rows, vocab) * 2.5).to(dtype))
    e = Array(rows, vocab, torch.float32, int(rng.integers(0, 4)), int(rng.integers(0, 5)),
              data=torch.empty(rows, vocab, device="cuda").exponential_(generator=g))
    x.raw[:, vocab:] = float("inf")                # what would win if it were read
    e.raw[:, vocab:] = 0.0
    sets = [pick(rng, (1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.02), (0.0, 0, 1.0, 0.0), (1.0, 7, 1.0, 0.0), (1.3, 0, 0.9, 0.0),
                 (1.0, 0, 1.0, 0.1)) for _ in range(rows)]
    t, k, p, m = (torch.tensor(v, dtype=d, device="cuda") for v, d in
                  zip(zip(*sets), (torch.float32, torch.int32, torch.float32, torch.float32)))
    tok, prob = Array(1, rows, torch.int32, 1, fill=77), Array(1, rows, torch.float32, 1, fill=7.0)
    rc = N.lib().engine_sample_device(x.ptr, x.stride, CODE[dtype], e.ptr, e.stride, t.data_ptr(), k.data_ptr(), p.data_ptr(), m.data_ptr(),
                                      rows, vocab, tok.ptr, prob.ptr, 0, stream())
    assert rc == 0
    assert tok.untouched_around() and prob.untouched_around()
    xs, es = x.value().float().cpu().numpy(), e.value().cpu().numpy()
    f = lambda v: float(np.float32(v))   # noqa: E731
    for i, (ti, ki, pi, mi) in enumerate(sets):
        ok, share = acceptable(xs[i], es[i], f(ti), ki, f(pi), f(mi))
        got = int(tok.value()[0, i])
        assert got in ok
        assert abs(float(prob.value()[0, i]) - share[got]) <= 1e-5 * share[got] + 1e-38

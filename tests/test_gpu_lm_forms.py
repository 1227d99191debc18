"""The language-model operators in every form of their kernels: sizes that the plans send to wide
tiles and pairs, split tiles, several tiles per CTA, many experts and streaming accesses, against
their definitions in 64 bits (bounds as in test_gpu_lm.py)."""
import threading

import numpy as np
import pytest

import pdefa_b200 as pb
import test_gpu_lm as base
from pdefa_b200 import _native as N
from test_gpu_lm import DTYPES, check_product, gen, ids, logits_of, noise_of, operands, randn, spaced
from test_lm_plans import FORMS, GROUP_FORMS

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
shape_ids = lambda f: "x".join(str(v) for v in f[:-2])   # noqa: E731


@pytest.mark.parametrize("form", FORMS, ids=shape_ids)
def test_matmul_forms(form):
    m, n, k = form[:3]
    a, sa, b, sb = operands(gen(m + n + k), m, n, k)
    for out in DTYPES:
        check_product(pb.ops_matmul_fp8(a, sa, b, sb, out_dtype=out), a, sa, b, sb)


@pytest.mark.parametrize("m,n,k", [(2600, 5000, 400), (300, 20000, 400), (20, 45000, 130)])
def test_matmul_forms_with_strides(m, n, k):
    """Spaced rows that TMA reads in place, and ones that are copied first."""
    a, sa, b, sb = operands(gen(3), m, n, k)
    want = pb.ops_matmul_fp8(a, sa, b, sb)
    for ga, gb in ((16, 112), (0, 5)):
        assert torch.equal(pb.ops_matmul_fp8(spaced(a, ga), spaced(sa, 3), spaced(b, gb), spaced(sb, 1)), want)


@pytest.mark.parametrize("out", DTYPES, ids=ids)
@pytest.mark.parametrize("m,n,k,gap", [(2600, 4999, 400, 9), (2600, 5000, 400, 8), (700, 4001, 256, 7), (700, 4001, 256, 2),
                                       (300, 6001, 1000, 3), (33, 40001, 400, 1)])
def test_matmul_output_rows_apart(m, n, k, gap, out):
    """Through the C entry point: the last columns of aligned and unaligned rows, nothing written between rows."""
    a, sa, b, sb = operands(gen(n), m, n, k)
    wide = torch.full((m, n + gap), 7.0, device="cuda", dtype=out)
    rc = N.lib().engine_matmul_fp8_device(a.data_ptr(), k, sa.data_ptr(), sa.shape[1], b.data_ptr(), k, sb.data_ptr(), sb.shape[1],
                                          wide.data_ptr(), n + gap, CODE[out], m, n, k, 0,
                                          torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    check_product(wide[:, :n], a, sa, b, sb)
    assert (wide[:, n:] == 7.0).all()


@pytest.mark.parametrize("m,n,k", [(5, 300, 100), (140, 260, 399), (300, 20000, 130), (2600, 5000, 403), (255, 640, 2063)])
def test_matmul_rows_that_end_inside_16_bytes(m, n, k):
    """Rows that TMA reads in place although k is not a multiple of 16: what follows them (NaN) stays out."""
    a, sa, b, sb = operands(gen(k), m, n, k)
    gap = -k % 16
    got = pb.ops_matmul_fp8(spaced(a, gap), sa, spaced(b, gap), sb, out_dtype=torch.float32)
    check_product(got, a, sa, b, sb)
    assert torch.equal(got, pb.ops_matmul_fp8(a, sa, b, sb, out_dtype=torch.float32))


def uneven(rng, rows, experts):
    """Counts that fall steeply, with a run of empty experts over a boundary of 32."""
    p = rng.random(experts) ** 3 + 0.01
    p[25:min(36, experts - 1)] = 0
    return rng.multinomial(rows, p / p.sum())


def check_groups(got, off, a, sa, b, sb):
    for e, (lo, hi) in enumerate(zip(off, off[1:])):
        if hi > lo:
            check_product(got[lo:hi], a[lo:hi], sa[lo:hi], b[e], sb[e])


@pytest.mark.parametrize("form", GROUP_FORMS, ids=shape_ids)
def test_grouped_forms(form):
    rows, experts, n, k = form[:4]
    counts = uneven(np.random.default_rng(rows), rows, experts)
    a, sa, b, sb = operands(gen(rows + experts), rows, n, k, experts=experts)
    off = [0, *np.cumsum(counts).tolist()]
    assert 0 in counts and off[-1] == rows
    for out in DTYPES:
        got = pb.ops_matmul_grouped_fp8(a, sa, b, sb, torch.tensor(off, dtype=torch.int32, device="cuda"), out_dtype=out)
        check_groups(got, off, a, sa, b, sb)


@pytest.mark.parametrize("rows,n", [(700, 300), (6500, 904)])
@pytest.mark.parametrize("out", DTYPES, ids=ids)
def test_grouped_odd_offsets_of_many_experts(rows, n, out):
    """Offsets that fall, also from one chunk of 32 experts to the next, or lie outside; rows of no expert."""
    experts, k = 70, 272
    rng = np.random.default_rng(n)
    a, sa, b, sb = operands(gen(n), rows, n, k, experts=experts)
    off = np.sort(rng.integers(3, rows - 3, experts + 1))
    off[5], off[31], off[32], off[33] = 0, off[40], off[20], off[10]
    off[64], off[65] = off[66] + 1, -4
    # what they count as: the nearest value within 0 .. rows that is not below one before it
    counts_as = np.maximum.accumulate(np.clip(off, 0, rows)).tolist()
    got = pb.ops_matmul_grouped_fp8(a, sa, b, sb, torch.from_numpy(off.astype(np.int32)).cuda(), out_dtype=out)
    check_groups(got, counts_as, a, sa, b, sb)
    assert (got[:counts_as[0]] == 0).all() and (got[counts_as[-1]:] == 0).all()


@pytest.mark.parametrize("dtype,cols", [(torch.bfloat16, 8192), (torch.float16, 4096), (torch.float32, 4096)], ids=str)
@pytest.mark.parametrize("gap", [0, 8])
def test_norm_beyond_the_cache(dtype, cols, gap):
    """Over 64 MB with a residual, where accesses stream."""
    rows = (72 << 20) // (3 * dtype.itemsize * cols)
    base.test_norm(rows, cols, dtype, True, gap)


def test_two_threads():
    """Calls from two host threads, each on its own stream."""
    g = gen(4)
    x, w = randn(g, 300, 1031).to(torch.bfloat16), randn(g, 1031).to(torch.bfloat16)
    products = [operands(g, m, n, k) for m, n, k in ((20, 1000, 2064), (2600, 5000, 400), (7, 300, 133))]
    lg, e = logits_of(g, 20, 30000, torch.float32), noise_of(g, 20, 30000)

    def all_of():
        return [*pb.ops_rms_norm_fp8(x, w, residual=x), *(pb.ops_matmul_fp8(*p) for p in products), *pb.ops_sample(lg, e)]

    want = all_of()
    torch.cuda.synchronize()
    wrong = []

    def work():
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got = [all_of() for _ in range(20)]
        side.synchronize()
        wrong.extend(1 for run in got for u, v in zip(run, want) if not torch.equal(u.view(torch.uint8), v.view(torch.uint8)))
        done.append(1)

    done = []
    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(done) == 2 and not wrong


def test_offsets_beyond_32_bits():
    """The last rows of arrays of more than 2^31 elements."""
    g = gen(5)
    rows, cols = 270000, 8191
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[:2], x[-3:] = randn(g, 2, cols).bfloat16(), randn(g, 3, cols).bfloat16()
    w = torch.ones(cols, dtype=torch.bfloat16, device="cuda")
    y64, _ = base.norm_ref(x[-3:], w, None, 1e-5)
    y = pb.ops_rms_norm(x, w, eps=1e-5)[-3:]
    assert ((y.double() - y64).abs() <= (96 * base.U + 2.0 ** -8) * y64.abs() * 1.0001).all()
    del x
    m, n, k = 17000, 131072, 128
    a, sa, b, sb = operands(g, m, n, k)
    out = pb.ops_matmul_fp8(a, sa, b, sb)
    for lo in (0, 16250, 16990):
        check_product(out[lo:lo + 10], a[lo:lo + 10], sa[lo:lo + 10], b, sb)
    tail = out[-40:].float()
    e = torch.empty(m, n, device="cuda")
    e[-40:].exponential_(generator=g)
    t = torch.full((m,), 0.9, device="cuda")
    t[:-40] = 0
    tok, prob = pb.ops_sample(out, e, temperature=t)
    want = pb.ops_sample(out[-40:].clone(), e[-40:].clone(), temperature=t[-40:].clone())
    assert torch.equal(tok[-40:], want[0]) and torch.allclose(prob[-40:], want[1], rtol=1e-4, atol=1e-37)
    assert torch.equal(tok[:40].long(), out[:40].float().argmax(1)) and tail.isfinite().all()

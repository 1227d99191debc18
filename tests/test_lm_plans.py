"""Which form of a kernel a call gets, without a GPU: the rules over their ranges."""
import ctypes as C

import pytest

from pdefa_b200 import _native as N

F32, F16, BF16 = 0, 1, 2
RESIDENT = {8: 30, 4: 68, 2: 148}       # clusters of that many CTAs that run well at once


def sample_ctas(rows, vocab, dtype):
    n = C.c_int32(-1)
    assert N.lib().engine_sample_plan(rows, vocab, dtype, C.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [1, 1000, 1537, 8000, 32000, 50257, 60001, 100001, 131072, 262147])
def test_sample_clusters_are_resident_at_once(vocab, dtype):
    """No cluster is larger than leaves all rows' resident, unless the slices need it or long rows may wait; the
    limits are the same for rows of 1000 and of 262147, and more rows never get larger clusters."""
    size = vocab * (4 if dtype == F32 else 2)
    need = next(n for n in (1, 2, 4, 8) if n == 8 or size <= n * 102400)
    before = 8
    for rows in range(1, 400):
        n = sample_ctas(rows, vocab, dtype)
        assert n in (1, 2, 4, 8) and need <= n <= before
        assert n == need or rows <= (110 if n == 4 and vocab >= 80000 else RESIDENT[n]), rows
        assert n == need or size >= n * 3072
        before = n


def test_sample_rows_that_no_cluster_holds():
    assert sample_ctas(4, 409600, F32) == 8 and sample_ctas(4, 409701, F32) == 0
    assert sample_ctas(1000, 819200, BF16) == 8 and sample_ctas(1000, 900001, F16) == 0
    assert N.lib().engine_sample_plan(4, 0, F32, C.byref(C.c_int32())) == 6
    assert N.lib().engine_sample_plan(4, 10, 5, C.byref(C.c_int32())) == 7
    assert N.lib().engine_sample_plan(4, 10, F32, None) == 1


def matmul_plan(m, n, k, experts=0, dtype=BF16, aligned=True, sms=148, clusters=(74, 35, 16)):
    """(CTAs of a wide tile or 0, tokens of a tile, CTAs of a split)"""
    held, plan = (C.c_int32 * 3)(*clusters), (C.c_int32 * 3)()
    assert N.lib().engine_matmul_fp8_plan(m, n, k, experts, dtype, aligned, sms, held, plan) == 0
    return tuple(plan)


def wide_waves(m, n, pair):
    tiles = -(-m // (128 * pair)) * -(-n // 256)
    return -(-tiles // (148 // pair))


@pytest.mark.parametrize("n,k", [(4096, 4096), (8192, 4096), (28672, 8192), (50264, 4096), (128256, 4096), (151936, 2048)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_pairs_never_make_more_waves_than_single_ctas(n, k, dtype):
    """A pair's tile is 256 tokens: with few of them, or an odd number of 128s, its second half is empty."""
    seen = set()
    for m in [*range(1, 700, 9), 128, 129, 256, 257, 384, 640, 1000, 4096, 8192]:
        wide, tokens, split = matmul_plan(m, n, k, dtype=dtype)
        seen.add(wide)
        if wide == 2:
            assert m > 128 and tokens == 256 and wide_waves(m, n, 2) <= wide_waves(m, n, 1), m
    assert 2 in seen


def test_plan_of_head_shapes():
    assert matmul_plan(100, 128256, 4096) == (1, 128, 1)
    assert matmul_plan(300, 50264, 4096) == (1, 128, 1)
    assert matmul_plan(256, 128256, 4096) == (2, 256, 1)
    assert matmul_plan(8192, 8192, 4096) == (2, 256, 1)


def test_plan_refusals():
    held, plan = (C.c_int32 * 3)(74, 35, 16), (C.c_int32 * 3)()
    call = N.lib().engine_matmul_fp8_plan
    assert call(0, 1, 1, 0, F32, 1, 148, held, plan) == 6 and call(1, 1, 1, 1025, F32, 1, 148, held, plan) == 6
    assert call(1, 1, 1, 0, 3, 1, 148, held, plan) == 7 and call(1, 1, 1, 0, F32, 1, 1, held, plan) == 7
    assert call(1, 1, 1, 0, F32, 1, 148, None, plan) == 1 and call(1, 1, 1, 0, F32, 1, 148, held, None) == 1


# m, n, k and the plan for 32- and for 16-bit outputs: every form of the product's kernels, with
# several tiles per CTA, partial tiles and blocks, and output rows aligned or not. The GPU tests
# compute these, so a refit that changes a plan shows here.
FORMS = [
    (2600, 5000, 400, (2, 256, 1), (2, 256, 1)), (520, 9000, 640, (2, 256, 1), (2, 256, 1)),
    (20000, 304, 130, (2, 256, 1), (2, 256, 1)), (2000, 2600, 300, (2, 256, 1), (2, 256, 1)),
    (1500, 5001, 4000, (2, 256, 1), (2, 256, 1)), (2600, 5001, 400, (0, 128, 1), (2, 256, 1)),
    (300, 20000, 400, (1, 128, 1), (1, 128, 1)), (700, 4000, 256, (1, 128, 1), (1, 128, 1)),
    (777, 3001, 4000, (1, 128, 1), (1, 128, 1)),
    (5, 40000, 256, (0, 16, 1), (0, 16, 1)), (20, 45000, 130, (0, 32, 1), (0, 32, 1)),
    (33, 40000, 400, (0, 64, 1), (0, 64, 1)), (300, 6000, 1000, (0, 128, 1), (0, 128, 1)),
    (16, 5000, 2064, (0, 16, 2), (0, 16, 2)), (129, 203, 1040, (0, 16, 4), (0, 16, 4)), (50, 128, 4096, (0, 16, 8), (0, 16, 8)),
    (255, 640, 2064, (0, 32, 2), (0, 32, 2)), (257, 383, 2064, (0, 32, 4), (0, 32, 4)), (161, 200, 3000, (0, 32, 8), (0, 32, 8)),
    (255, 1279, 4096, (0, 64, 2), (0, 64, 2)), (257, 640, 4096, (0, 64, 4), (0, 64, 4)), (300, 203, 8192, (0, 64, 8), (0, 64, 8)),
    (255, 2600, 8192, (0, 128, 2), (0, 128, 2)), (255, 1279, 8192, (0, 128, 4), (0, 128, 4)),
]
# rows, experts, n, k: grouped plans
GROUP_FORMS = [
    (500, 64, 1300, 272, (0, 16, 1), (0, 16, 1)), (500, 33, 1300, 272, (0, 32, 1), (0, 32, 1)), (1500, 1024, 130, 128, (0, 16, 1), (0, 16, 1)),
    (2500, 200, 700, 400, (0, 32, 1), (0, 32, 1)), (2000, 64, 1301, 272, (0, 64, 1), (0, 64, 1)), (9000, 200, 300, 256, (0, 64, 1), (0, 64, 1)),
    (9000, 33, 1104, 400, (1, 128, 1), (1, 128, 1)), (9001, 65, 1101, 400, (0, 128, 1), (1, 128, 1)), (6500, 70, 900, 1040, (1, 128, 1), (0, 128, 1)),
]


@pytest.mark.parametrize("clusters", [(74, 35, 16), (60, 28, 12), (74, 37, 18)])
def test_plans_of_the_computed_forms(clusters):
    for m, n, k, f32, f16 in FORMS:
        for dtype, want in ((F32, f32), (F16, f16), (BF16, f16)):
            aligned = n * (4 if dtype == F32 else 2) % 16 == 0
            assert matmul_plan(m, n, k, dtype=dtype, aligned=aligned, clusters=clusters) == want, (m, n, k, dtype)
    for rows, experts, n, k, f32, f16 in GROUP_FORMS:
        for dtype, want in ((F32, f32), (F16, f16), (BF16, f16)):
            aligned = n * (4 if dtype == F32 else 2) % 16 == 0
            assert matmul_plan(rows, n, k, experts, dtype, aligned, clusters=clusters) == want, (rows, experts, n, k, dtype)
    plans = {p for form in FORMS for p in form[3:]}
    assert plans == {(2, 256, 1), (1, 128, 1), *((0, t, s) for t in (16, 32, 64, 128) for s in (1, 2, 4, 8))} - {(0, 128, 8)}

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

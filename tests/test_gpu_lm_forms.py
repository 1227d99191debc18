"""The language-model operators in every form of their kernels: sizes that the plans send to wide
tiles and pairs, split tiles, several tiles per CTA, many experts and streaming accesses, against
their definitions in 64 bits (bounds as in test_gpu_lm.py)."""
import pytest

from pdefa_b200 import _native as N
from test_gpu_lm import DTYPES, check_product, gen, ids, operands

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


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

"""Argument checks of the language-model operators' C entry points that come before any
device is touched, and what the Python functions refuse without a GPU."""
import ctypes as C

import pytest

import pdefa_b200 as pb
from pdefa_b200 import _native as N

NULL, SHAPE, ARG = 1, 6, 7          # ENGINE_ERR_NULL_PTR, _INVALID_SHAPE, _INVALID_ARG


@pytest.fixture(scope="module")
def buf():
    """An address that is never dereferenced: the checks come first."""
    b = C.create_string_buffer(256)
    a = C.addressof(b)
    yield a + (-a) % 16
    del b


def norm(buf, **kw):
    d = dict(x=buf, xs=64, r=None, rs=0, w=buf, h=None, hs=0, y=buf, ys=64, s=None, ss=0, rows=2, cols=64, dtype=2, wd=2,
             eps=1e-6, dev=0, stream=None)
    d.update(kw)
    return N.lib().engine_rms_norm_device(*d.values())


def matmul(buf, **kw):
    d = dict(a=buf, lda=64, sa=buf, ldsa=1, b=buf, ldb=64, sb=buf, ldsb=1, out=buf, ldo=32, od=2, m=4, n=32, k=64, dev=0,
             stream=None)
    d.update(kw)
    return N.lib().engine_matmul_fp8_device(*d.values())


def grouped(buf, **kw):
    d = dict(a=buf, lda=64, sa=buf, ldsa=1, b=buf, ldb=64, be=2048, sb=buf, ldsb=1, sbe=1, off=buf, experts=2, out=buf,
             ldo=32, od=2, rows=4, n=32, k=64, dev=0, stream=None)
    d.update(kw)
    return N.lib().engine_matmul_grouped_fp8_device(*d.values())


def sample(buf, **kw):
    d = dict(x=buf, xs=100, dt=2, e=buf, es=100, t=None, k=None, p=None, m=None, rows=2, vocab=100, tok=buf, prob=None,
             dev=0, stream=None)
    d.update(kw)
    return N.lib().engine_sample_device(*d.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(x=None), NULL), (dict(w=None), NULL), (dict(y=None), NULL), (dict(rows=-1), SHAPE), (dict(cols=-1), SHAPE),
    (dict(rows=1 << 31), SHAPE), (dict(dtype=3), ARG), (dict(wd=1), ARG), (dict(eps=-1.0), ARG),
    (dict(eps=float("nan")), ARG), (dict(eps=float("inf")), ARG), (dict(xs=-64), ARG), (dict(ys=63), ARG),
    (dict(xs=1 << 61), ARG), (dict(r="buf", rs=-1), ARG), (dict(h="buf", hs=1), ARG), (dict(s="buf", ss=0), ARG),
    (dict(x="odd"), ARG), (dict(y="odd"), ARG), (dict(rows=0), 0), (dict(cols=0), 0),
])
def test_norm_checks(buf, kw, rc):
    kw = {k: buf if v == "buf" else buf + 1 if v == "odd" else v for k, v in kw.items()}
    assert norm(buf, **kw) == rc
    assert rc == 0 or N.lib().pdefa_last_error().startswith(b"rms_norm:")


@pytest.mark.parametrize("kw,rc", [
    (dict(a=None), NULL), (dict(sb=None), NULL), (dict(out=None), NULL), (dict(m=-1), SHAPE), (dict(k=1 << 31), SHAPE),
    (dict(od=5), ARG), (dict(lda=-1), ARG), (dict(ldb=-1), ARG), (dict(ldo=31), ARG), (dict(ldsa=-1), ARG),
    (dict(sa="odd"), ARG), (dict(out="odd"), ARG), (dict(m=0), 0), (dict(n=0), 0),
])
def test_matmul_checks(buf, kw, rc):
    kw = {k: buf + 1 if v == "odd" else v for k, v in kw.items()}
    assert matmul(buf, **kw) == rc
    assert rc == 0 or N.lib().pdefa_last_error().startswith(b"matmul_fp8:")
    if "lda" not in kw or kw["lda"] is None:
        kw = {("rows" if k == "m" else k): v for k, v in kw.items()}
        assert grouped(buf, **kw) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(off=None), NULL), (dict(experts=0), SHAPE), (dict(experts=65536), SHAPE), (dict(be=-1), ARG),
    (dict(sbe=-1), ARG), (dict(off="odd"), ARG), (dict(rows=0), 0),
])
def test_grouped_checks(buf, kw, rc):
    kw = {k: buf + 1 if v == "odd" else v for k, v in kw.items()}
    assert grouped(buf, **kw) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(x=None), NULL), (dict(e=None), NULL), (dict(tok=None), NULL), (dict(rows=-1), SHAPE), (dict(vocab=0), SHAPE),
    (dict(vocab=1 << 31), SHAPE), (dict(dt=4), ARG), (dict(xs=-1), ARG), (dict(es=-1), ARG), (dict(x="odd"), ARG),
    (dict(e="odd"), ARG), (dict(p="odd"), ARG), (dict(rows=0), 0),
])
def test_sample_checks(buf, kw, rc):
    kw = {k: buf + 1 if v == "odd" else v for k, v in kw.items()}
    assert sample(buf, **kw) == rc
    assert rc == 0 or N.lib().pdefa_last_error().startswith(b"sample:")


def test_calls_without_a_gpu_fail_loudly(buf):
    if pb.device_count() > 0:
        pytest.skip("a GPU is present")
    for call in (norm, matmul, grouped, sample):
        assert call(buf) != 0
        assert N.lib().pdefa_last_error()


def test_python_refuses_what_is_not_on_a_gpu():
    torch = pytest.importorskip("torch")
    x = torch.zeros(2, 8)
    for call in (lambda: pb.ops_rms_norm(x, x[0]), lambda: pb.ops_rms_norm_fp8(x, x[0]), lambda: pb.ops_sample(x, x),
                 lambda: pb.ops_matmul_fp8(x, x, x, x), lambda: pb.ops_matmul_grouped_fp8(x, x, x, x, x),
                 lambda: pb.ops_sample(None, None), lambda: pb.ops_rms_norm(pb.zeros(2, 8), pb.zeros(8))):
        with pytest.raises(TypeError):
            call()

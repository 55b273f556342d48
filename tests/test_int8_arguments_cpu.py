"""8-bit integer products: what is refused on the host, before anything is launched."""
from flashrt_b200 import _lib

A = 4096                                                   # stands for an aligned device pointer; never read


def quantize(**kw):
    a = dict(x=A, stride=256, out=A, scale=A, rows=4, dim=256, flags=0, stream=None)
    a.update(kw)
    return _lib.call_status("frt_b200_quantize_int8_rows", *a.values())


def product(**kw):
    a = dict(a=A, w=A, d=A, m=8, n=128, k=256, ts=A, cs=A, bias=None, flags=0, stream=None)
    a.update(kw)
    return _lib.call_status("frt_b200_gemm_int8_nt", *a.values())


def test_quantize():
    assert quantize(rows=0) == 0
    for kw in (dict(rows=-1), dict(dim=-16), dict(stride=240), dict(stride=260), dict(x=None), dict(out=None), dict(scale=None),
               dict(x=A + 8), dict(out=A + 8), dict(scale=A + 2)):
        assert quantize(**kw) == -1, kw
    assert quantize(dim=248) == -2


def test_product():
    assert product(m=0) == 0 and product(n=0) == 0
    for kw in (dict(m=-1), dict(n=-1), dict(k=0), dict(a=None), dict(w=None), dict(d=None), dict(ts=None), dict(cs=None), dict(a=A + 8),
               dict(w=A + 4), dict(d=A + 2), dict(ts=A + 1), dict(cs=A + 2), dict(bias=A + 1)):
        assert product(**kw) == -1, kw
    for k in (8, 120, 131072, 1 << 20):
        assert product(k=k) == -2, k

"""Paged cache entry points: what is refused on the host, before anything is launched."""
import ctypes

import pytest

from flashrt_b200 import _lib

A = 4096                                                   # stands for an aligned device pointer; never read


def append(**kw):
    a = dict(qkv=A, qkv_stride=6144, rope=A, rope_rows=8, q=A, k=A, v=A, ks=A, vs=A, table=A, table_stride=4, cu=A, lens=A, tokens=8,
             batch=2, num_blocks=8, block_size=16, hq=32, hkv=8, d=128, flags=0, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.call_status("frt_b200_paged_kv_append_fp8", *a.values())


def attend(**kw):
    a = dict(q=A, q_stride=4096, o=A, o_stride=4096, lse=A, k=A, v=A, ks=A, vs=A, table=A, table_stride=4, cu=A, lens=A, tokens=8, batch=2,
             max_new=4, num_blocks=8, block_size=16, hq=32, hkv=8, d=128, scale=0.1, cap=0.0, window=0, work=A, work_bytes=1 << 30, flags=0,
             stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.call_status("frt_b200_paged_attention_fp8", *a.values())


@pytest.mark.parametrize("call", [append, attend])
def test_shapes_and_pointers(call):
    assert call(tokens=0) == 0 and call(batch=0) == 0 and call(tokens=0, batch=0, cu=None) == 0
    for kw in (dict(d=96), dict(d=512), dict(block_size=8), dict(block_size=24), dict(block_size=256)):
        assert call(**kw) == -2, kw
    for kw in (dict(tokens=-1), dict(batch=-1), dict(num_blocks=-1), dict(table_stride=-1), dict(hq=0), dict(hkv=0)):
        assert call(**kw) == -1, kw
    assert call(cu=None, tokens=8, batch=7) == -1          # one token per sequence, but not as many
    for name in ("k", "v", "ks", "vs", "table", "lens"):
        assert call(**{name: None}) == -1, name
    for name, off in (("k", 8), ("v", 4), ("ks", 2), ("vs", 1), ("table", 2), ("cu", 3), ("lens", 1), ("q", 8)):
        assert call(**{name: A + off}) == -1, name


def test_append():
    assert append(hq=2048) == -2
    assert append(qkv=None) == -1 and append(qkv=A + 2) == -1 and append(rope=A + 8) == -1
    assert append(qkv_stride=6143) == -1 and append(qkv_stride=6148) == -1 and append(rope_rows=-1) == -1


def test_attention():
    assert attend(hq=30) == -2                             # 30 query heads on 8
    assert attend(hq=2048, q_stride=2048 * 128, o_stride=2048 * 128) == -2
    assert attend(q=None) == -1 and attend(o=None) == -1 and attend(work=None) == -1 and attend(o=A + 2) == -1
    assert attend(q_stride=4095) == -1 and attend(o_stride=4100) == -1 and attend(q_stride=4000) == -1
    assert attend(window=-1) == -1 and attend(window=4, flags=2) == -2 and attend(max_new=-1) == -1
    for bad in (-1.0, float("nan"), float("inf")):
        assert attend(cap=bad) == -1
    assert attend(scale=float("nan")) == -1 and attend(scale=float("inf")) == -1
    assert attend(work=A + 8) == -1


def test_workspace():
    n = ctypes.c_longlong(0)
    size = lambda *a: (_lib.call_status("frt_b200_paged_attention_workspace_bytes", *a, ctypes.addressof(n)), n.value)  # noqa: E731
    for d in (64, 128, 256):
        rc, few = size(4, 4, 1, 32, 8, d)
        assert rc == 0 and few > 0 and few % 16 == 0
        rc, more = size(64, 4, 16, 32, 8, d)
        assert rc == 0 and more >= few
        at_most = size(8192, 16, 8192, 32, 8, d)[1]            # one for the largest figures serves all smaller ones
        assert all(size(b * n, b, n, 32, 8, d)[1] <= at_most for b in (1, 4, 16) for n in (1, 2, 4, 5, 6, 30, 200, 8192 // b))
    assert size(4, 4, 1, 32, 8, 96)[0] == -2 and size(4, 4, 1, 30, 8, 128)[0] == -2 and size(-1, 4, 1, 32, 8, 128)[0] == -1
    assert _lib.call_status("frt_b200_paged_attention_workspace_bytes", 4, 4, 1, 32, 8, 128, None) == -1

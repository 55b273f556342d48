"""Block-scaled products, probabilities, drafted tokens and blocks of the paged cache: what is refused on the host, before anything is
launched; and the plain statements that the GPU tests compare with."""
import numpy as np
import pytest
import torch

import decode_ref as R
from flashrt_b200 import _lib

A = 4096                                                   # stands for an aligned device pointer; never read


def status(name, base, kw):
    a = dict(base)
    a.update(kw)
    return _lib.call_status(name, *a.values())


def quantize(**kw):
    return status("frt_b200_quantize_fp8_groups", dict(x=A, stride=256, out=A, scale=A, sstride=4, rows=4, dim=256, flags=0, stream=None), kw)


def product(**kw):
    return status("frt_b200_gemm_fp8_block_nt", dict(a=A, w=A, d=A, m=8, n=128, k=256, asc=A, sstride=8, wsc=A, bias=None, flags=0, stream=None), kw)


def softmax(**kw):
    return status("frt_b200_softmax_rows", dict(x=A, istride=100, out=A + 64, ostride=100, t=None, rows=4, vocab=100, flags=0, stream=None), kw)


def verify(**kw):
    return status("frt_b200_verify_drafts", dict(p=A, ps=100, q=A, qs=100, tok=A, cu=A, lens=A, u=A, v=A, out=A + 64, acc=A, kept=A, n=6, batch=2,
                                                 vocab=100, flags=0, stream=None), kw)


def plan(**kw):
    return status("frt_b200_paged_plan", dict(kept=A, new=A, table=A, stride=8, free=A, fin=A, fout=A + 4, cu=A, lens=A + 64, pos=A, slots=A, ref=A,
                                              tokens=6, batch=2, pool=16, bs=16, flags=0, stream=None), kw)


def release(**kw):
    return status("frt_b200_paged_release", dict(kept=A, lens=A, table=A, stride=8, free=A, fin=A, fout=A + 4, batch=2, pool=16, bs=16, flags=0,
                                                 stream=None), kw)


def test_quantize():
    assert quantize(rows=0) == 0 and quantize(dim=0) == 0
    for kw in (dict(rows=-1), dict(dim=-16), dict(stride=240), dict(stride=260), dict(sstride=3), dict(x=None), dict(out=None), dict(scale=None),
               dict(x=A + 8), dict(out=A + 8), dict(scale=A + 2)):
        assert quantize(**kw) == -1, kw
    assert quantize(dim=248) == -2 and quantize(rows=1 << 30, sstride=1 << 30) == -2


def test_product():
    assert product(m=0) == 0 and product(n=0) == 0
    for kw in (dict(m=-1), dict(n=-1), dict(k=0), dict(sstride=7), dict(a=None), dict(w=None), dict(d=None), dict(asc=None), dict(wsc=None),
               dict(a=A + 8), dict(w=A + 4), dict(d=A + 2), dict(asc=A + 1), dict(wsc=A + 2), dict(bias=A + 1)):
        assert product(**kw) == -1, kw
    for kw in (dict(k=8), dict(k=120), dict(k=(1 << 20) + 16), dict(n=(1 << 30) + 1)):
        assert product(**kw) == -2, kw


def test_softmax():
    assert softmax(rows=0) == 0 and softmax(vocab=0) == 0
    for kw in (dict(rows=-1), dict(vocab=-1), dict(istride=99), dict(ostride=99), dict(x=None), dict(out=None), dict(x=A + 1), dict(x=A + 2, flags=2),
               dict(out=A + 2), dict(out=A), dict(t=A + 2)):
        assert softmax(**kw) == -1, kw
    assert softmax(vocab=(1 << 30) + 1, istride=1 << 31, ostride=1 << 31) == -2 and softmax(rows=(1 << 27) + 1) == -2


def test_verify():
    assert verify(batch=0) == 0
    for kw in (dict(n=-1), dict(batch=-1), dict(vocab=0), dict(ps=99), dict(qs=99), dict(p=None), dict(tok=None), dict(cu=None), dict(lens=None),
               dict(u=None), dict(v=None), dict(out=None), dict(acc=None), dict(out=A), dict(p=A + 2), dict(q=A + 1), dict(tok=A + 2), dict(cu=A + 2),
               dict(lens=A + 1), dict(u=A + 2), dict(v=A + 2), dict(out=A + 66), dict(acc=A + 2), dict(kept=A + 2)):
        assert verify(**kw) == -1, kw
    assert verify(batch=(1 << 27) + 1) == -2


def test_plan_and_release():
    for kw in (dict(batch=-1), dict(pool=-1), dict(stride=-1), dict(kept=None), dict(fin=None), dict(fout=None), dict(lens=None), dict(table=None),
               dict(free=None), dict(fout=A), dict(kept=A + 2), dict(table=A + 2), dict(free=A + 2), dict(fin=A + 1), dict(fout=A + 6)):
        assert plan(**kw) == -1 and release(**kw) == -1, kw
    for kw in (dict(tokens=-1), dict(new=None), dict(cu=None), dict(lens=A), dict(pos=A + 2), dict(slots=A + 4), dict(ref=A + 2), dict(cu=A + 2),
               dict(new=A + 2), dict(lens=A + 66)):
        assert plan(**kw) == -1, kw
    for kw in (dict(bs=8), dict(bs=48), dict(bs=256), dict(batch=8193), dict(batch=8192, stride=1 << 18), dict(pool=(1 << 30) + 1)):
        assert plan(**kw) == -2 and release(**kw) == -2, kw
    assert plan(tokens=(1 << 30) + 1) == -2


# ------------------------------------------------------------------ the statements themselves
def test_codes_of_the_statement_are_the_type_s():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    every = every[every.isfinite()]
    assert torch.equal(R.e4m3(every), every)
    grid = every.unique()
    middle = (grid[1:] + grid[:-1]) / 2
    assert torch.equal(R.e4m3(middle), middle.float().to(torch.float8_e4m3fn).double())
    x = torch.randn(4096, generator=torch.Generator().manual_seed(0)).double() * 100
    assert torch.equal(R.e4m3(x.float().double()), x.float().clamp(-448, 448).to(torch.float8_e4m3fn).double())


def test_verification_keeps_the_target_s_distribution():
    """One drafted token from q: what stands or takes its place is distributed as p.  20000 draws, expected counts to five sigma."""
    rng = np.random.default_rng(0)
    p, q = (rng.dirichlet(np.ones(6)).astype(np.float32) for _ in range(2))
    n = 20000
    drafted = rng.choice(6, size=n, p=q.astype(np.float64) / q.astype(np.float64).sum())
    hits = np.zeros(6)
    rows, qrows = np.stack([p, p]), np.stack([q, q])
    for d in drafted:
        out, acc, kept = R.verify(rows, qrows, [0, int(d)], [0, 2], [7], rng.random(2, dtype=np.float32), rng.random(1, dtype=np.float32))
        hits[out[0]] += 1
        assert kept[0] == 6 + acc[0]
    want = p.astype(np.float64) / p.astype(np.float64).sum() * n
    assert (np.abs(hits - want) <= 5 * np.sqrt(want)).all(), (hits, want)


@pytest.mark.parametrize("bs", [16, 64])
def test_release_and_plan_are_inverse(bs):
    rng = np.random.default_rng(bs)
    kept = rng.integers(0, 300, 9).tolist()
    new = rng.integers(0, 200, 9).tolist()
    table = [[-1] * 40 for _ in kept]
    free = rng.permutation(400).tolist()
    count, _, lens, *_ = R.plan([0] * 9, kept, table, free, 400, 400, bs, 10 ** 4)
    held = [row[:] for row in table]
    after, cu, lens, pos, slot, refused = R.plan(kept, new, table, free, count, 400, bs, 10 ** 4)
    assert refused == 0 and cu[-1] == sum(new) and len({s for s in slot if s >= 0}) == sum(new)
    assert R.release(kept, lens, table, free, after, 400, bs) == count and table == held

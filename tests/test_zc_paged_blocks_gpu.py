"""Blocks of the paged cache between two steps, against plain lists."""
import numpy as np
import pytest
import torch

import decode_ref as R

pytestmark = pytest.mark.gpu
I32, I64 = torch.int32, torch.int64


def _stream():
    return torch.cuda.current_stream().cuda_stream


def dev(x, t=I32):
    return torch.tensor(np.asarray(x), dtype=t, device="cuda")


def run_plan(kept, new, table, free, count, pool, bs, tokens, slots=True):
    from flashrt_b200 import flash_rt_kernels as fvk
    batch, stride = len(kept), len(table[0]) if table else 0
    d = [dev(kept), dev(new), dev(table).view(batch, stride), dev(free), dev([count, -9])]
    cu, lens, pos, ref = (torch.full((k,), -55, dtype=I32, device="cuda") for k in (batch + 2, batch + 1, tokens + 1, 2))
    slot = torch.full((tokens + 1,), -55, dtype=I64, device="cuda")
    fvk.paged_plan(d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), stride, d[3].data_ptr(), d[4].data_ptr(), d[4].data_ptr() + 4, cu.data_ptr(),
                   lens.data_ptr(), pos.data_ptr() if slots else 0, slot.data_ptr() if slots else 0, ref.data_ptr() if slots else 0, tokens, batch, pool,
                   bs, _stream())
    torch.cuda.synchronize()
    assert cu[-1] == -55 and lens[-1] == -55 and pos[-1] == -55 and slot[-1] == -55 and ref[1] == -55
    assert d[0].tolist() == list(kept) and d[1].tolist() == list(new) and d[3].tolist() == list(free) and d[4][0] == count
    return d[2].tolist(), (int(d[4][1]), cu[:-1].tolist(), lens[:-1].tolist(), pos[:-1].tolist(), slot[:-1].tolist(), int(ref[0]))


def check_plan(kept, new, table, free, count, pool, bs, tokens):
    got_table, got = run_plan(kept, new, table, free, count, pool, bs, tokens)
    want_table = [row[:] for row in table]
    want = R.plan(kept, new, want_table, free, count, pool, bs, tokens)
    for a, b in zip(got, want):
        assert a == b
    assert got_table == want_table
    same, less = run_plan(kept, new, table, free, count, pool, bs, tokens, slots=False)
    assert same == want_table and less[:3] == want[:3]
    return got_table, got


def check_release(kept, lens, table, free, count, pool, bs):
    from flashrt_b200 import flash_rt_kernels as fvk
    batch, stride = len(kept), len(table[0]) if table else 0
    d = [dev(kept), dev(lens), dev(table).view(batch, stride), dev(free), dev([count, -9])]
    fvk.paged_release(d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), stride, d[3].data_ptr(), d[4].data_ptr(), d[4].data_ptr() + 4, batch, pool, bs,
                      _stream())
    torch.cuda.synchronize()
    want_table, want_free = [row[:] for row in table], list(free)
    want = R.release(kept, lens, want_table, want_free, count, pool, bs)
    assert d[2].tolist() == want_table and d[3].tolist() == want_free and d[4].tolist() == [count, want]
    return want_table, want_free, want


def state(rng, batch, longest, most_new, bs, spare):
    kept = rng.integers(0, longest + 1, batch).tolist()
    new = rng.integers(0, most_new + 1, batch).tolist()
    held = [R.blocks_of(k, bs) for k in kept]
    stride = max(R.blocks_of(k + n, bs) for k, n in zip(kept, new)) + 2
    need = sum(R.blocks_of(k + n, bs) for k, n in zip(kept, new))
    pool = need + spare
    ids = rng.permutation(pool).tolist()
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-1] * (stride - h))
        at += h
    free = ids[at:] + [-1] * at
    return kept, new, table, free, pool - at, pool


@pytest.mark.parametrize("batch,longest,most_new,bs", [(1, 0, 1, 16), (1, 900, 5, 16), (2, 15, 1, 16), (7, 100, 40, 32), (64, 500, 6, 128), (255, 40, 3, 16),
                                                       (256, 300, 2, 32), (257, 64, 64, 64), (1000, 100, 8, 16), (8192, 60, 2, 32), (3, 9000, 5000, 16),
                                                       (20, 30000, 3000, 64)])
def test_plan_then_release(batch, longest, most_new, bs):
    rng = np.random.default_rng(batch + longest)
    kept, new, table, free, count, pool = state(rng, batch, longest, most_new, bs, 7)
    filled, (after, cu, lens, *_) = check_plan(kept, new, table, free, count, pool, bs, sum(new) + 5)
    assert lens == [k + n for k, n in zip(kept, new)]
    # some drafts do not stand, some sequences end
    stay = [max(0, n - int(rng.integers(0, 9))) if i % 6 else 0 for i, n in enumerate(lens)]
    t2, f2, c2 = check_release(stay, lens, filled, free, after, pool, bs)
    assert c2 + sum(R.blocks_of(s, bs) for s in stay) == pool
    # and the same number again finds them in their places
    t3, (c3, *_) = check_plan(stay, [n - s for n, s in zip(lens, stay)], t2, f2, c2, pool, bs, 1 << 20 if sum(lens) < 1 << 20 else sum(lens))
    assert t3 == filled and c3 == after


def test_shortage_and_refusals():
    rng = np.random.default_rng(5)
    kept, new, table, free, count, pool = state(rng, 40, 200, 60, 16, 0)
    for lack in (1, 5, 30, count):
        check_plan(kept, new, table, free, count - lack, pool, 16, 5000)
    for tokens in (0, 1, 17, sum(new) - 1, sum(new)):
        check_plan(kept, new, table, free, count, pool, 16, tokens)
    for bad in (-1, -2 ** 31, 2 ** 31 - 1):
        k, n = kept[:], new[:]
        k[3], n[9] = bad, bad
        _, got = check_plan(k, n, table, free, count, pool, 16, 5000)
        assert got[5] >= 2
    k = kept[:]
    k[0] = len(table[0]) * 16                                        # a full row: nothing more fits
    new[0] = 1
    _, got = check_plan(k, new, table, free, count, pool, 16, 5000)
    assert got[5] == 1 and got[1][1] == 0
    for count in (-5, pool + 100):                                   # a count outside the pool is taken into it
        check_plan(kept, new, table, free[:pool], count, pool, 16, 5000)
    check_plan([0, 3], [5, 0], [[-1, 4], [2, -1]], [-7, 99, 1], 2, 3, 16, 9)       # a list with entries that are no blocks: no slots


def test_empty_ones():
    check_plan([], [], [], [4, 5, 6], 3, 3, 16, 4)
    check_plan([0, 0], [0, 0], [[-1], [-1]], [0], 1, 1, 16, 0)
    check_plan([5, 0], [0, 0], [[0], [-1]], [0, 0], 0, 2, 16, 3)
    check_release([], [], [], [4], 0, 1, 16)
    check_release([3], [3], [[0]], [0], 0, 1, 16)


def test_release_holes_and_long_rows():
    rng = np.random.default_rng(9)
    for batch, stride, bs in ((3, 50, 16), (40, 60, 32), (30, 900, 16), (3, 30000, 128)):
        pool = batch * stride
        table = rng.permutation(pool).reshape(batch, stride)
        table[rng.random(table.shape) < 0.2] = -1                    # pages that are absent, or are no block of the pool
        table[rng.random(table.shape) < 0.1] = pool + 3
        lens = rng.integers(0, stride * bs + 100, batch)
        kept = np.minimum(lens, rng.integers(-20, stride * bs, batch))
        kept[0], lens[0] = 0, stride * bs + 999
        check_release(kept.tolist(), lens.tolist(), table.tolist(), [-1] * pool, 0, pool, bs)
        check_release(lens.tolist(), kept.tolist(), table.tolist(), [-1] * pool, 0, pool, bs)        # nothing to drop
    check_release([0], [64], [[1, 2, 0, 3]], [9, 9, 9, 9], 2, 4, 16)          # a list that would run over its end stops there


def test_a_captured_step_serves_other_lengths():
    from flashrt_b200 import flash_rt_kernels as fvk
    rng = np.random.default_rng(3)
    batch, bs, tokens = 33, 16, 400
    kept, new, table, free, count, pool = state(rng, batch, 300, 8, bs, 40)
    table = [row + [-1] * 8 for row in table]
    d = {k: dev(x) for k, x in dict(kept=kept, new=new, table=table, free=free, a=[count], b=[0]).items()}
    cu, lens, pos, ref = (torch.zeros(k, dtype=I32, device="cuda") for k in (batch + 1, batch, tokens, 1))
    lens.copy_(d["kept"])
    slot = torch.zeros(tokens, dtype=I64, device="cuda")
    stride = len(table[0])

    def step():
        fvk.paged_release(d["kept"].data_ptr(), lens.data_ptr(), d["table"].data_ptr(), stride, d["free"].data_ptr(), d["a"].data_ptr(), d["b"].data_ptr(),
                          batch, pool, bs, _stream())
        fvk.paged_plan(d["kept"].data_ptr(), d["new"].data_ptr(), d["table"].data_ptr(), stride, d["free"].data_ptr(), d["b"].data_ptr(),
                       d["a"].data_ptr(), cu.data_ptr(), lens.data_ptr(), pos.data_ptr(), slot.data_ptr(), ref.data_ptr(), tokens, batch, pool, bs,
                       _stream())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    hlens = kept[:]
    for i in range(6):
        graph.replay()
        torch.cuda.synchronize()
        mid = R.release(kept, hlens, table, free, count, pool, bs)
        count, wcu, hlens, wpos, wslot, wref = R.plan(kept, new, table, free, mid, pool, bs, tokens)
        assert cu.tolist() == wcu and lens.tolist() == hlens and pos.tolist() == wpos and slot.tolist() == wslot and int(ref) == wref
        assert d["table"].tolist() == table and d["free"].tolist() == free and int(d["a"]) == count and int(d["b"]) == mid
        kept = [max(0, n - int(rng.integers(0, 8))) if rng.random() > 0.1 else 0 for n in hlens]
        new = rng.integers(0, 12, batch).tolist()
        d["kept"].copy_(dev(kept))
        d["new"].copy_(dev(new))

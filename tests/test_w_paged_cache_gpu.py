"""Paged E4M3 cache: append and attention against 64-bit formulas (tests/paged_ref.py)."""
import math

import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
GUARD = 0x5A


def _stream():
    return torch.cuda.current_stream().cuda_stream


class Pool:
    """Caches and scales on the device, filled as an earlier call would have left them."""

    def __init__(self, num_blocks, hkv, block, d, seed, fill=True):
        g = torch.Generator().manual_seed(seed)
        shape = (num_blocks, hkv, block, d)
        self.block, self.num_blocks = block, num_blocks
        self.c, self.s = {}, {}
        for n in "kv":
            s = 0.004 + 0.008 * torch.rand(num_blocks, hkv, generator=g)
            x = (torch.randn(shape, generator=g) / s[:, :, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
            self.c[n] = (x if fill else torch.full(shape, GUARD, dtype=torch.uint8)).cuda()
            self.s[n] = s.cuda()

    def host(self):
        torch.cuda.synchronize()
        return {n: t.cpu() for n, t in self.c.items()}, {n: t.cpu() for n, t in self.s.items()}


def append(pool, qkv, rope, table, cu, lens, hq, hkv, d, halves=False, q=True, tokens=None, stride=0):
    from flashrt_b200 import flash_rt_kernels as fvk
    tokens = qkv.shape[0] if tokens is None else tokens
    out = torch.full((tokens, hq * d), -7.0, dtype=BF16, device="cuda") if q else None
    fvk.paged_kv_append_fp8(qkv.data_ptr(), rope.data_ptr() if rope is not None else 0, out.data_ptr() if q else 0, pool.c["k"].data_ptr(),
                            pool.c["v"].data_ptr(), pool.s["k"].data_ptr(), pool.s["v"].data_ptr(), table.data_ptr(), table.shape[1],
                            cu.data_ptr() if cu is not None else 0, lens.data_ptr(), tokens, len(lens), pool.num_blocks, pool.block, hq,
                            hkv, d, rope.shape[0] if rope is not None else 0, _stream(), halves=halves, qkv_stride=stride)
    return out


def check_append(pool, before, qkv, rope, table, cu, lens, hq, hkv, d, halves, out):
    """Scales to the rounding of their two operations and of the rotation (4 x 2^-24); codes within half a step of the value over the
    scale (2^-4 of it, at least 2^-10 of a unit), with room for a value that the fp32 rotation moved across the middle of two
    codes; everything that no new token touches as it was."""
    c0, s0 = before
    c1, s1 = pool.host()
    rot = lambda x, p: R.rotate(x, rope[p], halves) if rope is not None else x  # noqa: E731
    touched = torch.zeros(pool.num_blocks, pool.block, dtype=torch.bool)
    for b, n_all in enumerate(lens):
        new = cu[b + 1] - cu[b]
        first = max(0, n_all - new)
        x = qkv[cu[b + 1] - (n_all - first):cu[b + 1]].to(F64).view(-1, hq + 2 * hkv, d)
        pos = torch.arange(first, n_all)
        if rope is not None:
            x, pos = x[pos < len(rope)], pos[pos < len(rope)]
        if not len(pos):
            continue
        t0 = cu[b + 1] - (n_all - first)
        if out is not None:
            want = rot(x[:, :hq], pos)
            got = out[t0:t0 + len(pos)].cpu().to(F64).view(-1, hq, d)
            # a rotation is exact to 2^-22 of |a| + |b|, then half a bf16 step
            pair = R.rotate(x[:, :hq].abs(), torch.ones(len(pos), d), halves).abs() + x[:, :hq].abs()
            assert ((got - want).abs() <= want.abs() * 2.0 ** -8 + pair * 2.0 ** -21).all()
        for n, y in (("k", rot(x[:, hq:hq + hkv], pos)), ("v", x[:, hq + hkv:])):
            for j in range(int(pos[0]) // pool.block, int(pos[-1]) // pool.block + 1):
                page = int(table[b, j])
                if not 0 <= page < pool.num_blocks:
                    continue
                sel = (pos // pool.block) == j
                slot = pos[sel] % pool.block
                held = int(slot[0])
                touched[page, slot] = True
                touched[page, :held] = True
                old = s0[n][page].to(F64) if held else torch.zeros(hkv, dtype=F64)
                now = torch.maximum(old, y[sel].abs().amax((0, 2)) / 448).clamp_min(1e-12)
                got_s = s1[n][page].to(F64)
                assert ((got_s - now).abs() <= now * 2.0 ** -20).all()
                code = R.codes(c1[n][page, :, slot])
                want = y[sel].transpose(0, 1) / now[:, None, None]
                assert ((code - want).abs() <= (want.abs() * 2.0 ** -4 * (1 + 2.0 ** -12)).clamp_min(2.0 ** -10 * (1 + 2.0 ** -12)) + 2.0 ** -12).all()
                if n == "v":                               # no rotation: the fp32 sequence, code for code
                    inv = (1.0 / s1[n][page])[:, None, None]
                    same = (y[sel].transpose(0, 1).to(F32) * inv).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
                    assert torch.equal(same, c1[n][page, :, slot])
                if held:
                    was = c0[n][page, :, :held]
                    grown = (got_s != old)
                    ratio = (s0[n][page] / s1[n][page])[:, None, None]
                    back = (was.view(torch.float8_e4m3fn).to(F32) * ratio).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
                    assert torch.equal(torch.where(grown[:, None, None], back, was), c1[n][page, :, :held])
    for n in "kv":
        free = ~touched[:, None, :].expand(-1, hkv, -1)
        assert torch.equal(c1[n][free], c0[n][free])
        rest = ~touched.any(1)
        assert torch.equal(s1[n][rest], s0[n][rest])


def _run_append(hq, hkv, d, block, new, ctx, halves=False, rope=True, seed=0, null_cu=False, tail=0, strong=1.0):
    g = torch.Generator().manual_seed(seed)
    pool = Pool(sum((c + block - 1) // block for c in ctx) + 3, hkv, block, d, seed)
    table = R.pages(ctx, block, pool.num_blocks, seed)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    qkv = (torch.randn(cu[-1] + tail, (hq + 2 * hkv) * d, generator=g) * strong).to(BF16)
    tab = R.rope_table(max(ctx) + 1, d) if rope else None
    before = pool.host()
    dev = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    out = append(pool, qkv.cuda(), tab.cuda() if rope else None, table.cuda(), None if null_cu else dev(cu), dev(ctx), hq, hkv, d, halves)
    check_append(pool, before, qkv, tab, table, cu, ctx, hq, hkv, d, halves, out)
    assert (out[cu[-1]:] == -7.0).all()
    return pool


HEADS = [(8, 1), (32, 8), (4, 4), (12, 2), (28, 4), (16, 1)]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_append_ragged(d, halves, block):
    hq, hkv = HEADS[(d // 64 + block) % len(HEADS)]
    _run_append(hq, hkv, d, block, [1, 37, 130, 2, 16], [1, 40, 259, 129, 16], halves, seed=d + block)


@pytest.mark.parametrize("hq,hkv", HEADS)
def test_append_one_token_each(hq, hkv):
    ctx = [1, 2, 16, 17, 31, 32, 33, 47, 48, 100]
    _run_append(hq, hkv, 128, 16, [1] * len(ctx), ctx, True, seed=hq, null_cu=True)
    _run_append(hq, hkv, 256, 32, [1] * len(ctx), ctx, False, seed=hq)


def test_append_scale_grows_and_shrinks_not():
    for strong in (0.01, 1.0, 40.0):
        _run_append(8, 2, 128, 32, [1, 5, 33], [20, 37, 90], seed=3, strong=strong)


def test_append_without_rotation_and_rows_behind():
    _run_append(8, 2, 64, 16, [3, 0, 7], [9, 4, 7], rope=False, seed=5, tail=6)


def test_append_many_sequences():
    new = [(7 * i) % 4 for i in range(300)]
    _run_append(4, 1, 64, 16, new, [n + (5 * i) % 23 for i, n in enumerate(new)], True, seed=8)


def test_append_long_prompt():
    _run_append(8, 2, 128, 64, [1500], [1531], True, seed=9)


def test_append_twice_is_the_same():
    """The second call finds its own scale and codes."""
    hq, hkv, d, block = 8, 2, 128, 32
    pool = Pool(8, hkv, block, d, 11)
    table, lens, cu = R.pages([70, 33], block, 8, 2), [70, 33], [0, 9, 12]
    qkv = torch.randn(12, (hq + 2 * hkv) * d, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    rope = R.rope_table(80, d).cuda()
    dev = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    a = append(pool, qkv, rope, table.cuda(), dev(cu), dev(lens), hq, hkv, d)
    one = pool.host()
    b = append(pool, qkv, rope, table.cuda(), dev(cu), dev(lens), hq, hkv, d)
    two = pool.host()
    assert torch.equal(a, b) and all(torch.equal(one[i][n], two[i][n]) for i in (0, 1) for n in "kv")


def test_append_what_is_left_out():
    """Idle slots, positions before the first, pages that are none, positions without a rotation row, a table that is too short."""
    hq, hkv, d, block = 4, 2, 64, 16
    dev = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    rope = R.rope_table(40, d)
    lens = [0, 3, 20, 33, 44, -5]
    new = [1, 5, 4, 2, 8, 1]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    table = torch.tensor([[0, -1, -1], [1, -1, -1], [2, -1, -1], [3, 4, 99], [5, 6, 7], [8, 9, 10]], dtype=torch.int32)
    pool = Pool(12, hkv, block, d, 4)
    qkv = torch.randn(cu[-1], (hq + 2 * hkv) * d, generator=torch.Generator().manual_seed(2)).to(BF16)
    before = pool.host()
    out = append(pool, qkv.cuda(), rope.cuda(), table.cuda(), dev(cu), dev(lens), hq, hkv, d)
    check_append(pool, before, qkv, rope, table, cu, [max(n, 0) for n in lens], hq, hkv, d, False, out)
    assert (out[0] == -7).all() and (out[1:3] == -7).all() and (out[3:6] != -7).any(1).all() and (out[-1] == -7).all()
    short = table[:, :1].contiguous()
    pool2 = Pool(12, hkv, block, d, 4)
    append(pool2, qkv.cuda(), rope.cuda(), short.cuda(), dev(cu), dev(lens), hq, hkv, d)
    check_append(pool2, before, qkv, rope, torch.cat([short, torch.full((6, 2), -1, dtype=torch.int32)], 1), cu, [max(n, 0) for n in lens],
                 hq, hkv, d, False, None)


def test_append_infinities_and_nan():
    hq, hkv, d, block = 2, 1, 64, 16
    x = torch.randn(3, (hq + 2 * hkv) * d, generator=torch.Generator().manual_seed(7)).to(BF16)
    x[1, 3 * d + 5], x[1, 3 * d + 6], x[2, 3 * d + 7] = math.inf, -math.inf, math.nan
    pool = Pool(2, hkv, block, d, 1)
    dev = lambda y: torch.tensor(y, dtype=torch.int32).cuda()  # noqa: E731
    append(pool, x.cuda(), None, dev([[1]]), dev([0, 3]), dev([3]), hq, hkv, d)
    c, s = pool.host()
    v = R.codes(c["v"][1, 0, :3])
    fine = x[:, 3 * d:].float()
    top = torch.where(fine.isfinite(), fine.abs(), 0.0).max() / 448
    assert s["v"][1, 0] == top and v[1, 5] == 448 and v[1, 6] == -448 and v[2, 7] == -448
    zero = torch.zeros_like(x)
    append(pool, zero.cuda(), None, dev([[1]]), dev([0, 3]), dev([3]), hq, hkv, d)
    c, s = pool.host()
    assert s["v"][1, 0] == torch.tensor(1e-12) and (R.codes(c["v"][1, 0, :3]) == 0).all()


def test_append_row_stride_and_no_queries():
    hq, hkv, d, block = 4, 2, 64, 16
    width = (hq + 2 * hkv) * d
    wide = torch.randn(5, width + 72, generator=torch.Generator().manual_seed(3)).to(BF16)
    table, dev = R.pages([21], block, 4, 0), lambda y: torch.tensor(y, dtype=torch.int32).cuda()  # noqa: E731
    rope = R.rope_table(32, d)
    pool = Pool(4, hkv, block, d, 6)
    before = pool.host()
    append(pool, wide.cuda(), rope.cuda(), table.cuda(), dev([0, 5]), dev([21]), hq, hkv, d, q=False, stride=width + 72)
    check_append(pool, before, wide[:, :width], rope, table, [0, 5], [21], hq, hkv, d, False, None)


# ------------------------------------------------------------------------------------------------ attention
def attend(pool, q, table, cu, lens, hq, hkv, d, cap=0.0, window=0, causal=True, work=None, max_new=None, lse=True, o=None, scale=None):
    from flashrt_b200 import flash_rt_fa2 as fa2
    tokens = q.shape[0]
    new = max((b - a for a, b in zip(cu, cu[1:])), default=0) if max_new is None else max_new
    n = fa2.paged_workspace_bytes(tokens, len(lens), new, hq, hkv, d)
    work = torch.zeros(n, dtype=torch.uint8, device="cuda") if work is None else work
    o = torch.full((tokens, hq * d), -7.0, dtype=BF16, device="cuda") if o is None else o
    ls = torch.full((hq, tokens), -7.0, device="cuda") if lse else None
    dev = lambda y: torch.tensor(y, dtype=torch.int32).cuda()  # noqa: E731
    one = new == 1 and cu[-1] == tokens == len(lens)
    cu_d, lens_d, table_d = dev(cu), dev(lens), table.cuda()
    fa2.paged_fwd_fp8(q.data_ptr(), o.data_ptr(), ls.data_ptr() if lse else 0, pool.c["k"].data_ptr(), pool.c["v"].data_ptr(),
                      pool.s["k"].data_ptr(), pool.s["v"].data_ptr(), table_d.data_ptr(), table.shape[1], 0 if one else cu_d.data_ptr(),
                      lens_d.data_ptr(), tokens, len(lens), new, pool.num_blocks, pool.block, hq, hkv, d, scale or d ** -0.5,
                      work.data_ptr(), n, _stream(), softcap=cap, window=window, causal=causal)
    torch.cuda.synchronize()
    assert (work[:4096] == 0).all()                        # the arrival counters are ready for the next launch
    return o, ls


def close(o, lse, want):
    """Output: half a bf16 step (2^-8); each weight rounded to fp16 (2^-11) and its logit off by the fp32 sum of d products
    (d x 2^-23 of sum |q||k|, at most 2^-12 here) and a few operations: 2^-10 of the weighted mean of |v| in all.  lse: the logit's
    error and its own fp32 operations."""
    ow, lw, size, reach = want
    o = o.cpu().to(F64).view(ow.shape)
    n = ow.shape[0]
    err = (o[:n] - ow).abs()
    bar = ow.abs() * 2.0 ** -8 + size * 2.0 ** -10 + 1e-30
    assert (err <= bar).all(), float((err / bar).max())
    if lse is not None:
        l = lse.cpu().to(F64)[:, :n]
        assert torch.equal(l.isinf(), lw.isinf())
        fin = lw.isfinite()
        e = (l - lw).abs()[fin]
        b = ((1 + lw.abs() + reach) * 2.0 ** -18)[fin]
        assert (e <= b).all(), float((e / b).max())


def _run_attend(hq, hkv, d, block, new, ctx, seed=0, tail=0, **kw):
    pool = Pool(sum((max(c, 0) + block - 1) // block for c in ctx) + 2, hkv, block, d, seed)
    table = R.pages(ctx, block, pool.num_blocks, seed)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1] + tail, hq * d, generator=torch.Generator().manual_seed(seed + 1)).to(BF16)
    c, s = pool.host()
    o, lse = attend(pool, q.cuda(), table, cu, ctx, hq, hkv, d, **{k: v for k, v in kw.items()})
    if tail:
        assert (o[cu[-1]:] == -7.0).all() and (lse[:, cu[-1]:] == -7.0).all()
    kw = {k: v for k, v in kw.items() if k in ("cap", "window", "causal")}
    want = R.attention(q.view(-1, hq, d)[:cu[-1]], c["k"], c["v"], s["k"], s["v"], table, cu, ctx, d ** -0.5, **kw)
    close(o[:cu[-1]], lse[:, :cu[-1]], want)
    return pool, table, cu, q, o, lse


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_attention_one_token(d, hq, hkv):
    ctx = [1, 15, 16, 17, 31, 33, 64, 65, 130, 200]
    _run_attend(hq, hkv, d, 16 if d == 64 else 32, [1] * len(ctx), ctx, seed=hq + d)


@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_attention_long_context_is_split(block):
    _run_attend(8, 1, 128, block, [1], [3001], seed=block)
    _run_attend(4, 2, 256, block, [1, 1], [1537, 700], seed=block + 1)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,ctx", [([5, 1, 3], [5, 300, 77]), ([2, 0, 17, 40], [130, 50, 17, 61])])
def test_attention_several_tokens(d, new, ctx):
    _run_attend(8, 2, d, 16, new, ctx, seed=d, tail=3)
    _run_attend(6, 2, d, 32, new, ctx, seed=d + 1)


@pytest.mark.parametrize("kw", [dict(window=1), dict(window=16), dict(window=50), dict(window=4000), dict(cap=5.0), dict(cap=30.0, window=33),
                                dict(causal=False), dict(causal=False, cap=2.0)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_masks_and_caps(kw, d):
    _run_attend(8, 2, d, 16, [1, 6, 33], [150, 90, 33], seed=d, **kw)


def test_attention_rows_without_keys():
    """Idle slots (length 0), more new tokens than positions: zeros, lse -inf."""
    _, _, _, _, o, lse = _run_attend(8, 2, 128, 16, [1, 1, 1], [0, 40, 0], seed=1)
    assert (o[0] == 0).all() and (o[2] == 0).all() and lse[:, 0].isneginf().all()
    _, _, _, _, o, lse = _run_attend(4, 2, 64, 16, [5, 3], [2, 3], seed=2)
    assert (o[:3] == 0).all() and lse[:, :3].isneginf().all() and lse[:, 3:].isfinite().all()
    _run_attend(4, 2, 64, 16, [5], [0], seed=3, causal=False)


def test_attention_absent_pages_and_what_lies_around():
    """Negative and too large entries are absent keys; bytes behind a sequence's end, in front of its window and in pages of other
    tokens may be anything (NaN codes, infinite scales)."""
    hq, hkv, d, block = 8, 2, 128, 16
    lens, cu = [60, 85], [0, 2, 3]
    pool = Pool(12, hkv, block, d, 5)
    table = torch.tensor([[0, -1, 1, 2, 7, 7], [3, 4, 12, 5, 2 ** 31 - 1, 6]], dtype=torch.int32)
    q = torch.randn(3, hq * d, generator=torch.Generator().manual_seed(1)).to(BF16)
    c, s = pool.host()
    want = R.attention(q.view(-1, hq, d), c["k"], c["v"], s["k"], s["v"], table, cu, lens, 0.1)
    for n in "kv":
        pool.c[n][2, :, 60 % block:] = 0x7F
        pool.c[n][6, :, 85 % block:] = 0xFF
        for page in (7, 8, 9, 10, 11):
            pool.c[n][page], pool.s[n][page] = 0x7F, math.inf
    close(*attend(pool, q.cuda(), table, cu, lens, hq, hkv, d, scale=0.1), want)
    # a window: pages in front of it may be gone or hold others' bytes
    table2 = torch.tensor([[7, 8, 1, 2, 9, 9], [7, 2 ** 31 - 1, -1, 8, 5, 6]], dtype=torch.int32)
    want = R.attention(q.view(-1, hq, d), c["k"], c["v"], s["k"], s["v"], table2, cu, lens, 0.1, window=20)
    for n in "kv":
        pool.c[n][1, :, :(58 - 20 + 1) % block] = 0x7F
        pool.c[n][5, :, :(84 - 20 + 1) % block] = 0xFF
    close(*attend(pool, q.cuda(), table2, cu, lens, hq, hkv, d, scale=0.1, window=20), want)


def test_attention_scales_far_apart():
    """Weights meet codes as 2^(logit + log2 scale): pages whose scales differ by 10^8 neither overflow nor lose the small ones."""
    hq, hkv, d, block = 4, 1, 64, 16
    lens, cu = [96], [0, 1]
    for which in "kv":
        pool = Pool(6, hkv, block, d, 9)
        pool.s[which][::2] *= 1e-4 if which == "k" else 1e-8
        if which == "v":
            pool.s["v"][1] *= 1e4
        table = R.pages(lens, block, 6, 3)
        q = torch.randn(1, hq * d, generator=torch.Generator().manual_seed(1)).to(BF16)
        c, s = pool.host()
        want = R.attention(q.view(-1, hq, d), c["k"], c["v"], s["k"], s["v"], table, cu, lens, d ** -0.5)
        close(*attend(pool, q.cuda(), table, cu, lens, hq, hkv, d), want)


@pytest.mark.parametrize("factor", [1e-20, 1e-3, 300.0])
def test_attention_large_and_small_queries(factor):
    hq, hkv, d, block = 4, 1, 128, 32
    lens, cu = [200], [0, 2]
    pool = Pool(7, hkv, block, d, 10)
    table = R.pages(lens, block, 7, 3)
    q = (torch.randn(2, hq * d, generator=torch.Generator().manual_seed(1)) * factor).to(BF16)
    c, s = pool.host()
    scale = d ** -0.5 if factor < 1 else d ** -0.5 / 300
    want = R.attention(q.view(-1, hq, d), c["k"], c["v"], s["k"], s["v"], table, cu, lens, scale)
    close(*attend(pool, q.cuda(), table, cu, lens, hq, hkv, d, scale=scale), want)


def test_attention_many_sequences_and_repeats():
    """More sequences than threads of a block; the same bits again from a used workspace, also after another shape used it."""
    n = 300
    ctx = [1 + (37 * i) % 90 for i in range(n)]
    pool, table, cu, q, o, lse = _run_attend(4, 2, 64, 16, [1] * n, ctx, seed=4)
    from flashrt_b200 import flash_rt_fa2 as fa2
    size = max(fa2.paged_workspace_bytes(n, n, 1, 4, 2, 64), fa2.paged_workspace_bytes(40, 1, 40, 4, 2, 64))
    work = torch.zeros(size, dtype=torch.uint8, device="cuda")
    for _ in range(2):
        again, l2 = attend(pool, q.cuda(), table, cu, ctx, 4, 2, 64, work=work)
        assert torch.equal(o, again) and torch.equal(lse, l2)
        attend(pool, torch.randn(40, 256, device="cuda").to(BF16), table[:1], [0, 40], [80], 4, 2, 64, work=work)


def test_attention_captured():
    """One captured launch serves other lengths, tables and queries; the graph's stream is not the current one."""
    from flashrt_b200 import flash_rt_fa2 as fa2, flash_rt_kernels as fvk
    hq, hkv, d, block, B = 8, 2, 128, 16, 3
    pool = Pool(40, hkv, block, d, 2)
    rope = R.rope_table(200, d).cuda()
    qkv = torch.zeros(B, (hq + 2 * hkv) * d, dtype=BF16, device="cuda")
    q, o = torch.zeros(B, hq * d, dtype=BF16, device="cuda"), torch.zeros(B, hq * d, dtype=BF16, device="cuda")
    table, lens = torch.full((B, 12), -1, dtype=torch.int32, device="cuda"), torch.ones(B, dtype=torch.int32, device="cuda")
    n = fa2.paged_workspace_bytes(B, B, 1, hq, hkv, d)
    work = torch.zeros(n, dtype=torch.uint8, device="cuda")

    def step(st):
        fvk.paged_kv_append_fp8(qkv.data_ptr(), rope.data_ptr(), q.data_ptr(), pool.c["k"].data_ptr(), pool.c["v"].data_ptr(),
                                pool.s["k"].data_ptr(), pool.s["v"].data_ptr(), table.data_ptr(), 12, 0, lens.data_ptr(), B, B, 40, block,
                                hq, hkv, d, 200, st)
        fa2.paged_fwd_fp8(q.data_ptr(), o.data_ptr(), 0, pool.c["k"].data_ptr(), pool.c["v"].data_ptr(), pool.s["k"].data_ptr(),
                          pool.s["v"].data_ptr(), table.data_ptr(), 12, 0, lens.data_ptr(), B, B, 1, 40, block, hq, hkv, d, d ** -0.5,
                          work.data_ptr(), n, st)

    graph = torch.cuda.CUDAGraph()
    step(_stream())
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(_stream())
    for i, ctx in enumerate(([5, 100, 33], [6, 0, 180])):
        table.copy_(R.pages(ctx, block, 40, i, width=12))
        lens.copy_(torch.tensor(ctx, dtype=torch.int32))
        qkv.copy_(torch.randn(qkv.shape, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        c, s = pool.host()
        want = R.attention(q.cpu().view(B, hq, d), c["k"], c["v"], s["k"], s["v"], table.cpu(), [0, 1, 2, 3], ctx, d ** -0.5)
        close(o, None, want)


# ---------------------------------------------------------------- chunks of prompts: the tensor-memory kernel
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_chunk_blocks(d, block):
    _run_attend(8, 2, d, block, [70, 33, 1], [390, 33, 200], seed=d + block)


@pytest.mark.parametrize("hq,hkv", [(3, 1), (5, 1), (7, 1), (16, 1), (4, 4), (12, 2)])
def test_chunk_groups(hq, hkv):
    """Groups that do not divide 128 rows: a token's heads lie in two tiles."""
    _run_attend(hq, hkv, 128, 32, [45, 100], [45, 350], seed=hq)


@pytest.mark.parametrize("kw", [dict(), dict(window=70), dict(window=1), dict(cap=0.3), dict(cap=20.0), dict(causal=False), dict(cap=0.3, window=130),
                                dict(causal=False, cap=20.0)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_chunk_masks(kw, d):
    _run_attend(4, 1, d, 32, [150, 65], [700, 65], seed=d + 3, tail=2, **kw)


def test_chunk_one_row_tile_and_key_splits():
    """One sequence of few rows and a long context: the keys are split over CTAs and the pieces joined."""
    for d, block in ((128, 64), (64, 16), (256, 128)):
        _run_attend(4, 1, d, block, [9], [2600], seed=d)
        _run_attend(8, 1, d, block, [40], [1900], seed=d + 1, window=300)
    _run_attend(2, 1, 128, 16, [20], [3], seed=5)                  # more splits than tiles, rows without keys


@pytest.mark.parametrize("d", [64, 128, 256])
def test_chunk_warps_that_run_ahead(d):
    """Second row tiles with warps without rows, whose neighbours in the first finish tiles before the others: a row is through only when
    its last product is, and the same call gives the same bits."""
    pool, table, cu, q, o, lse = _run_attend(8, 1, d, 16, [24, 25, 36, 23], [903, 1210, 640, 1100], seed=d, cap=30.0)
    for _ in range(3):
        again, l2 = attend(pool, q.cuda(), table, cu, [903, 1210, 640, 1100], 8, 1, d, cap=30.0)
        assert torch.equal(o, again) and torch.equal(lse, l2)


def test_chunk_many_sequences():
    """More sequences than threads of a block, all of them with more rows than the other kernel takes, or mixed."""
    n = 560
    _run_attend(4, 1, 64, 16, [7] * n, [7 + i % 12 for i in range(n)], seed=6)
    _run_attend(8, 2, 64, 16, [(1, 7, 2, 40)[i % 4] for i in range(40)], [45 + i for i in range(40)], seed=7)


def test_chunk_absent_pages_and_what_lies_around():
    hq, hkv, d, block = 4, 1, 128, 16
    lens, cu = [170], [0, 60]
    pool = Pool(14, hkv, block, d, 5)
    table = torch.tensor([[0, 1, -1, 2, 3, 99, 4, 5, 6, 7, 8, 9, 9]], dtype=torch.int32)
    q = torch.randn(60, hq * d, generator=torch.Generator().manual_seed(1)).to(BF16)
    c, s = pool.host()
    for kw in (dict(), dict(window=40)):
        want = R.attention(q.view(-1, hq, d), c["k"], c["v"], s["k"], s["v"], table, cu, lens, 0.1, **kw)
        for n in "kv":
            pool.c[n][8, :, 170 % block:] = 0x7F                  # behind the sequence's end (block 10 of it)
            for page in (10, 11, 12, 13):
                pool.c[n][page], pool.s[n][page] = 0xFF, math.inf
        if kw:
            table = table.clone()
            table[0, :4] = torch.tensor([12, 99, 13, -1], dtype=torch.int32)      # in front of every window (keys below 71)
            want = R.attention(q.view(-1, hq, d), c["k"], c["v"], s["k"], s["v"], table, cu, lens, 0.1, **kw)
        close(*attend(pool, q.cuda(), table, cu, lens, hq, hkv, d, scale=0.1, **kw), want)


@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 2], [40, 3, 100]])
def test_attention_strides_streams_and_captures(new):
    """Rows of Q and O inside wider ones, no lse, a larger max_new, another stream, a captured launch replayed: the same bits."""
    from flashrt_b200 import flash_rt_fa2 as fa2
    hq, hkv, d, block = 8, 2, 128, 32
    ctx = [n + 200 * i for i, n in enumerate(new)]
    pool, table, cu, q, o, lse = _run_attend(hq, hkv, d, block, new, ctx, seed=2)
    wide_q = torch.zeros(cu[-1], hq * d + 40, dtype=BF16, device="cuda")
    wide_q[:, :hq * d] = q.cuda()
    wide_o = torch.full((cu[-1], hq * d + 24), -7.0, dtype=BF16, device="cuda")
    n = fa2.paged_workspace_bytes(cu[-1], len(ctx), max(new), hq, hkv, d)
    work = torch.zeros(n, dtype=torch.uint8, device="cuda")
    dev = lambda y: torch.tensor(y, dtype=torch.int32).cuda()  # noqa: E731
    cu_d, lens_d, table_d = dev(cu), dev(ctx), table.cuda()

    def call(stream):
        fa2.paged_fwd_fp8(wide_q.data_ptr(), wide_o.data_ptr(), 0, pool.c["k"].data_ptr(), pool.c["v"].data_ptr(), pool.s["k"].data_ptr(),
                          pool.s["v"].data_ptr(), table_d.data_ptr(), table.shape[1], cu_d.data_ptr(), lens_d.data_ptr(), cu[-1], len(ctx),
                          max(new), pool.num_blocks, block, hq, hkv, d, d ** -0.5, work.data_ptr(), n, stream, q_stride=hq * d + 40,
                          o_stride=hq * d + 24)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    call(side.cuda_stream)
    side.synchronize()
    assert torch.equal(wide_o[:, :hq * d], o) and (wide_o[:, hq * d:] == -7).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(_stream())
    for _ in range(3):
        wide_o.fill_(-7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(wide_o[:, :hq * d], o) and (wide_o[:, hq * d:] == -7).all()
    o2, lse2 = attend(pool, q.cuda(), table, cu, ctx, hq, hkv, d, max_new=max(new) + 200)
    c, s = pool.host()
    close(o2, lse2, R.attention(q.view(-1, hq, d), c["k"], c["v"], s["k"], s["v"], table, cu, ctx, d ** -0.5))


@pytest.mark.parametrize("d,hq,new", [(64, 4, 1), (64, 8, 3), (128, 8, 1), (128, 8, 2), (256, 8, 1), (256, 4, 2), (256, 8, 9)])
def test_attention_many_pieces(d, hq, new):
    """One key/value head on a long context: an item in more pieces than a join has in flight."""
    _run_attend(hq, 1, d, 64, [new], [9001], seed=d + new)


@pytest.mark.parametrize("hq,hkv,new", [(8, 1, 2), (6, 3, 5), (16, 4, 4), (12, 1, 1)])
def test_attention_heads_of_256_many_sequences_of_few_rows(hq, hkv, new):
    """9 to 16 rows a sequence: with many sequences the kernel for few rows, with few the other one."""
    ctx = [new + (37 * i) % 211 for i in range(21)]
    _run_attend(hq, hkv, 256, 16, [new] * 21, ctx, seed=hq)
    _run_attend(hq, hkv, 256, 16, [new] * 2, ctx[:2], seed=hq)


@pytest.mark.parametrize("d,hq", [(64, 4), (128, 4), (256, 2)])
@pytest.mark.parametrize("new,ctx", [([40, 5], [90, 70]), ([40, 0, 1], [40, 33, 300]), ([3, 40, 2], [3, 40, 150])])
def test_attention_padded_to_the_longest(d, hq, new, ctx):
    """Room for max_new tokens of every sequence, some of which bring few: all are answered, the rows behind them left alone."""
    _run_attend(hq, 1, d, 16, new, ctx, seed=d, tail=len(new) * max(new) - sum(new))


@pytest.mark.parametrize("d,new", [(128, [1, 1, 1]), (64, [3, 1, 2]), (256, [1, 1, 1]), (128, [40, 9, 33])])
@pytest.mark.parametrize("window,causal", [(0, True), (150, True), (20, True), (0, False)])
def test_attention_of_sequences_longer_than_their_table(d, new, window, causal):
    """Keys behind the table's last entry are absent; positions, masks and windows are those of the whole sequence."""
    ctx, block, width, hq, hkv = [300, 176, 40], 16, 11, 8, 2          # room for 176 keys
    pool = Pool(60, hkv, block, d, 3)
    table = R.pages(ctx, block, 60, 3, width=19)
    table[:, width:] = -1
    cu = [0, new[0], new[0] + new[1], sum(new)]
    q = torch.randn(cu[-1], hq * d, generator=torch.Generator().manual_seed(4)).to(BF16)
    c, s = pool.host()
    o, lse = attend(pool, q.cuda(), table[:, :width].contiguous(), cu, ctx, hq, hkv, d, window=window, causal=causal)
    close(o, lse, R.attention(q.view(-1, hq, d), c["k"], c["v"], s["k"], s["v"], table, cu, ctx, d ** -0.5, window=window, causal=causal))


def test_attention_one_workspace_for_all_shapes():
    """A workspace that fits the largest serves every shape in any order: no launch leaves its partials where another one counts."""
    from flashrt_b200 import flash_rt_fa2 as fa2
    shapes = [(8, 1, 256, 16, [1, 1], [1500, 40]), (4, 1, 128, 32, [9], [2000]), (8, 2, 64, 64, [1], [3000]), (4, 1, 256, 128, [40], [900]),
              (6, 2, 128, 16, [7, 1, 30], [400, 900, 1100]), (32, 1, 128, 64, [1], [2500]), (4, 1, 64, 16, [70], [1300])]
    size = max(fa2.paged_workspace_bytes(sum(new), len(new), max(new), hq, hkv, d) for hq, hkv, d, _, new, _ in shapes)
    work = torch.zeros(size, dtype=torch.uint8, device="cuda")
    runs = []
    for i, (hq, hkv, d, block, new, ctx) in enumerate(shapes):
        pool, table, cu, q, o, lse = _run_attend(hq, hkv, d, block, new, ctx, seed=i)
        runs.append((pool, q.cuda(), table, cu, ctx, hq, hkv, d, o, lse))
    order = torch.randperm(3 * len(runs), generator=torch.Generator().manual_seed(0)) % len(runs)
    for i in order.tolist():
        pool, q, table, cu, ctx, hq, hkv, d, o, lse = runs[i]
        again, l2 = attend(pool, q, table, cu, ctx, hq, hkv, d, work=work)
        assert torch.equal(o, again) and torch.equal(lse, l2), i


def test_attention_workspace_too_small_is_refused():
    from flashrt_b200 import flash_rt_fa2 as fa2
    from flashrt_b200._lib import KernelError
    hq, hkv, d = 8, 2, 128
    t = torch.zeros(4096, dtype=torch.int32, device="cuda")
    for new in (1, 300):
        n = fa2.paged_workspace_bytes(new, 1, new, hq, hkv, d)
        with pytest.raises(KernelError, match="-1"):
            fa2.paged_fwd_fp8(*[t.data_ptr()] * 8, 1, t.data_ptr(), t.data_ptr(), new, 1, new, 4, 16, hq, hkv, d, 0.1, t.data_ptr(), n - 16, _stream())
    torch.cuda.synchronize()


def test_attention_offsets_beyond_32_bits():
    """A pool of more than 4 GB: blocks at its far end."""
    hq, hkv, d, block = 8, 8, 256, 128
    num = (1 << 32) // (hkv * block * d) + 40
    pool = Pool(4, hkv, block, d, 3)
    small_c, small_s = pool.host()
    big = {n: torch.zeros(num, hkv, block, d, dtype=torch.uint8, device="cuda") for n in "kv"}
    scl = {n: torch.ones(num, hkv, device="cuda") for n in "kv"}
    for n in "kv":
        big[n][num - 4:] = pool.c[n]
        scl[n][num - 4:] = pool.s[n]
    pool.c, pool.s, pool.num_blocks = big, scl, num
    q = torch.randn(1, hq * d, generator=torch.Generator().manual_seed(1)).to(BF16)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32)
    want = R.attention(q.view(-1, hq, d), small_c["k"], small_c["v"], small_s["k"], small_s["v"], table, [0, 1], [300], d ** -0.5)
    close(*attend(pool, q.cuda(), table + (num - 4), [0, 1], [300], hq, hkv, d), want)
    qkv = torch.randn(1, 3 * hq * d, generator=torch.Generator().manual_seed(2)).to(BF16)
    dev = lambda y: torch.tensor(y, dtype=torch.int32).cuda()  # noqa: E731
    append(pool, qkv.cuda(), None, (table + (num - 4)).cuda(), None, dev([301]), hq, hkv, d)
    torch.cuda.synchronize()
    got = R.codes(pool.c["v"][num - 1, :, 44].cpu()) * pool.s["v"][num - 1].cpu().to(F64)[:, None]
    want = qkv[0, 2 * hq * d:].view(hkv, d).to(F64)
    assert ((got - want).abs() <= want.abs() * 2.0 ** -4 * (1 + 2.0 ** -12) + pool.s["v"][num - 1].cpu().to(F64)[:, None] * 2.0 ** -9).all()
    torch.cuda.empty_cache()

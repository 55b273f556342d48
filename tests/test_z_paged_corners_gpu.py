"""Corners of the paged cache and of the attention over it: windows without end, infinite keys under the rotation, capped scores beside
hidden keys, what a block loses while its scale grows, single tokens beside chunks, calls at once and over one workspace, groups wider than
a tile, rows that are no numbers, shared blocks."""
import math

import pytest
import torch

import paged_ref as R
import test_w_paged_cache_gpu as W
import test_y_int8_block_gpu as Y

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def _dev(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 30, 2 ** 30])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_window_without_end_where_tokens_have_no_position(window, d):
    """More new tokens than positions, and a window of the largest numbers: positions before the first one see nothing, the others all
    keys up to their own.  Few rows a sequence, and chunks."""
    _, _, _, _, o, lse = W._run_attend(4, 2, d, 16, [5, 3, 1], [2, 3, 40], seed=2, window=window)
    assert (o[:3] == 0).all() and lse[:, :3].isneginf().all() and lse[:, 3:].isfinite().all()
    _, _, _, _, o, lse = W._run_attend(4, 1, d, 16, [40, 70], [17, 90], seed=3, window=window)
    assert (o[:23] == 0).all() and lse[:, :23].isneginf().all() and lse[:, 23:].isfinite().all()


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("d,block,tokens", [(64, 16, 9), (128, 32, 7), (64, 64, 200), (256, 64, 70)])
def test_append_infinities_under_the_rotation(halves, d, block, tokens):
    """Infinite elements of a key turn as the formula says: infinite where one term is or both agree (clamped), NaN where they differ
    (-448).  The queries of the row show the same.  Angles of all four quadrants; no sine or cosine is zero."""
    hq = hkv = 1
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, 3 * d, generator=g).to(BF16)
    kind = torch.randint(0, 12, (tokens, d), generator=g)               # a sixth of all elements
    x[:, d:2 * d] = torch.where(kind == 0, math.inf, torch.where(kind == 1, -math.inf, x[:, d:2 * d].float())).to(BF16)
    x[:, :d] = x[:, d:2 * d]
    angle = torch.arange(4)[torch.randint(0, 4, (tokens, d // 2), generator=g)] * (math.pi / 2) + 0.1 + 1.3 * torch.rand(tokens, d // 2, generator=g)
    rope = torch.stack([angle.cos(), angle.sin()], -1).reshape(tokens, d).float()
    table = R.pages([tokens], block, 8, 1)
    pool = W.Pool(8, hkv, block, d, 1)
    q = W.append(pool, x.cuda(), rope.cuda(), table.cuda(), _dev([0, tokens]), _dev([tokens]), hq, hkv, d, halves).cpu().double()
    c, s = pool.host()
    y = R.rotate(x.double().view(tokens, 3, d)[:, :2], rope, halves)
    yq, yk = y[:, 0], y[:, 1]
    assert yk.isnan().any() and (yk == math.inf).any() and (yk == -math.inf).any()
    assert torch.equal(q.isnan(), yq.isnan()) and torch.equal(q == math.inf, yq == math.inf) and torch.equal(q == -math.inf, yq == -math.inf)
    for j in range((tokens + block - 1) // block):
        rows, page = yk[j * block:(j + 1) * block], int(table[0, j])
        fin = rows.isfinite()
        now = torch.where(fin, rows.abs(), 0.0).max() / 448
        assert (s["k"][page, 0].double() - now).abs() <= now * 2.0 ** -20
        code = R.codes(c["k"][page, 0, :len(rows)])
        want = torch.where(rows.isnan(), -448.0, (rows / now).clamp(-448, 448))
        bar = (want.abs() * 2.0 ** -4 * (1 + 2.0 ** -12)).clamp_min(2.0 ** -10 * (1 + 2.0 ** -12)) + 2.0 ** -12
        assert ((code - want).abs() <= torch.where(fin, bar, 0.0)).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv,new,ctx", [(8, 2, [1, 3], [70, 100]), (4, 2, [1, 1], [70, 100]), (4, 1, [60], [62])])
def test_capped_scores_beside_hidden_keys(d, hq, hkv, new, ctx):
    """Finite codes that a row does not see -- behind its sequence's end, or of tokens after it -- change no bit of it, under a cap
    of which the hidden scores pass half and the seen ones stay far below."""
    cap, block = 30.0, 16
    pool = W.Pool(20, hkv, block, d, d)
    pool.s["k"] *= 3.0
    table = R.pages(ctx, block, 20, 1)
    cu = [0] + torch.tensor(new).cumsum(0).tolist()
    q = torch.randn(cu[-1], hq * d, generator=torch.Generator().manual_seed(2)).abs().to(BF16)
    hidden = q.double().view(-1, hq, d).sum(-1).min() * 448 * float(pool.s["k"].min()) * d ** -0.5
    assert hidden > cap / 2                               # where the form of tanh changes
    run = lambda: W.attend(pool, q.cuda(), table, cu, ctx, hq, hkv, d, cap=cap)  # noqa: E731
    last = [(int(table[b, (n - 1) // block]), n % block) for b, n in enumerate(ctx)]
    seen = []
    for code in (0x00, 0x7E, 0xFE):
        for page, used in last:
            if used:
                pool.c["k"][page, :, used:] = code
        seen.append(run())
    assert all(torch.equal(seen[0][i], s[i]) for s in seen for i in (0, 1))
    if new[-1] == 1:
        return
    seen = []
    for code in (0x00, 0x7E, 0xFE):                        # the key of the last token
        pool.c["k"][last[-1][0], :, (ctx[-1] - 1) % block] = code
        seen.append(run())
    assert all(torch.equal(seen[0][0][:-1], o[:-1]) and torch.equal(seen[0][1][:, :-1], lse[:, :-1]) for o, lse in seen)
    assert not torch.equal(seen[0][0][-1], seen[1][0][-1])
    c, s = pool.host()
    W.close(*seen[-1], R.attention(q.view(-1, hq, d), c["k"], c["v"], s["k"], s["v"], table, cu, ctx, d ** -0.5, cap=cap))


def lost(y, s, growths):
    """Largest error of a stored value after its block's scale has grown `growths` times, s the scale of now: each rounding is off by
    2^-4 of what it rounds or by 2^-10 of the scale, and rounds what the one before has left, so
    e_g <= e_{g-1} (1 + 2^-4) + 2^-4 |y| + 2^-10 s.  The fp32 operations in front of it by 2^-22: 2^-10 of a rounding is plenty."""
    r = 2.0 ** -4 * (1 + 2.0 ** -10)
    return ((1 + r) ** (growths + 1) - 1) * (y.abs() + 2.0 ** -6 * s)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("growth", [1.0, 1.07, 1.3])
def test_what_a_block_loses_while_its_scale_grows(block, growth):
    """A block filled token by token against the bound that the header gives; one filled at once is held to a single rounding."""
    hkv, d, n = 2, 64, 2 * block + 5
    x = (torch.randn(n, 3 * hkv * d, generator=torch.Generator().manual_seed(block)) * growth ** torch.arange(n)[:, None]).to(BF16)
    table = R.pages([n], block, 4, 1)
    for step in (1, 3, n):
        pool = W.Pool(4, hkv, block, d, 2)
        before = {m: torch.zeros(4, hkv) for m in "kv"}
        grown, records = ({m: torch.zeros(n, hkv) for m in "kv"} for _ in range(2))
        for a in range(0, n, step):
            e = min(a + step, n)
            W.append(pool, x[a:e].cuda(), None, table.cuda(), _dev([0, e - a]), _dev([e]), hkv, hkv, d)
            c, s = pool.host()
            for m, first in (("k", hkv), ("v", 2 * hkv)):
                # a scale grows when a call brings the block's largest magnitude so far
                size = x[:, first * d:(first + hkv) * d].float().abs().view(n, hkv, d).amax(2)
                for i in range(a):
                    lo, hi = i // block * block, min(i // block * block + block, e)
                    if hi > a:
                        records[m][i] += size[a:hi].amax(0) > size[lo:a].amax(0)
                for i in range(a):
                    grown[m][i] += s[m][table[0, i // block]] != before[m][table[0, i // block]]
                before[m] = s[m]
                for i in range(e):
                    page = int(table[0, i // block])
                    y = x[i, first * d:(first + hkv) * d].to(F64).view(hkv, d)
                    now = s[m][page].to(F64)[:, None]
                    assert ((R.codes(c[m][page, :, i % block]) * now - y).abs() <= lost(y, now, grown[m][i].to(F64)[:, None])).all()
                assert torch.equal(grown[m], records[m])
        assert (max(int(grown[m].max()) for m in "kv") > 0) == (step < n)


@pytest.mark.parametrize("hq,hkv,d,block", [(8, 2, 128, 32), (6, 2, 64, 64)])
def test_cache_of_the_block_holds_each_token_to_its_own_roundings(hq, hkv, d, block):
    """The attention block from prompts to tokens: a value just written is off by one rounding, an older one by one more for each time its
    block's scale has really grown."""
    batch, width = 3, 256 // block
    b = Y.Block(512, hq, hkv, d, block, 3 * width, batch, width, 128, seed=d)
    b.table.copy_(torch.randperm(3 * width, generator=torch.Generator().manual_seed(1)).view(batch, width))
    table, rope = b.table.cpu(), b.rope.cpu()
    g = torch.Generator().manual_seed(2)
    lens, tokens, before = [0] * batch, [], None
    for new in [[60, 1, 0], [25, 50, 30], [1, 1, 1], [1, 1, 1], [3, 1, 40], [1, 1, 1], [1, 2, 0]]:
        lens = [a + n for a, n in zip(lens, new)]
        cu = [0] + torch.tensor(new).cumsum(0).tolist()
        T = cu[-1]
        b.x[:T] = torch.randn(T, 512, generator=g).to(BF16)
        b.cu.copy_(torch.tensor(cu, dtype=torch.int32))
        b.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        b.step(T, max(new), new != [1] * batch)
        torch.cuda.synchronize()
        now = {"k": b.ks.cpu(), "v": b.vs.cpu()}
        codes = {"k": b.k.cpu(), "v": b.v.cpu()}
        for t in tokens:
            t["growths"] += now[t["of"]][t["page"]] != before[t["of"]][t["page"]]
        before = now
        qkv = b.qkv[:T].cpu().to(F64).view(T, hq + 2 * hkv, d)
        for s in range(batch):
            rows = qkv[cu[s]:cu[s + 1]]
            k = R.rotate(rows[:, hq:hq + hkv], rope[lens[s] - new[s]:lens[s]], True)
            for i in range(new[s]):
                at = lens[s] - new[s] + i
                for of, y in (("k", k[i]), ("v", rows[i, hq + hkv:])):
                    tokens.append({"of": of, "y": y, "page": int(table[s, at // block]), "slot": at % block, "growths": torch.zeros(hkv)})
        for t in tokens:
            scale = now[t["of"]][t["page"]].to(F64)[:, None]
            got = R.codes(codes[t["of"]][t["page"], :, t["slot"]]) * scale
            assert ((got - t["y"]).abs() <= lost(t["y"], scale, t["growths"].to(F64)[:, None])).all()
    assert max(int(t["growths"].max()) for t in tokens) >= 1


@pytest.mark.parametrize("kw", [dict(), dict(window=700), dict(cap=20.0)])
@pytest.mark.parametrize("d,hq,hkv", [(64, 8, 2), (128, 8, 1), (256, 4, 1)])
def test_single_tokens_and_a_chunk_in_one_call(d, hq, hkv, kw):
    """Decoding sequences, drafted tokens and a chunk of a prompt, each on a context of thousands; rows behind them left alone."""
    W._run_attend(hq, hkv, d, 32, [1, 1, 33, 1, 4, 1, 0], [2900, 17, 1700, 1, 900, 3001, 40], seed=d, tail=5, **kw)


def _call(pool, q, table, cu, ctx, hq, hkv, d, work, stream, o, lse):
    """A call over tensors that it keeps alive."""
    from flashrt_b200 import flash_rt_fa2 as fa2
    new = max(b - a for a, b in zip(cu, cu[1:]))
    q, cu_d, lens_d, table_d = q.cuda(), _dev(cu), _dev(ctx), table.cuda()
    return lambda: fa2.paged_fwd_fp8(
        q.data_ptr(), o.data_ptr(), lse.data_ptr(), pool.c["k"].data_ptr(), pool.c["v"].data_ptr(), pool.s["k"].data_ptr(),
        pool.s["v"].data_ptr(), table_d.data_ptr(), table.shape[1], cu_d.data_ptr(), lens_d.data_ptr(), q.shape[0], len(ctx), new,
        pool.num_blocks, pool.block, hq, hkv, d, d ** -0.5, work.data_ptr(), work.numel(), stream.cuda_stream)


def _work(shapes):
    from flashrt_b200 import flash_rt_fa2 as fa2
    size = max(fa2.paged_workspace_bytes(sum(n), len(n), max(n), hq, hkv, d) for hq, hkv, d, n, _ in shapes)
    return torch.zeros(size, dtype=torch.uint8, device="cuda")


def test_two_calls_at_once():
    """A decode batch and chunks on two streams, each with its workspace: the bits of the calls one behind the other."""
    calls, want, got = [], [], []
    for i, (hq, hkv, d, new, ctx) in enumerate([(8, 2, 128, [1, 1, 1, 1], [3000, 1200, 2500, 77]), (8, 2, 128, [50, 90], [1500, 2100])]):
        pool, table, cu, q, o, lse = W._run_attend(hq, hkv, d, 32, new, ctx, seed=i)
        want.append((o, lse))
        got.append((torch.zeros_like(o), torch.zeros_like(lse)))
        calls.append(_call(pool, q, table, cu, ctx, hq, hkv, d, _work([(hq, hkv, d, new, ctx)]), torch.cuda.Stream(), *got[-1]))
    torch.cuda.synchronize()
    for _ in range(20):
        for call in calls:
            call()
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_calls_behind_one_another_in_one_graph_share_a_workspace():
    """Layers of a model: captured calls of both kernels over one workspace, replayed."""
    shapes = [(8, 2, 128, [1, 1, 1], [900, 1200, 77]), (8, 2, 128, [50, 9], [1500, 700]), (8, 2, 128, [1, 40, 3], [2000, 300, 1100])]
    work, stream, calls, want, got = _work(shapes), torch.cuda.Stream(), [], [], []
    for i, (hq, hkv, d, new, ctx) in enumerate(shapes):
        pool, table, cu, q, o, lse = W._run_attend(hq, hkv, d, 32, new, ctx, seed=i)
        want.append((o, lse))
        got.append((torch.zeros_like(o), torch.zeros_like(lse)))
        calls.append(_call(pool, q, table, cu, ctx, hq, hkv, d, work, stream, *got[-1]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for _ in range(3):
            for call in calls:
                call()
    for _ in range(3):
        for o, lse in got:
            o.fill_(-7.0)
            lse.fill_(-7.0)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("hq,hkv,new", [(64, 1, [1, 1]), (200, 1, [1, 1, 1]), (300, 1, [2, 1, 3]), (96, 2, [5, 1, 0])])
def test_one_key_head_for_many_query_heads(hq, hkv, new):
    """More heads of a group than a row tile has rows: the rows of one token fill several."""
    W._run_attend(hq, hkv, 64, 16, new, [n + 61 * i + 40 for i, n in enumerate(new)], seed=hq)
    W._run_attend(hq // 4 * hkv, hkv, 128, 32, new, [n + 61 * i + 40 for i, n in enumerate(new)], seed=hq, window=50)


@pytest.mark.parametrize("max_new", [1, 40])
def test_no_sequence_brings_a_token(max_new):
    pool = W.Pool(4, 2, 16, 128, 1)
    q = torch.randn(5, 8 * 128, device="cuda").to(BF16)
    o, lse = W.attend(pool, q, R.pages([20, 3], 16, 4, 1), [0, 0, 0], [20, 3], 8, 2, 128, max_new=max_new)
    assert (o == -7).all() and (lse == -7).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,ctx", [([1, 2], [300, 90]), ([40, 30], [300, 90])])
def test_a_row_that_is_no_number_spoils_no_other(d, new, ctx):
    """NaN or infinite queries of one token and head: that row shows it, every other one keeps its bits."""
    hq, hkv = 8, 2
    pool, table, cu, q, o, lse = W._run_attend(hq, hkv, d, 16, new, ctx, seed=d, cap=20.0)
    token, head = cu[-1] - 1, 5
    others = torch.ones(cu[-1], hq, dtype=torch.bool, device="cuda")
    others[token, head] = False
    for bad in (math.nan, math.inf):
        q2 = q.clone().view(-1, hq, d)
        q2[token, head, ::2] = bad
        o2, lse2 = W.attend(pool, q2.view(-1, hq * d).cuda(), table, cu, ctx, hq, hkv, d, cap=20.0)
        assert torch.equal(o.view(-1, hq, d)[others], o2.view(-1, hq, d)[others]) and torch.equal(lse.T[others], lse2.T[others])
        if bad != bad:
            assert o2.view(-1, hq, d)[token, head].isnan().all() and lse2[head, token].isnan()


def test_sequences_share_the_blocks_of_a_prefix():
    """Blocks that are only read may stand in several tables, and twice in one."""
    hq, hkv, d, block = 8, 2, 128, 16
    pool = W.Pool(9, hkv, block, d, 3)
    table = torch.tensor([[0, 1, 2, 3, -1], [0, 1, 2, 4, 5], [0, 1, 0, 1, 6]], dtype=torch.int32)
    for new, ctx in (([1, 1, 1], [60, 77, 70]), ([12, 29, 6], [60, 77, 70])):
        cu = [0] + torch.tensor(new).cumsum(0).tolist()
        q = torch.randn(cu[-1], hq * d, generator=torch.Generator().manual_seed(4)).to(BF16)
        c, s = pool.host()
        want = R.attention(q.view(-1, hq, d), c["k"], c["v"], s["k"], s["v"], table, cu, ctx, d ** -0.5)
        W.close(*W.attend(pool, q.cuda(), table, cu, ctx, hq, hkv, d), want)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_refused_workspace_leaves_the_outputs_alone(d):
    """Single tokens and chunks: a workspace that is too small for one of the two kernels is refused in front of both."""
    from flashrt_b200._lib import KernelError
    hq, hkv, new, ctx = 8, 2, [1, 40, 2], [90, 50, 30]
    pool = W.Pool(16, hkv, 16, d, 1)
    q = torch.randn(43, hq * d, device="cuda").to(BF16)
    o, lse = torch.full((43, hq * d), -7.0, dtype=BF16, device="cuda"), torch.full((hq, 43), -7.0, device="cuda")
    work = _work([(hq, hkv, d, new, ctx)])
    args = (pool, q, R.pages(ctx, 16, 16, 1), [0, 1, 41, 43], ctx, hq, hkv, d)
    for size in (4096, work.numel() // 2):                 # too small for either, enough for single tokens alone
        with pytest.raises(KernelError, match="-1"):
            _call(*args, work[:size], torch.cuda.current_stream(), o, lse)()
    torch.cuda.synchronize()
    assert (o == -7).all() and (lse == -7).all()
    _call(*args, work, torch.cuda.current_stream(), o, lse)()
    torch.cuda.synchronize()
    assert (o != -7).any(1).all()

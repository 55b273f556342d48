"""Corners of the paged cache and of the attention over it: windows without end, infinite keys under the rotation, capped scores beside
hidden keys, what a block loses while its scale grows, batches of single tokens and chunks."""
import math

import pytest
import torch

import paged_ref as R
import test_w_paged_cache_gpu as W

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

"""Probabilities of logits, and drafted tokens verified against them."""
import numpy as np
import pytest
import torch

import decode_ref as R

pytestmark = pytest.mark.gpu
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
INF, NAN = float("inf"), float("nan")


def _stream():
    return torch.cuda.current_stream().cuda_stream


def softmax(x, t=None, in_stride=0, out_stride=0, rows=None, vocab=None):
    from flashrt_b200 import flash_rt_kernels as fvk
    rows, vocab = rows or x.shape[0], vocab or x.shape[1]
    width = out_stride or vocab
    p = torch.full((rows * width + 9,), -3.0, device="cuda")
    fvk.softmax_rows(x.data_ptr(), p.data_ptr(), rows, vocab, _stream(), temperature=t.data_ptr() if t is not None else 0,
                     in_f32=x.dtype == F32, in_stride=in_stride, out_stride=out_stride)
    torch.cuda.synchronize()
    assert (p[rows * width:] == -3).all()
    p = p[:rows * width].view(rows, width)
    assert (p[:, vocab:] == -3).all()
    return p[:, :vocab].cpu()


def close(p, x, t):
    """A probability p = w f / z: the weight's argument d c (c = log2(e) / T) has three roundings (2^-24 of it each, times ln 2 and the
    argument), the exponential is off by 2^-22, the factor's by 2^-22 and its two roundings, the sum of V weights, each off as much, by
    2^-24 times the depth of its tree (at most V / 4096 values a thread and 20 steps behind)."""
    want = R.softmax_rows(x.cpu(), t.cpu())
    arg = torch.where(want > 0, -torch.log2(want.clamp_min(1e-300)), 0.0) + np.log2(x.shape[1]) + 2
    rel = 2.0 ** -24 * (4 * arg) + 4 * 2.0 ** -22 + 2.0 ** -24 * (x.shape[1] / 4096 + 64)
    assert ((p.to(F64) - want).abs() <= want * rel + 2.0 ** -120).all(), ((p.to(F64) - want).abs() / (want * rel + 2.0 ** -120)).max()
    if (t <= 0).any():
        assert torch.equal(p[t.cpu() <= 0].to(F64), want[t.cpu() <= 0])


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 31), (5, 500), (300, 33), (7, 4096), (1, 50257), (4, 50257), (150, 1003), (2, 131072),
                                        (37, 16385), (1, 262143), (3, 300001), (1, 700000), (160, 9000)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_softmax(rows, vocab, dtype):
    g = torch.Generator().manual_seed(rows + vocab)
    x = (torch.randn(rows, vocab, generator=g) * 4).to(dtype).cuda()
    t = (0.3 + torch.rand(rows, generator=g)).cuda()
    t[rows // 2::5] = 0.0
    close(softmax(x, t), x, t)
    one = torch.ones(rows).cuda()
    close(softmax(x), x, one)


def test_softmax_masks_and_special_values():
    for vocab in (40, 5000, 70001):
        for dtype in (BF16, F32):
            x = torch.randn(12, vocab, generator=torch.Generator().manual_seed(vocab)).to(dtype)
            x[0] = -INF
            x[1] = NAN
            x[2, 1:] = -INF
            x[3, ::2] = -INF
            x[4] = torch.finfo(dtype).min
            x[5, 3], x[5, 39] = INF, INF
            x[6, 7] = NAN
            x[7] = 0
            x[8, vocab - 1] = 50
            x[9, : vocab - 1] = torch.finfo(dtype).min
            x[10] = -INF
            x[10, vocab - 1] = -1e4
            x[11, 5:] = NAN
            x = x.cuda()
            for temps in ([1.0] * 12, [0.0] * 12, [0.5, 0.0, 2.0, -1.0, 1.0, 1.0, 0.0, 0.0, 1e-3, 1.0, 1.0, 1.0]):
                t = torch.tensor(temps).cuda()
                p = softmax(x, t)
                assert not p.isnan().any()
                close(p, x, t)
                assert (p[0] == 0).all() and (p[1] == 0).all() and p[2, 0] == 1 and p[10, vocab - 1] == 1
            t = torch.tensor([NAN, 1e-42, INF] * 4).cuda()
            p = softmax(x, t)
            assert not p.isnan().any() and set(p[3].unique().tolist()) <= {0.0, 1.0}
            assert torch.allclose(p[4], torch.full((vocab,), 1.0 / vocab), rtol=1e-6, atol=0)      # equal logits, a temperature next to nothing
            for r in (2, 5, 8, 11):                                                 # an infinite temperature: even over what is not masked
                hit = (x[r] == INF) if (x[r] == INF).any() else (x[r] > -INF)
                assert torch.allclose(p[r], (hit / hit.sum()).float().cpu(), rtol=1e-6, atol=0)


@pytest.mark.parametrize("rows,vocab", [(700, 20001), (320, 50257), (170, 131071), (160, 131072), (80, 230001)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_softmax_clusters_that_go_from_row_to_row(rows, vocab, dtype):
    """More rows than clusters find room, of every kind, one behind the other."""
    x = (torch.randn(rows, vocab, device="cuda", generator=torch.Generator("cuda").manual_seed(vocab)) * 4).to(dtype)
    x[3::17] = -INF
    x[5::17, 1:] = -INF
    x[7::17, ::3] = NAN
    x[8::17, vocab // 2] = INF
    x[11::17, :vocab - 1] = torch.finfo(dtype).min
    t = torch.full((rows,), 0.7)
    t[2::5], t[4::7] = 0.0, 3.0
    t = t.cuda()
    p = softmax(x, t)
    assert not p.isnan().any()
    for r in range(0, rows, 64):
        close(p[r:r + 64], x[r:r + 64], t[r:r + 64])
    assert torch.equal(p, softmax(x, t))


def test_softmax_ties_and_strides():
    x = torch.zeros(6, 30000)
    x[1, 29999], x[2, 777], x[2, 20000], x[3, :] = 1, 2, 2, -5
    x[4, 16384:] = 1
    x = x.to(BF16).cuda()
    p = softmax(x, torch.zeros(6).cuda())
    assert p.argmax(1).tolist() == [0, 29999, 777, 0, 16384, 0] and (p.sum(1) == 1).all()
    wide = torch.randn(7, 1009, device="cuda")
    t = torch.full((7,), 0.8).cuda()
    close(softmax(wide, t, in_stride=1009, out_stride=1024, rows=7, vocab=1001), wide[:, :1001], t)


def test_softmax_rows_that_start_anywhere():
    """Inputs one value, outputs one or three values behind a boundary."""
    from flashrt_b200 import flash_rt_kernels as fvk
    g = torch.Generator().manual_seed(8)
    for dtype in (BF16, F32):
        for vocab, rows in ((5000, 3), (40000, 2), (70, 9), (131072, 40)):
            for i, j in ((1, 0), (0, 1), (3, 3), (1, 3), (7, 2)):
                x = (torch.randn(rows * vocab + 8, generator=g) * 3).to(dtype).cuda()
                p = torch.full((rows * vocab + 8,), -3.0, device="cuda")
                es = 2 if dtype == BF16 else 4
                t = torch.full((rows,), 0.9).cuda()
                fvk.softmax_rows(x.data_ptr() + i * es, p.data_ptr() + 4 * j, rows, vocab, _stream(), temperature=t.data_ptr(), in_f32=dtype == F32)
                torch.cuda.synchronize()
                assert (p[:j] == -3).all() and (p[j + rows * vocab:] == -3).all()
                close(p[j:j + rows * vocab].view(rows, vocab).cpu(), x[i:i + rows * vocab].view(rows, vocab), t)


# ------------------------------------------------------------------------------------------------ verification
def rows_of(rng, n, vocab, zeros=0.0):
    p = rng.exponential(size=(n, vocab)) ** 3
    if zeros:
        p[rng.random((n, vocab)) < zeros] = 0
        p[:, rng.integers(vocab)] += 1e-3
    return (p / p.sum(1, keepdims=True)).astype(np.float32)


def run(p, q, tokens, cu, lens, u, v, n_tokens=None, p_pad=0, q_pad=0, alias=False):
    from flashrt_b200 import flash_rt_kernels as fvk
    dev = lambda x, t: torch.tensor(np.asarray(x), dtype=t, device="cuda")  # noqa: E731
    n, vocab = p.shape
    pad = lambda x, k: torch.nn.functional.pad(dev(x, F32), (0, k), value=NAN).contiguous()  # noqa: E731
    dp, dq = pad(p, p_pad), None if q is None else pad(q, q_pad)
    tok, dcu, dlen, du, dv = dev(tokens, I32), dev(cu, I32), dev(lens, I32), dev(u, F32), dev(v, F32)
    batch = len(cu) - 1
    out = torch.full((n + 5,), -77, dtype=I32, device="cuda")
    acc = torch.full((batch + 1,), -77, dtype=I32, device="cuda")
    kept = dlen if alias else torch.full((batch + 1,), -77, dtype=I32, device="cuda")
    fvk.verify_drafts(dp.data_ptr(), dq.data_ptr() if dq is not None else 0, tok.data_ptr(), dcu.data_ptr(), dlen.data_ptr(), du.data_ptr(),
                      dv.data_ptr(), out.data_ptr(), acc.data_ptr(), kept.data_ptr(), n if n_tokens is None else n_tokens, batch, vocab, _stream(),
                      p_stride=vocab + p_pad, q_stride=vocab + q_pad)
    torch.cuda.synchronize()
    assert acc[batch] == -77 and (alias or kept[batch] == -77)
    return out.tolist(), acc[:batch].tolist(), kept[:batch].tolist()


def check(p, q, tokens, cu, lens, u, v, **kw):
    out, acc, kept = run(p, q, tokens, cu, lens, u, v, **kw)
    want, wacc, wkept = R.verify(p, q, tokens, cu, lens, u, v)
    assert acc == wacc and kept == wkept
    assert out == [-77 if w is None else w for w in want] + [-77] * 5


@pytest.mark.parametrize("batch,drafts,vocab", [(1, 0, 1), (1, 4, 5), (3, 2, 31), (2, 33, 100), (5, 70, 64), (40, 3, 513), (1, 4, 50257), (6, 5, 4097),
                                                (300, 1, 1000), (9, 8, 33333), (2, 3, 262144), (700, 2, 200)])
@pytest.mark.parametrize("with_q", [True, False])
def test_verify(batch, drafts, vocab, with_q):
    """Sums in 64 bits of fp32 values: two orders differ by 2^-50 or so, and a random number that close to a border has not been drawn."""
    rng = np.random.default_rng(batch + drafts + vocab)
    rows = [int(rng.integers(0, drafts + 2)) if b else drafts + 1 for b in range(batch)]
    cu = np.concatenate([[0], np.cumsum(rows)])
    n = int(cu[-1]) + 3                                              # rows behind the last sequence
    p = rows_of(rng, n, vocab, 0.3)
    q = rows_of(rng, n, vocab) if with_q else None
    if with_q and vocab > 4:                                         # drafts near the target: many stand
        q = ((p.astype(np.float64) + 0.1 * q) / 1.1).astype(np.float32)
    src = q if with_q else p
    tokens = np.array([0] + [int(rng.choice(vocab, p=r.astype(np.float64) / r.astype(np.float64).sum())) for r in src[:-1]])
    tokens[1 + int(rng.integers(n - 1)) if n > 1 else 0] = vocab
    lens = rng.integers(drafts + 1, 5000, batch)
    u, v = rng.random(n, dtype=np.float32), rng.random(batch, dtype=np.float32)
    check(p, q, tokens.tolist(), cu.tolist(), lens.tolist(), u, v, p_pad=int(vocab % 5), q_pad=int(vocab % 3))
    check(p, q, tokens.tolist(), cu.tolist(), lens.tolist(), u, v, alias=True)


def test_verify_borders():
    """Exact borders: sums of powers of two are exact in any order."""
    p = np.array([[0.5, 0.0, 0.25, 0.25]], np.float32)
    for v, want in ((0.0, 0), (0.49999997, 0), (0.5, 2), (0.75, 3), (0.99999994, 3), (1.0, 3), (-1.0, 0), (NAN, 0), (INF, 3)):
        assert run(p, None, [0], [0, 1], [9], [0.0], [v])[0][0] == want, v
    lead = np.zeros((1, 70000), np.float32)
    lead[0, 69999], lead[0, 3] = 0.5, 0.5
    for v, want in ((0.0, 3), (0.5, 69999), (0.25, 3), (1.0, 69999)):
        assert run(lead, None, [0], [0, 1], [9], [0.0], [v])[0][0] == want
    even = np.full((1, 65536), 2.0 ** -16, np.float32)
    for v in (0.0, 2.0 ** -16, 0.25, 0.5, 4097 / 65536, 0.75 - 2.0 ** -16, 1 - 2.0 ** -16):
        assert run(even, None, [0], [0, 1], [9], [0.0], [v])[0][0] == int(v * 65536)
    # a probability that equals u q does not stand; u 0 against q 0 neither where p is 0
    p = np.array([[0.5, 0.5, 0.0, 0.0]] * 2, np.float32)
    q = np.array([[0.25, 0.75, 0.0, 0.0]] * 2, np.float32)
    assert run(p, q, [0, 1], [0, 2], [9], [0.6666666, 0.0], [0.3])[1] == [1]
    assert run(p, q, [0, 1], [0, 2], [9], [np.float32(2 / 3) + np.float32(1e-6), 0.0], [0.3])[:2] == ([0, -1, -77, -77, -77, -77, -77], [0])
    half = np.array([[0.5, 0.5, 0.0, 0.0]] * 2, np.float32)
    assert run(p, half, [0, 1], [0, 2], [9], [1.0, 0.0], [0.7])[:2] == ([1, -1, -77, -77, -77, -77, -77], [0])     # nothing left of p - q: p
    assert run(p, q, [0, 2], [0, 2], [9], [0.0, 0.0], [0.9])[1] == [0]
    assert run(p, None, [0, 0], [0, 2], [9], [0.5, 0.0], [0.9])[:2] == ([1, -1, -77, -77, -77, -77, -77], [0])     # p without that token
    # no probability at all; tokens outside; malformed offsets
    none = np.zeros((3, 40), np.float32)
    assert run(none, None, [0, 1, 2], [0, 3], [9], [0.0] * 3, [0.5]) == ([-1, -1, -1] + [-77] * 5, [0], [7])
    ok = np.full((4, 40), 0.025, np.float32)
    assert run(ok, None, [0, -1, 3, 4], [0, 4], [9], [0.0] * 4, [0.5])[1] == [0]
    assert run(ok, None, [0, 40, 3, 4], [0, 4], [9], [0.0] * 4, [0.5])[1] == [0]
    for cu in ([0, 5], [-1, 2], [2, 1], [3, 3]):
        assert run(ok, None, [0, 1, 2, 3], cu, [9], [0.0] * 4, [0.5]) == ([-77] * 9, [0], [9]), cu


def test_verify_without_rows_and_two_calls_at_once():
    from flashrt_b200 import flash_rt_kernels as fvk
    z = torch.zeros(4, dtype=I32, device="cuda")
    f = torch.zeros(4, device="cuda")
    acc, kept = torch.full((3,), 9, dtype=I32, device="cuda"), torch.full((3,), 9, dtype=I32, device="cuda")
    lens = torch.tensor([5, 6, 7], dtype=I32, device="cuda")
    fvk.verify_drafts(0, 0, 0, z.data_ptr(), lens.data_ptr(), 0, f.data_ptr(), 0, acc.data_ptr(), kept.data_ptr(), 0, 3, 100, _stream())
    torch.cuda.synchronize()
    assert acc.tolist() == [0, 0, 0] and kept.tolist() == [5, 6, 7]
    rng = np.random.default_rng(3)
    n, vocab = 64, 20000
    p, q = torch.tensor(rows_of(rng, n, vocab)).cuda(), torch.tensor(rows_of(rng, n, vocab)).cuda()
    tokens = q.argmax(1).roll(1).to(I32)
    cu = torch.arange(0, n + 1, 4, dtype=I32, device="cuda")
    u, v = torch.rand(n, device="cuda"), torch.rand(16, device="cuda")
    lens = torch.full((16,), 50, dtype=I32, device="cuda")
    want = R.verify(p.cpu().numpy(), q.cpu().numpy(), tokens.tolist(), cu.tolist(), lens.tolist(), u.cpu().numpy(), v.cpu().numpy())
    sides = [torch.cuda.Stream() for _ in range(3)]
    outs = [[torch.zeros(k, dtype=I32, device="cuda") for k in (n, 16, 16)] for _ in sides]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, o in zip(sides, outs):
            with torch.cuda.stream(s):
                fvk.verify_drafts(p.data_ptr(), q.data_ptr(), tokens.data_ptr(), cu.data_ptr(), lens.data_ptr(), u.data_ptr(), v.data_ptr(),
                                  o[0].data_ptr(), o[1].data_ptr(), o[2].data_ptr(), n, 16, vocab, _stream())
    torch.cuda.synchronize()
    for o in outs:
        assert tuple(x.tolist() for x in o) == want


def test_greedy_rows_are_the_argmax():
    """Temperature zero: drafted tokens stand as long as they are the target's largest, the next is the largest, whatever the random numbers."""
    from flashrt_b200 import flash_rt_kernels as fvk
    vocab, n = 3001, 6
    x = torch.randn(n, vocab, generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    p = softmax(x, torch.zeros(n).cuda()).numpy()
    best = x.float().argmax(1).tolist()
    assert fvk is not None
    for wrong in range(6):
        tokens = [9] + best[:5]
        if wrong < 5:
            tokens[wrong + 1] = (best[wrong] + 1) % vocab
        for q in (None, p):
            out, acc, kept = run(p, q, tokens, [0, 6], [50], [0.999] * 6, [0.999])
            assert acc == [wrong] and kept == [50 - 5 + wrong] and out[:6] == best[:wrong + 1] + [-1] * (5 - wrong)


def test_two_streams_and_a_graph():
    from flashrt_b200 import flash_rt_kernels as fvk
    rng = np.random.default_rng(1)
    batch, drafts, vocab = 12, 3, 9001
    n = batch * (drafts + 1)
    x = torch.randn(n, vocab, generator=torch.Generator().manual_seed(4)).mul_(3).cuda()
    t, p = torch.full((n,), 0.7).cuda(), torch.empty(n, vocab, device="cuda")
    tok, cu = torch.zeros(n, dtype=I32, device="cuda"), torch.arange(0, n + 1, drafts + 1, dtype=I32, device="cuda")
    lens, u, v = torch.full((batch,), 100, dtype=I32, device="cuda"), torch.zeros(n, device="cuda"), torch.zeros(batch, device="cuda")
    out, acc, kept = (torch.empty(k, dtype=I32, device="cuda") for k in (n, batch, batch))

    def step():
        fvk.softmax_rows(x.data_ptr(), p.data_ptr(), n, vocab, _stream(), temperature=t.data_ptr(), in_f32=True)
        fvk.verify_drafts(p.data_ptr(), 0, tok.data_ptr(), cu.data_ptr(), lens.data_ptr(), u.data_ptr(), v.data_ptr(), out.data_ptr(),
                          acc.data_ptr(), kept.data_ptr(), n, batch, vocab, _stream())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.synchronize()
    for _ in range(3):
        x.normal_().mul_(3)
        u.copy_(torch.tensor(rng.random(n, dtype=np.float32)))
        v.copy_(torch.tensor(rng.random(batch, dtype=np.float32)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = R.verify(p.cpu().numpy(), None, tok.tolist(), cu.tolist(), lens.tolist(), u.cpu().numpy(), v.cpu().numpy())
        assert (out.tolist(), acc.tolist(), kept.tolist()) == want

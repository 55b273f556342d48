"""Probabilities where logits lie further apart than the largest number, or temperatures are as large as numbers get, against 64 bits."""
import pytest
import torch

import decode_ref as R

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
INF = float("inf")


def softmax(x, t):
    from flashrt_b200 import flash_rt_kernels as fvk
    rows, vocab = x.shape
    p = torch.full((rows, vocab), -3.0, device="cuda")
    fvk.softmax_rows(x.data_ptr(), p.data_ptr(), rows, vocab, torch.cuda.current_stream().cuda_stream, temperature=t.data_ptr(),
                     in_f32=x.dtype == F32)
    torch.cuda.synchronize()
    assert fvk._lib.call_status("frt_b200_gemm_status", 1) == 0
    return p.cpu()


# a CTA a row; clusters; clusters that stay; rows that are not held, one CTA in eight without a large entry
@pytest.mark.parametrize("rows,vocab", [(20, 33), (20, 9000), (300, 50257), (20, 50257), (20, 300001)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_logits_further_apart_than_the_largest_number(rows, vocab, dtype):
    g = torch.Generator().manual_seed(vocab)
    big = float(torch.finfo(dtype).max)
    kinds = [(-big, big), (-0.9 * big, 0.5 * big), (-big, 2.0 ** 103), (-big, 2.0 ** 101), (-0.5 * big, -0.25 * big)]
    temps = [INF, 1e38, 2.5e37, 3.4e38, 1.0]
    x, t = torch.empty(rows, vocab), torch.empty(rows)
    for r in range(rows):
        lo, hi = kinds[r % 5]
        x[r] = lo
        x[r, torch.randperm(vocab, generator=g)[:max(1, vocab // 3)]] = hi
        x[r, : vocab // 8] = lo                                  # the first CTA of eight has no large entry
        if r % 3 == 1:
            x[r, vocab // 2:] = -INF
        if r % 4 == 2:
            x[r, vocab - 1] = hi * 0.5
        t[r] = temps[r // 5 % 5 if r >= 5 else r]
    x, t = x.to(dtype).cuda(), t.cuda()
    p = softmax(x, t)
    want = R.softmax_rows(x.cpu(), t.cpu())
    assert not p.isnan().any()
    # the argument d c: a rounding of each half, of c (2^-22 of it where T is so large that c lies below the normal numbers) and of the product,
    # three of 2^-24 beside it, times an argument of at most 7 where the weight counts (2 x 3.4e38 / 1e38) or 28 (2.5e37); the exponential and
    # the factor 2^-22 each, their product and the quotient 2^-24 each; the sum of V weights, V / 4096 values a thread and 20 steps behind
    rel = 28 * (2.0 ** -22 + 3 * 2.0 ** -24) + 2 * 2.0 ** -22 + 2 * 2.0 ** -24 + 2.0 ** -24 * (vocab / 4096 + 64)
    off = (p.to(F64) - want).abs()
    assert (off <= want * rel + 2.0 ** -120).all(), (off / (want * rel + 2.0 ** -120)).max()
    spread = [r for r in range(rows) if r % 5 < 2 and float(t[r]) >= 1e38]
    assert all(len(p[r].unique()) >= 2 or t[r] == INF for r in spread) and spread       # far ones count there, they are not all or nothing


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_probabilities_between_the_rows_of_their_logits(dtype):
    """Rows of one buffer: logits, probabilities right behind them, a gap.  Only what shares bytes is refused."""
    from flashrt_b200 import flash_rt_kernels as fvk
    rows, vocab = 9, 1000
    es = 2 if dtype == BF16 else 4
    step = vocab * (es + 4) + 16
    buffer = torch.full((rows * step,), 0x5a, dtype=torch.uint8, device="cuda")
    rows_of = buffer.view(rows, step)
    x = (torch.randn(rows, vocab, generator=torch.Generator().manual_seed(1)) * 3).to(dtype).cuda()
    rows_of[:, :vocab * es] = x.view(torch.uint8)
    t = torch.full((rows,), 0.8, device="cuda")
    args = dict(temperature=t.data_ptr(), in_f32=dtype == F32, in_stride=step // es, out_stride=step // 4)
    stream = torch.cuda.current_stream().cuda_stream
    with pytest.raises(fvk.KernelError):
        fvk.softmax_rows(buffer.data_ptr(), buffer.data_ptr() + vocab * es - 4, rows, vocab, stream, **args)
    fvk.softmax_rows(buffer.data_ptr(), buffer.data_ptr() + vocab * es, rows, vocab, stream, **args)
    torch.cuda.synchronize()
    assert torch.equal(rows_of[:, vocab * es:-16].contiguous().view(F32).cpu(), softmax(x, t))
    assert torch.equal(rows_of[:, :vocab * es].contiguous().view(dtype), x) and (rows_of[:, -16:] == 0x5a).all()
    assert fvk._lib.call_status("frt_b200_gemm_status", 1) == 0

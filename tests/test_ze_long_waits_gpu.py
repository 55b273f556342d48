"""Launches that are resident behind a kernel of more than two seconds, and one that takes longer than that itself: no bounded wait counts
the time that the kernel in front, or the work, takes."""
import pytest
import torch

import decode_ref as R

pytestmark = pytest.mark.gpu
BF16, E4M3, F32, F64, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.float32, torch.float64, torch.int32

# lets the next kernel start at once and ends after `ms` (or a bounded number of looks)
LONG = r"""
extern "C" __global__ void lets_the_next_start(int ms) {
    asm volatile("griddepcontrol.launch_dependents;");
    unsigned long long now, start;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(start));
    for (int i = 0; i < 10000000; ++i) {
        asm volatile("nanosleep.u32 2000;");
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
        if (now - start > 1000000ull * ms) return;
    }
}
"""


@pytest.fixture(scope="module")
def long_kernel():
    kernel = torch.cuda._compile_kernel(LONG, "lets_the_next_start")

    def launch():
        kernel(grid=(1, 1, 1), block=(32, 1, 1), args=[2300])
    return launch


def _stream():
    return torch.cuda.current_stream().cuda_stream


def operands(m, n, k, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    a, w = ((torch.randn(r, k, generator=g, device="cuda") * 100).clamp(-448, 448).to(E4M3) for r in (m, n))
    return a, w, torch.rand(k // 128, m, generator=g, device="cuda"), torch.rand((n + 127) // 128, k // 128, generator=g, device="cuda")


def run(job, out):
    from flashrt_b200 import flash_rt_kernels as fvk
    a, w, sa, sw = job
    fvk.GemmRunner().fp8_block_nt(a.data_ptr(), w.data_ptr(), out.data_ptr(), a.shape[0], w.shape[0], a.shape[1], sa.data_ptr(), sw.data_ptr(),
                                  _stream(), d_f32=out.dtype == F32)


@pytest.mark.parametrize("m,n,k", [(3, 640, 1024), (96, 4096, 4096), (300, 1000, 1024)])
def test_products_behind_a_long_kernel(m, n, k, long_kernel):
    from flashrt_b200 import flash_rt_kernels as fvk
    job = operands(m, n, k, m)
    want, got = (torch.full((m, n), float("nan"), device="cuda") for _ in range(2))
    run(job, want)
    torch.cuda.synchronize()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    long_kernel()
    run(job, got)
    end.record()
    torch.cuda.synchronize()
    assert begin.elapsed_time(end) > 2250
    assert fvk._lib.call_status("frt_b200_gemm_status", 1) == 0
    assert torch.equal(got, want) and want.isfinite().all()


def test_a_product_of_more_than_two_seconds():
    """65536 x 65536 x 524288, 4.5e15 operations: more than two seconds at any rate of this GPU's products with these scales.  Codes repeat
    along K, scales do not; a hundred entries against 64 bits, and no tile left out."""
    from flashrt_b200 import flash_rt_kernels as fvk
    m = n = 1 << 16
    k, period = 1 << 19, 1 << 10
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        torch.cuda.empty_cache()
    g = torch.Generator("cuda").manual_seed(1)
    a, w = (torch.randint(0, 0x7f, (r, period), generator=g, device="cuda", dtype=torch.uint8)
            .add_(torch.randint(0, 2, (r, period), generator=g, device="cuda", dtype=torch.uint8).mul_(0x80)).repeat(1, k // period) for r in (m, n))
    sa, sw = torch.rand(k // 128, m, generator=g, device="cuda"), torch.rand(n // 128, k // 128, generator=g, device="cuda")
    out = torch.full((m, n), float("nan"), dtype=BF16, device="cuda")
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    run((a, w, sa, sw), out)
    end.record()
    torch.cuda.synchronize()
    assert fvk._lib.call_status("frt_b200_gemm_status", 1) == 0
    assert begin.elapsed_time(end) > 2000                            # otherwise this test is about nothing
    assert not any(out[i:i + 8192].isnan().any() for i in range(0, m, 8192))
    rows, cols = [0, 1, 127, 128, 4000, 33000, 50001, 65407, 65408, m - 1], [0, 3, 255, 256, 9999, 32768, 40000, 65279, 65280, n - 1]
    x, y = (t[i].view(E4M3).to(F64) for t, i in ((a, rows), (w, cols)))
    x *= sa[:, rows].to(F64).t().repeat_interleave(128, 1)
    y *= sw[[c // 128 for c in cols]].to(F64).repeat_interleave(128, 1)
    want, size = x @ y.t(), x.abs() @ y.abs().t()
    # a block's 128 additions in the tensor core (2^-23 of its magnitudes each), a rounding of each of k / 128 fma, two of scales; half a bf16 step
    bound = size * (128 * 2.0 ** -23 + (k // 128 + 2) * 2.0 ** -24)
    bound = bound * (1 + 2.0 ** -8) + want.abs() * 2.0 ** -8
    assert ((out[rows][:, cols].to(F64) - want).abs() <= bound).all()


def _logits(rows, vocab, dtype):
    x = torch.randn(rows, vocab, generator=torch.Generator("cuda").manual_seed(rows), device="cuda") * 3
    return x.to(dtype)


@pytest.mark.parametrize("rows,vocab,dtype", [(1, 50257, BF16), (300, 50257, F32), (40, 131072, F32), (20, 150001, BF16)])
def test_probabilities_and_verification_behind_a_long_kernel(rows, vocab, dtype, long_kernel):
    """Clusters of a row, clusters that stay, rows that are not held; a sequence of all rows, whose last tokens are the likeliest."""
    from flashrt_b200 import flash_rt_kernels as fvk
    x = _logits(rows, vocab, dtype)
    p, q = (torch.full((rows, vocab), float("nan"), device="cuda") for _ in range(2))
    cu, lens = torch.tensor([0, rows], dtype=I32, device="cuda"), torch.tensor([rows + 7], dtype=I32, device="cuda")
    tokens = torch.cat([torch.zeros(1, dtype=I32, device="cuda"), x.float().argmax(1)[:-1].to(I32)])
    u, v = torch.full((rows,), 0.001, device="cuda"), torch.full((1,), 0.6, device="cuda")
    outs = [torch.full((rows + 2,), -9, dtype=I32, device="cuda") for _ in range(2)]

    def step(probs, out):
        fvk.softmax_rows(x.data_ptr(), probs.data_ptr(), rows, vocab, _stream(), in_f32=dtype == F32)
        fvk.verify_drafts(probs.data_ptr(), 0, tokens.data_ptr(), cu.data_ptr(), lens.data_ptr(), u.data_ptr(), v.data_ptr(), out.data_ptr(),
                          out.data_ptr() + 4 * rows, out.data_ptr() + 4 * rows + 4, rows, 1, vocab, _stream())
    step(p, outs[0])
    torch.cuda.synchronize()
    long_kernel()
    step(q, outs[1])
    torch.cuda.synchronize()
    assert fvk._lib.call_status("frt_b200_gemm_status", 1) == 0
    assert torch.equal(p, q) and p.isfinite().all() and torch.equal(*outs) and (outs[0][:1] >= 0).all()
    want, accepted, kept = R.verify(p.cpu().numpy(), None, tokens.tolist(), [0, rows], [rows + 7], u.tolist(), v.tolist())
    assert outs[0].tolist() == want + accepted + kept

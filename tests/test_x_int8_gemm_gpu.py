"""8-bit integer products and their quantiser against 64-bit integers and the fp32 operations of the header."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32, F64, I64 = torch.bfloat16, torch.float32, torch.float64, torch.int64


def _stream():
    return torch.cuda.current_stream().cuda_stream


def quantize(x, stride=0, rows=None, dim=None):
    from flashrt_b200 import flash_rt_kernels as fvk
    rows, dim = rows or x.shape[0], dim or x.shape[1]
    q = torch.full((rows + 1, dim), 99, dtype=torch.int8, device="cuda")
    s = torch.full((rows + 1,), -1.0, device="cuda")
    fvk.quantize_int8_rows(x.data_ptr(), q.data_ptr(), s.data_ptr(), rows, dim, _stream(), in_stride=stride)
    torch.cuda.synchronize()
    assert (q[rows] == 99).all() and s[rows] == -1                  # nothing behind the last row
    return q[:rows], s[:rows]


def quantized(x):
    """The header's fp32 operations, each rounded once: code for code."""
    x = x.cpu().float()
    s = (torch.where(x.isfinite(), x.abs(), 0.0).amax(1) / 127.0).clamp_min(1e-12)
    q = torch.round(x * (1.0 / s)[:, None]).nan_to_num(0.0).clamp(-127, 127)
    return q.to(torch.int8), s


@pytest.mark.parametrize("rows,dim", [(1, 16), (1, 2048), (3, 48), (7, 1024), (5, 1040), (130, 2064), (9, 4096), (2, 8192), (3, 8208),
                                      (4, 16384), (2, 40000), (2000, 128), (5000, 1024), (1300, 4112)])
def test_quantize_rows(rows, dim):
    g = torch.Generator().manual_seed(rows + dim)
    x = (torch.randn(rows, dim, generator=g) * torch.exp(torch.randn(rows, 1, generator=g) * 3)).to(BF16)
    x[rows // 2] = 0
    q, s = quantize(x.cuda())
    qw, sw = quantized(x)
    assert torch.equal(s.cpu(), sw) and torch.equal(q.cpu(), qw)
    v = q.cpu().to(F64) * s.cpu().to(F64)[:, None]
    assert ((v - x.to(F64)).abs() <= s.cpu().to(F64)[:, None] * (0.5 + 2.0 ** -15)).all()      # half a step


def test_quantize_strided_and_special_values():
    x = torch.randn(6, 512, generator=torch.Generator().manual_seed(0)).to(BF16)
    x[0, 3], x[1, 4], x[1, 5], x[2, 6] = float("inf"), -float("inf"), 1e30, float("nan")
    x[3] = float("nan")
    x[4] = 1e-30
    q, s = quantize(x.cuda(), stride=512, rows=6, dim=256)
    qw, sw = quantized(x[:, :256])
    assert torch.equal(q.cpu(), qw) and torch.equal(s.cpu(), sw)
    assert q[0, 3] == 127 and q[1, 4] == -127 and q[2, 6] == 0 and (q[3] == 0).all()
    wide = torch.randn(9, 328, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    q, s = quantize(wide, stride=328, rows=9, dim=320)
    qw, sw = quantized(wide[:, :320])
    assert torch.equal(q.cpu(), qw) and torch.equal(s.cpu(), sw)


def product(a, w, ts, cs, bias=None, pdl=False):
    from flashrt_b200 import flash_rt_kernels as fvk
    m, k = a.shape
    n = w.shape[0]
    out = torch.full((m * n + 64,), -7.0, dtype=BF16, device="cuda")
    fvk.GemmRunner().int8_nt(a.data_ptr(), w.data_ptr(), out.data_ptr(), m, n, k, ts.data_ptr(), cs.data_ptr(), _stream(),
                             bias=bias.data_ptr() if bias is not None else 0, pdl=pdl)
    torch.cuda.synchronize()
    assert fvk._lib.call_status("frt_b200_gemm_status", 1) == 0
    assert (out[m * n:] == -7.0).all()
    return out[:m * n].view(m, n)


def check(m, n, k, seed=0, bias=True, extreme=False, pdl=False):
    """Exact integer sums (64-bit here); then fp32(sum) * ts * cs (+ bias in one fma) and one rounding: without a bias every bit, with
    one half a bf16 step (2^-8) and the three fp32 roundings (3 x 2^-24 of the product)."""
    g = torch.Generator(device="cuda").manual_seed(seed + m + n + k)
    if extreme:
        a = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
        w = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    else:
        a = torch.randint(-128, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
        w = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    ts, cs = (torch.rand(x, generator=g, device="cuda") * 0.01 + 1e-4 for x in (m, n))
    b = (torch.randn(n, generator=g, device="cuda") * 20).to(BF16) if bias else None
    out = product(a, w, ts, cs, b, pdl)
    acc = (a.to(F64) @ w.to(F64).T)                                  # integers below 2^53
    plain = acc.to(F32) * ts[:, None] * cs
    if not bias:
        assert torch.equal(out, plain.to(BF16))
        return
    want = acc * ts.to(F64)[:, None] * cs.to(F64)
    err = (out.to(F64) - (want + b.to(F64))).abs()
    assert (err <= (want + b.to(F64)).abs() * 2.0 ** -8 + want.abs() * 3 * 2.0 ** -24).all()


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 64, 65, 100, 128])
@pytest.mark.parametrize("n,k", [(128, 128), (2560, 2048), (333, 144)])
def test_few_rows(m, n, k):
    check(m, n, k, bias=False)


@pytest.mark.parametrize("m", [129, 255, 256, 257, 400, 817])
@pytest.mark.parametrize("n,k", [(64, 64), (257, 400), (1000, 16), (2048, 1040)])
def test_more_rows(m, n, k):
    check(m, n, k, bias=False)


@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 7, 4096), (5, 130, 16384), (128, 1, 272), (300, 1, 128), (129, 33, 48), (3000, 515, 512),
                                   (2049, 4100, 256), (700, 9000, 128)])
def test_odd_sizes_with_bias(m, n, k):
    check(m, n, k)
    check(m, n, k, bias=False)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_longest_sums(m):
    """The largest magnitude of 32-bit sums: 131056 products of 2^14."""
    check(m, 160, 131056, bias=False, extreme=True)
    check(m, 160, 131056, bias=False)


@pytest.mark.parametrize("m,n,k", [(817, 2048, 16384), (300, 2048, 2048), (129, 256, 8192), (256, 4096, 4096), (513, 1000, 10000), (400, 333, 16384),
                                   (200, 8192, 1024), (1024, 1024, 1040)])
def test_shared_sums(m, n, k):
    """Few tiles and a long K: two or four pairs share a tile's sum."""
    check(m, n, k, bias=False)
    check(m, n, k)


def test_many_tiles():
    check(4096, 8192, 256, bias=False)
    check(96, 32768, 2048, bias=False, pdl=True)


def test_rows_are_independent_of_the_others():
    """A row's result does not depend on how many rows come with it (integer sums): every kernel gives the same bits."""
    g = torch.Generator(device="cuda").manual_seed(4)
    a = torch.randint(-128, 128, (600, 784), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-128, 128, (500, 784), generator=g, device="cuda", dtype=torch.int8)
    ts, cs = (torch.rand(x, generator=g, device="cuda") for x in (600, 500))
    b = torch.randn(500, generator=g, device="cuda").to(BF16)
    full = product(a, w, ts, cs, b)
    for m in (1, 16, 30, 64, 128, 129, 300):
        assert torch.equal(product(a[:m], w, ts, cs, b), full[:m]), m


def test_captured_pair_of_quantiser_and_product():
    from flashrt_b200 import flash_rt_kernels as fvk
    m, n, k = 50, 1024, 4096
    x = torch.zeros(m, k, dtype=BF16, device="cuda")
    w = torch.randint(-128, 128, (n, k), device="cuda", dtype=torch.int8)
    cs = torch.rand(n, device="cuda") * 1e-3
    q, s, out = torch.zeros(m, k, dtype=torch.int8, device="cuda"), torch.zeros(m, device="cuda"), torch.zeros(m, n, dtype=BF16, device="cuda")
    gemm = fvk.GemmRunner()

    def step():
        fvk.quantize_int8_rows(x.data_ptr(), q.data_ptr(), s.data_ptr(), m, k, _stream())
        gemm.int8_nt(q.data_ptr(), w.data_ptr(), out.data_ptr(), m, n, k, s.data_ptr(), cs.data_ptr(), _stream(), pdl=True)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (1, 2):
        x.copy_(torch.randn(m, k, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        qw, sw = quantized(x)
        want = ((qw.cuda().to(F64) @ w.to(F64).T).to(F32) * sw.cuda()[:, None] * cs).to(BF16)
        assert torch.equal(q.cpu(), qw) and torch.equal(out, want)

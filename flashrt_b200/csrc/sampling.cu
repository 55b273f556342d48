// Probabilities of logits, and the verification of drafted tokens against them.
//
// Stand behind the products that make logits and in front of the paged cache's lengths; no counterpart in the reference.
//
// Both read rows of a vocabulary once: a row belongs to a cluster of 1 to 8 CTAs that hold it (softmax: in registers) and exchange a few
// numbers through distributed shared memory.  Rows start anywhere (odd vocabularies), so a lane reads one value at a time, 32
// neighbours a warp; enough of them are under way for that not to matter.
#include "common.cuh"
#include "tc05.cuh"
#include "flashrt_b200.h"

namespace frt {
namespace smp {

constexpr int THREADS = 512, WARPS = THREADS / 32;

__device__ __forceinline__ uint64_t dsmem_ld_u64(uint32_t cluster_addr) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(cluster_addr) : "memory");
    return v;
}
__device__ __forceinline__ uint4 dsmem_ld_u32x4(uint32_t cluster_addr) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(cluster_addr) : "memory");
    return v;
}
__device__ __forceinline__ float load_logit(const void* row, int i, bool f32) {
    const float x = f32 ? static_cast<const float*>(row)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(row)[i]);
    return x == x ? x : -INFINITY;                           // NaN: masked
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ------------------------------------------------------------------------------------------------ softmax
//   p = exp((x - max) / T) / sum;  T not above zero: one on the first of the largest;  nothing but -infinity and NaN: zeros.
// A CTA's part: exponentials against its own maximum, then one exchange of (maximum, sum) in the cluster, and a factor that takes them to
// the row's.  E values a thread; HELD false: rows too long for that are read twice.
struct SoftmaxParams {
    const void* x;
    float* p;
    const float* temperature;
    long long in_stride, out_stride;
    int vocab, ctas;             // ctas: of a row
};

template <int E, bool F32, bool HELD>
__global__ void __launch_bounds__(THREADS)
softmax_rows_kernel(SoftmaxParams p) {
    __shared__ float part[WARPS], part2[WARPS];
    __shared__ int part3[WARPS];
    __shared__ uint4 mine;                                   // maximum, sum, index of the first of the largest
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ctas = p.ctas, rank = (int)(blockIdx.x % (unsigned)ctas);
    const long long row = blockIdx.x / (unsigned)ctas;
    const int lo = (int)((long long)p.vocab * rank / ctas), hi = (int)((long long)p.vocab * (rank + 1) / ctas), len = hi - lo;
    const void* x = static_cast<const uint8_t*>(p.x) + (row * p.in_stride + lo) * (F32 ? 4 : 2);
    float* out = p.p + row * p.out_stride + lo;
    const float T = p.temperature ? p.temperature[row] : 1.0f;
    const bool hot = !(T > 0.0f);
    const float c = hot ? 0.0f : __fdiv_rn(1.4426950408889634f, T);
    float v[E], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int at = tid + i * THREADS;
        v[i] = at < len ? load_logit(x, at, F32) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) top = fmaxf(top, v[i]);
    if (!HELD)
        for (int at = tid + E * THREADS; at < len; at += THREADS) top = fmaxf(top, load_logit(x, at, F32));
    top = warp_max_butterfly(top);
    if (lane == 0) part[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, part[w]);
    // against this CTA's maximum; where that is infinite, the infinite ones share the mass
    auto weight = [&](float y) { return y == top ? 1.0f : exp2_approx(fmaxf(__fmul_rn(__fsub_rn(y, top), c), -3.0e38f)); };
    float sum = 0.0f;
    int first = 0x7fffffff;
    if (hot) {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (v[i] == top && tid + i * THREADS < len) first = min(first, lo + tid + i * THREADS);
        if (!HELD)
            for (int at = tid + E * THREADS; at < len; at += THREADS)
                if (load_logit(x, at, F32) == top) first = min(first, lo + at);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            v[i] = tid + i * THREADS < len ? weight(v[i]) : 0.0f;
            sum += v[i];
        }
        if (!HELD)
            for (int at = tid + E * THREADS; at < len; at += THREADS) sum += weight(load_logit(x, at, F32));
    }
    first = __reduce_min_sync(0xffffffffu, first);
    sum = warp_sum_butterfly(sum);
    if (lane == 0) {
        part2[warp] = sum;
        part3[warp] = first;
    }
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        sum += part2[w];
        first = min(first, part3[w]);
    }
    float factor;
    bool nothing;
    if (ctas > 1) {
        if (tid == 0) mine = make_uint4(__float_as_uint(top), __float_as_uint(sum), (uint32_t)first, 0);
        __syncwarp();
        tc::cluster_sync_all();
        uint4 all[8];
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < ctas) all[r] = dsmem_ld_u32x4(tc::dsmem_map(tc::smem_u32(&mine), (uint32_t)r));
        float m = -INFINITY, total = 0.0f;
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < ctas) m = fmaxf(m, __uint_as_float(all[r].x));
        int f = 0x7fffffff;
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < ctas) {
                const float x_r = __uint_as_float(all[r].x);
                const float w = x_r == m ? 1.0f : exp2_approx(fmaxf(__fmul_rn(__fsub_rn(x_r, m), c), -3.0e38f));
                total = __fmaf_rn(__uint_as_float(all[r].y), w, total);
                if (x_r == m) f = min(f, (int)all[r].z);
            }
        first = f;
        nothing = m == -INFINITY;
        const float w = top == m ? 1.0f : exp2_approx(fmaxf(__fmul_rn(__fsub_rn(top, m), c), -3.0e38f));
        factor = __fdiv_rn(w, total);
        __syncwarp();
        tc::cluster_sync_all();                              // nobody leaves while its numbers are read
    } else {
        nothing = top == -INFINITY;
        factor = __fdiv_rn(1.0f, sum);
    }
    if (nothing) first = -1;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int at = tid + i * THREADS;
        if (at < len) out[at] = hot ? (lo + at == first ? 1.0f : 0.0f) : nothing ? 0.0f : __fmul_rn(v[i], factor);
    }
    if (!HELD)
        for (int at = tid + E * THREADS; at < len; at += THREADS)
            out[at] = hot ? (lo + at == first ? 1.0f : 0.0f) : nothing ? 0.0f : __fmul_rn(weight(load_logit(x, at, F32)), factor);
}

// ------------------------------------------------------------------------------------------------ verification
//   row t answers with token t + 1.  Drafted token d = tokens[t + 1] stands if u[t] q[t][d] < p[t][d] (exact in 64 bits: two products of 24).
//   At the first that does not: a token from max(p - q, 0) of that row, from p where nothing is left of it; if all stand, from p of
//   the last row.  The token is the first whose running sum is above v times the sum of all, in 64 bits.
// A warp has a run of neighbouring entries; the runs' sums of the whole cluster say which warp has the token, and that one reads its run
// again.
struct VerifyParams {
    const float *p, *q;
    long long p_stride, q_stride;
    const int *tokens, *cu, *lens;
    const float *u, *v;
    int *out, *accepted, *kept;
    int n_tokens, batch, vocab, ctas;
};

__device__ __forceinline__ double warp_scan(double x) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    return x;
}

__global__ void __launch_bounds__(THREADS)
verify_drafts_kernel(VerifyParams a) {
    __shared__ double sums[2 * WARPS];                       // of each warp's run: what is left of p, p
    __shared__ double all[2][8 * WARPS];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ctas = a.ctas, rank = (int)(blockIdx.x % (unsigned)ctas), b = (int)(blockIdx.x / (unsigned)ctas);
    const int first = a.cu[b], end = a.cu[b + 1];
    const int len = a.lens ? a.lens[b] : 0;
    const bool idle = first < 0 || end > a.n_tokens || end <= first;
    const int drafts = idle ? 0 : end - first - 1;
    int stood = 0;
    for (; stood < drafts; stood += 32) {
        const int i = stood + lane;
        bool stands = false;
        if (i < drafts) {
            const int t = first + i, d = a.tokens[t + 1];
            if (d >= 0 && d < a.vocab) {
                const float q = a.q ? a.q[t * a.q_stride + d] : 1.0f;
                stands = (double)a.u[t] * (double)q < (double)a.p[t * a.p_stride + d];
            }
        }
        const unsigned fails = __ballot_sync(0xffffffffu, !stands);
        if (fails) {
            stood = min(stood + __ffs(fails) - 1, drafts);
            break;
        }
    }
    stood = min(stood, drafts);
    if (rank == 0) {
        if (tid == 0) {
            a.accepted[b] = stood;
            if (a.kept) a.kept[b] = len - (drafts - stood);
        }
        if (!idle)
            for (int i = tid; i <= drafts; i += THREADS)
                if (i != stood) a.out[first + i] = i < stood ? a.tokens[first + i + 1] : -1;
    }
    if (idle) return;                                        // all CTAs of the cluster
    const int t = first + stood;
    const bool rejected = stood < drafts;
    const int drafted = rejected ? a.tokens[t + 1] : -1;
    const float* p = a.p + t * a.p_stride;
    const float* q = rejected && a.q ? a.q + t * a.q_stride : nullptr;
    const bool minus = rejected && !a.q;
    auto left = [&](int i, float x) {                        // what is left of p at entry i
        if (q) return fmax((double)x - (double)q[i], 0.0);
        return minus && i == drafted ? 0.0 : (double)x;
    };
    auto prob = [&](int i) { return fmaxf(p[i], 0.0f); };
    const int runs = ctas * WARPS, run = rank * WARPS + warp;
    const int lo = (int)((long long)a.vocab * run / runs), hi = (int)((long long)a.vocab * (run + 1) / runs);
    double sr = 0.0, sp = 0.0;
    int i = lo + lane;
    for (; i + 7 * 32 < hi; i += 8 * 32) {
        float x[8], y[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = prob(i + 32 * k);
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = q ? q[i + 32 * k] : minus && i + 32 * k == drafted ? x[k] : 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            sr += fmax((double)x[k] - (double)y[k], 0.0);
            sp += (double)x[k];
        }
    }
    for (; i < hi; i += 32) {
        const float x = prob(i);
        sr += left(i, x);
        sp += (double)x;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        sr += __shfl_xor_sync(0xffffffffu, sr, d);
        sp += __shfl_xor_sync(0xffffffffu, sp, d);
    }
    if (lane == 0) { sums[warp] = sr; sums[WARPS + warp] = sp; }
    if (ctas > 1) {
        __syncwarp();
        tc::cluster_sync_all();
    } else {
        __syncthreads();
    }
    for (int k = tid; k < 2 * runs; k += THREADS) {
        const int which = k >= runs, w = which ? k - runs : k;
        const uint32_t from = tc::smem_u32(&sums[which * WARPS + w % WARPS]);
        all[which][w] = ctas > 1 ? __longlong_as_double((long long)dsmem_ld_u64(tc::dsmem_map(from, (uint32_t)(w / WARPS)))) : sums[which * WARPS + w];
    }
    if (ctas > 1) {
        __syncwarp();
        tc::cluster_sync_all();                              // nobody leaves while its sums are read
    } else {
        __syncthreads();
    }
    // every warp: running sums of the runs, four a lane
    double s4[4], total = 0.0;
    int which = 0;
    for (; which < 2; ++which) {
        double x = 0.0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int w = lane * 4 + k;
            s4[k] = w < runs ? all[which][w] : 0.0;
            x += s4[k];
        }
        const double upto = warp_scan(x);
        total = __shfl_sync(0xffffffffu, upto, 31);
        double at = __shfl_up_sync(0xffffffffu, upto, 1);    // in front of this lane's runs
        if (lane == 0) at = 0.0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const double y = s4[k];
            s4[k] = at;                                      // in front of run lane * 4 + k
            at += y;
        }
        if (total > 0.0) break;
    }
    if (!(total > 0.0)) {                                    // no probability anywhere
        if (rank == 0 && tid == 0) a.out[t] = -1;
        return;
    }
    const float v0 = a.v[b], v = v0 > 0.0f ? fminf(v0, 0.99999994f) : 0.0f;
    const double target = (double)v * total;
    // the last run that starts at or below the target and is not empty
    int mine = -1;
    double start = 0.0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int w = lane * 4 + k;
        if (w < runs && s4[k] <= target && all[which][w] > 0.0) { mine = w; start = s4[k]; }
    }
    const int owner = __reduce_max_sync(0xffffffffu, mine);
    if (owner < 0 && run == 0 && lane == 0) a.out[t] = -1;   // infinite probabilities
    if (owner != run) return;
    start = __shfl_sync(0xffffffffu, start, owner >> 2);
    auto value = [&](int e) { return which ? (double)prob(e) : left(e, prob(e)); };
    // a lane sums a stretch of the run, then the warp walks over the stretch that has the token
    const int each = (hi - lo + 31) / 32, e0 = min(lo + lane * each, hi), e1 = min(e0 + each, hi);
    double x = 0.0;
    for (int e = e0; e < e1; ++e) x += value(e);
    const double upto = warp_scan(x);
    double front = __shfl_up_sync(0xffffffffu, upto, 1);
    if (lane == 0) front = 0.0;
    const unsigned has = __ballot_sync(0xffffffffu, x > 0.0 && start + front <= target);
    const int src = has ? 31 - __clz(has) : 0;
    start += __shfl_sync(0xffffffffu, front, src);
    const int s0 = __shfl_sync(0xffffffffu, e0, src), s1 = __shfl_sync(0xffffffffu, e1, src);
    int token = -1, last = -1;
    for (int base = s0; base < s1 && token < 0; base += 32) {
        const int e = base + lane;
        const double y = e < s1 ? value(e) : 0.0;
        const double z = warp_scan(y);
        const unsigned above = __ballot_sync(0xffffffffu, y > 0.0 && start + z > target), some = __ballot_sync(0xffffffffu, y > 0.0);
        if (above) token = base + __ffs(above) - 1;
        if (some) last = base + 31 - __clz(some);
        start += __shfl_sync(0xffffffffu, z, 31);
    }
    if (lane == 0) a.out[t] = token >= 0 ? token : last;     // roundings left the target behind the last one: that one
}

template <typename P>
static int launch(void (*kernel)(P), const P& p, unsigned ctas, unsigned rows, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas * rows);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    return e == cudaSuccess ? FRT_OK : FRT_CUDA_ERR(e);
}

template <bool F32>
static int launch_softmax(SoftmaxParams p, int rows, cudaStream_t st) {
    // CTAs of a row: enough to hold it, 32 values a thread; more where the rows leave SMs idle
    int ctas = 1;
    while (ctas < 8 && ((long long)ctas * THREADS * 32 < p.vocab || ((long long)rows * ctas * 2 <= device_sm_count() && ctas * THREADS * 4 < p.vocab))) ctas *= 2;
    const int each = (p.vocab + ctas - 1) / ctas;
    p.ctas = ctas;
    if (each <= 8 * THREADS) return launch(softmax_rows_kernel<8, F32, true>, p, ctas, rows, st);
    if (each <= 16 * THREADS) return launch(softmax_rows_kernel<16, F32, true>, p, ctas, rows, st);
    if (each <= 32 * THREADS) return launch(softmax_rows_kernel<32, F32, true>, p, ctas, rows, st);
    if (each <= 64 * THREADS) return launch(softmax_rows_kernel<64, F32, true>, p, ctas, rows, st);
    return launch(softmax_rows_kernel<32, F32, false>, p, ctas, rows, st);
}

}  // namespace smp
}  // namespace frt

static bool misaligned(const void* a, uintptr_t n) { return (reinterpret_cast<uintptr_t>(a) & (n - 1)) != 0; }

extern "C" int frt_b200_softmax_rows(const void* in, long long in_stride, float* out, long long out_stride, const float* temperature, int rows,
                                     int vocab, int flags, void* stream) {
    using namespace frt;
    if (rows < 0 || vocab < 0 || in_stride < vocab || out_stride < vocab) return FRT_ERR_INVALID;
    if (rows > 1 << 27 || vocab > 1 << 30) return FRT_ERR_UNSUPPORTED;
    if (rows == 0 || vocab == 0) return FRT_OK;
    const bool f32 = flags & 2;
    if (!in || !out || misaligned(in, f32 ? 4 : 2) || misaligned(out, 4) || misaligned(temperature, 4)) return FRT_ERR_INVALID;
    const smp::SoftmaxParams p = {in, out, temperature, in_stride, out_stride, vocab, 1};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return f32 ? smp::launch_softmax<true>(p, rows, st) : smp::launch_softmax<false>(p, rows, st);
}

extern "C" int frt_b200_verify_drafts(const float* target_probs, long long p_stride, const float* draft_probs, long long q_stride,
                                      const int* tokens, const int* cu_seqlens, const int* seq_lens, const float* u_accept,
                                      const float* u_sample, int* out_tokens, int* accepted, int* kept_lens, int n_tokens, int batch,
                                      int vocab, int flags, void* stream) {
    using namespace frt;
    (void)flags;
    if (n_tokens < 0 || batch < 0 || vocab < 1 || p_stride < vocab || (draft_probs && q_stride < vocab)) return FRT_ERR_INVALID;
    if (batch > 1 << 27 || vocab > 1 << 30) return FRT_ERR_UNSUPPORTED;
    if (batch == 0) return FRT_OK;
    if (!target_probs || !tokens || !cu_seqlens || !u_accept || !u_sample || !out_tokens || !accepted || (kept_lens && !seq_lens) ||
        out_tokens == tokens)
        return FRT_ERR_INVALID;
    if (misaligned(target_probs, 4) || misaligned(draft_probs, 4) || misaligned(tokens, 4) || misaligned(cu_seqlens, 4) || misaligned(seq_lens, 4) ||
        misaligned(u_accept, 4) || misaligned(u_sample, 4) || misaligned(out_tokens, 4) || misaligned(accepted, 4) || misaligned(kept_lens, 4))
        return FRT_ERR_INVALID;
    smp::VerifyParams p = {target_probs, draft_probs, p_stride, q_stride, tokens, cu_seqlens, seq_lens, u_accept, u_sample,
                           out_tokens, accepted, kept_lens, n_tokens, batch, vocab, 1};
    int ctas = 1;
    while (ctas < 8 && ctas * 2 * smp::THREADS <= vocab && (long long)batch * ctas * 2 <= 4ll * device_sm_count()) ctas *= 2;
    p.ctas = ctas;
    return smp::launch(smp::verify_drafts_kernel, p, ctas, batch, static_cast<cudaStream_t>(stream));
}

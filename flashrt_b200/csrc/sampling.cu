// Probabilities of logits, and the verification of drafted tokens against them.
//
// Stand behind the products that make logits and in front of the paged cache's lengths; no counterpart in the reference.
//
// Both read rows of a vocabulary once: a row belongs to a cluster of 1 to 8 CTAs that hold it (softmax: in registers) and exchange a few
// numbers through distributed shared memory.  Rows start anywhere (odd vocabularies): 16-byte vectors lie where memory has them, and the
// first and last of a row are taken value by value.
#include "common.cuh"
#include "tc05.cuh"
#include "flashrt_b200.h"

namespace frt {
namespace smp {

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
// 16 bytes, or four times `other` and no access: no branch, so that the loads of an unrolled loop are all under way at once
__device__ __forceinline__ uint4 ld_v4_if(const void* p, bool in, uint32_t other) {
    uint4 v;
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "mov.b32 %0, %6;\n\tmov.b32 %1, %6;\n\tmov.b32 %2, %6;\n\tmov.b32 %3, %6;\n\t"
        "@q ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
        : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w) : "l"(p), "r"((uint32_t)in), "r"(other) : "memory");
    return v;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float warp_max(float x) {
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

// ------------------------------------------------------------------------------------------------ softmax
//   p = exp((x - max) / T) / sum;  T not above zero: one on the first of the largest;  nothing but -infinity and NaN: zeros.
// A CTA's part: exponentials against its own maximum, then one exchange of (maximum, sum) in the cluster, and a factor that takes them to
// the row's.  NV vectors a thread; HELD false: what is behind them is read twice.
struct SoftmaxParams {
    const void* x;
    float* p;
    const float* temperature;
    long long in_stride, out_stride;
    int vocab, ctas;             // ctas: of a row
};

template <int THREADS, int NV, bool F32, bool HELD>
__global__ void __launch_bounds__(THREADS, NV * (F32 ? 4 : 8) > 32 ? 1 : 1024 / THREADS)
softmax_rows_kernel(SoftmaxParams p) {
    constexpr int VE = F32 ? 4 : 8, WARPS = THREADS / 32;    // values of 16 bytes
    __shared__ float part[WARPS], part2[WARPS];
    __shared__ int part3[WARPS];
    __shared__ uint4 mine;                                   // maximum, sum, index of the first of the largest
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ctas = p.ctas, rank = (int)(blockIdx.x % (unsigned)ctas);
    const long long row = blockIdx.x / (unsigned)ctas;
    const uint8_t* x = static_cast<const uint8_t*>(p.x) + row * p.in_stride * (F32 ? 4 : 2);
    float* out = p.p + row * p.out_stride;
    // vector j has the entries VE j - skew ..: rows start anywhere, vectors at 16 bytes
    const int skew = (int)(reinterpret_cast<uintptr_t>(x) & 15) / (F32 ? 4 : 2), vectors = (p.vocab + skew + VE - 1) / VE;
    const bool wide = ((reinterpret_cast<uintptr_t>(out) - 4 * (uintptr_t)skew) & 15) == 0;
    const int j0 = (int)((long long)vectors * rank / ctas), j1 = (int)((long long)vectors * (rank + 1) / ctas);
    const float T = p.temperature ? p.temperature[row] : 1.0f;
    const bool hot = !(T > 0.0f);
    const float c = hot ? 0.0f : __fdiv_rn(1.4426950408889634f, T);
    const int ja = max(j0, skew ? 1 : 0), jb = min(j1, (p.vocab + skew) / VE);       // whole vectors of this CTA; one may lie at each end
    constexpr uint32_t MASKED = F32 ? 0xff800000u : 0xff80ff80u;
    auto raw = [&](int j) { return ld_v4_if(x + ((long long)j * VE - skew) * (F32 ? 4 : 2), j >= ja && j < jb, MASKED); };
    auto values = [&](const uint4& w, int j, float* v) {     // masked: -infinity, as NaN is
        if (F32) {
            v[0] = __uint_as_float(w.x);
            v[1] = __uint_as_float(w.y);
            v[2] = __uint_as_float(w.z);
            v[3] = __uint_as_float(w.w);
        } else {
            unpack_bf16x2(w.x, v[0], v[1]);
            unpack_bf16x2(w.y, v[2], v[3]);
            unpack_bf16x2(w.z, v[VE - 4], v[VE - 3]);
            unpack_bf16x2(w.w, v[VE - 2], v[VE - 1]);
        }
        if (j < j1 && (j < ja || j >= jb)) {
            const int e = j * VE - skew;
#pragma unroll
            for (int k = 0; k < VE; ++k)
                if (e + k >= 0 && e + k < p.vocab)
                    v[k] = F32 ? reinterpret_cast<const float*>(x)[e + k] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(x)[e + k]);
        }
#pragma unroll
        for (int k = 0; k < VE; ++k) v[k] = v[k] == v[k] ? v[k] : -INFINITY;
    };
    float v[NV * VE], top = -INFINITY;
    {
        uint4 w[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) w[i] = raw(j0 + tid + i * THREADS);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            values(w[i], j0 + tid + i * THREADS, v + i * VE);
#pragma unroll
            for (int k = 0; k < VE; ++k) top = fmaxf(top, v[i * VE + k]);
        }
    }
    auto rest = [&](auto f) {                                // what this thread does not hold
        if (!HELD)
            for (int j = j0 + tid + NV * THREADS; j < j1; j += THREADS) {
                float w[VE];
                values(raw(j), j, w);
                f(j, w);
            }
    };
    rest([&](int, const float* w) {
#pragma unroll
        for (int k = 0; k < VE; ++k) top = fmaxf(top, w[k]);
    });
    top = warp_max(top);
    if (lane == 0) part[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, part[w]);
    // against this CTA's maximum; where that is infinite, the infinite ones share the mass
    auto weight = [&](float y) { return y == top ? 1.0f : exp2_approx(fmaxf(__fmul_rn(__fsub_rn(y, top), c), -3.0e38f)); };
    float sum = 0.0f;
    int first = 0x7fffffff;
    if (hot) {
        auto look = [&](int j, const float* w) {
#pragma unroll
            for (int k = 0; k < VE; ++k) {
                const int e = j * VE - skew + k;
                if (j < j1 && e >= 0 && e < p.vocab && w[k] == top) first = min(first, e);
            }
        };
#pragma unroll
        for (int i = 0; i < NV; ++i) look(j0 + tid + i * THREADS, v + i * VE);
        rest(look);
    } else if (top != -INFINITY) {                           // otherwise every weight stays 0 through the factor
#pragma unroll
        for (int i = 0; i < NV * VE; ++i) {
            v[i] = weight(v[i]);
            sum += v[i];
        }
        rest([&](int, const float* w) {
#pragma unroll
            for (int k = 0; k < VE; ++k) sum += weight(w[k]);
        });
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
    bool nothing = top == -INFINITY;                         // this CTA's entries are all masked: zeros
    if (ctas > 1) {
        if (tid == 0) mine = make_uint4(__float_as_uint(top), __float_as_uint(sum), (uint32_t)first, 0);
        tc::cluster_sync_all();
        uint4 all[8];
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < ctas) all[r] = dsmem_ld_u32x4(tc::dsmem_map(tc::smem_u32(&mine), (uint32_t)r));
        tc::cluster_arrive();
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
        first = m == -INFINITY ? -1 : f;
        factor = __fdiv_rn(top == m ? 1.0f : exp2_approx(fmaxf(__fmul_rn(__fsub_rn(top, m), c), -3.0e38f)), total);
    } else {
        if (nothing) first = -1;
        factor = __fdiv_rn(1.0f, sum);
    }
    auto store = [&](int j, float* w) {
        const int e = j * VE - skew;
        if (j >= j1) return;
#pragma unroll
        for (int k = 0; k < VE; ++k) w[k] = hot ? (e + k == first ? 1.0f : 0.0f) : nothing ? 0.0f : __fmul_rn(w[k], factor);
        if (wide && j >= ja && j < jb) {
#pragma unroll
            for (int k = 0; k < VE; k += 4) *reinterpret_cast<float4*>(out + e + k) = make_float4(w[k], w[k + 1], w[k + 2], w[k + 3]);
        } else {
#pragma unroll
            for (int k = 0; k < VE; ++k)
                if (e + k >= 0 && e + k < p.vocab) out[e + k] = w[k];
        }
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) store(j0 + tid + i * THREADS, v + i * VE);
    if (!HELD)
        for (int j = j0 + tid + NV * THREADS; j < j1; j += THREADS) {
            float w[VE];
            values(raw(j), j, w);
#pragma unroll
            for (int k = 0; k < VE; ++k) w[k] = hot || nothing ? 0.0f : weight(w[k]);
            store(j, w);
        }
    if (ctas > 1) tc::cluster_wait();                        // nobody leaves while its numbers are read
}

// ------------------------------------------------------------------------------------------------ verification
//   row t answers with token t + 1.  Drafted token d = tokens[t + 1] stands if u[t] q[t][d] < p[t][d] (exact in 64 bits: two products of 24).
//   At the first that does not: a token from max(p - q, 0) of that row, from p where nothing is left of it; if all stand, from p of
//   the last row.  The token is the first whose running sum is above v times the sum of all, in 64 bits.
// A warp has a run of neighbouring entries in SLOTS stretches; the sums of stretches stay in registers, those of runs go through shared
// memory, those of CTAs through the cluster, and from there the search goes back down: CTA, warp, stretch, lane, and the lane's four.
constexpr int VERIFY_THREADS = 512, VERIFY_WARPS = VERIFY_THREADS / 32, SLOTS = 8;

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
__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}

__global__ void __launch_bounds__(VERIFY_THREADS, 2)
verify_drafts_kernel(VerifyParams a) {
    constexpr int WARPS = VERIFY_WARPS;
    __shared__ double sums[WARPS];
    __shared__ double mine;
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ctas = a.ctas, rank = (int)(blockIdx.x % (unsigned)ctas), b = (int)(blockIdx.x / (unsigned)ctas);
    const int first = a.cu[b], end = a.cu[b + 1];
    const int len = a.lens ? a.lens[b] : 0;
    const float v0 = a.v[b], v = v0 > 0.0f ? fminf(v0, 0.99999994f) : 0.0f;
    const bool idle = first < 0 || end > a.n_tokens || end <= first;
    const int drafts = idle ? 0 : end - first - 1;
    int stood = 0;
    for (; stood < drafts; stood += 32) {
        const int i = stood + lane;
        bool stands = false;
        if (i < drafts) {
            const int t = first + i, d = a.tokens[t + 1];
            const float u = a.u[t];
            if (d >= 0 && d < a.vocab) {
                const float q = a.q ? a.q[t * a.q_stride + d] : 1.0f;
                stands = (double)u * (double)q < (double)a.p[t * a.p_stride + d];
            }
        }
        const unsigned fails = __ballot_sync(0xffffffffu, !stands);
        if (fails) {
            stood += __ffs(fails) - 1;
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
            for (int i = tid; i <= drafts; i += VERIFY_THREADS)
                if (i != stood) a.out[first + i] = i < stood ? a.tokens[first + i + 1] : -1;
    }
    if (idle) return;                                        // all CTAs of the cluster
    const int t = first + stood;
    const bool rejected = stood < drafts;
    const float* p = a.p + t * a.p_stride;
    const float* q = rejected && a.q ? a.q + t * a.q_stride : nullptr;
    const int gone = rejected && !a.q ? a.tokens[t + 1] : -1;      // entry that has nothing left
    // vector j has the entries 4 j - skew ..: rows start anywhere, vectors at 16 bytes
    const int skew = (int)(reinterpret_cast<uintptr_t>(p) & 15) / 4, vectors = (a.vocab + skew + 3) / 4;
    const bool q_wide = q && ((reinterpret_cast<uintptr_t>(q) - 4 * (uintptr_t)skew) & 15) == 0;
    const int runs = ctas * WARPS, run = rank * WARPS + warp;
    const int j0 = (int)((long long)vectors * run / runs), j1 = (int)((long long)vectors * (run + 1) / runs);
    const int stretch = (j1 - j0 + SLOTS * 32 - 1) / (SLOTS * 32) * 32;
    const int ja = max(j0, skew ? 1 : 0), jb = min(j1, (a.vocab + skew) / 4);        // whole vectors of this run; one may lie at each end
    auto raw = [&](const float* row, bool wide, int j, int je) { return ld_v4_if(row + 4 * j - skew, wide && j >= ja && j < jb && j < je, 0); };
    auto values = [&](const uint4& w, const float* row, bool wide, int j, int je) {
        float4 x = make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w));
        if (j < j1 && j < je && (!wide || j < ja || j >= jb)) {
            const int e = 4 * j - skew;
            if (e >= 0) x.x = row[e];
            if (e + 1 >= 0 && e + 1 < a.vocab) x.y = row[e + 1];
            if (e + 2 >= 0 && e + 2 < a.vocab) x.z = row[e + 2];
            if (e + 3 < a.vocab) x.w = row[e + 3];
        }
        return x;
    };
    // what vector j weighs; from_p: its probabilities, otherwise what is left of them
    auto weigh = [&](const float4& x, const float4& y, int j, bool from_p, double (&w)[4]) {
        const float xs[4] = {fmaxf(x.x, 0.0f), fmaxf(x.y, 0.0f), fmaxf(x.z, 0.0f), fmaxf(x.w, 0.0f)}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (from_p || !q) w[k] = !from_p && 4 * j - skew + k == gone ? 0.0 : (double)xs[k];
            else w[k] = xs[k] > ys[k] ? (double)xs[k] - (double)ys[k] : 0.0;
        }
    };
    const float4 zero4 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    double slot[SLOTS], start = 0.0, total = 0.0, target = 0.0;
    bool from_p = false;
    int owner = -1;
    for (;; from_p = true) {
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) slot[k] = 0.0;
        for (int i = lane; i < stretch; i += 32) {
#pragma unroll
            for (int k0 = 0; k0 < SLOTS; k0 += 4) {
                uint4 x[4], y[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = raw(p, true, j0 + (k0 + k) * stretch + i, j1);
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] = raw(q, q_wide && !from_p, j0 + (k0 + k) * stretch + i, j1);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int j = j0 + (k0 + k) * stretch + i;
                    double w[4];
                    weigh(values(x[k], p, true, j, j1), q && !from_p ? values(y[k], q, q_wide, j, j1) : zero4, j, from_p, w);
                    slot[k0 + k] += (w[0] + w[1]) + (w[2] + w[3]);
                }
            }
        }
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) s += slot[k];
        s = warp_sum(s);
        __syncthreads();                                     // `sums` of a pass before are read
        if (lane == 0) sums[warp] = s;
        __syncthreads();
        double cta = 0.0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) cta += sums[w];
        double all[8];
        if (ctas > 1) {
            if (tid == 0) mine = cta;
            tc::cluster_sync_all();
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r < ctas) all[r] = __longlong_as_double((long long)dsmem_ld_u64(tc::dsmem_map(tc::smem_u32(&mine), (uint32_t)r)));
            tc::cluster_arrive();
        } else {
            all[0] = cta;
        }
        total = 0.0;
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < ctas) total += all[r];
        target = (double)v * total;
        // the last CTA that starts at or below the target and is not empty
        double at = 0.0;
        owner = -1;
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < ctas) {
                if (at <= target && all[r] > 0.0) {
                    owner = r;
                    if (r == rank) start = at;
                }
                at += all[r];
            }
        if (total > 0.0 || from_p) break;
        if (ctas > 1) tc::cluster_wait();                    // everyone has read: `mine` may change
    }
    if (owner < 0 && rank == 0 && tid == 0) a.out[t] = -1;   // no probability anywhere, or an infinite one
    if (owner == rank) {
        int w = -1;
        double at = start;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) {
            if (at <= target && sums[i] > 0.0) {
                w = i;
                start = at;
            }
            at += sums[i];
        }
        if (w == warp) {
            int hit = 0;
            double in_front = start;
            at = start;
#pragma unroll
            for (int k = 0; k < SLOTS; ++k) {
                const double s = warp_sum(slot[k]);
                if (at <= target && s > 0.0) {
                    hit = k;
                    in_front = at;
                }
                at += s;
            }
            // the stretch again, 128 entries at a time
            const int s0 = j0 + hit * stretch, s1 = min(s0 + stretch, j1);
            int token = -1, last = -1;
            for (int base = s0; base < s1 && token < 0; base += 32) {
                const int j = base + lane;
                double y[4];
                const uint4 xw = raw(p, true, j, s1), yw = raw(q, q_wide && !from_p, j, s1);
                weigh(values(xw, p, true, j, s1), q && !from_p ? values(yw, q, q_wide, j, s1) : zero4, j, from_p, y);
                const double upto = warp_scan((y[0] + y[1]) + (y[2] + y[3]));
                double x = __shfl_up_sync(0xffffffffu, upto, 1);
                x = in_front + (lane ? x : 0.0);
                int found = 0x7fffffff, some = -1;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    x += y[k];
                    const int e = 4 * j - skew + k;
                    if (y[k] > 0.0) {
                        some = e;
                        if (x > target) found = min(found, e);
                    }
                }
                found = __reduce_min_sync(0xffffffffu, found);
                some = __reduce_max_sync(0xffffffffu, some);
                if (found != 0x7fffffff) token = found;
                if (some >= 0) last = some;
                in_front += __shfl_sync(0xffffffffu, upto, 31);
            }
            if (lane == 0) a.out[t] = token >= 0 ? token : last;     // roundings left the target behind the last one: that one
        }
    }
    if (ctas > 1) tc::cluster_wait();                        // nobody leaves while its sum is read
}

template <typename P>
static int launch(void (*kernel)(P), const P& p, unsigned ctas, unsigned rows, unsigned threads, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas * rows);
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctas > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    return e == cudaSuccess ? FRT_OK : FRT_CUDA_ERR(e);
}

template <bool F32>
static int launch_softmax(SoftmaxParams p, int rows, cudaStream_t st) {
    constexpr int N16 = F32 ? 4 : 2, VE = F32 ? 4 : 8;       // vectors of 16 values; values of a vector
    // CTAs of a row: enough to hold it, 32 values a thread; more where the rows leave SMs idle
    int ctas = 1;
    while (ctas < 8 && ((long long)ctas * 512 * 32 < p.vocab || ((long long)rows * ctas * 2 <= device_sm_count() && ctas * 512 * 4 < p.vocab))) ctas *= 2;
    p.ctas = ctas;
    const bool aligned = ((reinterpret_cast<uintptr_t>(p.x) | (uintptr_t)(p.in_stride * (16 / VE))) & 15) == 0;
    const int vectors = (p.vocab + (aligned ? 0 : VE - 1) + VE - 1) / VE, each = (vectors + ctas - 1) / ctas;
    if (each <= N16 * 128) return launch(softmax_rows_kernel<128, N16, F32, true>, p, ctas, rows, 128, st);
    if (each <= N16 * 512) return launch(softmax_rows_kernel<512, N16, F32, true>, p, ctas, rows, 512, st);
    if (each <= 2 * N16 * 512) return launch(softmax_rows_kernel<512, 2 * N16, F32, true>, p, ctas, rows, 512, st);
    if (each <= 4 * N16 * 512) return launch(softmax_rows_kernel<512, 4 * N16, F32, true>, p, ctas, rows, 512, st);
    return launch(softmax_rows_kernel<512, 2 * N16, F32, false>, p, ctas, rows, 512, st);
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
    while (ctas < 8 && ctas * 8 * smp::VERIFY_THREADS <= vocab && (long long)batch * ctas * 2 <= 2ll * device_sm_count()) ctas *= 2;
    p.ctas = ctas;
    return smp::launch(smp::verify_drafts_kernel, p, ctas, batch, smp::VERIFY_THREADS, static_cast<cudaStream_t>(stream));
}

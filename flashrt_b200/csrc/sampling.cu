// Probabilities of logits, and the verification of drafted tokens against them.
//
// Stand behind the products that make logits and in front of the paged cache's lengths; no counterpart in the reference.
//
// Both read rows of a vocabulary once, where a cluster of 1 to 8 CTAs holds one (softmax: in registers); its CTAs send one another a
// few numbers.  Rows start anywhere (odd vocabularies): 16-byte vectors lie where memory has them, and the
// first and last of a row are taken value by value.
#include "common.cuh"
#include "tc05.cuh"
#include "flashrt_b200.h"

namespace frt {
namespace smp {

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

// exp((x - m) / T), c = log2(e) / T, x not above m.  By halves, since logits of both signs can lie further apart than the largest number while a large T
// brings them near; equal ones weigh one by comparison, since 0 times infinity (both infinite, or a T next to nothing) would stand there.  NaN
// (a masked one at infinite T) weighs nothing.
__device__ __forceinline__ float weight_of(float x, float m, float c) {
    const float half = __fmul_rn(__fmaf_rn(0.5f, x, __fmul_rn(-0.5f, m)), c);
    return x == m ? 1.0f : exp2_approx(fmaxf(__fadd_rn(half, half), -3.0e38f));
}

// A wait of this warp gave up: the warp asks for nothing and sends nothing any more, gives copies and messages on their way a bounded time (the
// CTA's shared memory is another's once its last warp has left), and leaves.  The CTA's barriers wait for threads that have not left,
// so its other warps go on until a wait of their own gives up, which it does where it needed this one.
__device__ __forceinline__ void gave_up(int* status, int code) {
    if ((threadIdx.x & 31) == 0) atomicCAS(status, 0, code);
    const uint64_t until = tc::global_timer_ns() + 1000000ull;
    while (tc::global_timer_ns() < until) {}
}

// ------------------------------------------------------------------------------------------------ softmax
//   p = exp((x - max) / T) / sum;  T not above zero: one on the first of the largest;  nothing but -infinity and NaN: zeros.
// Weights are exponentials against the warp's own maximum; the (maximum, sum) of warps meet in shared memory, those of the cluster's CTAs
// by st.async (a cluster barrier waits for every store in front of it: 384 rows of 131072 in fp32 103 us with two a row), and a factor
// takes a warp's weights to the row's probabilities.  NV vectors a thread.  FORM 0: a row a cluster; 1: the same, and what is behind NV vectors is
// read three times (maximum, sum, output; the last two find it in L2; bf16 spills 84 bytes of stores and 152 of loads a thread at 64 registers);
// 2: clusters stay and go from row to row, the next row's part is copied to shared memory meanwhile (384 rows of 131072 71 us in fp32, 5.7 TB/s,
// 63 in bf16; without the copy 124).  Clusters that stay let the next kernel in with their last row: at the start its CTAs take places beside
// them (88, when a row took 78).
struct SoftmaxParams {
    const void* x;
    float* p;
    const float* temperature;
    long long in_stride, out_stride;
    int rows, vocab, ctas;       // ctas: of a row
    int* status;
};
constexpr int ONE_ROW = 0, READ_AGAIN = 1, STAY = 2;
enum { ERR_MAIL = 1, ERR_ROW = 2 };

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

template <int THREADS, int NV, bool F32, int FORM>
__global__ void __launch_bounds__(THREADS, (NV * (F32 ? 4 : 8) > 32 ? 512 : 1024) / THREADS)
softmax_rows_kernel(SoftmaxParams p) {
    constexpr int VE = F32 ? 4 : 8, ES = F32 ? 4 : 2, WARPS = THREADS / 32;      // values of 16 bytes, bytes of a value
    constexpr bool HELD = FORM != READ_AGAIN, STAGED = FORM == STAY;
    extern __shared__ uint4 stage[];                         // STAY: the next row's part
    __shared__ float part[2][WARPS], part2[2][WARPS];        // of each warp: maximum, sum
    __shared__ int part3[2][WARPS];                          // first of its largest
    __shared__ uint4 box[2][8];                              // the same of each CTA of the cluster
    __shared__ uint64_t mail[2], there;
    if (!STAGED) pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ctas = p.ctas, rank = (int)(blockIdx.x % (unsigned)ctas), step = (int)(gridDim.x / (unsigned)ctas);
    int no_flag = 0;
    if (tid == 0 && (STAGED || ctas > 1)) {
        tc::mbar_init(&mail[0], 1);
        tc::mbar_init(&mail[1], 1);
        tc::mbar_init(&there, 1);
        tc::mbar_fence_init();
    }
    if (ctas > 1) tc::cluster_arrive();                      // waited for in front of the first message
    if (STAGED) __syncthreads();
    pdl_wait();
    // A row's part: vector j has the entries VE j - skew .., since rows start anywhere and vectors at 16 bytes; whole vectors [ja, jb) of
    // this CTA's [j0, j1), one may lie at each end of the row.
    struct Place { const uint8_t* base; int skew, j0, j1, ja, jb; };
    auto place = [&](int row) {
        Place w;
        const uint8_t* x = static_cast<const uint8_t*>(p.x) + row * p.in_stride * ES;
        w.skew = (int)(reinterpret_cast<uintptr_t>(x) & 15) / ES;
        w.base = x - w.skew * ES;
        const int vectors = (p.vocab + w.skew + VE - 1) / VE;
        w.j0 = (int)((long long)vectors * rank / ctas);
        w.j1 = (int)((long long)vectors * (rank + 1) / ctas);
        w.ja = max(w.j0, w.skew ? 1 : 0);
        w.jb = min(w.j1, (p.vocab + w.skew) / VE);
        return w;
    };
    auto fetch = [&](int row) {                              // one thread
        if (row >= p.rows) return;
        const Place w = place(row);
        tc::mbar_arrive_expect_tx(&there, (uint32_t)max(w.jb - w.ja, 0) * 16u);
        for (int j = w.ja; j < w.jb; j += 1024)
            tc::bulk_load(&stage[j - w.j0], w.base + (size_t)j * 16, (uint32_t)min(w.jb - j, 1024) * 16u, &there);
    };
    int row = (int)(blockIdx.x / (unsigned)ctas);
    if (STAGED && tid == 0) fetch(row);
    for (int turn = 0; row < p.rows; row += step, ++turn) {
        const Place at = place(row);
        const int odd = turn & 1, me = at.j0 + tid;
        float* out = p.p + row * p.out_stride;
        const float* xf = reinterpret_cast<const float*>(at.base) + at.skew;
        const __nv_bfloat16* xh = reinterpret_cast<const __nv_bfloat16*>(at.base) + at.skew;
        const bool edges = at.ja > at.j0 || at.jb < at.j1, wide = ((reinterpret_cast<uintptr_t>(out) - 4 * (uintptr_t)at.skew) & 15) == 0;
        const bool wide32 = ((reinterpret_cast<uintptr_t>(out) - 4 * (uintptr_t)at.skew) & 31) == 0;
        const float T = p.temperature ? p.temperature[row] : 1.0f;
        const bool hot = !(T > 0.0f);
        const float c = hot ? 0.0f : __fdiv_rn(1.4426950408889634f, T);
        constexpr uint32_t MASKED = F32 ? 0xff800000u : 0xff80ff80u;
        auto unpack = [&](const uint4& w, float* v) {
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
        };
        auto at_edge = [&](int j) { return j < at.j1 && (j < at.ja || j >= at.jb); };
        auto edge = [&](int j, float* v) {                   // value by value
            const int e = j * VE - at.skew;
#pragma unroll
            for (int k = 0; k < VE; ++k) {
                v[k] = -INFINITY;
                if (e + k >= 0 && e + k < p.vocab) v[k] = F32 ? xf[e + k] : __bfloat162float(xh[e + k]);
            }
        };
        // NaN: fmaxf leaves it out, here and in a weight's argument, which it puts at the lower end
        float v[NV * VE], top = -INFINITY;
        if (STAGED && !tc::warp_wait_limited(tc::smem_u32(&there), (uint32_t)odd, false, &no_flag)) return gave_up(p.status, ERR_ROW);
        {
            uint4 w[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int j = me + i * THREADS;
                const bool in = j >= at.ja && j < at.jb;
                if (STAGED) w[i] = in ? stage[j - at.j0] : make_uint4(MASKED, MASKED, MASKED, MASKED);
                else w[i] = ld_v4_if(at.base + (size_t)(unsigned)j * 16, in, MASKED);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) unpack(w[i], v + i * VE);
        }
        if (edges)
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (at_edge(me + i * THREADS)) edge(me + i * THREADS, v + i * VE);
#pragma unroll
        for (int i = 0; i < NV * VE; ++i) top = fmaxf(top, v[i]);
        auto rest = [&](auto f) {                            // what this thread does not hold
            if (!HELD)
                for (int j = me + NV * THREADS; j < at.j1; j += THREADS) {
                    float w[VE];
                    if (at_edge(j)) edge(j, w);
                    else unpack(ld_v4_if(at.base + (size_t)(unsigned)j * 16, true, MASKED), w);
                    f(j, w);
                }
        };
        rest([&](int, float* w) {
#pragma unroll
            for (int k = 0; k < VE; ++k) top = fmaxf(top, w[k]);
        });
        top = warp_max(top);
        // weights two at a time; one by one where the maximum is infinite (the infinite ones share the mass) or so large that differences could be,
        // or where the temperature is so small that its reciprocal is
        const bool nothing = top == -INFINITY;               // this warp's entries are all masked: zeros
        const bool plain = !nothing && top < 0x1p102f && c < INFINITY;
        const uint64_t minus_top = f32x2(-top, -top), c2 = f32x2(c, c);
        auto weigh = [&](float* w, auto slow) {
            if (!decltype(slow)::value) {
#pragma unroll
                for (int k = 0; k < VE; k += 2) {
                    float a, b;
                    f32x2_parts(mul_f32x2(add_f32x2(f32x2(w[k], w[k + 1]), minus_top), c2), a, b);
                    w[k] = exp2_approx(fmaxf(a, -3.0e38f));
                    w[k + 1] = exp2_approx(fmaxf(b, -3.0e38f));
                }
            } else {
#pragma unroll
                for (int k = 0; k < VE; ++k) w[k] = weight_of(w[k], top, c);
            }
        };
        uint64_t sum2 = 0;
        int first = 0x7fffffff;
        auto look = [&](int j, float* w) {
#pragma unroll
            for (int k = 0; k < VE; ++k) {
                const int e = j * VE - at.skew + k;
                if (j < at.j1 && e >= 0 && e < p.vocab && w[k] == top) first = min(first, e);
            }
        };
        auto add = [&](float* w) {
#pragma unroll
            for (int k = 0; k < VE; k += 2) sum2 = add_f32x2(sum2, f32x2(w[k], w[k + 1]));
        };
        if (hot) {
#pragma unroll
            for (int i = 0; i < NV; ++i) look(me + i * THREADS, v + i * VE);
            rest(look);
            first = __reduce_min_sync(0xffffffffu, first);
        } else if (plain) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                weigh(v + i * VE, No());
                add(v + i * VE);
            }
            rest([&](int, float* w) {
                weigh(w, No());
                add(w);
            });
        } else if (!nothing) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                weigh(v + i * VE, Yes());
                add(v + i * VE);
            }
            rest([&](int, float* w) {
                weigh(w, Yes());
                add(w);
            });
        }
        float sum, sum_odd;
        f32x2_parts(sum2, sum, sum_odd);
        sum = warp_sum_butterfly(__fadd_rn(sum, sum_odd));
        if (lane == 0) {
            part[odd][warp] = top;
            part2[odd][warp] = sum;
            part3[odd][warp] = first;
        }
        __syncthreads();
        if (STAGED && tid == 0) fetch(row + step);           // everyone has taken this row's part
        if (STAGED && row + step >= p.rows) pdl_launch_dependents();        // earlier, the next kernel's CTAs would be in the way of clusters
        // lane w of every warp has warp w's, later CTA w's
        auto join = [&](float& m, float& s, int& f) {
            const float its = m;
            m = warp_max(its);
            s = warp_sum_butterfly(__fmul_rn(s, weight_of(its, m, c)));
            f = __reduce_min_sync(0xffffffffu, its == m ? f : 0x7fffffff);
        };
        float m = lane < WARPS ? part[odd][lane] : -INFINITY, total = lane < WARPS ? part2[odd][lane] : 0.0f;
        int f = lane < WARPS ? part3[odd][lane] : 0x7fffffff;
        if (ctas == 1 || warp == 0) join(m, total, f);
        if (ctas > 1) {
            if (turn == 0) tc::cluster_wait();               // the peers' barriers exist
            if (tid == 0) tc::mbar_arrive_expect_tx(&mail[odd], (uint32_t)ctas * 16u);
            if (warp == 0 && lane < ctas)
                tc::st_async_v4(tc::dsmem_map(tc::smem_u32(&box[odd][rank]), (uint32_t)lane), tc::dsmem_map(tc::smem_u32(&mail[odd]), (uint32_t)lane),
                                __float_as_uint(m), __float_as_uint(total), (uint32_t)f, 0u);
            // a box is written again two rows on, when every CTA has sent the row between, and so has read this one
            if (!tc::warp_wait_limited(tc::smem_u32(&mail[odd]), (uint32_t)(turn >> 1) & 1u, false, &no_flag)) return gave_up(p.status, ERR_MAIL);
            const uint4 its = lane < ctas ? box[odd][lane] : make_uint4(0xff800000u, 0u, 0x7fffffffu, 0u);
            m = __uint_as_float(its.x);
            total = __uint_as_float(its.y);
            f = (int)its.z;
            join(m, total, f);
        }
        if (m == -INFINITY) f = -1;
        const float factor = __fdiv_rn(weight_of(top, m, c), total);
        const uint64_t factor2 = f32x2(factor, factor);
        auto store = [&](int j, float* w) {
            const int e = j * VE - at.skew;
            if (hot || nothing) {
#pragma unroll
                for (int k = 0; k < VE; ++k) w[k] = hot && e + k == f ? 1.0f : 0.0f;
            } else {
#pragma unroll
                for (int k = 0; k < VE; k += 2) f32x2_parts(mul_f32x2(f32x2(w[k], w[k + 1]), factor2), w[k], w[k + 1]);
            }
            if (!F32 && wide32 && j >= at.ja && j < at.jb) {
                uint32_t r[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) r[k] = __float_as_uint(w[k % VE]);
                st_global_32(out + e, true, true, r);
            } else if (wide && j >= at.ja && j < at.jb) {
#pragma unroll
                for (int k = 0; k < VE; k += 4) *reinterpret_cast<float4*>(out + e + k) = make_float4(w[k], w[k + 1], w[k + 2], w[k + 3]);
            } else if (j < at.j1) {
#pragma unroll
                for (int k = 0; k < VE; ++k)
                    if (e + k >= 0 && e + k < p.vocab) out[e + k] = w[k];
            }
        };
#pragma unroll
        for (int i = 0; i < NV; ++i) store(me + i * THREADS, v + i * VE);
        rest([&](int j, float* w) {
            if (plain) weigh(w, No());
            else if (!hot && !nothing) weigh(w, Yes());
            store(j, w);
        });
        if (!STAGED) break;                                  // a cluster for each row
    }
}

// ------------------------------------------------------------------------------------------------ verification
//   row t answers with token t + 1.  Drafted token d = tokens[t + 1] stands if u[t] q[t][d] < p[t][d] (exact in 64 bits: two products of 24).
//   At the first that does not: a token from max(p - q, 0) of that row, from p where nothing is left of it; if all stand, from p of
//   the last row.  The token is the first whose running sum is above v times the sum of all, in 64 bits.
// A warp has a run of neighbouring entries in SLOTS stretches; the sums of stretches stay in registers, those of runs go through shared
// memory, those of CTAs through the cluster, and from there the search goes back down: CTA, warp, stretch, lane, and the lane's four.
// Two CTAs an SM leave 64 registers a thread; 176 bytes of stores and 200 of loads spill.  Rows of q that lie otherwise to 16 bytes than p's
// (another stride) are read value by value: 64 sequences of 131072 19.9 us instead of 14.8.
constexpr int VERIFY_THREADS = 512, VERIFY_WARPS = VERIFY_THREADS / 32, SLOTS = 8;

struct VerifyParams {
    const float *p, *q;
    long long p_stride, q_stride;
    const int *tokens, *cu, *lens;
    const float *u, *v;
    int *out, *accepted, *kept;
    int n_tokens, batch, vocab, ctas;
    int* status;
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
    __shared__ uint4 box[2][8];                              // sums of the cluster's CTAs, of what is left and of p
    __shared__ uint64_t mail[2];
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int no_flag = 0;
    if (a.ctas > 1) {
        if (tid == 0) {
            for (int i = 0; i < 2; ++i) {
                tc::mbar_init(&mail[i], 1);
                tc::mbar_arrive_expect_tx(&mail[i], (uint32_t)a.ctas * 16u);
            }
            tc::mbar_fence_init();
        }
        tc::cluster_arrive();                                // waited for in front of the first message
    }
    pdl_wait();
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
    if (idle) {                                              // all CTAs of the cluster
        if (ctas > 1) tc::cluster_wait();
        return;
    }
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
    const int at_gone = gone >= 0 ? (gone + skew) / 4 : -1;
    // Whole vectors weigh alike; those at the row's ends and the one with the token that is gone are left out there and added by a lane.
    const bool easy = !q || q_wide;
    double slot[SLOTS], start = 0.0, total = 0.0, target = 0.0;
    bool from_p = false;
    int owner = -1;
    for (int turn = 0;; ++turn, from_p = true) {
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) slot[k] = 0.0;
        const bool minus = q && !from_p;
        for (int i = lane; i < stretch; i += 32) {
#pragma unroll
            for (int k0 = 0; k0 < SLOTS; k0 += 4) {
                uint4 x[4], y[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = raw(p, !easy || j0 + (k0 + k) * stretch + i != at_gone, j0 + (k0 + k) * stretch + i, j1);
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] = raw(q, q_wide && minus, j0 + (k0 + k) * stretch + i, j1);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (easy) {                              // larger of both less q: two conversions, no selection
                        const float xs[4] = {__uint_as_float(x[k].x), __uint_as_float(x[k].y), __uint_as_float(x[k].z), __uint_as_float(x[k].w)};
                        const float ys[4] = {__uint_as_float(y[k].x), __uint_as_float(y[k].y), __uint_as_float(y[k].z), __uint_as_float(y[k].w)};
                        double w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = (double)fmaxf(xs[e], ys[e]) - (double)ys[e];
                        slot[k0 + k] += (w[0] + w[1]) + (w[2] + w[3]);
                    } else {
                        const int j = j0 + (k0 + k) * stretch + i;
                        double w[4];
                        weigh(values(x[k], p, true, j, j1), minus ? values(y[k], q, q_wide, j, j1) : zero4, j, from_p, w);
                        slot[k0 + k] += (w[0] + w[1]) + (w[2] + w[3]);
                    }
                }
            }
        }
        if (easy && lane == 0) {
            auto add = [&](int j) {
                const uint4 zero = make_uint4(0, 0, 0, 0);
                const bool whole = j >= ja && j < jb;        // the one whose token is gone
                double w[4];
                weigh(values(whole ? raw(p, true, j, j1) : zero, p, true, j, j1), minus ? values(zero, q, true, j, j1) : zero4, j, from_p, w);
                const double sum = (w[0] + w[1]) + (w[2] + w[3]);
#pragma unroll
                for (int k = 0; k < SLOTS; ++k)
                    if (j >= j0 + k * stretch && j < j0 + (k + 1) * stretch) slot[k] += sum;
            };
            const bool head = ja > j0, tail = jb < j1 && !(head && j1 == 1);
            if (head) add(0);
            if (tail) add(j1 - 1);
            if (at_gone >= j0 && at_gone < j1 && !(head && at_gone == 0) && !(tail && at_gone == j1 - 1)) add(at_gone);
        }
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) s += slot[k];
        s = warp_sum(s);
        if (turn) __syncthreads();                           // `sums` of the turn before are read
        if (lane == 0) sums[warp] = s;
        __syncthreads();
        double cta = 0.0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) cta += sums[w];
        double all[8];
        if (ctas > 1) {
            if (turn == 0) tc::cluster_wait();
            if (warp == 0 && lane < ctas) {
                const unsigned long long bits = (unsigned long long)__double_as_longlong(cta);
                tc::st_async_v4(tc::dsmem_map(tc::smem_u32(&box[turn][rank]), (uint32_t)lane), tc::dsmem_map(tc::smem_u32(&mail[turn]), (uint32_t)lane),
                                (uint32_t)bits, (uint32_t)(bits >> 32), 0u, 0u);
            }
            if (!tc::warp_wait_limited(tc::smem_u32(&mail[turn]), 0, false, &no_flag)) return gave_up(a.status, ERR_MAIL);
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r < ctas) {
                    const uint4 w = box[turn][r];
                    all[r] = __longlong_as_double((long long)((unsigned long long)w.x | (unsigned long long)w.y << 32));
                }
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
}

static int* status_word() {
    static PerDevicePointer status;
    return status.get(gemm_status_device_ptr);
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

// Form 2.  Clusters that the device holds at once: asked once per device and cluster size.
template <int THREADS, int NV, bool F32>
static int launch_staying(SoftmaxParams p, int rows, cudaStream_t st) {
    constexpr int SMEM = THREADS * NV * 16;
    static int known[64][4] = {};
    int c = 0;
    while (1 << c < p.ctas) ++c;
    auto kernel = softmax_rows_kernel<THREADS, NV, F32, STAY>;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return FRT_ERR_UNSUPPORTED;
    if (!known[dev][c]) {
        int n = 0;
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        cfg.gridDim = dim3(p.ctas);
        cfg.numAttrs = 1;
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
        if (e != cudaSuccess) return FRT_CUDA_ERR(e);
        known[dev][c] = n > 0 ? n : 1;
    }
    cfg.gridDim = dim3(p.ctas * (unsigned)(rows < known[dev][c] ? rows : known[dev][c]));
    cfg.numAttrs = 2;
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
    const bool few = (long long)rows * ctas <= 2 * device_sm_count();
    if (few && each <= N16 * 512) return launch(softmax_rows_kernel<512, N16, F32, ONE_ROW>, p, ctas, rows, 512, st);
    if (each <= 2 * N16 * 64) return launch(softmax_rows_kernel<64, 2 * N16, F32, ONE_ROW>, p, ctas, rows, 64, st);
    if (each <= 2 * N16 * 128) return launch(softmax_rows_kernel<128, 2 * N16, F32, ONE_ROW>, p, ctas, rows, 128, st);
    if (each <= 2 * N16 * 256) return launch(softmax_rows_kernel<256, 2 * N16, F32, ONE_ROW>, p, ctas, rows, 256, st);
    if (each <= 2 * N16 * 512) {
        if (few || ctas == 1) return launch(softmax_rows_kernel<512, 2 * N16, F32, ONE_ROW>, p, ctas, rows, 512, st);
        // 64 values a thread: with 32, twice the threads and as many rows under way, 384 rows of 131072 79 us instead of 71 (bf16 73 instead
        // of 63), 300 of 50257 27.2 instead of 25.2; on 16 CTAs a row, which needs leave, 90
        return launch_staying<256, 4 * N16, F32>(p, rows, st);
    }
    // A little more (a row that starts inside a vector has one more of them) is read again rather than held by clusters of twice the threads, of
    // which an SM has one: 384 rows of 131071 90 us against 150 (bf16 91 against 130), of 140000 113 against 139 (108 against 124), of 151936
    // 140 against 139.5 (113 against 124), 16 rows of them 8.5 against 11.5.  From five quarters on they are held: 384 of 163848 144 against
    // 147 (bf16 129 against 120), of 180000 148 against 171 (130 against 141), of 262136 169 against 301 (149 against 211).
    if (each > 2 * N16 * 640 && each <= 4 * N16 * 512) return launch_staying<512, 4 * N16, F32>(p, rows, st);
    return launch(softmax_rows_kernel<512, 2 * N16, F32, READ_AGAIN>, p, ctas, rows, 512, st);
}

}  // namespace smp
}  // namespace frt

static bool misaligned(const void* a, uintptr_t n) { return (reinterpret_cast<uintptr_t>(a) & (n - 1)) != 0; }
// a and b share bytes: rows of a_bytes every a_step (rows of one buffer may lie between those of another)
static bool rows_meet(const void* a, long long a_bytes, long long a_step, const void* b, long long b_bytes, long long b_step, int rows) {
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
    if (a0 >= b0 + (uintptr_t)(rows - 1) * b_step + b_bytes || b0 >= a0 + (uintptr_t)(rows - 1) * a_step + a_bytes) return false;
    for (long long i = 0, j = 0; i < rows && j < rows;) {
        const uintptr_t x = a0 + (uintptr_t)i * a_step, y = b0 + (uintptr_t)j * b_step;
        if (x < y + b_bytes && y < x + a_bytes) return true;
        if (x < y) ++i;
        else ++j;
    }
    return false;
}

extern "C" int frt_b200_softmax_rows(const void* in, long long in_stride, float* out, long long out_stride, const float* temperature, int rows,
                                     int vocab, int flags, void* stream) {
    using namespace frt;
    if (rows < 0 || vocab < 0 || in_stride < vocab || out_stride < vocab) return FRT_ERR_INVALID;
    if (rows > 1 << 27 || vocab > 1 << 30) return FRT_ERR_UNSUPPORTED;
    if (rows == 0 || vocab == 0) return FRT_OK;
    const bool f32 = flags & 2;
    if (!in || !out || misaligned(in, f32 ? 4 : 2) || misaligned(out, 4) || misaligned(temperature, 4)) return FRT_ERR_INVALID;
    const long long es = f32 ? 4 : 2;                        // rows are read while others are written
    if (rows_meet(in, vocab * es, in_stride * es, out, vocab * 4ll, out_stride * 4, rows)) return FRT_ERR_INVALID;
    smp::SoftmaxParams p = {in, out, temperature, in_stride, out_stride, rows, vocab, 1, smp::status_word()};
    if (!p.status) return FRT_ERR_UNSUPPORTED;
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
    if (!cu_seqlens || !u_sample || !accepted || (kept_lens && !seq_lens)) return FRT_ERR_INVALID;
    if (n_tokens && (!target_probs || !tokens || !u_accept || !out_tokens)) return FRT_ERR_INVALID;
    if (n_tokens && rows_meet(tokens, 4ll * n_tokens, 0, out_tokens, 4ll * n_tokens, 0, 1)) return FRT_ERR_INVALID;     // read while they are written
    if (misaligned(target_probs, 4) || misaligned(draft_probs, 4) || misaligned(tokens, 4) || misaligned(cu_seqlens, 4) || misaligned(seq_lens, 4) ||
        misaligned(u_accept, 4) || misaligned(u_sample, 4) || misaligned(out_tokens, 4) || misaligned(accepted, 4) || misaligned(kept_lens, 4))
        return FRT_ERR_INVALID;
    smp::VerifyParams p = {target_probs, draft_probs, p_stride, q_stride, tokens, cu_seqlens, seq_lens, u_accept, u_sample,
                           out_tokens, accepted, kept_lens, n_tokens, batch, vocab, 1, smp::status_word()};
    if (!p.status) return FRT_ERR_UNSUPPORTED;
    int ctas = 1;
    while (ctas < 8 && ctas * 8 * smp::VERIFY_THREADS <= vocab && (long long)batch * ctas * 2 <= 2ll * device_sm_count()) ctas *= 2;
    p.ctas = ctas;
    return smp::launch(smp::verify_drafts_kernel, p, ctas, batch, smp::VERIFY_THREADS, static_cast<cudaStream_t>(stream));
}

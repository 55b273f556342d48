// 8-bit integer products with a scale for each token and each output channel, and the quantiser of the activations.
//
// Stands beside the FP8 products (GemmRunner::fp8_nt_dev of the reference, csrc/gemm/gemm_runner.cu:67-76, whose scales are one per
// tensor); no counterpart in the reference.
//
//   D(M,N) = bf16((sum_k A[m,k] W[n,k]) * token_scale[m] * channel_scale[n] + bias[n])
//
// tcgen05.mma kind::i8: signed bytes, 32-bit integer sums in tensor memory, so the sum is exact and its order -- tiles, K splits --
// changes no bit; the conversion to fp32 and the two scales round at 2^-24 each, the store to bf16 once.
//
// More than 128 rows: 256 x 128 or 256 x 256 tiles on CTA pairs (cta_group::2, each CTA stages its 128 rows of A and half of the
// weight rows), persistent, two accumulators.  The tensor pipe bounds these.  The finish takes the accumulator through shared memory
// as fp32 -- a thread then owns four fixed columns of a tile's 32 rows and keeps their scales and bias in registers -- instead of
// reading every column's scale in every thread, since an accumulator row belongs to one thread.
// Up to 128 rows: the weights are the 128 lanes of a tile and the tokens its columns (16 to 128), because nothing is left but
// streaming the weights; K split over a cluster when there are few tiles, integer partials added through distributed shared memory.
// A tile stages its tokens beside its weights, with 65 to 128 tokens in as much room again (from L2): 96 x 32768 x 2048 21.7 us with its
// quantiser, 3.4 TB/s.
#include "common.cuh"
#include "tc05.cuh"
#include "flashrt_b200.h"

namespace frt {

int make_tmap_2d_u8(CUtensorMap* out, const void* base, uint64_t rows, uint64_t row_bytes, uint64_t pitch_bytes, uint32_t box_rows);

namespace i8 {

// ------------------------------------------------------------------------------------------------ quantise rows
//   s = max(max |finite x| / 127, 1e-12),  q = clamp(rint(x * (1 / s)), +-127); NaN -> 0.
// WPR warps of a row keep it in registers (NV x 8 values each) between the maximum and the codes: one read.  What a row
// has beyond 8192 values is read twice, the second time from L2: 817 x 16384 12 us, 3.3 TB/s.
constexpr int QR_NV = 4;

__device__ __forceinline__ float finite_max8(const uint4& v, float m) {
    const uint32_t* w = &v.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a, b;
        unpack_bf16x2(w[i], a, b);
        a = fabsf(a);
        b = fabsf(b);
        if (a < INFINITY) m = fmaxf(m, a);
        if (b < INFINITY) m = fmaxf(m, b);
    }
    return m;
}
__device__ __forceinline__ uint32_t to_s8(float v) {
    int r;
    asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(r) : "f"(v));     // NaN: 0
    return (uint32_t)max(r, -127) & 0xffu;
}
__device__ __forceinline__ uint2 codes8(const uint4& v, float inv) {
    const uint32_t* w = &v.x;
    uint32_t o[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a, b;
        unpack_bf16x2(w[i], a, b);
        o[i >> 1] |= (to_s8(__fmul_rn(a, inv)) | (to_s8(__fmul_rn(b, inv)) << 8)) << (16 * (i & 1));
    }
    return make_uint2(o[0], o[1]);
}

template <int WPR>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const __nv_bfloat16* x, long long x_stride, uint8_t* out, float* scale, int rows, int dim) {
    constexpr int RPB = 8 / WPR, T = 32 * WPR;
    __shared__ float part[8];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, slot = warp / WPR, me = threadIdx.x % T, vecs = dim >> 3;
    const long long row = (long long)blockIdx.x * RPB + slot;
    const bool in = row < rows;
    const __nv_bfloat16* src = x + (in ? row : 0) * x_stride;
    uint4 v[QR_NV];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < QR_NV; ++i)
        if (in && me + i * T < vecs) v[i] = ld_stream_v4(src + (size_t)(me + i * T) * 8);
#pragma unroll
    for (int i = 0; i < QR_NV; ++i)
        if (in && me + i * T < vecs) top = finite_max8(v[i], top);
    if (in)
        for (int i = me + QR_NV * T; i < vecs; i += T) top = finite_max8(ld_global_v4(src + (size_t)i * 8), top);
    top = warp_max_butterfly(top);
    if (WPR > 1) {
        if ((threadIdx.x & 31) == 0) part[warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WPR; ++w) top = fmaxf(top, part[slot * WPR + w]);
    }
    if (!in) return;
    const float s = fmaxf(__fdiv_rn(top, 127.0f), 1e-12f), inv = __fdiv_rn(1.0f, s);
    if (me == 0) scale[row] = s;
    uint8_t* dst = out + row * dim;
#pragma unroll
    for (int i = 0; i < QR_NV; ++i)
        if (me + i * T < vecs) st_global_v2(dst + (size_t)(me + i * T) * 8, codes8(v[i], inv));
    for (int i = me + QR_NV * T; i < vecs; i += T) st_global_v2(dst + (size_t)i * 8, codes8(ld_global_v4(src + (size_t)i * 8), inv));
}

// ------------------------------------------------------------------------------------------------ products
struct Params {
    __nv_bfloat16* out;
    const float *token_scale, *channel_scale;
    const __nv_bfloat16* bias;
    int* status;
    int M, N, kb;                // kb: k-blocks of 128
    int early;                   // the weights may be read before the kernel in front has ended
    int gm;                      // pair kernel: m-tiles of a group
};
enum { ERR_PRODUCER = 1, ERR_MMA = 2, ERR_EPILOGUE = 3 };

// signed bytes, 32-bit integer accumulators (formats as make_idesc: D 2 = s32, A and B 1 = s8)
__host__ __device__ constexpr uint32_t idesc_i8(uint32_t M, uint32_t N) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | ((M >> 4) << 24);
}
__device__ __forceinline__ void mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* slot, uint32_t ncols) {                  // same warp of both CTAs
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(slot)), "r"(ncols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* m, uint32_t bar_cluster_addr, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"(m), "r"(bar_cluster_addr), "r"(x), "r"(y)
        : "memory");
}
__device__ __forceinline__ void commit_both(uint32_t bar_addr, uint32_t leader) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar_addr),
        "h"((uint16_t)(3u << leader))
        : "memory");
}
__device__ __forceinline__ float finish(int acc, float ts, float cs, float bias, bool has_bias) {
    const float v = __fmul_rn(__int2float_rn(acc), ts);
    return has_bias ? __fmaf_rn(v, cs, bias) : __fmul_rn(v, cs);
}
__device__ __forceinline__ void gave_up(int* status, volatile int* abort_flag, int code) {
    if (!*abort_flag) atomicCAS(status, 0, code | (blockIdx.x << 8));
    *abort_flag = 1;
}

// A CTA that gave up may have copies in flight: a bounded time for them before its shared memory goes to another.
__device__ __forceinline__ void let_copies_land() {
    const uint64_t until = tc::global_timer_ns() + 1000000ull;
    while (tc::global_timer_ns() < until) {}
}

// ---------------------------------------------------------------- up to 128 rows: weights on the lanes, tokens on the columns
template <int BN>
struct LaneCfg {
    static constexpr int A_BYTES = 128 * 128, B_BYTES = BN * 128, STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int STAGES = BN <= 32 ? 5 : BN == 64 ? 4 : 3;           // about 100 KB: two CTAs per SM
    static constexpr int RED_BYTES = 128 * BN * 4;                           // a rank's partial, where the ring was
    static constexpr int RING_BYTES = STAGES * STAGE_BYTES > RED_BYTES ? STAGES * STAGE_BYTES : RED_BYTES;
    static constexpr int SMEM_BYTES = RING_BYTES + 1024 + 256;
    static constexpr int TMEM_COLS = BN < 32 ? 32 : BN;
};

// grid (n tiles, K splits), cluster (1, splits): rank r takes the k-blocks [kb r / S, kb (r + 1) / S)
template <int BN>
__global__ void __launch_bounds__(192, 2)
gemm_int8_lane_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW, Params p) {
    using Cfg = LaneCfg<BN>;
    constexpr int STAGES = Cfg::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::RING_BYTES);
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const uint64_t deadline = tc::global_timer_ns() + FRT_KERNEL_DEADLINE_NS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = (int)gridDim.y, rank = (int)blockIdx.y, n0 = (int)blockIdx.x * 128;
    const int kb0 = (int)((long long)p.kb * rank / S), kb1 = (int)((long long)p.kb * (rank + 1) / S);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            tc::mbar_init(&full[s], 1);
            tc::mbar_init(&empty[s], 1);
        }
        tc::mbar_init(acc_full, 1);
        *abort_flag = 0;
        tc::mbar_fence_init();
        tc::tma_prefetch_desc(&tmA);
        tc::tma_prefetch_desc(&tmW);
    }
    if (warp == 1) {
        tc::tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before_sync();
    __syncthreads();
    tc::tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();

    if (warp == 0) {
        // ---------------- producer (whole warp); settled weights: the first ring of them before the wait
        const uint32_t ring = tc::smem_u32(smem), full_a = tc::smem_u32(full), empty_a = tc::smem_u32(empty);
        const int ahead = p.early ? min(STAGES, kb1 - kb0) : 0;
        if (tc::elect_one())
            for (int s = 0; s < ahead; ++s) {
                tc::mbar_arrive_expect_tx(full_a + 8 * s, Cfg::STAGE_BYTES);
                tc::tma_load_2d(ring + s * Cfg::STAGE_BYTES, &tmW, full_a + 8 * s, (kb0 + s) * 128, n0);
            }
        __syncwarp();
        pdl_wait();
        if (tc::elect_one())
            for (int s = 0; s < ahead; ++s)
                tc::tma_load_2d(ring + s * Cfg::STAGE_BYTES + Cfg::A_BYTES, &tmA, full_a + 8 * s, (kb0 + s) * 128, 0);
        __syncwarp();
        int s = ahead % STAGES;
        uint32_t ph = ahead < STAGES;
        for (int kb = kb0 + ahead; kb < kb1; ++kb) {
            if (!tc::warp_wait(empty_a + 8 * s, ph, false, deadline, abort_flag)) {
                if (lane == 0) gave_up(p.status, abort_flag, ERR_PRODUCER);
                break;
            }
            if (tc::elect_one()) {
                const uint32_t dst = ring + s * Cfg::STAGE_BYTES, bar = full_a + 8 * s;
                tc::mbar_arrive_expect_tx(bar, Cfg::STAGE_BYTES);
                tc::tma_load_2d(dst, &tmW, bar, kb * 128, n0);
                tc::tma_load_2d(dst + Cfg::A_BYTES, &tmA, bar, kb * 128, 0);
            }
            __syncwarp();
            if (++s == STAGES) { s = 0; ph ^= 1; }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (whole warp)
        constexpr uint32_t idesc = idesc_i8(128, BN);
        const uint32_t full_a = tc::smem_u32(full), empty_a = tc::smem_u32(empty);
        const uint64_t dA0 = tc::make_desc_kmajor_sw128(tc::smem_u32(smem));
        const uint64_t dB0 = tc::make_desc_kmajor_sw128(tc::smem_u32(smem + Cfg::A_BYTES));
        int s = 0;
        uint32_t ph = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!tc::warp_wait(full_a + 8 * s, ph, false, deadline, abort_flag)) {
                if (lane == 0) gave_up(p.status, abort_flag, ERR_MMA);
                break;
            }
            tc::tc_fence_after_sync();
            if (tc::elect_one()) {
                const uint64_t so = (uint64_t)(s * (Cfg::STAGE_BYTES >> 4));
#pragma unroll
                for (int k = 0; k < 4; ++k) mma(tmem, dA0 + so + 2 * k, dB0 + so + 2 * k, idesc, kb > kb0 || k > 0 ? 1u : 0u);
                tc::mma_commit(empty_a + 8 * s);
                if (kb == kb1 - 1) tc::mma_commit(acc_full);
            }
            __syncwarp();
            if (++s == STAGES) { s = 0; ph ^= 1; }
        }
    } else {
        // ---------------- epilogue: warps 2..5, lane quadrant = warp % 4; a thread's lane is one output channel
        pdl_wait();
        const int q = warp & 3, n = n0 + q * 32 + lane;
        const uint32_t t_src = tmem + ((uint32_t)(q * 32) << 16);
        const bool in = n < p.N;
        const float cs = in ? p.channel_scale[n] : 0.0f;
        const float bias = in && p.bias ? __bfloat162float(p.bias[n]) : 0.0f;
        const bool ok = kb1 > kb0 ? tc::mbar_wait_until(acc_full, 0, deadline, abort_flag) : true;
        if (!__all_sync(0xffffffffu, ok)) {
            if (lane == 0) gave_up(p.status, abort_flag, ERR_EPILOGUE);
        } else {
            tc::tc_fence_after_sync();
#pragma unroll 1
            for (int c0 = 0; c0 < BN; c0 += 16) {
                if (c0 >= p.M) break;
                uint32_t v[16];
                __syncwarp();
                tc::tmem_ld16(t_src + c0, v);
                tc::tmem_ld_wait();
                if (S > 1) {
                    // [four tokens][channel]: a warp's store is 512 contiguous bytes
                    const uint32_t red = tc::smem_u32(smem) + (uint32_t)(c0 / 4 * 128 + q * 32 + lane) * 16;
#pragma unroll
                    for (int j = 0; j < 16; j += 4)
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(red + j * 512), "r"(v[j]), "r"(v[j + 1]), "r"(v[j + 2]),
                                     "r"(v[j + 3]) : "memory");
                    continue;
                }
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (in && c0 + j < p.M)
                        p.out[(size_t)(c0 + j) * p.N + n] =
                            __float2bfloat16_rn(finish((int)v[j], p.token_scale[c0 + j], cs, bias, p.bias != nullptr));
            }
        }
    }
    if (S > 1) {
        tc::cluster_sync_all();                              // all partials are there
        if (warp >= 2 && !*abort_flag) {
            const int q = warp & 3, n = n0 + q * 32 + lane;
            const bool in = n < p.N;
            const float cs = in ? p.channel_scale[n] : 0.0f;
            const float bias = in && p.bias ? __bfloat162float(p.bias[n]) : 0.0f;
            const uint32_t red = tc::smem_u32(smem) + (uint32_t)(q * 32 + lane) * 16;
            for (int g = rank; 4 * g < p.M; g += S) {        // four tokens; the ranks' partials are all on their way before the first is added
                float4 w[8];
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < S) w[r] = tc::dsmem_ld_f32x4(tc::dsmem_map(red + (uint32_t)g * 2048, (uint32_t)r));
                int sum[4] = {0, 0, 0, 0};
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < S) {
                        sum[0] += __float_as_int(w[r].x);
                        sum[1] += __float_as_int(w[r].y);
                        sum[2] += __float_as_int(w[r].z);
                        sum[3] += __float_as_int(w[r].w);
                    }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int m = 4 * g + e;
                    if (in && m < p.M) p.out[(size_t)m * p.N + n] = __float2bfloat16_rn(finish(sum[e], p.token_scale[m], cs, bias, p.bias != nullptr));
                }
            }
        }
        tc::cluster_sync_all();                              // nobody leaves while its partial is read
    }
    if (*abort_flag && threadIdx.x == 0) let_copies_land();
    tc::tc_fence_before_sync();
    __syncthreads();
    tc::tc_fence_after_sync();
    if (warp == 1) tc::tmem_dealloc(tmem, Cfg::TMEM_COLS);
}

// ---------------------------------------------------------------- more rows: CTA pairs, 256 x BN tiles
template <int BN>
struct PairCfg {
    static constexpr int A_BYTES = 128 * 128, B_BYTES = BN / 2 * 128, STAGE_BYTES = A_BYTES + B_BYTES;   // per CTA
    static constexpr int STAGES = BN == 256 ? 6 : 8;
    static constexpr int EPI_BYTES = 8 * 32 * 128;           // 32 rows x 32 fp32 columns of each epilogue warp
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + 256 + EPI_BYTES;
    static constexpr int TMEM_COLS = 2 * BN;                 // two accumulators
};

// Tiles in groups of gm m-tiles, m fastest inside a group: the pairs of a wave then share operand rows in L2.
__device__ __forceinline__ void tile_at(int t, int gm, int m_tiles, int n_tiles, int& m, int& n) {
    const int per = gm * n_tiles, g = t / per, r = t - g * per, h = min(m_tiles - g * gm, gm);
    n = r / h;
    m = g * gm + (r - n * h);
}

// 32 rows x 32 columns of an accumulator: token scale in the thread that holds the row, then through shared memory (16-byte chunks
// of a 128-byte row, chunk index xor row % 8) to threads that own four columns, channel scale and bias, stores of 64 bytes a row.
__device__ __forceinline__ void store_block(const Params& p, const uint32_t* v, int m_base, int nb, uint8_t* stg, float ts, bool vec) {
    const int lane = threadIdx.x & 31, ch = lane & 7, r0 = lane >> 3, n = nb + ch * 4;
    const uint32_t base = tc::smem_u32(stg), sw = (uint32_t)(lane & 7) << 4;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = __fmul_rn(__int2float_rn((int)v[4 * k + e]), ts);
        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(base + lane * 128 + (((uint32_t)k << 4) ^ sw)), "f"(f[0]), "f"(f[1]),
                     "f"(f[2]), "f"(f[3]) : "memory");
    }
    if (!vec) {
        // rows that start anywhere: a lane takes a column, a store two to three sectors of one row (four columns a lane and 2-byte stores
        // 8 bytes apart: 8192 x 1001 x 2048 41 us)
        const int col = nb + lane;
        const float cs = col < p.N ? p.channel_scale[col] : 0.0f;
        const float bias = p.bias && col < p.N ? __bfloat162float(p.bias[col]) : 0.0f;
        __syncwarp();
        __nv_bfloat16* dst = p.out + (size_t)m_base * p.N + col;
        const int rows = min(32, p.M - m_base);
#pragma unroll 8
        for (int r = 0; r < 32; ++r) {
            float f;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(base + r * 128 + ((uint32_t)((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) : "memory");
            f = p.bias ? __fmaf_rn(f, cs, bias) : __fmul_rn(f, cs);
            if (r < rows && col < p.N) dst[(size_t)r * p.N] = __float2bfloat16_rn(f);
        }
        __syncwarp();
        return;
    }
    float cs[4], bias[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        cs[e] = n + e < p.N ? p.channel_scale[n + e] : 0.0f;
        bias[e] = p.bias && n + e < p.N ? __bfloat162float(p.bias[n + e]) : 0.0f;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + r0, m = m_base + r;
        float f[4];
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3])
                     : "r"(base + r * 128 + ((uint32_t)(ch ^ (r & 7)) << 4)) : "memory");
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = p.bias ? __fmaf_rn(f[e], cs[e], bias[e]) : __fmul_rn(f[e], cs[e]);
        if (m < p.M && n < p.N)                              // N % 4 == 0: all four
            st_global_v2(p.out + (size_t)m * p.N + n, make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])));
    }
    __syncwarp();
}

// S > 1: a cluster of S pairs takes one tile, a pair the k-blocks [kb s / S, kb (s + 1) / S); the pairs then lay their integer partials into
// shared memory, where their rings were, and each finishes BN / S of the columns.
template <int BN, int S>
__global__ void __launch_bounds__(320, 1)
gemm_int8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW, Params p) {
    using Cfg = PairCfg<BN>;
    constexpr int STAGES = Cfg::STAGES;
    static_assert(S == 1 || (BN / S >= 64 && 128 * BN * 4 <= STAGES * Cfg::STAGE_BYTES), "columns of a half of the warps, partials in the ring");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * Cfg::STAGE_BYTES);   // the leader's count both CTAs' bytes
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;      // [2]
    uint64_t* acc_empty = acc_full + 2;       // [2] the leader's
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const uint64_t deadline = tc::global_timer_ns() + FRT_KERNEL_DEADLINE_NS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t cluster_rank = tc::cluster_ctarank(), rank = cluster_rank & 1, leader = cluster_rank & ~1u;
    const int split = (int)(cluster_rank >> 1);
    const int pair = (int)blockIdx.x / (2 * S), pairs = (int)gridDim.x / (2 * S);     // S > 1: as many as tiles
    const int kb0 = S == 1 ? 0 : (int)((long long)p.kb * split / S), kb1 = S == 1 ? p.kb : (int)((long long)p.kb * (split + 1) / S);
    const int m_tiles = (p.M + 255) / 256, n_tiles = (p.N + BN - 1) / BN, total = m_tiles * n_tiles;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            tc::mbar_init(&full[s], 1);
            tc::mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&acc_full[i], 1);
            tc::mbar_init(&acc_empty[i], 2 * 256);
        }
        *abort_flag = 0;
        tc::mbar_fence_init();
        tc::tma_prefetch_desc(&tmA);
        tc::tma_prefetch_desc(&tmW);
    }
    if (warp == 1) tmem_alloc_pair(tmem_slot, Cfg::TMEM_COLS);
    tc::tc_fence_before_sync();
    tc::cluster_sync_all();                    // both CTAs' barriers exist before anything signals across
    tc::tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();

    if (warp == 0) {
        // ---------------- producer of this CTA's rows, bytes counted at the leader
        const uint32_t ring = tc::smem_u32(smem), empty_a = tc::smem_u32(empty), full_a = tc::smem_u32(full);
        const uint32_t lead_full = tc::dsmem_map(full_a, leader);
        pdl_wait();
        int s = 0;
        uint32_t ph = 1;
        bool ready = true;
        for (int t = pair; t < total; t += pairs) {
            int mt, nt;
            tile_at(t, p.gm, m_tiles, n_tiles, mt, nt);
            const int m0 = mt * 256 + (int)rank * 128, n0 = nt * BN + (int)rank * (BN / 2);
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!tc::warp_wait(empty_a + 8 * s, ph, ready, deadline, abort_flag)) {
                    if (lane == 0) gave_up(p.status, abort_flag, ERR_PRODUCER);
                    t = total;
                    break;
                }
                const uint32_t dst = ring + s * Cfg::STAGE_BYTES, bar = lead_full + 8 * s, own = full_a + 8 * s;
                if (++s == STAGES) { s = 0; ph ^= 1; }
                ready = tc::mbar_test(empty_a + 8 * s, ph);
                if (tc::elect_one()) {
                    if (rank == 0) tc::mbar_arrive_expect_tx(own, 2 * Cfg::STAGE_BYTES);
                    tma_load_pair(dst, &tmA, bar, kb * 128, m0);
                    tma_load_pair(dst + Cfg::A_BYTES, &tmW, bar, kb * 128, n0);
                }
            }
        }
    } else if (warp == 1 && rank == 0) {
        // ---------------- MMA issuer for both CTAs
        constexpr uint32_t idesc = idesc_i8(256, BN);
        const uint64_t dA0 = tc::make_desc_kmajor_sw128(tc::smem_u32(smem));
        const uint64_t dB0 = tc::make_desc_kmajor_sw128(tc::smem_u32(smem + Cfg::A_BYTES));
        const uint32_t full_a = tc::smem_u32(full), empty_a = tc::smem_u32(empty);
        const uint32_t accF_a = tc::smem_u32(acc_full), accE_a = tc::smem_u32(acc_empty);
        int s = 0, i = 0;
        uint32_t ph = 0;
        bool ready = false, failed = false;
        for (int t = pair; t < total && !failed; t += pairs, ++i) {
            const int buf = i & 1;
            if (!tc::warp_wait(accE_a + 8 * buf, (uint32_t)(((i >> 1) - 1) & 1), i < 2, deadline, abort_flag)) {
                if (lane == 0) gave_up(p.status, abort_flag, ERR_MMA);
                break;
            }
            tc::tc_fence_after_sync();
            const uint32_t d_tm = tmem + buf * BN;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!tc::warp_wait(full_a + 8 * s, ph, ready, deadline, abort_flag)) {
                    if (lane == 0) gave_up(p.status, abort_flag, ERR_MMA);
                    failed = true;
                    break;
                }
                tc::tc_fence_after_sync();
                const uint64_t so = (uint64_t)(s * (Cfg::STAGE_BYTES >> 4));
                const uint32_t done = empty_a + 8 * s;
                if (++s == STAGES) { s = 0; ph ^= 1; }
                ready = tc::mbar_test(full_a + 8 * s, ph);
                if (tc::elect_one()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma_pair(d_tm, dA0 + so + 2 * k, dB0 + so + 2 * k, idesc, kb > kb0 || k > 0 ? 1u : 0u);
                    commit_both(done, leader);
                    if (kb == kb1 - 1) commit_both(accF_a + 8 * buf, leader);
                }
            }
        }
    } else if (warp >= 2) {
        // ---------------- epilogue: this CTA's 128 rows; a warp's lane quadrant and half of the columns
        pdl_wait();
        const int q = warp & 3, half = (warp - 2) >> 2;
        const uint32_t lane_off = (uint32_t)(q * 32) << 16;
        const bool vec = (p.N & 3) == 0;
        uint8_t* stg = smem + STAGES * Cfg::STAGE_BYTES + 256 + (warp - 2) * (32 * 128);
        int i = 0;
        for (int t = pair; t < total; t += pairs, ++i) {
            const int buf = i & 1;
            int mt, nt;
            tile_at(t, p.gm, m_tiles, n_tiles, mt, nt);
            const int m_base = mt * 256 + (int)rank * 128 + q * 32, n_base = nt * BN + half * (BN / 2);
            const float ts = m_base + lane < p.M ? p.token_scale[m_base + lane] : 0.0f;
            const bool ok = tc::mbar_wait_until(&acc_full[buf], (uint32_t)((i >> 1) & 1), deadline, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) {
                if (lane == 0) gave_up(p.status, abort_flag, ERR_EPILOGUE);
                break;
            }
            tc::tc_fence_after_sync();
            const uint32_t t_acc = tmem + buf * BN + half * (BN / 2) + lane_off;
#pragma unroll 1
            for (int c = 0; c < BN / 2; c += 32) {
                uint32_t v[32];
                __syncwarp();
                tc::tmem_ld32(t_acc + c, v);
                tc::tmem_ld_wait();
                if constexpr (S > 1) {                       // [four columns][row]: a warp's store is 512 contiguous bytes
                    const uint32_t red = tc::smem_u32(smem) + ((half * (BN / 2) + c) / 4 * 128 + q * 32 + lane) * 16;
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(red + j * 512), "r"(v[j]), "r"(v[j + 1]), "r"(v[j + 2]),
                                     "r"(v[j + 3]) : "memory");
                } else if (m_base < p.M && n_base + c < p.N) store_block(p, v, m_base, n_base + c, stg, ts, vec);
            }
            if constexpr (S > 1) break;
            tc::tc_fence_before_sync();
            tc::mbar_arrive_cluster(tc::dsmem_map(tc::smem_u32(&acc_empty[buf]), leader));
        }
    }
    if constexpr (S > 1) {
        tc::cluster_sync_all();                // all partials are there
        if (warp >= 2 && !*abort_flag) {
            constexpr int W = BN / S / 2;      // columns of this warp
            const int q = warp & 3, half = (warp - 2) >> 2, col = split * (BN / S) + half * W;
            int mt, nt;
            tile_at(pair, p.gm, m_tiles, n_tiles, mt, nt);
            const int m_base = mt * 256 + (int)rank * 128 + q * 32, n_base = nt * BN + col;
            const float ts = m_base + lane < p.M ? p.token_scale[m_base + lane] : 0.0f;
            uint8_t* stg = smem + STAGES * Cfg::STAGE_BYTES + 256 + (warp - 2) * (32 * 128);
            const uint32_t red = tc::smem_u32(smem) + (uint32_t)(col / 4 * 128 + q * 32 + lane) * 16;
#pragma unroll 1
            for (int c = 0; c < W; c += 32) {
                uint32_t v[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = 0;
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    const uint32_t from = tc::dsmem_map(red + (uint32_t)c * 512, (uint32_t)(2 * s) + rank);
                    float4 w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = tc::dsmem_ld_f32x4(from + (uint32_t)j * 2048);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        v[4 * j] += __float_as_uint(w[j].x);
                        v[4 * j + 1] += __float_as_uint(w[j].y);
                        v[4 * j + 2] += __float_as_uint(w[j].z);
                        v[4 * j + 3] += __float_as_uint(w[j].w);
                    }
                }
                if (m_base < p.M && n_base + c < p.N) store_block(p, v, m_base, n_base + c, stg, ts, (p.N & 3) == 0);
            }
        }
    }
    if (*abort_flag && threadIdx.x == 0) let_copies_land();
    __syncwarp();
    tc::tc_fence_before_sync();
    tc::cluster_sync_all();                    // the leader's MMAs read the peer's shared memory until the end
    if (warp == 1) tmem_dealloc_pair(tmem, Cfg::TMEM_COLS);
}

// ------------------------------------------------------------------------------------------------ host
template <int BN>
static int launch_lane(const void* A, const void* W, Params p, int K, int splits, cudaStream_t stream) {
    using Cfg = LaneCfg<BN>;
    static PerDeviceOnce once;
    CUtensorMap tmA, tmW;
    int dev = 0;
    if (once.need(dev)) {
        const cudaError_t e = cudaFuncSetAttribute(gemm_int8_lane_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES);
        if (e != cudaSuccess) return FRT_CUDA_ERR(e);
        once.set(dev);
    }
    int rc = make_tmap_2d_u8(&tmA, A, (uint64_t)p.M, (uint64_t)K, (uint64_t)K, BN);
    if (!rc) rc = make_tmap_2d_u8(&tmW, W, (uint64_t)p.N, (uint64_t)K, (uint64_t)K, 128);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((p.N + 127) / 128, splits);
    cfg.blockDim = dim3(192);
    cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = splits;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, gemm_int8_lane_kernel<BN>, tmA, tmW, p);
    return e == cudaSuccess ? FRT_OK : FRT_CUDA_ERR(e);
}

template <int BN, int S>
static int launch_pair(const void* A, const void* W, Params p, int K, cudaStream_t stream) {
    using Cfg = PairCfg<BN>;
    static PerDeviceOnce once;
    CUtensorMap tmA, tmW;
    int dev = 0;
    if (once.need(dev)) {
        const cudaError_t e = cudaFuncSetAttribute(gemm_int8_pair_kernel<BN, S>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES);
        if (e != cudaSuccess) return FRT_CUDA_ERR(e);
        once.set(dev);
    }
    int rc = make_tmap_2d_u8(&tmA, A, (uint64_t)p.M, (uint64_t)K, (uint64_t)K, 128);
    if (!rc) rc = make_tmap_2d_u8(&tmW, W, (uint64_t)p.N, (uint64_t)K, (uint64_t)K, BN / 2);
    if (rc) return rc;
    const int m_tiles = (p.M + 255) / 256, n_tiles = (p.N + BN - 1) / BN, workers = device_sm_count() / 2;
    const long long total = (long long)m_tiles * n_tiles;
    if (total > 0x7fffffffLL - workers) return FRT_ERR_UNSUPPORTED;
    // rows of A and of W that a wave reads: 256 gm and BN workers / gm, fewest when they are alike
    p.gm = 1;
    if (total <= workers) p.gm = m_tiles;
    else
        while (p.gm < m_tiles && (long long)(p.gm + 1) * (p.gm + 1) * 256 <= (long long)BN * workers) ++p.gm;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(S > 1 ? 2 * S * (unsigned)total : 2 * (unsigned)(total < workers ? total : workers));
    cfg.blockDim = dim3(320);
    cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2 * S;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, gemm_int8_pair_kernel<BN, S>, tmA, tmW, p);
    return e == cudaSuccess ? FRT_OK : FRT_CUDA_ERR(e);
}

// Clusters of the sharing form that the device holds at once (a cluster lies in one GPC, whose SMs its size need not divide): asked once.
template <int BN, int S>
static long long pair_clusters() {
    using Cfg = PairCfg<BN>;
    static int known[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    if (!known[dev]) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * S);
        cfg.blockDim = dim3(320);
        cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2 * S;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        cudaError_t e = cudaFuncSetAttribute(gemm_int8_pair_kernel<BN, S>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES);
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&n, gemm_int8_pair_kernel<BN, S>, &cfg);
        if (e != cudaSuccess) {
            cudaGetLastError();                              // not this launch's error: the form is not offered
            n = 0;
        }
        known[dev] = n + 1;
    }
    return known[dev] - 1;
}

template <int WPR>
static int launch_quantize(const void* x, long long stride, void* out, float* scale, int rows, int dim, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(((long long)rows + 8 / WPR - 1) / (8 / WPR)));
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, quantize_rows_kernel<WPR>, static_cast<const __nv_bfloat16*>(x), stride,
                                             static_cast<uint8_t*>(out), scale, rows, dim);
    return e == cudaSuccess ? FRT_OK : FRT_CUDA_ERR(e);
}

}  // namespace i8
}  // namespace frt

static bool misaligned(const void* a, uintptr_t n) { return (reinterpret_cast<uintptr_t>(a) & (n - 1)) != 0; }

extern "C" int frt_b200_quantize_int8_rows(const void* in_bf16, long long in_stride, void* out_s8, float* row_scale, int rows, int dim,
                                           int flags, void* stream) {
    using namespace frt;
    (void)flags;
    if (rows < 0 || dim < 0 || in_stride < dim || in_stride % 8) return FRT_ERR_INVALID;
    if (dim % 16) return FRT_ERR_UNSUPPORTED;
    if (rows == 0) return FRT_OK;
    if (!row_scale || (dim && (!in_bf16 || !out_s8))) return FRT_ERR_INVALID;
    if (misaligned(in_bf16, 16) || misaligned(out_s8, 16) || misaligned(row_scale, 4)) return FRT_ERR_INVALID;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    // warps of a row: enough to hold it in registers; where the rows alone do not fill the SMs, as many as have a vector to read
    int wpr = 1;
    const int hold = 32 * 8 * i8::QR_NV, few = 4 * device_sm_count();
    while (wpr < 8 && (wpr * hold < dim || ((long long)rows * wpr < few * 2 && wpr * 256 < dim))) wpr *= 2;
    if (wpr == 1) return i8::launch_quantize<1>(in_bf16, in_stride, out_s8, row_scale, rows, dim, st);
    if (wpr == 2) return i8::launch_quantize<2>(in_bf16, in_stride, out_s8, row_scale, rows, dim, st);
    if (wpr == 4) return i8::launch_quantize<4>(in_bf16, in_stride, out_s8, row_scale, rows, dim, st);
    return i8::launch_quantize<8>(in_bf16, in_stride, out_s8, row_scale, rows, dim, st);
}

extern "C" int frt_b200_gemm_int8_nt(const void* A, const void* W, void* D, int M, int N, int K, const float* token_scale,
                                     const float* channel_scale, const void* bias, int flags, void* stream) {
    using namespace frt;
    if (M < 0 || N < 0 || K < 1) return FRT_ERR_INVALID;
    if (K % 16 || K >= 131072 || M > 1 << 30 || N > 1 << 30) return FRT_ERR_UNSUPPORTED;      // 2^17 products of 2^14 leave 32 bits
    if (M == 0 || N == 0) return FRT_OK;
    if (!A || !W || !D || !token_scale || !channel_scale) return FRT_ERR_INVALID;
    if (misaligned(A, 16) || misaligned(W, 16) || misaligned(D, 16) || misaligned(token_scale, 4) || misaligned(channel_scale, 4) ||
        misaligned(bias, 2))
        return FRT_ERR_INVALID;
    i8::Params p = {};
    p.out = static_cast<__nv_bfloat16*>(D);
    p.token_scale = token_scale;
    p.channel_scale = channel_scale;
    p.bias = static_cast<const __nv_bfloat16*>(bias);
    static PerDevicePointer status;
    p.status = status.get(gemm_status_device_ptr);
    if (!p.status) return FRT_ERR_UNSUPPORTED;
    p.M = M;
    p.N = N;
    p.kb = (K + 127) / 128;
    p.early = flags & 1;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (M <= 128) {
        // K splits (a cluster) while the tiles alone leave SMs idle and every rank keeps two k-blocks
        const int tiles = (N + 127) / 128;
        int splits = 1;
        while (splits < 8 && tiles * splits * 2 <= 2 * device_sm_count() && p.kb / (splits * 2) >= 2) splits *= 2;
        if (M <= 16) return i8::launch_lane<16>(A, W, p, K, splits, st);
        if (M <= 32) return i8::launch_lane<32>(A, W, p, K, splits, st);
        if (M <= 64) return i8::launch_lane<64>(A, W, p, K, splits, st);
        return i8::launch_lane<128>(A, W, p, K, splits, st);
    }
    // The cheapest of: tiles of 256 or 128 columns in whole waves of CTA pairs, or, where the device holds them all at once, tiles whose K
    // two or four pairs share.  A k-block takes 0.30 us on 256 columns and 0.235 on 128 (operands from L2 bound it), an exchange of
    // partials 5.  817 x 2048 x 16384 30.0 us on 64 pairs of 128 columns, 26.7 with two pairs a tile; 256 x 2048 x 8192 on 16 pairs 18.9,
    // with four pairs a tile 14.5; 300 x 2048 x 2048 7.2 unshared, 22.7 shared.
    const long long pairs = device_sm_count() / 2, mt = (M + 255) / 256, wide = mt * ((N + 255) / 256), narrow = mt * ((N + 127) / 128);
    auto waves = [&](long long tiles) { return (double)((tiles + pairs - 1) / pairs); };
    double best = waves(wide) * p.kb * 0.30;
    int form = 0;
    if (waves(narrow) * p.kb * 0.235 < best) {
        best = waves(narrow) * p.kb * 0.235;
        form = 1;
    }
    auto shared = [&](int f, long long tiles, int S, double per_kb, long long (*clusters)()) {
        const double cost = (p.kb + S - 1) / S * per_kb + 5.0;
        if (cost < best && p.kb >= 4 * S && tiles <= clusters()) { best = cost; form = f; }
    };
    shared(2, wide, 2, 0.30, i8::pair_clusters<256, 2>);
    shared(3, wide, 4, 0.30, i8::pair_clusters<256, 4>);
    shared(4, narrow, 2, 0.235, i8::pair_clusters<128, 2>);
    switch (form) {
        case 1: return i8::launch_pair<128, 1>(A, W, p, K, st);
        case 2: return i8::launch_pair<256, 2>(A, W, p, K, st);
        case 3: return i8::launch_pair<256, 4>(A, W, p, K, st);
        case 4: return i8::launch_pair<128, 2>(A, W, p, K, st);
        default: return i8::launch_pair<256, 1>(A, W, p, K, st);
    }
}

// E4M3 products with a scale for each row and 128 of K of the activations and for each 128 x 128 block of the weights, and the quantiser
// of the activations.
//
// Stands beside the FP8 products with one scale per tensor (GemmRunner::fp8_nt_dev of the reference, csrc/gemm/gemm_runner.cu:67-76) and
// the int8 ones of gemm_int8.cu; no counterpart in the reference.
//
//   D(M,N) = sum_kb a_scale[kb][m] * w_scale[n / 128][kb] * (sum_{k in block kb} A[m,k] W[n,k]) + bias[n]
//
// tcgen05.mma kind::f8f6f4 sums one k-block of 128 into a buffer of tensor memory; the epilogue warps take it out, multiply by the block's
// scales and add it to the tile's sums, which they keep in registers (fp32: the block's scales differ, so tensor memory cannot hold them).
// The buffers go round, so that the next block's products run meanwhile.  That taking out is what bounds many rows: 256 x 256 x 128 on a CTA
// pair are 512 cycles of products, and a warp's 128 columns come out of tensor memory in 370 cycles when it is idle but in 850 beside the
// products, which go there for their sums too.  With the signals between the warps a k-block takes 0.53 us, 2.3 PFLOP/s on all pairs, where the
// products with one scale per tensor, taken out once a tile, take 0.41 (3.0; both from K 1024 to 8192 of 8192 x 9472, sixteen whole waves).  A
// tile's fill and store add 1.4 us: 8191 x 4096 x 4096, seven waves of which the last is not full, 120 to 128 us by the data, 2.1 to 2.3 PFLOP/s.
//
// Up to 64 rows the weights are the 128 lanes and the tokens the columns, because nothing is left but streaming the weights; so are tiles of 96
// or 128 tokens where four or eight CTAs share K and all their clusters fit on the device (few tiles).  Otherwise the tokens are the rows of a
// tile (a thread of the epilogue owns a row, its scale is one register), on CTA pairs or single CTAs.
#include "common.cuh"
#include "tc05.cuh"
#include "flashrt_b200.h"

namespace frt {

int make_tmap_2d_u8(CUtensorMap* out, const void* base, uint64_t rows, uint64_t row_bytes, uint64_t pitch_bytes, uint32_t box_rows);

namespace f8b {

// ------------------------------------------------------------------------------------------------ quantise groups of 128
//   t = max(max |finite x|, 448e-12),  s = t / 448,  code = e4m3(clamp(x 448 / t, +-448)); infinities are clamped, NaN becomes -448.
// The quotient is the correctly rounded one (Markstein, IBM J. Res. Dev. 34, 1990: the product with the rounded reciprocal, its exact
// remainder, one correction): bf16 values and the largest of them are short enough for quotients that lie exactly between two codes, one
// in some hundred, and a product with 1 / s puts those on either side.
// Eight lanes have a group, 16 values each; U groups a lane, whose loads are all under way at once.  What a row of groups costs beside its
// bytes is the scale, one of four bytes in a line of its own; DOWN: a block has 32 rows of U neighbouring groups, so that scales fill lines.
// Issue is busy for 76 % of the time and memory waits for it: blocks of two groups a lane, six an SM (40 registers), overlap their ends better
// than four of four groups (817 x 16384 9.1 us against 10.1, 8191 x 4096 19.7 against 19.9) or of one (11.0, 24.0); eight bytes a thread spill for it.
struct Quotient {
    uint64_t t, r;                                           // -t / 1024 and its reciprocal, twice: normal numbers for every bf16 t
    __device__ __forceinline__ explicit Quotient(float top) {
        const float s = __fmul_rn(top, 9.765625e-4f), inv = __fdiv_rn(1.0f, s);
        t = f32x2(-s, -s);
        r = f32x2(inv, inv);
    }
    // codes of four values, none infinite
    __device__ __forceinline__ uint32_t operator()(const float* x) const {
        float q[4];
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const uint64_t a = mul_f32x2(f32x2(x[i], x[i + 1]), f32x2(0.4375f, 0.4375f));      // 448 / 1024: three bits, exact
            const uint64_t y = mul_f32x2(a, r);
            f32x2_parts(fma_f32x2(fma_f32x2(y, t, a), r, y), q[i], q[i + 1]);
        }
        return f32x4_to_e4m3x4(clamp448(q[0]), clamp448(q[1]), clamp448(q[2]), clamp448(q[3]));
    }
};

template <int U, bool DOWN>
__global__ void __launch_bounds__(256, U == 2 ? 6 : 1)
quantize_groups_kernel(const __nv_bfloat16* x, long long x_stride, uint8_t* out, float* scale, long long scale_stride, int rows, int dim,
                       int groups) {
    pdl_launch_dependents();
    pdl_wait();
    const int me = threadIdx.x & 7;
    const unsigned slot = threadIdx.x >> 3, across = (unsigned)(groups + U - 1) / U;
    const unsigned block_row = DOWN ? blockIdx.x / across : 0, item = DOWN ? 0 : blockIdx.x * 32u + slot;
    const int row = DOWN ? (int)(block_row * 32u + slot) : (int)(item / (unsigned)groups);
    const int grp = DOWN ? (int)((blockIdx.x - block_row * across) * U) : (int)(item - (unsigned)row * (unsigned)groups);
    const bool wide = ((reinterpret_cast<uintptr_t>(x) | (uintptr_t)(x_stride * 2)) & 31) == 0;
    auto there = [&](int i) { return row < rows && grp + i < groups; };
    auto in = [&](int i) { return there(i) && (grp + i) * 128 + me * 16 < dim; };
    uint32_t v[U][8];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const __nv_bfloat16* src = x + (in(i) ? row * x_stride + (grp + i) * 128 + me * 16 : 0);
        ld_stream_32(src, wide, true, v[i]);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        float f[16], top = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) unpack_bf16x2(in(i) ? v[i][j] : 0u, f[2 * j], f[2 * j + 1]);
#pragma unroll
        for (int j = 0; j < 16; ++j) top = fmaxf(top, fabsf(f[j]));
#pragma unroll
        for (int d = 4; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        if (top == INFINITY) {                               // the group's lanes agree; the finite ones count
            top = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (fabsf(f[j]) < INFINITY) top = fmaxf(top, fabsf(f[j]));
            const unsigned group = 0xffu << (threadIdx.x & 24);
#pragma unroll
            for (int d = 4; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(group, top, d));
            top = fmaxf(top, 448e-12f);
#pragma unroll
            for (int j = 0; j < 16; ++j)                     // clamped: the quotient of the largest
                if (fabsf(f[j]) == INFINITY) f[j] = copysignf(top, f[j]);
        }
        top = fmaxf(top, 448e-12f);
        const Quotient q(top);
        if (in(i)) {
            uint4 o;
            uint32_t* w = &o.x;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = q(f + 4 * j);
            st_global_v4(out + (size_t)row * dim + (grp + i) * 128 + me * 16, o);
        }
        if (me == 0 && there(i)) scale[(grp + i) * scale_stride + row] = __fdiv_rn(top, 448.0f);
        __syncwarp();
    }
}

// ------------------------------------------------------------------------------------------------ products
struct Params {
    void* out;
    const float* a_scale;        // (kb, a_stride)
    long long a_stride;
    const float* w_scale;        // (ceil(N / 128), kb)
    const __nv_bfloat16* bias;
    int* status;
    int M, N, kb;                // kb: k-blocks of 128
    int early;                   // the weights may be read before the kernel in front has ended
    int gm;                      // tile kernel: m-tiles of a group
    int f32;                     // out is fp32
    int tma;                     // tile kernel: rows of D start at 16 bytes
};
enum { ERR_PRODUCER = 1, ERR_MMA = 2, ERR_EPILOGUE = 3 };

template <int CG>
__device__ __forceinline__ void mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 1) {
        tc::mma_f8(tmem_d, adesc, bdesc, idesc, accumulate);
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
    }
}
template <int CG>
__device__ __forceinline__ void tmem_take(uint32_t* slot, uint32_t ncols) {
    if constexpr (CG == 1) {
        tc::tmem_alloc(slot, ncols);
        tc::tmem_relinquish();
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(slot)), "r"(ncols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CG>
__device__ __forceinline__ void tmem_give(uint32_t taddr, uint32_t ncols) {
    if constexpr (CG == 1) tc::tmem_dealloc(taddr, ncols);
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
template <int CG>
__device__ __forceinline__ void load(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int y) {
    if constexpr (CG == 1) {
        tc::tma_load_2d(dst, m, bar, x, y);
    } else {
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
            ::"r"(dst), "l"(m), "r"(bar), "r"(x), "r"(y)
            : "memory");
    }
}
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar, uint32_t leader) {
    if constexpr (CG == 1)
        tc::mma_commit(bar);
    else
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
            "h"((uint16_t)(3u << leader))
            : "memory");
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
__device__ __forceinline__ void sts_v4(uint32_t a, float x, float y, float z, float w) {
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(a), "f"(x), "f"(y), "f"(z), "f"(w) : "memory");
}
__device__ __forceinline__ float4 lds_v4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}
// 8 columns of this thread's TMEM lane
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(taddr) : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t* v) {
    if constexpr (N == 8) tmem_ld8(taddr, v);
    else tc::tmem_ld16(taddr, v);
}
__device__ __forceinline__ void store_one(const Params& p, size_t at, float v) {
    if (p.f32) static_cast<float*>(p.out)[at] = v;
    else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
}

// ------------------------------- weights on the lanes, tokens on the columns: up to 64 rows, or tiles of 96 or 128 whose K four or eight CTAs share
template <int BN>
struct LaneCfg {
    static constexpr int A_BYTES = 128 * 128, B_BYTES = BN * 128, STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int PER_SM = BN <= 64 ? 2 : 1;                          // CTAs: of about 100 KB, or of all there is
    static constexpr int STAGES = BN <= 32 ? 5 : BN == 64 ? 4 : BN == 96 ? 7 : 6;
    static constexpr int BUFS = BN <= 32 ? 8 : 4, BUF_COLS = BN == 96 ? 128 : BN, TMEM_COLS = BUFS * BUF_COLS;      // accumulators: k-blocks under way
    static constexpr int RED_BYTES = 128 * BN * 4;                           // a rank's partial, where the ring was
    static_assert(RED_BYTES <= STAGES * STAGE_BYTES, "partials in the ring");
    static constexpr int HALVES = BN >= 64 ? 2 : 1, W = BN / HALVES;         // four warps of the epilogue for each half of the columns
    static constexpr int THREADS = 32 * (3 + 4 * HALVES);                    // producer, issuer, scales
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + 256 + BUFS * BN * 4;
    static_assert(PER_SM * TMEM_COLS <= 512 && PER_SM * (SMEM_BYTES + 1024) <= 228 * 1024, "CTAs of an SM");
};

// S = 1: grid of as many CTAs as there is room for, each walks over n tiles.  S > 1: grid (n tiles, S, tiles of tokens), cluster (1, S), rank r takes the
// k-blocks [kb r / S, kb (r + 1) / S); the ranks then lay their partials into shared memory and each finishes every S-th four tokens.
template <int BN>
__global__ void __launch_bounds__(LaneCfg<BN>::THREADS, LaneCfg<BN>::PER_SM)
gemm_fp8_block_lane_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW, Params p) {
    using Cfg = LaneCfg<BN>;
    constexpr int STAGES = Cfg::STAGES, BUFS = Cfg::BUFS, W = Cfg::W, LW = (BN == 64 ? 8 : 16);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * Cfg::STAGE_BYTES);
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;       // [BUFS]
    uint64_t* acc_empty = acc_full + BUFS;     // [BUFS]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + BUFS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    static_assert((2 * STAGES + 2 * BUFS) * 8 + 8 <= 256, "barriers");
    const uint32_t scale_a = tc::smem_u32(smem + STAGES * Cfg::STAGE_BYTES + 256);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = (int)gridDim.y, rank = (int)blockIdx.y, tiles = (p.N + 127) / 128;
    const int m0 = (int)blockIdx.z * BN, M = min(p.M - m0, BN);          // the tokens of this CTA
    const int kb0 = (int)((long long)p.kb * rank / S), kb1 = (int)((long long)p.kb * (rank + 1) / S);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            tc::mbar_init(&full[s], 1);
            tc::mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < BUFS; ++i) {
            tc::mbar_init(&acc_full[i], 2);                  // the products, the scales
            tc::mbar_init(&acc_empty[i], 4 * Cfg::HALVES);
        }
        *abort_flag = 0;
        tc::mbar_fence_init();
        tc::tma_prefetch_desc(&tmA);
        tc::tma_prefetch_desc(&tmW);
    }
    if (warp == 1) tmem_take<1>(tmem_slot, Cfg::TMEM_COLS);
    tc::tc_fence_before_sync();
    __syncthreads();
    tc::tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();

    if (warp == 0) {
        // ---------------- producer (whole warp); settled weights: the first ring of them before the wait
        const uint32_t ring = tc::smem_u32(smem), full_a = tc::smem_u32(full), empty_a = tc::smem_u32(empty);
        const int ahead = p.early && (int)blockIdx.x < tiles ? min(STAGES, kb1 - kb0) : 0;
        if (tc::elect_one())
            for (int s = 0; s < ahead; ++s) {
                tc::mbar_arrive_expect_tx(full_a + 8 * s, Cfg::STAGE_BYTES);
                tc::tma_load_2d(ring + s * Cfg::STAGE_BYTES, &tmW, full_a + 8 * s, (kb0 + s) * 128, (int)blockIdx.x * 128);
            }
        __syncwarp();
        pdl_wait();
        if (tc::elect_one())
            for (int s = 0; s < ahead; ++s)
                tc::tma_load_2d(ring + s * Cfg::STAGE_BYTES + Cfg::A_BYTES, &tmA, full_a + 8 * s, (kb0 + s) * 128, m0);
        __syncwarp();
        int s = ahead % STAGES, skip = ahead;
        uint32_t ph = ahead < STAGES;
        for (int t = (int)blockIdx.x; t < tiles; t += (int)gridDim.x) {
            for (int kb = kb0 + skip; kb < kb1; ++kb) {
                if (!tc::warp_wait_limited(empty_a + 8 * s, ph, false, abort_flag)) {
                    if (lane == 0) gave_up(p.status, abort_flag, ERR_PRODUCER);
                    t = tiles;
                    break;
                }
                if (tc::elect_one()) {
                    const uint32_t dst = ring + s * Cfg::STAGE_BYTES, bar = full_a + 8 * s;
                    tc::mbar_arrive_expect_tx(bar, Cfg::STAGE_BYTES);
                    tc::tma_load_2d(dst, &tmW, bar, kb * 128, t * 128);
                    tc::tma_load_2d(dst + Cfg::A_BYTES, &tmA, bar, kb * 128, m0);
                }
                __syncwarp();
                if (++s == STAGES) { s = 0; ph ^= 1; }
            }
            skip = 0;
        }
        // the last stages' returns arrive in this CTA's shared memory too: not after it has gone to another
        for (int i = 0; i < STAGES; ++i) {
            if (!tc::warp_wait_limited(empty_a + 8 * s, ph, false, abort_flag)) break;
            if (++s == STAGES) { s = 0; ph ^= 1; }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (whole warp): a k-block, a buffer
        pdl_wait();                                          // the first stage's limit counts from here
        constexpr uint32_t idesc = tc::make_idesc(0, 0, 0, 0, 128, BN);
        const uint32_t full_a = tc::smem_u32(full), empty_a = tc::smem_u32(empty);
        const uint32_t accF_a = tc::smem_u32(acc_full), accE_a = tc::smem_u32(acc_empty);
        const uint64_t dA0 = tc::make_desc_kmajor_sw128(tc::smem_u32(smem));
        const uint64_t dB0 = tc::make_desc_kmajor_sw128(tc::smem_u32(smem + Cfg::A_BYTES));
        int s = 0, buf = 0;
        uint32_t ph = 0, bph = 1;                              // the first round of the buffers is empty
        for (int t = (int)blockIdx.x; t < tiles; t += (int)gridDim.x)
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!tc::warp_wait_limited(accE_a + 8 * buf, bph, false, abort_flag) ||
                    !tc::warp_wait_limited(full_a + 8 * s, ph, false, abort_flag)) {
                    if (lane == 0) gave_up(p.status, abort_flag, ERR_MMA);
                    t = tiles;
                    break;
                }
                tc::tc_fence_after_sync();
                if (tc::elect_one()) {
                    const uint64_t so = (uint64_t)(s * (Cfg::STAGE_BYTES >> 4));
#pragma unroll
                    for (int k = 0; k < 4; ++k) tc::mma_f8(tmem + buf * Cfg::BUF_COLS, dA0 + so + 2 * k, dB0 + so + 2 * k, idesc, k > 0 ? 1u : 0u);
                    tc::mma_commit(empty_a + 8 * s);
                    tc::mma_commit(accF_a + 8 * buf);
                }
                __syncwarp();
                if (++s == STAGES) { s = 0; ph ^= 1; }
                if (++buf == BUFS) { buf = 0; bph ^= 1; }
            }
    } else if (warp == 2) {
        // ---------------- scales of a k-block, a buffer's beside it: of its tokens times the weights', a lane has every 32nd.  Four blocks'
        // loads are under way.  Tokens behind the last have its scale: what they make of it is not stored.
        pdl_wait();
        constexpr int PER = (BN + 31) / 32;
        struct Scales { float a[PER], w; };
        int row[PER], buf = 0;
        uint32_t bph = 1;
#pragma unroll
        for (int i = 0; i < PER; ++i) row[i] = m0 + min(lane + 32 * i, M - 1);
        for (int t = (int)blockIdx.x; t < tiles; t += (int)gridDim.x) {
            const float* ws = p.w_scale + (size_t)t * p.kb + kb0;
            const float* as = p.a_scale + kb0 * p.a_stride;
            auto ask = [&](int kb, Scales& r) {              // block after block
                if (kb >= kb1) return;
                r.w = *ws++;
#pragma unroll
                for (int i = 0; i < PER; ++i) r.a[i] = as[row[i]];
                as += p.a_stride;
            };
            auto give = [&](const Scales& r) {
                if (!tc::mbar_wait_limited(tc::smem_u32(&acc_empty[buf]), bph, abort_flag)) gave_up(p.status, abort_flag, ERR_EPILOGUE);
                const uint32_t to = scale_a + buf * (BN * 4) + lane * 4;
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    if (BN >= 32 || lane < BN) asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + 128 * i), "f"(__fmul_rn(r.a[i], r.w)) : "memory");
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&acc_full[buf]);
                if (++buf == BUFS) { buf = 0; bph ^= 1; }
            };
            Scales r[4] = {};
#pragma unroll
            for (int i = 0; i < 4; ++i) ask(kb0 + i, r[i]);
            for (int kb = kb0; kb < kb1; kb += 4)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (kb + i < kb1) {
                        give(r[i]);
                        ask(kb + i + 4, r[i]);
                    }
            if (__any_sync(0xffffffffu, *abort_flag != 0)) break;
        }
    } else {
        // ---------------- epilogue: lane quadrant = warp % 4, a thread's lane is one output channel; a half of the tokens
        pdl_wait();
        const int q = warp & 3, half = (warp - 3) >> 2;
        const uint32_t t_src = tmem + ((uint32_t)(q * 32) << 16) + half * W;
        int buf = 0;
        uint32_t bph = 0;
        bool ok = true;
        for (int t = (int)blockIdx.x; t < tiles && ok; t += (int)gridDim.x) {
            const int n = t * 128 + q * 32 + lane;
            float acc[W];
#pragma unroll
            for (int j = 0; j < W; ++j) acc[j] = 0.0f;
            for (int kb = kb0; kb < kb1; ++kb) {
                ok = tc::warp_wait_limited(tc::smem_u32(&acc_full[buf]), bph, false, abort_flag);
                if (!ok) {
                    if (lane == 0) gave_up(p.status, abort_flag, ERR_EPILOGUE);
                    break;
                }
                tc::tc_fence_after_sync();
                const uint32_t src = t_src + buf * Cfg::BUF_COLS, slot = scale_a + buf * (BN * 4) + half * (W * 4);
#pragma unroll
                for (int c = 0; c < W; c += LW) {
                    if (half * W + c >= M) break;
                    uint32_t v[LW];
                    float4 f[LW / 4];
                    tmem_ld<LW>(src + c, v);
#pragma unroll
                    for (int j = 0; j < LW / 4; ++j) f[j] = lds_v4(slot + c * 4 + j * 16);
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < LW; j += 4) {
                        const float4 s = f[j / 4];
                        const uint64_t r0 = fma_f32x2(f32x2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), f32x2(s.x, s.y), f32x2(acc[c + j], acc[c + j + 1]));
                        const uint64_t r1 = fma_f32x2(f32x2(__uint_as_float(v[j + 2]), __uint_as_float(v[j + 3])), f32x2(s.z, s.w), f32x2(acc[c + j + 2], acc[c + j + 3]));
                        f32x2_parts(r0, acc[c + j], acc[c + j + 1]);
                        f32x2_parts(r1, acc[c + j + 2], acc[c + j + 3]);
                    }
                }
                tc::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&acc_empty[buf]);
                if (++buf == BUFS) { buf = 0; bph ^= 1; }
            }
            if (!ok) break;
            if (S > 1) {                                       // [four tokens][channel]: a warp's store is 512 contiguous bytes
                const uint32_t red = tc::smem_u32(smem) + (uint32_t)(half * (W / 4) * 128 + q * 32 + lane) * 16;
#pragma unroll
                for (int j = 0; j < W; j += 4)
                    if (half * W + j < M) sts_v4(red + j * 512, acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
            } else if (n < p.N) {
                const float bias = p.bias ? __bfloat162float(p.bias[n]) : 0.0f;
                const size_t at = (size_t)(m0 + half * W) * p.N + n;
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if (half * W + j < M) store_one(p, at + (size_t)j * p.N, p.bias ? __fadd_rn(acc[j], bias) : acc[j]);
            }
        }
    }
    if (S > 1) {
        // Tensor memory goes back before this CTA waits for its peers: one of them may wait for columns that a cluster of another stream's kernel
        // holds, whose CTA beside this one waits for these.  Between the issuer's arrival and its wait, so that nobody waits for it.
        __syncwarp();
        tc::tc_fence_before_sync();
        if (warp >= 3) asm volatile("barrier.cta.arrive 1, %0;" ::"n"(32 * (1 + 4 * Cfg::HALVES)) : "memory");
        tc::cluster_arrive();
        if (warp == 1) {
            asm volatile("barrier.cta.sync 1, %0;" ::"n"(32 * (1 + 4 * Cfg::HALVES)) : "memory");
            tc::tc_fence_after_sync();
            if (*abort_flag) let_copies_land();
            tmem_give<1>(tmem, Cfg::TMEM_COLS);
        }
        tc::cluster_wait();                                  // all partials are there
        if (warp >= 3 && !*abort_flag) {
            const int q = warp & 3, half = (warp - 3) >> 2, n = (int)blockIdx.x * 128 + q * 32 + lane;
            const bool in = n < p.N;
            const float bias = in && p.bias ? __bfloat162float(p.bias[n]) : 0.0f;
            const uint32_t red = tc::smem_u32(smem) + (uint32_t)(q * 32 + lane) * 16;
            for (int g = rank + S * half; 4 * g < M; g += S * Cfg::HALVES) {   // four tokens; the ranks' partials are all on their way before the first is added
                float4 w[8];
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < S) w[r] = tc::dsmem_ld_f32x4(tc::dsmem_map(red + (uint32_t)g * 2048, (uint32_t)r));
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < S) {                             // in the order of K
                        sum[0] = __fadd_rn(sum[0], w[r].x);
                        sum[1] = __fadd_rn(sum[1], w[r].y);
                        sum[2] = __fadd_rn(sum[2], w[r].z);
                        sum[3] = __fadd_rn(sum[3], w[r].w);
                    }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int m = 4 * g + e;
                    if (in && m < M) store_one(p, (size_t)(m0 + m) * p.N + n, p.bias ? __fadd_rn(sum[e], bias) : sum[e]);
                }
            }
        }
        __syncwarp();
        tc::cluster_sync_all();                              // nobody leaves while its partial is read
    }
    if (*abort_flag && threadIdx.x == 0) let_copies_land();
    if (S > 1) return;
    tc::tc_fence_before_sync();
    __syncthreads();
    tc::tc_fence_after_sync();
    if (warp == 1) tmem_give<1>(tmem, Cfg::TMEM_COLS);
}

// ---------------------------------------------------------------- more rows: tokens on the rows, tiles of 128 CG x BN
constexpr int SCALE_SLOT = 528;       // a buffer's scales: 128 rows, two blocks of weights
template <int CG, int BN>
struct TileCfg {
    static constexpr int A_BYTES = 128 * 128, B_BYTES = BN / CG * 128, STAGE_BYTES = A_BYTES + B_BYTES;  // per CTA
    // a warp's place for stores: 32 rows of its half of the columns in bf16 (half of it, and a stage more where that makes one, waits for the
    // first half's copy in every tile: 8191 x 4096 x 4096 on single CTAs 138 us instead of 129)
    static constexpr int OUT_BYTES = 32 * BN;
    static_assert(OUT_BYTES >= 32 * 32 * 4, "a block of store_block");
    static constexpr int BUFS = 512 / BN;                    // accumulators: k-blocks under way
    static constexpr int REST = 1024 + 256 + 8 * OUT_BYTES + BUFS * SCALE_SLOT;
    static constexpr int FIT = (227 * 1024 - REST) / STAGE_BYTES > 8 ? 8 : (227 * 1024 - REST) / STAGE_BYTES;
    // With 128 columns the waits, four products and two commits of a k-block take a warp longer than the products: two issue, every other
    // block each, with stages and buffers of their own -- of one that both wait for, who is a round ahead would take the phase before for its own.
    static constexpr int ISSUERS = BN == 128 ? 2 : 1;
    static constexpr int STAGES = FIT / ISSUERS * ISSUERS;
    static_assert(BUFS % ISSUERS == 0, "buffers of an issuer");
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + REST;
};

// Tiles in groups of gm m-tiles, m fastest inside a group: the CTAs of a wave then share operand rows in L2.
__device__ __forceinline__ void tile_at(int t, int gm, int m_tiles, int n_tiles, int& m, int& n) {
    const int per = gm * n_tiles, g = t / per, r = t - g * per, h = min(m_tiles - g * gm, gm);
    n = r / h;
    m = g * gm + (r - n * h);
}

// 128 bytes x 32 rows of shared memory (128-byte swizzle) to the output, what lies outside it is left out; x in bytes
__device__ __forceinline__ void store_box(const CUtensorMap* m, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(m), "r"(src), "r"(x), "r"(y) : "memory");
}
// A warp's 32 rows of W columns from registers, a thread holds a row: through its own shared memory to the output by TMA, which goes on while
// the next tile is summed (all SMs reach the ends of their tiles together, and with the stores in the way of the sums 8192 x 8192 x 8192 took
// 4 us a tile more).
template <int W>
__device__ __forceinline__ void store_rows(const Params& p, const CUtensorMap* tmD, const float* acc, int m_base, int nb, uint32_t stg) {
    const int lane = threadIdx.x & 31;
    constexpr int BOX = 32 * 128;
    const uint32_t row = stg + lane * 128, sw = (uint32_t)(lane & 7) << 4;
    const bool wide = p.f32 != 0;
#pragma unroll
    for (int half = 0; half < 2; ++half) {                   // fp32: W / 2 columns fill the warp's place
        if (half == 1 && !wide) continue;
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
#pragma unroll
        for (int c = half * (W / 2); c < W; c += 8) {
            if (half == 0 && c >= W / 2 && wide) continue;
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = acc[c + j];
            if (p.bias) {
                uint4 b = make_uint4(0, 0, 0, 0);
                if (nb + c < p.N) b = ld_global_v4(p.bias + nb + c);         // N % 8 == 0
                const uint32_t* w = &b.x;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float x, y;
                    unpack_bf16x2(w[j], x, y);
                    f[2 * j] = __fadd_rn(f[2 * j], x);
                    f[2 * j + 1] = __fadd_rn(f[2 * j + 1], y);
                }
            }
            if (wide) {
                const uint32_t at = row + (c - half * (W / 2)) / 32 * BOX, k = (uint32_t)(c % 32) * 4;
                sts_v4(at + (k ^ sw), f[0], f[1], f[2], f[3]);
                sts_v4(at + ((k + 16) ^ sw), f[4], f[5], f[6], f[7]);
            } else {
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(row + c / 64 * BOX + (((uint32_t)(c % 64) * 2) ^ sw)), "r"(pack_bf16x2(f[0], f[1])),
                             "r"(pack_bf16x2(f[2], f[3])), "r"(pack_bf16x2(f[4], f[5])), "r"(pack_bf16x2(f[6], f[7])) : "memory");
            }
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        const int n0 = nb + half * (W / 2), per = wide ? 32 : 64, boxes = (wide ? W / 2 : W) / per;
        if (lane == 0 && m_base < p.M) {
            for (int i = 0; i < boxes; ++i)
                if (n0 + i * per < p.N) store_box(tmD, stg + i * BOX, (n0 + i * per) * (wide ? 4 : 2), m_base);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
    }
}

// 32 rows x 32 columns of a tile, a thread holds a row: through shared memory (16-byte chunks of a 128-byte row, chunk index xor row % 8) to
// threads that own four columns of four rows at a time, so that a store covers whole sectors of a row.
__device__ __forceinline__ void store_block(const Params& p, const float* f, int m_base, int nb, uint8_t* stg, bool vec) {
    const int lane = threadIdx.x & 31, ch = lane & 7, r0 = lane >> 3, n = nb + ch * 4;
    const uint32_t base = tc::smem_u32(stg), sw = (uint32_t)(lane & 7) << 4;
#pragma unroll
    for (int k = 0; k < 8; ++k) sts_v4(base + lane * 128 + (((uint32_t)k << 4) ^ sw), f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
    if (!vec) {
        // rows that start anywhere: a lane takes a column, a store two to three sectors of one row
        const int col = nb + lane;
        const float bias = p.bias && col < p.N ? __bfloat162float(p.bias[col]) : 0.0f;
        __syncwarp();
        const int rows = min(32, p.M - m_base);
#pragma unroll 8
        for (int r = 0; r < 32; ++r) {
            float v;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(base + r * 128 + ((uint32_t)((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) : "memory");
            if (p.bias) v = __fadd_rn(v, bias);
            if (r < rows && col < p.N) store_one(p, (size_t)(m_base + r) * p.N + col, v);
        }
        __syncwarp();
        return;
    }
    float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p.bias && n < p.N)
#pragma unroll
        for (int e = 0; e < 4; ++e) bias[e] = __bfloat162float(p.bias[n + e]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + r0, m = m_base + r;
        float4 v = lds_v4(base + r * 128 + ((uint32_t)(ch ^ (r & 7)) << 4));
        if (p.bias) {
            v.x = __fadd_rn(v.x, bias[0]);
            v.y = __fadd_rn(v.y, bias[1]);
            v.z = __fadd_rn(v.z, bias[2]);
            v.w = __fadd_rn(v.w, bias[3]);
        }
        if (m < p.M && n < p.N) {                            // N % 4 == 0: all four
            const size_t at = (size_t)m * p.N + n;
            if (p.f32) *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = v;
            else st_global_v2(static_cast<__nv_bfloat16*>(p.out) + at, make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w)));
        }
    }
    __syncwarp();
}

// CG = 2: a CTA pair has a tile of 256 rows, each CTA stages its 128 rows of A and half of the weight rows.  S > 1: a cluster of S such
// takes one tile, unit s the k-blocks [kb s / S, kb (s + 1) / S); they then lay their partials into shared memory, where their rings were,
// and each finishes BN / S of the columns.
constexpr int TILE_THREADS = 384;     // producer, issuer, scales, second issuer or none; eight warps of the epilogue
template <int CG, int BN, int S>
__global__ void __launch_bounds__(TILE_THREADS, 1)
gemm_fp8_block_tile_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmD, Params p) {
    using Cfg = TileCfg<CG, BN>;
    constexpr int STAGES = Cfg::STAGES, BUFS = Cfg::BUFS, ISSUERS = Cfg::ISSUERS, W2 = BN / 2, LW = BN == 256 ? 8 : 16;
    static_assert(S == 1 || (BN / S >= 64 && 128 * BN * 4 <= STAGES * Cfg::STAGE_BYTES), "columns of a half of the warps, partials in the ring");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* outs = smem + STAGES * Cfg::STAGE_BYTES;        // 1024-byte boundaries, for the swizzle of the stores
    uint64_t* full = reinterpret_cast<uint64_t*>(outs + 8 * Cfg::OUT_BYTES);   // the leader's count both CTAs' bytes
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;       // [BUFS]
    uint64_t* acc_empty = acc_full + BUFS;     // [BUFS] the leader's
    uint64_t* scale_empty = acc_empty + BUFS;  // [BUFS]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(scale_empty + BUFS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    static_assert((2 * STAGES + 3 * BUFS) * 8 + 8 <= 256, "barriers");
    const uint32_t scale_a = tc::smem_u32(outs + 8 * Cfg::OUT_BYTES + 256);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t cluster_rank = CG * S > 1 ? tc::cluster_ctarank() : 0u, rank = cluster_rank % CG, leader = cluster_rank - rank;
    const int split = (int)cluster_rank / CG;
    const int unit = (int)blockIdx.x / (CG * S), units = (int)gridDim.x / (CG * S);     // S > 1: as many as tiles
    const int kb0 = S == 1 ? 0 : (int)((long long)p.kb * split / S), kb1 = S == 1 ? p.kb : (int)((long long)p.kb * (split + 1) / S);
    const int m_tiles = (p.M + 128 * CG - 1) / (128 * CG), n_tiles = (p.N + BN - 1) / BN, total = m_tiles * n_tiles;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            tc::mbar_init(&full[s], 1);
            tc::mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < BUFS; ++i) {
            tc::mbar_init(&acc_full[i], 2);                  // the products, the scales
            tc::mbar_init(&scale_empty[i], 8);
            tc::mbar_init(&acc_empty[i], CG * 8);
        }
        *abort_flag = 0;
        tc::mbar_fence_init();
        tc::tma_prefetch_desc(&tmA);
        tc::tma_prefetch_desc(&tmW);
    }
    if (warp == 1) tmem_take<CG>(tmem_slot, 512);
    tc::tc_fence_before_sync();
    if constexpr (CG * S > 1) tc::cluster_sync_all();        // the CTAs' barriers exist before anything signals across
    else __syncthreads();
    tc::tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();

    if (warp == 0) {
        // ---------------- producer of this CTA's rows, bytes counted at the leader; settled weights: the first ring of them before the wait
        const uint32_t ring = tc::smem_u32(smem), empty_a = tc::smem_u32(empty), full_a = tc::smem_u32(full);
        const uint32_t lead_full = CG == 1 ? full_a : tc::dsmem_map(full_a, leader);
        const int ahead = p.early && unit < total ? min(STAGES, kb1 - kb0) : 0;
        int s = 0;
        if (ahead) {
            int mt, nt;
            tile_at(unit, p.gm, m_tiles, n_tiles, mt, nt);
            if (tc::elect_one())
                for (int i = 0; i < ahead; ++i) {
                    if (rank == 0) tc::mbar_arrive_expect_tx(full_a + 8 * i, CG * Cfg::STAGE_BYTES);
                    load<CG>(ring + i * Cfg::STAGE_BYTES + Cfg::A_BYTES, &tmW, lead_full + 8 * i, (kb0 + i) * 128, nt * BN + (int)rank * (BN / CG));
                }
            __syncwarp();
            pdl_wait();
            if (tc::elect_one())
                for (int i = 0; i < ahead; ++i)
                    load<CG>(ring + i * Cfg::STAGE_BYTES, &tmA, lead_full + 8 * i, (kb0 + i) * 128, (mt * CG + (int)rank) * 128);
            __syncwarp();
            s = ahead % STAGES;
        } else {
            pdl_wait();
        }
        int skip = ahead;
        uint32_t ph = ahead < STAGES;
        bool ready = false;                                  // the first wait looks for itself
        for (int t = unit; t < total; t += units) {
            int mt, nt;
            tile_at(t, p.gm, m_tiles, n_tiles, mt, nt);
            const int m0 = (mt * CG + (int)rank) * 128, n0 = nt * BN + (int)rank * (BN / CG);
            for (int kb = kb0 + skip; kb < kb1; ++kb) {
                if (!tc::warp_wait_limited(empty_a + 8 * s, ph, ready, abort_flag)) {
                    if (lane == 0) gave_up(p.status, abort_flag, ERR_PRODUCER);
                    t = total;
                    break;
                }
                const uint32_t dst = ring + s * Cfg::STAGE_BYTES, bar = lead_full + 8 * s, own = full_a + 8 * s;
                if (++s == STAGES) { s = 0; ph ^= 1; }
                ready = tc::mbar_test(empty_a + 8 * s, ph);
                if (tc::elect_one()) {
                    if (rank == 0) tc::mbar_arrive_expect_tx(own, CG * Cfg::STAGE_BYTES);
                    load<CG>(dst, &tmA, bar, kb * 128, m0);
                    load<CG>(dst + Cfg::A_BYTES, &tmW, bar, kb * 128, n0);
                }
            }
            skip = 0;
        }
        // the last stages' returns arrive in this CTA's shared memory too: not after it has gone to another
        for (int i = 0; i < STAGES; ++i) {
            if (!tc::warp_wait_limited(empty_a + 8 * s, ph, false, abort_flag)) break;
            if (++s == STAGES) { s = 0; ph ^= 1; }
        }
    } else if ((warp & 1) && warp < 2 * ISSUERS && rank == 0) {
        // ---------------- MMA issuers for the tiles, warps 1 and (two issuers) 3: a k-block, a buffer
        pdl_wait();                                          // the first stage's limit counts from here
        constexpr uint32_t idesc = tc::make_idesc(0, 0, 0, 0, 128 * CG, BN);
        const uint64_t dA0 = tc::make_desc_kmajor_sw128(tc::smem_u32(smem));
        const uint64_t dB0 = tc::make_desc_kmajor_sw128(tc::smem_u32(smem + Cfg::A_BYTES));
        const uint32_t full_a = tc::smem_u32(full), empty_a = tc::smem_u32(empty);
        const uint32_t accF_a = tc::smem_u32(acc_full), accE_a = tc::smem_u32(acc_empty);
        const int mine = unit < total ? ((total - 1 - unit) / units + 1) * (kb1 - kb0) : 0;       // k-blocks of this unit's tiles
        int s = warp >> 1, buf = warp >> 1;
        uint32_t ph = 0, bph = 1;                            // the first round of the buffers is empty
        bool ready = false;
        for (int i = warp >> 1; i < mine; i += ISSUERS) {
            if (!tc::warp_wait_limited(full_a + 8 * s, ph, ready, abort_flag) ||
                !tc::warp_wait_limited(accE_a + 8 * buf, bph, false, abort_flag)) {
                if (lane == 0) gave_up(p.status, abort_flag, ERR_MMA);
                break;
            }
            tc::tc_fence_after_sync();
            const uint64_t so = (uint64_t)(s * (Cfg::STAGE_BYTES >> 4));
            const uint32_t done = empty_a + 8 * s, there = accF_a + 8 * buf, d_tm = tmem + buf * BN;
            s += ISSUERS;
            if (s >= STAGES) { s -= STAGES; ph ^= 1; }
            buf += ISSUERS;
            if (buf >= BUFS) { buf -= BUFS; bph ^= 1; }
            ready = tc::mbar_test(full_a + 8 * s, ph);
            if (tc::elect_one()) {
#pragma unroll
                for (int k = 0; k < 4; ++k) mma<CG>(d_tm, dA0 + so + 2 * k, dB0 + so + 2 * k, idesc, k > 0 ? 1u : 0u);
                commit<CG>(done, leader);
                commit<CG>(there, leader);
            }
        }
    } else if (warp == 2) {
        // ---------------- scales of this CTA's rows and of the tile's two blocks of weights, a buffer's beside it: a lane has four rows.  Four
        // blocks' loads are under way; whoever takes them from a register that a loop moves on waits for them a block earlier.  Rows behind the
        // last have its scale: what they make of it is not stored.
        pdl_wait();
        struct Scales { float a[4], w; };
        int buf = 0;
        uint32_t bph = 1;
        for (int t = unit; t < total; t += units) {
            int mt, nt;
            tile_at(t, p.gm, m_tiles, n_tiles, mt, nt);
            const int m0 = (mt * CG + (int)rank) * 128 + 4 * lane;
            int row[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) row[i] = min(m0 + i, p.M - 1);
            const float* ws = p.w_scale + (size_t)(min(nt * BN + (lane & 1) * W2, p.N - 1) / 128) * p.kb + kb0;
            const float* as = p.a_scale + kb0 * p.a_stride;
            auto ask = [&](int kb, Scales& r) {              // block after block
                if (kb >= kb1) return;
                r.w = *ws++;
#pragma unroll
                for (int i = 0; i < 4; ++i) r.a[i] = as[row[i]];
                as += p.a_stride;
            };
            auto give = [&](const Scales& r) {
                if (!tc::mbar_wait_limited(tc::smem_u32(&scale_empty[buf]), bph, abort_flag)) gave_up(p.status, abort_flag, ERR_EPILOGUE);
                const uint32_t to = scale_a + buf * SCALE_SLOT;
                sts_v4(to + lane * 16, r.a[0], r.a[1], r.a[2], r.a[3]);
                if (lane < 2) asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + 512 + lane * 4), "f"(r.w) : "memory");
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&acc_full[buf]);
                if (++buf == BUFS) { buf = 0; bph ^= 1; }
            };
            Scales r[4] = {};
#pragma unroll
            for (int i = 0; i < 4; ++i) ask(kb0 + i, r[i]);
            for (int kb = kb0; kb < kb1; kb += 4)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (kb + i < kb1) {
                        give(r[i]);
                        ask(kb + i + 4, r[i]);
                    }
            if (__any_sync(0xffffffffu, *abort_flag != 0)) break;
        }
    } else if (warp >= 4) {
        // ---------------- epilogue: this CTA's 128 rows; a warp's lane quadrant and half of the columns
        pdl_wait();
        const int q = warp & 3, half = (warp - 4) >> 2;
        const uint32_t t_src = tmem + ((uint32_t)(q * 32) << 16);
        uint8_t* stg = outs + (warp - 4) * Cfg::OUT_BYTES;
        const uint32_t accF_a = tc::smem_u32(acc_full), accE_a = tc::smem_u32(acc_empty);
        const uint32_t accE_lead = CG == 1 ? accE_a : tc::dsmem_map(accE_a, leader);
        int buf = 0;
        uint32_t bph = 0;
        for (int t = unit; t < total; t += units) {
            int mt, nt;
            tile_at(t, p.gm, m_tiles, n_tiles, mt, nt);
            const int m_base = (mt * CG + (int)rank) * 128 + q * 32, n_base = nt * BN + half * W2;
            float acc[W2];
#pragma unroll
            for (int j = 0; j < W2; ++j) acc[j] = 0.0f;
            bool ok = true;
            for (int kb = kb0; kb < kb1; ++kb) {
                ok = tc::warp_wait_limited(accF_a + 8 * buf, bph, false, abort_flag);
                if (!ok) {
                    if (lane == 0) gave_up(p.status, abort_flag, ERR_EPILOGUE);
                    break;
                }
                tc::tc_fence_after_sync();
                float a, w_s;
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(a) : "r"(scale_a + buf * SCALE_SLOT + (q * 32 + lane) * 4) : "memory");
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(w_s) : "r"(scale_a + buf * SCALE_SLOT + 512 + half * 4) : "memory");
                const float s = __fmul_rn(a, w_s);
                const uint64_t s2 = f32x2(s, s);
                const uint32_t src = t_src + buf * BN + half * W2;
                // LW columns on their way from tensor memory while the LW in front are added: eight, where 128 sums leave registers for no more
                // (16 spill: 138 us instead of 125 at 8191 x 4096 x 4096)
                uint32_t v[2][LW];
                tmem_ld<LW>(src, v[0]);
#pragma unroll
                for (int c = 0; c < W2; c += LW) {
                    tc::tmem_ld_wait();
                    if (c + LW < W2) {
                        tmem_ld<LW>(src + c + LW, v[(c / LW + 1) & 1]);
                    } else {                                 // all is taken: the buffer may be filled again
                        tc::tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) {
                            if constexpr (CG == 1) tc::mbar_arrive(&acc_empty[buf]);
                            else tc::mbar_arrive_cluster(accE_lead + 8 * buf);
                            tc::mbar_arrive(&scale_empty[buf]);
                        }
                    }
                    const uint32_t* w = v[(c / LW) & 1];
#pragma unroll
                    for (int j = 0; j < LW; j += 2) {
                        const uint64_t r = fma_f32x2(f32x2(__uint_as_float(w[j]), __uint_as_float(w[j + 1])), s2, f32x2(acc[c + j], acc[c + j + 1]));
                        f32x2_parts(r, acc[c + j], acc[c + j + 1]);
                    }
                }
                if (++buf == BUFS) { buf = 0; bph ^= 1; }
            }
            if (!ok) break;
            if constexpr (S > 1) {                           // [four columns][row]: a warp's store is 512 contiguous bytes
                const uint32_t red = tc::smem_u32(smem) + (half * (W2 / 4) * 128 + q * 32 + lane) * 16;
#pragma unroll
                for (int j = 0; j < W2; j += 4) sts_v4(red + j * 512, acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
                break;
            } else {
                if (p.tma) store_rows<W2>(p, &tmD, acc, m_base, n_base, tc::smem_u32(stg));
                else
#pragma unroll
                    for (int c = 0; c < W2; c += 32)
                        if (m_base < p.M && n_base + c < p.N) store_block(p, acc + c, m_base, n_base + c, stg, false);
            }
        }
    }
    if constexpr (S > 1) {
        __syncwarp();
        tc::cluster_sync_all();                // all partials are there
        if (warp >= 4 && !*abort_flag) {
            constexpr int W = BN / S / 2;      // columns of this warp
            const int q = warp & 3, half = (warp - 4) >> 2, col = split * (BN / S) + half * W;
            int mt, nt;
            tile_at(unit, p.gm, m_tiles, n_tiles, mt, nt);
            const int m_base = (mt * CG + (int)rank) * 128 + q * 32, n_base = nt * BN + col;
            uint8_t* stg = outs + (warp - 4) * Cfg::OUT_BYTES;
            const uint32_t red = tc::smem_u32(smem) + (uint32_t)(col / 4 * 128 + q * 32 + lane) * 16;
#pragma unroll 1
            for (int c = 0; c < W; c += 32) {
                float v[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = 0.0f;
#pragma unroll
                for (int s = 0; s < S; ++s) {                // in the order of K
                    const uint32_t from = tc::dsmem_map(red + (uint32_t)c * 512, (uint32_t)(CG * s) + rank);
                    float4 w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = tc::dsmem_ld_f32x4(from + (uint32_t)j * 2048);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        v[4 * j] = __fadd_rn(v[4 * j], w[j].x);
                        v[4 * j + 1] = __fadd_rn(v[4 * j + 1], w[j].y);
                        v[4 * j + 2] = __fadd_rn(v[4 * j + 2], w[j].z);
                        v[4 * j + 3] = __fadd_rn(v[4 * j + 3], w[j].w);
                    }
                }
                if (m_base < p.M && n_base + c < p.N) store_block(p, v, m_base, n_base + c, stg, (p.N & 3) == 0);
            }
        }
    }
    if (*abort_flag && threadIdx.x == 0) let_copies_land();
    if (warp >= 4 && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
    tc::tc_fence_before_sync();
    if constexpr (CG * S > 1) tc::cluster_sync_all();        // the leader's MMAs read the peer's shared memory until the end
    else __syncthreads();
    tc::tc_fence_after_sync();
    if (warp == 1) tmem_give<CG>(tmem, 512);
}

// ------------------------------------------------------------------------------------------------ host
static void set_attrs(cudaLaunchConfig_t& cfg, cudaLaunchAttribute (&attr)[2], unsigned cx, unsigned cy, cudaStream_t stream) {
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cx;
    attr[0].val.clusterDim.y = cy;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
}

template <int BN>
static int launch_lane(const void* A, const void* W, Params p, int K, int splits, cudaStream_t stream) {
    using Cfg = LaneCfg<BN>;
    static PerDeviceOnce once;
    CUtensorMap tmA, tmW;
    int dev = 0;
    if (once.need(dev)) {
        const cudaError_t e = cudaFuncSetAttribute(gemm_fp8_block_lane_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES);
        if (e != cudaSuccess) return FRT_CUDA_ERR(e);
        once.set(dev);
    }
    int rc = make_tmap_2d_u8(&tmA, A, (uint64_t)p.M, (uint64_t)K, (uint64_t)K, BN);
    if (!rc) rc = make_tmap_2d_u8(&tmW, W, (uint64_t)p.N, (uint64_t)K, (uint64_t)K, 128);
    if (rc) return rc;
    const int tiles = (p.N + 127) / 128, room = Cfg::PER_SM * device_sm_count();
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = dim3(splits > 1 || tiles < room ? tiles : room, splits, (unsigned)((p.M + BN - 1) / BN));       // S = 1: one tile of tokens
    cfg.blockDim = dim3(Cfg::THREADS);
    cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
    set_attrs(cfg, attr, 1, (unsigned)splits, stream);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, gemm_fp8_block_lane_kernel<BN>, tmA, tmW, p);
    return e == cudaSuccess ? FRT_OK : FRT_CUDA_ERR(e);
}

template <int CG, int BN, int S>
static int launch_tile(const void* A, const void* W, Params p, int K, cudaStream_t stream) {
    using Cfg = TileCfg<CG, BN>;
    static PerDeviceOnce once;
    CUtensorMap tmA, tmW, tmD;
    int dev = 0;
    if (once.need(dev)) {
        const cudaError_t e = cudaFuncSetAttribute(gemm_fp8_block_tile_kernel<CG, BN, S>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES);
        if (e != cudaSuccess) return FRT_CUDA_ERR(e);
        once.set(dev);
    }
    int rc = make_tmap_2d_u8(&tmA, A, (uint64_t)p.M, (uint64_t)K, (uint64_t)K, 128);
    if (!rc) rc = make_tmap_2d_u8(&tmW, W, (uint64_t)p.N, (uint64_t)K, (uint64_t)K, BN / CG);
    const uint64_t out_row = (uint64_t)p.N * (p.f32 ? 4 : 2);
    // Rows at 16 bytes, bias read so, and a byte's place in a row is a 32-bit coordinate.  Otherwise values are stored one by one and nothing is
    // summed meanwhile: 80 x 50257 x 2048 40 us (50256: 28, fp32 30.5), 384 rows 70 (46, 52), 2000 325 (215, 224), 8191 x 50257 x 512 831 (313, 404).
    p.tma = p.N % 8 == 0 && (reinterpret_cast<uintptr_t>(p.bias) & 15) == 0 && out_row <= 1u << 31;
    if (!rc && p.tma) rc = make_tmap_2d_u8(&tmD, p.out, (uint64_t)p.M, out_row, out_row, 32);
    if (!p.tma) tmD = tmA;
    if (rc) return rc;
    const int m_tiles = (p.M + 128 * CG - 1) / (128 * CG), n_tiles = (p.N + BN - 1) / BN, workers = device_sm_count() / CG;
    const long long total = (long long)m_tiles * n_tiles;
    if (total > 1 << 30) return FRT_ERR_UNSUPPORTED;
    // rows of A and of W that a wave reads: 128 CG gm and BN workers / gm, fewest when they are alike
    p.gm = 1;
    if (total <= workers) p.gm = m_tiles;
    else
        while (p.gm < m_tiles && (long long)(p.gm + 1) * (p.gm + 1) * 128 * CG <= (long long)BN * workers) ++p.gm;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = dim3(CG * (S > 1 ? S * (unsigned)total : (unsigned)(total < workers ? total : workers)));
    cfg.blockDim = dim3(TILE_THREADS);
    cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
    set_attrs(cfg, attr, CG * S, 1, stream);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, gemm_fp8_block_tile_kernel<CG, BN, S>, tmA, tmW, tmD, p);
    return e == cudaSuccess ? FRT_OK : FRT_CUDA_ERR(e);
}

// Clusters of a sharing form that the device holds at once (a cluster lies in one GPC, whose SMs its size need not divide): asked once.
template <int SMEM, typename K>
static long long clusters_held(int (&known)[64], K kernel, dim3 cluster, int threads) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    if (!known[dev]) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = cluster;
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = SMEM;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = cluster.x;
        attr[0].val.clusterDim.y = cluster.y;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
        if (e != cudaSuccess) {
            cudaGetLastError();                              // not this launch's error: the form is not offered
            n = 0;
        }
        known[dev] = n + 1;
    }
    return known[dev] - 1;
}
template <int CG, int BN, int S>
static long long tile_clusters() {
    static int known[64] = {0};
    return clusters_held<TileCfg<CG, BN>::SMEM_BYTES>(known, gemm_fp8_block_tile_kernel<CG, BN, S>, dim3(CG * S), TILE_THREADS);
}
template <int BN, int S>
static long long lane_clusters() {
    static int known[64] = {0};
    return clusters_held<LaneCfg<BN>::SMEM_BYTES>(known, gemm_fp8_block_lane_kernel<BN>, dim3(1, S), LaneCfg<BN>::THREADS);
}

template <int U, bool DOWN>
static int launch_quantize(const void* x, long long stride, void* out, float* scale, long long scale_stride, int rows, int dim, cudaStream_t stream) {
    const int groups = (dim + 127) / 128;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(DOWN ? (unsigned)((rows + 31) / 32) * (unsigned)((groups + U - 1) / U) : ((unsigned)rows * (unsigned)groups + 31u) / 32u);
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, quantize_groups_kernel<U, DOWN>, static_cast<const __nv_bfloat16*>(x), stride,
                                             static_cast<uint8_t*>(out), scale, scale_stride, rows, dim, groups);
    return e == cudaSuccess ? FRT_OK : FRT_CUDA_ERR(e);
}

}  // namespace f8b
}  // namespace frt

static bool misaligned(const void* a, uintptr_t n) { return (reinterpret_cast<uintptr_t>(a) & (n - 1)) != 0; }

extern "C" int frt_b200_quantize_fp8_groups(const void* in_bf16, long long in_stride, void* out8, float* group_scale, long long scale_stride,
                                            int rows, int dim, int flags, void* stream) {
    using namespace frt;
    (void)flags;
    if (rows < 0 || dim < 0 || in_stride < dim || in_stride % 8 || scale_stride < rows) return FRT_ERR_INVALID;
    if (dim % 16 || (long long)rows * ((dim + 127) / 128) > 1 << 30) return FRT_ERR_UNSUPPORTED;
    if (rows == 0 || dim == 0) return FRT_OK;
    if (!in_bf16 || !out8 || !group_scale) return FRT_ERR_INVALID;
    if (misaligned(in_bf16, 16) || misaligned(out8, 16) || misaligned(group_scale, 4)) return FRT_ERR_INVALID;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows < 32) return f8b::launch_quantize<1, false>(in_bf16, in_stride, out8, group_scale, scale_stride, rows, dim, st);
    const bool few = (long long)rows * ((dim + 127) / 128) < 256ll * device_sm_count();
    if (few) return f8b::launch_quantize<1, true>(in_bf16, in_stride, out8, group_scale, scale_stride, rows, dim, st);
    return f8b::launch_quantize<2, true>(in_bf16, in_stride, out8, group_scale, scale_stride, rows, dim, st);
}

extern "C" int frt_b200_gemm_fp8_block_nt(const void* A, const void* W, void* D, int M, int N, int K, const float* a_scale,
                                          long long a_scale_stride, const float* w_scale, const void* bias, int flags, void* stream) {
    using namespace frt;
    if (M < 0 || N < 0 || K < 1 || a_scale_stride < M) return FRT_ERR_INVALID;
    if (K % 16 || K > 1 << 20 || M > 1 << 30 || N > 1 << 30) return FRT_ERR_UNSUPPORTED;
    if (M == 0 || N == 0) return FRT_OK;
    if (!A || !W || !D || !a_scale || !w_scale) return FRT_ERR_INVALID;
    if (misaligned(A, 16) || misaligned(W, 16) || misaligned(D, 16) || misaligned(a_scale, 4) || misaligned(w_scale, 4) || misaligned(bias, 2))
        return FRT_ERR_INVALID;
    f8b::Params p = {};
    p.out = D;
    p.a_scale = a_scale;
    p.a_stride = a_scale_stride;
    p.w_scale = w_scale;
    p.bias = static_cast<const __nv_bfloat16*>(bias);
    static PerDevicePointer status;
    p.status = status.get(gemm_status_device_ptr);
    if (!p.status) return FRT_ERR_UNSUPPORTED;
    p.M = M;
    p.N = N;
    p.kb = (K + 127) / 128;
    p.early = flags & 1;
    p.f32 = flags & 2;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int sms = device_sm_count(), n128 = (N + 127) / 128, n256 = (N + 255) / 256;
    if (M <= 64) {
        // K splits (a cluster) while the tiles alone leave SMs idle and every rank keeps two k-blocks.  A cluster lies in one GPC, so 33 of eight and
        // 69 to 71 of four fit at two CTAs an SM: where this asks for a few more (34 to 37 tiles, 72 to 74), the last run behind the first (one
        // row, K 3584: 4224 columns 6.8 us, 4352 to 4736 10.6 to 10.9, 4864 7.1; 8832 8.9, 9216 to 9472 13.3, 9600 9.5).
        int splits = 1;
        while (splits < 8 && n128 * splits * 2 <= 2 * sms && p.kb / (splits * 2) >= 2) splits *= 2;
        if (M <= 16) return f8b::launch_lane<16>(A, W, p, K, splits, st);
        if (M <= 32) return f8b::launch_lane<32>(A, W, p, K, splits, st);
        return f8b::launch_lane<64>(A, W, p, K, splits, st);
    }
    // The cheapest of the forms: whole waves of tiles, k-blocks of a tile, the microseconds of one and of what a tile takes besides; where K is
    // shared, the exchange, and only if the device holds all clusters at once.  Measured at 128 x 4096 x 4096 (12 us in 128-column tiles, 10 with
    // K shared by two, 18 in 256-column ones), 256 x 2048 x 8192 (20 on pairs of 128 columns, 13 with K shared by two), 817 x 2048 x 16384 (66 in
    // 256-column tiles, 40 with K shared by two), 8191 x 4096 x 4096 (125 on pairs of 256 columns, 129 on single CTAs, 162 on pairs of 128).
    // A k-block's time is that of products; where memory is slower (96 x 32768 x 2048: 0.7 us a k-block, 128 CTAs at 32 KB, 0.64 at the copy rate)
    // all forms read the same weights, and whole waves decide.
    const long long m128 = (M + 127) / 128, m256 = (M + 255) / 256;
    double best = 1e30;
    int form = 0;
    auto offer = [&](int f, long long tiles, int ctas, int S, double per_kb, double exchange, long long (*clusters)()) {
        const long long room = sms / ctas, waves = S == 1 ? (tiles + room - 1) / room : 1;
        const double cost = (double)waves * ((p.kb + S - 1) / S * per_kb + 2.0) + exchange;
        if (cost < best && (S == 1 || (p.kb >= 4 * S && tiles <= clusters()))) { best = cost; form = f; }
    };
    offer(0, m256 * n256, 2, 1, 0.47, 0.0, nullptr);
    offer(1, m128 * n256, 1, 1, 0.50, 0.0, nullptr);
    offer(2, m256 * n128, 2, 1, 0.30, 0.8, nullptr);         // the pair's signals: 512 x 2048 x 2048 7.8 against 7.4 on single CTAs
    offer(3, m128 * n128, 1, 1, 0.345, 0.0, nullptr);
    offer(4, m128 * n128, 1, 2, 0.345, 2.5, f8b::tile_clusters<1, 128, 2>);
    offer(5, m256 * n128, 2, 2, 0.30, 3.8, f8b::tile_clusters<2, 128, 2>);
    offer(6, m128 * n256, 1, 2, 0.50, 5.0, f8b::tile_clusters<1, 256, 2>);
    offer(7, m128 * n256, 1, 4, 0.50, 7.0, f8b::tile_clusters<1, 256, 4>);
    // K shared by four or eight with the weights on the lanes, tiles of 96 or 128 tokens: 96 x 4096 x 4096 8.4 us against 9.5, 96 x 4096 x 14336 20
    // against 28, 129 x 2048 x 16384 18 against 30; by two, or by none, no gain (96 x 6144 x 4096 11.9 against
    // 11.2), and where the clusters do not all fit a loss (96 x 2048 x 2048 by eight 11, by four 6)
    const bool of96 = (M + 95) / 96 == m128;
    offer(8, m128 * n128, 1, 4, of96 ? 0.34 : 0.40, 2.7, of96 ? f8b::lane_clusters<96, 4> : f8b::lane_clusters<128, 4>);
    offer(9, m128 * n128, 1, 8, of96 ? 0.34 : 0.40, 2.7, of96 ? f8b::lane_clusters<96, 8> : f8b::lane_clusters<128, 8>);
    switch (form) {
        case 8: return of96 ? f8b::launch_lane<96>(A, W, p, K, 4, st) : f8b::launch_lane<128>(A, W, p, K, 4, st);
        case 9: return of96 ? f8b::launch_lane<96>(A, W, p, K, 8, st) : f8b::launch_lane<128>(A, W, p, K, 8, st);
        case 1: return f8b::launch_tile<1, 256, 1>(A, W, p, K, st);
        case 2: return f8b::launch_tile<2, 128, 1>(A, W, p, K, st);
        case 3: return f8b::launch_tile<1, 128, 1>(A, W, p, K, st);
        case 4: return f8b::launch_tile<1, 128, 2>(A, W, p, K, st);
        case 5: return f8b::launch_tile<2, 128, 2>(A, W, p, K, st);
        case 6: return f8b::launch_tile<1, 256, 2>(A, W, p, K, st);
        case 7: return f8b::launch_tile<1, 256, 4>(A, W, p, K, st);
        default: return f8b::launch_tile<2, 256, 1>(A, W, p, K, st);
    }
}

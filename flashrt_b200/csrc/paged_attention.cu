// Attention of new tokens over a paged E4M3 key/value cache (one scale per block and head), causal, ragged batches.
//
// No counterpart in the reference (its attention reads dense 16-bit K and V: csrc/attention/fa2_wrapper.cu).
//
// With c the stored codes, k_j = ks_p c_j and v_j = vs_p c_j (p: the page of key j), all in base 2:
//   t_ij = q_i . c_j * (softmax_scale * log2(e) * ks_p)        [capped: cap * tanh(s / cap)]
//   u_ij = t_ij + log2(vs_p),  m_i = max_j u_ij,  w_ij = 2^(u_ij - m_i + 15)
//   o_i = (sum_j w_ij c_j) / l_i,  l_i = sum_j w_ij / vs_p,  lse_i = ln 2 (m_i - 15 + log2 l_i)
// The values' scale goes into the exponent, so a weight that meets the codes is at most 2^15 whatever the scales are: it is rounded to
// fp16 (2^-12 relative down to 2^-29 of the largest; bf16 weights would give up four bits) while every sum stays in fp32.  E4M3 codes
// are fp16 values exactly; queries are brought to at most 1 by a power of two per row, which is exact too (elements under 2^-24 of
// the row's largest lose bits).
//
// What bounds it: a decode step reads every key and value once and does 4 x group flops per byte, so memory does, and the kernel is
// built to keep copies in flight.  Every warp works alone: it owns a ring of slots (KT keys and their values, 8 KB each) that it fills
// itself by TMA, two or three tiles ahead and across the items of its work, so neither the join of an item's warps nor the set-up of
// the next one lets the memory wait.  (The form before loaded into registers, one tile ahead: 64 sequences of 1500 .. 6000 tokens, 32
// heads on 8 of 128: 142 us, memory 42 % busy, every second cycle of a warp spent on a load.)
// Codes go from shared memory to the tensor cores as fp16: keys are the M rows of K . Q^T and dimensions the M rows of V^T . P^T
// (mma.sync m16n8k16), so a group of up to eight query rows fills the N side and no tensor work is wasted.  Which dimension a k index
// stands for is free, hence a lane's 16 contiguous bytes serve four k steps; the pairs of keys that V^T wants side by side come from
// one byte permutation.  The conversion itself is the hardware's e4m3x2 -> f16x2 (measured 86 values per clock and SM with its
// surroundings, where 25 arrive from memory; shifts and masks gave 43).  P^T comes from the scores by movmatrix.  TMA's swizzle, and an
// order of keys and dimensions over the lanes that sets neighbouring groups four rows or chunks apart, keep the reads free of bank
// conflicts (heads of 64: the values' reads meet twice).
//
// Split: the work is one line of (sequence, head, row tile, key tile) units, cut evenly over the CTAs whatever the lengths are.  A CTA
// whose range ends inside an item leaves fp32 partials in the workspace; the CTA that arrives last at the item adds them in
// order, so results do not depend on the order of arrival.  No host knowledge of lengths: a captured graph serves every step.
#include "common.cuh"
#include "tc05.cuh"
#include "flashrt_b200.h"

#include <cuda_fp16.h>

#include <type_traits>

namespace frt {

constexpr int PA_MAX_GRID = 1024;                     // counters at the head of the workspace

struct PagedAttnParams {
    const __nv_bfloat16* q;
    __nv_bfloat16* o;
    float* lse;
    long long q_stride, o_stride;
    const uint8_t *k, *v;
    const float *k_scale, *v_scale;
    const int *table, *cu, *lens;
    int table_stride, tokens, batch, num_blocks, block_size, block_shift, hq, hkv, group;
    float scale, cap;
    int window, causal;
    int pool_rows;               // rows of a cache seen as a matrix of head_dim columns
    int* status;
    unsigned* counters;
    float2* part_ml;             // [cta][2][rows] (m, l)
    float* part_o;               // [cta][2][rows][D]
};

template <int D, int NT>
struct PagedCfg {
    static constexpr int ROWS = 8 * NT;
    static constexpr int KT = 4096 / D;               // keys of a warp's tile: 4 KB of keys, 4 KB of values
    static constexpr int ST = KT / 16;                // 16-key steps
    static constexpr int NW = 8;
    static constexpr int THREADS = 32 * NW;
    static constexpr int SLOT_BYTES = 2 * KT * D;
    static constexpr int SLOTS = NT == 1 && D <= 128 ? 3 : 2;
    static constexpr int RING_BYTES = NW * SLOTS * SLOT_BYTES;
    static constexpr int WRITERS = NT == 1 && D != 128 ? NW : NW / 2;      // warps whose accumulators are in shared memory at once
    static constexpr int PITCH = D + 4;               // floats of an accumulator row in shared memory
    static constexpr int Q_BYTES = NT * (D / 16) * 32 * 8;
    static constexpr int ACC_BYTES = WRITERS * ROWS * PITCH * 4;
    static constexpr int SMEM_BYTES = 1024 + RING_BYTES + Q_BYTES + ACC_BYTES;
    static constexpr bool Q_REGS = NT == 1;           // query fragments stay in registers
    static_assert(SMEM_BYTES <= 232448 - 6 * 1024, "dynamic and static shared memory of a CTA");
};

// One sequence's share of the work line.
struct PagedSeq { int start, n, len, row_tiles, t0, tiles; };

template <int KT, int ROWS>
__device__ __forceinline__ PagedSeq paged_seq(const PagedAttnParams& p, int b) {
    PagedSeq s;
    s.start = p.cu ? min(max(p.cu[b], 0), p.tokens) : b;
    const int end = p.cu ? min(max(p.cu[b + 1], s.start), p.tokens) : b + 1;
    s.n = end - s.start;
    s.len = min(max(p.lens[b], 0), (int)min((long long)p.table_stride << p.block_shift, 0x7fffff00LL));
    s.row_tiles = (int)(((long long)s.n * p.group + ROWS - 1) / ROWS);
    const int lo = p.window > 0 ? max(0, s.len - s.n - p.window + 1) : 0;
    s.t0 = lo / KT;
    s.tiles = max(1, (s.len + KT - 1) / KT - s.t0);             // an item without keys still writes its rows
    return s;
}
template <int KT, int ROWS>
__device__ __forceinline__ long long paged_units(const PagedAttnParams& p, int b) {
    const PagedSeq s = paged_seq<KT, ROWS>(p, b);
    return (long long)s.row_tiles * s.tiles * p.hkv;
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// four codes -> (c0, c1) and (c2, c3)
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ void mma_f16_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t a) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
    return r;
}
__device__ __forceinline__ uint2 ld_shared_v2(uint32_t a) {
    uint2 r;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a) : "memory");
    return r;
}
__device__ __forceinline__ float ld_shared_f(uint32_t a) {
    float r;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r) : "r"(a) : "memory");
    return r;
}
// 4 bytes to shared memory (zero if !there); the thread's arrival at `bar` follows its copies
__device__ __forceinline__ void copy_scale(uint32_t dst, const float* src, bool there, uint32_t bar) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
    asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(bar) : "memory");
}

// tanh through the hardware's exp2 and reciprocal: 2^-22 absolute, where tanh.approx has 2^-11
__device__ __forceinline__ float soft_cap(float s, float cap, float inv_cap2) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + ex2(s * inv_cap2)));
    return cap * (1.0f - 2.0f * r);
}

// A stretch of the work line inside one item: what a warp has to know to copy its tiles, and where the item's rows are.
struct PagedSegment {
    int b, item;                 // sequence; (head, row tile) inside it
    long long first, end;        // line positions: of the item, behind the stretch
    int items, h, row0, rows, tiles;
    int len, n, start;
    int key_lo, key_hi;          // keys that any row sees
    int tile_lo, tile_hi;        // tiles of the stretch with such keys
};
// the stretch that begins at line position `at` < w1; b, item, first are set
template <int KT, int ROWS>
__device__ __forceinline__ void paged_segment(const PagedAttnParams& p, PagedSegment& g, long long at, long long w1) {
    PagedSeq s = paged_seq<KT, ROWS>(p, g.b);
    while (g.item >= s.row_tiles * p.hkv && g.b + 1 < p.batch) {             // through with the sequence, or one without new tokens
        ++g.b;
        g.item = 0;
        s = paged_seq<KT, ROWS>(p, g.b);
    }
    g.items = s.row_tiles * p.hkv;
    g.h = g.item / s.row_tiles;
    g.row0 = (g.item - g.h * s.row_tiles) * ROWS;
    g.rows = min(ROWS, s.n * p.group - g.row0);
    g.tiles = s.tiles;
    g.len = s.len;
    g.n = s.n;
    g.start = s.start;
    g.end = min(g.first + s.tiles, w1);
    const int p0 = s.len - s.n + g.row0 / p.group, p1 = s.len - s.n + (g.row0 + g.rows - 1) / p.group;
    g.key_lo = p.window > 0 ? max(0, p0 - p.window + 1) : 0;
    g.key_hi = p.causal ? min(s.len, p1 + 1) : s.len;
    g.tile_lo = max(s.t0 + (int)(at - g.first), g.key_lo / KT);
    g.tile_hi = min(s.t0 + (int)(g.end - g.first), g.key_hi > 0 ? (g.key_hi + KT - 1) / KT : 0);
}

template <int D, int NT>
__global__ void __launch_bounds__(256, 1)
paged_attention_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, PagedAttnParams p) {
    using Cfg = PagedCfg<D, NT>;
    constexpr int ST = Cfg::ST, KT = Cfg::KT, NW = Cfg::NW, ROWS = Cfg::ROWS, SEGS = D / 64, MT = D / 16, SLOTS = Cfg::SLOTS;
    constexpr float LOG2E = 1.4426950408889634f;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint2* q_s = reinterpret_cast<uint2*>(smem + Cfg::RING_BYTES);           // [nt][k step][lane]
    float* acc_s = reinterpret_cast<float*>(smem + Cfg::RING_BYTES + Cfg::Q_BYTES);       // [warp][row][PITCH]
    __shared__ float2 ml_s[NW][ROWS];
    __shared__ float rf_s[ROWS];
    __shared__ float scale_s[NW][SLOTS][ST][2];
    __shared__ uint64_t full_s[NW][SLOTS];
    __shared__ long long scan_s[256];
    __shared__ long long warp_s[8];
    __shared__ unsigned last_s;
    __shared__ volatile int abort_s;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    if (lane < SLOTS) tc::mbar_init(&full_s[warp][lane], 1 + 2 * ST);        // the copies' bytes, one arrival per scale
    if (tid == 0) {
        tc::tma_prefetch_desc(&tmK);
        tc::tma_prefetch_desc(&tmV);
    }
    tc::mbar_fence_init();
    const uint64_t deadline = tc::global_timer_ns() + FRT_KERNEL_DEADLINE_NS;
    if (tid == 0) abort_s = 0;
    pdl_launch_dependents();
    pdl_wait();

    // ---------------- the work line: thread t counts the units of sequences [t * per, (t + 1) * per)
    const int per = (p.batch + 255) / 256;
    long long mine = 0;
    for (int b = tid * per; b < min((tid + 1) * per, p.batch); ++b) mine += paged_units<KT, ROWS>(p, b);
    long long incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += o;
    }
    if (lane == 31) warp_s[warp] = incl;
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        if (w < warp) before += warp_s[w];
        total += warp_s[w];
    }
    scan_s[tid] = before + incl - mine;                                      // exclusive
    __syncthreads();
    // few units: as many CTAs as give every warp one
    const int grid = (int)max(1LL, min((long long)gridDim.x, (total + NW - 1) / NW));
    const int cta = blockIdx.x;
    if (cta >= grid || total == 0) return;
    const long long w0 = total * cta / grid, w1 = total * (cta + 1) / grid;
    PagedSegment cur;
    {
        int lo = 0, hi = 256;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (scan_s[mid] <= w0) lo = mid; else hi = mid;
        }
        cur.b = lo * per;
        cur.first = scan_s[lo];
        for (;;) {                                                           // ends before the chunk does: w0 lies in it
            const long long u = paged_units<KT, ROWS>(p, cur.b);
            if (w0 < cur.first + u || cur.b + 1 >= p.batch) break;
            cur.first += u;
            ++cur.b;
        }
        cur.item = (int)((w0 - cur.first) / paged_seq<KT, ROWS>(p, cur.b).tiles);
        cur.first += (long long)cur.item * paged_seq<KT, ROWS>(p, cur.b).tiles;
    }
    paged_segment<KT, ROWS>(p, cur, w0, w1);

    // ---------------- this warp's copies: `nx` runs ahead of the computation by the slots of the ring
    const uint32_t ring = tc::smem_u32(smem) + (uint32_t)warp * (SLOTS * Cfg::SLOT_BYTES);
    const uint32_t full_a = tc::smem_u32(&full_s[warp][0]), scale_a = tc::smem_u32(&scale_s[warp][0][0][0]);
    PagedSegment nx = cur;
    int nx_tile = cur.tile_lo + warp, nx_page = -1, nx_slot = 0;
    // to the next tile there is for this warp; lanes 2 st, 2 st + 1 ask for the page of its st-th 16 keys
    auto seek = [&] {
        while (nx_tile >= nx.tile_hi) {
            if (nx.end >= w1) { nx_tile = 0x7fffffff; return; }
            const long long at = nx.end;
            nx.first = at;                                                   // a stretch that does not end the work ends its item
            ++nx.item;
            paged_segment<KT, ROWS>(p, nx, at, w1);
            nx_tile = nx.tile_lo + warp;
        }
        const int k0 = nx_tile * KT + (lane >> 1) * 16, box = min(KT, p.block_size), head = k0 & ~(box - 1);
        nx_page = -1;                                                        // a box without keys of the item is not looked at
        if (lane < 2 * ST && head < nx.key_hi && head + box > nx.key_lo)
            nx_page = p.table[(size_t)nx.b * p.table_stride + (head >> p.block_shift)];
        if (nx_page >= p.num_blocks) nx_page = -1;
    };
    auto copy = [&] {
        if (nx_tile == 0x7fffffff) return;
        const uint32_t bar = full_a + 8 * nx_slot, dst = ring + nx_slot * Cfg::SLOT_BYTES;
        if (lane < 2 * ST) {
            const float* src = lane & 1 ? p.v_scale : p.k_scale;
            copy_scale(scale_a + (nx_slot * ST * 2 + lane) * 4, src + (size_t)max(nx_page, 0) * p.hkv + nx.h, nx_page >= 0, bar);
        }
        if (lane == 0) tc::mbar_arrive_expect_tx(bar, Cfg::SLOT_BYTES);
        // one box per block (or per tile inside one): lane 2 st of its first 16 keys issues it; rows beyond the pool arrive as zeros
        const int box = min(KT, p.block_size), st = lane >> 1;
        if (lane < 2 * ST && (st * 16) % box == 0) {
            const int k0 = nx_tile * KT + st * 16;
            const int row = nx_page >= 0 ? (nx_page * p.hkv + nx.h) * p.block_size + (k0 & (p.block_size - 1)) : p.pool_rows;
            const CUtensorMap* map = lane & 1 ? &tmV : &tmK;
            constexpr int INNER = D < 128 ? D : 128;
            const uint32_t to = dst + (lane & 1) * (KT * D) + st * 16 * INNER;
#pragma unroll
            for (int x = 0; x < D; x += INNER) tc::tma_load_2d(to + x * KT, map, bar, x, row);
        }
        if (++nx_slot == SLOTS) nx_slot = 0;
        nx_tile += NW;
    };
    for (int i = 0; i < SLOTS; ++i) {
        seek();
        copy();
    }
    seek();
    int slot = 0;
    uint32_t phase = 0;

    // where this lane's operands are in a slot (see the top: groups of lanes four rows or chunks apart)
    const int krow = D == 64 ? g : (g >> 1) | ((g & 1) << 2), dchunk = krow;
    const uint32_t k_off = D == 64 ? g * 64 + ((c ^ ((g >> 1) & 3)) << 4) : krow * 128 + ((c ^ krow) << 4);
    const uint32_t v_off = KT * D + (D == 64 ? 2 * c * 64 + (((g >> 1) ^ c) << 4) + (g & 1) * 8 : c * 128 + ((dchunk ^ c) << 4));
    constexpr int STEP = D == 64 ? 64 : 128;                                 // bytes from row to row

    for (long long at = w0; at < w1;) {
        if (at != w0) {
            cur.first = at;
            ++cur.item;
            paged_segment<KT, ROWS>(p, cur, at, w1);
        }
        const int rows = cur.rows, row0 = cur.row0, h = cur.h;

        // queries -> fp16 operand fragments, at most 1 in magnitude: one warp per row
        __syncthreads();                                                     // the item before is through with shared memory
        for (int r = warp; r < ROWS; r += NW) {
            constexpr int PL = D / 32;                                       // dimensions of a lane
            float x[PL];
            float top = 0.0f;
            if (r < rows) {
                const int i = (row0 + r) / p.group, hh = h * p.group + (row0 + r) % p.group;
                const uint32_t* src = reinterpret_cast<const uint32_t*>(p.q + (size_t)(cur.start + i) * p.q_stride + (size_t)hh * D + lane * PL);
#pragma unroll
                for (int j = 0; j < PL / 2; ++j) unpack_bf16x2(src[j], x[2 * j], x[2 * j + 1]);
            } else {
#pragma unroll
                for (int j = 0; j < PL; ++j) x[j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < PL; ++j) top = fmaxf(top, fabsf(x[j]));
            top = warp_max_butterfly(top);
            // 2^-e with 2^e > top (zero, tiny: no scaling; infinite: neither, the row is NaN or infinite as it should be)
            const int e = top > 1e-30f && top < INFINITY ? min((int)((__float_as_uint(top) >> 23) & 255) - 126, 126) : 0;
            const float down = __uint_as_float((uint32_t)(127 - e) << 23);
            if (lane == 0) rf_s[r] = __uint_as_float((uint32_t)(127 + e) << 23);
            __half* dst = reinterpret_cast<__half*>(q_s + (r >> 3) * MT * 32);
#pragma unroll
            for (int j = 0; j < PL; ++j) {
                // dimension -> (segment of 64, lane column, k step of the segment, place in the fragment)
                const int d = lane * PL + j, step = (d >> 6) * 4 + ((d >> 2) & 3), cc = (d >> 4) & 3, place = d & 3;
                dst[((step * 32 + (r & 7) * 4 + cc) << 2) + place] = __float2half_rn(x[j] * down);
            }
        }
        __syncthreads();

        // this lane's rows: 2c, 2c + 1 of every n tile
        float rf[NT][2];
        int row_hi[NT][2], row_lo[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int r = nt * 8 + 2 * c + x;
                rf[nt][x] = rf_s[r] * p.scale * (p.cap > 0.0f ? 1.0f : LOG2E);
                const int pos = cur.len - cur.n + (row0 + min(r, rows - 1)) / p.group;
                row_hi[nt][x] = p.causal ? min(pos + 1, cur.len) : cur.len;
                row_lo[nt][x] = p.window > 0 ? max(0, pos - p.window + 1) : 0;
            }
        const int p0 = cur.len - cur.n + row0 / p.group, p1 = cur.len - cur.n + (row0 + rows - 1) / p.group;
        const int all_hi = p.causal ? min(p0 + 1, cur.len) : cur.len;        // keys that every row sees
        const int all_lo = p.window > 0 ? max(0, p1 - p.window + 1) : 0;
        uint2 q_r[Cfg::Q_REGS ? MT : 1];
        if constexpr (Cfg::Q_REGS) {
#pragma unroll
            for (int j = 0; j < MT; ++j) q_r[j] = q_s[j * 32 + lane];
        }

        float m[NT][2], l[NT][2], acc[NT][MT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
            for (int j = 0; j < MT; ++j)
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[nt][j][x] = 0.0f;
        }

        for (int tile = cur.tile_lo + warp; tile < cur.tile_hi; tile += NW) {
            const uint32_t base = ring + slot * Cfg::SLOT_BYTES;
            if (!tc::mbar_wait_until(full_a + 8 * slot, phase, deadline, &abort_s)) {
                if (!abort_s && lane == 0) atomicCAS(p.status, 0, 1 | (blockIdx.x << 8));
                abort_s = 1;
            }
            __syncwarp();
            // ---- scores: [key][row]
            float sc[ST][NT][4];
#pragma unroll
            for (int st = 0; st < ST; ++st)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 4; ++x) sc[st][nt][x] = 0.0f;
#pragma unroll
            for (int sg = 0; sg < SEGS; ++sg) {
                uint32_t kw[ST][2][4];
                const uint32_t kb = base + (sg >> 1) * (KT * 128) + (sg & 1 ? k_off ^ 64 : k_off);
#pragma unroll
                for (int st = 0; st < ST; ++st)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint4 w = ld_shared_v4(kb + (st * 16 + x * 8) * STEP);
                        kw[st][x][0] = w.x; kw[st][x][1] = w.y; kw[st][x][2] = w.z; kw[st][x][3] = w.w;
                    }
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    uint2 qf[NT];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) qf[nt] = Cfg::Q_REGS ? q_r[sg * 4 + y] : q_s[(nt * MT + sg * 4 + y) * 32 + lane];
#pragma unroll
                    for (int st = 0; st < ST; ++st) {
                        uint32_t a[4];
                        e4m3x4_to_f16(kw[st][0][y], a[0], a[2]);
                        e4m3x4_to_f16(kw[st][1][y], a[1], a[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_f16_16816(sc[st][nt], a, qf[nt].x, qf[nt].y);
                    }
                }
            }
            // ---- base-2 logits with the values' scale, mask, running maximum
            const int key0 = tile * KT;
            bool open = key0 >= all_lo && key0 + KT <= all_hi;
            float ks[ST], lv[ST], inv_vs[ST], top[NT][2];
#pragma unroll
            for (int st = 0; st < ST; ++st) {
                ks[st] = ld_shared_f(scale_a + ((slot * ST + st) * 2) * 4);
                const float vs = ld_shared_f(scale_a + ((slot * ST + st) * 2 + 1) * 4);
                open = open && vs != 0.0f;                                   // zero: an absent page
                lv[st] = __log2f(fmaxf(vs, 1e-30f));
                inv_vs[st] = vs != 0.0f ? __frcp_rn(fmaxf(vs, 1e-30f)) : 0.0f;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) top[nt][0] = top[nt][1] = -INFINITY;
#pragma unroll
            for (int st = 0; st < ST; ++st)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float f = rf[nt][x & 1] * ks[st];
                        float u;
                        if (p.cap > 0.0f) u = fmaf(soft_cap(sc[st][nt][x] * f, p.cap, 2.0f * LOG2E / p.cap), LOG2E, lv[st]);
                        else u = fmaf(sc[st][nt][x], f, lv[st]);
                        sc[st][nt][x] = u;
                    }
            if (!open) {
#pragma unroll
                for (int st = 0; st < ST; ++st)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const int key = key0 + st * 16 + krow + 8 * (x >> 1);
                            if (inv_vs[st] == 0.0f || key >= row_hi[nt][x & 1] || key < row_lo[nt][x & 1]) sc[st][nt][x] = -INFINITY;
                        }
            }
#pragma unroll
            for (int st = 0; st < ST; ++st)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 4; ++x) top[nt][x & 1] = fmaxf(top[nt][x & 1], sc[st][nt][x]);
            bool grown = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float t = top[nt][x];
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
                    top[nt][x] = fmaxf(m[nt][x], t);
                    grown = grown || top[nt][x] > m[nt][x];
                }
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float down = ex2(m[nt][x] - (top[nt][x] == -INFINITY ? 0.0f : top[nt][x]));
                        m[nt][x] = top[nt][x];
                        l[nt][x] *= down;
#pragma unroll
                        for (int j = 0; j < MT; ++j) {
                            acc[nt][j][x] *= down;
                            acc[nt][j][2 + x] *= down;
                        }
                    }
            }
            // ---- weights -> P^T fragments
            uint32_t pf[ST][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float ref[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) ref[x] = 15.0f - (m[nt][x] == -INFINITY ? 0.0f : m[nt][x]);
#pragma unroll
                for (int st = 0; st < ST; ++st) {
                    float w[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        w[x] = ex2(sc[st][nt][x] + ref[x & 1]);
                        l[nt][x & 1] = fmaf(w[x], inv_vs[st], l[nt][x & 1]);
                    }
                    pf[st][nt][0] = transpose_8x8(pack_f16x2(w[0], w[1]));
                    pf[st][nt][1] = transpose_8x8(pack_f16x2(w[2], w[3]));
                }
            }
            // ---- values: [dimension][row]
#pragma unroll
            for (int st = 0; st < ST; ++st) {
#pragma unroll
                for (int half = 0; half < (D == 256 ? 2 : 1); ++half) {
                    constexpr int W = D == 64 ? 2 : 4;                       // words of a lane and key
                    uint32_t vw[4][W];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {                            // k indices 2c, 2c + 1, 2c + 8, 2c + 9
                        if constexpr (D == 64) {
                            const uint2 w = ld_shared_v2(base + v_off + (st * 16 + (x & 1) + 8 * (x >> 1)) * 64);
                            vw[x][0] = w.x; vw[x][1] = w.y;
                        } else {
                            const uint4 w = ld_shared_v4(base + (x & 1 ? (v_off ^ 64) + 512 : v_off) + (st * 16 + 8 * (x >> 1)) * 128 +
                                                         half * (KT * 128));
                            vw[x][0] = w.x; vw[x][1] = w.y; vw[x][2] = w.z; vw[x][3] = w.w;
                        }
                        if (!open) {
                            // what lies outside the item's keys may be anything, and 0 x NaN is NaN
                            const int key = key0 + st * 16 + (D == 64 ? 2 * c + (x & 1) : c + 4 * (x & 1)) + 8 * (x >> 1);
                            if (key >= cur.key_hi || key < cur.key_lo) {
#pragma unroll
                                for (int y = 0; y < W; ++y) vw[x][y] = 0;
                            }
                        }
                    }
#pragma unroll
                    for (int y = 0; y < W; ++y) {
                        const int j = 2 * (half * 4 + y);
                        uint32_t a[4], e[4];
                        e4m3x4_to_f16(__byte_perm(vw[0][y], vw[1][y], 0x5140), a[0], a[1]);
                        e4m3x4_to_f16(__byte_perm(vw[2][y], vw[3][y], 0x5140), a[2], a[3]);
                        e4m3x4_to_f16(__byte_perm(vw[0][y], vw[1][y], 0x7362), e[0], e[1]);
                        e4m3x4_to_f16(__byte_perm(vw[2][y], vw[3][y], 0x7362), e[2], e[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma_f16_16816(acc[nt][j], a, pf[st][nt][0], pf[st][nt][1]);
                            mma_f16_16816(acc[nt][j + 1], e, pf[st][nt][0], pf[st][nt][1]);
                        }
                    }
                }
            }
            __syncwarp();                                                    // the slot is read: the next tile may land there
            copy();
            seek();
            if (++slot == SLOTS) { slot = 0; phase ^= 1; }
        }

        // ---------------- the warps' results
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float t = l[nt][x];
                t += __shfl_xor_sync(0xffffffffu, t, 4);
                t += __shfl_xor_sync(0xffffffffu, t, 8);
                t += __shfl_xor_sync(0xffffffffu, t, 16);
                if (g == 0) ml_s[warp][nt * 8 + 2 * c + x] = make_float2(m[nt][x], t);
            }
        // this lane's row and dimensions 4 i .. 4 i + 3 of its piece in an accumulator
        auto place = [&](int w, int nt, int x, int i) {
            const int d = D == 64 ? g * 8 + 4 * i : (i >> 2) * 128 + dchunk * 16 + 4 * (i & 3);
            return reinterpret_cast<float4*>(acc_s + ((size_t)w * ROWS + nt * 8 + 2 * c + x) * Cfg::PITCH + d);
        };
        auto put = [&](int w) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int i = 0; i < MT / 2; ++i)
                        *place(w, nt, x, i) = make_float4(acc[nt][2 * i][x], acc[nt][2 * i][2 + x], acc[nt][2 * i + 1][x], acc[nt][2 * i + 1][2 + x]);
        };
        if constexpr (Cfg::WRITERS == NW) {
            put(warp);
            __syncthreads();
        } else {
            // the upper half's accumulators first, each into the registers of a warp of the lower half
            if (warp >= NW / 2) put(warp - NW / 2);
            __syncthreads();
            if (warp < NW / 2) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int r = nt * 8 + 2 * c + x;
                        const float2 a = ml_s[warp][r], b = ml_s[warp + NW / 2][r];
                        const float mm = fmaxf(a.x, b.x), safe = mm == -INFINITY ? 0.0f : mm, fa = ex2(a.x - safe), fb = ex2(b.x - safe);
#pragma unroll
                        for (int i = 0; i < MT / 2; ++i) {
                            const float4 o = *place(warp, nt, x, i);
                            acc[nt][2 * i][x] = acc[nt][2 * i][x] * fa + o.x * fb;
                            acc[nt][2 * i][2 + x] = acc[nt][2 * i][2 + x] * fa + o.y * fb;
                            acc[nt][2 * i + 1][x] = acc[nt][2 * i + 1][x] * fa + o.z * fb;
                            acc[nt][2 * i + 1][2 + x] = acc[nt][2 * i + 1][2 + x] * fa + o.w * fb;
                        }
                        __syncwarp();
                        if (g == 0) ml_s[warp][r] = make_float2(mm, a.y * fa + b.y * fb);
                    }
                put(warp);
            }
            __syncthreads();
        }
        const bool split = !(at == cur.first && cur.end == cur.first + cur.tiles);
        const int slot = at == w0 ? 0 : 1;
        const size_t part = (size_t)cta * 2 + slot;
        auto finish = [&](int r, int d4, float4 sum, float mm, float ll) {
            const int i = (row0 + r) / p.group, hh = h * p.group + (row0 + r) % p.group;
            const float inv = ll > 0.0f ? __frcp_rn(ll) : (ll == 0.0f ? 0.0f : ll);       // no key: zero; NaN stays
            uint2 out;
            out.x = pack_bf16x2(sum.x * inv, sum.y * inv);
            out.y = pack_bf16x2(sum.z * inv, sum.w * inv);
            const int token = cur.start + i;
            st_global_v2(p.o + (size_t)token * p.o_stride + (size_t)hh * D + d4 * 4, out);
            if (d4 == 0 && p.lse)
                p.lse[(size_t)hh * p.tokens + token] = ll == 0.0f ? -INFINITY : 0.6931471805599453f * (mm - 15.0f + log2f(ll));
        };
        for (int x = tid; x < rows * (D / 4); x += Cfg::THREADS) {
            const int r = x / (D / 4), d4 = x % (D / 4);
            float mm = -INFINITY, ll = 0.0f;
#pragma unroll
            for (int w = 0; w < Cfg::WRITERS; ++w) mm = fmaxf(mm, ml_s[w][r].x);
            const float safe = mm == -INFINITY ? 0.0f : mm;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < Cfg::WRITERS; ++w) {
                const float f = ex2(ml_s[w][r].x - safe);
                const float4 v = *reinterpret_cast<const float4*>(acc_s + ((size_t)w * ROWS + r) * Cfg::PITCH + d4 * 4);
                ll = fmaf(ml_s[w][r].y, f, ll);
                sum.x = fmaf(v.x, f, sum.x); sum.y = fmaf(v.y, f, sum.y);
                sum.z = fmaf(v.z, f, sum.z); sum.w = fmaf(v.w, f, sum.w);
            }
            if (!split) {
                finish(r, d4, sum, mm, ll);
            } else {
                __stcg(reinterpret_cast<float4*>(p.part_o + (part * ROWS + r) * D + d4 * 4), sum);
                if (d4 == 0) __stcg(p.part_ml + part * ROWS + r, make_float2(mm, ll));
            }
        }
        if (split) {
            // CTAs of the item: from the one with its first unit to the one with its last
            const long long first = cur.first, last_unit = first + cur.tiles - 1;
            auto owner = [&](long long u) { return (int)(((u + 1) * grid - 1) / total); };
            const int c0 = owner(first), c1 = owner(last_unit);
            __threadfence();
            __syncthreads();
            if (tid == 0) last_s = atomicInc(p.counters + c0, (unsigned)(c1 - c0)) == (unsigned)(c1 - c0);
            __syncthreads();
            if (last_s) {
                __threadfence();
                const int slot0 = total * c0 / grid < first;                 // the first CTA had another item in front
                for (int x = tid; x < rows * (D / 4); x += Cfg::THREADS) {
                    const int r = x / (D / 4), d4 = x % (D / 4);
                    auto piece = [&](int q) { return (size_t)q * 2 + (q == c0 ? slot0 : 0); };
                    float mm = -INFINITY, ll = 0.0f;
                    for (int q = c0; q <= c1; ++q) mm = fmaxf(mm, __ldcg(p.part_ml + piece(q) * ROWS + r).x);
                    const float safe = mm == -INFINITY ? 0.0f : mm;
                    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                    for (int q = c0; q <= c1; ++q) {
                        const size_t at_q = piece(q) * ROWS + r;
                        const float2 ml = __ldcg(p.part_ml + at_q);
                        const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part_o + at_q * D + d4 * 4));
                        const float f = ex2(ml.x - safe);
                        ll = fmaf(ml.y, f, ll);
                        sum.x = fmaf(v.x, f, sum.x); sum.y = fmaf(v.y, f, sum.y);
                        sum.z = fmaf(v.z, f, sum.z); sum.w = fmaf(v.w, f, sum.w);
                    }
                    finish(r, d4, sum, mm, ll);
                }
            }
        }
        at = cur.end;
    }
    if (abort_s) {                       // a wait gave up: copies may be in flight, a bounded time for them to land
        const uint64_t until = tc::global_timer_ns() + 1000000ull;
        while (tc::global_timer_ns() < until) {}
    }
}

template <int D, int NT>
static int paged_grid() { return min(device_sm_count(), PA_MAX_GRID); }
template <int D, int NT>
static long long paged_workspace() {
    return 4 * PA_MAX_GRID + (long long)paged_grid<D, NT>() * 2 * PagedCfg<D, NT>::ROWS * (D + 2) * 4;
}

// A cache as a matrix of head_dim bytes a row; boxes of `box` rows x 128 bytes (64 for heads of 64), swizzled over that width.  Rows
// behind the last one read as zeros.
static int paged_map(CUtensorMap* out, const void* base, int rows, int d, int box) {
    typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                               CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
        return e == cudaSuccess && q == cudaDriverEntryPointSuccess ? reinterpret_cast<Encode>(fn) : nullptr;
    }();
    if (!encode) return FRT_ERR_UNSUPPORTED;
    const cuuint64_t dims[2] = {(cuuint64_t)d, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)d};
    const cuuint32_t boxes[2] = {(cuuint32_t)(d < 128 ? d : 128), (cuuint32_t)box}, ones[2] = {1, 1};
    const CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, boxes, ones,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, d < 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? FRT_OK : FRT_ERR_INVALID;
}

template <int D, int NT>
static int launch_paged_attention(PagedAttnParams p, void* work, long long work_bytes, cudaStream_t stream) {
    using Cfg = PagedCfg<D, NT>;
    static PerDeviceOnce attr_once;
    int attr_dev = 0;
    if (attr_once.need(attr_dev)) {
        const cudaError_t e = cudaFuncSetAttribute(paged_attention_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   Cfg::SMEM_BYTES);
        if (e != cudaSuccess) return FRT_CUDA_ERR(e);
        attr_once.set(attr_dev);
    }
    const int grid = paged_grid<D, NT>();
    if (work_bytes < paged_workspace<D, NT>()) return FRT_ERR_INVALID;
    p.counters = static_cast<unsigned*>(work);
    p.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(work) + 4 * PA_MAX_GRID);
    p.part_o = reinterpret_cast<float*>(p.part_ml + (size_t)grid * 2 * Cfg::ROWS);
    CUtensorMap tmK, tmV;
    const int box = Cfg::KT < p.block_size ? Cfg::KT : p.block_size;
    int rc = paged_map(&tmK, p.k, p.pool_rows, D, box);
    if (!rc) rc = paged_map(&tmV, p.v, p.pool_rows, D, box);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(Cfg::THREADS);
    cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_attention_kernel<D, NT>, tmK, tmV, p);
    return e == cudaSuccess ? FRT_OK : FRT_CUDA_ERR(e);
}

}  // namespace frt

// Row tiles of 8 NT rows, so that the keys are read and converted as few times as the registers of the accumulators allow (heads of
// 256: 16 rows, else 32), and no wider than the rows need.
static int paged_nt(long long max_new, int group, int d) {
    const int most = d == 256 ? 2 : 4;
    const long long rows = max_new * group, tiles = (rows + 8 * most - 1) / (8 * most);
    return tiles < 1 ? 1 : tiles > 4 ? most : (int)((rows + 8 * tiles - 1) / (8 * tiles));
}
// f(kernel's head dim, row tile) for one of the instances
template <typename F>
static auto paged_dispatch(int d, int nt, F f) {
    using std::integral_constant;
    auto with = [&](auto D) {
        if constexpr (D() != 256) {
            if (nt == 4) return f(D, integral_constant<int, 4>());
            if (nt == 3) return f(D, integral_constant<int, 3>());
        }
        if (nt == 2) return f(D, integral_constant<int, 2>());
        return f(D, integral_constant<int, 1>());
    };
    if (d == 64) return with(integral_constant<int, 64>());
    if (d == 128) return with(integral_constant<int, 128>());
    return with(integral_constant<int, 256>());
}

extern "C" int frt_b200_paged_attention_workspace_bytes(int tokens, int batch, int max_new, int num_heads_q, int num_heads_kv,
                                                        int head_dim, long long* out_bytes) {
    using namespace frt;
    if (!out_bytes || tokens < 0 || batch < 0 || max_new < 0 || num_heads_q < 1 || num_heads_kv < 1) return FRT_ERR_INVALID;
    if (num_heads_q % num_heads_kv) return FRT_ERR_UNSUPPORTED;
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return FRT_ERR_UNSUPPORTED;
    *out_bytes = paged_dispatch(head_dim, paged_nt(max_new, num_heads_q / num_heads_kv, head_dim),
                                [](auto D, auto NT) { return paged_workspace<D(), NT()>(); });
    return FRT_OK;
}

extern "C" int frt_b200_paged_attention_fp8(const void* Q, long long q_stride, void* O, long long o_stride, float* lse,
                                            const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                                            const int* block_table, int table_stride, const int* cu_seqlens, const int* seq_lens,
                                            int tokens, int batch, int max_new, int num_blocks, int block_size, int num_heads_q,
                                            int num_heads_kv, int head_dim, float softmax_scale, float softcap, int window,
                                            void* workspace, long long workspace_bytes, int flags, void* stream) {
    using namespace frt;
    auto off = [](const void* a, uintptr_t n) { return (reinterpret_cast<uintptr_t>(a) & (n - 1)) != 0; };
    if (tokens < 0 || batch < 0 || max_new < 0 || num_blocks < 0 || table_stride < 0 || num_heads_q < 1 || num_heads_kv < 1 ||
        window < 0 || !(softcap >= 0.0f) || softcap > 1e30f || !(softmax_scale > -1e30f && softmax_scale < 1e30f))
        return FRT_ERR_INVALID;
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return FRT_ERR_UNSUPPORTED;
    if (block_size < 16 || block_size > 128 || (block_size & (block_size - 1))) return FRT_ERR_UNSUPPORTED;
    if (num_heads_q > 1024 || num_heads_q % num_heads_kv) return FRT_ERR_UNSUPPORTED;
    const bool causal = !(flags & 2);
    if (window && !causal) return FRT_ERR_UNSUPPORTED;
    const long long width = (long long)num_heads_q * head_dim;
    if (q_stride < width || o_stride < width || q_stride % 8 || o_stride % 8) return FRT_ERR_INVALID;
    if (!cu_seqlens && tokens != batch) return FRT_ERR_INVALID;
    if (tokens == 0 || batch == 0) return FRT_OK;
    if (!Q || !O || !k_cache || !v_cache || !k_scale || !v_scale || !block_table || !seq_lens || !workspace) return FRT_ERR_INVALID;
    if (off(Q, 16) || off(O, 16) || off(lse, 4) || off(k_cache, 16) || off(v_cache, 16) || off(k_scale, 4) || off(v_scale, 4) ||
        off(block_table, 4) || off(cu_seqlens, 4) || off(seq_lens, 4) || off(workspace, 16))
        return FRT_ERR_INVALID;
    PagedAttnParams p = {};
    p.q = static_cast<const __nv_bfloat16*>(Q);
    p.o = static_cast<__nv_bfloat16*>(O);
    p.lse = lse;
    p.q_stride = q_stride;
    p.o_stride = o_stride;
    p.k = static_cast<const uint8_t*>(k_cache);
    p.v = static_cast<const uint8_t*>(v_cache);
    p.k_scale = k_scale;
    p.v_scale = v_scale;
    p.table = block_table;
    p.cu = cu_seqlens;
    p.lens = seq_lens;
    p.table_stride = table_stride;
    p.tokens = tokens;
    p.batch = batch;
    p.num_blocks = num_blocks;
    p.block_size = block_size;
    while ((1 << p.block_shift) < block_size) ++p.block_shift;
    p.hq = num_heads_q;
    p.hkv = num_heads_kv;
    p.group = num_heads_q / num_heads_kv;
    p.scale = softmax_scale;
    p.cap = softcap;
    p.window = window;
    p.causal = causal;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const long long pool_rows = (long long)num_blocks * num_heads_kv * block_size;
    if (pool_rows > 0x7fffffffLL) return FRT_ERR_UNSUPPORTED;
    p.pool_rows = (int)pool_rows;
    p.status = attention_status_device_ptr();
    if (!p.status) return FRT_ERR_UNSUPPORTED;
    return paged_dispatch(head_dim, paged_nt(max_new, p.group, head_dim),
                          [&](auto D, auto NT) { return launch_paged_attention<D(), NT()>(p, workspace, workspace_bytes, st); });
}

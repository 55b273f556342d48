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
// built to keep loads in flight: no shared memory and no barrier on the way of keys and values.  A warp takes KT keys at a time with
// 16-byte loads straight into registers, whose layout IS the operand of mma.sync m16n8k16: keys are the M rows of K . Q^T and
// dimensions the M rows of V^T . P^T, so a group of up to eight query rows fills the N side and no tensor work is wasted; which
// dimension a k index stands for is free, hence a lane's 16 contiguous bytes serve four k steps.  The pairs of keys that V^T wants
// side by side come from one byte permutation, which unpacking 8-bit codes costs anyway; the conversion itself is the hardware's
// e4m3x2 -> f16x2 (measured 86 values per clock and SM with its surroundings, where 25 arrive from memory; shifts and masks gave 43).
// P^T comes from the scores by movmatrix.  The next tile's keys are requested as soon as this one's are converted, its values likewise.
//
// Split: the work is one line of (sequence, head, row tile, key tile) units, cut evenly over the CTAs whatever the lengths are.  A CTA
// whose range ends inside an item leaves fp32 partials in the workspace; the CTA that arrives last at the item adds them in
// order, so results do not depend on the order of arrival.  No host knowledge of lengths: a captured graph serves every step.
#include "common.cuh"
#include "flashrt_b200.h"

#include <cuda_fp16.h>

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
    unsigned* counters;
    float2* part_ml;             // [cta][2][rows] (m, l)
    float* part_o;               // [cta][2][rows][D]
};

template <int D, int NT>
struct PagedCfg {
    static constexpr int ROWS = 8 * NT;
    static constexpr int ST = D == 256 ? 1 : 2;       // 16-key steps of a warp's tile
    static constexpr int KT = 16 * ST;
    static constexpr int NW = 8;
    static constexpr int THREADS = 32 * NW;
    static constexpr int CTAS = D == 256 || NT == 2 ? 1 : 2;      // per SM (registers)
    static constexpr int PITCH = D + 4;               // floats of an accumulator row in shared memory
    static constexpr int Q_BYTES = NT * (D / 16) * 32 * 8;
    static constexpr int ACC_BYTES = NW * ROWS * PITCH * 4;
    static constexpr int SMEM_BYTES = Q_BYTES + ACC_BYTES;
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
// cache bytes: coherent (the append in front may still run when this kernel starts), not kept in L1, in program order
template <int WORDS>
__device__ __forceinline__ void ld_codes(const uint8_t* p, uint32_t* w) {
    if constexpr (WORDS == 2)
        asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
    else
#pragma unroll
        for (int i = 0; i < WORDS; i += 4)
            asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]) : "l"(p + 4 * i));
}

// tanh through the hardware's exp2 and reciprocal: 2^-22 absolute, where tanh.approx has 2^-11
__device__ __forceinline__ float soft_cap(float s, float cap, float inv_cap2) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + ex2(s * inv_cap2)));
    return cap * (1.0f - 2.0f * r);
}

template <int D, int NT>
__global__ void __launch_bounds__(256, (PagedCfg<D, NT>::CTAS))
paged_attention_kernel(PagedAttnParams p) {
    using Cfg = PagedCfg<D, NT>;
    constexpr int ST = Cfg::ST, KT = Cfg::KT, NW = Cfg::NW, ROWS = Cfg::ROWS, SEGS = D / 64, VW = D / 32, MT = D / 16;
    constexpr float LOG2E = 1.4426950408889634f;
    extern __shared__ __align__(16) uint8_t smem[];
    uint2* q_s = reinterpret_cast<uint2*>(smem);                             // [nt][k step][lane]
    float* acc_s = reinterpret_cast<float*>(smem + Cfg::Q_BYTES);            // [warp][row][PITCH]
    __shared__ float2 ml_s[NW][ROWS];
    __shared__ float rf_s[ROWS];
    __shared__ long long scan_s[256];
    __shared__ long long warp_s[8];
    __shared__ unsigned last_s;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
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
    int b, item;                                                             // sequence; (head, row tile) inside it
    long long at = w0, first;                                                // first: line position of the item
    {
        int lo = 0, hi = 256;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (scan_s[mid] <= w0) lo = mid; else hi = mid;
        }
        b = lo * per;
        first = scan_s[lo];
        for (;;) {                                                           // ends before the chunk does: w0 lies in it
            const long long u = paged_units<KT, ROWS>(p, b);
            if (w0 < first + u || b + 1 >= p.batch) break;
            first += u;
            ++b;
        }
        const PagedSeq s = paged_seq<KT, ROWS>(p, b);
        item = (int)((w0 - first) / s.tiles);
        first += (long long)item * s.tiles;
    }

    while (at < w1) {
        const PagedSeq s = paged_seq<KT, ROWS>(p, b);
        const int items = s.row_tiles * p.hkv;
        if (item >= items) { ++b; item = 0; continue; }                      // a sequence without new tokens has no items
        const int h = item / s.row_tiles, row0 = (item - h * s.row_tiles) * ROWS;
        const long long end = min(first + s.tiles, w1);
        const int rows = min(ROWS, s.n * p.group - row0);

        // queries -> fp16 operand fragments, at most 1 in magnitude: one warp per row
        __syncthreads();                                                     // the item before is through with shared memory
        for (int r = warp; r < ROWS; r += NW) {
            constexpr int PL = D / 32;                                       // dimensions of a lane
            float x[PL];
            float top = 0.0f;
            if (r < rows) {
                const int i = (row0 + r) / p.group, hh = h * p.group + (row0 + r) % p.group;
                const uint32_t* src = reinterpret_cast<const uint32_t*>(p.q + (size_t)(s.start + i) * p.q_stride + (size_t)hh * D + lane * PL);
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
        int all_hi = 0x7fffffff, all_lo = 0;                                 // keys that every row sees
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int r = nt * 8 + 2 * c + x;
                rf[nt][x] = rf_s[r] * p.scale * (p.cap > 0.0f ? 1.0f : LOG2E);
                const int pos = s.len - s.n + (row0 + min(r, rows - 1)) / p.group;
                row_hi[nt][x] = p.causal ? min(pos + 1, s.len) : s.len;
                row_lo[nt][x] = p.window > 0 ? max(0, pos - p.window + 1) : 0;
            }
        {
            const int p0 = s.len - s.n + row0 / p.group, p1 = s.len - s.n + (row0 + rows - 1) / p.group;
            all_hi = p.causal ? min(p0 + 1, s.len) : s.len;
            all_lo = p.window > 0 ? max(0, p1 - p.window + 1) : 0;
        }
        const int key_lo = p.window > 0 ? max(0, s.len - s.n + row0 / p.group - p.window + 1) : 0;
        const int key_hi = p.causal ? min(s.len, s.len - s.n + (row0 + rows - 1) / p.group + 1) : s.len;   // any row's keys
        // tiles of this CTA's share, without those that no row sees
        const int tile_lo = max(s.t0 + (int)(at - first), key_lo / KT);
        const int tile_hi = min(s.t0 + (int)(end - first), key_hi > 0 ? (key_hi + KT - 1) / KT : 0);

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
        uint32_t kw[ST][2][SEGS][4], vw[ST][4][VW];
        // pages and scales of a tile; a page that holds no key of the item, or is no block of the pool, reads as absent
        int page_n[ST];
        float ks_n[ST], vs_n[ST];
        const int* table = p.table + (size_t)b * p.table_stride;
        auto load_meta = [&](int tile) {
#pragma unroll
            for (int st = 0; st < ST; ++st) {
                const int k0 = tile * KT + st * 16;
                int page = -1;
                if (tile < tile_hi && k0 < key_hi && k0 + 16 > key_lo) page = table[k0 >> p.block_shift];
                if (page >= p.num_blocks) page = -1;
                page_n[st] = page;
                ks_n[st] = vs_n[st] = 1.0f;
                if (page >= 0) {
                    ks_n[st] = p.k_scale[(size_t)page * p.hkv + h];
                    vs_n[st] = fmaxf(p.v_scale[(size_t)page * p.hkv + h], 1e-30f);
                }
            }
        };
        auto block_base = [&](int page, int k0) {
            return (((size_t)max(page, 0) * p.hkv + h) * p.block_size + (k0 & (p.block_size - 1))) * D;
        };
        auto load_k = [&](int tile) {
#pragma unroll
            for (int st = 0; st < ST; ++st) {
                const int k0 = tile * KT + st * 16;
                const uint8_t* base = p.k + block_base(page_n[st], k0) + c * 16;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int r = g + 8 * x;
                    if (page_n[st] >= 0 && k0 + r < key_hi) {
#pragma unroll
                        for (int sg = 0; sg < SEGS; ++sg) ld_codes<4>(base + r * D + sg * 64, kw[st][x][sg]);
                    } else {
#pragma unroll
                        for (int sg = 0; sg < SEGS; ++sg)
#pragma unroll
                            for (int y = 0; y < 4; ++y) kw[st][x][sg][y] = 0;
                    }
                }
            }
        };
        auto load_v = [&](int tile) {
#pragma unroll
            for (int st = 0; st < ST; ++st) {
                const int k0 = tile * KT + st * 16;
                const uint8_t* base = p.v + block_base(page_n[st], k0) + g * (D / 8);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int r = 2 * c + (x & 1) + 8 * (x >> 1);
                    // what lies outside the item's keys may be anything, and 0 x NaN is NaN: it is not read
                    if (page_n[st] >= 0 && k0 + r < key_hi && k0 + r >= key_lo) ld_codes<VW>(base + r * D, vw[st][x]);
                    else {
#pragma unroll
                        for (int y = 0; y < VW; ++y) vw[st][x][y] = 0;
                    }
                }
            }
        };

        int tile = tile_lo + warp;
        load_meta(tile);
        if (tile < tile_hi) {
            load_k(tile);
            load_v(tile);
        }
        while (tile < tile_hi) {
            const int next = tile + NW;
            float ks[ST], vs[ST];
            bool there[ST];
#pragma unroll
            for (int st = 0; st < ST; ++st) {
                ks[st] = ks_n[st];
                vs[st] = vs_n[st];
                there[st] = page_n[st] >= 0;
            }
            load_meta(next);
            // ---- scores: [key][row]
            float sc[ST][NT][4];
#pragma unroll
            for (int st = 0; st < ST; ++st)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 4; ++x) sc[st][nt][x] = 0.0f;
#pragma unroll
            for (int sg = 0; sg < SEGS; ++sg)
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    uint2 qf[NT];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) qf[nt] = q_s[(nt * MT + sg * 4 + y) * 32 + lane];
#pragma unroll
                    for (int st = 0; st < ST; ++st) {
                        uint32_t a[4];
                        e4m3x4_to_f16(kw[st][0][sg][y], a[0], a[2]);
                        e4m3x4_to_f16(kw[st][1][sg][y], a[1], a[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_f16_16816(sc[st][nt], a, qf[nt].x, qf[nt].y);
                    }
                }
            if (next < tile_hi) load_k(next);
            // ---- base-2 logits with the values' scale, mask, running maximum
            const int key0 = tile * KT;
            bool open = key0 >= all_lo && key0 + KT <= all_hi;
#pragma unroll
            for (int st = 0; st < ST; ++st) open = open && there[st];
            float top[NT][2], inv_vs[ST];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) top[nt][0] = top[nt][1] = -INFINITY;
#pragma unroll
            for (int st = 0; st < ST; ++st) {
                const float lv = __log2f(vs[st]);
                inv_vs[st] = __frcp_rn(vs[st]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float f = rf[nt][x & 1] * ks[st];
                        float u;
                        if (p.cap > 0.0f) u = fmaf(soft_cap(sc[st][nt][x] * f, p.cap, 2.0f * LOG2E / p.cap), LOG2E, lv);
                        else u = fmaf(sc[st][nt][x], f, lv);
                        if (!open) {
                            const int key = key0 + st * 16 + g + 8 * (x >> 1);
                            if (!there[st] || key >= row_hi[nt][x & 1] || key < row_lo[nt][x & 1]) u = -INFINITY;
                        }
                        sc[st][nt][x] = u;
                        top[nt][x & 1] = fmaxf(top[nt][x & 1], u);
                    }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float t = top[nt][x];
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
                    const float mn = fmaxf(m[nt][x], t), safe = mn == -INFINITY ? 0.0f : mn;
                    const float down = ex2(m[nt][x] - safe);
                    m[nt][x] = mn;
                    l[nt][x] *= down;
#pragma unroll
                    for (int j = 0; j < MT; ++j) {
                        acc[nt][j][x] *= down;
                        acc[nt][j][2 + x] *= down;
                    }
                    top[nt][x] = 15.0f - safe;
                }
            // ---- weights -> P^T fragments
            uint32_t pf[ST][NT][2];
#pragma unroll
            for (int st = 0; st < ST; ++st)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float w[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        w[x] = ex2(sc[st][nt][x] + top[nt][x & 1]);
                        l[nt][x & 1] = fmaf(w[x], inv_vs[st], l[nt][x & 1]);
                    }
                    pf[st][nt][0] = transpose_8x8(pack_f16x2(w[0], w[1]));
                    pf[st][nt][1] = transpose_8x8(pack_f16x2(w[2], w[3]));
                }
            // ---- values: [dimension][row]
#pragma unroll
            for (int i = 0; i < VW; ++i)
#pragma unroll
                for (int st = 0; st < ST; ++st) {
                    uint32_t a[4], e[4];
                    e4m3x4_to_f16(__byte_perm(vw[st][0][i], vw[st][1][i], 0x5140), a[0], a[1]);
                    e4m3x4_to_f16(__byte_perm(vw[st][2][i], vw[st][3][i], 0x5140), a[2], a[3]);
                    e4m3x4_to_f16(__byte_perm(vw[st][0][i], vw[st][1][i], 0x7362), e[0], e[1]);
                    e4m3x4_to_f16(__byte_perm(vw[st][2][i], vw[st][3][i], 0x7362), e[2], e[3]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma_f16_16816(acc[nt][2 * i], a, pf[st][nt][0], pf[st][nt][1]);
                        mma_f16_16816(acc[nt][2 * i + 1], e, pf[st][nt][0], pf[st][nt][1]);
                    }
                }
            if (next < tile_hi) load_v(next);
            tile = next;
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
                const int r = nt * 8 + 2 * c + x;
                if (g == 0) ml_s[warp][r] = make_float2(m[nt][x], t);
                float* dst = acc_s + ((size_t)warp * ROWS + r) * Cfg::PITCH + g * (D / 8);
#pragma unroll
                for (int j = 0; j < MT; j += 2)
                    *reinterpret_cast<float4*>(dst + 2 * j) =
                        make_float4(acc[nt][j][x], acc[nt][j][2 + x], acc[nt][j + 1][x], acc[nt][j + 1][2 + x]);
            }
        __syncthreads();
        const bool split = !(at == first && end == first + s.tiles);
        const int slot = at == w0 ? 0 : 1;
        const size_t part = (size_t)cta * 2 + slot;
        auto finish = [&](int r, int d4, float4 sum, float mm, float ll) {
            const int i = (row0 + r) / p.group, hh = h * p.group + (row0 + r) % p.group;
            const float inv = ll > 0.0f ? __frcp_rn(ll) : (ll == 0.0f ? 0.0f : ll);       // no key: zero; NaN stays
            uint2 out;
            out.x = pack_bf16x2(sum.x * inv, sum.y * inv);
            out.y = pack_bf16x2(sum.z * inv, sum.w * inv);
            const int token = s.start + i;
            st_global_v2(p.o + (size_t)token * p.o_stride + (size_t)hh * D + d4 * 4, out);
            if (d4 == 0 && p.lse)
                p.lse[(size_t)hh * p.tokens + token] = ll == 0.0f ? -INFINITY : 0.6931471805599453f * (mm - 15.0f + log2f(ll));
        };
        for (int x = tid; x < rows * (D / 4); x += Cfg::THREADS) {
            const int r = x / (D / 4), d4 = x % (D / 4);
            float mm = -INFINITY, ll = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) mm = fmaxf(mm, ml_s[w][r].x);
            const float safe = mm == -INFINITY ? 0.0f : mm;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < NW; ++w) {
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
            const long long last_unit = first + s.tiles - 1;
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
        at = end;
        first += s.tiles;
        ++item;
    }
}

template <int D, int NT>
static int paged_grid() { return min(device_sm_count() * PagedCfg<D, NT>::CTAS, PA_MAX_GRID); }
template <int D, int NT>
static long long paged_workspace() {
    return 4 * PA_MAX_GRID + (long long)paged_grid<D, NT>() * 2 * PagedCfg<D, NT>::ROWS * (D + 2) * 4;
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
    const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_attention_kernel<D, NT>, p);
    return e == cudaSuccess ? FRT_OK : FRT_CUDA_ERR(e);
}

}  // namespace frt

// Row tiles of 8 or 16: a decode step's group, or more rows, which then read the keys once per 16.
static bool paged_two(long long max_new, int hq, int hkv) { return max_new * (hq / hkv) > 8; }

extern "C" int frt_b200_paged_attention_workspace_bytes(int tokens, int batch, int max_new, int num_heads_q, int num_heads_kv,
                                                        int head_dim, long long* out_bytes) {
    using namespace frt;
    if (!out_bytes || tokens < 0 || batch < 0 || max_new < 0 || num_heads_q < 1 || num_heads_kv < 1) return FRT_ERR_INVALID;
    if (num_heads_q % num_heads_kv) return FRT_ERR_UNSUPPORTED;
    const bool two = paged_two(max_new, num_heads_q, num_heads_kv);
    if (head_dim == 64) *out_bytes = two ? paged_workspace<64, 2>() : paged_workspace<64, 1>();
    else if (head_dim == 128) *out_bytes = two ? paged_workspace<128, 2>() : paged_workspace<128, 1>();
    else if (head_dim == 256) *out_bytes = two ? paged_workspace<256, 2>() : paged_workspace<256, 1>();
    else return FRT_ERR_UNSUPPORTED;
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
    const bool two = paged_two(max_new, num_heads_q, num_heads_kv);
    if (head_dim == 64)
        return two ? launch_paged_attention<64, 2>(p, workspace, workspace_bytes, st)
                   : launch_paged_attention<64, 1>(p, workspace, workspace_bytes, st);
    if (head_dim == 128)
        return two ? launch_paged_attention<128, 2>(p, workspace, workspace_bytes, st)
                   : launch_paged_attention<128, 1>(p, workspace, workspace_bytes, st);
    return two ? launch_paged_attention<256, 2>(p, workspace, workspace_bytes, st)
               : launch_paged_attention<256, 1>(p, workspace, workspace_bytes, st);
}

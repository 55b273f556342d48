// Attention of new tokens over a paged E4M3 key/value cache (one scale per block and head), causal, ragged batches.
//
// No counterpart in the reference (its attention reads dense 16-bit K and V: csrc/attention/fa2_wrapper.cu).
//
// With c the stored codes, k_j = ks_p c_j and v_j = vs_p c_j (p: the page of key j), all in base 2:
//   t_ij = q_i . c_j * (softmax_scale * log2(e) * ks_p)        [capped: cap * tanh(s / cap)]
//   u_ij = t_ij + log2(vs_p),  m_i = max_j u_ij,  w_ij = 2^(u_ij - m_i + 15)
//   o_i = (sum_j w_ij c_j) / l_i,  l_i = sum_j w_ij / vs_p,  lse_i = ln 2 (m_i - 15 + log2 l_i)
// The values' scale goes into the exponent, so a weight that meets the codes is at most 2^15 whatever the scales are: it is rounded to
// fp16 (2^-11 relative down to 2^-29 of the largest; bf16 weights, 2^-8, would give up three bits) while every sum stays in fp32.  E4M3
// codes are fp16 values exactly; queries are brought below 1 by a power of two per row, which is exact as well as long as the eight bits
// of an element lie above fp16's last one, 2^-24: elements under 2^-16 of the row's largest may lose bits, those under 2^-25 vanish.
//
// What bounds it: a decode step reads every key and value once and does 4 x group flops per byte, so memory does, and the kernel is
// built to keep copies in flight.  Up to four warps copy -- a lane per block, by TMA, into a ring of stages, across the items of the CTA's
// work, so that neither the join of an item's warps nor the set-up of the next lets the memory wait -- and one or two groups of four
// take the stages in turn, a warp KT keys.
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
//
// Measured (times of a replayed graph): 64 sequences of 1500 .. 6000 tokens, 32 query and 8 key heads of 128, 87 to 90 us, 5.6 TB/s; two of 48000
// and 131071 tokens 81 to 82 us, 5.6 TB/s; one token on 819 keys, heads of 256, 10.7 us, of which the chain of dependent trips to memory is
// nearly all: lengths 1.9, queries 0.8, keys 0.8, products 1.0, joins of warps 1.4, arrival 1.2, join of CTAs 2.3.
#include "common.cuh"
#include "tc05.cuh"
#include "flashrt_b200.h"

#include <cuda_fp16.h>

#include <algorithm>
#include <climits>
#include <type_traits>

namespace frt {

// The head of a workspace: arrival counters of the CTAs.  A place of their own, whatever the shapes: every launch leaves them at zero, and no
// partial is written over them.
constexpr int PA_MAX_GRID = 512, PA_HEAD_BYTES = 4096;

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
    int room;                    // keys that a table row has entries for
    int few_rows;                // sequences with more query rows than this are the other kernel's
    int pool_rows;               // rows of a cache seen as a matrix of head_dim columns
    int* status;
    unsigned* counters;
    float2* part_ml;             // [cta][2][rows] (m, l)
    float* part_o;               // [cta][2][rows][D]
};

template <int D, int NT>
struct PagedCfg {
    static constexpr int ROWS = 8 * NT;
    // Warps that compute, in groups of four: a group takes a stage, a warp KT of its keys.  With eight rows two CTAs share an SM, each
    // with a group and a share of the line of its own: one joins an item while the other streams (64 sequences of 1500 .. 6000 tokens
    // 98.7 -> 90.4 us; heads of 256 on one short sequence 11.8 -> 16.7, so they keep one CTA).
    static constexpr int CTAS = NT == 1 && D <= 128 ? 2 : 1;
    static constexpr int GROUPS = CTAS == 2 ? 1 : 2;
    static constexpr int NW = 4 * GROUPS;
    static constexpr int KT = D == 256 ? 16 : 32;
    static constexpr int ST = KT / 16;
    static constexpr int UK = 4 * KT;                 // keys of a stage, and unit of the work line
    static constexpr int THREADS = 32 * (NW + 4);     // and a group that copies
    // registers of a thread: 128 or 168 at launch; the warps that compute take what the others give (4 x 176 + 4 x 80 = 8 x 128,
    // 8 x 200 + 4 x 104 = 12 x 168)
    static constexpr int REGS_COMPUTE = CTAS == 2 ? 176 : 200, REGS_COPY = CTAS == 2 ? 80 : 104;
    static constexpr int STAGE_BYTES = 2 * UK * D;
    static constexpr int BUFS = CTAS == 2 ? 2 : 4;    // warps whose accumulators are in shared memory at once
    static constexpr int PITCH = D + 4;               // floats of an accumulator row in shared memory
    static constexpr int Q_BYTES = NT * (D / 16) * 32 * 8;
    static constexpr int ACC_BYTES = BUFS * ROWS * PITCH * 4;
    static constexpr int ROOM = (CTAS == 2 ? 115200 - 1024 - 1536 : 232448 - 1024 - 6 * 1024) - Q_BYTES - ACC_BYTES;    // static: below 1536 or 6 K
    static constexpr int FIT = ROOM / STAGE_BYTES < 12 ? ROOM / STAGE_BYTES : 12;
    static constexpr int STAGES = FIT / GROUPS * GROUPS;
    // Warps that copy, each every COPIERS-th unit.  A warp that waits for a stage's k-th release tells it by the phase's parity, which is
    // right as long as the release before the last has happened.  Its own unit before, COPIERS back, found a stage whose unit
    // before, STAGES further back, was released, and one group's releases are in order: the same group as this stage's, if
    // COPIERS and STAGES are multiples of GROUPS, and a later unit than the one in question, if COPIERS <= STAGES.
    static constexpr int COPIERS = STAGES < 4 ? STAGES / GROUPS * GROUPS : 4;
    static_assert(COPIERS <= STAGES && COPIERS % GROUPS == 0 && STAGES % GROUPS == 0 && STAGES >= 2, "parity of a stage's releases");
    static constexpr int RING_BYTES = STAGES * STAGE_BYTES;
    static constexpr int SMEM_BYTES = 1024 + RING_BYTES + Q_BYTES + ACC_BYTES;
    static constexpr bool Q_REGS = NT == 1;           // query fragments stay in registers
    // The next stretch's queries are asked for in front of this one's join.  More rows have no registers for it: 16 sequences x 16 rows of
    // 256 on 4000 keys 41 us without, 44 with.
    static constexpr bool EARLY = NT == 1;
};

// First position that a token at `pos` sees.  A sequence with more new tokens than positions has negative ones, and a window may be any
// positive number: compared first, so that nothing leaves 32 bits.
__device__ __forceinline__ int window_from(const PagedAttnParams& p, int pos) {
    return p.window > 0 && pos >= p.window ? pos - p.window + 1 : 0;
}

// One sequence's share of the work line.
struct PagedSeq { int start, n, len, row_tiles, t0, tiles; };

template <int UK, int ROWS>
__device__ __forceinline__ PagedSeq paged_seq(const PagedAttnParams& p, int b) {
    PagedSeq s;
    s.start = p.cu ? min(max(p.cu[b], 0), p.tokens) : b;
    const int end = p.cu ? min(max(p.cu[b + 1], s.start), p.tokens) : b + 1;
    s.n = end - s.start;
    if ((long long)s.n * p.group > p.few_rows) s.n = 0;
    s.len = min(max(p.lens[b], 0), 0x7fffff00);
    s.row_tiles = (int)(((long long)s.n * p.group + ROWS - 1) / ROWS);
    s.t0 = window_from(p, s.len - s.n) / UK;
    s.tiles = max(1, (min(s.len, p.room) + UK - 1) / UK - s.t0);             // an item without keys still writes its rows
    return s;
}
template <int UK, int ROWS>
__device__ __forceinline__ long long paged_units(const PagedAttnParams& p, int b) {
    const PagedSeq s = paged_seq<UK, ROWS>(p, b);
    return (long long)s.row_tiles * s.tiles * p.hkv;
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float lg2(float x) {
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
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
// a box that nobody reads again soon: with the default policy a cache larger than L2 pushes itself through it (64 sequences of 1500 .. 6000 tokens 96.6 us for 90.4)
__device__ __forceinline__ void tma_load_once(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int y, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;"
        ::"r"(dst), "l"(m), "r"(bar), "r"(x), "r"(y), "l"(policy)
        : "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void st_shared_zero(uint32_t a) { asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(a), "r"(0) : "memory"); }
// atomicInc between the fences that a hand-over wants, without two full ones around it: 1700 clocks for 3400
__device__ __forceinline__ unsigned arrive_inc(unsigned* a, unsigned limit) {
    unsigned old;
    asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;" : "=r"(old) : "l"(a), "r"(limit) : "memory");
    return old;
}
// the warps that compute meet without those that copy
__device__ __forceinline__ void sync_threads(int n) { asm volatile("bar.sync 1, %0;" ::"r"(n) : "memory"); }

__device__ __forceinline__ float inverse_sum(float l) { return l > 0.0f ? __frcp_rn(l) : l; }
// e with 2^e > top for a row whose largest magnitude is top (zero, tiny: 0; infinite: 0 too, the row is NaN or infinite as it should be)
__device__ __forceinline__ int query_exponent(float top) {
    return top > 1e-30f && top < INFINITY ? min((int)((__float_as_uint(top) >> 23) & 255) - 126, 126) : 0;
}
// cap * tanh(s / cap).  Through the hardware's exp2 and reciprocal: 2^-22 of the cap, where tanh.approx has 2^-11.  For |s| <= cap / 2,
// which scores seldom leave, the first seven terms of the series (the next is below 10^-7 of the value): the exponential unit has
// the softmax's own to do.  A score takes the form of its own size: were it the tile's largest that chose, keys that a row does not see --
// tokens after it, what a block holds behind its sequence -- would reach the row's last bits.
__device__ __forceinline__ float soft_cap_far(float s, float cap, float inv_cap) {
    constexpr float LOG2E2 = 2.8853900817779268f;
    return cap * (1.0f - 2.0f * rcp(1.0f + ex2(s * inv_cap * LOG2E2)));
}
__device__ __forceinline__ float soft_cap_low(float s, float inv_cap) {
    const float x = s * inv_cap, y = x * x;
    float q = fmaf(y, 21844.0f / 6081075.0f, -1382.0f / 155925.0f);
    q = fmaf(q, y, 62.0f / 2835.0f);
    q = fmaf(q, y, -17.0f / 315.0f);
    q = fmaf(q, y, 2.0f / 15.0f);
    q = fmaf(q, y, -1.0f / 3.0f);
    return fmaf(s * y, q, s);
}
__device__ __forceinline__ float soft_cap(float s, float cap, float inv_cap) {
    const float far = soft_cap_far(s, cap, inv_cap), low = soft_cap_low(s, inv_cap);
    return fabsf(s) <= 0.5f * cap ? low : far;
}

// The line cut into `grid` stretches whose lengths differ by one at most.
struct PagedShare {
    long long each;
    int longer;                  // the first ones have one unit more
    __device__ __forceinline__ PagedShare(long long total, int grid) {
        each = total < 0x7fffffffLL ? (long long)((unsigned)total / (unsigned)grid) : total / grid;
        longer = (int)(total - each * grid);
    }
    __device__ __forceinline__ long long begin(int cta) const { return each * cta + min(cta, longer); }
    __device__ __forceinline__ int owner(long long unit) const {
        const long long head = (each + 1) * longer;
        if (unit < head) return head < 0x7fffffffLL ? (int)((unsigned)unit / (unsigned)(each + 1)) : (int)(unit / (each + 1));
        return longer + (unit - head < 0x7fffffffLL && each < 0x7fffffffLL ? (int)((unsigned)(unit - head) / (unsigned)each)
                                                                          : (int)((unit - head) / each));
    }
};

// A stretch of the work line inside one item: the units to copy, and where the item's rows are.
struct PagedSegment {
    int b, item;                 // sequence; (head, row tile) inside it
    long long first, end;        // line positions: of the item, behind the stretch
    int items, h, row0, rows, tiles;
    int len, n, start;
    int key_lo, key_hi;          // keys that any row sees
    int unit_lo, unit_hi;        // units of the stretch with such keys
};
// the stretch that begins at line position `at` < w1; b, item, first are set
template <int UK, int ROWS>
__device__ __forceinline__ void paged_segment(const PagedAttnParams& p, PagedSegment& g, long long at, long long w1) {
    PagedSeq s = paged_seq<UK, ROWS>(p, g.b);
    while (g.item >= s.row_tiles * p.hkv && g.b + 1 < p.batch) {             // through with the sequence, or one without new tokens
        ++g.b;
        g.item = 0;
        s = paged_seq<UK, ROWS>(p, g.b);
    }
    g.items = s.row_tiles * p.hkv;
    // one new token: no divisions, some 100 clocks each of a chain that nothing hides (one token on 819 keys 10.9 -> 10.7 us).  With more rows
    // a sequence the short cuts cost registers: 24 rows 80 -> 85 us
    const bool one = ROWS == 8 && s.n == 1;
    g.h = ROWS == 8 && s.row_tiles == 1 ? g.item : g.item / s.row_tiles;
    g.row0 = (g.item - g.h * s.row_tiles) * ROWS;
    g.rows = min(ROWS, s.n * p.group - g.row0);
    g.tiles = s.tiles;
    g.len = s.len;
    g.n = s.n;
    g.start = s.start;
    g.end = min(g.first + s.tiles, w1);
    const int p0 = s.len - s.n + (one ? 0 : g.row0 / p.group), p1 = s.len - s.n + (one ? 0 : (g.row0 + g.rows - 1) / p.group);
    g.key_lo = window_from(p, p0);
    g.key_hi = min(p.causal ? p1 + 1 : s.len, p.room);
    g.unit_lo = max(s.t0 + (int)(at - g.first), g.key_lo / UK);
    g.unit_hi = min(s.t0 + (int)(g.end - g.first), g.key_hi > 0 ? (g.key_hi + UK - 1) / UK : 0);
}

template <int D, int NT>
__global__ void __launch_bounds__((PagedCfg<D, NT>::THREADS), (PagedCfg<D, NT>::CTAS))
paged_attention_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, PagedAttnParams p) {
    using Cfg = PagedCfg<D, NT>;
    constexpr int ST = Cfg::ST, KT = Cfg::KT, UK = Cfg::UK, NW = Cfg::NW, ROWS = Cfg::ROWS, SEGS = D / 64, MT = D / 16;
    constexpr int STAGES = Cfg::STAGES, SCAN = 256;
    constexpr float LOG2E = 1.4426950408889634f;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint2* q_s = reinterpret_cast<uint2*>(smem + Cfg::RING_BYTES);           // [nt][k step][lane]
    float* acc_s = reinterpret_cast<float*>(smem + Cfg::RING_BYTES + Cfg::Q_BYTES);       // [warp][row][PITCH]
    __shared__ float2 ml_s[NW][ROWS];
    __shared__ float rf_s[ROWS];
    __shared__ float2 scale_s[STAGES][UK / 16];                              // per 16 keys: of the keys, of the values
    __shared__ uint64_t full_s[STAGES], empty_s[STAGES];
    __shared__ long long warp_s[SCAN / 32], first_s;
    __shared__ int begin_s[2];
    __shared__ unsigned last_s;
    __shared__ volatile int abort_s;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) {
            tc::mbar_init(&full_s[s], 2);                                    // the copies' bytes; the scales
            tc::mbar_init(&empty_s[s], 4);
        }
        abort_s = 0;
        tc::mbar_fence_init();
        tc::tma_prefetch_desc(&tmK);
        tc::tma_prefetch_desc(&tmV);
    }
    const uint64_t deadline = tc::global_timer_ns() + FRT_KERNEL_DEADLINE_NS;
    pdl_launch_dependents();
    pdl_wait();

    // ---------------- the work line: thread t counts the units of sequences [t * per, (t + 1) * per)
    const int per = (p.batch + SCAN - 1) / SCAN;
    long long mine = 0, incl;
    if (tid < SCAN) {
        for (int b = tid * per; b < min((tid + 1) * per, p.batch); ++b) mine += paged_units<UK, ROWS>(p, b);
        incl = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long o = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += o;
        }
        if (lane == 31) warp_s[warp] = incl;
    }
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < SCAN / 32; ++w) {
        if (w < warp) before += warp_s[w];
        total += warp_s[w];
    }
    // A unit for every CTA, which then meets one item: 16 rows of 64 on 300 keys 13.8 us with a unit for every group, 8.1 so.  Items of more
    // than 16 units (that many pieces' loads are in flight together at a join) keep every group busy: on 4000 keys 9.5 and 10.8.
    const bool dense = Cfg::GROUPS == 2 && total > 16LL * p.batch * p.hkv;
    const int grid = (int)max(1LL, min((long long)gridDim.x, dense ? (total + 1) >> 1 : total));
    const int cta = blockIdx.x;
    if (cta >= grid || total == 0) return;
    const PagedShare share(total, grid);
    const long long w0 = share.begin(cta), w1 = share.begin(cta + 1);
    if (tid < SCAN && mine > 0) {
        long long first = before + incl - mine;
        if (first <= w0 && w0 < first + mine) {                              // one thread's sequences hold the first unit
            int b = tid * per;
            for (;;) {
                const long long u = per == 1 ? mine : paged_units<UK, ROWS>(p, b);
                if (w0 < first + u) break;
                first += u;
                ++b;
            }
            const int units = paged_seq<UK, ROWS>(p, b).tiles;
            const long long in = w0 - first;
            const int item = in < 0x7fffffffLL ? (int)((unsigned)in / (unsigned)units) : (int)(in / units);
            begin_s[0] = b;
            begin_s[1] = item;
            first_s = first + (long long)item * units;
        }
    }
    __syncthreads();
    PagedSegment cur;
    cur.b = begin_s[0];
    cur.item = begin_s[1];
    cur.first = first_s;
    paged_segment<UK, ROWS>(p, cur, w0, w1);
    int stage = 0;
    uint32_t phase = 0;

    auto next_segment = [&](PagedSegment& s) {                               // a stretch that does not end the work ends its item
        const long long at = s.end;
        s.first = at;
        ++s.item;
        paged_segment<UK, ROWS>(p, s, at, w1);
    };
    if (warp >= NW) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::REGS_COPY));
        if (warp >= NW + Cfg::COPIERS) return;
        // ---------------- copies: a warp takes every COPIERS-th unit, a lane a block (or the unit's part of one) of its keys or of its values.
        // A unit costs its warp 1800 to 2600 clocks -- two dependent trips to memory for block number and scale, and some 100 a copy,
        // which its uniform operands make the lanes issue one by one -- where a stage takes 2700 to arrive (of 256 keys then): with one warp, 64 sequences
        // of 1500 .. 6000 tokens in blocks of 32 took 99.6 us
        const uint32_t ring = tc::smem_u32(smem), full_a = tc::smem_u32(full_s), empty_a = tc::smem_u32(empty_s);
        const int box = min(UK, p.block_size), boxes = UK / box;
        constexpr int INNER = D < 128 ? D : 128;
        constexpr int PER_LANE = UK / 16 * 2 / 32 > 0 ? UK / 16 * 2 / 32 : 1;       // copies of a lane at most
        const float* my_scale = lane & 1 ? p.v_scale : p.k_scale;
        const CUtensorMap* map = lane & 1 ? &tmV : &tmK;
        const uint64_t once = tc::l2_policy_evict_first();
        struct Unit {
            int page[PER_LANE];      // table entry; INT_MIN: no key of the item there
            int h, k0;               // key/value head, first key
            bool there;
        };
        int u = cur.unit_lo, skip = warp - NW;                               // this warp's next unit is `skip` behind u
        auto ask_pages = [&](Unit& n) {
            n.there = false;
            for (;;) {
                const int left = max(cur.unit_hi - u, 0);
                if (skip < left) break;
                skip -= left;
                if (cur.end >= w1) { u = cur.unit_hi; return; }
                next_segment(cur);
                u = cur.unit_lo;
            }
            u += skip;
            skip = Cfg::COPIERS;
            n.there = true;
            n.h = cur.h;
            n.k0 = u * UK;
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i) {
                const int k0 = u * UK + ((lane + 32 * i) >> 1) * box;
                const bool want = (lane + 32 * i) >> 1 < boxes && k0 < cur.key_hi && k0 + box > cur.key_lo;
                n.page[i] = want ? max(p.table[(size_t)cur.b * p.table_stride + (k0 >> p.block_shift)], -1) : INT_MIN;
            }
        };
        Unit now, next;
        float scale[PER_LANE];
        auto ask_scales = [&] {
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i) {
                if (now.page[i] >= p.num_blocks) now.page[i] = -1;
                if (now.there && now.page[i] >= 0) scale[i] = my_scale[(size_t)now.page[i] * p.hkv + now.h];
            }
        };
        auto step = [&](int n) {                                             // units -> stages
            stage += n;
            while (stage >= STAGES) { stage -= STAGES; phase ^= 1; }
        };
        step(warp - NW);
        ask_pages(now);
        ask_pages(next);
        ask_scales();
        while (now.there) {
            unsigned wanted = 0;
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i) wanted += __popc(__ballot_sync(0xffffffffu, now.page[i] != INT_MIN));
            if (!tc::warp_wait(empty_a + 8 * stage, phase ^ 1, false, deadline, &abort_s)) {
                if (lane == 0 && !abort_s) atomicCAS(p.status, 0, 1 | (blockIdx.x << 8));
                abort_s = 1;
                return;
            }
            const uint32_t bar = full_a + 8 * stage, dst = ring + stage * Cfg::STAGE_BYTES;
            if (lane == 0) tc::mbar_arrive_expect_tx(bar, wanted * (unsigned)(box * D));
            __syncwarp();
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i) {
                if (now.page[i] == INT_MIN) continue;
                const int n = (lane + 32 * i) >> 1, in_block = (now.k0 + n * box) & (p.block_size - 1);
                // no block of the pool: rows behind its end, which arrive as zeros
                const int row = now.page[i] >= 0 ? (now.page[i] * p.hkv + now.h) * p.block_size + in_block : p.pool_rows;
                const uint32_t to = dst + (lane & 1) * (UK * D) + n * box * INNER;
#pragma unroll
                for (int x = 0; x < D; x += INNER) tma_load_once(to + x * UK, map, bar, x, row, once);
                for (int j = 0; j < box / 16; ++j) (&scale_s[stage][n * (box / 16) + j].x)[lane & 1] = now.page[i] >= 0 ? fmaxf(scale[i], 1e-30f) : 0.0f;
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&full_s[stage]);
            step(Cfg::COPIERS);
            now = next;
            ask_scales();
            ask_pages(next);
        }
        return;
    }

    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::REGS_COMPUTE));

    // where this lane's operands are in its warp's part of a stage (see the top: groups of lanes four rows or chunks apart)
    const int krow = D == 64 ? g : (g >> 1) | ((g & 1) << 2), dchunk = krow;
    const uint32_t k_off = D == 64 ? g * 64 + ((c ^ ((g >> 1) & 3)) << 4) : krow * 128 + ((c ^ krow) << 4);
    const uint32_t v_off = (D == 64 ? 2 * c * 64 + (((g >> 1) ^ c) << 4) + (g & 1) * 8 : c * 128 + ((dchunk ^ c) << 4));
    constexpr int STEP = D == 64 ? 64 : 128;                                 // bytes from row to row
    const int group = warp >> 2, part_w = warp & 3;
    int turn = 0;
    const bool capped = p.cap > 0.0f;
    const float inv_cap = capped ? 1.0f / p.cap : 0.0f;

    // a warp's query rows of a stretch, asked for while the stretch before is joined
    constexpr int PL = D / 32, RW = ROWS / NW;                               // dimensions of a lane, rows of a warp
    uint32_t raw[RW][PL / 2];
    auto ask_queries = [&](const PagedSegment& s) {
#pragma unroll
        for (int k = 0; k < RW; ++k) {
            const int at_row = s.row0 + min(warp + k * NW, s.rows - 1), i = NT == 1 && s.n == 1 ? 0 : at_row / p.group, hh = s.h * p.group + at_row - i * p.group;
            const uint32_t* src = reinterpret_cast<const uint32_t*>(p.q + (size_t)(s.start + i) * p.q_stride + (size_t)hh * D + lane * PL);
#pragma unroll
            for (int j = 0; j < PL / 2; ++j) raw[k][j] = src[j];
        }
    };
    if constexpr (Cfg::EARLY) ask_queries(cur);
    for (long long at = w0; at < w1;) {
        if constexpr (!Cfg::EARLY) {
            if (at != w0) next_segment(cur);
            ask_queries(cur);
        }
        const int rows = cur.rows, row0 = cur.row0, h = cur.h;

        // queries -> fp16 operand fragments, at most 1 in magnitude: one warp per row
        sync_threads(32 * NW);                                               // the item before is through with shared memory
#pragma unroll
        for (int k = 0; k < RW; ++k) {
            const int r = warp + k * NW;
            float x[PL];
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < PL / 2; ++j) unpack_bf16x2(r < rows ? raw[k][j] : 0u, x[2 * j], x[2 * j + 1]);
#pragma unroll
            for (int j = 0; j < PL; ++j) top = fmaxf(top, fabsf(x[j]));
            top = warp_max_butterfly(top);
            const int e = query_exponent(top);
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
        sync_threads(32 * NW);

        // this lane's rows: 2c, 2c + 1 of every n tile
        float rf[NT][2];
        int row_hi[NT][2], row_lo[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int r = nt * 8 + 2 * c + x;
                rf[nt][x] = rf_s[r] * p.scale * (capped ? 1.0f : LOG2E);
                const int pos = cur.len - cur.n + (NT == 1 && cur.n == 1 ? 0 : (row0 + min(r, rows - 1)) / p.group);
                row_hi[nt][x] = min(p.causal ? pos + 1 : cur.len, cur.key_hi);
                row_lo[nt][x] = window_from(p, pos);
            }
        const bool one = NT == 1 && cur.n == 1;
        const int p0 = cur.len - cur.n + (one ? 0 : row0 / p.group), p1 = cur.len - cur.n + (one ? 0 : (row0 + rows - 1) / p.group);
        const int all_hi = min(p.causal ? p0 + 1 : cur.len, cur.key_hi);      // keys that every row sees
        const int all_lo = window_from(p, p1);
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

        // the group's units of the stretch; `stage`, `phase`, `turn`: of the stretch's first
        const int units = max(cur.unit_hi - cur.unit_lo, 0);
        int off = group - turn;
        if (off < 0) off += Cfg::GROUPS;
        int st_i = stage + off;
        uint32_t ph_i = phase;
        if (st_i >= STAGES) { st_i -= STAGES; ph_i ^= 1; }
        turn = (turn + units) % Cfg::GROUPS;
        phase ^= (uint32_t)((stage + units) / STAGES) & 1u;
        stage = (stage + units) % STAGES;
        for (; off < units; off += Cfg::GROUPS) {
            const int key0 = (cur.unit_lo + off) * UK + part_w * KT;
            if (!tc::mbar_wait_until(&full_s[st_i], ph_i, deadline, &abort_s)) {
                if (!abort_s && lane == 0) atomicCAS(p.status, 0, 2 | (blockIdx.x << 8));
                abort_s = 1;
            }
            __syncwarp();
            if (key0 < cur.key_hi && key0 + KT > cur.key_lo) {
            const uint32_t base = tc::smem_u32(smem) + st_i * Cfg::STAGE_BYTES + part_w * (KT * STEP), base_v = base + UK * D;
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
                const uint32_t kb = base + (sg >> 1) * (UK * 128) + (sg & 1 ? k_off ^ 64 : k_off);
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
            bool open = key0 >= all_lo && key0 + KT <= all_hi;
            float ks[ST], lv[ST], inv_vs[ST], top[NT][2];
#pragma unroll
            for (int st = 0; st < ST; ++st) {
                // a step without keys of the item has no scales: anything, all of it masked
                const float2 s = scale_s[st_i][part_w * ST + st];
                const bool there = s.y != 0.0f && key0 + st * 16 < cur.key_hi && key0 + st * 16 + 16 > cur.key_lo;
                open = open && there;
                ks[st] = there ? s.x : 0.0f;
                lv[st] = there ? lg2(s.y) : 0.0f;
                inv_vs[st] = there ? rcp(s.y) : 0.0f;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) top[nt][0] = top[nt][1] = -INFINITY;
#pragma unroll
            for (int st = 0; st < ST; ++st)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float f[2] = {rf[nt][0] * ks[st], rf[nt][1] * ks[st]};
#pragma unroll
                    for (int x = 0; x < 4; ++x) sc[st][nt][x] = fmaf(sc[st][nt][x], f[x & 1], capped ? 0.0f : lv[st]);
                }
            if (capped) {
                float far = 0.0f;
#pragma unroll
                for (int st = 0; st < ST; ++st)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int x = 0; x < 4; ++x) far = fmaxf(far, fabsf(sc[st][nt][x]));
                const bool low = __all_sync(0xffffffffu, far <= 0.5f * p.cap);
#pragma unroll
                for (int st = 0; st < ST; ++st)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const float s = sc[st][nt][x];
                            sc[st][nt][x] = fmaf(low ? soft_cap_low(s, inv_cap) : soft_cap(s, p.cap, inv_cap), LOG2E, lv[st]);
                        }
            }
            if (!open) {
                // values outside the item's keys may be anything, and 0 x NaN is NaN: zero their rows, 16 bytes a lane
                for (int i = lane; i < KT * (D / 16); i += 32) {
                    const int r = i / (D / 16), ch = i % (D / 16);
                    if (key0 + r >= cur.key_hi || key0 + r < cur.key_lo)
                        st_shared_zero(base_v + (D == 256 ? (ch >> 3) * (UK * 128) + r * 128 + (ch & 7) * 16 : r * STEP + ch * 16));
                }
                tc::fence_proxy_async_smem();                                // before the next copy of this stage
                __syncwarp();
#pragma unroll
                for (int st = 0; st < ST; ++st)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const int key = key0 + st * 16 + krow + 8 * (x >> 1);
                            if (ks[st] == 0.0f || key >= row_hi[nt][x & 1] || key < row_lo[nt][x & 1]) sc[st][nt][x] = -INFINITY;
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
                            const uint2 w = ld_shared_v2(base_v + v_off + (st * 16 + (x & 1) + 8 * (x >> 1)) * 64);
                            vw[x][0] = w.x; vw[x][1] = w.y;
                        } else {
                            const uint4 w = ld_shared_v4(base_v + (x & 1 ? (v_off ^ 64) + 512 : v_off) + (st * 16 + 8 * (x >> 1)) * 128 +
                                                         half * (UK * 128));
                            vw[x][0] = w.x; vw[x][1] = w.y; vw[x][2] = w.z; vw[x][3] = w.w;
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
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&empty_s[st_i]);
            st_i += Cfg::GROUPS;
            if (st_i >= STAGES) { st_i -= STAGES; ph_i ^= 1; }
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
        PagedSegment after = cur;
        if constexpr (Cfg::EARLY) {
            if (cur.end < w1) {
                next_segment(after);
                ask_queries(after);
            }
        }
        // four warps at a time hand theirs to the four below, until four are left
        constexpr int BUFS = Cfg::BUFS;
#pragma unroll 1
        for (int top_warp = NW; top_warp > BUFS; top_warp -= BUFS) {
            if (warp >= top_warp - BUFS && warp < top_warp) put(warp & (BUFS - 1));
            sync_threads(32 * NW);
            if (warp >= top_warp - 2 * BUFS && warp < top_warp - BUFS) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int r = nt * 8 + 2 * c + x;
                        const float2 a = ml_s[warp][r], b = ml_s[warp + BUFS][r];
                        const float mm = fmaxf(a.x, b.x), safe = mm == -INFINITY ? 0.0f : mm, fa = ex2(a.x - safe), fb = ex2(b.x - safe);
#pragma unroll
                        for (int i = 0; i < MT / 2; ++i) {
                            const float4 o = *place(warp & (BUFS - 1), nt, x, i);
                            acc[nt][2 * i][x] = acc[nt][2 * i][x] * fa + o.x * fb;
                            acc[nt][2 * i][2 + x] = acc[nt][2 * i][2 + x] * fa + o.y * fb;
                            acc[nt][2 * i + 1][x] = acc[nt][2 * i + 1][x] * fa + o.z * fb;
                            acc[nt][2 * i + 1][2 + x] = acc[nt][2 * i + 1][2 + x] * fa + o.w * fb;
                        }
                        __syncwarp();
                        if (g == 0) ml_s[warp][r] = make_float2(mm, a.y * fa + b.y * fb);
                    }
            }
        }
        if (warp < BUFS) put(warp);
        sync_threads(32 * NW);
        const bool split = !(at == cur.first && cur.end == cur.first + cur.tiles);
        const int slot = at == w0 ? 0 : 1;
        const size_t part = (size_t)cta * 2 + slot;
        auto finish = [&](int r, int d4, float4 sum, float mm, float ll) {
            const int i = NT == 1 && cur.n == 1 ? 0 : (row0 + r) / p.group, hh = h * p.group + row0 + r - i * p.group;
            const float inv = inverse_sum(ll);
            uint2 out;
            out.x = pack_bf16x2(sum.x * inv, sum.y * inv);
            out.y = pack_bf16x2(sum.z * inv, sum.w * inv);
            const int token = cur.start + i;
            st_global_v2(p.o + (size_t)token * p.o_stride + (size_t)hh * D + d4 * 4, out);
            if (d4 == 0 && p.lse)
                p.lse[(size_t)hh * p.tokens + token] = ll == 0.0f ? -INFINITY : 0.6931471805599453f * (mm - 15.0f + log2f(ll));
        };
        for (int x = tid; x < rows * (D / 4); x += 32 * NW) {
            const int r = x / (D / 4), d4 = x % (D / 4);
            float mm = -INFINITY, ll = 0.0f;
#pragma unroll
            for (int w = 0; w < BUFS; ++w) mm = fmaxf(mm, ml_s[w][r].x);
            const float safe = mm == -INFINITY ? 0.0f : mm;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < BUFS; ++w) {
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
            const int c0 = share.owner(first), c1 = share.owner(last_unit);
            sync_threads(32 * NW);
            if (tid == 0) {
                // releases the whole CTA's stores (it met at the barrier), acquires the others'
                last_s = arrive_inc(p.counters + c0, (unsigned)(c1 - c0)) == (unsigned)(c1 - c0);
            }
            sync_threads(32 * NW);
            if (last_s) {
                const int slot0 = share.begin(c0) < first;                   // the first CTA had another item in front
                const int pieces = c1 - c0 + 1;
                const size_t part0 = (size_t)c0 * 2 + slot0;                 // the others' are at 2 (c0 + q)
                auto part_of = [&](int q) { return (q ? ((size_t)c0 + q) * 2 : part0) * ROWS; };
                for (int x = tid; x < rows * (D / 4); x += 32 * NW) {
                    const int r = x / (D / 4), d4 = x % (D / 4);
                    float mm = -INFINITY, ll = 0.0f;
                    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    constexpr int B = 16;                                    // pieces whose loads are in flight together
#pragma unroll 1
                    for (int q0 = 0; q0 < pieces; q0 += B) {
                        float2 ml[B];
                        float4 v[B];
#pragma unroll
                        for (int q = 0; q < B; ++q) {
                            const bool there = q0 + q < pieces;
                            ml[q] = there ? __ldcg(p.part_ml + part_of(q0 + q) + r) : make_float2(-INFINITY, 0.0f);
                            v[q] = there ? __ldcg(reinterpret_cast<const float4*>(p.part_o + (part_of(q0 + q) + r) * D + d4 * 4))
                                         : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        }
                        float now = mm;
#pragma unroll
                        for (int q = 0; q < B; ++q) now = fmaxf(now, ml[q].x);
                        const float safe = now == -INFINITY ? 0.0f : now, keep = ex2(mm - safe);
                        mm = now;
                        ll *= keep;
                        sum.x *= keep; sum.y *= keep; sum.z *= keep; sum.w *= keep;
#pragma unroll
                        for (int q = 0; q < B; ++q) {
                            const float f = ex2(ml[q].x - safe);
                            ll = fmaf(ml[q].y, f, ll);
                            sum.x = fmaf(v[q].x, f, sum.x); sum.y = fmaf(v[q].y, f, sum.y);
                            sum.z = fmaf(v[q].z, f, sum.z); sum.w = fmaf(v[q].w, f, sum.w);
                        }
                    }
                    finish(r, d4, sum, mm, ll);
                }
            }
        }
        at = cur.end;
        if constexpr (Cfg::EARLY) cur = after;
    }
    if (abort_s) {                       // a wait gave up: copies may be in flight, a bounded time for them to land
        const uint64_t until = tc::global_timer_ns() + 1000000ull;
        while (tc::global_timer_ns() < until) {}
    }
}

template <int D, int NT>
static int paged_grid() { return min(device_sm_count() * PagedCfg<D, NT>::CTAS, PA_MAX_GRID); }
template <int D, int NT>
static long long paged_workspace() {
    return PA_HEAD_BYTES + (long long)paged_grid<D, NT>() * 2 * PagedCfg<D, NT>::ROWS * (D + 2) * 4;
}

// A cache as a matrix of head_dim bytes a row; boxes of `box` rows x 128 bytes (64 for heads of 64), swizzled over that width, or of whole
// rows as they are.  Rows
// behind the last one read as zeros.
static int paged_map(CUtensorMap* out, const void* base, int rows, int d, int box, bool swizzled) {
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
    const cuuint32_t boxes[2] = {(cuuint32_t)(swizzled && d > 128 ? 128 : d), (cuuint32_t)box}, ones[2] = {1, 1};
    const CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, boxes, ones,
                              CU_TENSOR_MAP_INTERLEAVE_NONE,
                              !swizzled ? CU_TENSOR_MAP_SWIZZLE_NONE : d < 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? FRT_OK : FRT_ERR_INVALID;
}

template <int D, int NT>
static int launch_paged_attention(PagedAttnParams p, void* work, cudaStream_t stream) {
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
    p.counters = static_cast<unsigned*>(work);
    p.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(work) + PA_HEAD_BYTES);
    p.part_o = reinterpret_cast<float*>(p.part_ml + (size_t)grid * 2 * Cfg::ROWS);
    CUtensorMap tmK, tmV;
    const int box = Cfg::UK < p.block_size ? Cfg::UK : p.block_size;
    int rc = paged_map(&tmK, p.k, p.pool_rows, D, box, true);
    if (!rc) rc = paged_map(&tmV, p.v, p.pool_rows, D, box, true);
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

#include "paged_prefill.cuh"

}  // namespace frt

// Row tiles of 8 NT rows, no wider than the rows need (at most paged_few of them).
static int paged_nt(long long rows) { return rows > 16 ? 3 : rows > 8 ? 2 : 1; }
// Query rows of a sequence up to which the kernel for few rows takes it.  16 sequences x 4 key/value heads on 4000 keys, this kernel and the
// other: heads of 128, 16 rows 25 and 38 us, 24 rows 32 and 38, 32 rows 66 and 42; of 64, 24 rows 23 and 31, 32 rows 36 and 33; of 256,
// 16 rows 41 and 63, 24 rows 108 and 64.  Heads of 256 in few sequences (one: 33 and 19, four: 31 and 26): a join of two row tiles by one
// CTA takes longer than the other kernel's launch for it.
static int paged_few(int d, long long items) { return d < 256 ? 24 : items > 16 ? 16 : 8; }
// f(head dim, row tiles of a CTA)
template <typename F>
static auto prefill_dispatch(int d, long long rows, F f) {
    using std::integral_constant;
    if (d == 256) return f(integral_constant<int, 256>(), integral_constant<int, 1>());
    if (d == 128) return rows > 128 ? f(integral_constant<int, 128>(), integral_constant<int, 2>())
                                    : f(integral_constant<int, 128>(), integral_constant<int, 1>());
    return rows > 128 ? f(integral_constant<int, 64>(), integral_constant<int, 2>())
                      : f(integral_constant<int, 64>(), integral_constant<int, 1>());
}
// f(kernel's head dim, row tile) for one of the instances
template <typename F>
static auto paged_dispatch(int d, int nt, F f) {
    using std::integral_constant;
    auto with = [&](auto D) {
        if constexpr (D() != 256) {
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
    const int group = num_heads_q / num_heads_kv, few = paged_few(head_dim, LLONG_MAX);
    const long long rows = (long long)max_new * group;
    *out_bytes = paged_dispatch(head_dim, paged_nt(rows < few ? rows : few), [](auto D, auto NT) { return paged_workspace<D(), NT()>(); });
    if (rows > paged_few(head_dim, 0)) *out_bytes += prefill_workspace(head_dim);        // fewer sequences may go there sooner
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
        window < 0 || !(softcap == 0.0f || (softcap >= 1e-30f && softcap <= 1e30f)) || !(softmax_scale > 0.0f && softmax_scale < 1e30f))
        return FRT_ERR_INVALID;                              // a cap's reciprocal is a number too
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
    p.room = (int)std::min((long long)table_stride * block_size, 0x7fffff00LL);
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
    const cudaStream_t stream_of = static_cast<cudaStream_t>(stream);
    const long long pool_rows = (long long)num_blocks * num_heads_kv * block_size;
    if (pool_rows > 0x7fffffffLL) return FRT_ERR_UNSUPPORTED;
    p.pool_rows = (int)pool_rows;
    static PerDevicePointer status;
    p.status = status.get(attention_status_device_ptr);
    if (!p.status) return FRT_ERR_UNSUPPORTED;
    // Sequences of few rows and of many go to different kernels.  A batch with room for max_new tokens of every sequence most likely has
    // them: the kernel for many rows takes all of it, whatever a padded batch holds in the end.
    const int few = paged_few(head_dim, (long long)batch * num_heads_kv);
    const long long rows = (long long)max_new * p.group;
    const bool many = rows > few, some_few = !many || (long long)batch * max_new != tokens;
    p.few_rows = !many ? INT_MAX : some_few ? few : 0;
    uint8_t* work = static_cast<uint8_t*>(workspace);
    int rc = paged_dispatch(head_dim, paged_nt(rows < few ? rows : few), [&](auto D, auto NT) {
        const long long need = paged_workspace<D(), NT()>();
        // of both kernels, in front of the first launch: a call that is refused has written nothing
        if (workspace_bytes < need + (many ? prefill_workspace(D()) : 0)) return (int)FRT_ERR_INVALID;
        const int r = some_few ? launch_paged_attention<D(), NT()>(p, work, stream_of) : FRT_OK;
        work += need;
        return r;
    });
    if (rc || !many) return rc;
    return prefill_dispatch(head_dim, rows, [&](auto D, auto T) { return launch_prefill<D(), T()>(p, max_new, work, stream_of); });
}

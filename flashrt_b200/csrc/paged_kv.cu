// New tokens into a paged E4M3 key/value cache with one scale per (block, head), the rotary position applied on the way.
//
// Stands beside qkv_split_rope[_devpos] (csrc/kernels/rope.cu:135-277 of the reference), which appends the rows of one sequence to a
// dense bf16 cache; the paged 8-bit form has no counterpart there.
//
//   position of new token i of a sequence: p = seq_len - new + i, block j = p / block_size, page = block_table[seq][j]
//   scale  s = max(s_old if the block holds earlier tokens, max |y| / 448 over the block's new tokens, 1e-12)
//   codes  e4m3(clamp(y * (1 / s), +-448)); codes that the block holds already: e4m3(c * (s_old / s)) where s has grown
//
// One group of threads owns a (block, head, K or V): it sees all new values of the block, so the scale needs no atomics and the result
// no order.  A warp is a group where sequences bring few tokens (a decode batch has batch x 2 heads such blocks of one row), 256
// threads where a block is filled at once.  A group walks the "leaders" of its chunk of packed tokens -- the first new token of a
// sequence and every token at the head of a block -- so nothing has to be known on the host about where sequences begin.  Values are
// kept in registers between the maximum and the codes, two pieces of 16 a thread; what is beyond that is read twice.
#include "common.cuh"
#include "flashrt_b200.h"

namespace frt {

struct PagedAppendParams {
    const __nv_bfloat16* qkv;
    long long qkv_stride;
    const float* rope;           // (rope_rows, head_dim): cos, sin of each pair; NULL: no rotation
    int rope_rows;
    __nv_bfloat16* q;            // (tokens, heads_q * head_dim) or NULL
    uint8_t *k, *v;              // (num_blocks, heads_kv, block_size, head_dim)
    float *k_scale, *v_scale;    // (num_blocks, heads_kv)
    const int *table, *cu, *lens;
    int table_stride, tokens, batch, num_blocks, block_size, hq, hkv, d;
    int chunk;                   // packed tokens of a group
    int q_heads;                 // query heads of a thread: one read of the angles for all of them
    unsigned kv_items, kv_blocks;
};

// Where a packed token stands.  `end`: first packed token behind its sequence.
struct TokenPlace { int seq, pos, start, end; };

__device__ __forceinline__ TokenPlace place_of(const int* cu, const int* lens, int batch, int tokens, int t) {
    TokenPlace r;
    if (!cu) {                                   // one token per sequence
        r.seq = t;
        r.start = t;
        r.end = t + 1;
        r.pos = t < batch ? lens[t] - 1 : -1;
        return r;
    }
    int lo = 0, hi = batch;                      // largest seq with cu[seq] <= t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= t) lo = mid; else hi = mid;
    }
    r.seq = lo;
    r.start = max(cu[lo], 0);
    r.end = min(cu[lo + 1], tokens);
    r.pos = t >= r.start && t < r.end ? lens[lo] - (r.end - t) : -1;
    if (t >= r.end) r.end = tokens;              // behind the last sequence
    return r;
}

// x c + y s, the rounding error of y s given back (Kahan): half a unit in the last place or little more, where the plain fma has two and
// more when the products nearly cancel.  Codes near the middle of two go the right way more often.  An infinite y s has no error to give
// back (infinity minus itself would make the element NaN): the plain sum stands, infinite, or NaN where x c is the other infinity.
__device__ __forceinline__ float two_products(float x, float c, float y, float s) {
    const float w = __fmul_rn(y, s), e = __fmaf_rn(y, s, -w), plain = __fmaf_rn(x, c, w), sum = __fadd_rn(plain, e);
    return sum == sum ? sum : plain;
}
// 16 values of one head: 16 neighbours, or (HALVES) 8 of the first half and their partners of the second.
template <bool HALVES>
struct Sixteen {
    float a[8], b[8];            // pairs (a[i], b[i])
    __device__ __forceinline__ void load(const __nv_bfloat16* row, int unit, int d) {
        const uint4 x = ld_stream_v4(row + (HALVES ? unit * 8 : unit * 16));
        const uint4 y = ld_stream_v4(row + (HALVES ? d / 2 + unit * 8 : unit * 16 + 8));
        const uint32_t* xw = &x.x;
        const uint32_t* yw = &y.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (HALVES) {
                unpack_bf16x2(xw[i], a[2 * i], a[2 * i + 1]);
                unpack_bf16x2(yw[i], b[2 * i], b[2 * i + 1]);
            } else {
                unpack_bf16x2(xw[i], a[i], b[i]);
                unpack_bf16x2(yw[i], a[4 + i], b[4 + i]);
            }
        }
    }
    // table row: pair i of the head at floats 2 i, 2 i + 1
    __device__ __forceinline__ void load_angles(const float* row, int unit, float4 (&t)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = ld_global_f4(row + unit * 16 + 4 * i);
    }
    // EXACT: for values that become codes; a query is rounded to bf16, which hides the plain fma's second rounding
    template <bool EXACT>
    __device__ __forceinline__ void turn(const float4 (&t)[4]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float cs = i & 1 ? t[i / 2].z : t[i / 2].x, sn = i & 1 ? t[i / 2].w : t[i / 2].y;
            const float x = a[i], y = b[i];
            a[i] = EXACT ? two_products(x, cs, -y, sn) : __fmaf_rn(x, cs, -__fmul_rn(y, sn));
            b[i] = EXACT ? two_products(y, cs, x, sn) : __fmaf_rn(y, cs, __fmul_rn(x, sn));
        }
    }
    // largest finite magnitude
    __device__ __forceinline__ float largest() const {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, fmaxf(fabsf(a[i]), fabsf(b[i])));
        if (m == INFINITY) {
            m = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = fabsf(a[i]), y = fabsf(b[i]);
                if (x < INFINITY) m = fmaxf(m, x);
                if (y < INFINITY) m = fmaxf(m, y);
            }
        }
        return m;
    }
    __device__ __forceinline__ void store_bf16(__nv_bfloat16* row, int unit, int d) const {
        uint4 x, y;
        uint32_t* xw = &x.x;
        uint32_t* yw = &y.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            xw[i] = HALVES ? pack_bf16x2(a[2 * i], a[2 * i + 1]) : pack_bf16x2(a[i], b[i]);
            yw[i] = HALVES ? pack_bf16x2(b[2 * i], b[2 * i + 1]) : pack_bf16x2(a[4 + i], b[4 + i]);
        }
        st_global_v4(row + (HALVES ? unit * 8 : unit * 16), x);
        st_global_v4(row + (HALVES ? d / 2 + unit * 8 : unit * 16 + 8), y);
    }
    __device__ __forceinline__ void store_e4m3(uint8_t* row, int unit, int d, float inv) const {
        auto q = [inv](float v) { return clamp448(__fmul_rn(v, inv)); };
        uint32_t w[4];
        if (HALVES) {
            w[0] = f32x4_to_e4m3x4(q(a[0]), q(a[1]), q(a[2]), q(a[3]));
            w[1] = f32x4_to_e4m3x4(q(a[4]), q(a[5]), q(a[6]), q(a[7]));
            w[2] = f32x4_to_e4m3x4(q(b[0]), q(b[1]), q(b[2]), q(b[3]));
            w[3] = f32x4_to_e4m3x4(q(b[4]), q(b[5]), q(b[6]), q(b[7]));
            st_global_v2(row + unit * 8, make_uint2(w[0], w[1]));
            st_global_v2(row + d / 2 + unit * 8, make_uint2(w[2], w[3]));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = f32x4_to_e4m3x4(q(a[2 * i]), q(b[2 * i]), q(a[2 * i + 1]), q(b[2 * i + 1]));
            st_global_v4(row + unit * 16, make_uint4(w[0], w[1], w[2], w[3]));
        }
    }
};

__device__ __forceinline__ float2 e4m3x2_to_f32x2(uint32_t two) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

constexpr int APPEND_THREADS = 256;

template <int GROUP, bool HALVES>
__global__ void __launch_bounds__(APPEND_THREADS, GROUP == 32 ? 2 : 4)
paged_append_kernel(PagedAppendParams p) {
    __shared__ float part[APPEND_THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int units = p.d >> 4;                              // 16-value pieces of a head
    if (blockIdx.x >= p.kv_blocks) {
        // ---------------- queries: (token, group of heads, piece)
        const long long n = (long long)(blockIdx.x - p.kv_blocks) * APPEND_THREADS + threadIdx.x;
        const int hgroups = (p.hq + p.q_heads - 1) / p.q_heads, per_token = hgroups * units;
        const long long t = n / per_token;
        if (t >= p.tokens) return;
        const int rest = (int)(n - t * per_token), h0 = rest / units * p.q_heads, unit = rest % units;
        const TokenPlace at = place_of(p.cu, p.lens, p.batch, p.tokens, (int)t);
        if (at.pos < 0 || (p.rope && at.pos >= p.rope_rows)) return;
        const __nv_bfloat16* row = p.qkv + t * p.qkv_stride;
        float4 angle[4];
        Sixteen<HALVES> x[2];
        if (p.rope) x[0].load_angles(p.rope + (size_t)at.pos * p.d, unit, angle);
        const int h1 = min(h0 + p.q_heads, p.hq);
        for (int hh = h0; hh < h1; hh += 2) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (hh + i < h1) x[i].load(row + (size_t)(hh + i) * p.d, unit, p.d);
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (hh + i < h1) {
                    if (p.rope) x[i].template turn<false>(angle);
                    x[i].store_bf16(p.q + ((size_t)t * p.hq + hh + i) * p.d, unit, p.d);
                }
        }
        return;
    }
    // ---------------- keys and values: the blocks whose first new token is in this group's chunk
    constexpr int GROUPS = APPEND_THREADS / GROUP;
    const unsigned item = blockIdx.x * GROUPS + threadIdx.x / GROUP;
    if (item >= p.kv_items) return;                          // whole groups: 256 threads are one group and never leave here alone
    const int me = threadIdx.x % GROUP;
    const int h2 = (int)(item % (2 * p.hkv)), chunk = (int)(item / (2 * p.hkv));
    const bool is_k = h2 < p.hkv;
    const int h = is_k ? h2 : h2 - p.hkv;
    uint8_t* cache = is_k ? p.k : p.v;
    float* scales = is_k ? p.k_scale : p.v_scale;
    const bool rotate = is_k && p.rope;
    const __nv_bfloat16* src = p.qkv + (size_t)(p.hq + h2) * p.d;
    const int bs = p.block_size, t_end = (int)min((long long)(chunk + 1) * p.chunk, (long long)p.tokens);
    int t = chunk * p.chunk;
    while (t < t_end) {
        const TokenPlace at = place_of(p.cu, p.lens, p.batch, p.tokens, t);
        if (t < at.start) { t = at.start; continue; }        // in front of the first sequence
        if (at.pos < 0) {                                    // behind the sequences, or before the first position of one
            const int first = at.end - (p.cu && at.seq < p.batch ? p.lens[at.seq] : 0);   // token at position 0
            t = first > t && first < at.end ? first : max(at.end, t + 1);
            continue;
        }
        const int slot = at.pos & (bs - 1);
        const int next = min(at.end, t + bs - slot);         // first token of another block
        if (t != at.start && slot != 0) { t = next; continue; }      // the group of an earlier chunk has this block
        const int j = at.pos / bs;
        const int page = j < p.table_stride ? p.table[(size_t)at.seq * p.table_stride + j] : -1;
        int rows = next - t;
        if (p.rope) rows = min(rows, p.rope_rows - at.pos);
        const int t_first = t;
        t = next;
        if (page < 0 || page >= p.num_blocks || rows <= 0) continue;
        const size_t block = (size_t)page * p.hkv + h;
        const float s_old = slot > 0 ? scales[block] : 0.0f;
        auto value = [&](Sixteen<HALVES>& x, int i) {
            const int r = i / units, unit = i - r * units;
            x.load(src + (size_t)(t_first + r) * p.qkv_stride, unit, p.d);
            if (rotate) {
                float4 angle[4];
                x.load_angles(p.rope + (size_t)(at.pos + r) * p.d, unit, angle);
                x.template turn<true>(angle);
            }
        };
        // up to two pieces a thread stay in registers between the maximum and the codes; the others are read again
        Sixteen<HALVES> keep[2];
        float top = 0.0f;
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (me + k * GROUP < rows * units) {
                value(keep[k], me + k * GROUP);
                top = fmaxf(top, keep[k].largest());
            }
        for (int i = me + 2 * GROUP; i < rows * units; i += GROUP) {
            Sixteen<HALVES> x;
            value(x, i);
            top = fmaxf(top, x.largest());
        }
        top = warp_max_butterfly(top);
        if (GROUP > 32) {
            if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < APPEND_THREADS / 32; ++w) top = fmaxf(top, part[w]);
        }
        // every thread of the group has read the old scale (and `part`) before it changes
        if (GROUP > 32) __syncthreads();
        else __syncwarp();
        const float s = fmaxf(fmaxf(s_old, __fdiv_rn(top, 448.0f)), 1e-12f), inv = __fdiv_rn(1.0f, s);
        uint8_t* base = cache + block * bs * p.d;
        if (me == 0) scales[block] = s;
        if (slot > 0 && s != s_old) {
            const float ratio = __fdiv_rn(s_old, s);
            for (int i = me; i < slot * units; i += GROUP) {
                uint4 w = ld_global_v4(base + (size_t)i * 16);
                uint32_t* ww = &w.x;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 lo = e4m3x2_to_f32x2(ww[k] & 0xffffu), hi = e4m3x2_to_f32x2(ww[k] >> 16);
                    ww[k] = f32x4_to_e4m3x4(clamp448(__fmul_rn(lo.x, ratio)), clamp448(__fmul_rn(lo.y, ratio)),
                                            clamp448(__fmul_rn(hi.x, ratio)), clamp448(__fmul_rn(hi.y, ratio)));
                }
                st_global_v4(base + (size_t)i * 16, w);
            }
        }
        auto code = [&](const Sixteen<HALVES>& x, int i) {
            const int r = i / units, unit = i - r * units;
            x.store_e4m3(base + (size_t)(slot + r) * p.d, unit, p.d, inv);
        };
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (me + k * GROUP < rows * units) code(keep[k], me + k * GROUP);
        for (int i = me + 2 * GROUP; i < rows * units; i += GROUP) {
            Sixteen<HALVES> x;
            value(x, i);
            code(x, i);
        }
    }
}

template <int GROUP, bool HALVES>
static int launch_append(PagedAppendParams p, cudaStream_t stream) {
    const long long chunks = (p.tokens + (long long)p.chunk - 1) / p.chunk, items = chunks * 2 * p.hkv;
    const long long kv_blocks = (items * GROUP + APPEND_THREADS - 1) / APPEND_THREADS;
    const long long q_items = p.q ? (long long)p.tokens * ((p.hq + p.q_heads - 1) / p.q_heads) * (p.d / 16) : 0;
    const long long blocks = kv_blocks + (q_items + APPEND_THREADS - 1) / APPEND_THREADS;
    if (blocks > 0x7fffffffLL || items > 0xffffffffLL) return FRT_ERR_UNSUPPORTED;
    p.kv_items = (unsigned)items;
    p.kv_blocks = (unsigned)kv_blocks;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(APPEND_THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_append_kernel<GROUP, HALVES>, p);
    return e == cudaSuccess ? FRT_OK : FRT_CUDA_ERR(e);
}

}  // namespace frt

extern "C" int frt_b200_paged_kv_append_fp8(const void* qkv, long long qkv_stride, const float* rope, int rope_rows, void* Q,
                                            void* k_cache, void* v_cache, float* k_scale, float* v_scale,
                                            const int* block_table, int table_stride, const int* cu_seqlens,
                                            const int* seq_lens, int tokens, int batch, int num_blocks, int block_size,
                                            int num_heads_q, int num_heads_kv, int head_dim, int flags, void* stream) {
    using namespace frt;
    auto off = [](const void* a, uintptr_t n) { return (reinterpret_cast<uintptr_t>(a) & (n - 1)) != 0; };
    if (tokens < 0 || batch < 0 || num_blocks < 0 || table_stride < 0 || num_heads_q < 1 || num_heads_kv < 1 || rope_rows < 0)
        return FRT_ERR_INVALID;
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return FRT_ERR_UNSUPPORTED;
    if (block_size < 16 || block_size > 128 || (block_size & (block_size - 1))) return FRT_ERR_UNSUPPORTED;
    if (num_heads_q > 1024 || num_heads_kv > 1024) return FRT_ERR_UNSUPPORTED;
    const long long width = (long long)(num_heads_q + 2 * num_heads_kv) * head_dim;
    if (qkv_stride < width || qkv_stride % 8) return FRT_ERR_INVALID;
    if (!cu_seqlens && tokens != batch) return FRT_ERR_INVALID;
    if (tokens == 0 || batch == 0) return FRT_OK;
    if (!qkv || !k_cache || !v_cache || !k_scale || !v_scale || !block_table || !seq_lens) return FRT_ERR_INVALID;
    if (off(qkv, 16) || off(rope, 16) || off(Q, 16) || off(k_cache, 16) || off(v_cache, 16) || off(k_scale, 4) || off(v_scale, 4) ||
        off(block_table, 4) || off(cu_seqlens, 4) || off(seq_lens, 4))
        return FRT_ERR_INVALID;
    PagedAppendParams p = {static_cast<const __nv_bfloat16*>(qkv), qkv_stride, rope, rope_rows, static_cast<__nv_bfloat16*>(Q),
                           static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(v_cache), k_scale, v_scale, block_table, cu_seqlens,
                           seq_lens, table_stride, tokens, batch, num_blocks, block_size, num_heads_q, num_heads_kv, head_dim, 1, 2, 0, 0};
    // chunk: about a sequence's tokens, at most a block, so that a group finds one leader or so; a power of two
    const int mean = tokens / batch;
    while (p.chunk * 2 <= mean && p.chunk < block_size) p.chunk *= 2;
    // 96 decoding tokens 3.8 us with two heads a thread, 4.4 with four, 5.8 with eight; 7700 of prompts 53, 51 and 51
    p.q_heads = (long long)tokens * num_heads_q * head_dim > 1 << 22 ? 8 : 2;
    const bool halves = flags & 2, warp = p.chunk * (head_dim / 16) <= 64;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (warp) return halves ? launch_append<32, true>(p, st) : launch_append<32, false>(p, st);
    return halves ? launch_append<APPEND_THREADS, true>(p, st) : launch_append<APPEND_THREADS, false>(p, st);
}

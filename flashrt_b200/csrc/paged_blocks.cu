// Blocks of the paged cache between two steps: what dropped tokens held goes back to the free list, the next tokens get theirs; block table,
// packed offsets, positions and slots on the device, so that a captured graph serves steps whose lengths the host does not know.
//
// Stands beside paged_kv_append_fp8 and paged_attention_fp8, which read these arrays; no counterpart in the reference.
//
// Nothing here moves much: a batch's lengths are a few KB, a table's new entries and the slots of a step about as much, so what counts is
// the number of launches and of dependent loads.  Every CTA scans the whole batch by itself (a thread has a run of sequences, sums that
// stop at 2^31 - 1 stay associative) and finds its own tokens' and blocks' sequences by bisection in shared memory: one launch, no
// order between CTAs, no atomics.
#include "common.cuh"
#include "tc05.cuh"
#include "flashrt_b200.h"

namespace frt {
namespace blk {

constexpr int PLAN_THREADS = 256, RELEASE_THREADS = 1024, MAX_BATCH = 8192;

__device__ __forceinline__ int sat_add(int a, int b) { return (int)min((unsigned)a + (unsigned)b, 0x7fffffffu); }    // both >= 0

// exclusive scan over the block's threads of two counts, sums stop at 2^31 - 1; `part`: 2 * warps ints
template <int THREADS>
__device__ __forceinline__ void block_scan2(int& a, int& b, int* part, int& all_a, int& all_b) {
    constexpr int WARPS = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = a, y = b;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, x, d), v = __shfl_up_sync(0xffffffffu, y, d);
        if (lane >= d) { x = sat_add(x, u); y = sat_add(y, v); }
    }
    if (lane == 31) { part[warp] = x; part[WARPS + warp] = y; }
    __syncthreads();
    int fa = 0, fb = 0, ta = 0, tb = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w == warp) { fa = ta; fb = tb; }
        ta = sat_add(ta, part[w]);
        tb = sat_add(tb, part[WARPS + w]);
    }
    const int px = __shfl_up_sync(0xffffffffu, x, 1), py = __shfl_up_sync(0xffffffffu, y, 1);
    a = sat_add(fa, lane ? px : 0);
    b = sat_add(fb, lane ? py : 0);
    all_a = ta;
    all_b = tb;
    __syncthreads();
}
// largest i in [0, n) with start[i] <= t (start ascending, start[0] <= t)
__device__ __forceinline__ int last_not_above(const int* start, int n, int t) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
}
__device__ __forceinline__ int blocks_of(int tokens, int shift) { return tokens > 0 ? (int)(((unsigned)tokens + ((1u << shift) - 1)) >> shift) : 0; }

struct PlanParams {
    const int *kept, *fresh;     // tokens that stay, tokens to come (batch)
    int* table;                  // (batch, table_stride)
    const int *free_list, *free_in;
    int *free_out, *cu, *lens, *positions;
    long long* slots;
    int* refused;
    int table_stride, tokens, batch, num_blocks, shift;
};

__global__ void __launch_bounds__(PLAN_THREADS)
paged_plan_kernel(PlanParams p) {
    extern __shared__ int start[];                           // (batch + 1) first token, (batch + 1) first new block of each sequence, tokens it keeps
    __shared__ int part[2 * PLAN_THREADS / 32];
    int *first = start + p.batch + 1, *stay = first + p.batch + 1;
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, per = (p.batch + PLAN_THREADS - 1) / PLAN_THREADS;
    const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
    const int room = min(max(*p.free_in, 0), p.num_blocks);
    // what a sequence asks for: nothing where its lengths are none or its table is too short
    auto asks = [&](int b, int& tokens, int& blocks) {
        const int k = p.kept[b], n = p.fresh[b];
        const long long all = (long long)k + n;
        const bool fits = k >= 0 && n >= 0 && all <= 0x7fffffffLL && blocks_of((int)all, p.shift) <= p.table_stride;
        tokens = fits ? n : 0;
        blocks = fits ? blocks_of((int)all, p.shift) - blocks_of(k, p.shift) : 0;
        return fits;
    };
    int t = 0, k = 0, all_t, all_k;
    for (int b = b0; b < b1; ++b) {
        int n, m;
        asks(b, n, m);
        t = sat_add(t, n);
        k = sat_add(k, m);
    }
    block_scan2<PLAN_THREADS>(t, k, part, all_t, all_k);
    // served: all in front and this one fit.  Sums grow along the batch, so the served ones are its beginning.
    int last_t = 0, last_k = 0, refused = 0;                 // of this thread's last served one
    for (int b = b0; b < b1; ++b) {
        int n, m;
        const bool fits = asks(b, n, m);
        start[b] = t;
        first[b] = k;
        t = sat_add(t, n);
        k = sat_add(k, m);
        const bool served = t <= p.tokens && k <= room;
        if (served) { last_t = t; last_k = k; }
        refused += !(fits && served);
        stay[b] = p.kept[b];
        if (blockIdx.x == 0) p.lens[b] = fits && served ? stay[b] + n : max(stay[b], 0);
    }
    const int total_t = __reduce_max_sync(0xffffffffu, last_t), total_k = __reduce_max_sync(0xffffffffu, last_k);
    const int warp_refused = __reduce_add_sync(0xffffffffu, refused);
    __shared__ int tops[3][PLAN_THREADS / 32];
    if ((tid & 31) == 0) {
        tops[0][tid >> 5] = total_t;
        tops[1][tid >> 5] = total_k;
        tops[2][tid >> 5] = warp_refused;
    }
    __syncthreads();
    int tokens = 0, blocks = 0, missing = 0;
#pragma unroll
    for (int w = 0; w < PLAN_THREADS / 32; ++w) {
        tokens = max(tokens, tops[0][w]);
        blocks = max(blocks, tops[1][w]);
        missing += tops[2][w];
    }
    // behind the served ones everything starts at the end
    for (int b = b0; b < b1; ++b) {
        start[b] = min(start[b], tokens);
        first[b] = min(first[b], blocks);
        if (blockIdx.x == 0) p.cu[b] = start[b];
    }
    if (tid == 0) {
        start[p.batch] = tokens;
        first[p.batch] = blocks;
        if (blockIdx.x == 0) {
            p.cu[p.batch] = tokens;
            *p.free_out = room - blocks;
            if (p.refused) *p.refused = missing;
        }
    }
    __syncthreads();
    const int gsize = gridDim.x * PLAN_THREADS, gid = blockIdx.x * PLAN_THREADS + tid;
    for (int i = gid; i < blocks; i += gsize) {
        const int b = last_not_above(first, p.batch, i);
        p.table[(size_t)b * p.table_stride + blocks_of(stay[b], p.shift) + (i - first[b])] = p.free_list[room - 1 - i];
    }
    if (!p.positions && !p.slots) return;
    for (long long i = gid; i < p.tokens; i += gsize) {
        int pos = -1;
        long long slot = -1;
        if (i < tokens) {
            const int b = last_not_above(start, p.batch, (int)i), have = blocks_of(stay[b], p.shift);
            pos = stay[b] + ((int)i - start[b]);
            const int j = pos >> p.shift;
            const int page = j < have ? p.table[(size_t)b * p.table_stride + j] : p.free_list[room - 1 - (first[b] + j - have)];
            if (page >= 0 && page < p.num_blocks) slot = ((long long)page << p.shift) + (pos & ((1 << p.shift) - 1));
        }
        if (p.positions) p.positions[i] = pos;
        if (p.slots) p.slots[i] = slot;
    }
}

struct ReleaseParams {
    const int *kept, *lens;
    int *table, *free_list;
    const int* free_in;
    int* free_out;
    int table_stride, batch, num_blocks, shift;
};

// One CTA, or one cluster of eight where tables are large.  The entries to drop, sequence by sequence, are one row of items; a CTA has a
// run of them, counts the blocks of the pool among them, and writes them from the end of the list's new part backwards, so that a plan
// that takes as many finds them in the order in which they were.
__global__ void __launch_bounds__(RELEASE_THREADS)
paged_release_kernel(ReleaseParams p) {
    extern __shared__ int first[];                           // first item of each sequence; blocks that it keeps
    __shared__ int part[2 * RELEASE_THREADS / 32];
    __shared__ int mine;
    int* stay = first + p.batch;
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, per = (p.batch + RELEASE_THREADS - 1) / RELEASE_THREADS;
    const int ctas = (int)gridDim.x, rank = (int)blockIdx.x;
    const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
    const int room = min(max(*p.free_in, 0), p.num_blocks);
    auto drops = [&](int b, int& from) {
        from = blocks_of(p.kept[b], p.shift);
        return max(min(blocks_of(p.lens[b], p.shift), p.table_stride) - from, 0);
    };
    int at = 0, zero = 0, items, none, from;
    for (int b = b0; b < b1; ++b) at = sat_add(at, drops(b, from));
    block_scan2<RELEASE_THREADS>(at, zero, part, items, none);
    for (int b = b0; b < b1; ++b) {
        first[b] = at;
        at = sat_add(at, drops(b, from));
        stay[b] = from;
    }
    __syncthreads();
    auto entry = [&](int i) {
        const int b = last_not_above(first, p.batch, i);
        return p.table + (size_t)b * p.table_stride + stay[b] + (i - first[b]);
    };
    // few items (the tables are large, but a step drops little): the first CTA's alone, and nobody waits for a count
    const bool alone = items <= RELEASE_THREADS;
    if (alone && rank > 0) return;
    const int i0 = alone ? 0 : (int)((long long)items * rank / ctas), i1 = alone ? items : (int)((long long)items * (rank + 1) / ctas);
    int before = 0, total = 0;                               // blocks of the pool in front of this CTA's items, and in all
    if (!alone) {
        int n = 0, unused = 0, all, none2;
        for (int i = i0 + tid; i < i1; i += RELEASE_THREADS) n += (unsigned)*entry(i) < (unsigned)p.num_blocks;
        block_scan2<RELEASE_THREADS>(n, unused, part, all, none2);
        if (ctas > 1) {
            if (tid == 0) mine = all;
            __syncwarp();
            tc::cluster_sync_all();
            for (int r = 0; r < ctas; ++r) {
                const int n_r = __float_as_int(tc::dsmem_ld_f32(tc::dsmem_map(tc::smem_u32(&mine), (uint32_t)r)));
                if (r < rank) before += n_r;
                total += n_r;
            }
            __syncwarp();
            tc::cluster_sync_all();                          // nobody leaves while its count is read
        } else {
            total = all;
        }
    }
    for (int base = i0; base < i1 || (alone && base == i0); base += RELEASE_THREADS) {
        const int i = base + tid;
        int* e = i < i1 ? entry(i) : nullptr;
        const int page = e ? *e : -1;
        int n = (unsigned)page < (unsigned)p.num_blocks, unused = 0, all, none2;
        const bool valid = n;
        block_scan2<RELEASE_THREADS>(n, unused, part, all, none2);
        if (alone) total = all;
        if (valid) {
            const int to = room + total - 1 - (before + n);
            if (to >= 0 && to < p.num_blocks) p.free_list[to] = page;
            *e = -1;
        }
        before += all;
    }
    if (rank == 0 && tid == 0) *p.free_out = min(room + total, p.num_blocks);
}

constexpr int PLAN_SMEM = 3 * (MAX_BATCH + 1) * 4;

static int launch_plan(const PlanParams& p, cudaStream_t stream) {
    static PerDeviceOnce once;
    int dev = 0;
    if (once.need(dev)) {
        const cudaError_t e = cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PLAN_SMEM);
        if (e != cudaSuccess) return FRT_CUDA_ERR(e);
        once.set(dev);
    }
    // two tokens a thread and more: the scan of the batch is the same in every CTA
    const long long want = ((long long)(p.tokens > p.batch ? p.tokens : p.batch) + 2 * PLAN_THREADS - 1) / (2 * PLAN_THREADS);
    const int most = device_sm_count();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(want < 1 ? 1 : want < most ? want : most));
    cfg.blockDim = dim3(PLAN_THREADS);
    cfg.dynamicSmemBytes = 3 * (size_t)(p.batch + 1) * 4;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_plan_kernel, p);
    return e == cudaSuccess ? FRT_OK : FRT_CUDA_ERR(e);
}

static int launch_release(const ReleaseParams& p, cudaStream_t stream) {
    static PerDeviceOnce once;
    int dev = 0;
    if (once.need(dev)) {
        const cudaError_t e = cudaFuncSetAttribute(paged_release_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PLAN_SMEM);
        if (e != cudaSuccess) return FRT_CUDA_ERR(e);
        once.set(dev);
    }
    cudaLaunchConfig_t cfg = {};
    const unsigned ctas = (long long)p.batch * p.table_stride > 16 * RELEASE_THREADS ? 8 : 1;
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(RELEASE_THREADS);
    cfg.dynamicSmemBytes = 2 * (size_t)p.batch * 4;
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
    const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_release_kernel, p);
    return e == cudaSuccess ? FRT_OK : FRT_CUDA_ERR(e);
}

// sums of the batch stay below 2^31 - 1, where they stop
static bool too_large(int tokens, int batch, int num_blocks, int table_stride, int block_size) {
    return block_size < 16 || block_size > 128 || (block_size & (block_size - 1)) || batch > MAX_BATCH || tokens > 1 << 30 ||
           num_blocks > 1 << 30 || (long long)batch * table_stride > 1 << 30;
}
static int shift_of(int block_size) {
    int s = 0;
    while ((1 << s) < block_size) ++s;
    return s;
}

}  // namespace blk
}  // namespace frt

static bool misaligned(const void* a, uintptr_t n) { return (reinterpret_cast<uintptr_t>(a) & (n - 1)) != 0; }

extern "C" int frt_b200_paged_plan(const int* kept_lens, const int* new_lens, int* block_table, int table_stride, const int* free_list,
                                   const int* free_in, int* free_out, int* cu_seqlens, int* seq_lens, int* positions,
                                   long long* slots, int* refused, int tokens, int batch, int num_blocks, int block_size, int flags,
                                   void* stream) {
    using namespace frt;
    (void)flags;
    if (tokens < 0 || batch < 0 || num_blocks < 0 || table_stride < 0) return FRT_ERR_INVALID;
    if (blk::too_large(tokens, batch, num_blocks, table_stride, block_size)) return FRT_ERR_UNSUPPORTED;
    if (!free_in || !free_out || !cu_seqlens || (!free_list && num_blocks)) return FRT_ERR_INVALID;
    if (batch && (!kept_lens || !new_lens || !seq_lens || (!block_table && table_stride))) return FRT_ERR_INVALID;
    auto meet = [&](const int* a) { return a < seq_lens + batch && seq_lens < a + batch; };
    if (free_in == free_out || (batch && (meet(kept_lens) || meet(new_lens)))) return FRT_ERR_INVALID;      // read while they are written
    if (misaligned(kept_lens, 4) || misaligned(new_lens, 4) || misaligned(block_table, 4) || misaligned(free_list, 4) || misaligned(free_in, 4) ||
        misaligned(free_out, 4) || misaligned(cu_seqlens, 4) || misaligned(seq_lens, 4) || misaligned(positions, 4) || misaligned(slots, 8) ||
        misaligned(refused, 4))
        return FRT_ERR_INVALID;
    const blk::PlanParams p = {kept_lens, new_lens, block_table, free_list, free_in, free_out, cu_seqlens, seq_lens, positions, slots, refused,
                               table_stride, tokens, batch, num_blocks, blk::shift_of(block_size)};
    return blk::launch_plan(p, static_cast<cudaStream_t>(stream));
}

extern "C" int frt_b200_paged_release(const int* kept_lens, const int* seq_lens, int* block_table, int table_stride, int* free_list,
                                      const int* free_in, int* free_out, int batch, int num_blocks, int block_size, int flags,
                                      void* stream) {
    using namespace frt;
    (void)flags;
    if (batch < 0 || num_blocks < 0 || table_stride < 0) return FRT_ERR_INVALID;
    if (blk::too_large(0, batch, num_blocks, table_stride, block_size)) return FRT_ERR_UNSUPPORTED;
    if (!free_in || !free_out || (!free_list && num_blocks) || free_in == free_out) return FRT_ERR_INVALID;
    if (batch && (!kept_lens || !seq_lens || (!block_table && table_stride))) return FRT_ERR_INVALID;
    if (misaligned(kept_lens, 4) || misaligned(seq_lens, 4) || misaligned(block_table, 4) || misaligned(free_list, 4) || misaligned(free_in, 4) ||
        misaligned(free_out, 4))
        return FRT_ERR_INVALID;
    const blk::ReleaseParams p = {kept_lens, seq_lens, block_table, free_list, free_in, free_out, table_stride, batch, num_blocks, blk::shift_of(block_size)};
    return blk::launch_release(p, static_cast<cudaStream_t>(stream));
}

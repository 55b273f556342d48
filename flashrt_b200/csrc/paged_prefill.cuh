#pragma once

// Many query rows over the paged E4M3 cache: chunks of prompts.  Included by paged_attention.cu inside namespace frt.
//
// Same formulas as the kernel for few rows.  128 query rows (tokens x the group's heads) are the lanes of a tcgen05 tile; two tiles share
// every converted tile of keys and values.
//   S = Q . K^T    kind::f16, queries and codes as fp16 (both exact, see the top of paged_attention.cu) in shared memory
//   O += P . V     P fp16 from tensor memory, written over S
// The block's scales stay out of the operands: a column of S has the factor softmax_scale * log2(e) * ks of its 16 keys and the addend
// log2(vs), which replace the one factor that a softmax has anyway; the sum takes 1 / vs per 16 keys.
// Every row tile has two S: the next scores are issued in front of this tile's P . V and stand when the softmax is through.  O is rescaled
// only when a row's maximum grows by more than 2^8: weights are 2^(u - m + 7) with the stale m, at most 2^15.
// Warps: 0-3 and 4-7 softmax (thread = row), 8-11 turn E4M3 bytes into swizzled fp16 operands, 12 and 14 issue a row tile's MMAs, 13 the copies.
// Heads of 256 (an O of 256 columns) and calls of at most 128 rows have one tile.
// Two row tiles with heads of 128 need 4 x 128 x 64 x 128 products for a tile of 64 keys, 1024 clocks of the tensor pipe, and
// 2 x 128 x 64 exponentials at 16 a clock, 1024 as well; a tile takes some 2400.
// Bound by: neither unit alone, each is active for 44 % of the time.  A row tile's softmax, a chain of dependent steps of one thread a row,
// hides behind the other's products only in part; and items are whole: of 472 on 148 SMs the last SM ends after 364 key tiles where the mean is
// 316 (longest first: 366).
// Measured: two chunks of up to 2048 tokens on up to 8191 keys, 32 query and 8 key heads of 128, 468 us, 0.83 PFLOP/s.
template <int D, int T>
struct PrefillCfg {
    static_assert(T == 1 || D <= 128, "tensor memory: two tiles of S and O");
    static constexpr int BKV = T == 2 || D == 256 ? 64 : 128;      // keys of a tile: two S a row tile beside its O
    static constexpr int GR = BKV / 16;                   // groups of 16 keys: one block each
    static constexpr int Q_BYTES = 128 * D * 2, KV_BYTES = BKV * D * 2, RAW_BYTES = BKV * D;
    // Keys and values alternate in both rings (operand 2 i: the keys of tile i, 2 i + 1: its values): slots of bytes, so that copies run
    // ahead, and of fp16 operands.
    static constexpr int RAWS = BKV == 64 && D <= 128 ? 6 : 4, OPS = BKV == 64 && D <= 128 ? 6 : 3;
    static constexpr int OFF_OP = T * Q_BYTES, OFF_RAW = OFF_OP + OPS * KV_BYTES;
    static constexpr int SMEM_BYTES = OFF_RAW + RAWS * RAW_BYTES + 1024;
    static_assert(SMEM_BYTES <= 232448 - (D == 256 ? 2 : 3) * 1024, "dynamic and static shared memory of a CTA");
    static constexpr int O_COL = T * 2 * BKV;             // accumulators behind the S
    static_assert(O_COL + T * D <= 512, "tensor memory");
    static constexpr int THREADS = 512;
    // registers of a thread: 128 at launch (8 x 192 + 4 x 80 + 4 x 48 = 16 x 128)
    static constexpr int REGS_SOFTMAX = 192, REGS_CONVERT = 80, REGS_ISSUE = 48;
    static constexpr int RING = 16;                       // scales of tiles; copies run at most RAWS / 2 + OPS / 2 + 2 tiles ahead of the softmax
    static constexpr float OFFSET = 7.0f, GROWTH = 8.0f;
};

struct PrefillParams {
    PagedAttnParams a;
    int splits;                  // along the keys, at most: an item's pieces have two tiles or more; paged_join_kernel joins them
    int tiles;                   // row tiles of all sequences, at most: items of one head
    int4* items;                 // [item] first token, first row, rows, pieces
    float* part_o;               // [item][split][tile][D][128]
    float2* part_ml;             // [item][split][tile][128]
};

template <int D, int T>
__global__ void __launch_bounds__(512, 1)
paged_prefill_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const PrefillParams pp) {
    using Cfg = PrefillCfg<D, T>;
    constexpr int BKV = Cfg::BKV, GR = Cfg::GR;
    constexpr float LOG2E = 1.4426950408889634f;
    const PagedAttnParams& p = pp.a;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t raw_full[Cfg::RAWS], raw_empty[Cfg::RAWS], op_full[Cfg::OPS], op_empty[Cfg::OPS], s_full[2 * T], p_half[2 * T], p_ready[2 * T], q_full, o_done[T];
    __shared__ float4 scale_s[Cfg::RING][GR];               // per 16 keys: ks, log2 vs, 1 / vs
    __shared__ float rf_s[T * 128];
    __shared__ int warp_s[16], item_s[2];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_s;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < Cfg::RAWS; ++i) {
            tc::mbar_init(&raw_full[i], 2);                 // bytes; scales
            tc::mbar_init(&raw_empty[i], 4);
        }
        for (int i = 0; i < Cfg::OPS; ++i) {
            tc::mbar_init(&op_full[i], 4);
            tc::mbar_init(&op_empty[i], T);
        }
        for (int i = 0; i < 2 * T; ++i) {
            tc::mbar_init(&s_full[i], 1);
            tc::mbar_init(&p_half[i], 128);
            tc::mbar_init(&p_ready[i], 128);
        }
        tc::mbar_init(&q_full, 128 * T);
        for (int i = 0; i < T; ++i) tc::mbar_init(&o_done[i], 1);
        abort_s = 0;
        tc::mbar_fence_init();
        tc::tma_prefetch_desc(&tmK);
        tc::tma_prefetch_desc(&tmV);
    }
    if (warp == 12) {
        tc::tmem_alloc(&tmem_slot, 512);
        tc::tmem_relinquish();
    }
    const uint64_t deadline = tc::global_timer_ns() + FRT_KERNEL_DEADLINE_NS;
    pdl_launch_dependents();
    pdl_wait();

    // ---------------- this CTA's item: tiles of the sequences with more than few_rows rows, a sequence's last (most keys) first
    const int per = (p.batch + 511) / 512;
    auto tiles_of = [&](int b) {
        const int start = p.cu ? min(max(p.cu[b], 0), p.tokens) : b, end = p.cu ? min(max(p.cu[b + 1], start), p.tokens) : b + 1;
        const long long rows = (long long)(end - start) * p.group;
        return rows > p.few_rows ? (int)((rows + 128 * T - 1) / (128 * T)) : 0;
    };
    int mine = 0;
    for (int b = tid * per; b < min((tid + 1) * per, p.batch); ++b) mine += tiles_of(b);
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += o;
    }
    if (lane == 31) warp_s[warp] = incl;
    if (tid == 0) item_s[0] = -1;
    tc::tc_fence_before_sync();
    __syncthreads();
    tc::tc_fence_after_sync();
    int first = incl - mine;
    for (int w = 0; w < warp; ++w) first += warp_s[w];
    const int want = (int)blockIdx.x;
    if (mine > 0 && first <= want && want < first + mine) {
        int b = tid * per;
        for (;; ++b) {
            const int n = tiles_of(b);
            if (want < first + n) {
                item_s[1] = n - 1 - (want - first);
                break;
            }
            first += n;
        }
        item_s[0] = b;
    }
    __syncthreads();
    const int b = item_s[0], item = (int)(blockIdx.y * gridDim.x + blockIdx.x);
    const uint32_t tmem = tmem_slot;
    if (b < 0) {                                            // fewer items than the grid's bound
        if (pp.splits > 1 && blockIdx.z == 0 && tid == 0) pp.items[item] = make_int4(0, 0, 0, 0);
        if (warp == 12) tc::tmem_dealloc(tmem, 512);
        return;
    }
    const int start = p.cu ? min(max(p.cu[b], 0), p.tokens) : b, stop = p.cu ? min(max(p.cu[b + 1], start), p.tokens) : b + 1;
    const int n_new = stop - start, h = (int)blockIdx.y, row0 = item_s[1] * (128 * T);
    const int rows = (int)min((long long)128 * T, (long long)n_new * p.group - row0);
    const int len = min(max(p.lens[b], 0), 0x7fffff00);
    const int p0 = len - n_new + row0 / p.group, p1 = len - n_new + (row0 + rows - 1) / p.group;
    const int key_lo = window_from(p, p0);
    const int key_hi = min(p.causal ? p1 + 1 : len, p.room);
    const int jl = key_lo / BKV, jn = max(key_hi > 0 ? (key_hi + BKV - 1) / BKV - jl : 0, 0);
    const int split = (int)blockIdx.z, pieces = max(min(pp.splits, (jn + 1) / 2), 1);
    if (pp.splits > 1 && split == 0 && tid == 0) pp.items[item] = make_int4(start, row0, rows, pieces);
    if (split >= pieces) {
        if (warp == 12) tc::tmem_dealloc(tmem, 512);
        return;
    }
    const int j0 = jl + (int)((long long)jn * split / pieces), j1 = jl + (int)((long long)jn * (split + 1) / pieces);
    const int nt = j1 - j0;
    const int* table = p.table + (size_t)b * p.table_stride;
    const uint32_t sm = tc::smem_u32(smem);
    auto gave_up = [&](int code) {
        if (!abort_s && lane == 0) atomicCAS(p.status, 0, code | (blockIdx.x << 8));
        abort_s = 1;
    };

    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::REGS_ISSUE));
        if (warp == 12 || (T == 2 && warp == 14)) {
            // ---------------- MMA issuer of a row tile (whole warp).  One warp for both tiles took some 80 clocks an MMA, 2900 of a pair's 4220
            // for a tile of keys, and made each tile wait for the other's turn.
            constexpr uint32_t idesc_s = tc::make_idesc(0, 0, 0, 0, 128, BKV);      // fp16, both K-major
            constexpr uint32_t idesc_o = tc::make_idesc(0, 0, 0, 1, 128, D);        // P from tensor memory, V MN-major
            const int t = (warp - 12) >> 1;
            const uint64_t dq = tc::make_desc_kmajor_sw128(sm + t * Cfg::Q_BYTES), dk0 = tc::make_desc_kmajor_sw128(sm + Cfg::OFF_OP);
            const uint64_t dv0 = tc::make_desc_mnmajor_sw128(sm + Cfg::OFF_OP, BKV * 128);
            const uint32_t tmem_o = tmem + Cfg::O_COL + t * D;
            auto buf = [&](int i) { return 2 * t + (i & 1); };              // S and its barriers: two in turn
            auto par = [&](int i) { return (uint32_t)((i >> 1) & 1); };
            auto qk = [&](int i) {
                const uint64_t dk = dk0 + (uint64_t)((2 * i % Cfg::OPS) * (Cfg::KV_BYTES >> 4));
                const uint32_t tmem_s = tmem + buf(i) * BKV;
                if (tc::elect_one()) {
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)        // 64-element blocks, 32 bytes per step inside
                        tc::mma_f16(tmem_s, dq + (uint64_t)((k / 4) * ((128 * 128) >> 4) + 2 * (k % 4)),
                                    dk + (uint64_t)((k / 4) * ((BKV * 128) >> 4) + 2 * (k % 4)), idesc_s, k > 0 ? 1u : 0u);
                    tc::mma_commit(&s_full[buf(i)]);
                    tc::mma_commit(&op_empty[2 * i % Cfg::OPS]);
                }
                __syncwarp();
            };
            auto pv = [&](int i, int half) {
                const uint64_t dv = dv0 + (uint64_t)(((2 * i + 1) % Cfg::OPS) * (Cfg::KV_BYTES >> 4));
                const uint32_t tmem_p = tmem + buf(i) * BKV;
                if (tc::elect_one()) {
#pragma unroll
                    for (int k = half * (BKV / 32); k < (half + 1) * (BKV / 32); ++k)
                        tc::mma_f16_ts(tmem_o, tmem_p + 8 * k, dv + (uint64_t)(k * ((16 * 128) >> 4)), idesc_o, i > 0 || k > 0 ? 1u : 0u);
                    if (half == 1) {
                        tc::mma_commit(&op_empty[(2 * i + 1) % Cfg::OPS]);
                        tc::mma_commit(&o_done[t]);
                    }
                }
                __syncwarp();
            };
            auto p_step = [&](int i) {
                if (!tc::warp_wait(tc::smem_u32(&p_half[buf(i)]), par(i), false, deadline, &abort_s)) return false;
                tc::tc_fence_after_sync();
                pv(i, 0);
                if (!tc::warp_wait(tc::smem_u32(&p_ready[buf(i)]), par(i), false, deadline, &abort_s)) return false;
                tc::tc_fence_after_sync();
                pv(i, 1);
                return true;
            };
            auto there = [&](int n) {
                const bool ok = tc::warp_wait(tc::smem_u32(&op_full[n % Cfg::OPS]), (uint32_t)((n / Cfg::OPS) & 1), false, deadline, &abort_s);
                tc::tc_fence_after_sync();
                return ok;
            };
            bool ok = nt == 0 || (tc::warp_wait(tc::smem_u32(&q_full), 0u, false, deadline, &abort_s) && there(0));
            if (ok && nt > 0) qk(0);
            for (int i = 0; ok && i < nt; ++i) {
                if (i + 1 < nt) {                            // the next scores first: the softmax finds them when it is through with these
                    ok = there(2 * i + 2);
                    if (!ok) break;
                    qk(i + 1);
                }
                ok = there(2 * i + 1) && p_step(i);
            }
            if (!ok) gave_up(3);
        } else if (warp == 13) {
            // ---------------- copies: lane = (box of a block, keys or values); scales by the lanes of 16 keys each
            const int box = min(BKV, p.block_size), boxes = BKV / box;
            const CUtensorMap* map = lane & 1 ? &tmV : &tmK;
            auto page_of = [&](int j, int k) {              // k: first key of the box in the tile; INT_MIN: no key of the item there
                const int k0 = j * BKV + k;
                if (k0 >= key_hi || k0 + box <= key_lo) return INT_MIN;
                const int page = table[k0 >> p.block_shift];
                return page < 0 || page >= p.num_blocks ? -1 : page;
            };
            int page = INT_MIN;
            const int my_k = (lane >> 1) * box;
            auto group_scales = [&](int j) {                // of group lane / 2: this lane's tensor
                const int pg = lane < 2 * GR ? page_of(j, (lane >> 1) * 16 / box * box) : INT_MIN;
                return pg >= 0 ? fmaxf((lane & 1 ? p.v_scale : p.k_scale)[(size_t)pg * p.hkv + h], 1e-30f) : 0.0f;
            };
            if (nt > 0 && (lane >> 1) < boxes) page = page_of(j0, my_k);
            float scale = nt > 0 ? group_scales(j0) : 0.0f;
            for (int i = 0; i < nt; ++i) {
                const int j = j0 + i;
                const int wanted = __popc(__ballot_sync(0xffffffffu, page != INT_MIN)) / 2;       // boxes of each tensor
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int slot = (2 * i + x) % Cfg::RAWS;
                    if (!tc::warp_wait(tc::smem_u32(&raw_empty[slot]), (uint32_t)(((2 * i + x) / Cfg::RAWS) & 1) ^ 1u, false, deadline, &abort_s)) {
                        gave_up(1);
                        i = nt;
                        break;
                    }
                    if (lane == 0) tc::mbar_arrive_expect_tx(&raw_full[slot], (unsigned)(wanted * box * D));
                    __syncwarp();
                    if (page != INT_MIN && (lane & 1) == x) {
                        const int row = page >= 0 ? (page * p.hkv + h) * p.block_size + ((j * BKV + my_k) & (p.block_size - 1)) : p.pool_rows;
                        tc::tma_load_2d(sm + Cfg::OFF_RAW + slot * Cfg::RAW_BYTES + my_k * D, map, tc::smem_u32(&raw_full[slot]), 0, row);
                    }
                    if (x == 0) {
                        const float vs = __shfl_down_sync(0xffffffffu, scale, 1);
                        if (lane < 2 * GR && !(lane & 1))
                            scale_s[i % Cfg::RING][lane >> 1] = scale > 0.0f ? make_float4(scale, lg2(vs), rcp(vs), 0.0f)
                                                                             : make_float4(0.0f, -INFINITY, 0.0f, 0.0f);
                        __syncwarp();
                    }
                    if (lane == 0) tc::mbar_arrive(&raw_full[slot]);
                }
                if (i + 1 < nt) {
                    page = (lane >> 1) < boxes ? page_of(j + 1, my_k) : INT_MIN;
                    scale = group_scales(j + 1);
                }
            }
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::REGS_CONVERT));
        // ---------------- E4M3 bytes -> fp16 operand rows of 128 bytes (64 dimensions), 128-byte swizzle.  A thread takes 16 bytes; the blocks
        // of 64 that neighbouring rows take differ, so that neither the reads nor the writes of eight lanes share banks.
        constexpr int BL = D / 64, PASSES = BKV / 32 * BL, AT_ONCE = PASSES < 4 ? PASSES : 4;
        const int c = tid - 256, sub = c & 3, r_in = c >> 2;
        for (int i = 0; i < nt; ++i) {
            const int key0 = (j0 + i) * BKV;
            const bool inside = key0 >= key_lo && key0 + BKV <= key_hi;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int n = 2 * i + x, slot = n % Cfg::RAWS, op = n % Cfg::OPS;
                const uint32_t src = sm + Cfg::OFF_RAW + slot * Cfg::RAW_BYTES, dst = sm + Cfg::OFF_OP + op * Cfg::KV_BYTES;
                bool ok = tc::mbar_wait_until(&raw_full[slot], (uint32_t)((n / Cfg::RAWS) & 1), deadline, &abort_s);
                ok = ok && tc::mbar_wait_until(&op_empty[op], (uint32_t)((n / Cfg::OPS) & 1) ^ 1u, deadline, &abort_s);
                if (!__all_sync(0xffffffffu, ok)) { gave_up(2); i = nt; break; }
#pragma unroll
                for (int q0 = 0; q0 < PASSES; q0 += AT_ONCE) {
                    uint4 w[AT_ONCE];
#pragma unroll
                    for (int q = 0; q < AT_ONCE; ++q) {
                        const int r = r_in + 32 * ((q0 + q) / BL), bl = BL == 1 ? 0 : ((q0 + q) % BL) ^ (r & 1);
                        w[q] = ld_shared_v4(src + r * D + (bl * 4 + sub) * 16);
                        // rows outside the item's keys may be anything, and 0 x NaN is NaN
                        if (!inside && (key0 + r < key_lo || key0 + r >= key_hi)) w[q] = make_uint4(0, 0, 0, 0);
                    }
#pragma unroll
                    for (int q = 0; q < AT_ONCE; ++q) {
                        const int r = r_in + 32 * ((q0 + q) / BL), bl = BL == 1 ? 0 : ((q0 + q) % BL) ^ (r & 1);
                        uint32_t f[8];
                        e4m3x4_to_f16(w[q].x, f[0], f[1]);
                        e4m3x4_to_f16(w[q].y, f[2], f[3]);
                        e4m3x4_to_f16(w[q].z, f[4], f[5]);
                        e4m3x4_to_f16(w[q].w, f[6], f[7]);
                        const uint32_t row = dst + bl * (BKV * 128) + r * 128;
                        st_shared_v4(row + (((2 * sub) ^ (r & 7)) << 4), f[0], f[1], f[2], f[3]);
                        st_shared_v4(row + (((2 * sub + 1) ^ (r & 7)) << 4), f[4], f[5], f[6], f[7]);
                    }
                }
                tc::fence_proxy_async_smem();               // operands are read by the tensor core, the bytes written by the next copy
                __syncwarp();
                if (lane == 0) {
                    tc::mbar_arrive(&raw_empty[slot]);
                    tc::mbar_arrive(&op_full[op]);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::REGS_SOFTMAX));
        const int t = warp >> 2;
        if (t < T) {
            // ---------------- softmax: thread = row
            const int row = (warp & 3) * 32 + lane, r = t * 128 + row;             // in the tile, in the item
            const bool real = r < rows;
            const int at_row = row0 + min(r, rows - 1);             // rows behind the last go along with it
            const int i_tok = at_row / p.group, hh = h * p.group + at_row % p.group, token = start + i_tok;
            const int pos = len - n_new + i_tok;
            const int hi = max(0, min(p.causal ? pos + 1 : len, key_hi)), lo = window_from(p, pos);
            // the warp's 32 queries, 16 bytes a lane: fp16 at most 1 in magnitude, 16-byte chunks at chunk xor row % 8
            float rf;
            {
                constexpr int CH = D / 8, RP = 32 / CH;                // chunks of a row, rows of a step
                const int ch = lane % CH;
#pragma unroll 1
                for (int s0 = 0; s0 < 32; s0 += 8 * RP) {
                    uint4 w[8];
#pragma unroll
                    for (int s = 0; s < 8; ++s) {
                        const int q_row = t * 128 + (warp & 3) * 32 + s0 + s * RP + lane / CH, q_at = row0 + min(q_row, rows - 1);
                        w[s] = make_uint4(0, 0, 0, 0);
                        if (q_row < rows)
                            w[s] = ld_global_v4(p.q + (size_t)(start + q_at / p.group) * p.q_stride + (size_t)(h * p.group + q_at % p.group) * D + ch * 8);
                    }
#pragma unroll
                    for (int s = 0; s < 8; ++s) {
                        const int r_w = s0 + s * RP + lane / CH;      // in the warp
                        const uint32_t* ww = &w[s].x;
                        float x[8], top = 0.0f;
#pragma unroll
                        for (int e = 0; e < 4; ++e) unpack_bf16x2(ww[e], x[2 * e], x[2 * e + 1]);
#pragma unroll
                        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
#pragma unroll
                        for (int d = 1; d < CH; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                        const int e2 = query_exponent(top);
                        const float down = __uint_as_float((uint32_t)(127 - e2) << 23);
                        const int q_row = (warp & 3) * 32 + r_w;
                        st_shared_v4(sm + t * Cfg::Q_BYTES + (ch >> 3) * (128 * 128) + q_row * 128 + (((ch & 7) ^ (q_row & 7)) << 4),
                                     pack_f16x2(x[0] * down, x[1] * down), pack_f16x2(x[2] * down, x[3] * down),
                                     pack_f16x2(x[4] * down, x[5] * down), pack_f16x2(x[6] * down, x[7] * down));
                        if (ch == 0) rf_s[t * 128 + q_row] = __uint_as_float((uint32_t)(127 + e2) << 23);
                    }
                }
                tc::fence_proxy_async_smem();
                __syncwarp();
                rf = rf_s[r] * p.scale * LOG2E;
                tc::mbar_arrive(&q_full);
            }
            const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t tmem_O = tmem + Cfg::O_COL + t * D + lane_off;
            const bool capped = p.cap > 0.0f;
            const float cap2 = p.cap * LOG2E, inv_cap2 = capped ? 1.0f / cap2 : 0.0f;       // of base-2 logits
            // keys that every row of the warp sees
            const int w_hi = (int)__reduce_min_sync(0xffffffffu, (unsigned)hi), w_lo = (int)__reduce_max_sync(0xffffffffu, (unsigned)lo);
            const bool idle = t * 128 + (warp & 3) * 32 >= rows;    // a warp behind the last row only signs
            float m = -INFINITY, l = 0.0f;
            bool alive = true;
            // A parity tells a phase of o_done from its neighbours only.  While a warp has not signed tile i, the products of tile i - 2 are
            // through (its scores stood behind them) and that of tile i is not, so it may wait for tile i - 1's; once it has signed, it may
            // find itself two behind, or two ahead of warps that have not.  Hence the last product but one is waited for before the
            // last tile is signed, and the last one after it.
            auto last_but_one = [&](int i) {
                if (i == 0 || i != nt - 1) return true;
                const bool ok = tc::mbar_wait_until(&o_done[t], (uint32_t)((i - 1) & 1), deadline, &abort_s);
                alive = __all_sync(0xffffffffu, ok) != 0;
                if (!alive) gave_up(5);
                return alive;
            };
            for (int i = 0; i < nt; ++i) {
                const int sb = 2 * t + (i & 1);
                const uint32_t par = (uint32_t)((i >> 1) & 1), tmem_S = tmem + sb * BKV + lane_off;
                const int key0 = (j0 + i) * BKV;
                const float4* sc = scale_s[i % Cfg::RING];
                const bool open = key0 >= w_lo && key0 + BKV <= w_hi, plain = !capped && open;     // warp-uniform
                const bool ok = tc::mbar_wait_until(&s_full[sb], par, deadline, &abort_s);
                if (!__all_sync(0xffffffffu, ok)) { gave_up(4); alive = false; break; }
                tc::tc_fence_after_sync();
                if (idle) {
                    if (!last_but_one(i)) break;
                    tc::tc_fence_before_sync();
                    tc::mbar_arrive(&p_half[sb]);
                    tc::mbar_arrive(&p_ready[sb]);
                    continue;
                }
                if (!plain) {
                    // Capped tiles that no mask cuts leave the comparisons out, and the cap works on base-2 logits: 16 x 5 drafted tokens under a
                    // window and a cap 48.6 -> 42.8 us, capped chunks of 2048 on 4096 keys 506 -> 417 (42.9 and 420 with the form of tanh
                    // chosen score by score where a warp's columns need both; 545 where most scores pass half of the cap).
                    // the base-2 logits themselves, masked, over S; factor 1 and addend 0 from here on.  In a loop of 32 columns: written out
                    // over a row of registers this was 40 KB of instructions, fetched anew for every tile
#pragma unroll 1
                    for (int k = 0; k < BKV; k += 32) {
                        uint32_t v[32];
                        tc::tmem_ld32(tmem_S + k, v);
                        const float2 s0 = *reinterpret_cast<const float2*>(&sc[k / 16]), s1 = *reinterpret_cast<const float2*>(&sc[k / 16 + 1]);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * (rf * (e < 16 ? s0.x : s1.x)));
                        if (capped) {
                            float far = 0.0f;
#pragma unroll
                            for (int e = 0; e < 32; ++e) far = fmaxf(far, fabsf(__uint_as_float(v[e])));
                            if (__all_sync(0xffffffffu, far <= 0.5f * cap2)) {
#pragma unroll
                                for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(soft_cap_low(__uint_as_float(v[e]), inv_cap2));
                            } else {
#pragma unroll
                                for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(soft_cap(__uint_as_float(v[e]), cap2, inv_cap2));
                            }
                        }
                        if (open) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) + (e < 16 ? s0.y : s1.y));
                        } else {
                            const int from = lo - key0 - k, to = hi - key0 - k;
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                v[e] = __float_as_uint(e >= from && e < to ? __uint_as_float(v[e]) + (e < 16 ? s0.y : s1.y) : -INFINITY);
                        }
                        tc::tmem_st32(tmem_S + k, v);
                    }
                    tc::tmem_st_wait();
                }
                uint32_t sv[BKV];
#pragma unroll
                for (int k = 0; k < BKV; k += 32) tc::tmem_ld32(tmem_S + k, sv + k);
                // factor and addend of each 16 keys, while the scores arrive
                float fac[GR], add[GR];
#pragma unroll
                for (int g = 0; g < GR; ++g) {
                    const float2 s = *reinterpret_cast<const float2*>(&sc[g]);
                    fac[g] = plain ? rf * s.x : 1.0f;
                    add[g] = plain ? s.y : 0.0f;
                }
                tc::tmem_ld_wait();
                float mx = -INFINITY;
#pragma unroll
                for (int g = 0; g < GR; ++g) {
                    const uint32_t* s = sv + g * 16;
                    auto v = [&](int e) { return __uint_as_float(s[e]); };
                    const float a = max3(max3(v(0), v(1), v(2)), v(3), v(4)), c = max3(max3(v(5), v(6), v(7)), v(8), v(9));
                    const float d = max3(max3(v(10), v(11), v(12)), max3(v(13), v(14), v(15)), a);
                    mx = fmaxf(mx, fmaf(fmaxf(c, d), fac[g], add[g]));
                }
                const bool grow = mx > m + Cfg::GROWTH;
                if (__any_sync(0xffffffffu, grow && i > 0)) {                     // warp-uniform: tensor-memory loads are collective
                    // the product before may still run: these scores were issued in front of it
                    const bool done = tc::mbar_wait_until(&o_done[t], (uint32_t)((i - 1) & 1), deadline, &abort_s);
                    if (!__all_sync(0xffffffffu, done)) { gave_up(5); alive = false; break; }
                    tc::tc_fence_after_sync();
                    const float f = grow ? ex2(m - mx) : 1.0f;
                    l *= f;
#pragma unroll 1
                    for (int k = 0; k < D; k += 32) {
                        uint32_t v[32];
                        tc::tmem_ld32(tmem_O + k, v);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
                        tc::tmem_st32(tmem_O + k, v);
                    }
                    tc::tmem_st_wait();
                }
                if (grow) m = mx;
                const float ref = Cfg::OFFSET - (m == -INFINITY ? 0.0f : m);
#pragma unroll
                for (int k = 0; k < BKV; k += 32) {
                    uint32_t u[16];
#pragma unroll
                    for (int gg = 0; gg < 2; ++gg) {
                        const int g = k / 16 + gg;
                        const uint64_t f2 = f32x2(fac[g], fac[g]), a2 = f32x2(add[g] + ref, add[g] + ref);
                        uint64_t sum = 0;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int at = k + gg * 16 + 2 * e;
                            float x, y;
                            f32x2_parts(fma_f32x2(f32x2(__uint_as_float(sv[at]), __uint_as_float(sv[at + 1])), f2, a2), x, y);
                            x = ex2(x);
                            y = ex2(y);
                            sum = add_f32x2(sum, f32x2(x, y));
                            u[gg * 8 + e] = pack_f16x2(x, y);
                        }
                        float s0, s1;
                        f32x2_parts(sum, s0, s1);
                        l = fmaf(s0 + s1, sc[g].z, l);
                    }
                    tc::tmem_st16(tmem_S + (k >> 1), u);
                    if (k == BKV / 2 - 32) {
                        tc::tmem_st_wait();
                        tc::tc_fence_before_sync();
                        tc::mbar_arrive(&p_half[sb]);
                    }
                }
                tc::tmem_st_wait();
                if (!last_but_one(i)) break;
                tc::tc_fence_before_sync();
                tc::mbar_arrive(&p_ready[sb]);
            }
            if (alive && nt > 0) {
                const bool ok = tc::mbar_wait_until(&o_done[t], (uint32_t)((nt - 1) & 1), deadline, &abort_s);
                alive = __all_sync(0xffffffffu, ok) != 0;
                if (!alive) gave_up(6);
                tc::tc_fence_after_sync();
            }
            const size_t part = (size_t)(item * pp.splits + split) * T + t;
            if (alive) {
                const float inv = inverse_sum(l);
#pragma unroll 1
                for (int k = 0; k < D; k += 32) {
                    uint32_t v[32];
                    __syncwarp();                               // the lanes part in the store
                    if (nt > 0) {
                        tc::tmem_ld32(tmem_O + k, v);
                        tc::tmem_ld_wait();
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = 0u;
                    }
                    if (!real) continue;
                    if (pieces > 1) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) __stcg(pp.part_o + (part * D + k + e) * 128 + row, __uint_as_float(v[e]));
                    } else {
                        __nv_bfloat16* dst = p.o + (size_t)token * p.o_stride + (size_t)hh * D + k;
#pragma unroll
                        for (int e = 0; e < 32; e += 8)
                            st_global_v4(dst + e, make_uint4(pack_bf16x2(__uint_as_float(v[e]) * inv, __uint_as_float(v[e + 1]) * inv),
                                                             pack_bf16x2(__uint_as_float(v[e + 2]) * inv, __uint_as_float(v[e + 3]) * inv),
                                                             pack_bf16x2(__uint_as_float(v[e + 4]) * inv, __uint_as_float(v[e + 5]) * inv),
                                                             pack_bf16x2(__uint_as_float(v[e + 6]) * inv, __uint_as_float(v[e + 7]) * inv)));
                    }
                }
                if (real) {
                    if (pieces > 1) __stcg(pp.part_ml + part * 128 + row, make_float2(m, l));
                    else if (p.lse) p.lse[(size_t)hh * p.tokens + token] = l == 0.0f ? -INFINITY : 0.6931471805599453f * (m - Cfg::OFFSET + log2f(l));
                }
            }
        }
    }
    if (abort_s && warp == 13) {                            // a wait gave up: copies may be in flight, a bounded time for them to land
        const uint64_t until = tc::global_timer_ns() + 1000000ull;
        while (tc::global_timer_ns() < until) {}
    }
    __syncwarp();
    tc::tc_fence_before_sync();
    __syncthreads();
    tc::tc_fence_after_sync();
    if (warp == 12) tc::tmem_dealloc(tmem, 512);
}

// Joins an item's pieces: row r has o = sum_z 2^(m_z - m) o_z / sum_z 2^(m_z - m) l_z, m = max_z m_z, in the order of z.  A block takes 32
// rows (lanes) x 32 columns (4 a warp), so that an item of 8 pieces of 128 x 256 sums, a megabyte, is read by 32 SMs.  One CTA of the kernel
// above, the last to arrive, took 26 us for it: 64 rows on 300 keys (heads of 256) 64 -> 18 us,
// on 16384 107 -> 35, now that an item may have more than 8 pieces.
template <int D>
__global__ void __launch_bounds__(256) paged_join_kernel(const PrefillParams pp, int row_tiles) {
    const PagedAttnParams& p = pp.a;
    pdl_launch_dependents();
    pdl_wait();
    const int item = (int)blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int4 it = __ldcg(pp.items + item);
    const int row = (int)blockIdx.y * 32 + lane, col = (int)blockIdx.z * 32 + warp * 4;
    if (it.w <= 1 || row >= it.z) return;
    const size_t step = (size_t)row_tiles * 128, first = (size_t)item * pp.splits * step + row;      // of (m, l): [piece][tile][row]
    const float2* ml = pp.part_ml + first;
    const float* o = pp.part_o + (first - (row & 127)) * D + (size_t)col * 128 + (row & 127);
    float m = -INFINITY, l = 0.0f, sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int z0 = 0; z0 < it.w; z0 += 8) {                  // all loads of 8 pieces in front of their sums
        float2 part[8];
        float v[8][4];
#pragma unroll
        for (int z = 0; z < 8; ++z) {
            const bool there = z0 + z < it.w;
            part[z] = there ? __ldcg(ml + (z0 + z) * step) : make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[z][e] = there ? __ldcg(o + (z0 + z) * step * D + e * 128) : 0.0f;
        }
        float now = m;
#pragma unroll
        for (int z = 0; z < 8; ++z) now = fmaxf(now, part[z].x);
        const float safe = now == -INFINITY ? 0.0f : now, keep = ex2(m - safe);
        m = now;
        l *= keep;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] *= keep;
#pragma unroll
        for (int z = 0; z < 8; ++z) {
            const float f = ex2(part[z].x - safe);
            l = fmaf(part[z].y, f, l);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = fmaf(v[z][e], f, sum[e]);
        }
    }
    const float inv = inverse_sum(l);
    const int at = it.y + row, token = it.x + at / p.group, hh = (item / pp.tiles) * p.group + at % p.group;
    st_global_v2(p.o + (size_t)token * p.o_stride + (size_t)hh * D + col,
                 make_uint2(pack_bf16x2(sum[0] * inv, sum[1] * inv), pack_bf16x2(sum[2] * inv, sum[3] * inv)));
    if (p.lse && col == 0)
        p.lse[(size_t)hh * p.tokens + token] = l == 0.0f ? -INFINITY : 0.6931471805599453f * (m - PrefillCfg<D, 1>::OFFSET + log2f(l));
}

// Row tiles of all sequences, at most: a sequence adds less than one to its rows' share, and has no more than max_new tokens.
static long long prefill_tiles(long long tokens, long long batch, long long max_new, int group, int tile_rows) {
    const long long by_rows = tokens * group / tile_rows + batch, by_sequence = batch * ((max_new * group + tile_rows - 1) / tile_rows);
    return by_rows < by_sequence ? by_rows : by_sequence;
}
// Splits of the keys where the items leave SMs idle; `tiles`: of keys that a table has room for.  Beyond 64 pieces the join takes longer
// than the tiles that it saves.
static int prefill_splits(long long items, long long tiles, int sms) {
    long long s = sms / (items < 1 ? 1 : items);
    s = s < 64 ? s : 64;
    s = s < (tiles + 1) / 2 ? s : (tiles + 1) / 2;
    return s < 1 ? 1 : (int)s;
}
// Pieces of all items where the keys are split (no more than SMs), at the larger of the row tiles: a workspace for many rows serves fewer,
// which may be split more.
static long long prefill_workspace(int d) {
    return (long long)device_sm_count() * (16 + (d == 256 ? 1 : 2) * 128 * (8 + 4 * d));
}

template <int D, int T>
static int launch_prefill(const PagedAttnParams& a, int max_new, void* work, cudaStream_t stream) {
    using Cfg = PrefillCfg<D, T>;
    static PerDeviceOnce attr_once;
    int attr_dev = 0;
    if (attr_once.need(attr_dev)) {
        const cudaError_t e = cudaFuncSetAttribute(paged_prefill_kernel<D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES);
        if (e != cudaSuccess) return FRT_CUDA_ERR(e);
        attr_once.set(attr_dev);
    }
    const long long tiles = prefill_tiles(a.tokens, a.batch, max_new, a.group, 128 * T), items = tiles * a.hkv;
    if (items > 0x7fffffffLL) return FRT_ERR_UNSUPPORTED;
    PrefillParams pp = {};
    pp.a = a;
    pp.splits = prefill_splits(items, ((long long)a.room + Cfg::BKV - 1) / Cfg::BKV, device_sm_count());
    pp.tiles = (int)tiles;
    pp.items = static_cast<int4*>(work);
    pp.part_ml = reinterpret_cast<float2*>(pp.items + items);
    pp.part_o = reinterpret_cast<float*>(pp.part_ml + items * pp.splits * T * 128);
    CUtensorMap tmK, tmV;
    const int box = Cfg::BKV < a.block_size ? Cfg::BKV : a.block_size;
    int rc = paged_map(&tmK, a.k, a.pool_rows, D, box, false);
    if (!rc) rc = paged_map(&tmV, a.v, a.pool_rows, D, box, false);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)tiles, (unsigned)a.hkv, (unsigned)pp.splits);
    cfg.blockDim = dim3(Cfg::THREADS);
    cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, paged_prefill_kernel<D, T>, tmK, tmV, pp);
    if (e != cudaSuccess || pp.splits == 1) return e == cudaSuccess ? FRT_OK : FRT_CUDA_ERR(e);
    cfg.gridDim = dim3((unsigned)items, T * 4, D / 32);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, paged_join_kernel<D>, pp, T);
    return e == cudaSuccess ? FRT_OK : FRT_CUDA_ERR(e);
}

// Attention over 4-bit pages on the tensor cores, few query rows per kv head (decode, short chunks): f16 / bf16, E == Ev == 64 or 128.
//
// By its bytes bound by HBM: 9/8 byte per (key, channel) of K and V together, 144 bytes per key and kv head at head size 128, against 512 in
// 16 bits -- so what a key costs on the SM counts: at the full copy rate an SM has to finish one every six cycles.  Bound by instruction issue:
// 350 instructions of a warp per 16 keys, the schedulers at 62 %.  2 sequences of 131,072 keys, 8 kv heads of 4 heads: 77.0 us = 3.92 TB/s;
// 24 of 6,000 keys down to 1,331, 5 heads: 40 us; 8 of 16,384 keys, 2 kv heads of 16 heads: 31.7 us, of which the walk is ten.
//
// Both products are taken transposed, keys or value channels as the M of mma.sync m16n8k16 and up to eight query rows as its N:
//     S^T [16 keys x 8 rows] = K [16 x E] Q^T,      O^T [E x 8 rows] += V^T [E x 16 keys] P^T
// With rows as the M (16) and four heads per kv head three quarters of the products would be padding.  The 4-bit operand is the A
// operand of both; its fragments are unpacked from shared memory straight into registers, two values per conversion:
//   * K: the order of a product's channels is free as long as Q has the same, so a thread's A fragments of all steps are 32 (16)
//     consecutive channels of two keys: one 16-byte (8-byte) load each, and two scales (one).
//   * V^T: a thread's rows of all tiles are the 16 (8) consecutive channels of one scale group, for four keys; pairs of keys at one
//     channel are put together from two words with masks and a shift.
// Values times scales are exact in fp16 (six significant bits), so the only rounding is that of P.  bf16 queries are brought to fp16 by a
// power of two per row, which loses nothing a float accumulator would keep: magnitudes down to 2^-39 of the row's largest are held.
// P goes from the accumulators of the first product to the B operand of the second by movmatrix.
//
// Every warp works alone: 16 keys of each 128-key tile, fetched by its own cp.async copies into its own ring, its own running maximum and
// sum; the eight (or four) warps meet only where a unit ends.  Rows are looked up in the block table one tile ahead of their copies.
//
// P in fp16: a row's reference lies 2^7 below its maximum and O is rescaled only when some score exceeds it by 2^15, so the largest probability stands
// between 2^7 and 2^15, and fp16's 11 bits reach down to 2^-21 of it, its last one to 2^-31.  (With the maximum itself as the reference all keys
// below 2^-25 of the largest were lost: beside a key that takes nearly all of the weight, thousands of others count together.)
//
// Split: units (<= 16 query rows that share keys, kv head) are cut into 128-key tiles, all units' tiles are one list, every CTA takes an
// equal contiguous share (two CTAs per SM), in which a unit's start and end count as some tiles.  A share's part of a unit is a partial; q4_mma_merge_kernel adds them up.  With as many units as
// CTAs each unit gets a CTA of its own, and no merge step; with more, CTAs of four warps, four per SM, whose starts and ends overlap.
#pragma once
#include <float.h>

#include <type_traits>

#include "hogatt_q4.cuh"

namespace hogatt {

constexpr int kQ4Ctas = 2;       // resident CTAs of eight warps per SM (four of four warps)
// Powers of two: a row's reference below its maximum, a score above it that moves it.  (Maxima of 2^24 and more round what is taken off: 7 becomes 8 at most, 8
// became 16, which is beyond fp16.)
constexpr float kQ4RefBelow = 7.f, kQ4RefAbove = 15.f;

struct Q4MmaArgs {
    PagedArgs p;                  // kcache / vcache: the codes; splits: unused; groups_bound: entries of the prefix
    const unsigned char* kscale;
    const unsigned char* vscale;
    int num_blocks;
    float vunit;
    FastDiv block;                // block size
    int ctas;                     // the list's shares; 0: a CTA per unit
    int unit_cost;                // what a unit counts for in the list beside its tiles
    int* plan;                    // [groups_bound + 1]: length of the list of one kv head's units in front of every group of query tokens
};

template <int HD, int WARPS>
struct Q4MmaCfg {
    static constexpr int THREADS = WARPS * 32, TILE = WARPS * 16;  // keys of a tile: 16 a warp
    static constexpr int ROW = HD / 2, SROW = HD / kGroup;         // bytes of a row's codes and scales
    static constexpr int STAGE = 16 * 2 * (ROW + SROW) + 16;       // K, V, K scales, V scales of 16 keys; which have no page
    static constexpr int OFF_V = 16 * ROW, OFF_KS = 32 * ROW, OFF_VS = OFF_KS + 16 * SROW, OFF_BAD = OFF_VS + 16 * SROW;
    // Three tiles of a ring: sixteen warps an SM hide one another's copies, and a shorter prologue comes sooner to its first tile.  us with 5 / 4 / 3 / 2 at
    // head size 128: 2 sequences of 131,072 keys 75.5 / 74.9 / 74.4 / 74.4, 24 ragged ones 43.5 / 43.1 / 43.0 / 42.8; with 8 / 6 / 5 / 3 at 64:
    // the latter 32.8 / 32.8 / 32.2 / 31.6.
    static constexpr int NSTAGE = 3;
    static constexpr int RING = WARPS * NSTAGE * STAGE;
    static constexpr int PITCH = HD + 4;                           // floats between rows of the fold
    static constexpr int fold_bytes(int rows) { return WARPS * rows * (PITCH + 2) * 4; }
    static constexpr int ring_bytes(int nt) { return RING > fold_bytes(8 * nt) ? RING : fold_bytes(8 * nt); }
    // sixteen query rows do not fit in registers beside O: their fragments, the same for every warp, lie in shared memory
    static constexpr int q_bytes(int nt) { return nt == 2 ? nt * (HD / 32) * 512 : 0; }
    static constexpr int work_bytes(int nt) { return ring_bytes(nt) + q_bytes(nt); }
};
template <int HD, int WARPS>
__host__ __device__ inline size_t q4_mma_smem_bytes(int nt, int W, int groups, bool list) {
    return Q4MmaCfg<HD, WARPS>::work_bytes(nt) + (list ? ((size_t)W + 1 + 2 * groups + 1) * sizeof(int) : 0);
}

// the 8x8 matrix of 16-bit elements that the warp holds (row lane / 4, columns 2 (lane % 4) and + 1), transposed
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// shared memory by its 32-bit address, `OFF` bytes further (generic pointers cost the loop an address per load)
template <int OFF>
__device__ __forceinline__ uint4 lds128(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4+%5];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at), "n"(OFF));
    return v;
}
template <int OFF>
__device__ __forceinline__ uint2 lds64(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2+%3];" : "=r"(v.x), "=r"(v.y) : "r"(at), "n"(OFF));
    return v;
}
template <int OFF>
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1+%2];" : "=r"(v) : "r"(at), "n"(OFF));
    return v;
}
template <int OFF>
__device__ __forceinline__ uint32_t lds16(uint32_t at) {
    uint16_t v;
    asm volatile("ld.shared.b16 %0, [%1+%2];" : "=h"(v) : "r"(at), "n"(OFF));
    return v;
}
template <int OFF>
__device__ __forceinline__ uint32_t lds8(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1+%2];" : "=r"(v) : "r"(at), "n"(OFF));
    return v;
}
// `n` of 16 (8, 4) bytes copied, the others zeros
template <int BYTES>
__device__ __forceinline__ void cp_async_zfill(uint32_t dst, const void* src, bool real) {
    const int n = real ? BYTES : 0;
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}

// Visible keys of (group of query tokens, fragment): the most that any of its rows sees.
__device__ __forceinline__ int group_visible(const PagedArgs& a, int f, int w, int s_base, int s_begin, int s_end) {
    int top = -1;
    for (int s = s_begin; s < s_end; ++s) top = max(top, a.loc[(size_t)f * a.loc_f + (size_t)w * a.loc_w + s_base + s]);
    return most_visible(a, top, a.flen[f * a.len_f + w * a.len_w]);
}
__device__ __forceinline__ int tokens_of(const PagedArgs& a, int w, int* start) {
    *start = a.cu_seqlens ? a.cu_seqlens[w] : 0;
    return a.cu_seqlens ? max(0, min(a.cu_seqlens[w + 1], a.total_q) - *start) : a.S;
}

// Sequence, tokens and heads of unit x, by a whole warp: a lane counts the groups of a run of sequences, its loads all under way at once.
__device__ __forceinline__ bool locate_unit(const PagedArgs& a, int x, PagedUnit* u) {
    const int lane = threadIdx.x & 31;
    u->hkv = x % a.Hkv;
    const int y = x / a.Hkv;
    u->g0 = (y % a.head_blocks) * 16;
    int grp = y / a.head_blocks;
    if (a.cu_seqlens == nullptr) {
        const int each = (a.S + a.tokens_per_group - 1) / a.tokens_per_group;
        u->w = grp / each;
        u->s_base = 0;
        u->s_begin = (grp - u->w * each) * a.tokens_per_group;
        u->s_end = min(a.S, u->s_begin + a.tokens_per_group);
        return u->w < a.W;
    }
    const int run = (a.W + 31) / 32, w0 = min(a.W, lane * run), w1 = min(a.W, w0 + run);
    auto groups_of = [&](int w) {
        int start;
        return (tokens_of(a, w, &start) + a.tokens_per_group - 1) / a.tokens_per_group;
    };
    int mine = 0;
#pragma unroll 8
    for (int w = w0; w < w1; ++w) mine += groups_of(w);
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int z = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += z;
    }
    const unsigned here = __ballot_sync(0xffffffffu, grp < inc);
    if (!here) return false;
    const int src = __ffs(here) - 1;
    grp -= __shfl_sync(0xffffffffu, inc - mine, src);
    int w = w0;
    if (lane == src)
        for (int n; grp >= (n = groups_of(w)); ++w) grp -= n;
    w = __shfl_sync(0xffffffffu, w, src);
    grp = __shfl_sync(0xffffffffu, grp, src);
    int start;
    const int tokens = tokens_of(a, w, &start);
    u->w = w;
    u->s_base = start;
    u->s_begin = grp * a.tokens_per_group;
    u->s_end = min(tokens, u->s_begin + a.tokens_per_group);
    return true;
}

template <class T, int HD, int NT, bool ALIGNED, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, kQ4Ctas * 8 / WARPS) q4_mma_kernel(const __grid_constant__ Q4MmaArgs x) {
    using C = Q4MmaCfg<HD, WARPS>;
    constexpr int KS = HD / 16;              // steps of S^T = tiles of O^T
    constexpr int CPT = HD / 4, DPT = HD / 8;        // channels of a key, of a value that a thread holds
    const PagedArgs& a = x.p;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    unsigned char* const ring = smem_raw + warp * C::NSTAGE * C::STAGE;
    const uint32_t ring_u32 = smem_u32(ring);
    int* const first_group = reinterpret_cast<int*>(smem_raw + C::work_bytes(NT));      // [W + 1]
    int* const pre = first_group + a.W + 1;                                              // [groups + 1]
    int* const seen = pre + a.groups_bound + 1;                                          // [groups]: the group's visible keys, of the last fragment
    const unsigned char* const kc = static_cast<const unsigned char*>(a.kcache);
    const unsigned char* const vc = static_cast<const unsigned char*>(a.vcache);
    const int per_group = a.Hkv * a.head_blocks;          // units of a group of query tokens

    pdl_wait();
    pdl_trigger();

    // ---- the list: tiles of every group, and this CTA's share ----
    int64_t item = 0, item_end = 0;
    int groups = 0;
    if (x.ctas) {
        int before = 0;
        if (a.cu_seqlens) {
            for (int w0 = 0; w0 < a.W; w0 += C::THREADS) {
                int start, n = 0, total;
                if (w0 + tid < a.W) n = (tokens_of(a, w0 + tid, &start) + a.tokens_per_group - 1) / a.tokens_per_group;
                const int at = before + block_exclusive(n, &total);
                if (w0 + tid < a.W) first_group[w0 + tid] = at;
                before += total;
            }
        } else {
            const int each = (a.S + a.tokens_per_group - 1) / a.tokens_per_group;
            for (int w = tid; w < a.W; w += C::THREADS) first_group[w] = w * each;
            before = a.W * each;
        }
        groups = min(before, a.groups_bound);
        if (tid == 0) first_group[a.W] = before;
        __syncthreads();
        before = 0;
        for (int e0 = 0; e0 < groups; e0 += C::THREADS) {
            const int e = e0 + tid;
            int n = 0, total;
            if (e < groups) {
                int lo = 0, hi = a.W;                     // the sequence: the last one that starts at or in front of e
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (first_group[mid] <= e) lo = mid;
                    else hi = mid;
                }
                int start;
                const int tokens = tokens_of(a, lo, &start), s0 = (e - first_group[lo]) * a.tokens_per_group;
                int vis = 0;
                for (int f = 0; f < a.F; ++f) {
                    vis = group_visible(a, f, lo, start, s0, min(tokens, s0 + a.tokens_per_group));
                    n += ceil_div(vis, C::TILE);
                }
                seen[e] = vis;
                n += n ? x.unit_cost : 0;
            }
            const int at = before + block_exclusive(n, &total);
            if (e < groups) pre[e] = at;
            before += total;
        }
        if (tid == 0) pre[groups] = before;
        __syncthreads();
        if (blockIdx.x == 0)
            for (int e = tid; e <= a.groups_bound; e += C::THREADS) x.plan[e] = pre[min(e, groups)];
        const int64_t N = (int64_t)before * per_group;
        const int shares = effective_ctas(N, x.ctas);     // none of them empty
        if ((int)blockIdx.x >= shares) return;
        item = cta_first_tile(blockIdx.x, N, shares);
        item_end = cta_first_tile(blockIdx.x + 1, N, shares);
    }

    int grp = 0;
    bool again = true;
    while (again) {
        // ---- the next unit of the share: its tiles [j0, j1) ----
        PagedUnit u;
        int unit = blockIdx.x, j0 = 0, j1 = INT_MAX;
        if (x.ctas) {
            int lo = grp, hi = groups;                    // the group: the last one that starts at or in front of `item`, with tiles
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if ((int64_t)pre[mid] * per_group <= item) lo = mid;
                else hi = mid;
            }
            grp = lo;
            const int n = pre[grp + 1] - pre[grp];
            const int64_t off = item - (int64_t)pre[grp] * per_group;
            const int of_group = (int)floor_div(off, n);
            unit = grp * per_group + of_group;
            j0 = (int)(off - (int64_t)of_group * n);
            j1 = (int)min((int64_t)n, j0 + (item_end - item));
            item += j1 - j0;
            again = item < item_end;
            j0 = max(0, j0 - x.unit_cost);                // (the tiles stand behind what the unit costs)
            j1 -= x.unit_cost;
            if (j0 >= j1) continue;
            int wl = 0, wh = a.W;
            while (wh - wl > 1) {
                const int mid = (wl + wh) >> 1;
                if (first_group[mid] <= grp) wl = mid;
                else wh = mid;
            }
            int start;
            const int tokens = tokens_of(a, wl, &start);
            u.w = wl;
            u.s_base = start;
            u.s_begin = (grp - first_group[wl]) * a.tokens_per_group;
            u.s_end = min(tokens, u.s_begin + a.tokens_per_group);
            u.hkv = of_group % a.Hkv;
            u.g0 = of_group / a.Hkv * 16;
        } else {
            again = false;
            if (!locate_unit(a, unit, &u)) return;        // (uniform: the grid is an upper bound)
        }
        const int* const table = a.block_table + (size_t)u.w * a.max_blocks;

        float o[NT][KS][4];
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = -FLT_MAX;                 // (nothing seen yet; finite, so that differences with it are)
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int k = 0; k < KS; ++k) o[n][k][0] = o[n][k][1] = o[n][k][2] = o[n][k][3] = 0.f;
        }

        int tiles_before = 0;
        bool whole = true;                                // this CTA has all of the unit's tiles
        for (int f = 0; f < a.F; ++f) {
            // ---- this fragment's tiles of the share ----
            const int vis = x.ctas && a.F == 1 ? seen[grp] : group_visible(a, f, u.w, u.s_base, u.s_begin, u.s_end);
            const int tiles = ceil_div(vis, C::TILE);
            const int b0 = max(j0, tiles_before) - tiles_before, b1 = min(j1, tiles_before + tiles) - tiles_before;
            whole = whole && (tiles == 0 || (b0 == 0 && b1 == tiles));
            tiles_before += tiles;
            if (b0 >= b1) continue;

            // ---- copies of 16 keys: rows of 4 (2) 16-byte chunks, dealt over the lanes; scales of K by lanes 0-15, of V by 16-31 ----
            constexpr int CPR = C::ROW / 16, PASSES = 16 * CPR / 32, RPP = 32 / CPR;
            const int row0 = lane / CPR, srow = lane & 15;                 // this lane's first row, and its scales' row
            const uint32_t dst0 = ring_u32 + row0 * C::ROW + (HD == 128 ? ((lane % CPR) ^ (row0 & 2)) * 16 : (lane % CPR) * 16);
            const uint32_t sdst0 = ring_u32 + (lane < 16 ? C::OFF_KS : C::OFF_VS) + srow * C::SROW;
            const unsigned char* const scales = lane < 16 ? x.kscale : x.vscale;
            // Where key `key`'s row is in either cache (rows of all pages and heads numbered through; ALIGNED: sixteens of rows, which 32 bits hold
            // however large the cache); -1: behind the keys, -2: a key without a page.
            using Row = std::conditional_t<ALIGNED, int, int64_t>;
            constexpr int PER = ALIGNED ? 16 : 1;
            auto row_of = [&](int key) -> Row {
                if (key >= vis) return -1;
                const int at = (int)fast_div((uint32_t)key, x.block);
                const int p = at < a.max_blocks ? table[at] : -1;
                if (p < 0 || p >= x.num_blocks) return -2;
                return ((Row)p * a.Hkv + u.hkv) * (a.block_size / PER) + (key - at * (int)x.block.d) / PER;
            };
            // ALIGNED: the 16 keys of a tile lie in one block, and the lanes look up 32 tiles at a time, the next 32 ahead of their use;
            // otherwise every lane looks its rows of the next tile up
            constexpr int LOOKUPS = ALIGNED ? 2 : PASSES + 1;
            Row from[LOOKUPS];
            int looked = b0;                              // ALIGNED: from[0] has tiles `looked` ..., from[1] the 32 behind them
            auto look_up = [&](int j) {
                const int k0 = j * C::TILE + warp * 16;
                if constexpr (ALIGNED) {
                    if (j - looked == 32) {
                        looked = j;
                        from[0] = from[1];
                        from[1] = row_of(k0 + (32 + lane) * C::TILE);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < PASSES; ++i) from[i] = row_of(k0 + i * RPP + row0);
                    from[PASSES] = row_of(k0 + srow);
                }
            };
            const unsigned char* const k_lane = kc + row0 * C::ROW + lane % CPR * 16;
            const unsigned char* const v_lane = vc + row0 * C::ROW + lane % CPR * 16;
            const unsigned char* const s_lane = scales + srow * C::SROW;
            const int whole_tiles = (vis - warp * 16) / C::TILE + ((vis - warp * 16) % C::TILE >= 16);        // tiles of which this warp has all 16 keys
            bool any_bad = false;                         // a tile with keys that have no page has been met: their bits are looked at
            auto fetch = [&](int j, uint32_t base) {      // base: the stage's bytes from the ring's start
                const Row tile_from = ALIGNED ? __shfl_sync(0xffffffffu, from[0], j - looked) : 0;       // (the lane: modulo 32)
                if (ALIGNED && j < whole_tiles && tile_from >= 0) {
                    const unsigned char* const ks = k_lane + (int64_t)tile_from * (16 * C::ROW);
                    const unsigned char* const vs = v_lane + (int64_t)tile_from * (16 * C::ROW);
#pragma unroll
                    for (int i = 0; i < PASSES; ++i) {
                        cp_async_16(dst0 + base + i * RPP * C::ROW, ks + i * RPP * C::ROW, true);
                        cp_async_16(dst0 + base + C::OFF_V + i * RPP * C::ROW, vs + i * RPP * C::ROW, true);
                    }
                    cp_async_zfill<C::SROW>(sdst0 + base, s_lane + (int64_t)tile_from * (16 * C::SROW), true);
                    if (any_bad && lane == 0) *reinterpret_cast<uint32_t*>(ring + base + C::OFF_BAD) = 0u;
                } else {                                  // (rows that are not there: zeros, from an address inside the cache)
                    const int left = vis - (j * C::TILE + warp * 16);      // keys there are from here on
#pragma unroll
                    for (int i = 0; i < PASSES; ++i) {
                        const Row row = ALIGNED ? tile_from : from[i];
                        const bool real = row >= 0 && row0 + i * RPP < left;
                        const int64_t at = (real ? (int64_t)row * PER + (ALIGNED ? row0 + i * RPP : 0) : 0) * C::ROW + lane % CPR * 16;
                        cp_async_zfill<16>(dst0 + base + i * RPP * C::ROW, kc + at, real);
                        cp_async_zfill<16>(dst0 + base + C::OFF_V + i * RPP * C::ROW, vc + at, real);
                    }
                    const Row row = ALIGNED ? tile_from : from[LOOKUPS - 1];
                    const bool real = row >= 0 && srow < left;
                    cp_async_zfill<C::SROW>(sdst0 + base, scales + (real ? (int64_t)row * PER + (ALIGNED ? srow : 0) : 0) * C::SROW, real);
                    const uint32_t bad = __ballot_sync(0xffffffffu, row == -2 && srow < left) & 0xffffu;
                    if (bad && lane == 0 && a.status) atomicOr(a.status, STATUS_BAD_BLOCK);
                    any_bad = any_bad || bad != 0;
                    if (any_bad && lane == 0) *reinterpret_cast<uint32_t*>(ring + base + C::OFF_BAD) = bad;
                }
                cp_async_commit();
            };

            // ---- the walk ----
            if constexpr (ALIGNED) {
                from[0] = row_of(b0 * C::TILE + warp * 16 + lane * C::TILE);
                from[1] = row_of(b0 * C::TILE + warp * 16 + (32 + lane) * C::TILE);
            } else {
                look_up(b0);
            }
            // (a stage's bits of keys without a page are first read after a tile that has some has been met: zero until then)
            if (lane < C::NSTAGE) *reinterpret_cast<uint32_t*>(ring + lane * C::STAGE + C::OFF_BAD) = 0u;
            __syncwarp();
#pragma unroll 1
            for (int k = 0; k < C::NSTAGE - 1; ++k) {
                if (b0 + k < b1) {
                    fetch(b0 + k, k * C::STAGE);
                    if (b0 + k + 1 < b1) look_up(b0 + k + 1);
                } else {
                    cp_async_commit();
                }
            }
            // ---- the query rows as B fragments (the first copies are under way): thread (g, t) has channels CPT t ... of row g of each eight ----
            uint32_t q[NT == 1 ? KS : 1][2];
            uint4* const q_smem = reinterpret_cast<uint4*>(smem_raw + C::ring_bytes(NT)) + lane;
            if (NT == 2 && f > 0) __syncthreads();        // (every warp has left the last fragment)
            float factor[NT][2];                          // what a product of columns 2 t, 2 t + 1 is multiplied with: log2 e * scale / row's power
            int lim[NT][2], lowest = INT_MAX;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                int s_abs, hq;
                const bool real = paged_row(a, u, n * 8 + g, &s_abs, &hq);
                uint4 raw[CPT / 8];
#pragma unroll
                for (int k = 0; k < CPT / 8; ++k) raw[k] = make_uint4(0u, 0u, 0u, 0u);
                if (real) {
                    const T* src = static_cast<const T*>(a.q) + f * a.q_f + u.w * a.q_w + s_abs * a.q_s + hq * a.q_h + t * CPT;
#pragma unroll
                    for (int k = 0; k < CPT / 8; ++k) {
                        const int4 v = load_16(src + k * 8);
                        raw[k] = make_uint4(v.x, v.y, v.z, v.w);
                    }
                }
                float mine = fabsf(a.l2scale);
                uint32_t* r = reinterpret_cast<uint32_t*>(raw);
                // a row with an infinity or a NaN becomes NaN (every row, if the scale is one); the factor stays a number, so that a key which the
                // row does not see is -inf times it
                constexpr bool half = std::is_same<T, __half>::value;
                uint32_t top = 0;                         // the largest magnitude's bits, in the upper half
#pragma unroll
                for (int k = 0; k < CPT / 2; ++k) top = max(top, max(r[k] & 0x7fff0000u, (r[k] & 0x7fffu) << 16));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const bool finite = top < (half ? 0x7c000000u : 0x7f800000u) && fabsf(a.l2scale) <= FLT_MAX;
                if constexpr (half) {
#pragma unroll
                    for (int k = 0; k < CPT / 2; ++k) r[k] = finite ? r[k] : 0x7fff7fffu;
                } else {                                  // times 2^e so that the largest lies in [2^14, 2^15)
                    const int e = min(120, 14 - ((int)(top >> 23) - 127));
                    const float up = finite ? __int_as_float((e + 127) << 23) : NAN;
                    mine *= finite ? __int_as_float((127 - e) << 23) : 1.f;
#pragma unroll
                    for (int k = 0; k < CPT / 2; ++k) {
                        const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&r[k]);
                        r[k] = pack2<__half>(__low2float(v) * up, __high2float(v) * up);
                    }
                }
                mine = fminf(fmaxf(mine, FLT_MIN), FLT_MAX);      // (a masked score is -inf and has to stay it; scores this small are none)
                if (a.l2scale < 0.f) {                    // (the row's maximum is taken before the factor)
#pragma unroll
                    for (int k = 0; k < CPT / 2; ++k) r[k] ^= 0x80008000u;
                }
                if constexpr (NT == 1) {
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        q[k][0] = r[2 * k];
                        q[k][1] = r[2 * k + 1];
                    }
                } else if (warp == 0) {
#pragma unroll
                    for (int k = 0; k < KS / 2; ++k) q_smem[(n * (KS / 2) + k) * 32] = raw[k];
                }
                int mylim = INT_MAX;                      // (a row that is not there is never masked, nor stored)
                if (real) {
                    const int loc = a.loc[(size_t)f * a.loc_f + (size_t)u.w * a.loc_w + s_abs];
                    mylim = most_visible(a, loc, a.flen[f * a.len_f + u.w * a.len_w]);
                }
                lowest = min(lowest, mylim);
#pragma unroll
                for (int c = 0; c < 2; ++c) {             // row 2 t + c is lane 8 t + 4 c's
                    lim[n][c] = __shfl_sync(0xffffffffu, mylim, 8 * t + 4 * c);
                    factor[n][c] = __shfl_sync(0xffffffffu, mine, 8 * t + 4 * c);
                }
            }
#pragma unroll
            for (int k = 4; k < 32; k <<= 1) lowest = min(lowest, __shfl_xor_sync(0xffffffffu, lowest, k));
            if (NT == 2) __syncthreads();

            // row i of the product is key i with the last bit flipped in every second four: the loads of V then hit all banks
            const int ka = g ^ ((g >> 2) & 1), kb = ka + 8;
            const int flip = (t >> 1) & 1, v0 = 2 * t + flip, v1 = 2 * t + 1 - flip;
            const uint32_t k_at = ring_u32 + (HD == 128 ? ka * 64 + ((t ^ (ka & 2)) * 16) : ka * 32 + t * 8);
            const uint32_t ks_at = ring_u32 + C::OFF_KS + ka * C::SROW + t * (HD / 64);
            auto v_of = [&](int key) { return ring_u32 + C::OFF_V + key * C::ROW + (HD == 128 ? ((g >> 1) ^ (key & 2)) * 16 + (g & 1) * 8 : g * 4); };
            const uint32_t va_at = v_of(v0), vb_at = v_of(v1), vs_at = ring_u32 + C::OFF_VS + v0 * C::SROW + (HD == 128 ? g : g >> 1);
            const int vs_step = (v1 - v0) * C::SROW;
            uint32_t base = 0, base_ahead = (C::NSTAGE - 1) * C::STAGE;
            int k0 = b0 * C::TILE + warp * 16;
#pragma unroll 1
            for (int j = b0; j < b1; ++j, k0 += C::TILE) {
                cp_async_wait<C::NSTAGE - 2>();
                __syncwarp();                             // every lane's copies have landed, and every lane has left the last stage
                const int ahead = j + C::NSTAGE - 1;
                if (ahead < b1) {
                    fetch(ahead, base_ahead);
                    look_up(ahead + 1);
                } else {
                    cp_async_commit();
                }
                const uint32_t s = base;
                base_ahead = base;
                base = base == (C::NSTAGE - 1) * C::STAGE ? 0u : base + C::STAGE;
                if (k0 >= vis) continue;

                float c[NT][4];
                {
                    // one tile of rows: two chains of products, so that a step waits for the one before the last
                    float d[NT][4];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.f;
                        d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.f;
                    }
                    uint32_t wa[CPT / 8], wb[CPT / 8], sa, sb;
                    if constexpr (HD == 128) {
                        *reinterpret_cast<uint4*>(wa) = lds128<0>(k_at + s);
                        *reinterpret_cast<uint4*>(wb) = lds128<8 * C::ROW>(k_at + s);
                        sa = from_e4m3x2(lds16<0>(ks_at + s));
                        sb = from_e4m3x2(lds16<8 * C::SROW>(ks_at + s));
                    } else {
                        *reinterpret_cast<uint2*>(wa) = lds64<0>(k_at + s);
                        *reinterpret_cast<uint2*>(wb) = lds64<8 * C::ROW>(k_at + s);
                        sa = from_e4m3x2(lds8<0>(ks_at + s));
                        sb = from_e4m3x2(lds8<8 * C::SROW>(ks_at + s));
                    }
#pragma unroll
                    for (int k = 0; k < KS; k += 2) {     // a word of either key: two steps
                        const uint32_t ya = __byte_perm(sa, sa, k < KS / 2 || HD == 64 ? 0x1010 : 0x3232);
                        const uint32_t yb = __byte_perm(sb, sb, k < KS / 2 || HD == 64 ? 0x1010 : 0x3232);
                        uint32_t xa[4], xb[4];
                        from_e2m1x8(wa[k / 2], xa);
                        from_e2m1x8(wb[k / 2], xb);
                        uint4 qq[NT];
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if constexpr (NT == 1) qq[n] = make_uint4(q[k][0], q[k][1], q[k + 1][0], q[k + 1][1]);
                            else qq[n] = q_smem[(n * (KS / 2) + k / 2) * 32];
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t frag[4] = {mul_half2(xa[2 * h], ya), mul_half2(xb[2 * h], yb), mul_half2(xa[2 * h + 1], ya), mul_half2(xb[2 * h + 1], yb)};
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma_16816<__half>(NT == 1 && h ? d[n] : c[n], frag, h ? qq[n].z : qq[n].x, h ? qq[n].w : qq[n].y);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) c[n][i] += NT == 1 ? d[n][i] : 0.f;
                }
                const uint32_t bad = any_bad ? *reinterpret_cast<const uint32_t*>(ring + s + C::OFF_BAD) : 0u;
                const bool edge = k0 + 16 > lowest || bad != 0;
                if (edge) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int key = i < 2 ? ka : kb;
                            if (k0 + key >= lim[n][i & 1] || (bad >> key & 1)) c[n][i] = -INFINITY;
                        }
                }
                // (scores rounded in front of the difference: fused, the rounding of m would be what is left of scores beyond 2^27; and the
                // difference is compared, not m + 15, which from 2^24 on is rounded upwards)
                bool grow = false;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) c[n][i] = __fmul_rn(c[n][i], factor[n][i & 1]);
#pragma unroll
                    for (int i = 0; i < 2; ++i) grow = grow || fmaxf(c[n][i], c[n][i + 2]) - m[n][i] > kQ4RefAbove;
                }
                if (__any_sync(0xffffffffu, grow)) {      // (rare behind the first tiles) every row's reference follows its maximum so far
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float top = fmaxf(m[n][i], fmaxf(c[n][i], c[n][i + 2]) - kQ4RefBelow);
#pragma unroll
                            for (int k = 4; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
                            const float down = exp2_fast(m[n][i] - top);
                            m[n][i] = top;
                            l[n][i] *= down;
#pragma unroll
                            for (int k = 0; k < KS; ++k) {
                                o[n][k][i] *= down;
                                o[n][k][i + 2] *= down;
                            }
                        }
                }
                uint32_t pb[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) c[n][i] = exp2_fast(c[n][i] - m[n][i & 1]);
                    l[n][0] += c[n][0] + c[n][2];
                    l[n][1] += c[n][1] + c[n][3];
                    pb[n][0] = movmatrix(pack2<__half>(c[n][0], c[n][1]));
                    pb[n][1] = movmatrix(pack2<__half>(c[n][2], c[n][3]));
                }
                // ---- O^T += V^T P^T: columns of the product are keys 2 t, 2 t + 1 and eight further, in the order of the rows above ----
                {
                    uint32_t w[4][DPT / 8], sc[4];
                    if constexpr (HD == 128) {
                        *reinterpret_cast<uint2*>(w[0]) = lds64<0>(va_at + s);
                        *reinterpret_cast<uint2*>(w[1]) = lds64<0>(vb_at + s);
                        *reinterpret_cast<uint2*>(w[2]) = lds64<8 * C::ROW>(va_at + s);
                        *reinterpret_cast<uint2*>(w[3]) = lds64<8 * C::ROW>(vb_at + s);
                    } else {
                        w[0][0] = lds32<0>(va_at + s);
                        w[1][0] = lds32<0>(vb_at + s);
                        w[2][0] = lds32<8 * C::ROW>(va_at + s);
                        w[3][0] = lds32<8 * C::ROW>(vb_at + s);
                    }
                    sc[0] = lds8<0>(vs_at + s);
                    sc[1] = lds8<0>(vs_at + s + vs_step);
                    sc[2] = lds8<8 * C::SROW>(vs_at + s);
                    sc[3] = lds8<8 * C::SROW>(vs_at + s + vs_step);
                    if (edge) {
                        // a value that is not a number reaches the rows that see its key, and no others (0 * NaN would)
                        uint32_t odd = 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (is_nan_e4m3(sc[i])) {
                                odd |= 1u << ((i & 1 ? v1 : v0) + (i >> 1) * 8);
                                sc[i] = 0u;
                            }
                        if (__any_sync(0xffffffffu, odd != 0)) {
                            odd |= __shfl_xor_sync(0xffffffffu, odd, 1);
                            odd |= __shfl_xor_sync(0xffffffffu, odd, 2);
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int i = 0; i < 2; ++i) {
                                    const int seen = max(0, min(16, lim[n][i] - k0));
                                    if (odd & ((1u << seen) - 1u) & ~bad) {
#pragma unroll
                                        for (int k = 0; k < KS; ++k) o[n][k][i] = o[n][k][i + 2] = NAN;
                                    }
                                }
                        }
                    }
                    const uint32_t ya = from_e4m3x2(sc[0] | sc[1] << 8), yb = from_e4m3x2(sc[2] | sc[3] << 8);
#pragma unroll
                    for (int h = 0; h < DPT / 8; ++h) {
                        // byte k: channel 2 k of both keys (even), channel 2 k + 1 (odd)
                        uint32_t ae[4], ao[4], be[4], bo[4];
                        from_e2m1x8((w[0][h] & 0x0f0f0f0fu) | ((w[1][h] << 4) & 0xf0f0f0f0u), ae);
                        from_e2m1x8(((w[0][h] >> 4) & 0x0f0f0f0fu) | (w[1][h] & 0xf0f0f0f0u), ao);
                        from_e2m1x8((w[2][h] & 0x0f0f0f0fu) | ((w[3][h] << 4) & 0xf0f0f0f0u), be);
                        from_e2m1x8(((w[2][h] >> 4) & 0x0f0f0f0fu) | (w[3][h] & 0xf0f0f0f0u), bo);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t frag[4] = {mul_half2(ae[k], ya), mul_half2(ao[k], ya), mul_half2(be[k], yb), mul_half2(bo[k], yb)};
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma_16816<__half>(o[n][h * 4 + k], frag, pb[n][0], pb[n][1]);
                        }
                    }
                }
            }
            cp_async_wait<0>();
            __syncwarp();
        }

        // ---- the warps' results become one ----
        __syncthreads();                                  // (the fold lies on the rings)
        float* const fold = reinterpret_cast<float*>(smem_raw);
        float* const fold_m = fold + WARPS * 8 * NT * C::PITCH;
        float* const fold_l = fold_m + WARPS * 8 * NT;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float sum = l[n][i];
#pragma unroll
                for (int k = 4; k < 32; k <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
                const int row = warp * 8 * NT + n * 8 + 2 * t + i;
                float* dst = fold + row * C::PITCH + g * DPT;
#pragma unroll
                for (int k = 0; k < KS; k += 2)
                    *reinterpret_cast<float4*>(dst + 2 * k) = make_float4(o[n][k][i], o[n][k][i + 2], o[n][k + 1][i], o[n][k + 1][i + 2]);
                if (g == 0) {
                    fold_m[row] = m[n][i];
                    fold_l[row] = sum;
                }
            }
        __syncthreads();
        for (int i = tid; i < 8 * NT * (HD / 4); i += C::THREADS) {
            const int r = i / (HD / 4), col = (i - r * (HD / 4)) * 4;
            int s_abs, hq;
            if (!paged_row(a, u, r, &s_abs, &hq)) continue;
            float M = -FLT_MAX;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) M = fmaxf(M, fold_m[w * 8 * NT + r]);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            float L = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float wgt = exp2_fast(fold_m[w * 8 * NT + r] - M);
                const float4 v = *reinterpret_cast<const float4*>(fold + (w * 8 * NT + r) * C::PITCH + col);
                acc.x = fmaf(v.x, wgt, acc.x);
                acc.y = fmaf(v.y, wgt, acc.y);
                acc.z = fmaf(v.z, wgt, acc.z);
                acc.w = fmaf(v.w, wgt, acc.w);
                L = fmaf(fold_l[w * 8 * NT + r], wgt, L);
            }
            if (whole) {
                const float inv = L == 0.f ? 0.f : x.vunit / L;
                store4<T>(static_cast<T*>(a.out) + u.w * a.o_w + s_abs * a.o_s + hq * a.o_h + col, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
            } else {
                const size_t slot = (size_t)blockIdx.x + unit;            // (both only grow along the list)
                *reinterpret_cast<float4*>(a.ws_o + (slot * kFmaRows + r) * HD + col) = acc;
                if (col == 0) {
                    a.ws_m[slot * kFmaRows + r] = M;
                    a.ws_l[slot * kFmaRows + r] = L;
                }
            }
        }
        __syncthreads();
    }
}

// Adds up the partials of an output row, a lane four (two) columns.  WIDE: a CTA per row, warp w takes every fourth partial (few units have many
// partials each); otherwise a warp per row.  Units that one CTA had to itself are stored already; rows that see nothing, of which the list
// has no tile, are zeros.
template <class T, int HD, bool WIDE>
__global__ void __launch_bounds__(128) q4_mma_merge_kernel(const __grid_constant__ Q4MmaArgs x) {
    constexpr int VEC = HD / 32, STRIDE = WIDE ? 4 : 1;
    const PagedArgs& a = x.p;
    __shared__ float sm_m[4], sm_l[4], sm_o[WIDE ? 4 : 1][HD];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, unit = blockIdx.x, row = WIDE ? blockIdx.y : blockIdx.y * 4 + warp;
    const int per_group = a.Hkv * a.head_blocks, grp = unit / per_group;
    PagedUnit u;
    pdl_wait();
    pdl_trigger();
    const bool there = locate_unit(a, unit, &u);          // (its loads beside the plan's)
    const int before = __ldcg(x.plan + grp), n = __ldcg(x.plan + grp + 1) - before;
    const int64_t N = (int64_t)__ldcg(x.plan + a.groups_bound) * per_group;
    int first = 0, count = 0;
    if (n > 0) {
        const int64_t start = (int64_t)before * per_group + (int64_t)(unit - grp * per_group) * n;
        const int shares = effective_ctas(N, x.ctas);
        first = cta_of_tile(start + x.unit_cost, N, shares);
        count = cta_of_tile(start + n - 1, N, shares) - first + 1;
        if (count == 1) return;
    }
    int s_abs, hq;
    if (!there || !paged_row(a, u, row, &s_abs, &hq)) return;
    T* const out = static_cast<T*>(a.out) + u.w * a.o_w + s_abs * a.o_s + hq * a.o_h;
    float M = -FLT_MAX, L = 0.f, acc[VEC] = {};
    for (int p0 = WIDE ? warp : 0; p0 < count; p0 += 8 * STRIDE) {        // eight partials of a warp in flight
        float mp[8], lp[8], v[8][VEC];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const size_t at = ((size_t)(first + p0 + STRIDE * k) + unit) * kFmaRows + row;
            const bool have = p0 + STRIDE * k < count;
            mp[k] = have ? __ldcg(a.ws_m + at) : -FLT_MAX;
            lp[k] = have ? __ldcg(a.ws_l + at) : 0.f;
            if constexpr (VEC == 4) {
                const float4 y = have ? __ldcg(reinterpret_cast<const float4*>(a.ws_o + at * HD + lane * 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
                v[k][0] = y.x; v[k][1] = y.y; v[k][2] = y.z; v[k][3] = y.w;
            } else {
                const float2 y = have ? __ldcg(reinterpret_cast<const float2*>(a.ws_o + at * HD + lane * 2)) : make_float2(0.f, 0.f);
                v[k][0] = y.x; v[k][1] = y.y;
            }
        }
        float top = M;
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, mp[k]);
        const float down = exp2_fast(M - top);
        M = top;
        L *= down;
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] *= down;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float wgt = exp2_fast(mp[k] - top);
            L = fmaf(lp[k], wgt, L);
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] = fmaf(v[k][i], wgt, acc[i]);
        }
    }
    if constexpr (WIDE) {
        if (lane == 0) {
            sm_m[warp] = M;
            sm_l[warp] = L;
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) sm_o[warp][lane * VEC + i] = acc[i];
        __syncthreads();
        if (warp != 0) return;
        const float top = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
        L = 0.f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float wgt = exp2_fast(sm_m[w] - top);
            L = fmaf(sm_l[w], wgt, L);
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] = fmaf(sm_o[w][lane * VEC + i], wgt, acc[i]);
        }
    }
    const float inv = L == 0.f ? 0.f : x.vunit / L;
    if constexpr (VEC == 4) store4<T>(out + lane * 4, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    else *reinterpret_cast<uint32_t*>(out + lane * 2) = pack2<T>(acc[0] * inv, acc[1] * inv);
}

}  // namespace hogatt

// Pages of a paged cache: who holds which, on the device (step_blocks_kernel, compact_blocks_kernel), and copies of pages in all of a
// model's caches at once (copy_pages_kernel).  refs[p] is the number of block-table entries that name page p, plus what the
// caller adds to keep a page; a page with refs[p] == 0 is free.  There is no list of free pages to keep consistent: pages are given out
// lowest first, found by counting the zeros of refs.
//
// Both bookkeeping kernels are one thread-block cluster each: phases that need all of the previous one's results are separated by the
// cluster's hardware barrier instead of by launches, and eight SMs read the few hundred KB of refs and tables at once.  Nothing depends
// on the order of atomics: sums of integers, and pages are dealt by rank.  What one phase writes and another reads goes through
// L2 (__ldcg).
#pragma once
#include "hogatt_device.cuh"
#include "hogatt_q4.cuh"

namespace hogatt {

constexpr int kBlocksCluster = 8, kBlocksThreads = 1024;

// this CTA's share [begin, end) of `n` things
__device__ __forceinline__ void cluster_share(int n, int* begin, int* end) {
    const int rank = cluster_ctarank(), ctas = cluster_nctarank();
    *begin = (int)((int64_t)n * rank / ctas);
    *end = (int)((int64_t)n * (rank + 1) / ctas);
}

struct StepBlocksArgs {
    int num_blocks, block_size, max_blocks, rows_in, rows_out;
    const int* refs_in;
    const int* table_in;          // [rows_in, max_blocks]
    const int* lengths_in;        // [rows_in]
    const int* source;            // [rows_out] or nullptr: every row stays
    const int* new_tokens;        // [rows_out] or nullptr: none
    int* refs_out;
    int* table_out;               // [rows_out, max_blocks]
    int* lengths_out;             // [rows_out]
    int* room;                    // [rows_out]
    int* ws;                      // StepBlocksWs
    int* status;
};
// Workspace, ints: [0] copies listed, [1 .. 8] free pages per CTA, [16 + 3 w] pages of row w that are kept x 2 + takes a copy, its last page,
// pages that rows before it need (INT_MAX: that or more); behind them one entry more of the last kind (the total); then the list of copies (from, to).
constexpr int kStepHead = 16;
__host__ __device__ inline int64_t step_blocks_pairs(int64_t rows) { return kStepHead + 3 * (rows + 1); }
__host__ __device__ inline int64_t step_blocks_ints(int64_t rows) { return step_blocks_pairs(rows) + 2 * rows; }

struct StepRow {
    int length, kept, want, add;  // tokens; pages of them; pages with the new tokens; new tokens
    int from;                     // row of the old table, -1: none
    bool over;
};
__device__ __forceinline__ StepRow step_row(const StepBlocksArgs& a, int w) {
    StepRow r;
    r.from = a.source ? a.source[w] : w;
    const bool bad = r.from >= a.rows_in;
    if (bad || r.from < 0) r.from = -1;
    r.length = r.from >= 0 ? max(0, __ldcg(a.lengths_in + r.from)) : 0;
    r.add = a.new_tokens ? max(0, a.new_tokens[w]) : 0;
    // (a length and a block size are below 2^31: the sum fits 32 bits without sign; with new tokens it may not)
    const uint32_t bs = (uint32_t)a.block_size;
    const int64_t kept = ((uint32_t)r.length + bs - 1) / bs, all = (int64_t)r.length + r.add + bs - 1;
    const int64_t want = all >> 32 ? all / bs : (int64_t)((uint32_t)all / bs);
    r.kept = (int)min(kept, (int64_t)a.max_blocks);
    r.over = bad || kept > a.max_blocks || want > a.max_blocks;
    r.want = r.over ? r.kept : (int)want;
    return r;
}

// grid = one cluster
__global__ void __launch_bounds__(kBlocksThreads, 1) step_blocks_kernel(const __grid_constant__ StepBlocksArgs a) {
    const int rank = cluster_ctarank(), ctas = cluster_nctarank(), tid = threadIdx.x;
    const int64_t gtid = (int64_t)rank * kBlocksThreads + tid, gthreads = (int64_t)ctas * kBlocksThreads;
    int* const rows_ws = a.ws + kStepHead;
    int* const pairs = a.ws + step_blocks_pairs(a.rows_out);
    pdl_wait();
    pdl_trigger();
    int begin, end;
    cluster_share(a.num_blocks, &begin, &end);
    int flags = 0;

    // ---- 1: the rows as they are taken over, and what that does to the pages' counts ----
    if (a.refs_out != a.refs_in)
        for (int p = begin + tid; p < end; p += kBlocksThreads) a.refs_out[p] = a.refs_in[p];
    if (gtid == 0) a.ws[0] = 0;
    cluster_sync_all();
    if (a.source)
        for (int64_t i = gtid; i < (int64_t)a.rows_in * a.max_blocks; i += gthreads) {
            const int p = a.table_in[i];
            if (p >= 0 && p < a.num_blocks) atomicAdd(a.refs_out + p, -1);
        }
    // (a warp takes 128 entries of a row at a time: what the row is, once for all of them)
    const int pieces = (a.max_blocks + 127) / 128;
    for (int64_t i = gtid >> 5; i < (int64_t)a.rows_out * pieces; i += gthreads >> 5) {
        const int w = (int)floor_div(i, pieces), c0 = (int)(i - (int64_t)w * pieces) * 128 + (tid & 31);
        const int64_t row = (int64_t)w * a.max_blocks;
        const int from = a.source ? a.source[w] : w;
        int p[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            p[k] = from >= 0 && from < a.rows_in && c0 + 32 * k < a.max_blocks ? a.table_in[(int64_t)from * a.max_blocks + c0 + 32 * k] : -1;
        const StepRow r = step_row(a, w);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int c = c0 + 32 * k;
            if (c >= a.max_blocks) break;
            const bool there = p[k] >= 0 && p[k] < a.num_blocks, kept = c < r.kept;
            if (kept && !there) flags |= STATUS_BAD_BLOCK;
            if (a.source) {
                if (kept && there) atomicAdd(a.refs_out + p[k], 1);
            } else if (!kept && there) {
                atomicAdd(a.refs_out + p[k], -1);
            }
            a.table_out[row + c] = kept && there ? p[k] : -1;
        }
    }
    cluster_sync_all();

    // ---- 2: what every row needs (CTA 0), free pages of every share ----
    __shared__ __align__(16) int last_of[kBlocksThreads];
    if (rank == 0) {
        // (65,536 rows may ask for more pages than 32 bits count; more than the pool has is all the same)
        int64_t before = 0;
        for (int w0 = 0; w0 < a.rows_out; w0 += kBlocksThreads) {
            const int w = w0 + tid;
            StepRow r = {};
            int last = -1;
            if (w < a.rows_out) {
                r = step_row(a, w);
                if (r.over) flags |= STATUS_TABLE_FULL;
                if (!r.over && r.add > 0 && r.length % a.block_size != 0) last = __ldcg(a.table_out + (int64_t)w * a.max_blocks + r.kept - 1);
                __stcg(rows_ws + 3 * w + 1, last);
            }
            __syncthreads();                              // (the last chunk's have been read)
            last_of[tid] = last;
            __syncthreads();
            // a last page that is partly filled and shared: its writers take copies in row order while others still hold it
            bool copy = false;
            if (last >= 0) {
                const int holders = __ldcg(a.refs_out + last);
                if (holders > 1) {
                    int earlier = 0, v = 0;
                    for (; v + 3 < tid; v += 4) {
                        const int4 x = *reinterpret_cast<const int4*>(last_of + v);
                        earlier += (x.x == last) + (x.y == last) + (x.z == last) + (x.w == last);
                    }
                    for (; v < tid; ++v) earlier += last_of[v] == last;
#pragma unroll 8
                    for (v = 0; v < w0; ++v) earlier += __ldcg(rows_ws + 3 * v + 1) == last;
                    copy = holders - earlier > 1;
                }
            }
            const int need = w < a.rows_out ? r.want - r.kept + copy : 0;
            int64_t total;
            const int64_t at = block_exclusive((int64_t)need, &total);
            if (w < a.rows_out) {
                __stcg(rows_ws + 3 * w, r.kept * 2 + copy);
                __stcg(rows_ws + 3 * w + 2, (int)min(before + at, (int64_t)INT_MAX));
            }
            before += total;
        }
        if (tid == 0) __stcg(rows_ws + 3 * a.rows_out + 2, (int)min(before, (int64_t)INT_MAX));
    }
    int mine = 0;
    for (int p = begin + tid; p < end; p += kBlocksThreads) mine += __ldcg(a.refs_out + p) == 0;
    int free_here;
    block_exclusive(mine, &free_here);
    if (tid == 0) __stcg(a.ws + 1 + rank, free_here);
    cluster_sync_all();

    // ---- 3: free page number k, lowest first, goes to whoever needs the k-th ----
    int free_all = 0, base = 0;
    for (int i = 0; i < ctas; ++i) {
        const int n = __ldcg(a.ws + 1 + i);
        if (i < rank) base += n;
        free_all += n;
    }
    const int needed = __ldcg(rows_ws + 3 * a.rows_out + 2);
    for (int p0 = begin; p0 < end && base < needed; p0 += kBlocksThreads) {
        const int p = p0 + tid;
        const bool unused = p < end && __ldcg(a.refs_out + p) == 0;
        int total;
        const int k = base + block_exclusive((int)unused, &total);
        base += total;
        if (!unused || k >= needed) continue;
        int lo = 0, hi = a.rows_out;                      // the row: the last one whose predecessors need at most k
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (__ldcg(rows_ws + 3 * mid + 2) <= k) lo = mid;
            else hi = mid;
        }
        // (rows are served in order until one cannot be; from there on none is)
        if (__ldcg(rows_ws + 3 * (lo + 1) + 2) > free_all) continue;
        const int what = __ldcg(rows_ws + 3 * lo), kept = what >> 1, copy = what & 1, o = k - __ldcg(rows_ws + 3 * lo + 2);
        a.refs_out[p] = 1;
        if (copy && o == 0) {
            const int from = __ldcg(rows_ws + 3 * lo + 1);
            atomicAdd(a.refs_out + from, -1);             // (at least one holder is left: the page does not become free)
            const int at = atomicAdd(a.ws, 1);
            pairs[2 * at] = from;
            pairs[2 * at + 1] = p;
            a.table_out[(int64_t)lo * a.max_blocks + kept - 1] = p;
        } else {
            a.table_out[(int64_t)lo * a.max_blocks + kept + o - copy] = p;
        }
    }
    for (int64_t w = gtid; w < a.rows_out; w += gthreads) {
        const StepRow r = step_row(a, (int)w);
        const bool served = __ldcg(rows_ws + 3 * (w + 1) + 2) <= free_all && !r.over;
        if (!served && !r.over && r.add > 0) flags |= STATUS_NO_BLOCKS;
        a.room[w] = served ? r.add : 0;
        a.lengths_out[w] = r.length;                      // (in place too: a length below zero is none)
    }
    if (flags && a.status) atomicOr(a.status, flags);
}

struct CompactBlocksArgs {
    int num_blocks;
    int64_t entries;              // of the block table
    const int* refs_in;
    const int* table_in;
    int* refs_out;
    int* table_out;
    int* moved;                   // [num_blocks]: the page's new number, -1 for a free one
    int* ws;                      // CompactBlocksWs
    int* status;
};
// Workspace, ints: [0] moves, [1 .. 24] per CTA: live pages, free ones in front, live ones behind; then the moves (from, to).
constexpr int kCompactHead = 32;
__host__ __device__ inline int64_t compact_blocks_ints(int64_t blocks) { return kCompactHead + 2 * (blocks / 2 + 1); }

// n live pages: the k-th live page at or behind place n (lowest first) goes to the k-th free place in front of it.  No page is both, so
// the copies can run in any order.
__global__ void __launch_bounds__(kBlocksThreads, 1) compact_blocks_kernel(const __grid_constant__ CompactBlocksArgs a) {
    const int rank = cluster_ctarank(), ctas = cluster_nctarank(), tid = threadIdx.x;
    const int64_t gtid = (int64_t)rank * kBlocksThreads + tid, gthreads = (int64_t)ctas * kBlocksThreads;
    int* const pairs = a.ws + kCompactHead;
    pdl_wait();
    pdl_trigger();
    int begin, end, n = 0;
    cluster_share(a.num_blocks, &begin, &end);
    {
        int mine = 0, total;
        for (int p = begin + tid; p < end; p += kBlocksThreads) mine += a.refs_in[p] != 0;
        block_exclusive(mine, &total);
        if (tid == 0) __stcg(a.ws + 1 + rank, total);
    }
    cluster_sync_all();
    for (int i = 0; i < ctas; ++i) n += __ldcg(a.ws + 1 + i);
    {
        int holes = 0, movers = 0, h, m;
        for (int p = begin + tid; p < end; p += kBlocksThreads) {
            holes += p < n && a.refs_in[p] == 0;
            movers += p >= n && a.refs_in[p] != 0;
        }
        block_exclusive(holes, &h);
        block_exclusive(movers, &m);
        if (tid == 0) {
            __stcg(a.ws + 1 + kBlocksCluster + rank, h);
            __stcg(a.ws + 1 + 2 * kBlocksCluster + rank, m);
        }
    }
    cluster_sync_all();
    int hole = 0, mover = 0, moves = 0;
    for (int i = 0; i < ctas; ++i) {
        const int h = __ldcg(a.ws + 1 + kBlocksCluster + i), m = __ldcg(a.ws + 1 + 2 * kBlocksCluster + i);
        if (i < rank) {
            hole += h;
            mover += m;
        }
        moves += h;
    }
    for (int p0 = begin; p0 < end; p0 += kBlocksThreads) {
        const int p = p0 + tid;
        const int refs = p < end ? a.refs_in[p] : 0;
        const bool is_hole = p < end && p < n && refs == 0, is_mover = p < end && p >= n && refs != 0;
        int th, tm;
        const int h = hole + block_exclusive((int)is_hole, &th), m = mover + block_exclusive((int)is_mover, &tm);
        hole += th;
        mover += tm;
        if (is_hole) __stcg(pairs + 2 * h + 1, p);
        if (is_mover) __stcg(pairs + 2 * m, p);
        if (p < end) {
            if (!is_mover) a.moved[p] = refs != 0 ? p : -1;
            if (!is_hole && !is_mover && a.refs_out != a.refs_in) a.refs_out[p] = refs;
        }
    }
    cluster_sync_all();
    for (int64_t k = gtid; k < moves; k += gthreads) {
        const int from = __ldcg(pairs + 2 * k), to = __ldcg(pairs + 2 * k + 1);
        const int refs = __ldcg(a.refs_in + from);
        a.refs_out[to] = refs;
        a.refs_out[from] = 0;
        a.moved[from] = to;
    }
    if (gtid == 0) a.ws[0] = moves;
    cluster_sync_all();
    bool bad = false;
    for (int64_t i = gtid; i < a.entries; i += gthreads) {
        const int p = a.table_in[i];
        const bool there = p >= 0 && p < a.num_blocks;
        const int to = there ? __ldcg(a.moved + p) : -1;
        bad |= p >= 0 && to < 0;                          // (a page that is not there, or free)
        a.table_out[i] = to;
    }
    if (bad && a.status) atomicOr(a.status, STATUS_BAD_BLOCK);
}

// ---- copies ---------------------------------------------------------------------------------------------------------------
constexpr int kMaxPageTensors = 128;      // per launch: the table travels in the kernel arguments
constexpr int kPagePiece = 4096;          // bytes a warp copies at a time: eight 16-byte loads of every lane in flight
struct PageTensor {
    char* base;
    int64_t bytes;                // of a page
    int first;                    // pieces of a page in the tensors before this one
    int vectorised;               // base and bytes are multiples of 16
};
struct CopyPagesArgs {
    int n, pieces;                // tensors; pieces of a page in all of them
    const int* count;             // device
    const int* pairs;             // (from, to)
    PageTensor t[kMaxPageTensors];
};
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CopyPagesArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5);
    pdl_wait();
    pdl_trigger();
    const int64_t items = (int64_t)__ldcg(a.count) * a.pieces;
    for (int64_t i = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < items; i += warps) {
        const int64_t k = floor_div(i, a.pieces);
        const int piece = (int)(i - k * a.pieces);
        int lo = 0, hi = a.n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.t[mid].first <= piece) lo = mid;
            else hi = mid;
        }
        const PageTensor& t = a.t[lo];
        const int64_t at = (int64_t)(piece - t.first) * kPagePiece;
        const int n = (int)min((int64_t)kPagePiece, t.bytes - at);
        const char* src = t.base + (int64_t)__ldcg(a.pairs + 2 * k) * t.bytes + at;
        char* dst = t.base + (int64_t)__ldcg(a.pairs + 2 * k + 1) * t.bytes + at;
        if (t.vectorised) {
            int4 v[kPagePiece / 512];
#pragma unroll
            for (int j = 0; j < kPagePiece / 512; ++j)
                if (j * 512 + lane * 16 < n) v[j] = load_16(src + j * 512 + lane * 16);
#pragma unroll
            for (int j = 0; j < kPagePiece / 512; ++j)
                if (j * 512 + lane * 16 < n) *reinterpret_cast<int4*>(dst + j * 512 + lane * 16) = v[j];
        } else {
            for (int j = lane; j < n; j += 32) dst[j] = src[j];
        }
    }
}

}  // namespace hogatt

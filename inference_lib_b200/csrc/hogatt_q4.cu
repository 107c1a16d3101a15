// C ABI of the 4-bit paged cache and of page bookkeeping (declared in include/hogatt.h): argument validation, kernel choice, workspace
// carving and launches, like hogatt_api.cu.
#include <limits.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <type_traits>

#include "hogatt_host.h"
#include "hogatt_blocks.cuh"
#include "hogatt_q4.cuh"
#include "hogatt_q4_mma.cuh"
#include "hogatt_q4_dense.cuh"

namespace hogatt {
namespace {

// A power of two far enough from the ends of fp32 that a scale times it, and six times it, are normal numbers.
bool unit_ok(float u) {
    int e;
    return u > 0.f && std::isfinite(u) && std::frexp(u, &e) == 0.5f && e >= -63 && e <= 65;
}

FastDiv fast_div_by(uint32_t d) {
    uint32_t shift = 0;
    while (shift < 32 && ((uint64_t)1 << shift) < d) ++shift;
    return {(uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1), shift, d};
}

int cache_shape(int Hkv, int E, int Ev, int block_size, int max_blocks, int num_blocks, int dtype) {
    if (Hkv <= 0 || E <= 0 || Ev <= 0 || block_size <= 0 || max_blocks <= 0 || num_blocks <= 0) return HOGATT_ERR_BAD_SHAPE;
    if (Hkv > 65535) return HOGATT_ERR_TOO_LARGE;
    if (dtype != HOGATT_F32 && dtype != HOGATT_F16 && dtype != HOGATT_BF16) return HOGATT_ERR_UNSUPPORTED_DTYPE;
    if (E % kGroup != 0 || Ev % kGroup != 0 || E > 256 || Ev > 256) return HOGATT_ERR_UNSUPPORTED_HEAD_DIM;
    return HOGATT_OK;
}

// The tcgen05 kernel's workspace for packed queries: the plan, then one slot of 256 rows per (CTA, unit) pair that can meet.
struct DenseLayout {
    size_t pre, cost, vis, start, merge, fold, rec, o, m, l, total;
};
DenseLayout carve_dense_plan(int64_t blocks, int Hkv, int F, int grid) {
    const size_t slots = (size_t)grid + (size_t)blocks * Hkv;
    DenseLayout w;
    w.pre = 256;
    w.cost = w.pre + align_up((size_t)(blocks + 1) * sizeof(long long), 256);
    w.vis = w.cost + align_up((size_t)(blocks + 1) * sizeof(long long), 256);
    w.start = w.vis + align_up((size_t)blocks * 2 * F * sizeof(int), 256);
    w.merge = w.start + align_up((size_t)grid * sizeof(int4), 256);
    w.fold = w.merge + align_up((size_t)blocks * Hkv * sizeof(int4), 256);
    w.rec = w.fold + align_up((size_t)blocks * Hkv * kDenseFoldInts * sizeof(int), 256);
    w.o = w.rec + align_up((size_t)blocks * sizeof(int4), 256);
    w.m = w.o + slots * kDenseBlock * 128 * sizeof(float);
    w.l = w.m + align_up(slots * kDenseBlock * sizeof(float), 256);
    w.total = w.l + align_up(slots * kDenseBlock * sizeof(float), 256);
    return w;
}

struct Q4Plan {
    int kernel;                     // HOGATT_KERNEL_FMA or HOGATT_KERNEL_MMA
    int tokens_per_group, head_blocks, groups_bound, units, splits;
    int rows;                       // (MMA) query rows of a unit at most
    int ctas;                       // (MMA) shares of the list of tiles; 0: a CTA per unit
    int unit_cost;                  // (MMA) what a unit counts for in the list beside its tiles
    bool small;                     // (MMA) CTAs of four warps
    size_t o, m, l, plan, total;
    int tokens, blocks;             // (DENSE) query tokens per tile, blocks per kv head at most
    DenseLayout w;                  // (DENSE) its workspace
    size_t queries, factor;
};

// What scores are multiplied with: the products of queries and of what the codes and scales alone stand for.
float score_factor(const hogatt_paged_q4_problem* x) { return (float)((double)x->paged.scale * 1.4426950408889634 * x->key_unit); }

// Packed queries on the tcgen05 kernel: head size 128, blocks of a multiple of eight rows.  The factor of the scores lies where neither it nor 8 / factor
// leaves fp32, not even times the power of two, 2^-120 to 2^113, that a row of bf16 queries is scaled by (clamped at 1e-36).
bool dense_eligible(const hogatt_paged_q4_problem* x) {
    const hogatt_paged_problem* p = &x->paged;
    const float factor = score_factor(x);
    return p->cu_seqlens_q != nullptr && (p->dtype == HOGATT_F16 || p->dtype == HOGATT_BF16) && p->E == 128 && p->Ev == 128 && p->block_size % 8 == 0 &&
           p->Hq / p->Hkv <= kDenseRows && (int64_t)p->num_blocks * p->Hkv * p->block_size < ((int64_t)1 << 31) &&
           (int64_t)p->total_q_tokens * p->Hq * p->F < ((int64_t)1 << 31) && factor >= 1e-30f && factor <= 8192.f;
}
// AUTO takes it where the tokens beyond one per sequence, over as many keys as the block table has room for, would keep the other
// kernel busy for long (as for 16-bit pages).
bool dense_wanted(const hogatt_paged_problem* p) {
    if (dense_disabled() || paged_mma_disabled()) return false;
    const int64_t tokens = (int64_t)p->total_q_tokens - p->W;
    if (tokens * (p->Hq / p->Hkv) < kDenseRows || tokens * p->Hq < 8 * kDenseRows) return false;
    return (double)tokens * p->Hq * p->max_blocks_per_seq * p->block_size >= 4.5e6;
}

int plan_q4(const hogatt_paged_q4_problem* x, int sms, Q4Plan* pl) {
    if (x == nullptr) return HOGATT_ERR_NULL_POINTER;
    const hogatt_paged_problem* p = &x->paged;
    const bool packed = p->cu_seqlens_q != nullptr;
    if (p->F <= 0 || p->W <= 0 || p->Hq <= 0 || p->Hkv <= 0 || p->Hq % p->Hkv != 0 || (packed ? p->total_q_tokens < 0 : p->S <= 0))
        return HOGATT_ERR_BAD_SHAPE;
    if (const int rc = cache_shape(p->Hkv, p->E, p->Ev, p->block_size, p->max_blocks_per_seq, p->num_blocks, p->dtype)) return rc;
    if (p->Ev != 32 && p->Ev != 64 && p->Ev != 128 && p->Ev != 256) return HOGATT_ERR_UNSUPPORTED_HEAD_DIM;
    if (p->F > 4096) return HOGATT_ERR_TOO_MANY_FRAGMENTS;
    const bool mma = p->dtype != HOGATT_F32 && p->E == p->Ev && (p->E == 64 || p->E == 128);
    const bool dense = dense_eligible(x);
    if (p->kernel != HOGATT_KERNEL_AUTO && p->kernel != HOGATT_KERNEL_FMA && !(p->kernel == HOGATT_KERNEL_MMA && mma) &&
        !(p->kernel == HOGATT_KERNEL_DENSE && dense))
        return HOGATT_ERR_BAD_KERNEL_CHOICE;
    pl->kernel = mma && (p->kernel == HOGATT_KERNEL_MMA || (p->kernel == HOGATT_KERNEL_AUTO && !paged_mma_disabled())) ? HOGATT_KERNEL_MMA : HOGATT_KERNEL_FMA;
    if (dense && (p->kernel == HOGATT_KERNEL_DENSE || (p->kernel == HOGATT_KERNEL_AUTO && dense_wanted(p)))) pl->kernel = HOGATT_KERNEL_DENSE;
    if (!packed && (int64_t)p->F * p->W * p->S >= ((int64_t)1 << 31)) return HOGATT_ERR_TOO_LARGE;
    if (packed && (int64_t)p->F * std::max(p->total_q_tokens, p->W) >= ((int64_t)1 << 31)) return HOGATT_ERR_TOO_LARGE;
    const int G = p->Hq / p->Hkv, most = G >= 16 ? 1 : 16 / G;
    if (pl->kernel == HOGATT_KERNEL_DENSE) {
        pl->tokens = kDenseRows / G;
        const int64_t blocks = (int64_t)p->total_q_tokens / (2 * pl->tokens) + p->W;
        if (blocks * p->Hkv > (1 << 24)) return HOGATT_ERR_TOO_LARGE;
        pl->blocks = (int)blocks;
        pl->ctas = std::min(sms, kDenseMaxCtas);
        pl->w = carve_dense_plan(pl->blocks, p->Hkv, p->F, pl->ctas);
        pl->queries = pl->w.total;
        const size_t rows = (size_t)p->total_q_tokens * p->Hq * p->F;
        pl->factor = pl->queries + (p->dtype == HOGATT_BF16 ? align_up(rows * 128 * sizeof(__half), 256) : 0);
        pl->total = pl->factor + align_up(rows * sizeof(float), 256);
        return HOGATT_OK;
    }
    // (tokens that a sequence is likely to have: a group of more would be empty rows; one of fewer is another reader of the same keys)
    const int64_t tokens = packed ? ((int64_t)p->total_q_tokens + p->W - 1) / p->W : p->S;
    pl->tokens_per_group = pl->kernel == HOGATT_KERNEL_MMA ? (int)std::max<int64_t>(1, std::min<int64_t>(most, tokens)) : most;
    pl->head_blocks = (G + 15) / 16;
    pl->rows = std::min(G, 16) * pl->tokens_per_group;
    const int64_t groups = packed ? ((int64_t)p->total_q_tokens + pl->tokens_per_group - 1) / pl->tokens_per_group + p->W
                                  : (int64_t)p->W * ((p->S + pl->tokens_per_group - 1) / pl->tokens_per_group);
    const int64_t units = groups * pl->head_blocks * p->Hkv;
    if (units > (1 << 24)) return HOGATT_ERR_TOO_LARGE;
    pl->groups_bound = (int)groups;
    pl->units = (int)std::max<int64_t>(units, 1);
    // tiles are counted in 32 bits, a unit's where it has a CTA to itself, otherwise all units'
    const int64_t keys = std::min<int64_t>((int64_t)p->max_blocks_per_seq * p->block_size + 1, INT_MAX), tiles = p->F * (keys / 32 + 1) + 16;
    size_t slots;
    if (pl->kernel == HOGATT_KERNEL_MMA) {
        pl->splits = 0;
        // With at least as many units as resident CTAs each gets one to itself: shares of the list would hold ends of units (the warps' fold, the next
        // unit's first copies), which do not overlap inside a CTA, and the merge step is saved.  us per call with shares / without, 8 kv heads
        // of 5 heads: 24 sequences of 6,000 keys 53.5 / 57.9, 37 of them 65.0 / 58.5, 46 of 2,000 keys 46.0 / 40.0 (40 of 6,000 79 / 93: the second
        // round of CTAs is short there).
        const int64_t likely = (packed ? std::max<int64_t>(p->W, p->total_q_tokens / pl->tokens_per_group) : groups) * pl->head_blocks * p->Hkv;
        // CTAs of four warps, twice as many resident, from three times as many units: a long unit takes them twice as long, which shows where lengths
        // differ.  us with eight / four: 200 sequences of 1,000 keys 88 / 67, 148 of 200 keys 35.8 / 22.5; from 6,000 keys down in equal steps 64 of them
        // 60 / 101, 100 of them 93 / 101, 120 of 5,100 down 98 / 90.
        // What a unit costs beside its tiles (the fold, the first copies), in tiles: us with 0 / 2 / 4 / 6, 24 sequences of 6,000 keys down to 1,331
        // 44.0 / 42.2 / 40.7 / 41.6, 30 of 4,000 down to 230 49.1 / 36.7 / 34.9 / 36.3, 20 of 1,500 down to 740 23.5 / 22.9 / 22.7 / 23.4.  Few units have hardly
        // any ends in a share, but a tile more in it would show.
        pl->ctas = likely >= kQ4Ctas * sms ? 0 : kQ4Ctas * sms;
        pl->small = likely >= 3 * kQ4Ctas * sms;
        pl->unit_cost = 2 * likely > pl->ctas ? 4 : 0;
        if (tiles > INT_MAX / (pl->ctas ? groups : 1)) return HOGATT_ERR_TOO_LARGE;
        slots = pl->ctas ? ((size_t)pl->units + pl->ctas) * kFmaRows : 0;
    } else {
        pl->ctas = 0;
        pl->splits = std::max(1, std::min(24, (3 * sms + pl->units - 1) / pl->units));      // (24: the merge step's one round trip)
        slots = (size_t)pl->units * pl->splits * kFmaRows;
        if (tiles > INT_MAX) return HOGATT_ERR_TOO_LARGE;
    }
    pl->o = 0;
    pl->m = pl->o + align_up(slots * p->Ev * sizeof(float), 256);
    pl->l = pl->m + align_up(slots * sizeof(float), 256);
    pl->plan = pl->l + align_up(slots * sizeof(float), 256);
    pl->total = pl->plan + align_up(((size_t)pl->groups_bound + 1) * sizeof(int), 256);
    return HOGATT_OK;
}

template <class T, int HD, int NT, bool ALIGNED, int WARPS>
int launch_q4_mma(const Q4MmaArgs& x, const Q4Plan& pl, int dev, int smem_optin, cudaStream_t stream) {
    static std::atomic<size_t> granted[kMaxDevices];
    const size_t smem = q4_mma_smem_bytes<HD, WARPS>(NT, x.p.W, pl.groups_bound, x.ctas > 0);
    if (smem > (size_t)smem_optin) return HOGATT_ERR_TOO_LARGE;
    const int rc = ensure_smem_limit(q4_mma_kernel<T, HD, NT, ALIGNED, WARPS>, dev, smem, granted);
    if (rc != HOGATT_OK) return rc;
    HOGATT_CUDA_OK(launch_kernel(q4_mma_kernel<T, HD, NT, ALIGNED, WARPS>, dim3(x.ctas ? x.ctas : pl.units), dim3(WARPS * 32), smem, stream, x));
    if (!x.ctas) return HOGATT_OK;
    // a unit's partials: about ctas / units and one more at either end
    if (x.ctas / pl.units + 2 > 8) HOGATT_CUDA_OK(launch_kernel(q4_mma_merge_kernel<T, HD, true>, dim3(pl.units, pl.rows), dim3(128), 0, stream, x));
    else HOGATT_CUDA_OK(launch_kernel(q4_mma_merge_kernel<T, HD, false>, dim3(pl.units, (pl.rows + 3) / 4), dim3(128), 0, stream, x));
    return HOGATT_OK;
}
template <class T, int HD, int NT>
int launch_q4_mma_blocks(const Q4MmaArgs& x, const Q4Plan& pl, int dev, int smem_optin, cudaStream_t stream) {
    if (x.p.block_size % 16 == 0)
        return pl.small ? launch_q4_mma<T, HD, NT, true, 4>(x, pl, dev, smem_optin, stream) : launch_q4_mma<T, HD, NT, true, 8>(x, pl, dev, smem_optin, stream);
    return pl.small ? launch_q4_mma<T, HD, NT, false, 4>(x, pl, dev, smem_optin, stream) : launch_q4_mma<T, HD, NT, false, 8>(x, pl, dev, smem_optin, stream);
}
template <class T, int HD>
int launch_q4_mma_rows(const Q4MmaArgs& x, const Q4Plan& pl, int dev, int smem_optin, cudaStream_t stream) {
    return pl.rows <= 8 ? launch_q4_mma_blocks<T, HD, 1>(x, pl, dev, smem_optin, stream) : launch_q4_mma_blocks<T, HD, 2>(x, pl, dev, smem_optin, stream);
}

template <class T>
int launch_q4_merge(const Q4Args& x, const Q4Plan& pl, cudaStream_t stream) {
    HOGATT_CUDA_OK(launch_kernel(q4_merge_kernel<T>, dim3(pl.units, kFmaRows / kMergeWarps), dim3(kMergeWarps * 32), 0, stream, x.p));
    return HOGATT_OK;
}

template <class T, int EV>
int launch_q4_fma(const Q4Args& x, const Q4Plan& pl, int dev, int smem_optin, cudaStream_t stream) {
    static std::atomic<size_t> granted[kMaxDevices];
    const size_t smem = q4_smem_bytes(x.p.E, EV, x.p.F);
    if (smem > (size_t)smem_optin) return HOGATT_ERR_TOO_MANY_FRAGMENTS;
    const int rc = ensure_smem_limit(q4_attention_kernel<T, EV>, dev, smem, granted);
    if (rc != HOGATT_OK) return rc;
    HOGATT_CUDA_OK(launch_kernel(q4_attention_kernel<T, EV>, dim3(pl.units, pl.splits), dim3(kFmaThreads), smem, stream, x));
    return launch_q4_merge<T>(x, pl, stream);
}

template <class T>
int launch_q4(const Q4Args& x, const Q4Plan& pl, int dev, int smem_optin, cudaStream_t stream) {
    if constexpr (!std::is_same<T, float>::value) {
        if (pl.kernel == HOGATT_KERNEL_MMA) {
            Q4MmaArgs y;
            y.p = x.p;
            y.kscale = x.kscale; y.vscale = x.vscale; y.num_blocks = x.num_blocks; y.vunit = x.vunit;
            y.block = fast_div_by((uint32_t)x.p.block_size);
            y.ctas = pl.ctas;
            y.unit_cost = pl.unit_cost;
            y.plan = x.plan;
            return x.p.E == 128 ? launch_q4_mma_rows<T, 128>(y, pl, dev, smem_optin, stream) : launch_q4_mma_rows<T, 64>(y, pl, dev, smem_optin, stream);
        }
    }
    switch (x.p.Ev) {
        case 32: return launch_q4_fma<T, 32>(x, pl, dev, smem_optin, stream);
        case 64: return launch_q4_fma<T, 64>(x, pl, dev, smem_optin, stream);
        case 128: return launch_q4_fma<T, 128>(x, pl, dev, smem_optin, stream);
        default: return launch_q4_fma<T, 256>(x, pl, dev, smem_optin, stream);
    }
}

// The limits of the bounded waits in this translation unit's kernels (hogatt_api.cu sets its own; see hogatt_device.cuh).
int ensure_wait_limits(int dev) {
    static std::atomic<bool> done[kMaxDevices];
    if (done[dev].load(std::memory_order_acquire)) return HOGATT_OK;
    if (const char* ms = getenv("HOGATT_WAIT_LIMIT_MS")) {
        const unsigned int polls = (unsigned int)std::min(std::max(1ll, atoll(ms)), 1000000ll) * kPollsPerMs;
        HOGATT_CUDA_OK(cudaMemcpyToSymbol(g_wait_polls, &polls, sizeof(polls)));
    }
    done[dev].store(true, std::memory_order_release);
    return HOGATT_OK;
}

template <class T>
int launch_q4_dense(const hogatt_paged_q4_problem* x, const Q4Plan& pl, int dev, int smem_optin, cudaStream_t stream) {
    const hogatt_paged_problem* p = &x->paged;
    int rc = ensure_wait_limits(dev);
    if (rc != HOGATT_OK) return rc;
    unsigned char* const ws = static_cast<unsigned char*>(p->workspace);
    DenseArgs d;
    memset(&d, 0, sizeof(d));
    d.F = p->F; d.W = p->W; d.Hq = p->Hq; d.Hkv = p->Hkv; d.G = p->Hq / p->Hkv;
    d.tiles = 2 * pl.blocks;
    d.blocks = pl.blocks;
    d.tile_span = pl.tokens;
    d.total_q = p->total_q_tokens;
    d.block_size = p->block_size;
    d.max_blocks = p->max_blocks_per_seq;
    d.l2scale = score_factor(x);
    d.loc = p->locations;
    d.flen = p->fragment_lengths;
    d.cu = p->cu_seqlens_q;
    d.block_table = p->block_table;
    d.nmerge = reinterpret_cast<int*>(ws);
    d.start = reinterpret_cast<int4*>(ws + pl.w.start);
    d.merge = reinterpret_cast<int4*>(ws + pl.w.merge);
    d.fold = reinterpret_cast<int*>(ws + pl.w.fold);
    d.pre = reinterpret_cast<long long*>(ws + pl.w.pre);
    d.cost = reinterpret_cast<long long*>(ws + pl.w.cost);
    d.vis = reinterpret_cast<int*>(ws + pl.w.vis);
    d.rec = reinterpret_cast<int4*>(ws + pl.w.rec);
    d.ws_o = reinterpret_cast<float4*>(ws + pl.w.o);
    d.ws_m = reinterpret_cast<float*>(ws + pl.w.m);
    d.ws_l = reinterpret_cast<float*>(ws + pl.w.l);
    d.ctas = pl.ctas;
    d.status = p->device_status;
    d.out = p->out;
    d.codes[0] = static_cast<const unsigned char*>(p->key_cache);
    d.codes[1] = static_cast<const unsigned char*>(p->value_cache);
    d.scales[0] = static_cast<const unsigned char*>(x->key_scales);
    d.scales[1] = static_cast<const unsigned char*>(x->value_scales);
    d.num_blocks = p->num_blocks;
    d.most_keys = (int)std::min<int64_t>((int64_t)p->max_blocks_per_seq * p->block_size + 1, INT_MAX - 4096);
    const FastDiv by_block = fast_div_by((uint32_t)p->block_size);
    d.block_mul = by_block.mul;
    d.block_shift = by_block.shift;
    d.out_scale = x->value_unit;
    constexpr bool convert = std::is_same<T, __nv_bfloat16>::value;
    d.factor = reinterpret_cast<float*>(ws + pl.factor);
    const void* const q = convert ? ws + pl.queries : p->queries;
    DenseMaps maps;
    memset(&maps, 0, sizeof(maps));
    const cuuint64_t qdims[5] = {128, (cuuint64_t)d.G, (cuuint64_t)d.Hkv, (cuuint64_t)d.total_q, (cuuint64_t)d.F};
    const cuuint32_t qbox[5] = {64, (cuuint32_t)d.G, 1, (cuuint32_t)d.tile_span, 1};
    rc = encode_map(&maps.q, q, HOGATT_F16, 5, qdims, qbox);
    if (rc != HOGATT_OK) return rc;
    HOGATT_CUDA_OK(launch_kernel(dense_plan_kernel<true>, dim3(1), dim3(kDensePlanThreads), 0, stream, d));
    const int rows = p->F * p->total_q_tokens * p->Hq;
    HOGATT_CUDA_OK(launch_kernel(q4_dense_queries_kernel<T>, dim3((rows + 7) / 8), dim3(256), 0, stream, static_cast<const T*>(p->queries),
                                 reinterpret_cast<__half*>(ws + pl.queries), reinterpret_cast<float*>(ws + pl.factor), rows, d.l2scale));
    static std::atomic<size_t> granted[kMaxDevices];
    constexpr size_t smem = DenseCfgOf<true>::OFF_END;
    if (smem > (size_t)smem_optin) return HOGATT_ERR_CUDA;
    rc = ensure_smem_limit(dense_attention_kernel<T, true, true>, dev, smem, granted);
    if (rc != HOGATT_OK) return rc;
    HOGATT_CUDA_OK(launch_kernel(dense_attention_kernel<T, true, true>, dim3(d.ctas), dim3(DenseCfgOf<true>::WARPS * 32), smem, stream, d, maps));
    // (as for 16-bit pages: few units have many partials, whose eight warps share a row's)
    const int64_t units = (int64_t)d.blocks * d.Hkv, resident = 2 * (int64_t)d.ctas;
    const dim3 block(kDenseMergeWarps * 32);
    if (d.ctas <= 8 * units)
        HOGATT_CUDA_OK(launch_kernel(dense_merge_kernel<T, true, false, kDenseMergeBatch>, dim3((unsigned)std::min(8 * units, resident)), block, 0, stream, d));
    else
        HOGATT_CUDA_OK(launch_kernel(dense_merge_kernel<T, true, true, 1>, dim3((unsigned)(64 * units)), block, 0, stream, d));
    return HOGATT_OK;
}

// (rows x groups, kv heads, sequences), eight CTAs of 256 threads per SM at most
dim3 rows_grid(int64_t rows, int64_t groups, int Hkv, int B, int sms) {
    const int64_t z = std::min(B, 65535), per = std::max<int64_t>(1, (int64_t)sms * 8 / (Hkv * z));
    return dim3((unsigned)std::min((rows * groups + 255) / 256, per), (unsigned)Hkv, (unsigned)z);
}

// Bookkeeping runs as one cluster; the copies follow on the whole GPU.
int launch_copies(const hogatt_block_tensors* t, const int* count, const int* pairs, int64_t most, int sms, cudaStream_t stream) {
    for (int first = 0; first < t->count; first += kMaxPageTensors) {
        CopyPagesArgs c;
        memset(&c, 0, sizeof(c));
        c.n = std::min(kMaxPageTensors, t->count - first);
        c.count = count;
        c.pairs = pairs;
        int64_t pieces = 0;
        for (int i = 0; i < c.n; ++i) {
            const int64_t bytes = t->block_bytes[first + i];
            c.t[i] = {static_cast<char*>(t->data[first + i]), bytes, (int)pieces, aligned16(t->data[first + i]) && bytes % 16 == 0};
            pieces += (bytes + kPagePiece - 1) / kPagePiece;
            if (pieces >= ((int64_t)1 << 31)) return HOGATT_ERR_TOO_LARGE;
        }
        c.pieces = (int)pieces;
        const int64_t ctas = (most * pieces + 7) / 8;
        HOGATT_CUDA_OK(launch_kernel(copy_pages_kernel, dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(ctas, (int64_t)sms * 6))), dim3(256), 0, stream, c));
    }
    return HOGATT_OK;
}

// CTAs of the bookkeeping cluster by what there is to read (pages' counts and table entries): a barrier over several costs more than it
// saves where one has little to do.  us per call, copies included, with 1 / 2 / 4 / 8: compaction of 512 pages 9.6 / 9.8 / 10.1 / 12.0; a fork of 8 rows
// into 32, 2,048 pages, 6,000 entries 20.2 / 18.4 / 18.7 / 19.1; 64 rows of 250 entries, 20,480 pages 15.9 / 12.4 / 10.5 / 10.4.
int cluster_ctas(int64_t cells) { return cells <= 2048 ? 1 : cells <= 8192 ? 2 : cells <= 65536 ? 4 : kBlocksCluster; }

template <class Args>
cudaError_t launch_cluster(void (*kernel)(Args), int ctas, cudaStream_t stream, const Args& args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kBlocksThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args);
}

int check_tensors(const hogatt_block_tensors* t) {
    if (t->count < 0) return HOGATT_ERR_BAD_SHAPE;
    if (t->count > 0 && (!t->data || !t->block_bytes)) return HOGATT_ERR_NULL_POINTER;
    for (int i = 0; i < t->count; ++i) {
        if (!t->data[i]) return HOGATT_ERR_NULL_POINTER;
        if (t->block_bytes[i] <= 0) return HOGATT_ERR_BAD_SHAPE;
    }
    return HOGATT_OK;
}

}  // namespace
}  // namespace hogatt

using namespace hogatt;

extern "C" {

size_t hogatt_paged_q4_workspace_bytes(const hogatt_paged_q4_problem* p) {
    int dev, sms, smem_optin;
    if (current_device_info(&dev, &sms, &smem_optin) != HOGATT_OK) return 0;
    Q4Plan pl;
    return plan_q4(p, sms, &pl) == HOGATT_OK ? pl.total : 0;
}

int hogatt_paged_q4_sdpa_launch(const hogatt_paged_q4_problem* x, hogatt_stream_t stream_) {
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    Q4Plan pl;
    int rc = plan_q4(x, 1, &pl);                          // (arguments before anything about the device)
    if (rc != HOGATT_OK) return rc;
    const hogatt_paged_problem* p = &x->paged;
    if (!unit_ok(x->key_unit) || !unit_ok(x->value_unit)) return HOGATT_ERR_BAD_UNIT;
    if (std::isfinite(p->scale) && !std::isfinite(score_factor(x))) return HOGATT_ERR_BAD_UNIT;
    if (!p->out || !p->queries || !p->locations || !p->fragment_lengths || !p->key_cache || !p->value_cache || !x->key_scales ||
        !x->value_scales || !p->block_table || !p->workspace)
        return HOGATT_ERR_NULL_POINTER;
    if (!aligned16(p->out) || !aligned16(p->queries) || !aligned16(p->key_cache) || !aligned16(p->value_cache) || !aligned16(x->key_scales) ||
        !aligned16(x->value_scales) || ((uintptr_t)p->workspace & 255u))
        return HOGATT_ERR_MISALIGNED;
    const bool packed = p->cu_seqlens_q != nullptr;
    if (packed && p->total_q_tokens == 0) return HOGATT_OK;
    int dev, sms, smem_optin;
    rc = current_device_info(&dev, &sms, &smem_optin);
    if (rc == HOGATT_OK) rc = plan_q4(x, sms, &pl);
    if (rc != HOGATT_OK) return rc;
    if (p->workspace_bytes < pl.total) return HOGATT_ERR_WORKSPACE_TOO_SMALL;

    if (pl.kernel == HOGATT_KERNEL_DENSE)
        return p->dtype == HOGATT_F16 ? launch_q4_dense<__half>(x, pl, dev, smem_optin, stream) : launch_q4_dense<__nv_bfloat16>(x, pl, dev, smem_optin, stream);
    Q4Args args;
    memset(&args, 0, sizeof(args));
    PagedArgs& a = args.p;
    a.F = p->F; a.W = p->W; a.Hq = p->Hq; a.Hkv = p->Hkv; a.G = p->Hq / p->Hkv; a.E = p->E; a.Ev = p->Ev;
    a.S = p->S; a.total_q = packed ? p->total_q_tokens : p->W * p->S;
    a.block_size = p->block_size; a.max_blocks = p->max_blocks_per_seq;
    a.tokens_per_group = pl.tokens_per_group; a.head_blocks = pl.head_blocks; a.groups_bound = pl.groups_bound;
    a.splits = pl.splits;
    // (a scale that is no number: every score is inf - inf or 0 * inf, NaN)
    a.l2scale = std::isfinite(p->scale) ? score_factor(x) : NAN;
    if (packed) {     // q [F,total_q,Hq,E], out [total_q,Hq,Ev], loc [F,total_q], len [F,W]; s is the packed token index
        a.q_f = (long long)a.total_q * p->Hq * p->E; a.q_w = 0; a.q_s = (long long)p->Hq * p->E; a.q_h = p->E;
        a.o_w = 0; a.o_s = (long long)p->Hq * p->Ev; a.o_h = p->Ev;
        a.loc_f = a.total_q; a.loc_w = 0; a.len_f = p->W; a.len_w = 1;
    } else {          // q [F,W,Hq,S,E], out [W,Hq,S,Ev], loc [F,W,S], len [F]
        a.q_f = (long long)p->W * p->Hq * p->S * p->E; a.q_w = (long long)p->Hq * p->S * p->E; a.q_s = p->E;
        a.q_h = (long long)p->S * p->E;
        a.o_w = (long long)p->Hq * p->S * p->Ev; a.o_s = p->Ev; a.o_h = (long long)p->S * p->Ev;
        a.loc_f = p->W * p->S; a.loc_w = p->S; a.len_f = 1; a.len_w = 0;
    }
    a.out = p->out; a.q = p->queries; a.loc = p->locations; a.flen = p->fragment_lengths;
    a.kcache = p->key_cache; a.vcache = p->value_cache; a.block_table = p->block_table; a.cu_seqlens = p->cu_seqlens_q;
    unsigned char* ws = static_cast<unsigned char*>(p->workspace);
    a.ws_o = reinterpret_cast<float*>(ws + pl.o);
    a.ws_m = reinterpret_cast<float*>(ws + pl.m);
    a.ws_l = reinterpret_cast<float*>(ws + pl.l);
    a.status = p->device_status;
    args.kscale = static_cast<const unsigned char*>(x->key_scales);
    args.vscale = static_cast<const unsigned char*>(x->value_scales);
    args.num_blocks = p->num_blocks;
    args.vunit = x->value_unit;
    args.plan = reinterpret_cast<int*>(ws + pl.plan);
    switch (p->dtype) {
        case HOGATT_F32: return launch_q4<float>(args, pl, dev, smem_optin, stream);
        case HOGATT_F16: return launch_q4<__half>(args, pl, dev, smem_optin, stream);
        default: return launch_q4<__nv_bfloat16>(args, pl, dev, smem_optin, stream);
    }
}

int hogatt_copy_to_blocks_q4_launch(const hogatt_q4_append* p, hogatt_stream_t stream_) {
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    if (p == nullptr) return HOGATT_ERR_NULL_POINTER;
    const bool packed = p->cu_seqlens != nullptr;
    if (p->B <= 0 || p->S < 0) return HOGATT_ERR_BAD_SHAPE;
    if (const int rc = cache_shape(p->Hkv, p->E, p->Ev, p->block_size, p->max_blocks, p->num_blocks, p->dtype)) return rc;
    if (!unit_ok(p->key_unit) || !unit_ok(p->value_unit)) return HOGATT_ERR_BAD_UNIT;
    if (!p->keys || !p->values || !p->key_cache || !p->value_cache || !p->key_scales || !p->value_scales || !p->block_table || !p->seq_lengths)
        return HOGATT_ERR_NULL_POINTER;
    if (!aligned16(p->key_cache) || !aligned16(p->value_cache) || !aligned16(p->key_scales) || !aligned16(p->value_scales)) return HOGATT_ERR_MISALIGNED;
    if (p->S == 0) return HOGATT_OK;
    Q4AppendArgs a;
    memset(&a, 0, sizeof(a));
    a.B = p->B; a.Hkv = p->Hkv; a.S = p->S; a.E = p->E; a.Ev = p->Ev;
    a.max_blocks = p->max_blocks; a.num_blocks = p->num_blocks;
    a.block = fast_div_by((uint32_t)p->block_size);
    a.groups = fast_div_by((uint32_t)(std::max(p->E, p->Ev) / kGroup));
    a.packed_tokens = packed ? p->S : 0;
    const int vec = 16 / (int)dtype_size(p->dtype);
    bool vectorised = aligned16(p->keys) && aligned16(p->values);
    for (int i = 0; i < 3; ++i) {
        a.ks[i] = p->key_strides[i];
        a.vs[i] = p->value_strides[i];
        vectorised = vectorised && a.ks[i] % vec == 0 && a.vs[i] % vec == 0;
    }
    a.key_unit = p->key_unit; a.value_unit = p->value_unit;
    a.k = p->keys; a.v = p->values;
    a.codes[0] = static_cast<unsigned char*>(p->key_cache); a.codes[1] = static_cast<unsigned char*>(p->value_cache);
    a.scales[0] = static_cast<unsigned char*>(p->key_scales); a.scales[1] = static_cast<unsigned char*>(p->value_scales);
    a.table = p->block_table; a.lengths = p->seq_lengths; a.cu = p->cu_seqlens; a.new_rows = p->new_rows; a.status = p->device_status;
    int dev, sms, smem_optin;
    if (const int rc = current_device_info(&dev, &sms, &smem_optin)) return rc;
    const dim3 grid = rows_grid(p->S, a.groups.d, p->Hkv, packed ? 1 : p->B, sms);
    cudaError_t err;
    switch (p->dtype) {
        case HOGATT_F32: err = launch_kernel(q4_append_kernel<float>, grid, dim3(256), 0, stream, a, (int)vectorised); break;
        case HOGATT_F16: err = launch_kernel(q4_append_kernel<__half>, grid, dim3(256), 0, stream, a, (int)vectorised); break;
        default: err = launch_kernel(q4_append_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, a, (int)vectorised); break;
    }
    HOGATT_CUDA_OK(err);
    return HOGATT_OK;
}

int hogatt_copy_from_blocks_q4_launch(const hogatt_q4_read* p, hogatt_stream_t stream_) {
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    if (p == nullptr) return HOGATT_ERR_NULL_POINTER;
    if (p->B <= 0 || p->S < 0) return HOGATT_ERR_BAD_SHAPE;
    if (const int rc = cache_shape(p->Hkv, p->E, p->Ev, p->block_size, p->max_blocks, p->num_blocks, p->dtype)) return rc;
    if (!unit_ok(p->key_unit) || !unit_ok(p->value_unit)) return HOGATT_ERR_BAD_UNIT;
    if (p->S == 0) return HOGATT_OK;
    if (!p->keys || !p->values || !p->key_cache || !p->value_cache || !p->key_scales || !p->value_scales || !p->block_table || !p->first_rows)
        return HOGATT_ERR_NULL_POINTER;
    if (!aligned16(p->keys) || !aligned16(p->values) || !aligned16(p->key_cache) || !aligned16(p->value_cache) || !aligned16(p->key_scales) ||
        !aligned16(p->value_scales))
        return HOGATT_ERR_MISALIGNED;
    Q4ReadArgs a;
    memset(&a, 0, sizeof(a));
    a.B = p->B; a.Hkv = p->Hkv; a.S = p->S; a.E = p->E; a.Ev = p->Ev;
    a.max_blocks = p->max_blocks; a.num_blocks = p->num_blocks;
    a.block = fast_div_by((uint32_t)p->block_size);
    a.groups = fast_div_by((uint32_t)(std::max(p->E, p->Ev) / kGroup));
    a.key_unit = p->key_unit; a.value_unit = p->value_unit;
    a.k = p->keys; a.v = p->values;
    a.codes[0] = static_cast<const unsigned char*>(p->key_cache); a.codes[1] = static_cast<const unsigned char*>(p->value_cache);
    a.scales[0] = static_cast<const unsigned char*>(p->key_scales); a.scales[1] = static_cast<const unsigned char*>(p->value_scales);
    a.table = p->block_table; a.first = p->first_rows; a.status = p->device_status;
    int dev, sms, smem_optin;
    if (const int rc = current_device_info(&dev, &sms, &smem_optin)) return rc;
    const dim3 grid = rows_grid(p->S, a.groups.d, p->Hkv, p->B, sms);
    cudaError_t err;
    switch (p->dtype) {
        case HOGATT_F32: err = launch_kernel(q4_read_kernel<float>, grid, dim3(256), 0, stream, a); break;
        case HOGATT_F16: err = launch_kernel(q4_read_kernel<__half>, grid, dim3(256), 0, stream, a); break;
        default: err = launch_kernel(q4_read_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, a); break;
    }
    HOGATT_CUDA_OK(err);
    return HOGATT_OK;
}

size_t hogatt_step_blocks_workspace_bytes(int32_t rows_out) {
    return rows_out > 0 && rows_out <= HOGATT_MAX_BLOCK_ROWS ? align_up((size_t)step_blocks_ints(rows_out) * sizeof(int), 256) : 0;
}

int hogatt_step_blocks_launch(const hogatt_step_blocks* p, hogatt_stream_t stream_) {
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    if (p == nullptr) return HOGATT_ERR_NULL_POINTER;
    if (p->num_blocks <= 0 || p->block_size <= 0 || p->max_blocks <= 0 || p->rows_in <= 0 || p->rows_out <= 0 || (!p->source && p->rows_out != p->rows_in))
        return HOGATT_ERR_BAD_SHAPE;
    if (p->rows_in > HOGATT_MAX_BLOCK_ROWS || p->rows_out > HOGATT_MAX_BLOCK_ROWS || p->num_blocks == INT_MAX) return HOGATT_ERR_TOO_LARGE;
    if (p->max_blocks >= 1 << 30) return HOGATT_ERR_TOO_LARGE;      // (a row's pages travel twice themselves, with a bit behind)
    if (!p->refs_in || !p->table_in || !p->lengths_in || !p->refs_out || !p->table_out || !p->lengths_out || !p->room || !p->workspace)
        return HOGATT_ERR_NULL_POINTER;
    // rows that change places cannot be taken over in place
    if (p->source && (p->table_out == p->table_in || p->lengths_out == p->lengths_in)) return HOGATT_ERR_BAD_SHAPE;
    if (const int rc = check_tensors(&p->caches)) return rc;
    if ((uintptr_t)p->workspace & 255u) return HOGATT_ERR_MISALIGNED;
    if (p->workspace_bytes < hogatt_step_blocks_workspace_bytes(p->rows_out)) return HOGATT_ERR_WORKSPACE_TOO_SMALL;
    int dev, sms, smem_optin;
    if (const int rc = current_device_info(&dev, &sms, &smem_optin)) return rc;
    StepBlocksArgs a;
    a.num_blocks = p->num_blocks; a.block_size = p->block_size; a.max_blocks = p->max_blocks; a.rows_in = p->rows_in; a.rows_out = p->rows_out;
    a.refs_in = p->refs_in; a.table_in = p->table_in; a.lengths_in = p->lengths_in; a.source = p->source; a.new_tokens = p->new_tokens;
    a.refs_out = p->refs_out; a.table_out = p->table_out; a.lengths_out = p->lengths_out; a.room = p->room;
    a.ws = static_cast<int*>(p->workspace);
    a.status = p->device_status;
    HOGATT_CUDA_OK(launch_cluster(step_blocks_kernel, cluster_ctas(p->num_blocks + (int64_t)p->rows_out * p->max_blocks), stream, a));
    if (p->new_tokens == nullptr) return HOGATT_OK;                 // (nobody writes: nothing is copied)
    return launch_copies(&p->caches, a.ws, a.ws + step_blocks_pairs(p->rows_out), p->rows_out, sms, stream);
}

size_t hogatt_compact_blocks_workspace_bytes(int32_t num_blocks) {
    return num_blocks > 0 ? align_up((size_t)compact_blocks_ints(num_blocks) * sizeof(int), 256) : 0;
}

int hogatt_compact_blocks_launch(const hogatt_compact_blocks* p, hogatt_stream_t stream_) {
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    if (p == nullptr) return HOGATT_ERR_NULL_POINTER;
    if (p->num_blocks <= 0 || p->table_entries < 0) return HOGATT_ERR_BAD_SHAPE;
    if (!p->refs_in || !p->refs_out || !p->moved || !p->workspace || (p->table_entries > 0 && (!p->table_in || !p->table_out)))
        return HOGATT_ERR_NULL_POINTER;
    if (const int rc = check_tensors(&p->caches)) return rc;
    if ((uintptr_t)p->workspace & 255u) return HOGATT_ERR_MISALIGNED;
    if (p->workspace_bytes < hogatt_compact_blocks_workspace_bytes(p->num_blocks)) return HOGATT_ERR_WORKSPACE_TOO_SMALL;
    int dev, sms, smem_optin;
    if (const int rc = current_device_info(&dev, &sms, &smem_optin)) return rc;
    CompactBlocksArgs a;
    a.num_blocks = p->num_blocks; a.entries = p->table_entries;
    a.refs_in = p->refs_in; a.table_in = p->table_in; a.refs_out = p->refs_out; a.table_out = p->table_out; a.moved = p->moved;
    a.ws = static_cast<int*>(p->workspace);
    a.status = p->device_status;
    HOGATT_CUDA_OK(launch_cluster(compact_blocks_kernel, cluster_ctas(p->num_blocks + p->table_entries), stream, a));
    return launch_copies(&p->caches, a.ws, a.ws + kCompactHead, p->num_blocks / 2 + 1, sms, stream);
}

}  // extern "C"

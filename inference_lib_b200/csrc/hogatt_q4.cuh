// Pages in 4 bits.  A row of E channels is E/2 bytes of e2m1 codes (the even channel in the low half of a byte) and E/16 e4m3 scales,
// one per 16 consecutive channels:
//     value[e] = e2m1(code[e]) * e4m3(scale[e / 16]) * unit,        unit a power of two that the caller keeps per cache
// Writing a group with largest magnitude a: scale = a / (6 unit) rounded to e4m3 (to the nearest, ties to even, at most 448), code = x /
// (scale unit) rounded to e2m1 the same way, at most 6.  A group with an infinity or a NaN gets a NaN scale.
// e2m1 has two significant bits and e4m3 four: code * scale has at most six, between 2^-10 and 2688, and is exact in fp16 and bf16.
// scale * unit is exact as well, so the one rounded operation in front of a choice between two codes is a division, whose
// quotient is on the same side of every border as the exact one (the border times the divisor has at most six bits).
//
// Here: the write path (q4_append_kernel), the way back (q4_read_kernel) and attention for every type and head size
// (q4_attention_kernel, CUDA cores).
#pragma once
#include "hogatt_device.cuh"
#include "hogatt_fma.cuh"
#include "hogatt_merge.cuh"
#include "hogatt_paged.cuh"

namespace hogatt {

enum BlockStatusBits : int {
    STATUS_NO_BLOCKS = 512,       // a row's pages did not fit into the pool
    STATUS_BAD_BLOCK = 1024,      // a page that the block table does not name, or names outside the cache
    STATUS_TABLE_FULL = 2048      // a row is longer than the block table is wide
};

constexpr int kGroup = 16;        // channels per scale

// two fp32 values -> two e2m1 codes, `lo` in the low half of the byte
__device__ __forceinline__ uint32_t to_e2m1x2(float lo, float hi) {
    uint32_t r;
    asm("{\n\t.reg .b8 b;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %1, %2;\n\tcvt.u32.u8 %0, b;\n\t}" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// two e2m1 codes of a byte -> two fp16 values, the low half's first
__device__ __forceinline__ uint32_t from_e2m1x2(uint32_t byte) {
    uint32_t r;
    asm("{\n\t.reg .b8 b;\n\tcvt.u8.u32 b, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(r) : "r"(byte));
    return r;
}
// the eight codes of a word as fp16, byte by byte
__device__ __forceinline__ void from_e2m1x8(uint32_t w, uint32_t (&out)[4]) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\tcvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(out[0]), "=r"(out[1]), "=r"(out[2]), "=r"(out[3]) : "r"(w));
}
__device__ __forceinline__ uint32_t to_e4m3(float x) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(x));
    return r & 0xffu;
}
// two e4m3 values of 16 bits -> two fp16 values
__device__ __forceinline__ uint32_t from_e4m3x2(uint32_t pair) {
    uint32_t r;
    asm("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(pair));
    return r;
}
__device__ __forceinline__ float from_e4m3(uint32_t byte) {
    const uint32_t h = from_e4m3x2(byte & 0xffu);
    return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}
__device__ __forceinline__ bool is_nan_e4m3(uint32_t byte) { return (byte & 0x7fu) == 0x7fu; }
__device__ __forceinline__ float2 half2_of(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

// n / d for 0 <= n < 2^31
struct FastDiv {
    uint32_t mul, shift, d;
};
__device__ __forceinline__ uint32_t fast_div(uint32_t n, const FastDiv& f) { return (__umulhi(n, f.mul) + n) >> f.shift; }

// Row `pos` of a sequence in the cache (rows of all pages and heads are numbered through), or -1: no page there.
__device__ __forceinline__ long long paged_row_at(const int* table, int pos, const FastDiv& block, int max_blocks, int num_blocks, int Hkv, int h) {
    const int at = (int)fast_div((uint32_t)pos, block);
    if (pos < 0 || at >= max_blocks) return -1;
    const int page = table[at];
    if (page < 0 || page >= num_blocks) return -1;
    return ((long long)page * Hkv + h) * block.d + (pos - at * (int)block.d);
}
__device__ __forceinline__ long long paged_row_at(const int* table, int pos, int block_size, int max_blocks, int num_blocks, int Hkv, int h) {
    const int at = pos / block_size;
    if (pos < 0 || at >= max_blocks) return -1;
    const int page = table[at];
    if (page < 0 || page >= num_blocks) return -1;
    return ((long long)page * Hkv + h) * block_size + (pos - at * block_size);
}

// exclusive prefix of `x` over the CTA's threads; the total comes back in *total.  Called by all threads.
template <class I>
__device__ __forceinline__ I block_exclusive(I x, I* total) {
    __shared__ I warp_sum[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    I inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const I y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
    }
    __syncthreads();                                      // (the array may still be in use from the last call)
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        I s = lane < (int)(blockDim.x >> 5) ? warp_sum[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const I y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        warp_sum[lane] = s;
    }
    __syncthreads();
    *total = warp_sum[31];
    return inc - x + (warp ? warp_sum[warp - 1] : 0);
}
struct Q4AppendArgs {
    int B, Hkv, S, E, Ev, max_blocks, num_blocks;
    int packed_tokens;            // packed layout: rows of the source; fixed layout: 0
    FastDiv block, groups;        // block size; max(E, Ev) / 16
    long long ks[3], vs[3];       // element strides of (sequence, kv head, token)
    float key_unit, value_unit;
    const void* k;
    const void* v;
    unsigned char* codes[2];      // keys, values
    unsigned char* scales[2];
    const int* table;
    const int* lengths;
    const int* cu;                // packed layout: [B + 1]
    const int* new_rows;          // [B] or nullptr: rows of a sequence behind this many stay out
    int* status;
};

// The sequence that packed token `i` belongs to: the last b with cu[b] <= i (sequences may be empty), -1 past the end.
__device__ __forceinline__ int packed_sequence(const int* cu, int B, int i) {
    if (i < cu[0] || i >= cu[B]) return -1;
    int lo = 0, hi = B;                                   // cu[lo] <= i < cu[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

// 16 consecutive channels as fp32
template <class T>
__device__ __forceinline__ void load_group(const T* src, bool vectorised, float (&x)[kGroup]) {
    constexpr int VEC = 16 / (int)sizeof(T), N = kGroup / VEC;
    if (vectorised) {
        int4 raw[N];
#pragma unroll
        for (int i = 0; i < N; ++i) raw[i] = load_16(src + i * VEC);
#pragma unroll
        for (int i = 0; i < kGroup; ++i) x[i] = Scalar<T>::to_float(reinterpret_cast<const T*>(raw)[i]);
    } else {
#pragma unroll
        for (int i = 0; i < kGroup; ++i) x[i] = Scalar<T>::to_float(src[i]);
    }
}

// A group's scale and codes.  x / step is the correctly rounded quotient, from a correctly rounded reciprocal r of the step and one
// correction, q + (x - q step) r (Markstein, IBM J. Res. Dev. 34, 1990).  It stays below 10 unless the scale is the largest; then a first
// quotient beyond 8 is taken for 8, so that nothing overflows into a NaN, and its correction only takes it further out.  A group
// whose scale is zero or not a number has codes of zero.  (A division per channel: 12,000 rows of 4 groups 9.3 us.)
__device__ __forceinline__ void quantise_group(const float (&x)[kGroup], float unit, uint32_t (&code)[2], uint32_t* scale) {
    uint32_t top = 0;                                     // largest magnitude, as bits: NaN > infinity > every number
#pragma unroll
    for (int e = 0; e < kGroup; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
    *scale = top >= 0x7f800000u ? 0x7fu : to_e4m3(__fdiv_rn(__uint_as_float(top), 6.f * unit));
    const float step = from_e4m3(*scale) * unit, r = __fdiv_rn(1.f, step);
    float q[kGroup];
#pragma unroll
    for (int e = 0; e < kGroup; ++e) q[e] = x[e] * r;
    if (*scale == 0x7eu) {
#pragma unroll
        for (int e = 0; e < kGroup; ++e) q[e] = fminf(fmaxf(q[e], -8.f), 8.f);
    }
#pragma unroll
    for (int e = 0; e < kGroup; ++e) q[e] = fmaf(fmaf(q[e], -step, x[e]), r, q[e]);
    code[0] = code[1] = 0u;
#pragma unroll
    for (int e = 0; e < kGroup; e += 2) code[e / 8] |= to_e2m1x2(q[e], q[e + 1]) << (e % 8 * 4);
    if (!(step > 0.f)) code[0] = code[1] = 0u;
}

// A thread: one group of a key row and of the value row beside it.  grid: (groups of rows, kv heads, sequences), packed layout one "sequence".
template <class T>
__global__ void __launch_bounds__(256) q4_append_kernel(const __grid_constant__ Q4AppendArgs a, const int vectorised) {
    const int gk = a.E / kGroup, gv = a.Ev / kGroup, h = blockIdx.y;
    pdl_wait();
    pdl_trigger();
    for (int z = blockIdx.z; z < (a.cu ? 1 : a.B); z += gridDim.z) {
        const int rows = a.cu ? a.packed_tokens : a.S;
        for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < (int64_t)rows * a.groups.d; i += (int64_t)gridDim.x * blockDim.x) {
            const int row = i < INT_MAX ? (int)fast_div((uint32_t)i, a.groups) : (int)(i / a.groups.d), g = (int)(i - (int64_t)row * a.groups.d);
            // both rows' loads first: where they go takes two more round trips
            float x[2][kGroup];
            if (g < gk) load_group<T>(static_cast<const T*>(a.k) + z * a.ks[0] + h * a.ks[1] + row * a.ks[2] + g * kGroup, vectorised, x[0]);
            if (g < gv) load_group<T>(static_cast<const T*>(a.v) + z * a.vs[0] + h * a.vs[1] + row * a.vs[2] + g * kGroup, vectorised, x[1]);
            int b = z, t = row;
            if (a.cu) {
                b = packed_sequence(a.cu, a.B, row);
                if (b < 0) continue;
                t = row - a.cu[b];
            }
            if (a.new_rows && t >= a.new_rows[b]) continue;
            const long long dst = paged_row_at(a.table + (size_t)b * a.max_blocks, a.lengths[b] + t, a.block, a.max_blocks, a.num_blocks, a.Hkv, h);
            if (dst < 0) {
                if (a.status && g == 0) atomicOr(a.status, STATUS_BAD_BLOCK);
                continue;
            }
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int groups = v ? gv : gk;
                if (g >= groups) continue;
                uint32_t code[2], scale;
                quantise_group(x[v], v ? a.value_unit : a.key_unit, code, &scale);
                *reinterpret_cast<uint2*>(a.codes[v] + ((size_t)dst * groups + g) * (kGroup / 2)) = make_uint2(code[0], code[1]);
                a.scales[v][(size_t)dst * groups + g] = (unsigned char)scale;
            }
        }
    }
}

struct Q4ReadArgs {
    int B, Hkv, S, E, Ev, max_blocks, num_blocks;
    FastDiv block, groups;
    float key_unit, value_unit;
    void* k;                      // [B, Hkv, S, E]
    void* v;
    const unsigned char* codes[2];
    const unsigned char* scales[2];
    const int* table;
    const int* first;             // [B]: the first row of each sequence that is read
    int* status;
};

// Rows first[b] ... first[b] + S - 1 of every sequence as numbers; a row without a page is NaN.  Threads and grid as above.
template <class T>
__global__ void __launch_bounds__(256) q4_read_kernel(const __grid_constant__ Q4ReadArgs a) {
    const int gk = a.E / kGroup, gv = a.Ev / kGroup, h = blockIdx.y;
    pdl_wait();
    pdl_trigger();
    for (int b = blockIdx.z; b < a.B; b += gridDim.z) {
        const int first = a.first[b];
        for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < (int64_t)a.S * a.groups.d; i += (int64_t)gridDim.x * blockDim.x) {
            const int t = i < INT_MAX ? (int)fast_div((uint32_t)i, a.groups) : (int)(i / a.groups.d), g = (int)(i - (int64_t)t * a.groups.d);
            const long long src = paged_row_at(a.table + (size_t)b * a.max_blocks, first + t, a.block, a.max_blocks, a.num_blocks, a.Hkv, h);
            if (src < 0 && a.status && g == 0) atomicOr(a.status, STATUS_BAD_BLOCK);
            const size_t row = ((size_t)b * a.Hkv + h) * a.S + t;
            uint2 code[2] = {make_uint2(0u, 0u), make_uint2(0u, 0u)};
            uint32_t scale[2] = {0x7fu, 0x7fu};
#pragma unroll
            for (int v = 0; v < 2; ++v)
                if (src >= 0 && g < (v ? gv : gk)) {
                    const size_t at = (size_t)src * (v ? gv : gk) + g;
                    code[v] = *reinterpret_cast<const uint2*>(a.codes[v] + at * (kGroup / 2));
                    scale[v] = a.scales[v][at];
                }
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int groups = v ? gv : gk;
                if (g >= groups) continue;
                const float step = from_e4m3(scale[v]) * (v ? a.value_unit : a.key_unit);
                __align__(16) T out[kGroup];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t x[4];
                    from_e2m1x8(e ? code[v].y : code[v].x, x);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float2 y = half2_of(x[k]);
                        out[e * 8 + 2 * k] = Scalar<T>::from_float(y.x * step);
                        out[e * 8 + 2 * k + 1] = Scalar<T>::from_float(y.y * step);
                    }
                }
                uint4* const dst = reinterpret_cast<uint4*>(static_cast<T*>(v ? a.v : a.k) + (row * groups + g) * kGroup);
#pragma unroll
                for (int k = 0; k < (int)(kGroup * sizeof(T) / 16); ++k) dst[k] = reinterpret_cast<const uint4*>(out)[k];
            }
        }
    }
}

// ---- attention -----------------------------------------------------------------------------------------------------------
// Keys that a row at `loc` of a sequence of `len` sees, as far as the kernels walk: the block table's and one more, which says that there are more
// than it has pages for (a length that is wrong would be a walk over two billion keys).
__device__ __forceinline__ int most_visible(const PagedArgs& a, int loc, int len) {
    const int64_t most = min((int64_t)a.max_blocks * a.block_size + 1, (int64_t)INT_MAX - 4096);
    return (int)min((int64_t)(max(0, min(loc, max(len, 0) - 1) + 1)), most);
}

struct Q4Args {
    PagedArgs p;                  // kcache / vcache: the codes
    const unsigned char* kscale;
    const unsigned char* vscale;
    int num_blocks;
    float vunit;                  // (the keys' unit is in p.l2scale)
    int* plan;                    // (the tensor-core kernel's)
};

// Any type, any head size: the units, splits and partials of paged_attention_kernel and its arithmetic, rows unpacked to fp32 as they are
// staged.  Values that are not numbers are staged as zeros; which groups of which rows they are in is kept beside the tile, and a
// query row that sees one has NaN in that group's channels and no others (0 * NaN would reach every row).
__host__ __device__ inline size_t q4_smem_bytes(int E, int Ev, int F) {
    return paged_smem_bytes(E, Ev, F) + (size_t)(2 * kFmaTile + kFmaRows) * sizeof(int);
}

template <class T, int EV>
__global__ void __launch_bounds__(kFmaThreads) q4_attention_kernel(const __grid_constant__ Q4Args x) {
    const PagedArgs& a = x.p;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const int E = a.E, tid = threadIdx.x;
    FmaCore<EV> core;
    int* vis = reinterpret_cast<int*>(core.carve(smem_raw, E));    // [F] visible keys per fragment for this unit
    int* pre = vis + a.F;                                           // [F+1] tile prefix
    int* odd = pre + a.F + 1;                                       // [32] per key: value groups that are not numbers; 1 << 16: no page
    int* row_odd = odd + kFmaTile;                                  // [16] per query row: groups that have become NaN

    pdl_wait();
    pdl_trigger();
    PagedUnit u;
    if (!locate_paged_unit(a, blockIdx.x, &u)) return;
    const int split = blockIdx.y;
    const T* q = static_cast<const T*>(a.q);
    const unsigned char* kc = static_cast<const unsigned char*>(a.kcache);
    const unsigned char* vc = static_cast<const unsigned char*>(a.vcache);
    const int* table = a.block_table + (size_t)u.w * a.max_blocks;

    for (int f = tid; f < a.F; f += kFmaThreads) vis[f] = 0;
    if (tid < kFmaRows) row_odd[tid] = 0;
    __syncthreads();
    for (int i = tid; i < a.F * kFmaRows; i += kFmaThreads) {
        const int f = i / kFmaRows, r = i % kFmaRows;
        int s_abs, hq;
        if (paged_row(a, u, r, &s_abs, &hq)) {
            const int len = a.flen[f * a.len_f + u.w * a.len_w];
            const int loc = a.loc[(size_t)f * a.loc_f + (size_t)u.w * a.loc_w + s_abs];
            atomicMax(&vis[f], most_visible(a, loc, len));
        }
    }
    __syncthreads();
    if (tid == 0) {
        int acc = 0;
        for (int f = 0; f < a.F; ++f) {
            pre[f] = acc;
            acc += ceil_div(vis[f], kFmaTile);
        }
        pre[a.F] = acc;
    }
    __syncthreads();
    const int T_u = pre[a.F];
    const int t0 = (int)((int64_t)split * T_u / a.splits), t1 = (int)((int64_t)(split + 1) * T_u / a.splits);

    core.reset();
    int cur_f = -1, fscan = 0;
    for (int t = t0; t < t1; ++t) {
        while (t >= pre[fscan + 1]) ++fscan;
        const int f = fscan;
        const bool new_f = f != cur_f;
        if (new_f) {
            cur_f = f;
            for (int idx = tid; idx < kFmaRows * E; idx += kFmaThreads) {
                const int r = idx / E, e = idx - r * E;
                int s_abs, hq;
                float val = 0.f;
                if (paged_row(a, u, r, &s_abs, &hq))
                    val = Scalar<T>::to_float(q[f * a.q_f + u.w * a.q_w + s_abs * a.q_s + hq * a.q_h + e]);
                core.Qs[idx] = fabsf(val) == INFINITY ? NAN : val;        // (scores of -infinity would look like keys that are not seen)
            }
            if (tid < kFmaRows) {
                int s_abs, hq, lim = 0;
                if (paged_row(a, u, tid, &s_abs, &hq)) {
                    const int len = a.flen[f * a.len_f + u.w * a.len_w];
                    const int loc = a.loc[(size_t)f * a.loc_f + (size_t)u.w * a.loc_w + s_abs];
                    lim = most_visible(a, loc, len);
                }
                core.lim_s[tid] = lim;
            }
        }
        const int tok0 = (t - pre[f]) * kFmaTile;
        const int ntok = min(kFmaTile, vis[f] - tok0);
        if (tid < kFmaTile) odd[tid] = 0;
        __syncthreads();
        const int gk = E / kGroup, gv = EV / kGroup;
        for (int i = tid; i < kFmaTile * (gk + gv); i += kFmaThreads) {
            const int tok = i / (gk + gv), c = i - tok * (gk + gv);
            const bool value = c >= gk;
            const int g = value ? c - gk : c, groups = value ? gv : gk;
            long long row = -1;
            if (tok < ntok) row = paged_row_at(table, tok0 + tok, a.block_size, a.max_blocks, x.num_blocks, a.Hkv, u.hkv);
            uint2 code = make_uint2(0u, 0u);
            float step = 0.f;
            if (row >= 0) {
                code = *reinterpret_cast<const uint2*>((value ? vc : kc) + ((size_t)row * groups + g) * (kGroup / 2));
                const uint32_t s = (value ? x.vscale : x.kscale)[(size_t)row * groups + g];
                if (value && is_nan_e4m3(s)) atomicOr(&odd[tok], 1 << g);
                else step = from_e4m3(s) * (value ? x.vunit : 1.f);
            } else if (tok < ntok) {
                atomicOr(&odd[tok], 1 << 16);
                if (a.status && c == 0) atomicOr(a.status, STATUS_BAD_BLOCK);
            }
            float* dst = value ? core.Vs + tok * EV + g * kGroup : core.Ks + tok * (E + 1) + g * kGroup;
#pragma unroll
            for (int e = 0; e < kGroup; e += 2) {
                const float2 v = half2_of(from_e2m1x2((e < 8 ? code.x : code.y) >> (e % 8 * 4)));
                dst[e] = v.x * step;
                dst[e + 1] = v.y * step;
            }
        }
        __syncthreads();
        // (keys without a page were staged as zeros; compute() takes them out key by key)
        int any = 0;
        for (int k = 0; k < ntok; ++k) any |= odd[k];
        if (any && tid < kFmaRows) {
            int mine = 0;
            for (int k = 0; k < ntok; ++k)
                if (tok0 + k < core.lim_s[tid] && !(odd[k] >> 16)) mine |= odd[k] & 0xffff;
            row_odd[tid] |= mine;
        }
        core.compute(tok0, ntok, a.l2scale, any >> 16 ? odd : nullptr);
        __syncthreads();
    }
    __syncthreads();
    const size_t slot = (size_t)blockIdx.x * a.splits + split;
    core.flush(a.ws_o, a.ws_m, a.ws_l, slot);
    __syncthreads();
    for (int i = tid; i < kFmaRows * EV; i += kFmaThreads) {
        const int r = i / EV, e = i - r * EV;
        if (row_odd[r] >> (e / kGroup) & 1) a.ws_o[(slot * kFmaRows + r) * EV + e] = NAN;
    }
}

// One warp per output row folds the splits' partials (the grid is units x row groups).
template <class T>
__global__ void __launch_bounds__(kMergeWarps * 32) q4_merge_kernel(const __grid_constant__ PagedArgs a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    pdl_trigger();
    PagedUnit u;
    if (!locate_paged_unit(a, blockIdx.x, &u)) return;
    T* const out = static_cast<T*>(a.out);
    for (int row = blockIdx.y * kMergeWarps + warp; row < kFmaRows; row += gridDim.y * kMergeWarps) {
        int s_abs, hq;
        if (!paged_row(a, u, row, &s_abs, &hq)) continue;
        const int splits = a.splits;
#pragma unroll 1
        for (int e0 = 0; e0 < a.Ev; e0 += 128)
            merge_partials_rows<T, 1, 24>(a.ws_o, a.ws_m, a.ws_l, (size_t)blockIdx.x * a.splits, kFmaRows, a.Ev, row, splits,
                                      [splits]() { return splits; }, &out, 1,
                                      (size_t)(u.w * a.o_w + s_abs * a.o_s + hq * a.o_h), lane, e0);
    }
}

}  // namespace hogatt

// Packed prompt chunks over 4-bit pages on the tcgen05 kernel (hogatt_dense.cuh with Q4): head size 128, blocks of a multiple of eight rows.
//
// The tensor cores take both operands in one 16-bit type from swizzled shared memory, so what the TMA does for 16-bit pages a warp does
// here: one unpacks K tiles, one V tiles (128 keys).  A key is a row of 64 bytes of codes and 8 of scales, copied 32 keys at a time by
// cp.async into a ring of six such units a warp (a third K tile would lie there), converted two values per instruction, multiplied by
// their scales -- exact in fp16 -- and stored where the 128-byte swizzle wants them.  Unpacking into 16-bit pages in the workspace first would
// take four times the cache's memory.
//
// Bound by those two warps, which share their schedulers with the softmax warps: 2,048 tokens of 4,000 keys, 32 / 8 heads, fp16: 164 us (of 159,
// when that was measured, 145 were left without the copies, 120 without the conversions, 106 without either); two chunks of 512 tokens of 6,000
// keys beside six single tokens, bf16: 181 us.
// Slower: four unpacking warps of 24 (registers spill: 220 us); a third one for a quarter of both tiles, both products issued by one warp (219 us).
// 96 registers for every thread: nothing is left to take from the other warps.
//
// fp16 for both products: six significant bits times a probability; bf16 queries become fp16 once per call, a power of two per row
// taken out (q4_dense_queries_kernel), which the softmax multiplies back in.  A row's largest probability stands between 2^7 and 2^15 of fp16's range
// (the running maximum may lag by 2^8), so that those below it keep their bits down to 2^-21 of it.
//
// Values that are not numbers are stored as zeros, keys without a page as zeros too; what is special about a tile travels to the softmax
// warps in a ring of eight entries (K tiles are at most three ahead of the scores that are read), and only for such tiles they look
// the scales and the block table up again: a row that sees such a value has NaN in that group's channels.
#pragma once
#include "hogatt_dense.cuh"
#include "hogatt_q4_mma.cuh"

namespace hogatt {

// row (of all pages and heads: fewer than 2^31, 64 bytes each) of key `key` of sequence w; -1 behind the keys, -2 a key without a page
__device__ __forceinline__ int q4_dense_row(const DenseArgs& a, int w, int h, int key, int len) {
    if (key >= len) return -1;
    const int at = (int)fast_div((uint32_t)key, {a.block_mul, a.block_shift, 0u});
    const int p = at < a.max_blocks ? a.block_table[(size_t)w * a.max_blocks + at] : -1;
    if (p < 0 || p >= a.num_blocks) return -2;
    return (p * a.Hkv + h) * a.block_size + (key - at * a.block_size);
}

// Tile t (128 keys) of sequence w's K (which 0) or V (1), kv head h, into the tile at `dst`; `len` keys are seen by anybody, the segment's
// tiles are t0 ... t1 - 1.  Whole warp.  `pack`: the warp's ring of packed units of 32 keys, all but one of which are under way.  (A copy takes
// two microseconds here: with two under way a tile took four.  One unit's loads are in front of its conversions: with each load in front of
// its own, a tile took four as well.)
template <class C>
__device__ __forceinline__ void q4_unpack(const DenseArgs& a, int which, int w, int h, int t, int t0, int t1, int len, uint32_t pack, uint32_t dst,
                                          unsigned char* odd, Q4Pipe& pipe, int lane) {
    constexpr int AHEAD = C::NPACK - 1;
    // a lane's row of eight and quarter of it: eight lanes in a row are four rows and one half of their channels, which all stores below take to
    // different banks; in the ring the halves of every second pair of rows change places, for the loads
    const int r = (lane >> 4) * 4 + ((lane >> 1) & 3), q = ((lane >> 3) & 1) * 2 + (lane & 1), in_ring = r * 64 + (q ^ (r & 2)) * 16;
    const unsigned char* const codes = a.codes[which] + r * 64 + q * 16;
    // scales, two rows a lane: K's or V's by lanes 0-15; behind K's the values', to see what is special about them
    const bool second = lane >= 16;
    const unsigned char* const scales = a.scales[second ? 1 : which] + (lane & 3) * 16;
    auto look_up = [&](int window) { return q4_dense_row(a, w, h, window * 256 + lane * 8, len); };
    // the next unit's turn: its window, and its copies if it belongs to the segment: 4 groups of 8 rows (a group lies in one block), a row's four
    // 16-byte pieces by four lanes
    auto fetch = [&](int unit) {
        if ((unit & 7) == 0 && unit != 4 * t0) {
            pipe.rows = pipe.next;
            pipe.next = look_up((unit >> 3) + 1);
            pipe.before = pipe.none;
            pipe.none = __ballot_sync(0xffffffffu, pipe.rows == -2);
            if (which == 0 && pipe.none && lane == 0 && a.status) atomicOr(a.status, STATUS_BAD_BLOCK);
        }
        if (unit < 4 * t1) {
            const int left = len - unit * 32, from = (unit & 7) * 4;
            const uint32_t at = pack + (uint32_t)(unit % C::NPACK) * C::PACK_BYTES;
            if (left >= 32 && (pipe.none >> from & 0xfu) == 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    cp_async_16(at + i * 512 + in_ring, codes + (int64_t)__shfl_sync(0xffffffffu, pipe.rows, from + i) * 64, true);
                const int64_t row0 = __shfl_sync(0xffffffffu, pipe.rows, from + ((lane >> 2) & 3));
                if (!second || which == 0) cp_async_16(at + 2048 + lane * 16, scales + row0 * 8, true);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row0 = __shfl_sync(0xffffffffu, pipe.rows, from + i);
                    const bool real = row0 >= 0 && i * 8 + r < left;
                    cp_async_zfill<16>(at + i * 512 + in_ring, codes + (real ? (int64_t)row0 * 64 : 0), real);
                }
                const int row0 = __shfl_sync(0xffffffffu, pipe.rows, from + ((lane >> 2) & 3));
                const int rows = row0 >= 0 ? max(0, min(2, left - (lane & 15) * 2)) : 0;
                if (!second || which == 0)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at + 2048 + lane * 16), "l"(scales + (rows > 0 ? (int64_t)row0 * 8 : 0)), "r"(rows * 8)
                                 : "memory");
            }
        }
        cp_async_commit();
    };
    if (t == t0) {
        __syncwarp();
        pipe.rows = look_up(4 * t >> 3);
        pipe.next = look_up((4 * t >> 3) + 1);
        pipe.none = __ballot_sync(0xffffffffu, pipe.rows == -2);
        if (which == 0 && pipe.none && lane == 0 && a.status) atomicOr(a.status, STATUS_BAD_BLOCK);
#pragma unroll 1
        for (int k = 0; k < AHEAD; ++k) fetch(4 * t + k);
    }
    const uint32_t to = dst + (uint32_t)((q >> 1) * C::ATOM_BYTES + r * 128 + ((((q & 1) * 4) ^ r) * 16));       // (word k of a row: this address ^ 16 k)
    bool special = false;
#pragma unroll 1
    for (int k = 0; k < 4; ++k) {
        const int unit = 4 * t + k;
        __syncwarp();                                     // (every lane has left the unit whose place is next)
        fetch(unit + AHEAD);
        cp_async_wait<AHEAD>();
        __syncwarp();
        const uint32_t at = pack + (uint32_t)(unit % C::NPACK) * C::PACK_BYTES, from = at + in_ring, sfrom = at + 2048 + r * 8 + q * 2;
        const uint32_t put = to + k * 32 * 128;
        const uint4 w[4] = {lds128<0>(from), lds128<512>(from), lds128<1024>(from), lds128<1536>(from)};
        const uint32_t sc[4] = {lds16<0>(sfrom), lds16<64>(sfrom), lds16<128>(sfrom), lds16<192>(sfrom)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t s = sc[i];
            if (which == 1) {                             // a NaN scale becomes zero (0x7f + 1 reaches the sign bit)
                const uint32_t bits = ((s & 0x7f7fu) + 0x0101u) & 0x8080u;
                s &= ~(bits | (bits - (bits >> 7)));
            }
            s = from_e4m3x2(s);
            const uint32_t y0 = __byte_perm(s, s, 0x1010), y1 = __byte_perm(s, s, 0x3232);
            const uint32_t words[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t x[4];
                const uint32_t y = j < 2 ? y0 : y1;
                from_e2m1x8(words[j], x);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"((put ^ (16 * j)) + i * 1024), "r"(mul_half2(x[0], y)), "r"(mul_half2(x[1], y)),
                             "r"(mul_half2(x[2], y)), "r"(mul_half2(x[3], y)) : "memory");
            }
        }
        if (which == 0) {
            const uint4 v = lds128<2304>(at + (lane & 15) * 16);
            const uint32_t nan = ((v.x & 0x7f7f7f7fu) + 0x01010101u) | ((v.y & 0x7f7f7f7fu) + 0x01010101u) | ((v.z & 0x7f7f7f7fu) + 0x01010101u) |
                                 ((v.w & 0x7f7f7f7fu) + 0x01010101u);
            special = special || __any_sync(0xffffffffu, (nan & 0x80808080u) != 0);
            // four bits, one per eight keys, to bits of the unit's keys
            const uint32_t g = ~((unit >> 3 == (unit + AHEAD) >> 3 ? pipe.none : pipe.before) >> (unit & 7) * 4);
            if (lane == 0) *reinterpret_cast<volatile uint32_t*>(odd + k * 4) = ((g & 1u) | (g & 2u) << 7 | (g & 4u) << 14 | (g & 8u) << 21) * 0xffu;
        }
    }
    if (which == 0 && lane == 0) *reinterpret_cast<volatile uint32_t*>(odd + 16) = special;
    fence_proxy_async_smem();                             // generic-proxy writes before the MMA's async-proxy reads
    __syncwarp();
}

// Groups of channels in which some value of keys tok0 ... tok0 + n - 1 is not a number.
__device__ __forceinline__ uint32_t q4_odd_groups(const DenseArgs& a, int w, int h, int tok0, int n) {
    uint32_t odd = 0;
#pragma unroll 1
    for (int k = 0; k < n; ++k) {
        const int row = q4_dense_row(a, w, h, tok0 + k, INT_MAX);
        if (row < 0) continue;
#pragma unroll 1
        for (int g = 0; g < 8; ++g)
            if (is_nan_e4m3(a.scales[1][(int64_t)row * 8 + g])) odd |= 1u << g;
    }
    return odd;
}

// factor: what a row's (fragment, token, head) products are multiplied with.
// bf16: queries as fp16, the row's largest magnitude brought to [2^14, 2^15); factor is what brings its scores back, with the scale.  (One power of two
// for all fragments would be the largest one's, also of a fragment that the row does not see, where anything may stand.)  A row with an infinity or a
// NaN becomes NaN.
// fp16: queries go to the products as they are; an infinite one's scores may all be -infinity, which looks like keys that are not seen, so the
// factor of such a row is NaN.  (The pass over 2,048 tokens of 32 heads: 163.6 -> 165.6 us.)
// One warp per row, four channels per lane.  It starts beside the plan kernel, which is behind everything that may still write the queries, and ends
// after it: its first CTA does, the others make room.  (All of them waiting for the plan: the grid's later waves came behind it, these tokens 175 us.)
template <class T>
__global__ void __launch_bounds__(256) q4_dense_queries_kernel(const T* q, __half* out, float* factor, int rows, float l2scale) {
    constexpr bool half = std::is_same<T, __half>::value;
    const int lane = threadIdx.x & 31, row = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row < rows) {
        const uint2 x = *reinterpret_cast<const uint2*>(q + (size_t)row * 128 + lane * 4);
        const uint32_t mine = max(max(x.x & 0x7fff0000u, (x.x & 0x7fffu) << 16), max(x.y & 0x7fff0000u, (x.y & 0x7fffu) << 16));
        const uint32_t top = __reduce_max_sync(0xffffffffu, mine);        // the largest magnitude's bits, in the upper half
        const bool finite = top < (half ? 0x7c000000u : 0x7f800000u);
        if constexpr (half) {
            if (lane == 0) factor[row] = finite ? l2scale : NAN;
        } else {
            const int e = finite ? min(120, 14 - ((int)(top >> 23) - 127)) : 0;
            if (lane == 0) factor[row] = fmaxf(l2scale * __int_as_float((127 - e) << 23), 1e-36f);
            const float up = finite ? __int_as_float((e + 127) << 23) : NAN;
            const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(&x);
            *reinterpret_cast<uint2*>(out + (size_t)row * 128 + lane * 4) =
                make_uint2(pack2<__half>(__low2float(v[0]) * up, __high2float(v[0]) * up), pack2<__half>(__low2float(v[1]) * up, __high2float(v[1]) * up));
        }
    }
    if (blockIdx.x == 0) {
        pdl_trigger();
        pdl_wait();
    }
}

}  // namespace hogatt

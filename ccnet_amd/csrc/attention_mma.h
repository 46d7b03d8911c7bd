// What the two attentions over tokens (attention_cache.hip, attention_cross.hip) share: the transposed products S^T = K Q^T and
// O^T = V^T P^T, in which a lane keeps ONE query column through both (col = lane & 15 or & 31), so that the running maximum, the sum
// and the probabilities never change lanes: the C rows of S^T that a lane holds are exactly the contraction slots it has to feed
// as P^T, once the keys are dealt to the rows of the first product in that order.
#pragma once
#include "token_ops.h"

#ifdef __HIPCC__
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

constexpr float LOG2E = 1.44269504088896340736f;

__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// maximum / sum over the lanes l, l ^ 16, l ^ 32, l ^ 48 (the four quarters of a column)
__device__ __forceinline__ float quarters_max(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quarters_sum(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// a * b rounded by itself.  A score and the running maximum have to be the SAME rounded product: fused into score * scale - maximum, the
// rounding of the maximum alone would show as an exponent, and past 2^24 (where it is more than a power of two) as a wrong weight.
__device__ __forceinline__ float mul_rn(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}
// Eight weights as two bf16 terms, hi + lo: 2^-16 relative.  One term (2^-8) would add as much error to the result as its own rounding to bf16
// does.  Taken for few rows (one or two tiles to a workgroup), where the keys' bytes bound the kernel and it costs nothing (16 rows) to 3 % (32 rows);
// 64 rows would pay 15-30 %.  For values that are finite (codes): lo may be of either sign, or zero.
__device__ __forceinline__ void pack_two(const float* e, u32x4& hi, u32x4& lo) {
    hi = __builtin_bit_cast(u32x4, pack8(e));
    float h[8], r[8];
    unpack8(__builtin_bit_cast(uint4, hi), h);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = e[i] - h[i];
    lo = __builtin_bit_cast(u32x4, pack8(r));
}
// The same for weights >= 0 of values that may be infinite: hi is cut off one step of bf16 below e, so that lo, one to two steps, is above zero wherever
// e is and both products with an infinity have its sign (the nearest hi gave inf - inf or 0 * inf: NaN).  lo has 2^-6 of e at most: 2^-14 relative.
__device__ __forceinline__ void pack_two_above(const float* e, u32x4& hi, u32x4& lo) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t h[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            h[x] = __builtin_elementwise_sub_sat(__float_as_uint(e[2 * i + x]), 0x10000u) & 0xFFFF0000u;
            r[2 * i + x] = e[2 * i + x] - __uint_as_float(h[x]);
        }
        hi[i] = __builtin_amdgcn_perm(h[1], h[0], 0x07060302u);
    }
    lo = __builtin_bit_cast(u32x4, pack8(r));
}
// x = hi + mid + lo, three bf16 of 8 bits each: all 24 bits of a float (of its normal range)
__device__ __forceinline__ void split3(float x, float& mid_in, float& lo_in) {
    const float h = bf16_bits_to_f32(f32_to_bf16_bits(x));
    mid_in = x - h;
    lo_in = mid_in - bf16_bits_to_f32(f32_to_bf16_bits(mid_in));
}

// One split's partial result of a 16-query tile: the unnormalised O^T as D*16 floats in registers' order (groups [i][lane] of four),
// then 16 references of the weights (base 2) and 16 sums.
__host__ __device__ static inline size_t partial_floats(int D) { return (size_t)D * 16 + 32; }

// The reference m of a row's weights 2^(score - m) when its tile's largest score is mx: where that rose above m, 2^8 above it, so that O is rescaled only
// where scores rise by more than that again (some row of 16 to 64 would ask for it in nearly every tile otherwise).  Weights stay at or below 1, the
// largest at or above 2^-8: sums of weights times values have the range that weights relative to the maximum itself give them, and the relative
// precision is the same; weights below 2^-118 of a row's largest may count as zero.  A row's references depend on its own scores alone.
__device__ __forceinline__ float raised(float m, float mx) { return mx > m ? mx + 8.0f : m; }

// Two running softmaxes become one
struct Join {
    float m, a, c;  // the common reference and what each side is scaled with
    __device__ __forceinline__ Join(float m1, float m2) {
        m = fmaxf(m1, m2);
        const float base = m == -INFINITY ? 0.0f : m;
        a = __builtin_amdgcn_exp2f(m1 - base);
        c = __builtin_amdgcn_exp2f(m2 - base);
    }
};

// Which tiles of a sequence a key range takes: an even share of ITS tiles (a tile per wave at least), so that every workgroup of a ragged batch
// starts at once and the long sequences are not left for last (ranges of 2048 keys each, whatever the length: 90 instead of 75 us for 32 sequences of
// up to 8192 tokens).
struct Ranges {
    int per, used;
    __device__ __forceinline__ Ranges(int ntile, int nsplit) {
        per = max(4, (ntile + nsplit - 1) / nsplit);
        used = (ntile + per - 1) / per;
    }
};
// The host's side: as many ranges as make 512 workgroups (two to a compute unit), of eight tiles at least: below that the join costs more than it
// hides.
static inline int split_keys(long long base, long long ntile) {
    long long ns = (512 + base - 1) / base;
    if (ns > ntile / 8) ns = ntile / 8;
    return (int)(ns < 1 ? 1 : ns > 256 ? 256 : ns);
}

// Joins the partial results of the `nsplit` key ranges that a sequence used; `live`: this lane's query row exists.  One workgroup per (16-query tile, register group i): its four waves take every fourth
// split, each with a running maximum, and meet in LDS.  put(col, r, value) stores value r of the lane's group.
template <typename F>
__device__ __forceinline__ void combine_tile(const float* part, int nsplit, size_t split_stride, int D, int i, bool live, F put) {
    __shared__ f32x4 ob[3][64];
    __shared__ float mb[3][16], lb[3][16];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, col = lane & 15;
    float m = -INFINITY, l = 0.0f;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
    // four splits' loads in flight at a time (64 splits of 5 queries x 32 heads of 128: 5.6 us; one at a time: 12.5)
    for (int s0 = wave; s0 < nsplit; s0 += 16) {
        float ms[4], ls[4];
        f32x4 os[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float* p = part + (size_t)min(s0 + 4 * u, nsplit - 1) * split_stride;
            ms[u] = ls[u] = 0.0f;
            if (live && s0 + 4 * u < nsplit) {
                ms[u] = p[D * 16 + col];
                ls[u] = p[D * 16 + 16 + col];
                os[u] = ((const f32x4*)p)[i * 64 + lane];
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            // (a range that held nothing for these queries, or a sum of nothing)
            const bool any = ls[u] != 0.0f;
            const Join j(m, any ? ms[u] : -INFINITY);
            l = l * j.a + (any ? ls[u] * j.c : 0.0f);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = o[r] * j.a + (any ? os[u][r] * j.c : 0.0f);
            m = j.m;
        }
    }
    if (wave > 0) {
        ob[wave - 1][lane] = o;
        if (lane < 16) { mb[wave - 1][lane] = m; lb[wave - 1][lane] = l; }
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 0; w < 3; ++w) {
        const Join j(m, mb[w][col]);
        l = l * j.a + lb[w][col] * j.c;
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = o[r] * j.a + ob[w][lane][r] * j.c;
        m = j.m;
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) put(col, lane >> 4, r, o[r] * inv);
}
#endif  // __HIPCC__

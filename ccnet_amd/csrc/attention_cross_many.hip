// Cross attention, bfloat16 with many query rows: bound by the matrix cores (attention_cross.hip has the rest).
// Measured: 2 x 4096 queries over 8191 keys, 32/8 heads of 128: 1083 TFLOP/s (a large matrix product: 1128); heads of 64: 971, of 96: 951, of 256: 922; with a
// fifth of the keys masked, 128 dims: 933 of the unmasked work.  The matrix instructions are busy 46 % of the cycles and the vector ones 43 %: a wave's do
// not run beside each other.  Weights go into the value product as one bf16 term (2^-8): the result's error against 64 bits is 1.4 times that of its own rounding.
#include "attention_cross.h"

namespace {

// bfloat16: 32x32x16 products, 64-key tiles in two buffers, units of 32 keys.  S^T: lane (col = l & 31, half = l >> 5) holds scores of keys
// 8g + 4*half + r; O^T takes them unchanged as slots of k-step s = keys {16s + 4*half + 0..3, 16s + 8 + 4*half + 0..3}, for which two
// transposing LDS reads fetch the values.  The scores of unit u + 1 are formed while unit u goes through the softmax.
//   LDS rows of P chunks of 16 bytes.  Keys: chunk c of row r at c ^ ((r / R) & 15), R rows to a 256-byte line, so that 16 lanes that read
//   one chunk of 16 rows hit all banks; values: at c ^ ((r & 3) << 2) (64-dim rows: ((r >> 1) & 1) << 2), for the 4 rows x 64 bytes of
//   a transposing read.
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short s16x4v;
typedef __attribute__((ext_vector_type(8))) short s16x8v;

template <int DP, int QT>
__global__ __launch_bounds__(256) void cross_many_kernel(const CrossP p, int rt_n) {
    constexpr int P = DP == 96 ? 16 : DP / 8;            // chunks per LDS row
    constexpr int KS = DP / 16, DT = DP / 32;            // k-steps of S, 32-dim tiles of O
    constexpr int TILE = 64 * P * 16, NPC = P / 4;       // bytes of a tile; pieces of 1024 bytes per wave
    constexpr int RB = P * 16;                           // row bytes
    extern __shared__ __align__(16) unsigned char smem[];  // keys [2][TILE], values [2][TILE]
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int col = lane & 31, half = lane >> 5;
    int split, b, h, rt;
    many_place(p, rt_n, split, b, h, rt);
    const int D = p.D, row0 = (rt * 4 + wave) * 32 * QT;
    const int n = p.lens ? min(max(p.lens[b], 0), p.Sk) : p.Sk;
    const int ntile = (n + 63) / 64;
    const Ranges ranges(ntile, p.nsplit);
    const int t0 = split * ranges.per, t1 = min(t0 + ranges.per, ntile);
    if (split > 0 && t0 >= ntile) return;  // (range 0 always runs: it writes the zeros of an empty sequence)
    const __bf16* K = heads_at<__bf16>(p.k, b, 0, h);
    const __bf16* V = heads_at<__bf16>(p.v, b, 0, h);
    auto fk = [](int r) { return P >= 16 ? (r & 15) : P == 8 ? ((r >> 1) & 7) : ((r >> 2) & 3); };
    auto fv = [](int r) { return P >= 16 ? ((r & 3) << 2) : P == 8 ? (((r >> 1) & 1) << 2) : 0; };

    u32x4 qf[QT][KS];
#pragma unroll
    for (int j = 0; j < QT; ++j) {
        const int row = row0 + j * 32 + col;
        const int s = row / p.G;
        const __bf16* src = heads_at<__bf16>(p.q, b, row < p.rows ? s : 0, h * p.G + (row < p.rows ? row - s * p.G : 0)) + half * 8;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            qf[j][k] = u32x4{0u, 0u, 0u, 0u};
            if (row < p.rows && k * 16 + half * 8 < D) qf[j][k] = *(const u32x4*)(src + k * 16);
            if (p.neg) {
#pragma unroll
                for (int e = 0; e < 4; ++e) qf[j][k][e] ^= 0x80008000u;
            }
        }
    }
    float m[QT], l[QT];
    f32x16 o[QT][DT];
#pragma unroll
    for (int j = 0; j < QT; ++j) {
        m[j] = -INFINITY;
        l[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[j][i][r] = 0.0f;
    }
    // what this lane stages: chunk positions are fixed, rows advance with the tile's base
    unsigned ko[NPC], vo[NPC];
    int srow[NPC];
#pragma unroll
    for (int i = 0; i < NPC; ++i) {
        const int slot = (wave + 4 * i) * 64 + lane, row = slot / P, cp = slot % P;
        const int ck = cp ^ fk(row), cv = cp ^ fv(row);
        srow[i] = row;
        ko[i] = ck * 8 < D ? (unsigned)(row * (int)p.k.st + ck * 8) * 2u : PAST_END;
        vo[i] = cv * 8 < D ? (unsigned)(row * (int)p.v.st + cv * 8) * 2u : PAST_END;
    }
    auto seen_of = [&](int tile) -> unsigned long long {
        if (!p.mask) return n - tile * 64 >= 64 ? ~0ull : n - tile * 64 <= 0 ? 0ull : (1ull << (n - tile * 64)) - 1ull;
        return __builtin_amdgcn_ballot_w64(see_byte(p, b, tile * 64 + lane, n) != 0);
    };
    auto stage = [&](const __bf16* base, long long st, const unsigned* off, unsigned char* to, int tile, unsigned long long seen) {
        const __amdgpu_buffer_rsrc_t rs = rows_rsrc(base + (long long)tile * 64 * st);
#pragma unroll
        for (int i = 0; i < NPC; ++i) {
            unsigned v = off[i];
            if (seen != ~0ull) v = (seen >> srow[i]) & 1ull ? v : PAST_END;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)(to + (wave + 4 * i) * 1024), 16, (int)v, 0, 0, 0);
        }
    };
    // LDS addresses of the fragments
    unsigned ka[KS], va[DT];
    {
        const int li = lane & 15, vr = 4 * half + (li >> 2);
#pragma unroll
        for (int k = 0; k < KS; ++k) ka[k] = (unsigned)(col * RB + (((k * 2 + half) ^ fk(col)) << 4));
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            const int c = i * 4 + ((lane >> 4) & 1) * 2 + ((li & 3) >> 1);
            va[i] = (unsigned)(vr * RB + ((c ^ fv(vr)) << 4) + (li & 1) * 8);
        }
    }
    unsigned char* const kbase = smem;
    unsigned char* const vbase = smem + 2 * TILE;
    // One unit of 32 keys, in program order: a wave issues matrix instructions and vector instructions in turn, so the scores of the NEXT unit
    // (keys kn), this unit's exponentials and its products with the values (vt) are dealt into small steps by hand -- the fences keep the
    // compiler from gathering them.  Steps: KS k-steps of the next scores beside three quarters of the exponentials, DT value products
    // (keys 0..15 of the unit) beside the rest, DT value products (keys 16..31) beside the next scores' maximum.
    constexpr int NS = 16 * QT, E1 = (3 * NS / 4 + KS - 1) / KS, E2 = (NS - E1 * KS + DT - 1) / DT, M3 = (NS + DT - 1) / DT;
    float base[QT], c_use = p.scale;
    bool huge = false;
    auto unit = [&](const unsigned char* kn, const unsigned char* vt, f32x16* s, f32x16* sn, float* mx, auto fetch) {
        u32x4 pf[QT][2];
        float e[QT][16];
        // exponential i of the unit, in the order in which the products take them: keys 0..15 of every row tile first
        auto soft = [&](int i) {
            const int hf = i / (8 * QT), j = i / 8 % QT, r = hf * 8 + i % 8;
            e[j][r] = __builtin_amdgcn_exp2f(fmaf(s[j][r], c_use, -base[j]));
            l[j] += e[j][r];
            if (i % 8 == 7) pf[j][hf] = __builtin_bit_cast(u32x4, pack8(&e[j][hf * 8]));
        };
        auto vfrag = [&](int k, int i) {
            const unsigned char* a = vt + va[i] + k * 16 * RB;
            const s16x4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4v*)a);
            const s16x4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4v*)(a + 8 * RB));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        };
        if constexpr (QT * DP >= 256) {
            // queries in accumulation registers, from where the products take them as they are: left to itself the compiler copies some of them out for
            // every product (1100 -> 1056 us at 128 dims; nothing at fewer)
#pragma unroll
            for (int j = 0; j < QT; ++j)
#pragma unroll
                for (int k = 0; k < KS; ++k) asm volatile("" : "+a"(qf[j][k]));
        }
        u32x4 a[KS];
        s16x8v f[2 * DT];
        a[0] = *(const u32x4*)(kn + ka[0]);
        a[1] = *(const u32x4*)(kn + ka[1]);
#pragma unroll
        for (int j = 0; j < QT; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) sn[j][r] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            __builtin_amdgcn_sched_barrier(0);
            if (k + 2 < KS) a[k + 2] = *(const u32x4*)(kn + ka[k + 2]);
            else f[k + 2 - KS] = vfrag((k + 2 - KS) / DT, (k + 2 - KS) % DT);
#pragma unroll
            for (int j = 0; j < QT; ++j)
                sn[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a[k]), __builtin_bit_cast(bf16x8, qf[j][k]), sn[j], 0, 0, 0);
#pragma unroll
            for (int x = 0; x < E1; ++x)
                if (k * E1 + x < NS) soft(k * E1 + x);
        }
#pragma unroll
        for (int w = 0; w < 2 * DT; ++w) {
            __builtin_amdgcn_sched_barrier(0);
            const int i = w % DT;
            if (w + 2 < 2 * DT) f[w + 2] = vfrag((w + 2) / DT, (w + 2) % DT);
            else if (w + 2 == 2 * DT) fetch();  // behind the last LDS read of the unit: the compiler waits for every LDS write in flight before one
#pragma unroll
            for (int j = 0; j < QT; ++j)
                o[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, f[w]), __builtin_bit_cast(bf16x8, pf[j][w / DT]), o[j][i], 0, 0, 0);
            if (w < DT) {
#pragma unroll
                for (int x = 0; x < E2; ++x)
                    if (E1 * KS + w * E2 + x < NS) soft(E1 * KS + w * E2 + x);
            } else {
#pragma unroll
                for (int x = 0; x < M3; ++x) {
                    const int y = (w - DT) * M3 + x;
                    if (y < NS) mx[y / 16] = y % 16 ? fmaxf(mx[y / 16], sn[y / 16][y % 16]) : sn[y / 16][0];
                }
            }
        }
#pragma unroll
        for (int j = 0; j < QT; ++j) asm volatile("" : "+v"(l[j]), "+v"(mx[j]));  // sums and maxima stay in the steps they are written in
        __builtin_amdgcn_sched_barrier(0);
    };
    // Before a unit: hides keys, and moves the reference of the weights where a score rose above it (attention_mma.h: raised).
    auto settle = [&](f32x16* s, uint32_t seen, float* mx) {
        if (seen != 0xFFFFFFFFu) {
            const uint32_t mine = seen >> (4 * half);
#pragma unroll
            for (int j = 0; j < QT; ++j) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[j][r] = (mine >> (8 * (r >> 2) + (r & 3))) & 1u ? s[j][r] : -INFINITY;
                mx[j] = s[j][0];
#pragma unroll
                for (int r = 1; r < 16; ++r) mx[j] = fmaxf(mx[j], s[j][r]);
            }
        }
        bool up = false;
#pragma unroll
        for (int j = 0; j < QT; ++j) {
            auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx[j]), __float_as_uint(mx[j]), false, false);
            mx[j] = mul_rn(fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])), p.scale);
            up = up || mx[j] > m[j];
        }
        if (__builtin_amdgcn_ballot_w64(up) != 0) {
            bool far = false;
#pragma unroll
            for (int j = 0; j < QT; ++j) {
                const float mn = raised(m[j], mx[j]);
                base[j] = mn == -INFINITY ? 0.0f : mn;
                const float alpha = __builtin_amdgcn_exp2f(m[j] - base[j]);
                m[j] = mn;
                l[j] *= alpha;
                far = far || fabsf(base[j]) >= 16777216.0f;
#pragma unroll
                for (int i = 0; i < DT; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[j][i][r] *= alpha;
            }
            huge = __builtin_amdgcn_ballot_w64(far) != 0;
        }
        // s*scale - maximum as one fused operation is as good as two while the maximum's own rounding stays below one (under 2^24)
        c_use = p.scale;
        if (huge) {
#pragma unroll
            for (int j = 0; j < QT; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[j][r] = mul_rn(s[j][r], p.scale);
            c_use = 1.0f;
        }
    };
    if (t0 < t1) {
        // values of tile t + 1 are asked for at the end of tile t's first unit, keys of t + 2 at the end of its second (their buffers are
        // free by then).  The waits below would let them stay under way for a whole tile; but the compiler, which cannot tell the buffers apart, waits
        // for all of them before a unit's first transposing read, so they have the rest of their unit and the next one's first k-steps to arrive.  With a
        // mask they have less: the byte of tile t + 2 is used at once, and waiting for it waits for the keys asked for before it.
        unsigned long long seen = seen_of(t0), seen1 = t0 + 1 < t1 ? seen_of(t0 + 1) : 0ull, seen2 = 0ull;
        stage(K, p.k.st, ko, kbase, t0, seen);
        stage(V, p.v.st, vo, vbase, t0, seen);
        stage(K, p.k.st, ko, kbase + TILE, t0 + 1, seen1);  // (a tile behind the last is all hidden: zeros, nothing is read)
        __builtin_amdgcn_s_waitcnt(0x0F70 | NPC);           // vmcnt(NPC): all but the last keys
        __builtin_amdgcn_s_barrier();
        f32x16 sa[QT], sb[QT];
        float mx[QT];
#pragma unroll
        for (int j = 0; j < QT; ++j) {
            base[j] = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; ++r) sa[j][r] = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k)
                sa[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, *(const u32x4*)(kbase + ka[k])), __builtin_bit_cast(bf16x8, qf[j][k]), sa[j], 0, 0, 0);
            mx[j] = sa[j][0];
#pragma unroll
            for (int r = 1; r < 16; ++r) mx[j] = fmaxf(mx[j], sa[j][r]);
        }
        settle(sa, (uint32_t)seen, mx);
        for (int tile = t0; tile < t1; ++tile) {
            const int buf = (tile - t0) & 1;
            unsigned char* const kt = kbase + buf * TILE;
            unsigned char* const kn = kbase + (buf ^ 1) * TILE;
            unsigned char* const vt = vbase + buf * TILE;
            seen2 = tile + 2 < t1 ? seen_of(tile + 2) : 0ull;
            unit(kt + 32 * RB, vt, sa, sb, mx, [&] { stage(V, p.v.st, vo, vbase + (buf ^ 1) * TILE, tile + 1, seen1); });
            settle(sb, (uint32_t)(seen >> 32), mx);
            // this wave's keys of tile + 1 are there (only the values just asked for may be missing), its reads of kt are done
            __builtin_amdgcn_s_waitcnt(0x0070 | NPC);
            __builtin_amdgcn_s_barrier();
            unit(kn, vt + 32 * RB, sb, sa, mx, [&] { stage(K, p.k.st, ko, kt, tile + 2, seen2); });
            settle(sa, (uint32_t)seen1, mx);           // behind the last tile: all hidden, not used
            __builtin_amdgcn_s_waitcnt(0x0070 | NPC);  // the values of tile + 1
            __builtin_amdgcn_s_barrier();
            seen = seen1;
            seen1 = seen2;
        }
        __builtin_amdgcn_s_waitcnt(0x0070);  // nothing is in flight towards LDS when the workgroup ends
    }
#pragma unroll
    for (int j = 0; j < QT; ++j) {
        auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l[j]), __float_as_uint(l[j]), false, false);
        l[j] = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
        const int row = row0 + j * 32 + col;
        if (p.nsplit > 1) {
            // as 16-query tiles: lane l holds the groups of tile (col >> 4)
            const int t16 = row0 / 16 + j * 2 + (col >> 4);
            if (t16 >= p.tiles16) continue;
            float* part = p.part + ((((size_t)split * p.B + b) * p.Hk + h) * p.tiles16 + t16) * partial_floats(DP);
            if (half == 0) { part[DP * 16 + (col & 15)] = m[j]; part[DP * 16 + 16 + (col & 15)] = l[j]; }
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    ((f32x4*)part)[(i * 2 + (g >> 1)) * 64 + ((g & 1) * 2 + half) * 16 + (col & 15)] = f32x4{o[j][i][g * 4], o[j][i][g * 4 + 1], o[j][i][g * 4 + 2], o[j][i][g * 4 + 3]};
            continue;
        }
        if (row >= p.rows) continue;
        const int s = row / p.G;
        __bf16* out = heads_at<__bf16>(p.o, b, s, h * p.G + row - s * p.G);
        const float inv = l[j] != 0.0f ? 1.0f / l[j] : 0.0f;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = i * 32 + g * 8 + half * 4;
                if (d < D)
                    *(uint2*)(out + d) = make_uint2(pack_bf16x2(o[j][i][g * 4] * inv, o[j][i][g * 4 + 1] * inv), pack_bf16x2(o[j][i][g * 4 + 2] * inv, o[j][i][g * 4 + 3] * inv));
            }
    }
}

}  // namespace

int cross_launch_many_bf16(const CrossP& p, const CrossCfg& c, hipStream_t st) {
    if (c.groups == 2) return c.qt == 2 ? launch_many(cross_many_kernel<32, 2>, p, c, st) : launch_many(cross_many_kernel<32, 1>, p, c, st);
    if (c.groups == 4) return c.qt == 2 ? launch_many(cross_many_kernel<64, 2>, p, c, st) : launch_many(cross_many_kernel<64, 1>, p, c, st);
    if (c.groups == 6) return c.qt == 2 ? launch_many(cross_many_kernel<96, 2>, p, c, st) : launch_many(cross_many_kernel<96, 1>, p, c, st);
    if (c.groups == 8) return c.qt == 2 ? launch_many(cross_many_kernel<128, 2>, p, c, st) : launch_many(cross_many_kernel<128, 1>, p, c, st);
    return launch_many(cross_many_kernel<256, 1>, p, c, st);
}

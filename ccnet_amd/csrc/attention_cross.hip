// Cross attention: softmax(scale * q.k) v over keys of another length, with lengths, a key mask and shared key heads.
//
// Query rows: the Sq * G rows (s, head of the group) of one (batch, key head) share its keys, so they share tiles.  All kernels form the
// transposed products S^T = K Q^T, O^T = V^T P^T (attention_mma.h).
//   few rows (cross_few_kernel, cross_few_f32_kernel): bound by reading the keys and values.  Each wave takes its own key tiles, straight
//     from memory into registers; rows wait in registers.
//     Measured: 32 single queries over up to 1600 masked keys, 16 heads of 64, bfloat16: 24.6 us, 4.4 TB/s (a read-only pass over memory: 6.0).
//     Weights go into the value product as two bf16 terms (bfloat16, up to 32 rows) or one (above): attention_mma.h.
//   many rows (cross_many_kernel, cross_many_f32_kernel): bound by the matrix cores.  Key tiles pass through LDS, shared by the waves.
//     Measured, float32: 4096 queries over 8191 keys, 32/8 heads of 128: 133 TFLOP/s (a large matrix product: 152).
// Keys are split over workgroups where there would be few of them; a second kernel joins the parts in a fixed order.
#include "attention_cross.h"

namespace {

// ---- few rows, bfloat16.  16x16x32: a tile of 32*KS keys; lane (m, q) of sub-tile i loads key row (m >> 2)*8*KS + i*4 + (m & 3), dims
// (k >> 1)*64 + q*16 + (k & 1)*8 of k-step k, and so holds scores of keys q*8*KS .. + 8*KS - 1.  Values: the lane takes the SAME keys'
// EV dims m*EV .. (16 lanes: a whole row), and its k-step operand of product e is dim m*EV + e of eight keys: two-element permutes
// within the lane, no LDS.
template <int DC, int EV, int NQ, int KS>
__global__ __launch_bounds__(256) void cross_few_kernel(const CrossP p) {
    constexpr int NK = DC * 2, KT = 32 * KS, NI = 2 * KS, KPL = 8 * KS, EL = EV > 8 ? 8 : EV, EH = EV / EL;  // EH: halves of 128 dims
    __shared__ f32x4 ob[2][EV * 64];
    __shared__ float mb[2][16], lb[2][16];
    const int t = threadIdx.x, lane = t & 63, nw = blockDim.x >> 6;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int col = lane & 15, q = lane >> 4;
    const int split = blockIdx.x % p.nsplit, rt = blockIdx.x / p.nsplit, h = blockIdx.y, b = blockIdx.z;
    const int D = p.D;
    const int n = p.lens ? min(max(p.lens[b], 0), p.Sk) : p.Sk;
    const int ntile = (n + KT - 1) / KT;
    const Ranges ranges(ntile, p.nsplit);
    const int t0 = split * ranges.per, t1 = min(t0 + ranges.per, ntile);
    if (split > 0 && t0 >= ntile) return;  // (range 0 always runs: it writes the zeros of an empty sequence)
    const __bf16* K = heads_at<__bf16>(p.k, b, 0, h);
    const __bf16* V = heads_at<__bf16>(p.v, b, 0, h);

    u32x4 qf[NQ][NK];
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        const int row = (rt * NQ + j) * 16 + col;
        const int s = row / p.G;
        const __bf16* src = heads_at<__bf16>(p.q, b, row < p.rows ? s : 0, h * p.G + (row < p.rows ? row - s * p.G : 0));
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            const int d = (k >> 1) * 64 + q * 16 + (k & 1) * 8;
            qf[j][k] = u32x4{0u, 0u, 0u, 0u};
            if (row < p.rows && d < D) qf[j][k] = *(const u32x4*)(src + d);
            if (p.neg) {
#pragma unroll
                for (int e = 0; e < 4; ++e) qf[j][k][e] ^= 0x80008000u;
            }
        }
    }
    float m[NQ], l[NQ], base[NQ];
    f32x4 o[NQ][EV];
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        m[j] = -INFINITY;
        l[j] = base[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < EV; ++i) o[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    u32x4 kr[NI][NK];
    uint32_t vr[KPL][EV / 2];
    // Dims behind D are read again from the row's start, without a branch: keys are cleared before their use, what such values give is dropped
    int kd[NK], vd[EH];
#pragma unroll
    for (int k = 0; k < NK; ++k) kd[k] = (k >> 1) * 64 + q * 16 + (k & 1) * 8 < D ? (k >> 1) * 64 + q * 16 + (k & 1) * 8 : 0;
#pragma unroll
    for (int e = 0; e < EH; ++e) vd[e] = e * 128 + col * EL < D ? e * 128 + col * EL : 0;
    auto load_k = [&](int tile) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int key = min(tile * KT + (col >> 2) * KPL + i * 4 + (col & 3), n - 1);  // rows behind the last are hidden below
            const __bf16* a = K + (long long)key * p.k.st;
#pragma unroll
            for (int k = 0; k < NK; ++k) kr[i][k] = *(const u32x4*)(a + kd[k]);
        }
    };
    auto load_v = [&](int tile) {
#pragma unroll
        for (int i = 0; i < KPL; ++i) {
            const int key = min(tile * KT + q * KPL + i, n - 1);
            const __bf16* a = V + (long long)key * p.v.st;
#pragma unroll
            for (int e = 0; e < EH; ++e) {
                uint32_t* to = &vr[i][e * (EL / 2)];
                if constexpr (EL == 8) *(u32x4*)to = *(const u32x4*)(a + vd[e]);
                else *(uint2*)to = *(const uint2*)(a + vd[e]);
            }
        }
    };
    int tile = t0 + wave, byte = 0;
    if (tile < t1) {
        byte = see_byte(p, b, tile * KT + lane % KT, n);
        load_k(tile);
        load_v(tile);
    }
    for (; tile < t1; tile += nw) {
        const int next = tile + nw;
        unsigned long long seen = __builtin_amdgcn_ballot_w64(byte != 0);
        if constexpr (KS == 1) seen &= 0xFFFFFFFFull;
        const bool part = seen != (KS == 2 ? ~0ull : 0xFFFFFFFFull);
        if (next < t1) byte = see_byte(p, b, next * KT + lane % KT, n);
        if (D != DC * 64) {
#pragma unroll
            for (int k = 0; k < NK; ++k)
                if ((k >> 1) * 64 + q * 16 + (k & 1) * 8 >= D) {
#pragma unroll
                    for (int i = 0; i < NI; ++i) kr[i][k] = u32x4{0u, 0u, 0u, 0u};
                }
        }
        f32x4 s[NQ][NI];
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
                s[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < NK; ++k) s[j][i] = mfma16(kr[i][k], qf[j][k], s[j][i]);
            }
        if (next < t1) load_k(next);
        const uint32_t mine = (uint32_t)(seen >> (q * KPL));
        if (part) {
            // a hidden row's values may be anything: they leave as zeros
#pragma unroll
            for (int i = 0; i < KPL; ++i)
#pragma unroll
                for (int x = 0; x < EV / 2; ++x) vr[i][x] = (mine >> i) & 1u ? vr[i][x] : 0u;
        }
        constexpr int PTERMS = NQ <= 2 ? 2 : 1;  // bf16 terms of a weight (pack_two_above)
        u32x4 pf[NQ][KS][PTERMS];
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            if (part) {
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[j][i][r] = (mine >> (i * 4 + r)) & 1u ? s[j][i][r] : -INFINITY;
            }
            float mx = s[j][0][0];
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[j][i][r]);
            mx = quarters_max(mul_rn(mx, p.scale));
            if (__builtin_amdgcn_ballot_w64(mx > m[j]) != 0) {
                const float mn = raised(m[j], mx);
                base[j] = mn == -INFINITY ? 0.0f : mn;
                const float alpha = __builtin_amdgcn_exp2f(m[j] - base[j]);
                m[j] = mn;
                l[j] *= alpha;
#pragma unroll
                for (int i = 0; i < EV; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[j][i][r] *= alpha;
            }
            float e[KPL];
#pragma unroll
            for (int i = 0; i < KPL; ++i) {
                e[i] = __builtin_amdgcn_exp2f(mul_rn(s[j][i >> 2][i & 3], p.scale) - base[j]);
                l[j] += e[i];
            }
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                if constexpr (PTERMS == 2) pack_two_above(e + 8 * k, pf[j][k][0], pf[j][k][1]);
                else pf[j][k][0] = __builtin_bit_cast(u32x4, pack8(e + 8 * k));
            }
        }
#pragma unroll
        for (int e = 0; e < EV; ++e)
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                u32x4 a;
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    a[x] = __builtin_amdgcn_perm(vr[k * 8 + 2 * x + 1][e / 2], vr[k * 8 + 2 * x][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
                for (int j = 0; j < NQ; ++j)
#pragma unroll
                    for (int u = PTERMS - 1; u >= 0; --u) o[j][e] = mfma16(a, pf[j][k][u], o[j][e]);
            }
        if (next < t1) load_v(next);
    }
    // join the waves: the upper half hands its part to the lower, then wave 1 to wave 0
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        l[j] = quarters_sum(l[j]);
        for (int half = nw >> 1; half > 0; half >>= 1) {
            __syncthreads();
            if (wave >= half && wave < 2 * half) {
#pragma unroll
                for (int i = 0; i < EV; ++i) ob[wave - half][i * 64 + lane] = o[j][i];
                if (q == 0) { mb[wave - half][col] = m[j]; lb[wave - half][col] = l[j]; }
            }
            __syncthreads();
            if (wave < half) {
                const Join jn(m[j], mb[wave][col]);
                l[j] = l[j] * jn.a + lb[wave][col] * jn.c;
                m[j] = jn.m;
#pragma unroll
                for (int i = 0; i < EV; ++i) {
                    const f32x4 o2 = ob[wave][i * 64 + lane];
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[j][i][r] = o[j][i][r] * jn.a + o2[r] * jn.c;
                }
            }
        }
        const int t16 = rt * NQ + j;
        if (wave != 0 || t16 >= p.tiles16) continue;
        if (p.nsplit > 1) {
            const size_t pf_ = partial_floats(EV * 16);
            float* part = p.part + ((((size_t)split * p.B + b) * p.Hk + h) * p.tiles16 + t16) * pf_;
            if (q == 0) { part[EV * 256 + col] = m[j]; part[EV * 256 + 16 + col] = l[j]; }
            if (t16 * 16 + col < p.rows) {
#pragma unroll
                for (int i = 0; i < EV; ++i) ((f32x4*)part)[i * 64 + lane] = o[j][i];
            }
        } else {
            const int row = t16 * 16 + col;
            if (row < p.rows) {
                const int s = row / p.G;
                __bf16* out = heads_at<__bf16>(p.o, b, s, h * p.G + row - s * p.G);
                const float inv = l[j] != 0.0f ? 1.0f / l[j] : 0.0f;
#pragma unroll
                for (int i = 0; i < EV; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int d = (i / EL) * 128 + (q * 4 + r) * EL + i % EL;
                        if (d < D) store1<__bf16>(out + d, o[j][i][r] * inv);
                    }
            }
        }
    }
}

// ---- few rows, float32.  16x16x4: a tile of 16*NI keys; lane (m, q) loads key row i*16 + m, four dims at c*16 + q*4 (step x of a chunk contracts
// dims c*16 + 4q + x of the quarters), and holds scores of keys i*16 + q*4 + r.  Values: keys i*16 + q*4 + r, dims c*64 + m*4 .. + 3, product x
// takes dim m*4 + x.
template <int DC, int NQ>
__global__ __launch_bounds__(256) void cross_few_f32_kernel(const CrossP p) {
    constexpr int NC = DC * 4, EV = DC * 4, NI = DC == 4 ? 1 : 2, KT = 16 * NI;  // (32 keys of 256 dims do not fit the registers)
    constexpr uint32_t ALL = NI == 1 ? 0xFFFFu : 0xFFFFFFFFu;
    __shared__ f32x4 ob[2][EV * 64];
    __shared__ float mb[2][16], lb[2][16];
    const int t = threadIdx.x, lane = t & 63, nw = blockDim.x >> 6;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int col = lane & 15, q = lane >> 4;
    const int split = blockIdx.x % p.nsplit, rt = blockIdx.x / p.nsplit, h = blockIdx.y, b = blockIdx.z;
    const int D = p.D;
    const int n = p.lens ? min(max(p.lens[b], 0), p.Sk) : p.Sk;
    const int ntile = (n + KT - 1) / KT;
    const Ranges ranges(ntile, p.nsplit);
    const int t0 = split * ranges.per, t1 = min(t0 + ranges.per, ntile);
    if (split > 0 && t0 >= ntile) return;  // (range 0 always runs: it writes the zeros of an empty sequence)
    const float* K = heads_at<float>(p.k, b, 0, h);
    const float* V = heads_at<float>(p.v, b, 0, h);
    f32x4 qf[NQ][NC];
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        const int row = (rt * NQ + j) * 16 + col;
        const int s = row / p.G;
        const float* src = heads_at<float>(p.q, b, row < p.rows ? s : 0, h * p.G + (row < p.rows ? row - s * p.G : 0)) + q * 4;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            qf[j][c] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (row < p.rows && c * 16 + q * 4 < D) qf[j][c] = *(const f32x4*)(src + c * 16);
            if (p.neg) qf[j][c] = -qf[j][c];
        }
    }
    float m[NQ], l[NQ], base[NQ];
    f32x4 o[NQ][EV];
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        m[j] = -INFINITY;
        l[j] = base[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < EV; ++i) o[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    f32x4 kr[NI][NC], vr[NI][4][DC];
    // dims behind D: as in cross_few_kernel
    int kd[NC], vd[DC];
#pragma unroll
    for (int c = 0; c < NC; ++c) kd[c] = c * 16 + q * 4 < D ? c * 16 + q * 4 : 0;
#pragma unroll
    for (int c = 0; c < DC; ++c) vd[c] = c * 64 + col * 4 < D ? c * 64 + col * 4 : 0;
    auto load_k = [&](int tile) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const float* a = K + (long long)min(tile * KT + i * 16 + col, n - 1) * p.k.st;
#pragma unroll
            for (int c = 0; c < NC; ++c) kr[i][c] = *(const f32x4*)(a + kd[c]);
        }
    };
    auto load_v = [&](int tile) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float* a = V + (long long)min(tile * KT + i * 16 + q * 4 + r, n - 1) * p.v.st;
#pragma unroll
                for (int c = 0; c < DC; ++c) vr[i][r][c] = *(const f32x4*)(a + vd[c]);
            }
    };
    int tile = t0 + wave, byte = 0;
    if (tile < t1) {
        byte = see_byte(p, b, tile * KT + lane % KT, n);
        load_k(tile);
        load_v(tile);
    }
    for (; tile < t1; tile += nw) {
        const int next = tile + nw;
        const uint32_t seen = (uint32_t)__builtin_amdgcn_ballot_w64(byte != 0) & ALL;
        const bool part = seen != ALL;
        if (next < t1) byte = see_byte(p, b, next * KT + lane % KT, n);
        if (D != DC * 64) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (c * 16 + q * 4 >= D) {
#pragma unroll
                    for (int i = 0; i < NI; ++i) kr[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
                }
        }
        f32x4 s[NQ][NI];
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int i = 0; i < NI; ++i) s[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int j = 0; j < NQ; ++j)
#pragma unroll
                    for (int i = 0; i < NI; ++i) s[j][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[i][c][x], qf[j][c][x], s[j][i], 0, 0, 0);
        if (next < t1) load_k(next);
        if (part) {
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool see = (seen >> (i * 16 + q * 4 + r)) & 1u;
#pragma unroll
                    for (int j = 0; j < NQ; ++j) s[j][i][r] = see ? s[j][i][r] : -INFINITY;
                    if (!see) {
#pragma unroll
                        for (int c = 0; c < DC; ++c) vr[i][r][c] = f32x4{0.f, 0.f, 0.f, 0.f};
                    }
                }
        }
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            float mx = s[j][0][0];
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[j][i][r]);
            mx = quarters_max(mul_rn(mx, p.scale));
            if (__builtin_amdgcn_ballot_w64(mx > m[j]) != 0) {
                const float mn = raised(m[j], mx);
                base[j] = mn == -INFINITY ? 0.0f : mn;
                const float alpha = __builtin_amdgcn_exp2f(m[j] - base[j]);
                m[j] = mn;
                l[j] *= alpha;
#pragma unroll
                for (int i = 0; i < EV; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[j][i][r] *= alpha;
            }
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[j][i][r] = __builtin_amdgcn_exp2f(mul_rn(s[j][i][r], p.scale) - base[j]);
                    l[j] += s[j][i][r];
                }
        }
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < DC; ++c)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
#pragma unroll
                        for (int j = 0; j < NQ; ++j)
                            o[j][c * 4 + x] = __builtin_amdgcn_mfma_f32_16x16x4f32(vr[i][r][c][x], s[j][i][r], o[j][c * 4 + x], 0, 0, 0);
        if (next < t1) load_v(next);
    }
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        l[j] = quarters_sum(l[j]);
        for (int half = nw >> 1; half > 0; half >>= 1) {
            __syncthreads();
            if (wave >= half && wave < 2 * half) {
#pragma unroll
                for (int i = 0; i < EV; ++i) ob[wave - half][i * 64 + lane] = o[j][i];
                if (q == 0) { mb[wave - half][col] = m[j]; lb[wave - half][col] = l[j]; }
            }
            __syncthreads();
            if (wave < half) {
                const Join jn(m[j], mb[wave][col]);
                l[j] = l[j] * jn.a + lb[wave][col] * jn.c;
                m[j] = jn.m;
#pragma unroll
                for (int i = 0; i < EV; ++i) {
                    const f32x4 o2 = ob[wave][i * 64 + lane];
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[j][i][r] = o[j][i][r] * jn.a + o2[r] * jn.c;
                }
            }
        }
        const int t16 = rt * NQ + j;
        if (wave != 0 || t16 >= p.tiles16) continue;
        if (p.nsplit > 1) {
            float* part = p.part + ((((size_t)split * p.B + b) * p.Hk + h) * p.tiles16 + t16) * partial_floats(EV * 16);
            if (q == 0) { part[EV * 256 + col] = m[j]; part[EV * 256 + 16 + col] = l[j]; }
            if (t16 * 16 + col < p.rows) {
#pragma unroll
                for (int i = 0; i < EV; ++i) ((f32x4*)part)[i * 64 + lane] = o[j][i];
            }
        } else {
            const int row = t16 * 16 + col;
            if (row < p.rows) {
                const int s = row / p.G;
                float* out = heads_at<float>(p.o, b, s, h * p.G + row - s * p.G);
                const float inv = l[j] != 0.0f ? 1.0f / l[j] : 0.0f;
#pragma unroll
                for (int c = 0; c < DC; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int d = c * 64 + (q * 4 + r) * 4;
                        if (d < D)
                            *(float4*)(out + d) = make_float4(o[j][c * 4][r] * inv, o[j][c * 4 + 1][r] * inv, o[j][c * 4 + 2][r] * inv, o[j][c * 4 + 3][r] * inv);
                    }
            }
        }
    }
}

// Where value r of register group i, lane quarter q, lies in a row: the order of the kernel that wrote the partial results
enum { FEW_BF16, ANY_F32, MANY_BF16 };
template <typename T, int KIND>
__global__ __launch_bounds__(256) void cross_combine_kernel(const CrossP p, int groups, int kt) {
    const int i = blockIdx.x % groups, t16 = blockIdx.x / groups, h = blockIdx.y, b = blockIdx.z;
    const size_t pf = partial_floats(groups * 16);
    const float* part = p.part + (((size_t)b * p.Hk + h) * p.tiles16 + t16) * pf;
    const int n = p.lens ? min(max(p.lens[b], 0), p.Sk) : p.Sk;
    const Ranges ranges((n + kt - 1) / kt, p.nsplit);
    combine_tile(part, max(ranges.used, 1), (size_t)p.B * p.Hk * p.tiles16 * pf, groups * 16, i, t16 * 16 + (int)(threadIdx.x & 15) < p.rows, [&](int col, int q, int r, float v) {
        const int row = t16 * 16 + col, s = row / p.G, at = q * 4 + r;
        const int d = KIND == MANY_BF16 ? i * 16 + at : KIND == ANY_F32 ? (i / 4) * 64 + at * 4 + i % 4 : groups == 4 ? at * 4 + i : (i / 8) * 128 + at * 8 + i % 8;
        if (row < p.rows && d < p.D) store1<T>(heads_at<T>(p.o, b, s, h * p.G + row - s * p.G) + d, v);
    });
}

// float32, many rows: 16x16x4 products as in cross_few_f32_kernel.  Tiles of 16 keys (32 of 64 dims) in two buffers: 32 KB to 128 dims, so four workgroups share
// a compute unit and one's loads run beside another's products.  (400 x 2 heads of 64 queries over 48 keys of 128: 26.8 us; when it took 29.5, tiles
// of 32 with two workgroups took 39.8, three buffers of 16 with three workgroups 35.7.)
//   LDS rows of DC*16 chunks of 16 bytes; keys: chunk c of row r at c ^ (r & 15) (16 lanes read one chunk of 16 rows); values: in order.
template <int DC, int QT>
__global__ __launch_bounds__(256, DC <= 2 && QT == 1 ? 4 : 1) void cross_many_f32_kernel(const CrossP p, int rt_n) {
    constexpr int NI = DC == 1 ? 2 : 1, KT = 16 * NI;                         // keys of a tile
    constexpr int NC = DC * 4, EV = DC * 4, CH = DC * 16, TILE = KT * CH * 16;  // 16-byte chunks of a row; bytes of a key (or value) tile
    constexpr uint32_t ALL = NI == 1 ? 0xFFFFu : 0xFFFFFFFFu;
    extern __shared__ __align__(16) unsigned char smem[];                       // [2][keys, values]
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int col = lane & 15, q = lane >> 4;
    int split, b, h, rt;
    many_place(p, rt_n, split, b, h, rt);
    const int D = p.D, row0 = (rt * 4 + wave) * 16 * QT;
    const int n = p.lens ? min(max(p.lens[b], 0), p.Sk) : p.Sk;
    const int ntile = (n + KT - 1) / KT;
    const Ranges ranges(ntile, p.nsplit);
    const int t0 = split * ranges.per, t1 = min(t0 + ranges.per, ntile);
    if (split > 0 && t0 >= ntile) return;  // (range 0 always runs: it writes the zeros of an empty sequence)
    const float* K = heads_at<float>(p.k, b, 0, h);
    const float* V = heads_at<float>(p.v, b, 0, h);

    f32x4 qf[QT][NC];
#pragma unroll
    for (int j = 0; j < QT; ++j) {
        const int row = row0 + j * 16 + col;
        const int s = row / p.G;
        const float* src = heads_at<float>(p.q, b, row < p.rows ? s : 0, h * p.G + (row < p.rows ? row - s * p.G : 0)) + q * 4;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            qf[j][c] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (row < p.rows && c * 16 + q * 4 < D) qf[j][c] = *(const f32x4*)(src + c * 16);
            if (p.neg) qf[j][c] = -qf[j][c];
        }
    }
    float m[QT], l[QT], base[QT];
    f32x4 o[QT][EV];
#pragma unroll
    for (int j = 0; j < QT; ++j) {
        m[j] = -INFINITY;
        l[j] = base[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < EV; ++i) o[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    auto seen_of = [&](int tile) -> uint32_t {
        if (tile >= t1) return 0u;  // behind the last tile: all hidden, zeros, nothing is read
        return (uint32_t)__builtin_amdgcn_ballot_w64(see_byte(p, b, tile * KT + lane % KT, n) != 0) & ALL;
    };
    auto stage = [&](int tile, int buf, uint32_t seen) {
        const __amdgpu_buffer_rsrc_t rk = rows_rsrc(K + (long long)tile * KT * p.k.st), rv = rows_rsrc(V + (long long)tile * KT * p.v.st);
#pragma unroll
        for (int i = 0; i < DC * NI; ++i) {  // pieces of 64 chunks
            const int pc = wave + 4 * i, slot = pc * 64 + lane, row = slot / CH, cp = slot % CH, ck = cp ^ (row & 15);
            const bool see = (seen >> row) & 1u;
            const unsigned ok = see && ck * 4 < D ? (unsigned)(row * (int)p.k.st + ck * 4) * 4u : PAST_END;
            const unsigned ov = see && cp * 4 < D ? (unsigned)(row * (int)p.v.st + cp * 4) * 4u : PAST_END;
            unsigned char* at = smem + buf * 2 * TILE + pc * 1024;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_void_t*)at, 16, (int)ok, 0, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_void_t*)(at + TILE), 16, (int)ov, 0, 0, 0);
        }
    };
    if (t0 < t1) {
        uint32_t seen = seen_of(t0);
        int buf = 0;
        stage(t0, 0, seen);
        for (int tile = t0; tile < t1; ++tile) {
            const uint32_t next = seen_of(tile + 1);
            __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0): this wave's pieces of the tile are there, its reads of the other buffer are done
            __builtin_amdgcn_s_barrier();
            stage(tile + 1, buf ^ 1, next);
            const unsigned char* kt = smem + buf * 2 * TILE;
            const unsigned char* vt = kt + TILE;
            f32x4 s[QT][NI];
#pragma unroll
            for (int j = 0; j < QT; ++j)
#pragma unroll
                for (int i = 0; i < NI; ++i) s[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                f32x4 a[NI];
#pragma unroll
                for (int i = 0; i < NI; ++i) a[i] = *(const f32x4*)(kt + ((i * 16 + col) * CH + ((c * 4 + q) ^ col)) * 16);
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int i = 0; i < NI; ++i)
#pragma unroll
                        for (int j = 0; j < QT; ++j) s[j][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][x], qf[j][c][x], s[j][i], 0, 0, 0);
            }
            if (seen != ALL) {
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int j = 0; j < QT; ++j) s[j][i][r] = (seen >> (i * 16 + q * 4 + r)) & 1u ? s[j][i][r] : -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < QT; ++j) {
                float mx = s[j][0][0];
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[j][i][r]);
                mx = quarters_max(mul_rn(mx, p.scale));
                if (__builtin_amdgcn_ballot_w64(mx > m[j]) != 0) {
                    const float mn = raised(m[j], mx);
                    base[j] = mn == -INFINITY ? 0.0f : mn;
                    const float alpha = __builtin_amdgcn_exp2f(m[j] - base[j]);
                    m[j] = mn;
                    l[j] *= alpha;
#pragma unroll
                    for (int i = 0; i < EV; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[j][i][r] *= alpha;
                }
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[j][i][r] = __builtin_amdgcn_exp2f(mul_rn(s[j][i][r], p.scale) - base[j]);
                        l[j] += s[j][i][r];
                    }
            }
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int c = 0; c < DC; ++c) {
                        const f32x4 a = *(const f32x4*)(vt + ((i * 16 + q * 4 + r) * CH + c * 16 + col) * 16);
#pragma unroll
                        for (int x = 0; x < 4; ++x)
#pragma unroll
                            for (int j = 0; j < QT; ++j)
                                o[j][c * 4 + x] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[x], s[j][i][r], o[j][c * 4 + x], 0, 0, 0);
                    }
            seen = next;
            buf ^= 1;
        }
        __builtin_amdgcn_s_waitcnt(0x0070);  // nothing is in flight towards LDS when the workgroup ends
    }
#pragma unroll
    for (int j = 0; j < QT; ++j) {
        l[j] = quarters_sum(l[j]);
        const int t16 = row0 / 16 + j;
        if (t16 >= p.tiles16) continue;
        if (p.nsplit > 1) {
            float* part = p.part + ((((size_t)split * p.B + b) * p.Hk + h) * p.tiles16 + t16) * partial_floats(EV * 16);
            if (q == 0) { part[EV * 256 + col] = m[j]; part[EV * 256 + 16 + col] = l[j]; }
            if (t16 * 16 + col < p.rows) {
#pragma unroll
                for (int i = 0; i < EV; ++i) ((f32x4*)part)[i * 64 + lane] = o[j][i];
            }
            continue;
        }
        const int row = t16 * 16 + col;
        if (row >= p.rows) continue;
        const int s = row / p.G;
        float* out = heads_at<float>(p.o, b, s, h * p.G + row - s * p.G);
        const float inv = l[j] != 0.0f ? 1.0f / l[j] : 0.0f;
#pragma unroll
        for (int c = 0; c < DC; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = c * 64 + (q * 4 + r) * 4;
                if (d < D)
                    *(float4*)(out + d) = make_float4(o[j][c * 4][r] * inv, o[j][c * 4 + 1][r] * inv, o[j][c * 4 + 2][r] * inv, o[j][c * 4 + 3][r] * inv);
            }
    }
}

CrossCfg cross_cfg(int dtype, int B, int Sq, int Sk, int Hq, int Hk, int D) {
    CrossCfg c{};
    const long long rows = (long long)Sq * (Hq / Hk), pairs = (long long)B * Hk;
    const bool bf = dtype == CCNET_BF16;
    c.tiles16 = (int)((rows + 15) / 16);
    // 33 to 64 bfloat16 rows: to 64 dims they fit the registers of a few-row workgroup, which from 1024 keys on is as fast as the many-row kernel (64 pairs x 8
    // heads, 64 rows of 64: 42 against 38 us over 1400 keys, 56 / 58 over 2000, 372 / 372 over 12000) and faster under a mask (40 rows: 42 against 53 us over
    // 1500 keys, 250 / 270 over 8000); over 500 keys it is not (24 against 20 us).  Beyond 64 dims it is slower nearly throughout (64 rows of 128: 100 against
    // 82 us over 1400 keys, 231 / 214 over 4000, 425 / 415 over 8000).
    c.few = rows <= 32 || (rows <= 64 && bf && D <= 64 && Sk >= 1024);
    c.threads = 256;
    if (c.few) {
        c.groups = D <= 64 ? 4 : D <= 128 ? 8 : 16;
        c.qt = c.tiles16 > 2 ? 4 : c.tiles16 == 2 && (bf || D <= 128) ? 2 : 1;  // a second tile of float32 rows of 256 does not fit the registers
        c.rt_n = (c.tiles16 + c.qt - 1) / c.qt;
        c.kt = bf && c.qt == 1 && D <= 128 ? 64 : bf || D <= 128 ? 32 : 16;
        const long long ntile = ((long long)Sk + c.kt - 1) / c.kt;
        if (ntile <= 2) c.threads = ntile <= 1 ? 64 : 128;
        c.nsplit = split_keys(pairs * c.rt_n, ntile);
        return c;
    }
    // two row tiles per wave halve the LDS reads per product (3 to 10 % of the time); one where two would pad over a tenth more rows or leave compute
    // units without a workgroup
    auto padded = [&](long long tile) { return (rows + tile - 1) / tile * tile; };
    if (bf) {
        const int dp = D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : 256;
        c.groups = dp / 16;
        c.qt = dp <= 128 && pairs * ((rows + 255) / 256) >= 256 && 10 * padded(256) <= 11 * padded(128) ? 2 : 1;
        c.rt_n = (int)((rows + 128 * c.qt - 1) / (128 * c.qt));
        c.lds = (size_t)4 * 64 * (dp == 96 ? 256 : dp * 2);
        c.kt = 64;
    } else {
        const int dc = D <= 64 ? 1 : D <= 128 ? 2 : 4;
        c.groups = dc * 4;
        c.qt = dc <= 2 && pairs * ((rows + 127) / 128) >= 512 && 10 * padded(128) <= 11 * padded(64) ? 2 : 1;
        c.rt_n = (int)((rows + 64 * c.qt - 1) / (64 * c.qt));
        c.kt = dc == 1 ? 32 : 16;
        c.lds = (size_t)2 * 2 * c.kt * dc * 256;
    }
    c.nsplit = split_keys(pairs * c.rt_n, ((long long)Sk + c.kt - 1) / c.kt / (c.kt == 16 ? 2 : 1));  // (ranges of 256 keys at least)
    return c;
}

}  // namespace

extern "C" size_t ccnet_cross_attention_workspace_bytes(int dtype, int B, int Sq, int Sk, int Hq, int Hk, int D) {
    if (B <= 0 || Sq <= 0 || Sk <= 0 || Hq <= 0 || Hk <= 0 || D <= 0 || Hq < Hk) return 0;
    const CrossCfg c = cross_cfg(dtype, B, Sq, Sk, Hq, Hk, D);
    return c.nsplit > 1 ? (size_t)c.nsplit * B * Hk * c.tiles16 * partial_floats(c.groups * 16) * sizeof(float) : 0;
}

extern "C" int ccnet_cross_attention(ccnet_heads q, ccnet_heads k, ccnet_heads v, int dtype, int B, int Sq, int Sk, int Hq, int Hk, int D,
                                     const int32_t* lens_dev, const uint8_t* key_mask_dev, int64_t mask_sb, float scale, ccnet_heads out,
                                     void* workspace_dev, ccnet_stream stream) {
    CC_REQUIRE(cc_dtype_ok(dtype), "cross_attention: bad dtype");
    CC_REQUIRE(B >= 0 && B <= 65535 && Sq >= 0 && Sk >= 0 && Sq <= (1 << 18) && Sk <= (1 << 30), "cross_attention: bad sizes");
    CC_REQUIRE(Hk > 0 && Hq > 0 && Hq <= 4096 && (Hq % Hk) == 0, "cross_attention: query heads must be a multiple of key heads, at most 4096 (%d, %d)", Hq, Hk);
    CC_REQUIRE(D > 0 && D <= 256 && (D % 8) == 0, "cross_attention: head size must be a multiple of 8, at most 256 (got %d)", D);
    CC_REQUIRE(fabsf(scale) <= 1.0e38f, "cross_attention: the scale must be finite");
    if (B == 0 || Sq == 0) return CCNET_OK;
    CC_REQUIRE(cc_heads_ok(q, dtype, B, Sq, Hq) && cc_heads_ok(out, dtype, B, Sq, Hq), "cross_attention: q / out must be 16-byte aligned");
    CC_REQUIRE(Sk == 0 || (cc_heads_ok(k, dtype, B, Sk, Hk) && cc_heads_ok(v, dtype, B, Sk, Hk)), "cross_attention: k / v must be 16-byte aligned");
    // the tiles of the many-row kernels are addressed by 31 bits from their first row
    const int64_t far = 1 << 23;
    CC_REQUIRE((k.st >= 0 && k.st < far && v.st >= 0 && v.st < far) || Sk <= 1, "cross_attention: token strides of k / v must be below %lld elements", (long long)far);
    const CrossCfg c = cross_cfg(dtype, B, Sq, Sk, Hq, Hk, D);
    CC_REQUIRE(c.nsplit == 1 || (workspace_dev && ((uintptr_t)workspace_dev % 16) == 0), "cross_attention: a 16-byte aligned workspace is needed");
    CC_REQUIRE((long long)B * Hk * c.nsplit * c.rt_n < (1 << 23), "cross_attention: too many rows");
    const CrossP p{q, k, v, out, lens_dev, key_mask_dev, mask_sb, (float*)workspace_dev, B, Sq, Sk, Hq, Hk, Hq / Hk, D,
                   Sq * (Hq / Hk), c.tiles16, c.nsplit, scale < 0.0f ? 1 : 0, fmaxf(fabsf(scale) * LOG2E, 1.4e-45f)};  // (0 must not turn a hidden score's -inf into NaN)
    return ccnet_submit(
        [=](hipStream_t st, const float*) -> int {
            const bool bf = dtype == CCNET_BF16;
            if (c.few) {
                auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(c.rt_n * c.nsplit, Hk, B), dim3(c.threads), 0, st, p); };
                if (bf) {
                    if (D <= 64) c.qt == 1 ? go(cross_few_kernel<1, 4, 1, 2>) : c.qt == 2 ? go(cross_few_kernel<1, 4, 2, 1>) : go(cross_few_kernel<1, 4, 4, 1>);
                    else if (D <= 128) c.qt == 1 ? go(cross_few_kernel<2, 8, 1, 2>) : go(cross_few_kernel<2, 8, 2, 1>);
                    else c.qt == 1 ? go(cross_few_kernel<4, 16, 1, 1>) : go(cross_few_kernel<4, 16, 2, 1>);
                } else {
                    if (D <= 64) c.qt == 1 ? go(cross_few_f32_kernel<1, 1>) : go(cross_few_f32_kernel<1, 2>);
                    else if (D <= 128) c.qt == 1 ? go(cross_few_f32_kernel<2, 1>) : go(cross_few_f32_kernel<2, 2>);
                    else go(cross_few_f32_kernel<4, 1>);
                }
                CC_LAUNCH_CHECK();
            } else {
                int rc;
                if (bf) {
                    rc = cross_launch_many_bf16(p, c, st);
                } else {
                    if (c.groups == 4) rc = c.qt == 2 ? launch_many(cross_many_f32_kernel<1, 2>, p, c, st) : launch_many(cross_many_f32_kernel<1, 1>, p, c, st);
                    else if (c.groups == 8) rc = c.qt == 2 ? launch_many(cross_many_f32_kernel<2, 2>, p, c, st) : launch_many(cross_many_f32_kernel<2, 1>, p, c, st);
                    else rc = launch_many(cross_many_f32_kernel<4, 1>, p, c, st);
                }
                if (rc != CCNET_OK) return rc;
            }
            if (c.nsplit > 1) {
                const dim3 grid(c.tiles16 * c.groups, Hk, B);
                if (!bf) hipLaunchKernelGGL((cross_combine_kernel<float, ANY_F32>), grid, dim3(256), 0, st, p, c.groups, c.kt);
                else if (c.few) hipLaunchKernelGGL((cross_combine_kernel<__bf16, FEW_BF16>), grid, dim3(256), 0, st, p, c.groups, c.kt);
                else hipLaunchKernelGGL((cross_combine_kernel<__bf16, MANY_BF16>), grid, dim3(256), 0, st, p, c.groups, c.kt);
                CC_LAUNCH_CHECK();
            }
            return CCNET_OK;
        },
        stream, CCNET_OP_ATTENTION, 4.0 * B * Hq * Sq * (double)Sk * D, ((double)Sq * 2 * Hq + (double)Sk * 2 * Hk) * B * D * cc_esize(dtype));
}

// Attention over the 8-bit cache: softmax(scale * q . (ks kc)) (vs vc) over the pages of a sequence.
//
// The bytes of the context bound it: every code is read once per 16-64 query rows (all heads that share a cache head, all queries of
// the call: rows of one tile), straight from memory into registers in the layout that the matrix instructions take, and is exact in
// bf16 (int8: 7 bits + sign, e4m3: 4 bits), so no precision is lost behind the cache's own rounding.
//   S^T = K Q^T   16x16x32: A rows = keys, contraction = dims.  Lane (m = l & 15, q = l >> 4) of sub-tile i loads key row
//                 (m >> 2)*16 + i*4 + (m & 3) of the 64-key tile, 16 bytes at dim c*64 + q*16 (two k-steps).  With that deal of keys to rows,
//                 lane (col, q) holds scores of keys q*16 .. q*16 + 15, all of one page (a page is a multiple of 16): ONE key scale
//                 and ONE value scale per lane, and
//   O^T = V^T P^T  takes the same 16 keys as this lane's contraction slots: 16 contiguous bytes of a value row [dim][token].
// So P never leaves its lane, and nothing goes through LDS until the waves of a workgroup (each on every fourth tile) meet.
// The value scale is folded into P before it is rounded, to two bf16 terms (2^-16).  More than 48 bfloat16 rows of up to 128 dims, four tiles to a
// workgroup, take one term (2^-8, 1.4 times the plain form's error): there the second would cost matrix time.  float32 queries: q and p go in as
// three bf16 terms (24 bits), products and sums stay exact to 32 bits.
// Few rows, long contexts: the keys are split over workgroups, partial results (unnormalised O, maximum, sum) are joined by a second
// kernel in a fixed order.
// Measured: 64 contexts of 4096 tokens, 32/8 heads of 128, e4m3: 96 us, 5.6 TB/s (a read-only pass over memory: 6.0); 64 of 327 to 8192: 128 to 133 us,
// 4.4 TB/s, the last long ones run alone; one of 131071, 5 queries, int8: 53 us, 5.0 TB/s, + 6.6 us for the join.
#include "attention_mma.h"

namespace {

struct CacheAttnP {
    ccnet_heads q, o;
    const unsigned char *kc, *vc;
    const float *ks, *vs;
    const int32_t *table, *lens, *start;  // start: causal, the token of each sequence's first query; null: the queries end with the sequence
    float* part;
    int B, Sq, Hq, H, G, D, pages, page_log2, width, causal;
    int rows, tiles16, nsplit;  // rows = Sq * G query rows per (b, cache head), in tiles of 16
    int neg;                    // the softmax's scale is negative: q takes its sign
    float scale;                // its magnitude times log2(e): the softmax runs in base 2
};

template <int FMT>
__device__ __forceinline__ void widen8(uint32_t a, uint32_t b, u32x4& f);  // 8 codes -> 8 bf16
template <>
__device__ __forceinline__ void widen8<CCNET_FP8>(uint32_t a, uint32_t b, u32x4& f) {
    f[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false));
    f[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true));
    f[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false));
    f[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true));
}
template <>
__device__ __forceinline__ void widen8<CCNET_INT8>(uint32_t a, uint32_t b, u32x4& f) {
    float c[4];
    Code<CCNET_INT8>::dec4(a, c);  // at most 7 bits: the upper half of the float is its bf16
    f[0] = __builtin_amdgcn_perm(__float_as_uint(c[1]), __float_as_uint(c[0]), 0x07060302u);
    f[1] = __builtin_amdgcn_perm(__float_as_uint(c[3]), __float_as_uint(c[2]), 0x07060302u);
    Code<CCNET_INT8>::dec4(b, c);
    f[2] = __builtin_amdgcn_perm(__float_as_uint(c[1]), __float_as_uint(c[0]), 0x07060302u);
    f[3] = __builtin_amdgcn_perm(__float_as_uint(c[3]), __float_as_uint(c[2]), 0x07060302u);
}

// a 16-byte group with the bytes [n, 16) cleared
__device__ __forceinline__ u32x4 keep_bytes(u32x4 v, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = n - 4 * i;
        v[i] = k >= 4 ? v[i] : k <= 0 ? 0u : v[i] & ((1u << (8 * k)) - 1u);
    }
    return v;
}

// DC: 64-dim chunks of a head; NQ: 16-row query tiles per workgroup.
template <typename T, int FMT, int DC, int NQ>
__global__ __launch_bounds__(256, DC <= 2 && NQ == 1 ? 2 : 1) void cache_attn_kernel(const CacheAttnP p) {
    constexpr int TERMS = sizeof(T) == 4 ? 3 : 1, PTERMS = sizeof(T) == 4 ? 3 : NQ <= 2 ? 2 : 1;  // bf16 terms of a query, of a weight
    constexpr int NK = DC * 2, ND = DC * 4;
    __shared__ f32x4 ob[2][ND * 64];
    __shared__ float mb[2][16], lb[2][16];
    const int t = threadIdx.x, lane = t & 63, nw = blockDim.x >> 6;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int col = lane & 15, q = lane >> 4;
    const int split = blockIdx.x % p.nsplit, rt = blockIdx.x / p.nsplit, h = blockIdx.y, b = blockIdx.z;
    const int D = p.D, page = 1 << p.page_log2;
    const int len = max(p.lens[b], 0), n = min(len, p.width << p.page_log2);
    const int ntile = (n + 63) >> 6;
    const Ranges ranges(ntile, p.nsplit);
    const int t0 = split * ranges.per, t1 = min(t0 + ranges.per, ntile);
    if (split > 0 && t0 >= ntile) return;  // (range 0 always runs: it writes the zeros of an empty sequence)
    const int32_t* table = p.table + (long long)b * p.width;

    const int first = p.start ? min(max(p.start[b], 0), len) : 0, count = len - first;  // queries i < count are tokens first + i
    const int least = !p.causal ? n : p.start ? (count < p.Sq ? 0 : first + 1) : len - (p.Sq - 1);  // no query sees fewer keys

    // queries: B operand, column = row of the tile, k slots of (chunk c, step s): dims c*64 + q*16 + s*8 .. + 7
    u32x4 qf[NQ][NK][TERMS];
    int end[NQ];  // keys that this lane's query sees
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        const int row = (rt * NQ + j) * 16 + col;
        const bool live = row < p.rows;
        const int s = live ? row / p.G : 0, g = live ? row - s * p.G : 0;
        // (tokens past the table were dropped, their queries count)
        end[j] = !p.causal ? n : p.start ? (s < count ? min(first + s + 1, n) : 0) : min(len - (p.Sq - 1 - s), n);
        const T* src = heads_at<T>(p.q, b, s, h * p.G + g);
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            const int d = (k >> 1) * 64 + q * 16 + (k & 1) * 8;
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = 0.0f;
            if (live && d < D) Chan8<T>::load(src + d, f);
            if (p.neg) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = -f[e];
            }
            if constexpr (TERMS == 1) qf[j][k][0] = __builtin_bit_cast(u32x4, pack8(f));
            else {
                float mid[8], lo[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) split3(f[e], mid[e], lo[e]);
                qf[j][k][0] = __builtin_bit_cast(u32x4, pack8(f));
                qf[j][k][1] = __builtin_bit_cast(u32x4, pack8(mid));
                qf[j][k][2] = __builtin_bit_cast(u32x4, pack8(lo));
            }
        }
    }
    float m[NQ], l[NQ], base[NQ];
    f32x4 o[NQ][ND];
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        m[j] = -INFINITY;
        l[j] = base[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < ND; ++i) o[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // page of the 16 keys that start at key0, -1 where there are none
    auto page_of = [&](int key0) -> int { return key0 < n ? table[key0 >> p.page_log2] : -1; };
    auto valid = [&](int id) { return (unsigned)id < (unsigned)p.pages; };
    u32x4 kr[4][DC], vr[ND];
    // Dims behind D are read again from the row's start: no branch, no traffic (their queries are zeros, their output is dropped).
    int kd[DC];
#pragma unroll
    for (int c = 0; c < DC; ++c) kd[c] = c * 64 + q * 16 < D ? c * 64 + q * 16 : 0;
    auto load_k = [&](int tile, int id) {  // id: page of the quarter this lane's key rows belong to
        const long long blk = (long long)(valid(id) ? id : 0) * p.H + h;
        const int tok = (tile * 64 + (col >> 2) * 16 + (col & 3)) & (page - 1);
        const unsigned char* a = p.kc + ((blk << p.page_log2) + tok) * D;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < DC; ++c) kr[i][c] = *(const u32x4*)(a + i * 4 * D + kd[c]);
    };
    auto load_v = [&](int tile, int id) {  // id: page of this lane's own quarter
        const long long blk = (long long)(valid(id) ? id : 0) * p.H + h;
        const int tok = (tile * 64 + q * 16) & (page - 1);
        const unsigned char* a = p.vc + (((blk * D) + col) << p.page_log2) + tok;
#pragma unroll
        for (int i = 0; i < ND; ++i) vr[i] = *(const u32x4*)(a + ((i * 16 < D ? i * 16 : 0) << p.page_log2));
    };
    auto load_scales = [&](int id, float& ks, float& vs) {
        const long long blk = (long long)(valid(id) ? id : 0) * p.H + h;
        ks = p.ks[blk];
        vs = p.vs[blk];
    };
    int tile = t0 + wave;
    // pages are looked up two tiles ahead, keys asked for one ahead (when this tile's scores are formed), values when they are free
    int idk = -1, idv = -1, idk1 = -1, idv1 = -1;
    float ksc = 0.0f, vsc = 0.0f;
    if (tile < t1) {
        idk = page_of(tile * 64 + (col >> 2) * 16);
        idv = page_of(tile * 64 + q * 16);
        idk1 = page_of((tile + nw) * 64 + (col >> 2) * 16);
        idv1 = page_of((tile + nw) * 64 + q * 16);
        load_k(tile, idk);
        load_v(tile, idv);
        load_scales(idv, ksc, vsc);
    }
    for (; tile < t1; tile += nw) {
        const int next = tile + nw;
        const int idk2 = page_of((next + nw) * 64 + (col >> 2) * 16), idv2 = page_of((next + nw) * 64 + q * 16);
        f32x4 s[NQ][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < NQ; ++j) s[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                u32x4 a0, a1;
                widen8<FMT>(kr[i][c][0], kr[i][c][1], a0);
                widen8<FMT>(kr[i][c][2], kr[i][c][3], a1);
#pragma unroll
                for (int j = 0; j < NQ; ++j)
#pragma unroll
                    for (int u = TERMS - 1; u >= 0; --u) {
                        s[j][i] = mfma16(a0, qf[j][2 * c][u], s[j][i]);
                        s[j][i] = mfma16(a1, qf[j][2 * c + 1][u], s[j][i]);
                    }
            }
        }
        const float kf = ksc * p.scale, vf = vsc;
        const int key0 = tile * 64 + q * 16;
        const bool there = valid(idv);
        // a tile that some query of the call sees only in part: its end, the causal edge, or a page that is not there
        const bool part = (tile + 1) * 64 > min(least, n) || __builtin_amdgcn_ballot_w64(!there) != 0;
        if (next < t1) {
            load_k(next, idk1);
            load_scales(idv1, ksc, vsc);
        }
        if (part) {
            const int keep = there ? n - key0 : 0;
#pragma unroll
            for (int i = 0; i < ND; ++i) vr[i] = keep_bytes(vr[i], keep);
        }
        u32x4 pf[NQ][2][PTERMS];
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            float fv = vf;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[j][i][r] = mul_rn(s[j][i][r], kf);
            if (part) {
                // hidden keys: -inf.  A lane that sees none of its keys also drops their block's value scale (which may be NaN)
                const int lim = there ? end[j] - key0 : 0;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[j][i][r] = i * 4 + r < lim ? s[j][i][r] : -INFINITY;
                if (lim <= 0) fv = 0.0f;
            }
            float mx = s[j][0][0];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[j][i][r]);
            mx = quarters_max(mx);
            if (__builtin_amdgcn_ballot_w64(mx > m[j]) != 0) {
                const float mn = raised(m[j], mx);
                base[j] = mn == -INFINITY ? 0.0f : mn;
                const float alpha = __builtin_amdgcn_exp2f(m[j] - base[j]);
                m[j] = mn;
                l[j] *= alpha;
#pragma unroll
                for (int i = 0; i < ND; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[j][i][r] *= alpha;
            }
            float e[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float x = __builtin_amdgcn_exp2f(s[j][i >> 2][i & 3] - base[j]);
                l[j] += x;
                e[i] = x * fv;
            }
            if constexpr (PTERMS == 1) {
                pf[j][0][0] = __builtin_bit_cast(u32x4, pack8(e));
                pf[j][1][0] = __builtin_bit_cast(u32x4, pack8(e + 8));
            } else if constexpr (PTERMS == 2) {
                pack_two(e, pf[j][0][0], pf[j][0][1]);
                pack_two(e + 8, pf[j][1][0], pf[j][1][1]);
            } else {
                float mid[16], lo[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) split3(e[i], mid[i], lo[i]);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    pf[j][k][0] = __builtin_bit_cast(u32x4, pack8(e + 8 * k));
                    pf[j][k][1] = __builtin_bit_cast(u32x4, pack8(mid + 8 * k));
                    pf[j][k][2] = __builtin_bit_cast(u32x4, pack8(lo + 8 * k));
                }
            }
        }
#pragma unroll
        for (int i = 0; i < ND; ++i) {
            u32x4 a0, a1;
            widen8<FMT>(vr[i][0], vr[i][1], a0);
            widen8<FMT>(vr[i][2], vr[i][3], a1);
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int u = PTERMS - 1; u >= 0; --u) {
                    o[j][i] = mfma16(a0, pf[j][0][u], o[j][i]);
                    o[j][i] = mfma16(a1, pf[j][1][u], o[j][i]);
                }
        }
        if (next < t1) load_v(next, idv1);
        idv = idv1;
        idk1 = idk2;
        idv1 = idv2;
    }
    // join the waves: the upper half hands its part to the lower, then wave 1 to wave 0
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        l[j] = quarters_sum(l[j]);
        for (int half = nw >> 1; half > 0; half >>= 1) {
            __syncthreads();
            if (wave >= half && wave < 2 * half) {
                const int w = wave - half;
#pragma unroll
                for (int i = 0; i < ND; ++i) ob[w][i * 64 + lane] = o[j][i];
                if (q == 0) { mb[w][col] = m[j]; lb[w][col] = l[j]; }
            }
            __syncthreads();
            if (wave < half) {
                const Join jn(m[j], mb[wave][col]);
                l[j] = l[j] * jn.a + lb[wave][col] * jn.c;
                m[j] = jn.m;
#pragma unroll
                for (int i = 0; i < ND; ++i) {
                    const f32x4 o2 = ob[wave][i * 64 + lane];
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[j][i][r] = o[j][i][r] * jn.a + o2[r] * jn.c;
                }
            }
        }
        const int t16 = rt * NQ + j;
        if (wave != 0 || t16 >= p.tiles16) continue;
        if (p.nsplit > 1) {
            float* part = p.part + (((size_t)split * p.B + b) * p.H + h) * p.tiles16 * partial_floats(D) + (size_t)t16 * partial_floats(D);
            if (q == 0) { part[D * 16 + col] = m[j]; part[D * 16 + 16 + col] = l[j]; }
            if (t16 * 16 + col < p.rows) {
#pragma unroll
                for (int i = 0; i < ND; ++i)
                    if (i * 16 < D) ((f32x4*)part)[i * 64 + lane] = o[j][i];
            }
        } else {
            const int row = t16 * 16 + col;
            if (row < p.rows) {
                const int s = row / p.G, g = row - s * p.G;
                T* out = heads_at<T>(p.o, b, s, h * p.G + g);
                const float inv = l[j] != 0.0f ? 1.0f / l[j] : 0.0f;
#pragma unroll
                for (int i = 0; i < ND; ++i)
                    if (i * 16 < D) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) store1<T>(out + i * 16 + q * 4 + r, o[j][i][r] * inv);
                    }
            }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void cache_combine_kernel(const CacheAttnP p) {
    const int nd = p.D / 16, i = blockIdx.x % nd, t16 = blockIdx.x / nd, h = blockIdx.y, b = blockIdx.z;
    const size_t pf = partial_floats(p.D);
    const float* part = p.part + ((size_t)b * p.H + h) * p.tiles16 * pf + (size_t)t16 * pf;
    const int n = min(max(p.lens[b], 0), p.width << p.page_log2);
    const Ranges ranges((n + 63) >> 6, p.nsplit);
    combine_tile(part, max(ranges.used, 1), (size_t)p.B * p.H * p.tiles16 * pf, p.D, i, t16 * 16 + (int)(threadIdx.x & 15) < p.rows, [&](int col, int q, int r, float v) {
        const int row = t16 * 16 + col;
        if (row >= p.rows) return;
        const int s = row / p.G;
        store1<T>(heads_at<T>(p.o, b, s, h * p.G + row - s * p.G) + i * 16 + q * 4 + r, v);
    });
}

struct CacheCfg {
    int tiles16, dc, nq, rt, nsplit;  // 16-row query tiles, 64-dim chunks, tiles per workgroup, workgroups along the rows, key ranges
};
CacheCfg cache_cfg(int dtype, int B, int Sq, int Hq, int H, int D, int width, int page) {
    CacheCfg c;
    const long long rows = (long long)Sq * (Hq / H);
    c.tiles16 = (int)((rows + 15) / 16);
    c.dc = D <= 64 ? 1 : D <= 128 ? 2 : 4;
    // query tiles per workgroup: as many as there are, up to what the registers hold without spilling
    const int most = dtype == CCNET_BF16 ? (c.dc == 4 ? 2 : 4) : c.dc == 4 ? 1 : 2;
    c.nq = c.tiles16 >= 4 ? 4 : c.tiles16 >= 2 ? 2 : 1;
    if (c.nq > most) c.nq = most;
    c.rt = (c.tiles16 + c.nq - 1) / c.nq;
    c.nsplit = split_keys((long long)B * H * c.rt, ((long long)width * page + 63) / 64);
    return c;
}

}  // namespace

extern "C" size_t ccnet_cache_attention_workspace_bytes(int B, int Sq, int Hq, int H, int D, int width, int page) {
    if (B <= 0 || Sq <= 0 || Hq <= 0 || H <= 0 || D <= 0 || width <= 0 || page <= 0 || Hq < H) return 0;
    const CacheCfg c = cache_cfg(CCNET_BF16, B, Sq, Hq, H, D, width, page);  // float32 has as many workgroups or more, so no more ranges
    return c.nsplit > 1 ? (size_t)c.nsplit * B * H * c.tiles16 * partial_floats(D) * sizeof(float) : 0;
}

static int cache_attention(ccnet_heads q, int dtype, int B, int Sq, int Hq, const void* kc_dev, const void* vc_dev, const float* ks_dev,
                                     const float* vs_dev, int fmt, int pages, int H, int page, int D, const int32_t* table_dev, int width,
                                     const int32_t* lens_dev, const int32_t* start_dev, float scale, int causal, ccnet_heads out, void* workspace_dev, ccnet_stream stream) {
    CC_REQUIRE(cc_dtype_ok(dtype) && cc_code_ok(fmt), "cache_attention: bad dtype");
    CC_REQUIRE(B >= 0 && B <= 65535 && Sq >= 0 && Sq <= (1 << 16), "cache_attention: bad sizes");
    CC_REQUIRE(H > 0 && Hq > 0 && Hq <= 4096 && (Hq % H) == 0, "cache_attention: query heads must be a multiple of cache heads, at most 4096 (%d, %d)", Hq, H);
    CC_REQUIRE(D > 0 && D <= 256 && (D % 16) == 0, "cache_attention: head size must be a multiple of 16, at most 256 (got %d)", D);
    CC_REQUIRE(page == 16 || page == 32 || page == 64 || page == 128, "cache_attention: a page holds 16, 32, 64 or 128 tokens (got %d)", page);
    CC_REQUIRE(pages >= 0 && width >= 0 && (long long)width * page <= (1 << 30), "cache_attention: bad page table");
    CC_REQUIRE(fabsf(scale) <= 1.0e38f, "cache_attention: the scale must be finite");
    if (B == 0 || Sq == 0) return CCNET_OK;
    CC_REQUIRE(lens_dev && (width == 0 || table_dev) && (pages == 0 || (kc_dev && vc_dev && ks_dev && vs_dev)), "cache_attention: null pointer");
    CC_REQUIRE(((uintptr_t)kc_dev % 16) == 0 && ((uintptr_t)vc_dev % 16) == 0, "cache_attention: codes must be 16-byte aligned");
    CC_REQUIRE(cc_heads_ok(q, dtype, B, Sq, Hq) && cc_heads_ok(out, dtype, B, Sq, Hq), "cache_attention: q / out must be 16-byte aligned");
    const CacheCfg c = cache_cfg(dtype, B, Sq, Hq, H, D, pages ? width : 0, page);
    CC_REQUIRE(c.nsplit == 1 || (workspace_dev && ((uintptr_t)workspace_dev % 16) == 0), "cache_attention: a 16-byte aligned workspace is needed");
    CacheAttnP p{q, out, (const unsigned char*)kc_dev, (const unsigned char*)vc_dev, ks_dev, vs_dev, table_dev, lens_dev, start_dev, (float*)workspace_dev,
                 B, Sq, Hq, H, Hq / H, D, pages, 0, pages ? width : 0, causal ? 1 : 0, Sq * (Hq / H), c.tiles16, c.nsplit,
                 scale < 0.0f ? 1 : 0, fabsf(scale) * LOG2E};
    while ((1 << p.page_log2) < page) ++p.page_log2;
    CC_REQUIRE((long long)c.rt * c.nsplit < (1 << 23) && (long long)c.tiles16 * (D / 16) < (1 << 23), "cache_attention: too many rows");
    const int threads = (long long)p.width * page <= 128 ? 64 : 256;  // one or two tiles of keys: one wave
    return ccnet_submit(
        [=](hipStream_t st, const float*) -> int {
            auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(c.rt * c.nsplit, H, B), dim3(threads), 0, st, p); };
            auto by_nq = [&](auto* ty, auto fm, auto d) {
                using Ty = std::remove_pointer_t<decltype(ty)>;
                constexpr int FM = decltype(fm)::value, DCH = decltype(d)::value;
                if constexpr (sizeof(Ty) == 2 && DCH < 4) {
                    if (c.nq == 4) return go(cache_attn_kernel<Ty, FM, DCH, 4>);
                }
                if constexpr (sizeof(Ty) == 2 || DCH < 4) {
                    if (c.nq == 2) return go(cache_attn_kernel<Ty, FM, DCH, 2>);
                }
                go(cache_attn_kernel<Ty, FM, DCH, 1>);
            };
            auto by_d = [&](auto* ty, auto fm) {
                if (c.dc == 1) by_nq(ty, fm, std::integral_constant<int, 1>());
                else if (c.dc == 2) by_nq(ty, fm, std::integral_constant<int, 2>());
                else by_nq(ty, fm, std::integral_constant<int, 4>());
            };
            auto by_fmt = [&](auto* ty) {
                if (fmt == CCNET_INT8) by_d(ty, std::integral_constant<int, CCNET_INT8>());
                else by_d(ty, std::integral_constant<int, CCNET_FP8>());
            };
            if (dtype == CCNET_BF16) by_fmt((__bf16*)nullptr);
            else by_fmt((float*)nullptr);
            CC_LAUNCH_CHECK();
            if (c.nsplit > 1) {
                const dim3 grid(c.tiles16 * (D / 16), H, B);
                if (dtype == CCNET_BF16) hipLaunchKernelGGL(cache_combine_kernel<__bf16>, grid, dim3(256), 0, st, p);
                else hipLaunchKernelGGL(cache_combine_kernel<float>, grid, dim3(256), 0, st, p);
                CC_LAUNCH_CHECK();
            }
            return CCNET_OK;
        },
        stream, CCNET_OP_ATTENTION, 4.0 * B * Sq * Hq * (double)width * page * D, 2.0 * B * Sq * Hq * D * cc_esize(dtype) + 2.0 * B * (double)width * page * H * D);
}

extern "C" int ccnet_cache_attention(ccnet_heads q, int dtype, int B, int Sq, int Hq, const void* kc_dev, const void* vc_dev, const float* ks_dev,
                                     const float* vs_dev, int fmt, int pages, int H, int page, int D, const int32_t* table_dev, int width,
                                     const int32_t* lens_dev, float scale, int causal, ccnet_heads out, void* workspace_dev, ccnet_stream stream) {
    return cache_attention(q, dtype, B, Sq, Hq, kc_dev, vc_dev, ks_dev, vs_dev, fmt, pages, H, page, D, table_dev, width, lens_dev, nullptr, scale, causal, out,
                           workspace_dev, stream);
}

extern "C" int ccnet_cache_attention_from(ccnet_heads q, int dtype, int B, int Sq, int Hq, const void* kc_dev, const void* vc_dev, const float* ks_dev,
                                          const float* vs_dev, int fmt, int pages, int H, int page, int D, const int32_t* table_dev, int width,
                                          const int32_t* lens_dev, const int32_t* start_dev, float scale, ccnet_heads out, void* workspace_dev,
                                          ccnet_stream stream) {
    CC_REQUIRE(start_dev || B == 0 || Sq == 0, "cache_attention: null start");
    return cache_attention(q, dtype, B, Sq, Hq, kc_dev, vc_dev, ks_dev, vs_dev, fmt, pages, H, page, D, table_dev, width, lens_dev, start_dev, scale, 1, out,
                           workspace_dev, stream);
}

// The 8-bit key/value cache: quantised as it is written, and read back.
//   A block = the tokens of one page x one head, with one scale for its keys and one for its values.
//   write:  s' = max(s of the tokens already there, max|new| / Q);  code = round(x / s');  codes already there, where s' > s:
//           round(code * s / s').   read:  code * s.
// Keys lie [page][head][token][dim], values [page][head][dim][token]: that is how cache_attention's matrix instructions take them
// (dims are the contraction of q.k, tokens that of p.v), so the transposition is paid once, here.
// Both directions move bytes and do little else: memory bound.  Measured: 6 prompts of up to 4096 tokens x 8 heads of 128 from bfloat16 to e4m3 21.8 us
// (75 MB, 3.4 TB/s); 8 x up to 8192 tokens back to bfloat16 47.6 us (210 MB, 4.4 TB/s).
#include "token_ops.h"

namespace {

struct CacheP {
    ccnet_heads k, v;          // write: sources; read: destinations
    unsigned char *kc, *vc;
    float *ks, *vs;
    const int32_t *table, *start, *lens;
    int B, T, H, D, pages, page, page_log2, width;
    int slots, tile;  // workgroups along a sequence, and (read) the tokens of one
};

// the scale below which a block counts as zero: 1 / scale has to stay finite
constexpr float SCALE_MIN = 1.17549435e-38f;

__device__ __forceinline__ float amax_nan(float a, float b) { return (b > a || b != b) ? b : a; }  // keeps a NaN

// Quantises 16 values into a 16-byte group
template <int FMT>
__device__ __forceinline__ uint4 enc16(const float* f, float inv, bool finite) {
    float g[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) g[i] = finite ? f[i] * inv : 0.0f;
    return make_uint4(Code<FMT>::enc4(g), Code<FMT>::enc4(g + 4), Code<FMT>::enc4(g + 8), Code<FMT>::enc4(g + 12));
}
template <int FMT>
__device__ __forceinline__ void dec16(const uint4& c, float s, float* f) {
    Code<FMT>::dec4(c.x, f); Code<FMT>::dec4(c.y, f + 4); Code<FMT>::dec4(c.z, f + 8); Code<FMT>::dec4(c.w, f + 12);
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] *= s;
}

// 16 bytes of a row: PC = 8 bfloat16 or 4 float32 values, and their PC codes
template <typename T>
__device__ __forceinline__ void load_piece(const T* p, float* f) {
    if constexpr (sizeof(T) == 2) Chan8<T>::load(p, f);
    else {
        const float4 v = *(const float4*)p;
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    }
}
// Two neighbouring dims of one token
template <typename T>
__device__ __forceinline__ float2 load2(const T* p) {
    if constexpr (sizeof(T) == 4) return *(const float2*)p;
    else {
        const uint32_t v = *(const uint32_t*)p;
        return make_float2(bf16_bits_to_f32(v & 0xFFFFu), bf16_bits_to_f32(v >> 16));
    }
}

// One workgroup per (page slot of a sequence, head, keys / values).  The block's new tokens are read once and wait in registers for the largest
// magnitude: a thread holds N groups of 32 values -- of the keys 16-byte pieces of rows (neighbouring threads, neighbouring pieces), of the values 16
// tokens of two dims, which leave transposed as 16-byte stores.
template <typename T, int FMT, int N>
__global__ __launch_bounds__(256) void cache_write_kernel(const CacheP p) {
    constexpr int PC = 16 / sizeof(T), NP = 32 / PC;
    __shared__ float red[4];
    const int t = threadIdx.x, nt = blockDim.x, b = blockIdx.y, isv = blockIdx.z;
    const int h = blockIdx.x % p.H, slot = blockIdx.x / p.H;  // heads side by side: their rows are neighbours in memory
    const int page = p.page, D = p.D;
    const int cap = p.width * page;
    const int s0 = min(max(p.start[b], 0), cap);
    const int n = p.lens ? min(max(p.lens[b], 0), p.T) : p.T;
    const int end = min(s0 + n, cap);
    const int first = ((s0 >> p.page_log2) + slot) << p.page_log2;  // the page's first token
    if (n == 0 || first >= end) return;
    const int id = p.table[(long long)b * p.width + (first >> p.page_log2)];
    const int a = max(s0 - first, 0), z = min(end - first, page);  // new tokens of the page: [a, z); [0, a) are there already
    const ccnet_heads& src = isv ? p.v : p.k;
    const T* const rows = heads_at<T>(src, b, first - s0, h);      // token i of the page is source row first - s0 + i
    const int G = D / 16, D2 = D / 2, c0 = a / 16, P = D / PC, items = isv ? ((z + 15) / 16 - c0) * D2 : (z - a) * P;
    const float inv_d2 = 1.0f / (float)D2, inv_p = 1.0f / (float)P;  // e / P and e / D2 by them: e < 2^14, far from a tie
    float f[N][2][16];
    float m = 0.0f;
#pragma unroll
    for (int u = 0; u < N; ++u)
        if (isv) {
            const int e = t + u * nt, r = (int)(((float)e + 0.5f) * inv_d2), c = c0 + r, d = (e - r * D2) * 2;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int k = c * 16 + i;
                float2 x = make_float2(0.0f, 0.0f);
                if (e < items && k >= a && k < z) x = load2<T>(rows + (long long)k * src.st + d);
                f[u][0][i] = x.x;
                f[u][1][i] = x.y;
                m = amax_nan(m, fabsf(x.x));
                m = amax_nan(m, fabsf(x.y));
            }
        } else {
#pragma unroll
            for (int v = 0; v < NP; ++v) {
                const int e = t + (u * NP + v) * nt, r = (int)(((float)e + 0.5f) * inv_p);
                float* x = &f[u][0][0] + v * PC;
#pragma unroll
                for (int q = 0; q < PC; ++q) x[q] = 0.0f;
                if (e < items) load_piece<T>(rows + (long long)(a + r) * src.st + (e - r * P) * PC, x);
#pragma unroll
                for (int q = 0; q < PC; ++q) m = amax_nan(m, fabsf(x[q]));
            }
        }
    if ((unsigned)id >= (unsigned)p.pages) return;  // (looked up while the tokens were on their way)
    const long long blk = (long long)id * p.H + h;
    unsigned char* codes = (isv ? p.vc : p.kc) + blk * page * D;
    float* scale_at = (isv ? p.vs : p.ks) + blk;
    const float was = a > 0 ? *scale_at : 0.0f;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = amax_nan(m, __shfl_xor(m, o, 64));
    if ((t & 63) == 0) red[t >> 6] = m;
    __syncthreads();  // (every thread also has the old scale)
    m = red[0];
    for (int w = 1; w < nt / 64; ++w) m = amax_nan(m, red[w]);
    float sc = amax_nan(was, m * (1.0f / Code<FMT>::qmax));
    if (sc < SCALE_MIN) sc = 0.0f;
    const bool finite = sc - sc == 0.0f;
    const float inv = sc > 0.0f ? 1.0f / sc : 0.0f;
    const bool redo = a > 0 && !(sc == was);  // the scale grew: the codes already there are rounded again
    if (t == 0) *scale_at = sc;
    if (!isv) {
        if (redo)
            for (int e = t; e < a * G; e += nt) {
                uint4* c = (uint4*)(codes + (size_t)e * 16);
                float x[16];
                dec16<FMT>(*c, was, x);
                *c = enc16<FMT>(x, inv, finite);
            }
#pragma unroll
        for (int u = 0; u < N * NP; ++u) {
            const int e = t + u * nt;
            if (e >= items) continue;
            const float* x = &f[u / NP][0][0] + (u % NP) * PC;
            float y[PC];
#pragma unroll
            for (int q = 0; q < PC; ++q) y[q] = finite ? x[q] * inv : 0.0f;
            uint32_t* to = (uint32_t*)(codes + (size_t)a * D + (size_t)e * PC);
            if constexpr (PC == 8) *(uint2*)to = make_uint2(Code<FMT>::enc4(y), Code<FMT>::enc4(y + 4));
            else *to = Code<FMT>::enc4(y);
        }
        return;
    }
    if (redo)
        for (int e = t; e < c0 * D; e += nt) {  // (whole groups of tokens before the first new one's)
            uint4* c = (uint4*)(codes + (size_t)(e / c0) * page + (e % c0) * 16);
            float x[16];
            dec16<FMT>(*c, was, x);
            *c = enc16<FMT>(x, inv, finite);
        }
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int e = t + u * nt, r = (int)(((float)e + 0.5f) * inv_d2), c = c0 + r, d = (e - r * D2) * 2;
        if (e >= items) continue;
        const int keep = a - c * 16, last = z - c * 16;  // new tokens of the group: [keep, last)
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            uint4* at = (uint4*)(codes + (size_t)(d + v) * page + c * 16);
            uint4 now = enc16<FMT>(f[u][v], inv, finite);
            if (keep > 0 || last < 16) {
                // those before them keep their codes, or get them rounded again; those behind keep theirs
                const uint4 o = *at;
                uint4 r = o;
                if (redo) {
                    float x[16];
                    dec16<FMT>(o, was, x);
                    r = enc16<FMT>(x, inv, finite);
                }
                uint32_t ow[4] = {o.x, o.y, o.z, o.w}, rw[4] = {r.x, r.y, r.z, r.w}, nw[4] = {now.x, now.y, now.z, now.w};
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint32_t mask = 0xFFu << (8 * (i & 3));
                    const uint32_t from = i < keep ? rw[i >> 2] : i >= last ? ow[i >> 2] : nw[i >> 2];
                    nw[i >> 2] = (nw[i >> 2] & ~mask) | (from & mask);
                }
                now = make_uint4(nw[0], nw[1], nw[2], nw[3]);
            }
            *at = now;
        }
    }
}

// One workgroup per (tile of p.tile tokens, head, keys / values); a tile may hold several pages or part of one.  Values: a thread
// takes 16 tokens of four dims (four 16-byte loads) and stores four neighbouring dims of each token.
template <typename T, int FMT>
__global__ __launch_bounds__(256) void cache_read_kernel(const CacheP p) {
    const int t = threadIdx.x, b = blockIdx.y, isv = blockIdx.z;
    const int h = blockIdx.x % p.H, slot = blockIdx.x / p.H;  // heads side by side: their rows are neighbours in memory
    const int page = p.page, D = p.D;
    const int n = min(min(max(p.lens[b], 0), p.T), p.width * page);
    const int first = slot * p.tile;
    if (first >= n) return;
    const int z = min(n - first, p.tile);
    const int32_t* table = p.table + (long long)b * p.width;
    if (!isv) {
        // 16 bytes out per thread, neighbouring threads side by side; four pieces' look-ups and loads in flight at a time
        constexpr int PC = 16 / sizeof(T), U = 4;
        const int P = D / PC, items = z * P;
        const float inv_p = 1.0f / (float)P;
        for (int e0 = t; e0 < items; e0 += 256 * U) {
            int i[U], g[U], id[U];
            uint32_t c[U][PC / 4];
            float sc[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int e = min(e0 + 256 * u, items - 1), r = (int)(((float)e + 0.5f) * inv_p);  // e / P (e < 2^13: far from a tie)
                i[u] = first + r;
                g[u] = (e - r * P) * PC;
                id[u] = table[i[u] >> p.page_log2];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool there = (unsigned)id[u] < (unsigned)p.pages;  // an entry outside the cache reads as zeros
                const long long blk = there ? (long long)id[u] * p.H + h : 0;
                const uint32_t* from = (const uint32_t*)(p.kc + ((blk << p.page_log2) + (i[u] & (page - 1))) * D + g[u]);
                sc[u] = there ? p.ks[blk] : 0.0f;
#pragma unroll
                for (int x = 0; x < PC / 4; ++x) c[u][x] = there ? from[x] : 0u;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (e0 + 256 * u >= items) continue;
                float f[PC];
#pragma unroll
                for (int x = 0; x < PC / 4; ++x) Code<FMT>::dec4(c[u][x], f + 4 * x);
#pragma unroll
                for (int x = 0; x < PC; ++x) f[x] *= sc[u];
                T* o = heads_at<T>(p.k, b, i[u], h) + g[u];
                if constexpr (PC == 8) Chan8<T>::store(o, f);
                else *(float4*)o = make_float4(f[0], f[1], f[2], f[3]);
            }
        }
        return;
    }
    const int D4 = D / 4;
    const float inv_d4 = 1.0f / (float)D4;
    for (int e = t; e < ((z + 15) / 16) * D4; e += 256) {
        const int c = (int)(((float)e + 0.5f) * inv_d4), i0 = first + c * 16, d = (e - c * D4) * 4;
        const int id = table[i0 >> p.page_log2];
        const bool there = (unsigned)id < (unsigned)p.pages;
        const long long blk = there ? (long long)id * p.H + h : 0;
        const unsigned char* from = p.vc + ((blk * D + d) << p.page_log2) + (i0 & (page - 1));
        const float sc = there ? p.vs[blk] : 0.0f;
        float f[4][16];
#pragma unroll
        for (int v = 0; v < 4; ++v) dec16<FMT>(there ? *(const uint4*)(from + (v << p.page_log2)) : make_uint4(0, 0, 0, 0), sc, f[v]);
        T* o = heads_at<T>(p.v, b, i0, h) + d;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i0 + i < n) {
                if constexpr (sizeof(T) == 4) *(float4*)(o + (long long)i * p.v.st) = make_float4(f[0][i], f[1][i], f[2][i], f[3][i]);
                else *(uint2*)(o + (long long)i * p.v.st) = make_uint2(pack_bf16x2(f[0][i], f[1][i]), pack_bf16x2(f[2][i], f[3][i]));
            }
    }
}

int log2_of(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7; }

int check(const char* who, const ccnet_heads& k, const ccnet_heads& v, int dtype, int B, int T, int H, int D, int fmt, const void* kc, const void* vc,
          const float* ks, const float* vs, int pages, int page, const int32_t* table, int width) {
    CC_REQUIRE(cc_dtype_ok(dtype) && cc_code_ok(fmt), "%s: bad dtype", who);
    CC_REQUIRE(B >= 0 && B <= 65535 && T >= 0 && T <= (1 << 29) && H > 0 && H <= 65535, "%s: bad sizes", who);
    CC_REQUIRE(D > 0 && D <= 256 && (D % 16) == 0, "%s: head size must be a multiple of 16, at most 256 (got %d)", who, D);
    CC_REQUIRE(page == 16 || page == 32 || page == 64 || page == 128, "%s: a page holds 16, 32, 64 or 128 tokens (got %d)", who, page);
    CC_REQUIRE(pages >= 0 && width >= 0 && (long long)width * page <= (1 << 30), "%s: bad page table", who);
    if (B == 0 || T == 0 || width == 0) return CCNET_OK;
    CC_REQUIRE(table && (pages == 0 || (kc && vc && ks && vs)), "%s: null pointer", who);
    CC_REQUIRE(((uintptr_t)kc % 16) == 0 && ((uintptr_t)vc % 16) == 0, "%s: codes must be 16-byte aligned", who);
    CC_REQUIRE(cc_heads_ok(k, dtype, B, T, H) && cc_heads_ok(v, dtype, B, T, H), "%s: k / v must be 16-byte aligned", who);
    return CCNET_OK;
}

template <typename F>
int by_type(int dtype, int fmt, F f) {
    if (dtype == CCNET_BF16) return fmt == CCNET_INT8 ? f((__bf16*)nullptr, std::integral_constant<int, CCNET_INT8>()) : f((__bf16*)nullptr, std::integral_constant<int, CCNET_FP8>());
    return fmt == CCNET_INT8 ? f((float*)nullptr, std::integral_constant<int, CCNET_INT8>()) : f((float*)nullptr, std::integral_constant<int, CCNET_FP8>());
}

}  // namespace

extern "C" int ccnet_kv_cache_write(ccnet_heads k, ccnet_heads v, int dtype, int B, int T, int H, int D, int fmt, void* kc_dev, void* vc_dev,
                                    float* ks_dev, float* vs_dev, int pages, int page, const int32_t* table_dev, int width,
                                    const int32_t* start_dev, const int32_t* lens_dev, ccnet_stream stream) {
    int rc = check("kv_cache_write", k, v, dtype, B, T, H, D, fmt, kc_dev, vc_dev, ks_dev, vs_dev, pages, page, table_dev, width);
    if (rc != CCNET_OK) return rc;
    if (B == 0 || T == 0 || width == 0 || pages == 0) return CCNET_OK;
    CC_REQUIRE(start_dev, "kv_cache_write: null start");
    int slots = (T + page - 2) / page + 1;
    if (slots > width) slots = width;
    CC_REQUIRE((long long)slots * H <= (1 << 23), "kv_cache_write: too many pages");
    const CacheP p{k, v, (unsigned char*)kc_dev, (unsigned char*)vc_dev, ks_dev, vs_dev, table_dev, start_dev, lens_dev, B, T, H, D, pages, page, log2_of(page), width, slots, 0};
    // groups of 32 values in the largest block of this call (T tokens touch at most (T + 14)/16 + 1 groups of 16); one wave where two groups per
    // thread do for it (single tokens)
    const int groups = (T + 14) / 16 + 1 < page / 16 ? (T + 14) / 16 + 1 : page / 16;
    const int most = (T == 1 ? 1 : groups) * (D / 2), threads = most <= 64 ? 64 : 256, per = (most + threads - 1) / threads;
    return ccnet_submit(
        [=](hipStream_t st, const float*) -> int {
            return by_type(dtype, fmt, [&](auto* ty, auto f) -> int {
                using Ty = std::remove_pointer_t<decltype(ty)>;
                const dim3 grid(slots * H, B, 2);
                if (per <= 1) hipLaunchKernelGGL((cache_write_kernel<Ty, decltype(f)::value, 1>), grid, dim3(threads), 0, st, p);
                else if (per <= 2) hipLaunchKernelGGL((cache_write_kernel<Ty, decltype(f)::value, 2>), grid, dim3(threads), 0, st, p);
                else hipLaunchKernelGGL((cache_write_kernel<Ty, decltype(f)::value, 4>), grid, dim3(threads), 0, st, p);
                CC_LAUNCH_CHECK();
                return CCNET_OK;
            });
        },
        stream, CCNET_OP_KV_CACHE, 4.0 * B * T * H * D, 2.0 * B * T * H * D * (cc_esize(dtype) + 1.0));
}

extern "C" int ccnet_kv_cache_read(const void* kc_dev, const void* vc_dev, const float* ks_dev, const float* vs_dev, int fmt, int pages, int page,
                                   const int32_t* table_dev, int width, const int32_t* lens_dev, int dtype, int B, int T, int H, int D,
                                   ccnet_heads k_out, ccnet_heads v_out, ccnet_stream stream) {
    int rc = check("kv_cache_read", k_out, v_out, dtype, B, T, H, D, fmt, kc_dev, vc_dev, ks_dev, vs_dev, pages, page, table_dev, width);
    if (rc != CCNET_OK) return rc;
    if (B == 0 || T == 0 || width == 0) return CCNET_OK;
    CC_REQUIRE(lens_dev, "kv_cache_read: null lens");
    const int tile = T <= 64 ? 64 : 128, slots = (T + tile - 1) / tile;
    CC_REQUIRE((long long)slots * H <= (1 << 23), "kv_cache_read: too many pages");
    const CacheP p{k_out, v_out, (unsigned char*)kc_dev, (unsigned char*)vc_dev, (float*)ks_dev, (float*)vs_dev, table_dev, nullptr, lens_dev,
                   B, T, H, D, pages, page, log2_of(page), width, slots, tile};
    return ccnet_submit(
        [=](hipStream_t st, const float*) -> int {
            return by_type(dtype, fmt, [&](auto* ty, auto f) -> int {
                using Ty = std::remove_pointer_t<decltype(ty)>;
                hipLaunchKernelGGL((cache_read_kernel<Ty, decltype(f)::value>), dim3(slots * H, B, 2), dim3(256), 0, st, p);
                CC_LAUNCH_CHECK();
                return CCNET_OK;
            });
        },
        stream, CCNET_OP_KV_CACHE, 2.0 * B * T * H * D, 2.0 * B * T * H * D * (cc_esize(dtype) + 1.0));
}

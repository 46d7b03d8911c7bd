// The 8-bit key/value cache: quantised as it is written, and read back.
//   A block = the tokens of one page x one head, with one scale for its keys and one for its values.
//   write:  s' = max(s of the tokens already there, max|new| / Q);  code = round(x / s');  codes already there, where s' > s:
//           round(code * s / s').   read:  code * s.
// Keys lie [page][head][token][dim], values [page][head][dim][token]: that is how cache_attention's matrix instructions take them
// (dims are the contraction of q.k, tokens that of p.v), so the transposition is paid once, here.
// Both directions move bytes and do little else: memory bound.
#include "token_ops.h"

namespace {

struct CacheP {
    ccnet_heads k, v;          // write: sources; read: destinations
    unsigned char *kc, *vc;
    float *ks, *vs;
    const int32_t *table, *start, *lens;
    int B, T, H, D, pages, page, width, slots;
};

// the scale below which a block counts as zero: 1 / scale has to stay finite
constexpr float SCALE_MIN = 1.17549435e-38f;

__device__ __forceinline__ float amax_nan(float a, float b) { return (b > a || b != b) ? b : a; }  // keeps a NaN

__device__ __forceinline__ float block_amax(float v, float* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = amax_nan(v, __shfl_xor(v, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return amax_nan(amax_nan(red[0], red[1]), amax_nan(red[2], red[3]));
}

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

// One workgroup per (page slot of a sequence, head, keys / values).  Two passes over the new tokens of the block: the largest
// magnitude, then the codes (the second pass finds them in L2).
template <typename T, int FMT>
__global__ __launch_bounds__(256) void cache_write_kernel(const CacheP p) {
    __shared__ float red[4];
    const int t = threadIdx.x, b = blockIdx.y, isv = blockIdx.z;
    const int slot = blockIdx.x % p.slots, h = blockIdx.x / p.slots;
    const int page = p.page, D = p.D;
    const int cap = p.width * page;
    const int s0 = min(max(p.start[b], 0), cap);
    const int n = p.lens ? min(max(p.lens[b], 0), p.T) : p.T;
    const int end = min(s0 + n, cap);
    const int first = (s0 / page + slot) * page;  // the page's first token
    if (n == 0 || first >= end) return;
    const int id = p.table[(long long)b * p.width + first / page];
    if ((unsigned)id >= (unsigned)p.pages) return;
    const int a = max(s0 - first, 0), z = min(end - first, page);  // new tokens of the page: [a, z); [0, a) are there already
    const ccnet_heads& src = isv ? p.v : p.k;
    const long long blk = (long long)id * p.H + h;
    unsigned char* codes = (isv ? p.vc : p.kc) + blk * page * D;
    float* scale_at = (isv ? p.vs : p.ks) + blk;
    const int tsrc = first - s0;  // token i of the page is source row tsrc + i
    const int G = D / 16;
    float m = 0.0f;
    for (int e = t; e < (z - a) * G; e += 256) {
        const int i = e / G, g = e - i * G;
        float f[16];
        const T* s = heads_at<T>(src, b, tsrc + a + i, h) + g * 16;
        Chan8<T>::load(s, f);
        Chan8<T>::load(s + 8, f + 8);
#pragma unroll
        for (int q = 0; q < 16; ++q) m = amax_nan(m, fabsf(f[q]));
    }
    m = block_amax(m, red);
    const float old = a > 0 ? *scale_at : 0.0f;
    float sc = amax_nan(old, m * (1.0f / Code<FMT>::qmax));
    if (sc < SCALE_MIN) sc = 0.0f;
    const bool finite = sc - sc == 0.0f;
    const float inv = sc > 0.0f ? 1.0f / sc : 0.0f;
    const bool redo = a > 0 && !(sc == old);
    __syncthreads();  // every thread has the old scale
    if (t == 0) *scale_at = sc;
    if (!isv) {
        if (redo)
            for (int e = t; e < a * G; e += 256) {
                uint4* c = (uint4*)(codes + (size_t)e * 16);
                float f[16];
                dec16<FMT>(*c, old, f);
                *c = enc16<FMT>(f, inv, finite);
            }
        for (int e = t; e < (z - a) * G; e += 256) {
            const int i = e / G, g = e - i * G;
            float f[16];
            const T* s = heads_at<T>(src, b, tsrc + a + i, h) + g * 16;
            Chan8<T>::load(s, f);
            Chan8<T>::load(s + 8, f + 8);
            *(uint4*)(codes + ((size_t)(a + i) * D + g * 16)) = enc16<FMT>(f, inv, finite);
        }
        return;
    }
    // values: a thread takes 16 tokens of one dim, neighbouring threads neighbouring dims
    const int c0 = redo ? 0 : a / 16, c1 = (z + 15) / 16;
    for (int e = t; e < (c1 - c0) * D; e += 256) {
        const int c = c0 + e / D, d = e % D;
        uint4* at = (uint4*)(codes + (size_t)d * page + c * 16);
        float f[16];
        uint4 was = make_uint4(0, 0, 0, 0);
        const bool whole = c * 16 >= a && c * 16 + 16 <= z;
        if (!whole) was = *at;
        if (c * 16 < a) dec16<FMT>(was, old, f);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int k = c * 16 + i;
            if (k >= a && k < z) f[i] = load1<T>(heads_at<T>(src, b, tsrc + k, h) + d);
            else if (c * 16 >= a) f[i] = 0.0f;
        }
        uint4 now = enc16<FMT>(f, inv, finite);
        if (!whole) {
            // tokens behind the new ones keep their codes; so do those before them where the scale stays
            const int keep = redo ? 0 : a - c * 16, last = z - c * 16;
            uint32_t w[4] = {was.x, was.y, was.z, was.w}, nw[4] = {now.x, now.y, now.z, now.w};
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t mask = 0xFFu << (8 * (i & 3));
                if (i < keep || i >= last) nw[i >> 2] = (nw[i >> 2] & ~mask) | (w[i >> 2] & mask);
            }
            now = make_uint4(nw[0], nw[1], nw[2], nw[3]);
        }
        *at = now;
    }
}

// One workgroup per (page slot of a sequence, head, keys / values)
template <typename T, int FMT>
__global__ __launch_bounds__(256) void cache_read_kernel(const CacheP p) {
    const int t = threadIdx.x, b = blockIdx.y, isv = blockIdx.z;
    const int slot = blockIdx.x % p.slots, h = blockIdx.x / p.slots;
    const int page = p.page, D = p.D;
    const int n = min(min(max(p.lens[b], 0), p.T), p.width * page);
    const int first = slot * page;
    if (first >= n) return;
    const int z = min(n - first, page);
    const int id = p.table[(long long)b * p.width + slot];
    const bool there = (unsigned)id < (unsigned)p.pages;  // an entry outside the cache reads as zeros
    const ccnet_heads& dst = isv ? p.v : p.k;
    const long long blk = there ? (long long)id * p.H + h : 0;
    const unsigned char* codes = (isv ? p.vc : p.kc) + blk * page * D;
    const float sc = there ? (isv ? p.vs : p.ks)[blk] : 0.0f;
    if (!isv) {
        const int G = D / 16;
        for (int e = t; e < z * G; e += 256) {
            const int i = e / G, g = e - i * G;
            float f[16];
            dec16<FMT>(there ? *(const uint4*)(codes + (size_t)e * 16) : make_uint4(0, 0, 0, 0), sc, f);
            T* o = heads_at<T>(dst, b, first + i, h) + g * 16;
            Chan8<T>::store(o, f);
            Chan8<T>::store(o + 8, f + 8);
        }
        return;
    }
    for (int e = t; e < ((z + 15) / 16) * D; e += 256) {
        const int c = e / D, d = e % D;
        float f[16];
        dec16<FMT>(there ? *(const uint4*)(codes + (size_t)d * page + c * 16) : make_uint4(0, 0, 0, 0), sc, f);
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (c * 16 + i < z) store1<T>(heads_at<T>(dst, b, first + c * 16 + i, h) + d, f[i]);
    }
}

int check(const char* who, const ccnet_heads& k, const ccnet_heads& v, int dtype, int B, int T, int H, int D, int fmt, const void* kc, const void* vc,
          const float* ks, const float* vs, int pages, int page, const int32_t* table, int width) {
    CC_REQUIRE(cc_dtype_ok(dtype) && cc_code_ok(fmt), "%s: bad dtype", who);
    CC_REQUIRE(B >= 0 && B <= 65535 && T >= 0 && T <= (1 << 30) && H > 0 && H <= 65535, "%s: bad sizes", who);
    CC_REQUIRE(D > 0 && D <= 256 && (D % 16) == 0, "%s: head size must be a multiple of 16, at most 256 (got %d)", who, D);
    CC_REQUIRE(page == 16 || page == 32 || page == 64 || page == 128, "%s: a page holds 16, 32, 64 or 128 tokens (got %d)", who, page);
    CC_REQUIRE(pages >= 0 && width >= 0 && (long long)width * page <= (1 << 30), "%s: bad page table", who);
    if (B == 0 || T == 0 || width == 0 || pages == 0) return CCNET_OK;
    CC_REQUIRE(kc && vc && ks && vs && table, "%s: null pointer", who);
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
    const CacheP p{k, v, (unsigned char*)kc_dev, (unsigned char*)vc_dev, ks_dev, vs_dev, table_dev, start_dev, lens_dev, B, T, H, D, pages, page, width, slots};
    return ccnet_submit(
        [=](hipStream_t st, const float*) -> int {
            return by_type(dtype, fmt, [&](auto* ty, auto f) -> int {
                using Ty = std::remove_pointer_t<decltype(ty)>;
                hipLaunchKernelGGL((cache_write_kernel<Ty, decltype(f)::value>), dim3(slots * H, B, 2), dim3(256), 0, st, p);
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
    if (B == 0 || T == 0 || width == 0 || pages == 0) return CCNET_OK;
    CC_REQUIRE(lens_dev, "kv_cache_read: null lens");
    int slots = (T + page - 1) / page;
    if (slots > width) slots = width;
    CC_REQUIRE((long long)slots * H <= (1 << 23), "kv_cache_read: too many pages");
    const CacheP p{k_out, v_out, (unsigned char*)kc_dev, (unsigned char*)vc_dev, (float*)ks_dev, (float*)vs_dev, table_dev, nullptr, lens_dev,
                   B, T, H, D, pages, page, width, slots};
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

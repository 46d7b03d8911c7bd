// Attention over the 8-bit cache: softmax(scale * q . (ks kc)) (vs vc) over the pages of a sequence.
// One wave per query row: 64 keys at a time, one per lane, with a running maximum and sum.
#include "token_ops.h"

namespace {

struct CacheAttnP {
    ccnet_heads q, o;
    const unsigned char *kc, *vc;
    const float *ks, *vs;
    const int32_t *table, *lens;
    int B, Sq, Hq, H, G, D, pages, page, width, causal;
    long long rows;
    float scale;
};

template <typename T, int FMT>
__global__ __launch_bounds__(256) void cache_simple_kernel(const CacheAttnP p) {
    __shared__ float qs[4][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long row = (long long)blockIdx.x * 4 + wave;
    if (row >= p.rows) return;
    const int h = (int)(row % p.Hq), hk = h / p.G;
    const long long bs = row / p.Hq, b = bs / p.Sq;
    const int s = (int)(bs - b * p.Sq);
    const T* q = heads_at<T>(p.q, b, s, h);
    for (int d = lane; d < p.D; d += 64) qs[wave][d] = load1<T>(q + d);
    int n = min(max(p.lens[b], 0), p.width * p.page);
    if (p.causal) n -= p.Sq - 1 - s;
    float m = -INFINITY, l = 0.0f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < n; k0 += 64) {
        const int j = k0 + lane;
        int id = -1;
        if (j < n) id = p.table[b * p.width + j / p.page];
        const bool see = (unsigned)id < (unsigned)p.pages;
        const long long blk = see ? (long long)id * p.H + hk : 0;
        float x = -INFINITY, vsc = 0.0f;
        if (see) {
            const unsigned char* k = p.kc + (blk * p.page + j % p.page) * p.D;
            float a = 0.0f, f[4];
            for (int d = 0; d < p.D; d += 4) {
                Code<FMT>::dec4(*(const uint32_t*)(k + d), f);
#pragma unroll
                for (int e = 0; e < 4; ++e) a = fmaf(qs[wave][d + e], f[e], a);
            }
            x = a * p.ks[blk] * p.scale;
            vsc = p.vs[blk];
        }
        const unsigned long long seen = __ballot(see);
        if (seen == 0) continue;
        const float mn = fmaxf(m, wave_max(x));
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float e = see ? __expf(x - base) : 0.0f, alpha = __expf(m - base);
        l = l * alpha + wave_sum(e);
        m = mn;
        const float ev = see ? e * vsc : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= alpha;
        for (unsigned long long w = seen; w; w &= w - 1) {
            const int jj = __builtin_ctzll(w);
            const float pj = __shfl(ev, jj, 64);
            const long long bj = (long long)__shfl(id, jj, 64) * p.H + hk;
            const unsigned char* v = p.vc + bj * p.page * p.D + (k0 + jj) % p.page;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (lane + 64 * i < p.D) {
                    float f[4];
                    Code<FMT>::dec4(v[(lane + 64 * i) * p.page], f);
                    o[i] = fmaf(pj, f[0], o[i]);
                }
        }
    }
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    T* out = heads_at<T>(p.o, b, s, h);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < p.D) store1<T>(out + lane + 64 * i, o[i] * inv);
}

}  // namespace

extern "C" size_t ccnet_cache_attention_workspace_bytes(int B, int Sq, int Hq, int H, int D, int width, int page) { return 0; }

extern "C" int ccnet_cache_attention(ccnet_heads q, int dtype, int B, int Sq, int Hq, const void* kc_dev, const void* vc_dev, const float* ks_dev,
                                     const float* vs_dev, int fmt, int pages, int H, int page, int D, const int32_t* table_dev, int width,
                                     const int32_t* lens_dev, float scale, int causal, ccnet_heads out, void* workspace_dev, ccnet_stream stream) {
    CC_REQUIRE(cc_dtype_ok(dtype) && cc_code_ok(fmt), "cache_attention: bad dtype");
    CC_REQUIRE(B >= 0 && B <= 65535 && Sq >= 0 && Sq <= (1 << 20), "cache_attention: bad sizes");
    CC_REQUIRE(H > 0 && Hq > 0 && Hq <= 65535 && (Hq % H) == 0, "cache_attention: query heads must be a multiple of cache heads (%d, %d)", Hq, H);
    CC_REQUIRE(D > 0 && D <= 256 && (D % 16) == 0, "cache_attention: head size must be a multiple of 16, at most 256 (got %d)", D);
    CC_REQUIRE(page == 16 || page == 32 || page == 64 || page == 128, "cache_attention: a page holds 16, 32, 64 or 128 tokens (got %d)", page);
    CC_REQUIRE(pages >= 0 && width >= 0 && (long long)width * page <= (1 << 30), "cache_attention: bad page table");
    if (B == 0 || Sq == 0) return CCNET_OK;
    CC_REQUIRE(lens_dev && (width == 0 || table_dev) && (pages == 0 || (kc_dev && vc_dev && ks_dev && vs_dev)), "cache_attention: null pointer");
    CC_REQUIRE(((uintptr_t)kc_dev % 16) == 0 && ((uintptr_t)vc_dev % 16) == 0, "cache_attention: codes must be 16-byte aligned");
    CC_REQUIRE(cc_heads_ok(q, dtype, B, Sq, Hq) && cc_heads_ok(out, dtype, B, Sq, Hq), "cache_attention: q / out must be 16-byte aligned");
    const CacheAttnP p{q, out, (const unsigned char*)kc_dev, (const unsigned char*)vc_dev, ks_dev, vs_dev, table_dev, lens_dev,
                       B, Sq, Hq, H, Hq / H, D, pages, page, width, causal ? 1 : 0, (long long)B * Sq * Hq, scale};
    const unsigned blocks = (unsigned)((p.rows + 3) / 4);
    return ccnet_submit(
        [=](hipStream_t st, const float*) -> int {
            auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(blocks), dim3(256), 0, st, p); };
            if (dtype == CCNET_BF16) {
                if (fmt == CCNET_INT8) go(cache_simple_kernel<__bf16, CCNET_INT8>);
                else go(cache_simple_kernel<__bf16, CCNET_FP8>);
            } else {
                if (fmt == CCNET_INT8) go(cache_simple_kernel<float, CCNET_INT8>);
                else go(cache_simple_kernel<float, CCNET_FP8>);
            }
            CC_LAUNCH_CHECK();
            return CCNET_OK;
        },
        stream, CCNET_OP_ATTENTION, 4.0 * B * Sq * Hq * (double)width * page * D, 2.0 * B * Sq * Hq * D * cc_esize(dtype) + 2.0 * B * (double)width * page * H * D);
}

// Cross attention: softmax(scale * q.k) v over keys of another length, with lengths, a key mask and shared key heads.
// One wave per query row: 64 keys at a time, one per lane, with a running maximum and sum.
#include "token_ops.h"

namespace {

struct CrossP {
    ccnet_heads q, k, v, o;
    const int32_t* lens;
    const uint8_t* mask;
    long long mask_sb;
    int B, Sq, Sk, Hq, G, D;
    long long rows;
    float scale;
};

template <typename T>
__global__ __launch_bounds__(256) void cross_simple_kernel(const CrossP p) {
    __shared__ float qs[4][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long row = (long long)blockIdx.x * 4 + wave;
    if (row >= p.rows) return;
    const int h = (int)(row % p.Hq);
    const long long bs = row / p.Hq, b = bs / p.Sq, s = bs - b * p.Sq;
    const T* q = heads_at<T>(p.q, b, s, h);
    for (int d = lane; d < p.D; d += 64) qs[wave][d] = load1<T>(q + d);
    const int n = p.lens ? min(max(p.lens[b], 0), p.Sk) : p.Sk;
    float m = -INFINITY, l = 0.0f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < n; k0 += 64) {
        const int j = k0 + lane;
        const bool see = j < n && (!p.mask || p.mask[b * p.mask_sb + j] != 0);
        float x = -INFINITY;
        if (see) {
            const T* k = heads_at<T>(p.k, b, j, h / p.G);
            float a = 0.0f, f[8];
            for (int d = 0; d < p.D; d += 8) {
                Chan8<T>::load(k + d, f);
#pragma unroll
                for (int e = 0; e < 8; ++e) a = fmaf(qs[wave][d + e], f[e], a);
            }
            x = a * p.scale;
        }
        const unsigned long long seen = __ballot(see);
        if (seen == 0) continue;
        const float mn = fmaxf(m, wave_max(x));
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float e = see ? __expf(x - base) : 0.0f, alpha = __expf(m - base);
        l = l * alpha + wave_sum(e);
        m = mn;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= alpha;
        for (unsigned long long w = seen; w; w &= w - 1) {
            const int jj = __builtin_ctzll(w);
            const float pj = __shfl(e, jj, 64);
            const T* v = heads_at<T>(p.v, b, k0 + jj, h / p.G);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (lane + 64 * i < p.D) o[i] = fmaf(pj, load1<T>(v + lane + 64 * i), o[i]);
        }
    }
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    T* out = heads_at<T>(p.o, b, s, h);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < p.D) store1<T>(out + lane + 64 * i, o[i] * inv);
}

}  // namespace

extern "C" size_t ccnet_cross_attention_workspace_bytes(int dtype, int B, int Sq, int Sk, int Hq, int Hk, int D) { return 0; }

extern "C" int ccnet_cross_attention(ccnet_heads q, ccnet_heads k, ccnet_heads v, int dtype, int B, int Sq, int Sk, int Hq, int Hk, int D,
                                     const int32_t* lens_dev, const uint8_t* key_mask_dev, int64_t mask_sb, float scale, ccnet_heads out,
                                     void* workspace_dev, ccnet_stream stream) {
    CC_REQUIRE(cc_dtype_ok(dtype), "cross_attention: bad dtype");
    CC_REQUIRE(B >= 0 && B <= 65535 && Sq >= 0 && Sk >= 0 && Sq <= (1 << 30) && Sk <= (1 << 30), "cross_attention: bad sizes");
    CC_REQUIRE(Hk > 0 && Hq > 0 && Hq <= 65535 && (Hq % Hk) == 0, "cross_attention: query heads must be a multiple of key heads (%d, %d)", Hq, Hk);
    CC_REQUIRE(D > 0 && D <= 256 && (D % 8) == 0, "cross_attention: head size must be a multiple of 8, at most 256 (got %d)", D);
    if (B == 0 || Sq == 0) return CCNET_OK;
    CC_REQUIRE(cc_heads_ok(q, dtype, B, Sq, Hq) && cc_heads_ok(out, dtype, B, Sq, Hq), "cross_attention: q / out must be 16-byte aligned");
    CC_REQUIRE(Sk == 0 || (cc_heads_ok(k, dtype, B, Sk, Hk) && cc_heads_ok(v, dtype, B, Sk, Hk)), "cross_attention: k / v must be 16-byte aligned");
    const CrossP p{q, k, v, out, lens_dev, key_mask_dev, mask_sb, B, Sq, Sk, Hq, Hq / Hk, D, (long long)B * Sq * Hq, scale};
    const unsigned blocks = (unsigned)((p.rows + 3) / 4);
    return ccnet_submit(
        [=](hipStream_t st, const float*) -> int {
            if (dtype == CCNET_BF16) hipLaunchKernelGGL(cross_simple_kernel<__bf16>, dim3(blocks), dim3(256), 0, st, p);
            else hipLaunchKernelGGL(cross_simple_kernel<float>, dim3(blocks), dim3(256), 0, st, p);
            CC_LAUNCH_CHECK();
            return CCNET_OK;
        },
        stream, CCNET_OP_ATTENTION, 4.0 * B * Hq * Sq * (double)Sk * D, ((double)Sq * 2 * Hq + (double)Sk * 2 * Hk) * B * D * cc_esize(dtype));
}

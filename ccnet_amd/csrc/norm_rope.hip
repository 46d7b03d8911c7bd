// RMS norm of every query and key head with the position rotation in the same pass.
//   n = x * rsqrt(mean_d(x^2) + eps) * w;   (x1, x2) -> (n1 cos a - n2 sin a, n2 cos a + n1 sin a),  a = pos * freq
// Memory bound: each element is read once and written once.  A workgroup takes a few tokens: first every (token, pair) gets its cosine
// and sine once through LDS, then LP lanes per row hold a row in registers -- lane s the two halves of the pairs s*V .. s*V + V - 1, so the
// rotation needs no exchange between lanes -- and walk over heads of one token with its cosines, sines and weights in registers.
// Measured: 16396 tokens x 40 heads of 128, bfloat16: 79 us, 4.3 TB/s (a large copy: 4.9).
#include "token_ops.h"

namespace {

struct NormRopeP {
    ccnet_heads q, k, qo, ko;
    const float *wq, *wk;
    const int32_t* pos;
    long long pos_sb;
    const double* freqs;
    int B, T, Hq, Hk, D, half, interleaved, LP, NT;  // half: rotated pairs; LP: lanes per row; NT: tokens per workgroup
    long long tokens;
    float eps;
};

template <typename T, int V>
__device__ __forceinline__ void load_v(const T* p, float* f) {
    if constexpr (V == 8) Chan8<T>::load(p, f);
    else if constexpr (V == 4 && sizeof(T) == 4) {
        const float4 a = *(const float4*)p;
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    } else
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = load1<T>(p + i);
}
template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const float* f) {
    if constexpr (V == 8) Chan8<T>::store(p, f);
    else if constexpr (V == 4 && sizeof(T) == 4) *(float4*)p = make_float4(f[0], f[1], f[2], f[3]);
    else
#pragma unroll
        for (int i = 0; i < V; ++i) store1<T>(p + i, f[i]);
}

// IT slots per lane: 1 everywhere but with single-element slots (V = 1) on rows of more than 128 elements
template <typename T, int V, int IT>
__global__ __launch_bounds__(256) void norm_rope_kernel(const NormRopeP p) {
    extern __shared__ __align__(16) float2 turn[];  // [NT][half] (cos, sin)
    const int t = threadIdx.x;
    const unsigned tok0 = blockIdx.x * (unsigned)p.NT;
    const int nt = (int)min((unsigned)p.NT, (unsigned)p.tokens - tok0);
    // lanes of a row, rows side by side: GT groups of LP lanes share a token and deal its heads among them, the keys' behind the queries'
    const int sub = t % p.LP, GT = 256 / p.LP / p.NT, g = t / p.LP, j = g / GT, h0 = g - j * GT, rot = 2 * p.half;
    const int h1 = (h0 + GT - p.Hq % GT) % GT;  // the group's first query and key head
    const unsigned tok = tok0 + min(j, nt - 1), b = tok / (unsigned)p.T, tt = tok - b * p.T;
    int at1[IT], at2[IT];
    bool in1[IT], in2[IT], turned[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int s = (sub + i * p.LP) * V;  // first pair of the slot
        turned[i] = s < p.half;
        if (turned[i]) {
            at1[i] = p.interleaved ? 2 * s : s;
            at2[i] = p.interleaved ? 2 * s + V : p.half + s;
        } else {
            at1[i] = rot + 2 * (s - p.half);
            at2[i] = at1[i] + V;
        }
        in1[i] = at1[i] < p.D;
        in2[i] = at2[i] < p.D;
    }
    float x1[IT][V], x2[IT][V];
    auto load_row = [&](const T* src) {
#pragma unroll
        for (int i = 0; i < IT; ++i) {
#pragma unroll
            for (int e = 0; e < V; ++e) x1[i][e] = x2[i][e] = 0.0f;
            if (in1[i]) load_v<T, V>(src + at1[i], x1[i]);
            if (in2[i]) load_v<T, V>(src + at2[i], x2[i]);
        }
    };
    // the first row is asked for before the angles are worked out (400 tokens x 4 heads: 5.4 -> 5.2 us); asking for each next row ahead cost more in waves than it
    // hid (16396 tokens x 40 heads: 103 instead of 79 us)
    if (j < nt && h0 < p.Hq) load_row(heads_at<T>(p.q, b, tt, h0));
    else if (j < nt && h1 < p.Hk) load_row(heads_at<T>(p.k, b, tt, h1));
    for (int i = t; i < nt * p.half; i += 256) {
        const unsigned jj = (unsigned)i / (unsigned)p.half, tk = tok0 + jj, bb = tk / (unsigned)p.T;
        // whole turns leave in 64 bits: a position of 2^31 still has its angle to 2^-22 of a turn
        const double a = (double)p.pos[bb * p.pos_sb + (tk - bb * p.T)] * p.freqs[i - jj * p.half] * 0.15915494309189533577;
        float s, c;
        sincospif(2.0f * (float)(a - rint(a)), &s, &c);
        turn[i] = make_float2(c, s);
    }
    __syncthreads();
    float2 cs[IT][V];
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) cs[i][e] = turned[i] ? turn[min(j, nt - 1) * p.half + (sub + i * p.LP) * V + e] : make_float2(1.0f, 0.0f);
    const float inv_d = 1.0f / (float)p.D;
    if (j >= nt) return;  // (whole lane groups: the sums below stay inside a group)
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        const float* w = part ? p.wk : p.wq;
        const int H = part ? p.Hk : p.Hq;
        if ((part ? h1 : h0) >= H) continue;
        float w1[IT][V], w2[IT][V];
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                w1[i][e] = w && in1[i] ? w[at1[i] + e] : 1.0f;
                w2[i][e] = w && in2[i] ? w[at2[i] + e] : 1.0f;
            }
        for (int h = part ? h1 : h0; h < H; h += GT) {
            if (part ? h != h1 || h0 < p.Hq : h != h0) load_row(heads_at<T>(part ? p.k : p.q, b, tt, h));
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < IT; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) ss += x1[i][e] * x1[i][e] + x2[i][e] * x2[i][e];
            for (int o = p.LP >> 1; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
            const float var = ss * inv_d + p.eps;
            float rstd = __builtin_amdgcn_rsqf(var);  // 1 ulp; not for denormals
            if (var < 1e-30f) rstd = 1.0f / sqrtf(var);
            T* dst = heads_at<T>(part ? p.ko : p.qo, b, tt, h);
#pragma unroll
            for (int i = 0; i < IT; ++i) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    x1[i][e] = x1[i][e] * rstd * w1[i][e];
                    x2[i][e] = x2[i][e] * rstd * w2[i][e];
                }
                if (turned[i]) {
                    if (V > 1 && p.interleaved) {
                        // the slot's 2V elements are pairs (0,1), (2,3), ...: the first chunk's, then the second's
#pragma unroll
                        for (int e = 0; e + 1 < V; e += 2) {
                            const float2 c1 = cs[i][e / 2], c2 = cs[i][V / 2 + e / 2];
                            const float a0 = x1[i][e], a1 = x1[i][e + 1], b0 = x2[i][e], b1 = x2[i][e + 1];
                            x1[i][e] = a0 * c1.x - a1 * c1.y;
                            x1[i][e + 1] = a1 * c1.x + a0 * c1.y;
                            x2[i][e] = b0 * c2.x - b1 * c2.y;
                            x2[i][e + 1] = b1 * c2.x + b0 * c2.y;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            const float a0 = x1[i][e], a1 = x2[i][e];
                            x1[i][e] = a0 * cs[i][e].x - a1 * cs[i][e].y;
                            x2[i][e] = a1 * cs[i][e].x + a0 * cs[i][e].y;
                        }
                    }
                }
                if (in1[i]) store_v<T, V>(dst + at1[i], x1[i]);
                if (in2[i]) store_v<T, V>(dst + at2[i], x2[i]);
            }
        }
    }
}

}  // namespace

extern "C" int ccnet_qk_norm_rope(ccnet_heads q, ccnet_heads k, int dtype, int B, int T, int Hq, int Hk, int D, const float* wq, const float* wk,
                                  float eps, const int32_t* pos_dev, int64_t pos_sb, const double* freqs_dev, int rot, int interleaved,
                                  ccnet_heads q_out, ccnet_heads k_out, ccnet_stream stream) {
    CC_REQUIRE(cc_dtype_ok(dtype), "qk_norm_rope: bad dtype");
    CC_REQUIRE(B >= 0 && T >= 0 && Hq >= 0 && Hk >= 0 && Hq + Hk > 0 && Hq <= 65535 && Hk <= 65535, "qk_norm_rope: bad sizes");
    CC_REQUIRE(D > 0 && D <= 256 && (D % 8) == 0, "qk_norm_rope: head size must be a multiple of 8, at most 256 (got %d)", D);
    CC_REQUIRE(rot >= 0 && rot <= D && (rot % 2) == 0 && (rot == 0 || freqs_dev), "qk_norm_rope: rot must be even, at most D (got %d)", rot);
    CC_REQUIRE(eps >= 0.0f, "qk_norm_rope: negative eps");
    if (B == 0 || T == 0) return CCNET_OK;
    CC_REQUIRE((long long)B * T < (1ll << 31), "qk_norm_rope: too many tokens");
    CC_REQUIRE(rot == 0 || pos_dev, "qk_norm_rope: null positions");
    CC_REQUIRE(Hq == 0 || (cc_heads_ok(q, dtype, B, T, Hq) && cc_heads_ok(q_out, dtype, B, T, Hq)), "qk_norm_rope: q / q_out must be 16-byte aligned");
    CC_REQUIRE(Hk == 0 || (cc_heads_ok(k, dtype, B, T, Hk) && cc_heads_ok(k_out, dtype, B, T, Hk)), "qk_norm_rope: k / k_out must be 16-byte aligned");
    const int half = rot / 2, esz = cc_esize(dtype);
    // 8 pairs per lane (16-byte loads of bf16) or 4 (of fp32) where the halves start on such groups, single pairs otherwise
    const int want = dtype == CCNET_BF16 ? 8 : 4;
    const int V = ((interleaved ? rot : half) % want) == 0 && ((D - rot) % want) == 0 && (half % want) == 0 ? want : 1;
    const int slots = half / V + (D - rot + 2 * V - 1) / (2 * V);
    int LP = 1;
    while (LP < slots && LP < 64) LP <<= 1;
    NormRopeP p{q, k, q_out, k_out, wq, wk, pos_dev, pos_sb, freqs_dev, B, T, Hq, Hk, D, half, interleaved ? 1 : 0, LP, 1, (long long)B * T, eps};
    // tokens per workgroup: a power of two, so that a lane group keeps a token's cosines and sines in registers for 8 to 16 rows (16396 tokens
    // x 40 heads: 2 tokens, 2.5 rows 101 us; 8 tokens, 10 rows 79 us), fewer while the launch would leave compute units without a workgroup
    int NT = 1;
    while (2 * NT <= 256 / LP && NT < 16 && (Hq + Hk) * NT * 2 <= 16 * (256 / LP) && p.tokens / (2 * NT) >= 512) NT *= 2;
    p.NT = NT;
    CC_REQUIRE((p.tokens + NT - 1) / NT < (1 << 24), "qk_norm_rope: too many tokens");
    const unsigned blocks = (unsigned)((p.tokens + NT - 1) / NT);
    const size_t lds = (size_t)NT * half * sizeof(float2);
    return ccnet_submit(
        [=](hipStream_t st, const float*) -> int {
            const bool two = slots > 64;
            if (dtype == CCNET_BF16) {
                if (V == 8) hipLaunchKernelGGL((norm_rope_kernel<__bf16, 8, 1>), dim3(blocks), dim3(256), lds, st, p);
                else if (two) hipLaunchKernelGGL((norm_rope_kernel<__bf16, 1, 2>), dim3(blocks), dim3(256), lds, st, p);
                else hipLaunchKernelGGL((norm_rope_kernel<__bf16, 1, 1>), dim3(blocks), dim3(256), lds, st, p);
            } else {
                if (V == 4) hipLaunchKernelGGL((norm_rope_kernel<float, 4, 1>), dim3(blocks), dim3(256), lds, st, p);
                else if (two) hipLaunchKernelGGL((norm_rope_kernel<float, 1, 2>), dim3(blocks), dim3(256), lds, st, p);
                else hipLaunchKernelGGL((norm_rope_kernel<float, 1, 1>), dim3(blocks), dim3(256), lds, st, p);
            }
            CC_LAUNCH_CHECK();
            return CCNET_OK;
        },
        stream, CCNET_OP_NORM_ROPE, (double)p.tokens * (Hq + Hk) * (4.0 * D + 3.0 * rot), 2.0 * p.tokens * (Hq + Hk) * D * esz);
}

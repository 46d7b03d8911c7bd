// Cross attention, what its sources share: the problem, how keys are hidden, and how the many-row kernels stage their tiles.
#pragma once
#include "attention_mma.h"

struct CrossP {
    ccnet_heads q, k, v, o;
    const int32_t* lens;
    const uint8_t* mask;
    long long mask_sb;
    float* part;
    int B, Sq, Sk, Hq, Hk, G, D;
    int rows, tiles16, nsplit, neg;  // rows = Sq * G per (b, key head), in tiles of 16
    float scale;                     // magnitude times log2(e)
};

// Which keys of [key0, key0 + 64) are seen, a bit each.  `byte`: this lane's mask byte, loaded ahead (see_byte).
__device__ __forceinline__ int see_byte(const CrossP& p, int b, int key, int n) {
    return key < n ? (p.mask ? (int)p.mask[b * p.mask_sb + key] : 1) : 0;
}

struct CrossCfg {
    bool few;
    int tiles16, groups;        // 16-row tiles; register groups (16 dims each, padded) of a partial result
    int qt, rt_n, threads;
    int kt, nsplit;             // keys per tile; key ranges
    size_t lds;
};

// bfloat16, many rows (attention_cross_many.hip)
int cross_launch_many_bf16(const CrossP& p, const CrossCfg& c, hipStream_t st);

template <typename K>
static int launch_many(K kern, const CrossP& p, const CrossCfg& c, hipStream_t st) {
    if (c.lds > 64 * 1024) CC_HIP(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)c.lds));
    hipLaunchKernelGGL(kern, dim3((unsigned)p.B * p.Hk * c.nsplit * c.rt_n), dim3(c.threads), c.lds, st, p, c.rt_n);
    CC_LAUNCH_CHECK();
    return CCNET_OK;
}

// ---- many rows: bound by the matrix cores.  A workgroup takes a tile of rows, each wave its own 16*QT or 32*QT of them, all keys pass through
// LDS in tiles that every wave reads.  Tiles go memory -> LDS without registers (buffer loads with an LDS destination): a lane whose row
// is hidden or whose dims are behind D asks for an address past the descriptor's end, which fills its 16 bytes with zeros -- so padding, lengths
// and masks cost nothing here and no stale NaN can reach a product.
constexpr unsigned PAST_END = 0x80000000u;
typedef __attribute__((address_space(3))) void lds_void_t;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* base) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)0x7FFFFFFF, 0x00020000);
}

// Which (batch, key head, key range, row tile) a block works on: row tiles fastest, so that the eight XCDs (blocks are dealt to them in turn)
// share every sequence evenly whatever its length.  Giving each XCD sequences of its own kept their keys in one L2, but left half
// the XCDs idle on ragged batches (two sequences of 8191 and 1320 keys: 1105 us, this order: 747 us).
__device__ __forceinline__ void many_place(const CrossP& p, int rt_n, int& split, int& b, int& h, int& rt) {
    unsigned r = blockIdx.x;
    rt = (int)(r % rt_n);
    r /= rt_n;
    split = (int)(r % p.nsplit);
    r /= p.nsplit;
    h = (int)(r % p.Hk);
    b = (int)(r / p.Hk);
}

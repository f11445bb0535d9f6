// Declarations shared by the key-weight translation units.
#pragma once
#include "common.cuh"

namespace omni {

constexpr int kWsStepCols = 8;                     // columns up to which the warp-level kernel serves a call
constexpr float kWsLog2e = 1.4426950408889634f;

// A column is one (query head of the kv head's group, query token); columns per kv head = Hq / Hkv * T, head-major.
struct WeightArgs {
    const void* q;
    const uint8_t* k_nib; const uint8_t* k_qjl; const float* k_norms;
    const float* codebooks; int cb_per_head;
    const int32_t* user_ids; int32_t user_id; const int32_t* seq_lens;
    int64_t B; int Hq, Hkv, T; int64_t S; float scale;
    int with_qjl, rotate_q, causal, accumulate;
    const uint32_t* g_rows;
    float2* partial;                               // per span and column (and warp): maximum (base 2) and sum
    float* scores;                                 // warp-level kernel: [B * Hkv][S][columns, rounded up to even]
    int32_t* tiles_before;                         // [B + 1] tiles of one kv head in front of every user
    void* prepared;                                // the columns, ready for registers or tensor memory
    float* sums;
};

__device__ __forceinline__ int ws_len(const WeightArgs& a, int64_t b) {
    if (!a.seq_lens) return (int)a.S;
    const int64_t n = __ldg(a.seq_lens + b);
    return (int)(n < 0 ? 0 : (n > a.S ? a.S : n));
}
__device__ __forceinline__ float ws_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// power of two that brings `top` into [8192, 16384) (2^60 at most: products of two of them stay finite); 1 for zero, infinite, NaN
__device__ __forceinline__ float ws_pow2(float top) {
    if (!(top > 0.f) || !(top < INFINITY)) return 1.f;
    int e;
    frexpf(top, &e);
    e = 14 - e;
    return exp2f((float)(e > 60 ? 60 : e));
}
__device__ __forceinline__ uint32_t ws_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// what the fp16 pair h leaves of (lo, hi), as an fp16 pair: together 22 bits of each
__device__ __forceinline__ uint32_t ws_rest2(float lo, float hi, uint32_t h) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    return ws_half2(lo - f.x, hi - f.y);
}
// +-1 as fp16 for bits 0 and 1 of `bits` (1 = +1)
__device__ __forceinline__ uint32_t ws_signs2(uint32_t bits) {
    return 0xBC00BC00u ^ (((bits & 1u) << 15) | ((bits & 2u) << 30));
}

// Centroid table of a head in shared memory: the entry of a code byte holds the fp16 values of both centroids and what they
// leave, 8 bytes in COPIES copies side by side.  An 8-byte load is served in two half-warps, so sixteen copies (128 bytes per entry,
// 32 KiB) keep the lanes in banks of their own; thirty-two (256 bytes, 64 KiB) let one byte permutation make a lane's address.
// 256 threads build it; the centroids are scaled by ws_pow2 of the largest, returned.
template <int COPIES>
__device__ __forceinline__ float ws_build_lut(unsigned char* lut, const float* cb, int tid) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(__ldg(cb + i)));
    const float mul = ws_pow2(top);
    if (tid < 256) {
        const float x0 = __ldg(cb + (tid & 15)) * mul, x1 = __ldg(cb + (tid >> 4)) * mul;
        const uint32_t v = ws_half2(x0, x1), r = ws_rest2(x0, x1, v);
#pragma unroll
        for (int k = 0; k < COPIES / 2; ++k)       // every thread starts at another copy: the stores of a warp spread over the banks
            *reinterpret_cast<uint4*>(lut + tid * (8 * COPIES) + 16 * ((k + tid) & (COPIES / 2 - 1))) = make_uint4(v, r, v, r);
    }
    return mul;
}

// The keys of all (user, head) in tiles of 128 lie in one row, which is cut into equal shares, one per CTA: lengths differ, and only the
// device knows them.  A run of tiles of one head inside a share is a span.  tiles_before[b]: tiles of one kv head of the users in front of
// b, written by one CTA of WARPS warps of the launch that prepares the columns.
constexpr int kWsTile = 128;
template <int WARPS>
__device__ __forceinline__ void ws_tiles_before(const WeightArgs& a, int tid) {
    __shared__ int part[WARPS];
    const int lane = tid & 31, warp = tid >> 5;
    int before = 0;
    for (int64_t b0 = 0; b0 <= a.B; b0 += WARPS * 32) {
        const int64_t b = b0 + tid;
        const int n = b < a.B ? (ws_len(a, b) + kWsTile - 1) / kWsTile : 0;
        int upto = n;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const int o = __shfl_up_sync(kFullMask, upto, x);
            if (lane >= x) upto += o;
        }
        if (lane == 31) part[warp] = upto;
        __syncthreads();
        int total = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) upto += part[w];
            total += part[w];
        }
        if (b <= a.B) a.tiles_before[b] = before + upto - n;
        before += total;
        __syncthreads();
    }
}
// The last user with at most x / `heads` tiles in front of it, by a warp.
__device__ __forceinline__ int ws_user_of(const WeightArgs& a, int64_t x, int64_t heads, int lane) {
    int64_t lo = 0, n = a.B;                       // it lies in [lo, lo + n)
    while (n > 1) {
        const int64_t step = (n + 31) / 32, i = lo + lane * step;
        const bool below = lane == 0 || (i < lo + n && (int64_t)a.tiles_before[i] * heads <= x);
        const int64_t next = lo + (31 - __clz((int)__ballot_sync(kFullMask, below))) * step;
        n = lo + n - next < step ? lo + n - next : step;
        lo = next;
    }
    return (int)lo;
}
// The CTAs that have a share: no more than there are tiles, so that every CTA between two spans of a head has one of it as well.
__device__ __forceinline__ int64_t ws_sharers(int64_t ctas, int64_t all) { return ctas < all ? ctas : all; }
// The CTA of `ctas` launched ones whose share of `all` tiles holds tile x.
__device__ __forceinline__ int64_t ws_cta_of(int64_t x, int64_t ctas, int64_t all) { return ((x + 1) * ws_sharers(ctas, all) + all - 1) / all - 1; }
__host__ __device__ __forceinline__ size_t ws_before_bytes(int64_t B) { return ((size_t)(B + 1) * 4 + 15) & ~(size_t)15; }

// tcgen05 kernel for more columns (weight_window.cu)
int32_t launch_weight_window(WeightArgs a, int q_dtype, int32_t* status, cudaStream_t st);
size_t weight_window_workspace(int64_t B, int Hq, int Hkv, int T, int64_t S);

}  // namespace omni

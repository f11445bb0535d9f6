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
    float2* partial;                               // [B * Hkv][chunks][columns] maximum (base 2) and sum
    float* scores;                                 // warp-level kernel: [B * Hkv][S][columns, rounded up to even]
    int64_t chunk_keys, chunks;
    int32_t* tiles_before;                         // tcgen05 kernel: [B + 1] tiles of one kv head in front of every user
    void* prepared;                                // tcgen05 kernel: the columns, ready for tensor memory
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
// leave, 8 bytes in sixteen copies side by side, one per lane of a half-warp (an 8-byte load is served in two halves), so
// that lookups never meet in a bank.  256 threads build it; the centroids are scaled by ws_pow2 of the largest, returned.
constexpr int kWsLutBytes = 256 * 16 * 8;
__device__ __forceinline__ float ws_build_lut(unsigned char* lut, const float* cb, int tid) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(__ldg(cb + i)));
    const float mul = ws_pow2(top);
    if (tid < 256) {
        const float x0 = __ldg(cb + (tid & 15)) * mul, x1 = __ldg(cb + (tid >> 4)) * mul;
        const uint32_t v = ws_half2(x0, x1), r = ws_rest2(x0, x1, v);
#pragma unroll
        for (int k = 0; k < 8; ++k)                // every thread starts at another copy: the stores of a warp spread over the banks
            *reinterpret_cast<uint4*>(lut + tid * 128 + 16 * ((k + tid) & 7)) = make_uint4(v, r, v, r);
    }
    return mul;
}

// tcgen05 kernel for more columns (weight_window.cu)
int32_t launch_weight_window(WeightArgs a, int q_dtype, int32_t* status, cudaStream_t st);
size_t weight_window_workspace(int64_t B, int Hq, int Hkv, int T, int64_t S);

}  // namespace omni

// Declarations shared by the key-weight translation units.
#pragma once
#include "common.cuh"

namespace omni {

// Columns up to which the warp-level kernel serves a call: the eight of one product.  There it takes 43 us (16 users of up to 8,192 keys, 8
// heads; one column 40) and the tcgen05 kernel, whose time does not go with the columns, 159; 64 users of up to 1,500 keys 39 and 149.
constexpr int kWsStepCols = 8;
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
    int32_t* tiles_before;                         // [B + 1] tiles of one kv head in front of every user, then the [B] lengths they belong to
    void* prepared;                                // the columns, ready for registers or tensor memory
    float* sums;
};

__device__ __forceinline__ int ws_len_given(const WeightArgs& a, int64_t b) {
    if (!a.seq_lens) return (int)a.S;
    const int64_t n = __ldg(a.seq_lens + b);
    return (int)(n < 0 ? 0 : (n > a.S ? a.S : n));
}
// The length as the call's first launch read it: every later one walks over the same tiles, whatever is written to seq_lens meanwhile
// (a share that ends elsewhere than its tiles would walk on past the last user).  Behind that launch only.
__device__ __forceinline__ int ws_len(const WeightArgs& a, int64_t b) { return a.tiles_before[a.B + 1 + b]; }
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

__device__ __forceinline__ void wm_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight columns of one head by a warp: lane (g, c) = (lane / 4, lane % 4) has dims 32c .. 32c + 31 of its column `col` (of the head's;
// -1: zeros), rotated where asked and scaled by the power of two returned, which takes the sign of `sign`: qv[ks] holds dims 32c + 4ks .. + 3 as
// fp16, qr what those leave (QLO).  p: projections 16c .. 16c + 15 of G . q (G is +-1: exact products), handed over through `hand`.
template <int DT, bool QLO>
__device__ __forceinline__ float ws_columns8(const WeightArgs& a, int64_t b, int h, int col, float sign, float (*hand)[kQjlDim + 4], int lane,
                                             uint32_t (&qv)[8][2], uint32_t (&qr)[QLO ? 8 : 1][2], float (&p)[16]) {
    const int g = lane >> 2, c = lane & 3, G = a.Hq / a.Hkv;
    float q[32];
    const int64_t qrow = col >= 0 ? (b * a.Hq + (int64_t)h * G + col / a.T) * a.T + col % a.T : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (col >= 0) load8<DT>(a.q, qrow * kHeadDim + 32 * c + 8 * i, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) q[8 * i + k] = v[k];
    }
    uint32_t gw[4][2];
    if (a.with_qjl) {
        const int32_t uid = a.user_ids ? __ldg(a.user_ids + b) : a.user_id;
        const uint32_t* gr = a.g_rows + (size_t)seed_of(uid, h) * kQjlDim * 4 + g * 4 + c;
#pragma unroll
        for (int t = 0; t < 4; ++t) { gw[t][0] = __ldg(gr + 64 * t); gw[t][1] = __ldg(gr + 64 * t + 32); }
    }
    if (a.rotate_q) {                                                // Walsh-Hadamard over 4 lanes x 32 elements, stages in order
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                if ((i & s) == 0) {
                    const float x = q[i], y = q[i | s];
                    q[i] = __fadd_rn(x, y);
                    q[i | s] = __fsub_rn(x, y);
                }
            }
        }
#pragma unroll
        for (int s = 1; s < 4; s <<= 1) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float o = __shfl_xor_sync(kFullMask, q[i], s);
                q[i] = (c & s) ? __fsub_rn(o, q[i]) : __fadd_rn(q[i], o);
            }
        }
        const float s = __uint_as_float(OMNI_WHT_SCALE_BITS);
#pragma unroll
        for (int i = 0; i < 32; ++i) q[i] = __fmul_rn(q[i], s);
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) top = fmaxf(top, fabsf(q[i]));
    top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 1));
    top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 2));
    const float q_mul = copysignf(ws_pow2(top), sign);
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const float u = q[4 * ks + 2 * x] * q_mul, v = q[4 * ks + 2 * x + 1] * q_mul;
            qv[ks][x] = ws_half2(u, v);
            if (QLO) qr[ks][x] = ws_rest2(u, v, qv[ks][x]);
        }
    }
    if (a.with_qjl) {                                                // sixteen projections at a time
        __syncwarp();
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                const uint32_t a0 = ws_signs2(gw[t][0] >> (4 * ks)), a1 = ws_signs2(gw[t][1] >> (4 * ks));
                const uint32_t a2 = ws_signs2(gw[t][0] >> (4 * ks + 2)), a3 = ws_signs2(gw[t][1] >> (4 * ks + 2));
                wm_mma(d, a0, a1, a2, a3, qv[ks][0], qv[ks][1]);
                if (QLO) wm_mma(d, a0, a1, a2, a3, qr[ks][0], qr[ks][1]);
            }
            hand[2 * c][16 * t + g] = d[0];
            hand[2 * c + 1][16 * t + g] = d[1];
            hand[2 * c][16 * t + g + 8] = d[2];
            hand[2 * c + 1][16 * t + g + 8] = d[3];
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(&hand[g][16 * c + i]);
            p[i] = v.x; p[i + 1] = v.y; p[i + 2] = v.z; p[i + 3] = v.w;
        }
    }
    return q_mul;
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
        const int len = b < a.B ? ws_len_given(a, b) : 0, n = (len + kWsTile - 1) / kWsTile;
        if (b < a.B) a.tiles_before[a.B + 1 + b] = len;
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
__host__ __device__ __forceinline__ size_t ws_before_bytes(int64_t B) { return ((size_t)(2 * B + 1) * 4 + 15) & ~(size_t)15; }

// tcgen05 kernel for more columns (weight_window.cu)
int32_t launch_weight_window(WeightArgs a, int q_dtype, int32_t* status, cudaStream_t st);
size_t weight_window_workspace(int64_t B, int Hq, int Hkv, int T, int64_t S);

}  // namespace omni

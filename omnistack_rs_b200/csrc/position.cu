// Per-head norm of queries and keys and their position rotation in one pass over the rows.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                        over the 128 elements of a row (one head of one token)
//   (y_u, y_v) -> (y_u cos a - y_v sin a, y_v cos a + y_u sin a)   for pair i < P, (u, v) = (i, i + P) or (2i, 2i + 1)
//   a = position[axis of pair i] * inv_freq[i]                in fp64, reduced to one turn there: a position of 10^6
//                                                            leaves fp32 with an angle error of 0.06, fp64 with 10^-10
//
// Everything between the load and the one rounding at the store is fp32.  Bound by memory: a row is read once and written
// once, and nothing else of its size moves.  Sixteen lanes hold a row (8 elements, 16 bytes of a 16-bit type, per lane) and
// take the heads of one token in turn, so the angles are computed once per token and lane and stay in registers, with the
// weights multiplied in:   out_e = rsqrt(..) (x_e A_e + x_partner(e) B_e),   A_e = w_e cos, B_e = -+ w_partner(e) sin.
// The rows' factor being common, partners trade the rows' raw words (4 shuffles instead of 8 for a 16-bit type).
// 8 x 2,048 tokens of 40 heads in bf16: 71 us, 4.7 TB/s of the 6.5 a plain copy reaches (118 us with the angles and weights apart and no
// rows requested ahead; six CTAs per SM leave 80 registers, and up to 120 bytes per thread spill); a decode step of 64 users 5.5 us, launch,
// positions, angles and rows one after the other.
#include "common.cuh"

namespace omni {

constexpr int kPosThreads = 128;
constexpr int kPosRows = kPosThreads / 16;         // sixteen-lane units per CTA

// Rows a unit works on at a time; as many more are on their way meanwhile.
template <int DT> struct PosBatch { static constexpr int kRows = DT == OMNI_F32 ? 2 : 4, kWords = DT == OMNI_F32 ? 8 : 4; };

// two fp32 operations in one instruction
__device__ __forceinline__ float2 pos_fma2(float2 a, float2 b, float2 c) {
    uint64_t x, y, z, r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(x) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(y) : "f"(b.x), "f"(b.y));
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(z) : "f"(c.x), "f"(c.y));
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    float2 v;
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(v.x), "=f"(v.y) : "l"(r));
    return v;
}
__device__ __forceinline__ float2 pos_mul2(float2 a, float2 b) {
    uint64_t x, y, r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(x) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(y) : "f"(b.x), "f"(b.y));
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(x), "l"(y));
    float2 v;
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(v.x), "=f"(v.y) : "l"(r));
    return v;
}
// a lane's eight elements from their raw words
template <int DT> __device__ __forceinline__ void pos_unpack8(const uint32_t* w, float2 (&v)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (DT == OMNI_F32) v[k] = make_float2(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
        else if constexpr (DT == OMNI_BF16) v[k] = make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
        else v[k] = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
    }
}
template <int DT> __device__ __forceinline__ void pos_store8(typename Elem<DT>::T* p, const float2 (&v)[4]) {
    if constexpr (DT == OMNI_F32) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (DT == OMNI_BF16) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[k].x, v[k].y);
                w[k] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __half2 h = __floats2half2_rn(v[k].x, v[k].y);
                w[k] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
__device__ __forceinline__ float pos_weight(const void* w, int dtype, int i) {
    if (!w) return 1.f;
    if (dtype == OMNI_F32) return __ldg(reinterpret_cast<const float*>(w) + i);
    if (dtype == OMNI_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(w)[i]);
    return __half2float(reinterpret_cast<const __half*>(w)[i]);
}

__device__ __forceinline__ void pos_weight8(const void* w, int dtype, int i, float (&v)[8]) {
    if (!w) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = 1.f;
    } else if (dtype == OMNI_F32) {
        load8<OMNI_F32>(w, i, v);
    } else if (dtype == OMNI_BF16) {
        load8<OMNI_BF16>(w, i, v);
    } else {
        load8<OMNI_F16>(w, i, v);
    }
}

enum { kPosHalves = 0, kPosNeighbours = 1, kPosHalvesAny = 2 };   // pairs (i, i + P) with P % 8 == 0; (2i, 2i + 1); (i, i + P), any P

struct PosCall {
    omni_norm_rope_t a;
    int heads_per_unit, groups;                    // a unit takes heads_per_unit of the token's query and key heads
    int64_t units;
};

template <int DT, int MODE>
__global__ void __launch_bounds__(kPosThreads, 6) norm_rope_kernel(const __grid_constant__ PosCall c) {
    const omni_norm_rope_t& a = c.a;
    using E = typename Elem<DT>::T;
    constexpr int R = PosBatch<DT>::kRows, NW = PosBatch<DT>::kWords;
    const int lane = threadIdx.x & 15;                                       // 8 elements of the row: 8 * lane ..
    const int64_t unit = (int64_t)blockIdx.x * kPosRows + (threadIdx.x >> 4);
    if (unit >= c.units) return;                                             // a whole half-warp: the shuffles below name one
    const int group = (int)(unit % c.groups);
    const int64_t token = unit / c.groups;
    const int64_t b = token / a.T, t = token % a.T;
    const int P = a.n_pairs;
    const unsigned half_mask = 0xffffu << (threadIdx.x & 16);

    // ---- this unit's heads [h, h_end) of the queries and keys together; the first rows are requested right away --------------
    const int H0 = a.heads[0];
    int h = group * c.heads_per_unit;
    const int h_end = h + c.heads_per_unit < H0 + a.heads[1] ? h + c.heads_per_unit : H0 + a.heads[1];
    auto batch_end = [&](int h0) {                                           // a batch holds rows of one kind
        const int e = h0 + R < h_end ? h0 + R : h_end;
        return h0 < H0 && e > H0 ? H0 : e;
    };
    uint32_t ahead[R][NW];
    auto fetch = [&](int h0) {                                               // rows past the batch repeat its last one
        const int e = batch_end(h0), s = h0 >= H0;
        const E* p = reinterpret_cast<const E*>(a.x[s]) + b * a.xs[s][0] + t * a.xs[s][2] + (int64_t)(h0 - (s ? H0 : 0)) * a.xs[s][1] + 8 * lane;
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int k = 0; k < NW; k += 4) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + k / 4);           // read once
                ahead[r][k] = v.x; ahead[r][k + 1] = v.y; ahead[r][k + 2] = v.z; ahead[r][k + 3] = v.w;
            }
            if (h0 + r + 1 < e) p += a.xs[s][1];
        }
    };
    fetch(h);

    // ---- cos and sin: the lane computes pairs 4 lane .. 4 lane + 3 and, unless it needs just those, reads its elements' from the unit's row
    __shared__ __align__(16) float2 turn_s[kPosRows][64 + 2];                // (a row's start moves by four banks from unit to unit)
    float cs[8], sn[8];                                                      // sn: the factor of the partner, with its sign
    auto partner_of = [&](int e) { return MODE == kPosNeighbours ? e ^ 1 : (e < P ? e + P : e - P); };
    {
        double pos[OMNI_MAX_AXES];
#pragma unroll
        for (int x = 0; x < OMNI_MAX_AXES; ++x) {
            const int64_t at = (x < a.n_axes ? x : 0) * a.ps[0] + b * a.ps[1] + t * a.ps[2];
            if (x == 0 || x < a.n_axes)
                pos[x] = P == 0 ? 0.0 : (a.positions64 ? (double)__ldg(reinterpret_cast<const int64_t*>(a.positions) + at)
                                                       : (double)__ldg(reinterpret_cast<const int32_t*>(a.positions) + at));
            else
                pos[x] = 0.0;
        }
        float2 mine[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = 4 * lane + k;
            mine[k] = make_float2(1.f, 0.f);
            if (i < P) {
                double p = pos[0];
#pragma unroll
                for (int x = 1; x < OMNI_MAX_AXES; ++x)
                    if (x < a.n_axes && i >= a.axis_end[x - 1]) p = pos[x];
                const double f = a.inv_freq64 ? __ldg(reinterpret_cast<const double*>(a.inv_freq) + i) : (double)__ldg(reinterpret_cast<const float*>(a.inv_freq) + i);
                const double turns = p * f * 0.15915494309189533577;         // 1 / (2 pi)
                sincospif((float)(2.0 * (turns - rint(turns))), &mine[k].y, &mine[k].x);
            }
        }
        if (MODE == kPosNeighbours) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                cs[2 * k] = cs[2 * k + 1] = mine[k].x;
                sn[2 * k] = -mine[k].y;
                sn[2 * k + 1] = mine[k].y;
            }
        } else {
            float2* row = turn_s[threadIdx.x >> 4];
            *reinterpret_cast<float4*>(row + 4 * lane) = make_float4(mine[0].x, mine[0].y, mine[1].x, mine[1].y);
            *reinterpret_cast<float4*>(row + 4 * lane + 2) = make_float4(mine[2].x, mine[2].y, mine[3].x, mine[3].y);
            __syncwarp(half_mask);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int e = 8 * lane + k;
                const float2 v = e < 2 * P ? row[e < P ? e : e - P] : make_float2(1.f, 0.f);
                cs[k] = v.x;
                sn[k] = e < P ? -v.y : v.y;
            }
        }
    }
    const int P8 = P >> 3;
    const int from = lane < P8 ? lane + P8 : lane - P8;                      // halves: the lane that holds the partners (lanes < 2 P8)
    __shared__ float row_s[MODE == kPosHalvesAny ? kPosRows * 128 : 1];

    int kind = -1;
    float2 A[4], B[4];
    E* dst = nullptr;
    while (h < h_end) {
        const int e = batch_end(h), s = h >= H0;
        if (s != kind) {                                                     // the first batch of the queries, and of the keys
            kind = s;
            float own[8], other[8];
            pos_weight8(a.weight[s], a.weight_dtype[s], 8 * lane, own);
            if (MODE == kPosHalves) {
                pos_weight8(a.weight[s], a.weight_dtype[s], 8 * (from & 15), other);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int e0 = 8 * lane + k;
                    other[k] = MODE == kPosNeighbours ? own[k ^ 1] : (e0 < 2 * P ? pos_weight(a.weight[s], a.weight_dtype[s], partner_of(e0)) : 0.f);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                A[k] = make_float2(own[2 * k] * cs[2 * k], own[2 * k + 1] * cs[2 * k + 1]);
                B[k] = make_float2(other[2 * k] * sn[2 * k], other[2 * k + 1] * sn[2 * k + 1]);
            }
            dst = reinterpret_cast<E*>(a.y[s]) + ((b * a.heads[s] + (h - (s ? H0 : 0))) * a.T + t) * kHeadDim + 8 * lane;
        }
        uint32_t raw[R][NW];
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int k = 0; k < NW; ++k) raw[r][k] = ahead[r][k];
        }
        if (e < h_end) fetch(e);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float2 v[4], u[4];
            pos_unpack8<DT>(raw[r], v);
            float inv = 1.f;
            if (a.normalize) {
                float2 sq = pos_mul2(v[0], v[0]);
#pragma unroll
                for (int k = 1; k < 4; ++k) sq = pos_fma2(v[k], v[k], sq);
                float ss = sq.x + sq.y;
#pragma unroll
                for (int m = 8; m >= 1; m >>= 1) ss += __shfl_xor_sync(half_mask, ss, m);
                inv = rsqrtf(fmaf(ss, 1.f / 128.f, a.eps));
            }
            if (MODE == kPosNeighbours) {
#pragma unroll
                for (int k = 0; k < 4; ++k) u[k] = make_float2(v[k].y, v[k].x);
            } else if (MODE == kPosHalves) {
                uint32_t w[NW];
#pragma unroll
                for (int k = 0; k < NW; ++k) w[k] = __shfl_sync(half_mask, raw[r][k], from & 15, 16);
                pos_unpack8<DT>(w, u);
            } else {
                float* row = row_s + (threadIdx.x >> 4) * 128;
                __syncwarp(half_mask);
#pragma unroll
                for (int k = 0; k < 4; ++k) *reinterpret_cast<float2*>(row + 8 * lane + 2 * k) = v[k];
                __syncwarp(half_mask);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int e0 = 8 * lane + 2 * k;
                    u[k] = make_float2(e0 < 2 * P ? row[partner_of(e0)] : 0.f, e0 + 1 < 2 * P ? row[partner_of(e0 + 1)] : 0.f);
                }
            }
            if (MODE != kPosHalvesAny && P < 64) {                           // dims behind the pairs have no partner, not one times zero
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (8 * lane + 2 * k >= 2 * P) u[k] = make_float2(0.f, 0.f);
            }
            if (h + r < e) {
                float2 o[4];
                const float2 i2 = make_float2(inv, inv);
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = pos_mul2(pos_fma2(v[k], A[k], pos_mul2(u[k], B[k])), i2);
                pos_store8<DT>(dst, o);
                dst += a.T * kHeadDim;
            }
        }
        h = e;
    }
}

template <int DT>
static int32_t launch_norm_rope(const PosCall& c, cudaStream_t st) {
    const int64_t blocks = (c.units + kPosRows - 1) / kPosRows;
    OMNI_REQUIRE(blocks <= 0x7fffffffLL, OMNI_ERR_UNSUPPORTED, "omni_qk_norm_rope: too many rows");
    if (c.a.interleaved) norm_rope_kernel<DT, kPosNeighbours><<<(unsigned)blocks, kPosThreads, 0, st>>>(c);
    else if (c.a.n_pairs % 8 == 0) norm_rope_kernel<DT, kPosHalves><<<(unsigned)blocks, kPosThreads, 0, st>>>(c);
    else norm_rope_kernel<DT, kPosHalvesAny><<<(unsigned)blocks, kPosThreads, 0, st>>>(c);
    return check_cuda(cudaGetLastError(), "norm_rope_kernel launch");
}

}  // namespace omni

using namespace omni;

extern "C" int32_t omni_qk_norm_rope(const omni_norm_rope_t* call, void* stream) {
    OMNI_REQUIRE(call != nullptr, OMNI_ERR_ARG, "omni_qk_norm_rope: NULL call");
    const omni_norm_rope_t& a = *call;
    OMNI_REQUIRE(a.B >= 0 && a.T >= 0 && a.heads[0] >= 0 && a.heads[1] >= 0, OMNI_ERR_ARG, "omni_qk_norm_rope: negative extent");
    OMNI_REQUIRE(a.n_pairs >= 0 && a.n_pairs <= kHeadDim / 2, OMNI_ERR_ARG, "omni_qk_norm_rope: %d pairs, at most %d", a.n_pairs, kHeadDim / 2);
    OMNI_REQUIRE(a.n_axes >= 1 && a.n_axes <= OMNI_MAX_AXES, OMNI_ERR_UNSUPPORTED, "omni_qk_norm_rope: %d position axes, at most %d", a.n_axes, OMNI_MAX_AXES);
    for (int x = 0; x < a.n_axes; ++x)
        OMNI_REQUIRE(a.axis_end[x] >= (x ? a.axis_end[x - 1] : 0) && a.axis_end[x] <= a.n_pairs, OMNI_ERR_ARG, "omni_qk_norm_rope: axis_end must ascend to n_pairs");
    OMNI_REQUIRE(a.axis_end[a.n_axes - 1] == a.n_pairs, OMNI_ERR_ARG, "omni_qk_norm_rope: axis_end must ascend to n_pairs");
    const int64_t H = (int64_t)a.heads[0] + a.heads[1];
    if (a.B == 0 || a.T == 0 || H == 0) return OMNI_OK;
    for (int s = 0; s < 2; ++s) {
        if (a.heads[s] == 0) continue;
        OMNI_REQUIRE(a.x[s] && a.y[s], OMNI_ERR_ARG, "omni_qk_norm_rope: NULL rows");
        const int64_t unit = a.dtype == OMNI_F32 ? 4 : 8;
        OMNI_REQUIRE((((uintptr_t)a.x[s] | (uintptr_t)a.y[s] | (uintptr_t)a.weight[s]) & 15) == 0 && a.xs[s][0] % unit == 0 &&
                     a.xs[s][1] % unit == 0 && a.xs[s][2] % unit == 0, OMNI_ERR_ARG, "omni_qk_norm_rope: rows must start on 16-byte boundaries");
        OMNI_REQUIRE(!a.weight[s] || (a.weight_dtype[s] >= 0 && a.weight_dtype[s] <= 2), OMNI_ERR_ARG, "omni_qk_norm_rope: unknown weight dtype code %d", a.weight_dtype[s]);
    }
    OMNI_REQUIRE(a.n_pairs == 0 || (a.positions && a.inv_freq), OMNI_ERR_ARG, "omni_qk_norm_rope: NULL positions or frequencies");
    PosCall c{};
    c.a = a;
    // Few tokens: a unit takes few heads, so that the call still fills the device (the angles are then computed once per unit)
    const int64_t tokens = a.B * a.T;
    int64_t groups = 1;
    while (groups < H && tokens * groups < (int64_t)148 * 2 * kPosRows) groups *= 2;
    c.heads_per_unit = (int)((H + groups - 1) / groups);
    c.groups = (int)((H + c.heads_per_unit - 1) / c.heads_per_unit);
    c.units = tokens * c.groups;
    cudaStream_t st = (cudaStream_t)stream;
    switch (a.dtype) {
        case OMNI_F32:  return launch_norm_rope<OMNI_F32>(c, st);
        case OMNI_BF16: return launch_norm_rope<OMNI_BF16>(c, st);
        case OMNI_F16:  return launch_norm_rope<OMNI_F16>(c, st);
    }
    return set_error(OMNI_ERR_ARG, "omni_qk_norm_rope: unknown dtype code %d", a.dtype);
}

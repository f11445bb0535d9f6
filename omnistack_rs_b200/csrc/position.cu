// Per-head norm of queries and keys and their position rotation in one pass over the rows.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                        over the 128 elements of a row (one head of one token)
//   (y_u, y_v) -> (y_u cos a - y_v sin a, y_v cos a + y_u sin a)   for pair i < P, (u, v) = (i, i + P) or (2i, 2i + 1)
//   a = position[axis of pair i] * inv_freq[i]                in fp64, reduced to one turn there: a position of 10^6
//                                                            leaves fp32 with an angle error of 0.06, fp64 with 10^-10
//
// Everything between the load and the one rounding at the store is fp32.  Bound by memory: a row is read once and written
// once, and nothing else of its size moves.  Sixteen lanes hold a row (8 elements, 16 bytes of a 16-bit type, per lane) and
// take the heads of one token in turn, so the angles are computed once per token and lane and stay in registers.
#include "common.cuh"

namespace omni {

constexpr int kPosThreads = 256;
constexpr int kPosRows = kPosThreads / 16;         // sixteen-lane units per CTA
constexpr int kPosUnroll = 4;                      // rows a unit has in flight

template <int DT> __device__ __forceinline__ void pos_store8(void* p, int64_t i, const float (&v)[8]) {
    if constexpr (DT == OMNI_F32) {
        float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i);
        d[0] = make_float4(v[0], v[1], v[2], v[3]);
        d[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (DT == OMNI_BF16) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
                w[k] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __half2 h = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
                w[k] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
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
__global__ void __launch_bounds__(kPosThreads) norm_rope_kernel(const __grid_constant__ PosCall c) {
    const omni_norm_rope_t& a = c.a;
    const int lane = threadIdx.x & 15;                                       // 8 elements of the row: 8 * lane ..
    const int64_t unit = (int64_t)blockIdx.x * kPosRows + (threadIdx.x >> 4);
    const bool live = unit < c.units;                                        // lanes of a dead unit take part in the shuffles
    const int64_t u = live ? unit : 0;
    const int group = (int)(u % c.groups);
    const int64_t token = u / c.groups;
    const int64_t b = token / a.T, t = token % a.T;
    const int P = a.n_pairs;
    const unsigned half_mask = 0xffffu << (threadIdx.x & 16);

    // ---- cos and sin of this lane's pairs: pair (8 lane + k) mod P for the halves, pair 4 lane + k / 2 for neighbours ----
    constexpr int NA = MODE == kPosNeighbours ? 4 : 8;
    float cs[NA], sn[NA];
#pragma unroll
    for (int k = 0; k < NA; ++k) {
        int i;
        bool on;
        if (MODE == kPosNeighbours) { i = 4 * lane + k; on = i < P; }
        else { const int e = 8 * lane + k; on = e < 2 * P; i = e < P ? e : e - P; }
        cs[k] = 1.f;
        sn[k] = 0.f;
        if (on) {
            int axis = 0;
#pragma unroll
            for (int x = 0; x < OMNI_MAX_AXES - 1; ++x) axis += (x < a.n_axes - 1 && i >= a.axis_end[x]) ? 1 : 0;
            const int64_t pi = axis * a.ps[0] + b * a.ps[1] + t * a.ps[2];
            const double pos = a.positions64 ? (double)reinterpret_cast<const int64_t*>(a.positions)[pi]
                                             : (double)reinterpret_cast<const int32_t*>(a.positions)[pi];
            const double f = a.inv_freq64 ? reinterpret_cast<const double*>(a.inv_freq)[i] : (double)reinterpret_cast<const float*>(a.inv_freq)[i];
            const double turns = pos * f * 0.15915494309189533577;           // 1 / (2 pi)
            sincospif((float)(2.0 * (turns - rint(turns))), &sn[k], &cs[k]);
            if (MODE != kPosNeighbours && 8 * lane + k < P) sn[k] = -sn[k];  // first half: u cos - v sin
        }
    }

    const int H0 = a.heads[0], H = a.heads[0] + a.heads[1];
    const int h_begin = group * c.heads_per_unit;
    const int h_end = h_begin + c.heads_per_unit < H ? h_begin + c.heads_per_unit : H;
    float wq[8], wk[8];
    pos_weight8(a.weight[0], a.weight_dtype[0], 8 * lane, wq);
    pos_weight8(a.weight[1], a.weight_dtype[1], 8 * lane, wk);
    // partner of this lane's elements in the other half
    const int P8 = P >> 3;
    const int partner = lane < P8 ? lane + P8 : (lane < 2 * P8 ? lane - P8 : lane);
    __shared__ float row_s[MODE == kPosHalvesAny ? kPosRows * 128 : 1];

    for (int h0 = h_begin; h0 < h_end; h0 += kPosUnroll) {
        float v[kPosUnroll][8];
#pragma unroll
        for (int r = 0; r < kPosUnroll; ++r) {
            const int h = h0 + r < h_end ? h0 + r : h_end - 1;
            const int s = h >= H0;
            load8<DT>(a.x[s], b * a.xs[s][0] + (int64_t)(h - (s ? H0 : 0)) * a.xs[s][1] + t * a.xs[s][2] + 8 * lane, v[r]);
        }
#pragma unroll
        for (int r = 0; r < kPosUnroll; ++r) {
            const bool is_k = h0 + r >= H0;
            if (a.normalize) {
                float ss = 0.f;
#pragma unroll
                for (int k = 0; k < 8; ++k) ss = fmaf(v[r][k], v[r][k], ss);
#pragma unroll
                for (int m = 8; m >= 1; m >>= 1) ss += __shfl_xor_sync(half_mask, ss, m);
                const float inv = rsqrtf(fmaf(ss, 1.f / 128.f, a.eps));
#pragma unroll
                for (int k = 0; k < 8; ++k) v[r][k] = v[r][k] * inv * (is_k ? wk[k] : wq[k]);
            }
            float o[8];
            if (MODE == kPosNeighbours) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float x0 = v[r][2 * k], x1 = v[r][2 * k + 1];
                    o[2 * k] = fmaf(x0, cs[k], -(x1 * sn[k]));
                    o[2 * k + 1] = fmaf(x1, cs[k], x0 * sn[k]);
                }
            } else if (MODE == kPosHalves) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float other = __shfl_sync(half_mask, v[r][k], partner, 16);
                    o[k] = fmaf(v[r][k], cs[k], other * sn[k]);
                }
            } else {
                float* row = row_s + (threadIdx.x >> 4) * 128;
                __syncwarp(half_mask);
#pragma unroll
                for (int k = 0; k < 8; ++k) row[8 * lane + k] = v[r][k];
                __syncwarp(half_mask);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int e = 8 * lane + k;
                    const float other = e < 2 * P ? row[e < P ? e + P : e - P] : 0.f;
                    o[k] = e < 2 * P ? fmaf(v[r][k], cs[k], other * sn[k]) : v[r][k];
                }
            }
            // dims behind the pairs pass through (their cos and sin are 1 and 0, but 0 * infinity is not a pass)
            if (MODE != kPosHalvesAny && 2 * P < 128) {
#pragma unroll
                for (int k = 0; k < 8; ++k) o[k] = 8 * lane + k < 2 * P ? o[k] : v[r][k];
            }
            if (live && h0 + r < h_end) {
                const int h = h0 + r, s = h >= H0;
                pos_store8<DT>(a.y[s], (((b * a.heads[s] + (h - (s ? H0 : 0))) * a.T) + t) * kHeadDim + 8 * lane, o);
            }
        }
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
    while (groups < H && tokens * groups < (int64_t)148 * 8 * kPosRows) groups *= 2;
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

// The softmax weight every cached key receives from a set of queries.
//
//   s_jc = scale q_c . k^_j,   k^_j = cb[code_j] + norm_j (sqrt(2/pi)/128) sum_i sign_ji G_i      (c: a query of the kv head's group)
//   w_j = sum_c exp(s_jc - lse_c),   lse_c = log sum_j exp(s_jc)
//
// Two passes over the keys, since a weight needs the sum over all of them: the first leaves each chunk's maximum and sum
// per column, a small merge makes lse, the second forms the scores again and adds up the weights.  G_i . q is formed once
// per column, so a key's sign term is 64 additions.  fp32 throughout; a key's columns are added in order by one thread, so
// the result does not depend on scheduling.
#include "common.cuh"

namespace omni {

constexpr int kWsKeys = 128;                       // keys per CTA, one per thread
constexpr int kWsCols = 8;                         // columns per round
constexpr float kWsLog2e = 1.4426950408889634f;

struct WeightArgs {
    const void* q;
    const uint8_t* k_nib; const uint8_t* k_qjl; const float* k_norms;
    const float* codebooks; int cb_per_head;
    const int32_t* user_ids; int32_t user_id; const int32_t* seq_lens;
    int64_t B; int Hq, Hkv, T; int64_t S; float scale;
    int with_qjl, rotate_q, causal, accumulate;
    const uint32_t* g_rows;
    float2* partial;                               // [B * Hkv][chunks][columns] maximum (base 2) and sum
    float* lse;                                    // [B * Hkv][columns], base 2
    int64_t chunks;
    float* sums;
};

__device__ __forceinline__ int ws_len(const WeightArgs& a, int64_t b) {
    if (!a.seq_lens) return (int)a.S;
    const int64_t n = __ldg(a.seq_lens + b);
    return (int)(n < 0 ? 0 : (n > a.S ? a.S : n));
}

template <int DT, int PASS>
__global__ void __launch_bounds__(kWsKeys) weight_scores_kernel(const __grid_constant__ WeightArgs a) {
    __shared__ float q_s[kHeadDim][kWsCols];
    __shared__ float c_s[kQjlDim][kWsCols];
    __shared__ float cb_s[16];
    __shared__ float red[4][kWsCols];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t bh = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, b = bh / a.Hkv;
    const int h = (int)(bh % a.Hkv), G = a.Hq / a.Hkv, cols = G * a.T;
    const int len = ws_len(a, b);
    const int64_t key = chunk * kWsKeys + tid;
    const bool live = key < len;
    if (PASS == 1 && chunk * kWsKeys >= len) return;                     // the merge reads the chunks below the length only
    const int64_t row = bh * a.S + (live ? key : 0);
    if (tid < 16) cb_s[tid] = __ldg(a.codebooks + (a.cb_per_head ? h * 16 : 0) + tid);
    uint4 nib[4];
    uint2 sign = make_uint2(0u, 0u);
    float norm = 0.f, total = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) nib[i] = live ? __ldg(reinterpret_cast<const uint4*>(a.k_nib + row * kNibBytes) + i) : make_uint4(0u, 0u, 0u, 0u);
    if (live && a.with_qjl) {
        sign = __ldg(reinterpret_cast<const uint2*>(a.k_qjl + row * kQjlBytes));
        norm = __ldg(a.k_norms + row) * kQjlCoef;
    }
    const int32_t uid = a.user_ids ? __ldg(a.user_ids + b) : a.user_id;
    const uint32_t* g = a.g_rows + (size_t)seed_of(uid, h) * kQjlDim * 4;

    for (int c0 = 0; c0 < cols; c0 += kWsCols) {
        if (PASS == 2 && chunk * kWsKeys >= len) break;
        __syncthreads();
        for (int c = warp; c < kWsCols; c += 4) {                        // a warp per column: four elements per lane
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            const int col = c0 + c;
            if (col < cols) Elem<DT>::load4(a.q, ((b * a.Hq + (int64_t)h * G + col / a.T) * a.T + col % a.T) * kHeadDim + 4 * lane, v);
            if (a.rotate_q) wht128_warp(v, lane);
#pragma unroll
            for (int k = 0; k < 4; ++k) q_s[4 * lane + k][c] = v[k] * (a.scale * kWsLog2e);
        }
        __syncthreads();
        if (a.with_qjl) {
            for (int at = tid; at < kQjlDim * kWsCols; at += kWsKeys) {
                const int i = at / kWsCols, c = at % kWsCols;
                float s = 0.f;
                for (int wd = 0; wd < 4; ++wd) {
                    const uint32_t bits = __ldg(g + i * 4 + wd);
#pragma unroll
                    for (int d = 0; d < 32; ++d) s += __uint_as_float(__float_as_uint(q_s[32 * wd + d][c]) ^ (((~bits >> d) & 1u) << 31));
                }
                c_s[i][c] = s;
            }
            __syncthreads();
        }
        float s[kWsCols], sg[kWsCols];
#pragma unroll
        for (int c = 0; c < kWsCols; ++c) { s[c] = 0.f; sg[c] = 0.f; }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t w = i % 4 == 0 ? nib[i / 4].x : i % 4 == 1 ? nib[i / 4].y : i % 4 == 2 ? nib[i / 4].z : nib[i / 4].w;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float x = cb_s[(w >> (4 * k)) & 15];
#pragma unroll
                for (int c = 0; c < kWsCols; ++c) s[c] = fmaf(x, q_s[8 * i + k][c], s[c]);
            }
        }
        if (a.with_qjl) {
#pragma unroll 8
            for (int i = 0; i < kQjlDim; ++i) {
                const uint32_t flip = (~(i < 32 ? sign.x >> i : sign.y >> (i - 32)) & 1u) << 31;
#pragma unroll
                for (int c = 0; c < kWsCols; ++c) sg[c] += __uint_as_float(__float_as_uint(c_s[i][c]) ^ flip);
            }
#pragma unroll
            for (int c = 0; c < kWsCols; ++c) s[c] = fmaf(norm, sg[c], s[c]);
        }
#pragma unroll
        for (int c = 0; c < kWsCols; ++c) {
            const int col = c0 + c;
            const int64_t last = a.causal ? (int64_t)len - a.T + col % a.T : (int64_t)len - 1;
            if (!live || key > last) s[c] = -INFINITY;
        }
        if (PASS == 2) {
#pragma unroll
            for (int c = 0; c < kWsCols; ++c)
                if (c0 + c < cols && s[c] != -INFINITY) total += exp2f(s[c] - __ldg(a.lse + bh * cols + c0 + c));
            continue;
        }
        float m[kWsCols], l[kWsCols];
#pragma unroll
        for (int c = 0; c < kWsCols; ++c) {
            m[c] = s[c];
#pragma unroll
            for (int x = 16; x >= 1; x >>= 1) m[c] = fmaxf(m[c], __shfl_xor_sync(kFullMask, m[c], x));
            if (lane == 0) red[warp][c] = m[c];
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kWsCols; ++c) m[c] = fmaxf(fmaxf(red[0][c], red[1][c]), fmaxf(red[2][c], red[3][c]));
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kWsCols; ++c) {
            l[c] = s[c] == -INFINITY ? 0.f : exp2f(s[c] - m[c]);
#pragma unroll
            for (int x = 16; x >= 1; x >>= 1) l[c] += __shfl_xor_sync(kFullMask, l[c], x);
            if (lane == 0) red[warp][c] = l[c];
        }
        __syncthreads();
        if (tid < kWsCols && c0 + tid < cols) {
            float mm = -INFINITY;
#pragma unroll
            for (int c = 0; c < kWsCols; ++c) if (c == tid) mm = m[c];
            a.partial[(bh * a.chunks + chunk) * cols + c0 + tid] = make_float2(mm, red[0][tid] + red[1][tid] + red[2][tid] + red[3][tid]);
        }
    }
    if (PASS == 2 && key < a.S) {
        float* d = a.sums + bh * a.S + key;
        if (a.accumulate) { if (live) *d += total; }
        else *d = live ? total : 0.f;
    }
}

__global__ void __launch_bounds__(128) weight_lse_kernel(const __grid_constant__ WeightArgs a) {
    const int cols = a.Hq / a.Hkv * a.T;
    const int64_t at = (int64_t)blockIdx.x * 128 + threadIdx.x;
    if (at >= a.B * a.Hkv * cols) return;
    const int64_t bh = at / cols;
    const int len = ws_len(a, bh / a.Hkv);
    const int64_t n = (len + kWsKeys - 1) / kWsKeys;
    const float2* p = a.partial + bh * a.chunks * cols + at % cols;
    float m = -INFINITY, l = 0.f;
    for (int64_t i = 0; i < n; ++i) m = fmaxf(m, p[i * cols].x);
    for (int64_t i = 0; i < n; ++i) {
        const float2 v = p[i * cols];
        if (v.x != -INFINITY) l = fmaf(v.y, exp2f(v.x - m), l);
    }
    a.lse[at] = m + log2f(l);                                            // no open key: -inf, and no score refers to it
}

template <int DT>
static int32_t launch_weight_sums(const WeightArgs& a, cudaStream_t st) {
    const unsigned grid = (unsigned)(a.B * a.Hkv * a.chunks);
    const int64_t n = a.B * a.Hq * a.T;
    weight_scores_kernel<DT, 1><<<grid, kWsKeys, 0, st>>>(a);
    OMNI_CUDA(cudaGetLastError());
    weight_lse_kernel<<<(unsigned)((n + 127) / 128), 128, 0, st>>>(a);
    OMNI_CUDA(cudaGetLastError());
    weight_scores_kernel<DT, 2><<<grid, kWsKeys, 0, st>>>(a);
    return check_cuda(cudaGetLastError(), "weight_scores_kernel launch");
}

}  // namespace omni

using namespace omni;

extern "C" size_t omni_attn_weight_sums_workspace_bytes(int64_t B, int32_t Hq, int32_t Hkv, int32_t T, int64_t S) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || T <= 0 || S <= 0) return 0;
    const size_t rows = (size_t)B * Hq * T, chunks = (size_t)((S + kWsKeys - 1) / kWsKeys);
    return rows * chunks * sizeof(float2) + rows * sizeof(float);
}

extern "C" int32_t omni_attn_weight_sums(const void* q, int32_t q_dtype, const uint8_t* k_nib, const uint8_t* k_qjl,
                                         const float* k_norms, const float* codebooks, int32_t cb_per_head,
                                         const int32_t* user_ids, int32_t user_id, const int32_t* seq_lens,
                                         int64_t B, int32_t Hq, int32_t Hkv, int32_t T, int64_t S, float scale, int32_t with_qjl,
                                         int32_t rotate_q, int32_t causal, int32_t accumulate, void* workspace,
                                         size_t workspace_bytes, float* sums, void* stream) {
    OMNI_REQUIRE(B >= 0 && S >= 0 && T >= 0 && Hq > 0 && Hkv > 0, OMNI_ERR_ARG, "omni_attn_weight_sums: bad extent");
    OMNI_REQUIRE(Hq % Hkv == 0, OMNI_ERR_ARG, "omni_attn_weight_sums: Hq=%d is not a multiple of Hkv=%d", Hq, Hkv);
    OMNI_REQUIRE(Hkv <= kSeeds, OMNI_ERR_UNSUPPORTED, "omni_attn_weight_sums: Hkv=%d exceeds %d heads", Hkv, kSeeds);
    OMNI_REQUIRE(q_dtype >= 0 && q_dtype <= 2, OMNI_ERR_ARG, "omni_attn_weight_sums: unknown dtype code %d", q_dtype);
    if (B == 0 || S == 0) return OMNI_OK;
    OMNI_REQUIRE(sums != nullptr, OMNI_ERR_ARG, "omni_attn_weight_sums: NULL buffer");
    cudaStream_t st = (cudaStream_t)stream;
    if (T == 0) {
        if (!accumulate) OMNI_CUDA(cudaMemsetAsync(sums, 0, (size_t)(B * Hkv * S) * sizeof(float), st));
        return OMNI_OK;
    }
    OMNI_REQUIRE(q && k_nib && codebooks && (!with_qjl || (k_qjl && k_norms)), OMNI_ERR_ARG, "omni_attn_weight_sums: NULL buffer");
    OMNI_REQUIRE((((uintptr_t)q | (uintptr_t)k_nib) & 15) == 0 && ((uintptr_t)k_qjl & 7) == 0, OMNI_ERR_ARG, "omni_attn_weight_sums: misaligned buffer");
    OMNI_REQUIRE(workspace && workspace_bytes >= omni_attn_weight_sums_workspace_bytes(B, Hq, Hkv, T, S) && ((uintptr_t)workspace & 15) == 0,
                 OMNI_ERR_ARG, "omni_attn_weight_sums: workspace too small or misaligned");
    const DeviceTables* tab = tables_for_current_device();
    if (!tab) return OMNI_ERR_NOT_INIT;
    WeightArgs a{};
    a.q = q; a.k_nib = k_nib; a.k_qjl = k_qjl; a.k_norms = k_norms; a.codebooks = codebooks; a.cb_per_head = cb_per_head;
    a.user_ids = user_ids; a.user_id = user_id; a.seq_lens = seq_lens; a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.T = T; a.S = S;
    a.scale = scale; a.with_qjl = with_qjl; a.rotate_q = rotate_q; a.causal = causal; a.accumulate = accumulate;
    a.g_rows = tab->rows; a.chunks = (S + kWsKeys - 1) / kWsKeys; a.sums = sums;
    OMNI_REQUIRE(S <= 0x7fffff00LL && B * Hkv * a.chunks <= 0x7fffffffLL && B * Hq * T <= 0x7fffffffLL, OMNI_ERR_UNSUPPORTED, "omni_attn_weight_sums: too many keys");
    a.partial = reinterpret_cast<float2*>(workspace);
    a.lse = reinterpret_cast<float*>(a.partial + (size_t)B * Hq * T * a.chunks);
    switch (q_dtype) {
        case OMNI_F32:  return launch_weight_sums<OMNI_F32>(a, st);
        case OMNI_BF16: return launch_weight_sums<OMNI_BF16>(a, st);
        default:        return launch_weight_sums<OMNI_F16>(a, st);
    }
}

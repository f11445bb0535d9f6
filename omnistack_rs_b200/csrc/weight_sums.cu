// The softmax weight every cached key receives from a set of queries: entry point and the kernels for single tokens.
//
//   s_jc = scale q_c . k^_j,   k^_j = cb[code_j] + norm_j (sqrt(2/pi)/128) sum_i sign_ji G_i      (c: a column)
//   w_j = sum_c exp(s_jc - lse_c),   lse_c = log sum_j exp(s_jc)
//
// A weight needs its column's sum over all keys, so there are two passes.  G_i . q is formed once per column.  fp32 results
// need more than fp16 centroids, so products are split (see ws_build_lut); a key's columns are added in a fixed order.
//
// Up to eight columns (a decode step): the keys' 76 bytes are what has to move.  They are read once, the scores (4 bytes per
// key and column) wait in the workspace for the sum over all keys, and a second launch turns them into weights.
// mma.m16n8k16 with keys as rows and columns as columns: value and remainder of a centroid share one table lookup and one
// accumulator each, signs are exact (+-1), G_i . q is split like the centroids.  A query of a 16-bit type is exact in fp16 after a
// power-of-two scaling of its row; an fp32 or rotated one is split as well (QLO).
// Lane (g, c) = (lane / 4, lane % 4) reads bytes 16c .. 16c + 15 of the rows of keys g and g + 8: k-step ks takes its bytes 2ks
// and 2ks + 1, i.e. dims 32c + 4ks .. + 3, and the query fragments are laid out in the same order.
#include "weight_sums.cuh"

namespace omni {

constexpr int kWmWarps = 8;

__device__ __forceinline__ void wm_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
struct WmKeys { uint4 n0, n1; uint32_t s0, s1; float r0, r1; };          // this lane's part of keys g and g + 8 of a block of 16

template <int DT, bool QLO>
__global__ void __launch_bounds__(kWmWarps * 32, 2) weight_step_kernel(const __grid_constant__ WeightArgs a, int pad) {
    extern __shared__ __align__(128) unsigned char wm_smem[];
    __shared__ float c_s[kWsStepCols][kQjlDim + 4];
    __shared__ float2 part[kWmWarps][kWsStepCols];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int64_t bh = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, b = bh / a.Hkv;
    const int h = (int)(bh % a.Hkv), G = a.Hq / a.Hkv, cols = G * a.T;
    const int len = ws_len(a, b);
    const int k_begin = (int)(chunk * a.chunk_keys);
    const int k_end = len - k_begin < a.chunk_keys ? len : k_begin + (int)a.chunk_keys;
    if (k_begin >= k_end) return;
    const int64_t row0 = bh * a.S;
    auto load = [&](int k0, WmKeys& x) {                                 // keys past the end repeat the last one
        const int64_t ra = row0 + (k0 + g < k_end ? k0 + g : k_end - 1), rb = row0 + (k0 + g + 8 < k_end ? k0 + g + 8 : k_end - 1);
        x.n0 = __ldg(reinterpret_cast<const uint4*>(a.k_nib + ra * kNibBytes) + c);
        x.n1 = __ldg(reinterpret_cast<const uint4*>(a.k_nib + rb * kNibBytes) + c);
        if (a.with_qjl) {
            x.s0 = __ldg(reinterpret_cast<const uint16_t*>(a.k_qjl + ra * kQjlBytes) + c);
            x.s1 = __ldg(reinterpret_cast<const uint16_t*>(a.k_qjl + rb * kQjlBytes) + c);
            x.r0 = __ldg(a.k_norms + ra);
            x.r1 = __ldg(a.k_norms + rb);
        }
    };
    WmKeys next;
    next.s0 = next.s1 = 0; next.r0 = next.r1 = 0.f;
    int k0 = k_begin + 16 * warp;
    if (k0 < k_end) load(k0, next);

    // ---- table of the head's centroids --------------------------------------------------------------------------------
    const float cb_mul = ws_build_lut(wm_smem, a.codebooks + (a.cb_per_head ? h * 16 : 0), tid);
    // ---- query fragments: lane (g, c) has dims 32c .. 32c + 31 of column g ----------------------------------------------
    uint32_t qv[8][2], qr[QLO ? 8 : 1][2];
    float q_mul;
    {
        float q[32];
        const int64_t qrow = g < cols ? (b * a.Hq + (int64_t)h * G + g / a.T) * a.T + g % a.T : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            if (g < cols) Elem<DT>::load4(a.q, qrow * kHeadDim + 32 * c + 4 * i, v);
#pragma unroll
            for (int k = 0; k < 4; ++k) q[4 * i + k] = v[k];
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
        q_mul = ws_pow2(top);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const float u = q[4 * ks + 2 * x] * q_mul, v = q[4 * ks + 2 * x + 1] * q_mul;
                qv[ks][x] = ws_half2(u, v);
                if (QLO) qr[ks][x] = ws_rest2(u, v, qv[ks][x]);
            }
        }
    }
    // ---- G . q of the head's 64 projections (G is +-1: exact), four warps of 16 projections each ------------------------------
    uint32_t pv[4][2], pr[4][2];
    float p_mul = 1.f;
    if (a.with_qjl) {
        if (warp < 4) {
            const int32_t uid = a.user_ids ? __ldg(a.user_ids + b) : a.user_id;
            const uint32_t* gr = a.g_rows + ((size_t)seed_of(uid, h) * kQjlDim + 16 * warp) * 4;
            const uint32_t w0 = __ldg(gr + g * 4 + c), w1 = __ldg(gr + (g + 8) * 4 + c);
            float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                const uint32_t a0 = ws_signs2(w0 >> (4 * ks)), a1 = ws_signs2(w1 >> (4 * ks)), a2 = ws_signs2(w0 >> (4 * ks + 2)), a3 = ws_signs2(w1 >> (4 * ks + 2));
                wm_mma(d, a0, a1, a2, a3, qv[ks][0], qv[ks][1]);
                if (QLO) wm_mma(d, a0, a1, a2, a3, qr[ks][0], qr[ks][1]);
            }
            c_s[2 * c][16 * warp + g] = d[0];
            c_s[2 * c + 1][16 * warp + g] = d[1];
            c_s[2 * c][16 * warp + g + 8] = d[2];
            c_s[2 * c + 1][16 * warp + g + 8] = d[3];
        }
        __syncthreads();
        float p[16], top = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) { p[i] = c_s[g][16 * c + i]; top = fmaxf(top, fabsf(p[i])); }
        top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 1));
        top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 2));
        p_mul = ws_pow2(top);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const float u = p[4 * s + 2 * x] * p_mul, v = p[4 * s + 2 * x + 1] * p_mul;
                pv[s][x] = ws_half2(u, v);
                pr[s][x] = ws_rest2(u, v, pv[s][x]);
            }
        }
    }
    // factors of this lane's two result columns (they are lanes 8c and 8c + 4's columns); powers of two divide exactly
    float f_cb[2], f_sg[2];
    int last[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const float qm = __shfl_sync(kFullMask, q_mul, 8 * c + 4 * x), pm = __shfl_sync(kFullMask, p_mul, 8 * c + 4 * x);
        f_cb[x] = a.scale * kWsLog2e / qm / cb_mul;
        f_sg[x] = a.scale * kWsLog2e * kQjlCoef / qm / pm;
        const int col = 2 * c + x;
        last[x] = col < cols ? (a.causal ? len - a.T + col % a.T : len - 1) : -1;
    }
    __syncthreads();                                                     // the table is complete

    // ---- keys -----------------------------------------------------------------------------------------------------------
    const unsigned char* lut = wm_smem + 8 * (lane & 15);
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    for (; k0 < k_end; k0 += 16 * kWmWarps) {
        const WmKeys x = next;
        if (k0 + 16 * kWmWarps < k_end) load(k0 + 16 * kWmWarps, next);
        float d[4] = {0.f, 0.f, 0.f, 0.f}, e[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint32_t u0 = w == 0 ? x.n0.x : w == 1 ? x.n0.y : w == 2 ? x.n0.z : x.n0.w;
            const uint32_t u1 = w == 0 ? x.n1.x : w == 1 ? x.n1.y : w == 2 ? x.n1.z : x.n1.w;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int ks = 2 * w + k;
                const uint2 t0 = *reinterpret_cast<const uint2*>(lut + ((k ? u0 >> 9 : u0 << 7) & 0x7f80u));
                const uint2 t1 = *reinterpret_cast<const uint2*>(lut + ((k ? u1 >> 9 : u1 << 7) & 0x7f80u));
                const uint2 t2 = *reinterpret_cast<const uint2*>(lut + ((k ? u0 >> 17 : u0 >> 1) & 0x7f80u));
                const uint2 t3 = *reinterpret_cast<const uint2*>(lut + ((k ? u1 >> 17 : u1 >> 1) & 0x7f80u));
                wm_mma(d, t0.x, t1.x, t2.x, t3.x, qv[ks][0], qv[ks][1]);
                wm_mma(e, t0.y, t1.y, t2.y, t3.y, qv[ks][0], qv[ks][1]);
                if (QLO) wm_mma(e, t0.x, t1.x, t2.x, t3.x, qr[ks][0], qr[ks][1]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = (d[i] + e[i]) * f_cb[i & 1];
        if (a.with_qjl) {
            float s[4] = {0.f, 0.f, 0.f, 0.f}, t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a0 = ws_signs2(x.s0 >> (4 * i)), a1 = ws_signs2(x.s1 >> (4 * i)), a2 = ws_signs2(x.s0 >> (4 * i + 2)), a3 = ws_signs2(x.s1 >> (4 * i + 2));
                wm_mma(s, a0, a1, a2, a3, pv[i][0], pv[i][1]);
                wm_mma(t, a0, a1, a2, a3, pr[i][0], pr[i][1]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) d[i] = fmaf((s[i] + t[i]) * f_sg[i & 1], i < 2 ? x.r0 : x.r1, d[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int key = k0 + g + (i < 2 ? 0 : 8);
            if (key > last[i & 1] || key >= k_end) d[i] = -INFINITY;
        }
        if (2 * c < cols) {
            float* dst = a.scores + (row0 + k0 + g) * pad + 2 * c;
            if (k0 + g < k_end) *reinterpret_cast<float2*>(dst) = make_float2(d[0], d[1]);
            if (k0 + g + 8 < k_end) *reinterpret_cast<float2*>(dst + 8 * pad) = make_float2(d[2], d[3]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            // NaN scores: fmaxf drops them, the sum keeps them
            const float m_new = fmaxf(m[i], fmaxf(d[i], d[i + 2]));
            const float ref = m_new == -INFINITY ? 0.f : m_new;
            l[i] = l[i] * ws_ex2(m[i] - ref) + (ws_ex2(d[i] - ref) + ws_ex2(d[i + 2] - ref));
            m[i] = m_new;
        }
    }
    // ---- the chunk's maximum and sum per column ---------------------------------------------------------------------------
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float top = m[i];
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, s));
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = l[i] * ws_ex2(m[i] - ref);
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) sum += __shfl_xor_sync(kFullMask, sum, s);
        if (g == 0) part[warp][2 * c + i] = make_float2(top, sum);
    }
    __syncthreads();
    if (tid < cols) {
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWmWarps; ++w) top = fmaxf(top, part[w][tid].x);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < kWmWarps; ++w) sum += part[w][tid].y * ws_ex2(part[w][tid].x - ref);
        a.partial[(bh * a.chunks + chunk) * cols + tid] = make_float2(top, sum);
    }
}

// weights of the kept scores: sums[s] (+)= sum_c 2^(score_c - lse_c)
constexpr int kWfThreads = 256;
__global__ void __launch_bounds__(kWfThreads) weight_finish_kernel(const __grid_constant__ WeightArgs a, int pad, int64_t segments) {
    __shared__ float lse[kWsStepCols];
    const int tid = threadIdx.x;
    const int64_t bh = blockIdx.x / segments, s0 = blockIdx.x % segments * (4 * kWfThreads);
    const int len = ws_len(a, bh / a.Hkv), cols = a.Hq / a.Hkv * a.T;
    if (s0 < len) {
        const int n = (int)((len + a.chunk_keys - 1) / a.chunk_keys);
        const int warp = tid >> 5, lane = tid & 31;                      // a warp per column
        if (warp < cols) {
            const float2* p = a.partial + bh * a.chunks * cols + warp;
            float m = -INFINITY, l = 0.f;
            for (int i = lane; i < n; i += 32) m = fmaxf(m, p[(int64_t)i * cols].x);
#pragma unroll
            for (int x = 16; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, x));
            const float ref = m == -INFINITY ? 0.f : m;
            for (int i = lane; i < n; i += 32) l += p[(int64_t)i * cols].y * exp2f(p[(int64_t)i * cols].x - ref);
#pragma unroll
            for (int x = 16; x >= 1; x >>= 1) l += __shfl_xor_sync(kFullMask, l, x);
            if (lane == 0) lse[warp] = m == -INFINITY && l == 0.f ? 0.f : ref + log2f(l);   // no open key: its scores are -inf
        }
        __syncthreads();
    } else if (a.accumulate) {
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t s = s0 + k * kWfThreads + tid;
        if (s >= a.S) break;
        float total = 0.f;
        if (s < len) {
            const float2* p = reinterpret_cast<const float2*>(a.scores + (bh * a.S + s) * pad);
            for (int i = 0; i < cols; i += 2) {
                const float2 v = __ldg(p + (i >> 1));
                total += ws_ex2(v.x - lse[i]);
                if (i + 1 < cols) total += ws_ex2(v.y - lse[i + 1]);
            }
        }
        float* d = a.sums + bh * a.S + s;
        if (!a.accumulate) *d = total;
        else if (s < len) *d += total;
    }
}

// keys of a chunk: about two rounds of two CTAs per SM, at least 256 (the prologue of a CTA costs about as much as 128 keys)
static int64_t wm_chunk_keys(int64_t heads, int64_t S) {
    const int64_t per = (heads * S + 148 * 4 - 1) / (148 * 4);
    const int64_t keys = per < 256 ? 256 : (per > 4096 ? 4096 : per);
    return (keys + 127) / 128 * 128;
}

template <int DT, bool QLO>
static int32_t launch_weight_step(WeightArgs a, cudaStream_t st) {
    const int64_t heads = a.B * a.Hkv, segments = (a.S + 4 * kWfThreads - 1) / (4 * kWfThreads);
    const int pad = (a.Hq / a.Hkv * a.T + 1) & ~1;
    a.chunk_keys = wm_chunk_keys(heads, a.S);
    a.chunks = (a.S + a.chunk_keys - 1) / a.chunk_keys;
    a.scores = reinterpret_cast<float*>(a.partial + heads * a.chunks * (a.Hq / a.Hkv * a.T));
    OMNI_REQUIRE(heads * a.chunks <= 0x7fffffffLL && heads * segments <= 0x7fffffffLL, OMNI_ERR_UNSUPPORTED, "omni_attn_weight_sums: too many keys");
    weight_step_kernel<DT, QLO><<<(unsigned)(heads * a.chunks), kWmWarps * 32, kWsLutBytes, st>>>(a, pad);
    OMNI_CUDA(cudaGetLastError());
    weight_finish_kernel<<<(unsigned)(heads * segments), kWfThreads, 0, st>>>(a, pad, segments);
    return check_cuda(cudaGetLastError(), "weight_finish_kernel launch");
}

}  // namespace omni

using namespace omni;

extern "C" size_t omni_attn_weight_sums_workspace_bytes(int64_t B, int32_t Hq, int32_t Hkv, int32_t T, int64_t S) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || T <= 0 || S <= 0) return 0;
    const size_t heads = (size_t)B * Hkv, cols = (size_t)(Hq / Hkv) * T;
    if (cols > kWsStepCols) return weight_window_workspace(B, Hq, Hkv, T, S);
    const size_t keys = (size_t)wm_chunk_keys((int64_t)heads, S), chunks = ((size_t)S + keys - 1) / keys;
    return heads * cols * chunks * sizeof(float2) + heads * S * ((cols + 1) & ~(size_t)1) * sizeof(float);
}

extern "C" int32_t omni_attn_weight_sums(const void* q, int32_t q_dtype, const uint8_t* k_nib, const uint8_t* k_qjl,
                                         const float* k_norms, const float* codebooks, int32_t cb_per_head,
                                         const int32_t* user_ids, int32_t user_id, const int32_t* seq_lens,
                                         int64_t B, int32_t Hq, int32_t Hkv, int32_t T, int64_t S, float scale, int32_t with_qjl,
                                         int32_t rotate_q, int32_t causal, int32_t accumulate, void* workspace,
                                         size_t workspace_bytes, float* sums, int32_t* status_word, void* stream) {
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
    a.g_rows = tab->rows; a.partial = reinterpret_cast<float2*>(workspace); a.sums = sums;
    OMNI_REQUIRE(S <= 0x7fffff00LL && B * Hkv <= 0x7fffffffLL && (int64_t)(Hq / Hkv) * T <= 0x7fffffffLL, OMNI_ERR_UNSUPPORTED, "omni_attn_weight_sums: too many keys");
    if (Hq / Hkv * (int64_t)T > kWsStepCols) return launch_weight_window(a, q_dtype, status_word, st);
    switch (q_dtype) {
        case OMNI_F32:  return launch_weight_step<OMNI_F32, true>(a, st);
        case OMNI_BF16: return rotate_q ? launch_weight_step<OMNI_BF16, true>(a, st) : launch_weight_step<OMNI_BF16, false>(a, st);
        default:        return rotate_q ? launch_weight_step<OMNI_F16, true>(a, st) : launch_weight_step<OMNI_F16, false>(a, st);
    }
}

// Attention of whole prompts over themselves: entry point and the fp32 kernel.
//
//   s_ij = scale q_i . k_j (j of the same prompt, j <= i when causal),  o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i)
//
// One pass over the keys with the running maximum m and sum of each row.  64 x 64 tiles of scores on the FP32 units (two products per
// instruction): 256 threads, 4 x 4 scores and 4 x 8 outputs each; K and V share one buffer so that two CTAs fit an SM.  4 prompts of up
// to 611 tokens and 8 heads take 152 us (189 with one product per instruction), 1,500 tokens run at 33 TFLOP/s: bound by the loads
// between the phases of a tile, which only the other CTA covers (two CTAs leave 128 registers, and 68 to 76 bytes per thread spill).
// Tiles of 32 rows (three CTAs per SM) win below 100 tokens (18 us against 23) and lose above (180 us).
#include "prompt.cuh"

namespace omni {

constexpr int kPfM = 64, kPfN = 64;                // rows (token, head) and keys of a tile
constexpr int kPfR = kPfM / 16;                    // rows per thread
constexpr int kPfThreads = 256;
constexpr int kPfStride = kHeadDim + 4;            // floats: a warp's sixteen key rows start in different banks
constexpr int kPfPStride = kPfN + 4;
constexpr int kPfSmem = ((kPfM + kPfN) * kPfStride + kPfM * kPfPStride) * 4;
constexpr float kPfLog2e = 1.4426950408889634f;

// two fp32 operations in one instruction: (a.x b.x + c.x, a.y b.y + c.y)
__device__ __forceinline__ float2 pf_fma2(float2 a, float2 b, float2 c) {
    uint64_t x, y, z, r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(x) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(y) : "f"(b.x), "f"(b.y));
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(z) : "f"(c.x), "f"(c.y));
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    float2 v;
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(v.x), "=f"(v.y) : "l"(r));
    return v;
}

// rows [r0, r0 + 64) of a strided head into shared memory as fp32, zeros from row `end` on
template <int DT>
__device__ __forceinline__ void pf_load_tile(float* dst, const void* src, int64_t base, int64_t stride, int r0, int end) {
#pragma unroll
    for (int i = 0; i < kPfN * 32 / kPfThreads; ++i) {
        const int at = i * kPfThreads + threadIdx.x, row = at >> 5, c = (at & 31) * 4;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (r0 + row < end) Elem<DT>::load4(src, base + (int64_t)(r0 + row) * stride + c, v);
        *reinterpret_cast<float4*>(dst + row * kPfStride + c) = make_float4(v[0], v[1], v[2], v[3]);
    }
}

template <int DT>
__global__ void __launch_bounds__(kPfThreads, 2) prompt_fp32_kernel(const __grid_constant__ PromptArgs a) {
    constexpr int M = kPfM, R = kPfR;
    extern __shared__ __align__(16) float pf_shared[];
    float* Qs = pf_shared;
    float* Ks = Qs + M * kPfStride;                                   // keys, then the values of the same tile
    float* Ps = Ks + kPfN * kPfStride;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int64_t slot = (int64_t)gridDim.x - 1 - blockIdx.x;            // a prompt's last tiles have the most keys: first
    const PromptTile w = prompt_tile(a, slot, tid & 31);
    const int hg = blockIdx.y % a.n_hg, hkv = blockIdx.y / a.n_hg;
    const int G = a.Hq / a.Hkv, head0 = hkv * G + hg * a.gp;
    typename Elem<DT>::T* out = reinterpret_cast<typename Elem<DT>::T*>(a.out);

    prompt_zero_rows<DT>(a, w, slot, head0, tid, kPfThreads);
    if (w.t0 >= w.len) return;

    // ---- queries, scaled for exponents of two --------------------------------------------------------------------------
    const float qs = a.scale * kPfLog2e;
    for (int at = tid; at < M * 32; at += kPfThreads) {
        const int row = at >> 5, c = (at & 31) * 4;
        const int t = w.t0 + row % a.tpt, g = row / a.tpt;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (g < a.gp && t < w.len) Elem<DT>::load4(a.q, w.b * a.qs[0] + (int64_t)(head0 + g) * a.qs[1] + (w.row0 + t) * a.qs[2] + c, v);
        *reinterpret_cast<float4*>(Qs + row * kPfStride + c) = make_float4(v[0] * qs, v[1] * qs, v[2] * qs, v[3] * qs);
    }
    int lim[R];                                                          // newest key of this thread's rows (-1: no row)
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int row = R * ty + i, t = w.t0 + row % a.tpt;
        lim[i] = row / a.tpt < a.gp && t < w.len ? (a.causal ? t : w.len - 1) : -1;
    }
    const int t_last = w.t0 + a.tpt - 1 < w.len ? w.t0 + a.tpt - 1 : w.len - 1;
    const int n_keys = a.causal ? t_last + 1 : w.len;
    const int n_free = a.causal ? w.t0 + 1 : w.len;                      // keys below this are open to every row of the tile
    const int64_t kbase = w.b * a.ks[0] + (int64_t)hkv * a.ks[1] + w.row0 * a.ks[2];
    const int64_t vbase = w.b * a.vs[0] + (int64_t)hkv * a.vs[1] + w.row0 * a.vs[2];
    float m[R], l[R], o[R][8];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        m[i] = -INFINITY; l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < 8; ++c) o[i][c] = 0.f;
    }

    for (int j0 = 0; j0 < n_keys; j0 += kPfN) {
        const bool masked = j0 + kPfN > n_free;
        __syncthreads();                                                 // the previous tile's values are no longer read
        pf_load_tile<DT>(Ks, a.k, kbase, a.ks[2], j0, n_keys);
        __syncthreads();
        float2 s2[R][4];                                                 // even and odd dims apart
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s2[i][j] = make_float2(0.f, 0.f);
#pragma unroll 4
        for (int d = 0; d < kHeadDim; d += 4) {
            float4 qv[R], kv[4];
#pragma unroll
            for (int i = 0; i < R; ++i) qv[i] = *reinterpret_cast<const float4*>(Qs + (R * ty + i) * kPfStride + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) kv[j] = *reinterpret_cast<const float4*>(Ks + (tx + 16 * j) * kPfStride + d);
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s2[i][j] = pf_fma2(make_float2(qv[i].x, qv[i].y), make_float2(kv[j].x, kv[j].y), s2[i][j]);
                    s2[i][j] = pf_fma2(make_float2(qv[i].z, qv[i].w), make_float2(kv[j].z, kv[j].w), s2[i][j]);
                }
        }
        float s[R][4];
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = s2[i][j].x + s2[i][j].y;
        __syncthreads();                                                 // the keys have been read
        pf_load_tile<DT>(Ks, a.v, vbase, a.vs[2], j0, n_keys);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (masked) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j0 + tx + 16 * j > lim[i]) s[i][j] = -INFINITY;
            }
            float mx = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
#pragma unroll
            for (int x = 8; x >= 1; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFullMask, mx, x));
            const float m_new = fmaxf(m[i], mx);
            const float ref = m_new == -INFINITY ? 0.f : m_new;          // no open key so far: every weight below is zero
            const float alpha = exp2f(m[i] - ref);
            m[i] = m_new;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = exp2f(s[i][j] - ref);
                sum += p;
                Ps[(R * ty + i) * kPfPStride + tx + 16 * j] = p;
            }
#pragma unroll
            for (int x = 8; x >= 1; x >>= 1) sum += __shfl_xor_sync(kFullMask, sum, x);
            l[i] = fmaf(l[i], alpha, sum);
#pragma unroll
            for (int c = 0; c < 8; ++c) o[i][c] *= alpha;
        }
        __syncthreads();
        if (!masked || !a.causal) {                                      // without the causal mask, masked keys lie behind the end: zeros
#pragma unroll 2
            for (int j = 0; j < kPfN; j += 4) {
                float4 pv[R];
#pragma unroll
                for (int i = 0; i < R; ++i) pv[i] = *reinterpret_cast<const float4*>(Ps + (R * ty + i) * kPfPStride + j);
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                    const float4 va = *reinterpret_cast<const float4*>(Ks + (j + jj) * kPfStride + 4 * tx);
                    const float4 vb = *reinterpret_cast<const float4*>(Ks + (j + jj) * kPfStride + 64 + 4 * tx);
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        const float p = jj == 0 ? pv[i].x : jj == 1 ? pv[i].y : jj == 2 ? pv[i].z : pv[i].w;
                        const float2 p2 = make_float2(p, p), v2[4] = {{va.x, va.y}, {va.z, va.w}, {vb.x, vb.y}, {vb.z, vb.w}};
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float2 r = pf_fma2(p2, v2[c], make_float2(o[i][2 * c], o[i][2 * c + 1]));
                            o[i][2 * c] = r.x;
                            o[i][2 * c + 1] = r.y;
                        }
                    }
                }
            }
        } else {                                                         // zero weights must not meet a masked key's infinities
            for (int j = 0; j < kPfN && j0 + j < n_keys; ++j) {
                const float4 va = *reinterpret_cast<const float4*>(Ks + j * kPfStride + 4 * tx);
                const float4 vb = *reinterpret_cast<const float4*>(Ks + j * kPfStride + 64 + 4 * tx);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    if (j0 + j > lim[i]) continue;
                    const float p = Ps[(R * ty + i) * kPfPStride + j];
                    o[i][0] = fmaf(p, va.x, o[i][0]); o[i][1] = fmaf(p, va.y, o[i][1]);
                    o[i][2] = fmaf(p, va.z, o[i][2]); o[i][3] = fmaf(p, va.w, o[i][3]);
                    o[i][4] = fmaf(p, vb.x, o[i][4]); o[i][5] = fmaf(p, vb.y, o[i][5]);
                    o[i][6] = fmaf(p, vb.z, o[i][6]); o[i][7] = fmaf(p, vb.w, o[i][7]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int row = R * ty + i, t = w.t0 + row % a.tpt;
        if (lim[i] < 0) continue;
        const float inv = 1.f / l[i];
        const int64_t at = ((w.b * a.Hq + head0 + row / a.tpt) * a.T + w.row0 + t) * kHeadDim;
        const float lo[4] = {o[i][0] * inv, o[i][1] * inv, o[i][2] * inv, o[i][3] * inv};
        const float hi[4] = {o[i][4] * inv, o[i][5] * inv, o[i][6] * inv, o[i][7] * inv};
        Elem<DT>::store4(out, at + 4 * tx, lo);
        Elem<DT>::store4(out, at + 64 + 4 * tx, hi);
    }
}

template <int DT>
static int32_t launch_prompt_fp32(PromptArgs a, cudaStream_t st) {
    a.tpt = kPfM / a.gp;
    a.slots = a.cu ? a.T / a.tpt + a.n_seqs : a.B * ((a.T + a.tpt - 1) / a.tpt);
    OMNI_REQUIRE(a.slots <= 0x7fffffffLL && (int64_t)a.Hkv * a.n_hg <= 65535, OMNI_ERR_UNSUPPORTED, "omni_prompt_attn: too many tiles");
    OMNI_ALLOW_SMEM((prompt_fp32_kernel<DT>), kPfSmem);
    prompt_fp32_kernel<DT><<<dim3((unsigned)a.slots, (unsigned)(a.Hkv * a.n_hg)), kPfThreads, kPfSmem, st>>>(a);
    return check_cuda(cudaGetLastError(), "prompt_fp32_kernel launch");
}

}  // namespace omni

using namespace omni;

extern "C" int32_t omni_prompt_attn(const omni_prompt_t* call, void* stream) {
    OMNI_REQUIRE(call != nullptr, OMNI_ERR_ARG, "omni_prompt_attn: NULL call");
    const omni_prompt_t& p = *call;
    const int64_t B = p.B, T = p.T, n_seqs = p.n_seqs;
    const int32_t Hq = p.Hq, Hkv = p.Hkv, dtype = p.dtype;
    OMNI_REQUIRE(B >= 0 && T >= 0 && Hq > 0 && Hkv > 0 && n_seqs >= 0, OMNI_ERR_ARG, "omni_prompt_attn: bad extent");
    OMNI_REQUIRE(Hq % Hkv == 0, OMNI_ERR_ARG, "omni_prompt_attn: Hq=%d is not a multiple of Hkv=%d", Hq, Hkv);
    OMNI_REQUIRE(dtype >= 0 && dtype <= 2, OMNI_ERR_ARG, "omni_prompt_attn: unknown dtype code %d", dtype);
    OMNI_REQUIRE(T <= 0x3fffffffLL && n_seqs <= 0x3fffffffLL, OMNI_ERR_UNSUPPORTED, "omni_prompt_attn: more than 2^30 rows or prompts");
    OMNI_REQUIRE(p.cu_seqlens ? B == 1 && !p.seq_lens : n_seqs == B, OMNI_ERR_ARG, "omni_prompt_attn: packed prompts are the rows of one user; otherwise every user is one prompt");
    if (B == 0 || T == 0) return OMNI_OK;
    OMNI_REQUIRE(p.q && p.k && p.v && p.out, OMNI_ERR_ARG, "omni_prompt_attn: NULL buffer");
    const int64_t unit = dtype == OMNI_F32 ? 4 : 8;
    OMNI_REQUIRE((((uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v) & 15) == 0, OMNI_ERR_ARG, "omni_prompt_attn: rows must start on 16-byte boundaries");
    OMNI_REQUIRE(((uintptr_t)p.out & 31) == 0, OMNI_ERR_ARG, "omni_prompt_attn: out must start on a 32-byte boundary");
    PromptArgs a{};
    for (int i = 0; i < 3; ++i) {
        OMNI_REQUIRE(p.q_strides[i] % unit == 0 && p.k_strides[i] % unit == 0 && p.v_strides[i] % unit == 0, OMNI_ERR_ARG, "omni_prompt_attn: rows must start on 16-byte boundaries");
        a.qs[i] = p.q_strides[i]; a.ks[i] = p.k_strides[i]; a.vs[i] = p.v_strides[i];
    }
    cudaStream_t st = (cudaStream_t)stream;
    if (n_seqs == 0) {
        OMNI_CUDA(cudaMemsetAsync(p.out, 0, (size_t)(B * Hq * T) * kHeadDim * (dtype == OMNI_F32 ? 4 : 2), st));
        return OMNI_OK;
    }
    a.q = p.q; a.k = p.k; a.v = p.v; a.out = p.out; a.cu = p.cu_seqlens; a.seq_lens = p.seq_lens;
    a.B = B; a.T = T; a.n_seqs = n_seqs; a.Hq = Hq; a.Hkv = Hkv; a.scale = p.scale; a.causal = p.causal; a.status = p.status_word;
    // heads per tile: the largest divisor of the group up to sixteen
    const int G = Hq / Hkv;
    a.gp = 1;
    for (int g = 2; g <= 16; ++g) if (G % g == 0) a.gp = g;
    a.n_hg = G / a.gp;
    // The tensor-core kernel takes its running maximum over unscaled scores, which needs a positive scale.
    if (dtype != OMNI_F32 && p.scale > 0.f) return launch_prompt_umma(a, dtype, st);
    switch (dtype) {
        case OMNI_F32:  return launch_prompt_fp32<OMNI_F32>(a, st);
        case OMNI_BF16: return launch_prompt_fp32<OMNI_BF16>(a, st);
        default:        return launch_prompt_fp32<OMNI_F16>(a, st);
    }
}

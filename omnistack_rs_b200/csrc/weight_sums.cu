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

// ---- up to eight columns (single tokens): tensor-core products at the warp level, scores kept ----------------------------
//
// A decode step has few columns per kv head, so the keys' 76 bytes are what has to move: they are read once, the scores (4
// bytes per key and column) wait in the workspace for the sum over all keys, and a second launch turns them into weights.
//
// mma.m16n8k16 with keys as rows and query columns as columns.  fp32 results need more than fp16 centroids: the table that a
// code byte indexes holds both centroids' fp16 value AND what it leaves (2^-22 of the centroid together), the two products
// share one accumulator; the sign products are exact in A (+-1), their G_i . q split the same way.  A query of a 16-bit type is exact
// in fp16 after a power-of-two scaling of its row; an fp32 or rotated one is split as well (QLO).
// Lane (g, c) = (lane / 4, lane % 4) reads bytes 16c .. 16c + 15 of the rows of keys g and g + 8: k-step ks takes its bytes 2ks
// and 2ks + 1, i.e. dims 32c + 4ks .. + 3, and the query fragments are laid out in the same order.
constexpr int kWmWarps = 8;
constexpr int kWmLutBytes = 256 * 16 * 8;          // entry of a byte: (value pair, remainder pair), one copy per lane of a half-warp
constexpr float kWmTop = 8192.f;                   // power-of-two scalings put the largest magnitude in [8192, 16384)

__device__ __forceinline__ float wm_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// power of two that brings `top` into [8192, 16384); 1 for zero, infinite and NaN
__device__ __forceinline__ float wm_pow2(float top) {
    if (!(top > 0.f) || !(top < INFINITY)) return 1.f;
    int e;
    frexpf(top, &e);
    e = 14 - e;
    return exp2f((float)(e > 120 ? 120 : e));
}
__device__ __forceinline__ uint32_t wm_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t wm_rest2(float lo, float hi, uint32_t h) {       // what the fp16 pair h leaves of (lo, hi)
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    return wm_half2(lo - f.x, hi - f.y);
}
__device__ __forceinline__ void wm_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// +-1 as fp16 for bits 0 and 1 of `bits` (1 = +1)
__device__ __forceinline__ uint32_t wm_signs2(uint32_t bits) {
    return 0xBC00BC00u ^ (((bits & 1u) << 15) | ((bits & 2u) << 30));
}
struct WmKeys { uint4 n0, n1; uint32_t s0, s1; float r0, r1; };          // this lane's part of keys g and g + 8 of a block of 16

template <int DT, bool QLO>
__global__ void __launch_bounds__(kWmWarps * 32, 2) weight_step_kernel(const __grid_constant__ WeightArgs a, int64_t chunk_keys, float* scores, int pad) {
    extern __shared__ __align__(128) unsigned char wm_smem[];
    __shared__ float c_s[kWsCols][kQjlDim + 4];
    __shared__ float2 part[kWmWarps][kWsCols];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int64_t bh = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, b = bh / a.Hkv;
    const int h = (int)(bh % a.Hkv), G = a.Hq / a.Hkv, cols = G * a.T;
    const int len = ws_len(a, b);
    const int k_begin = (int)(chunk * chunk_keys);
    const int k_end = len - k_begin < chunk_keys ? len : k_begin + (int)chunk_keys;
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
    const float* cb = a.codebooks + (a.cb_per_head ? h * 16 : 0);
    float cb_top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) cb_top = fmaxf(cb_top, fabsf(__ldg(cb + i)));
    const float cb_mul = wm_pow2(cb_top);
    {
        const int byte = tid;                                            // one entry per thread, sixteen copies
        const float x0 = __ldg(cb + (byte & 15)) * cb_mul, x1 = __ldg(cb + (byte >> 4)) * cb_mul;
        const uint32_t v = wm_half2(x0, x1), r = wm_rest2(x0, x1, v);
#pragma unroll
        for (int k = 0; k < 8; ++k)                                      // start at another copy per thread: no bank meets all lanes
            *reinterpret_cast<uint4*>(wm_smem + byte * 128 + 16 * ((k + byte) & 7)) = make_uint4(v, r, v, r);
    }
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
        q_mul = wm_pow2(top);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const float u = q[4 * ks + 2 * x] * q_mul, v = q[4 * ks + 2 * x + 1] * q_mul;
                qv[ks][x] = wm_half2(u, v);
                if (QLO) qr[ks][x] = wm_rest2(u, v, qv[ks][x]);
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
                const uint32_t a0 = wm_signs2(w0 >> (4 * ks)), a1 = wm_signs2(w1 >> (4 * ks)), a2 = wm_signs2(w0 >> (4 * ks + 2)), a3 = wm_signs2(w1 >> (4 * ks + 2));
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
        p_mul = wm_pow2(top);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const float u = p[4 * s + 2 * x] * p_mul, v = p[4 * s + 2 * x + 1] * p_mul;
                pv[s][x] = wm_half2(u, v);
                pr[s][x] = wm_rest2(u, v, pv[s][x]);
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
                const uint32_t a0 = wm_signs2(x.s0 >> (4 * i)), a1 = wm_signs2(x.s1 >> (4 * i)), a2 = wm_signs2(x.s0 >> (4 * i + 2)), a3 = wm_signs2(x.s1 >> (4 * i + 2));
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
            float* dst = scores + (row0 + k0 + g) * pad + 2 * c;
            if (k0 + g < k_end) *reinterpret_cast<float2*>(dst) = make_float2(d[0], d[1]);
            if (k0 + g + 8 < k_end) *reinterpret_cast<float2*>(dst + 8 * pad) = make_float2(d[2], d[3]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            // NaN scores: fmaxf drops them, the sum keeps them
            const float m_new = fmaxf(m[i], fmaxf(d[i], d[i + 2]));
            const float ref = m_new == -INFINITY ? 0.f : m_new;
            l[i] = l[i] * wm_ex2(m[i] - ref) + (wm_ex2(d[i] - ref) + wm_ex2(d[i + 2] - ref));
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
        float sum = l[i] * wm_ex2(m[i] - ref);
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
        for (int w = 0; w < kWmWarps; ++w) sum += part[w][tid].y * wm_ex2(part[w][tid].x - ref);
        a.partial[(bh * a.chunks + chunk) * cols + tid] = make_float2(top, sum);
    }
}

// weights of the kept scores: sums[s] (+)= sum_c 2^(score_c - lse_c)
constexpr int kWfThreads = 256;
__global__ void __launch_bounds__(kWfThreads) weight_finish_kernel(const __grid_constant__ WeightArgs a, int64_t chunk_keys, const float* scores, int pad, int64_t segments) {
    __shared__ float lse[kWsCols];
    const int tid = threadIdx.x;
    const int64_t bh = blockIdx.x / segments, s0 = blockIdx.x % segments * (4 * kWfThreads);
    const int len = ws_len(a, bh / a.Hkv), cols = a.Hq / a.Hkv * a.T;
    if (s0 < len) {
        const int n = (int)((len + chunk_keys - 1) / chunk_keys);
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
            const float2* p = reinterpret_cast<const float2*>(scores + (bh * a.S + s) * pad);
            for (int i = 0; i < cols; i += 2) {
                const float2 v = __ldg(p + (i >> 1));
                total += wm_ex2(v.x - lse[i]);
                if (i + 1 < cols) total += wm_ex2(v.y - lse[i + 1]);
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
static int32_t launch_weight_step(WeightArgs a, float* scores, int pad, cudaStream_t st) {
    const int64_t heads = a.B * a.Hkv, keys = wm_chunk_keys(heads, a.S), segments = (a.S + 4 * kWfThreads - 1) / (4 * kWfThreads);
    a.chunks = (a.S + keys - 1) / keys;
    weight_step_kernel<DT, QLO><<<(unsigned)(heads * a.chunks), kWmWarps * 32, kWmLutBytes, st>>>(a, keys, scores, pad);
    OMNI_CUDA(cudaGetLastError());
    weight_finish_kernel<<<(unsigned)(heads * segments), kWfThreads, 0, st>>>(a, keys, scores, pad, segments);
    return check_cuda(cudaGetLastError(), "weight_finish_kernel launch");
}

}  // namespace omni

using namespace omni;

extern "C" size_t omni_attn_weight_sums_workspace_bytes(int64_t B, int32_t Hq, int32_t Hkv, int32_t T, int64_t S) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || T <= 0 || S <= 0) return 0;
    const size_t rows = (size_t)B * Hq * T, heads = (size_t)B * Hkv, cols = (size_t)(Hq / Hkv) * T;
    const size_t chunks = (size_t)((S + kWsKeys - 1) / kWsKeys);
    if (cols <= kWsCols) return rows * chunks * sizeof(float2) + heads * S * ((cols + 1) & ~(size_t)1) * sizeof(float);
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
    const int cols = Hq / Hkv * T;
    if (cols <= kWsCols) {
        float* scores = a.lse;                                           // behind the partial states
        const int pad = (cols + 1) & ~1;
        switch (q_dtype) {
            case OMNI_F32:  return launch_weight_step<OMNI_F32, true>(a, scores, pad, st);
            case OMNI_BF16: return rotate_q ? launch_weight_step<OMNI_BF16, true>(a, scores, pad, st) : launch_weight_step<OMNI_BF16, false>(a, scores, pad, st);
            default:        return rotate_q ? launch_weight_step<OMNI_F16, true>(a, scores, pad, st) : launch_weight_step<OMNI_F16, false>(a, scores, pad, st);
        }
    }
    switch (q_dtype) {
        case OMNI_F32:  return launch_weight_sums<OMNI_F32>(a, st);
        case OMNI_BF16: return launch_weight_sums<OMNI_BF16>(a, st);
        default:        return launch_weight_sums<OMNI_F16>(a, st);
    }
}

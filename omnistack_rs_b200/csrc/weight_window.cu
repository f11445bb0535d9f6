// Key weights of many columns (a prompt's last tokens): tcgen05 products in two passes over the keys.
//
// Query columns are the rows of the product (128 at a time), keys its columns:  S[col, key] = Q'[col, :] . K'[key, :].  Q' lives
// in tensor memory for the whole CTA, K' is dequantised tile by tile (128 keys) into shared memory, twice: values and what they
// leave of the centroids, plus the signs.  Two accumulators, since a key's norm multiplies the sign product alone and would have to
// be split as well to ride in it:   A = Qhi Khi + Qhi Klo (+ Qlo Khi),   B = Chi sign + Clo sign,   s = f_A A + f_B norm B.
//
// Pass 1: thread = column, running maximum and sum over the chunk's keys, one pair per (chunk, column) into the workspace.
// Pass 2: the same scores again (cheaper than 4 bytes per key and column written and read), weights 2^(s - lse), and their sum over
// the columns: a halving exchange between the lanes of a warp, then the four warps' parts in order.
//
// Warps 0-3: scores (thread = column).  Warps 4-7: dequantisation (thread = key), two buffers ahead of the products.  Warp 8
// issues the products.  Shared memory is what bounds a tile: 64 lookups of 8 bytes and 40 stores of 16 bytes per key, and the
// products' reads of K', about 1,900 cycles against 1,536 of the tensor pipe.
#include "weight_sums.cuh"

namespace omni {

constexpr int kWwThreads = 288;
constexpr int kWwTile = 128;                       // keys per tile, columns per CTA
constexpr uint32_t kWwLbo = 128;                   // K-major operands: bytes between the two 8-element chunks of a k-step
constexpr uint32_t kWwSbo = 16 * 128, kWwSboSign = 8 * 128;         // ... and between groups of eight keys
constexpr uint32_t kWwBytesV = 128 * 128 * 2, kWwBytesSign = 128 * 64 * 2;
constexpr uint32_t kWwBuf = 2 * kWwBytesV + kWwBytesSign;           // values, remainders, signs
constexpr uint32_t kWwOffLut = 2 * kWwBuf, kWwOffNorm = kWwOffLut + kWsLutBytes, kWwOffRed = kWwOffNorm + 4 * kWwTile * 4,
                   kWwOffBar = kWwOffRed + 4 * kWwTile * 4, kWwSmem = kWwOffBar + 128;
constexpr uint32_t kWwColA = 0, kWwColB = 128, kWwColQhi = 256, kWwColQlo = 320, kWwColChi = 384, kWwColClo = 416, kWwTmemCols = 512;
constexpr uint32_t kWwWaitLimit = 1u << 20;

__device__ __forceinline__ void ww_bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" :: "r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void ww_bar_arrive(uint32_t bar) {
    asm volatile("{\n .reg .b64 t;\n mbarrier.arrive.shared::cta.b64 t, [%0];\n}\n" :: "r"(bar) : "memory");
}
// bounded wait by all lanes of a warp, with one answer
__device__ __forceinline__ bool ww_bar_wait(uint32_t bar, uint32_t parity) {
    bool done = false;
    for (uint32_t i = 0; i < kWwWaitLimit && !done; ++i) {
        uint32_t ok;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        done = ok != 0;
    }
    return __all_sync(kFullMask, done);
}
__device__ __forceinline__ void ww_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void ww_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void ww_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void ww_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void ww_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" :: "r"(bar) : "memory");
}
__device__ __forceinline__ bool ww_elect() {
    uint32_t is;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(is));
    return is != 0;
}
// D[tmem] (+)= A[tmem] B[smem, K-major core matrices of 8 rows x 16 bytes]
__device__ __forceinline__ void ww_mma(uint32_t d, uint32_t a, uint32_t b, uint32_t sbo, uint32_t n, uint32_t accumulate) {
    const uint64_t desc = (uint64_t)((b & 0x3FFFFu) >> 4) | ((uint64_t)(kWwLbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | (1ull << 46);
    const uint32_t idesc = (1u << 4) | ((n >> 3) << 17) | ((128u >> 4) << 24);             // fp16 operands, fp32 accumulator
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                 :: "r"(d), "r"(a), "l"(desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void ww_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                   "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
                   "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
                   "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void ww_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n"
                 :: "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                    "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
                    "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
                    "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
                 : "memory");
}
__device__ __forceinline__ void ww_sts16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};\n" :: "r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint2 ww_lut(uint32_t lut_lane, uint32_t w, int byte) {
    const uint32_t off = (byte == 0 ? w << 7 : byte == 1 ? w >> 1 : byte == 2 ? w >> 9 : w >> 17) & 0x7f80u;
    uint2 v;
    asm("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(lut_lane + off));
    return v;
}

template <int DT, bool QLO, int PASS>
__global__ void __launch_bounds__(kWwThreads, 1) weight_window_kernel(const __grid_constant__ WeightArgs a, int col0, int32_t* status) {
    extern __shared__ __align__(1024) unsigned char ww_smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t bh = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, b = bh / a.Hkv;
    const int h = (int)(bh % a.Hkv), G = a.Hq / a.Hkv, cols = G * a.T;
    const int len = ws_len(a, b);
    const int64_t k_begin64 = chunk * a.chunk_keys;
    float* sums = a.sums + bh * a.S;
    if (k_begin64 >= len) {                                              // nothing but zeros, if anything
        if (PASS == 2 && !a.accumulate && col0 == 0)
            for (int64_t s = k_begin64 + tid; s < a.S && s < k_begin64 + a.chunk_keys; s += kWwThreads) sums[s] = 0.f;
        return;
    }
    const int k_begin = (int)k_begin64;
    const int k_end = len - k_begin < a.chunk_keys ? len : k_begin + (int)a.chunk_keys;
    const int n_tiles = (k_end - k_begin + kWwTile - 1) / kWwTile;
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(ww_smem);
    float* norm_s = reinterpret_cast<float*>(ww_smem + kWwOffNorm);      // ring of four tiles' norms
    float* red_s = reinterpret_cast<float*>(ww_smem + kWwOffRed);
    const uint32_t bar_full = base + kWwOffBar, bar_empty = bar_full + 16, bar_s = bar_empty + 16, bar_free = bar_s + 8, tmem_at = bar_free + 8;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            ww_bar_init(bar_full + 8 * i, 4);
            ww_bar_init(bar_empty + 8 * i, 1);
        }
        ww_bar_init(bar_s, 1);
        ww_bar_init(bar_free, 4);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" :: "r"(tmem_at), "r"(kWwTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    const float cb_mul = ws_build_lut(ww_smem + kWwOffLut, a.codebooks + (a.cb_per_head ? h * 16 : 0), tid);
    if (a.with_qjl && warp >= 4 && warp < 8) {                           // G as +-1, [64 projections][128 dims], where the first values will go
        const int32_t uid = a.user_ids ? __ldg(a.user_ids + b) : a.user_id;
        const int pi = (tid - 128) >> 1, half = tid & 1;                 // projection, and which 64 of its 128 dims
        const uint32_t* gr = a.g_rows + ((size_t)seed_of(uid, h) * kQjlDim + pi) * 4 + 2 * half;
        const uint32_t row = base + (uint32_t)(pi >> 3) * kWwSbo + (uint32_t)(pi & 7) * 16 + (uint32_t)half * 8 * kWwLbo;
#pragma unroll
        for (int wd = 0; wd < 2; ++wd) {
            const uint32_t bits = __ldg(gr + wd);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                ww_sts16(row + (uint32_t)(4 * wd + k) * kWwLbo, ws_signs2(bits >> (8 * k)), ws_signs2(bits >> (8 * k + 2)), ws_signs2(bits >> (8 * k + 4)),
                         ws_signs2(bits >> (8 * k + 6)));
        }
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    }
    ww_fence_before();
    __syncthreads();
    ww_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(tmem) : "r"(tmem_at));
    const uint32_t t_lane = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    const int col = col0 + tid;                                          // of warps 0-3
    const bool col_on = warp < 4 && col < cols;
    float q_mul = 1.f, p_mul = 1.f;

    // ---- Q' into tensor memory -----------------------------------------------------------------------------------------
    if (warp < 4) {
        float q[128];
        const int64_t qrow = col_on ? (b * a.Hq + (int64_t)h * G + col / a.T) * a.T + col % a.T : 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            if (col_on) Elem<DT>::load4(a.q, qrow * kHeadDim + 4 * i, v);
#pragma unroll
            for (int k = 0; k < 4; ++k) q[4 * i + k] = v[k];
        }
        if (a.rotate_q) {                                                // Walsh-Hadamard, stages in order, one rounding each
#pragma unroll
            for (int s = 1; s < 128; s <<= 1) {
#pragma unroll
                for (int i = 0; i < 128; ++i) {
                    if ((i & s) == 0) {
                        const float x = q[i], y = q[i | s];
                        q[i] = __fadd_rn(x, y);
                        q[i | s] = __fsub_rn(x, y);
                    }
                }
            }
            const float s = __uint_as_float(OMNI_WHT_SCALE_BITS);
#pragma unroll
            for (int i = 0; i < 128; ++i) q[i] = __fmul_rn(q[i], s);
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 128; ++i) top = fmaxf(top, fabsf(q[i]));
        q_mul = ws_pow2(top);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            uint32_t v[32], r[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float x = q[64 * j + 2 * i] * q_mul, y = q[64 * j + 2 * i + 1] * q_mul;
                v[i] = ws_half2(x, y);
                if (QLO) r[i] = ws_rest2(x, y, v[i]);
            }
            ww_st32(t_lane + kWwColQhi + 32 * j, v);
            if (QLO) ww_st32(t_lane + kWwColQlo + 32 * j, r);
        }
        ww_wait_st();
        ww_fence_before();
    }
    bool ok = true;
    uint32_t ph_s = 0;                                                   // parity of the next completion of bar_s
    if (a.with_qjl) {                                                    // C = G . q, then split like the centroids
        __syncthreads();
        if (warp == 8) {
            ww_fence_after();
            if (ww_elect()) {
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) ww_mma(tmem + kWwColA, tmem + kWwColQhi + 8 * ks, base + ks * 2 * kWwLbo, kWwSbo, 64, ks > 0);
                if (QLO) {
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) ww_mma(tmem + kWwColA, tmem + kWwColQlo + 8 * ks, base + ks * 2 * kWwLbo, kWwSbo, 64, 1);
                }
                ww_commit(bar_s);
            }
            __syncwarp();
        }
        ok = ww_bar_wait(bar_s, 0);                                      // G's buffer may be overwritten from here on
        ph_s = 1;
        if (ok && warp < 4) {
            ww_fence_after();
            uint32_t p[2][32], v[32], r[32];
            ww_ld32(t_lane + kWwColA, p[0]);
            ww_ld32(t_lane + kWwColA + 32, p[1]);
            ww_wait_ld();
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(p[0][i])), fabsf(__uint_as_float(p[1][i]))));
            p_mul = ws_pow2(top);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float x = __uint_as_float(p[i >> 4][2 * (i & 15)]) * p_mul, y = __uint_as_float(p[i >> 4][2 * (i & 15) + 1]) * p_mul;
                v[i] = ws_half2(x, y);
                r[i] = ws_rest2(x, y, v[i]);
            }
            ww_st32(t_lane + kWwColChi, v);
            ww_st32(t_lane + kWwColClo, r);
            ww_wait_st();
            ww_fence_before();
        }
    }
    ok = __syncthreads_and(ok) != 0;                                     // Q' and C are complete

    if (ok && warp == 8) {
        // ---- products ---------------------------------------------------------------------------------------------------
        ww_fence_after();
        for (int t = 0; ok && t < n_tiles; ++t) {
            const uint32_t kv = base + (t & 1) * kWwBuf;
            ok = ww_bar_wait(bar_full + 8 * (t & 1), (t >> 1) & 1);
            if (ok && t > 0) ok = ww_bar_wait(bar_free, (t - 1) & 1);
            if (!ok) break;
            ww_fence_after();
            if (ww_elect()) {
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) ww_mma(tmem + kWwColA, tmem + kWwColQhi + 8 * ks, kv + ks * 2 * kWwLbo, kWwSbo, 128, ks > 0);
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) ww_mma(tmem + kWwColA, tmem + kWwColQhi + 8 * ks, kv + kWwBytesV + ks * 2 * kWwLbo, kWwSbo, 128, 1);
                if (QLO) {
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) ww_mma(tmem + kWwColA, tmem + kWwColQlo + 8 * ks, kv + ks * 2 * kWwLbo, kWwSbo, 128, 1);
                }
                if (a.with_qjl) {
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) ww_mma(tmem + kWwColB, tmem + kWwColChi + 8 * ks, kv + 2 * kWwBytesV + ks * 2 * kWwLbo, kWwSboSign, 128, ks > 0);
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) ww_mma(tmem + kWwColB, tmem + kWwColClo + 8 * ks, kv + 2 * kWwBytesV + ks * 2 * kWwLbo, kWwSboSign, 128, 1);
                }
                ww_commit(bar_empty + 8 * (t & 1));
                ww_commit(bar_s);
            }
            __syncwarp();
        }
    } else if (ok && warp >= 4) {
        // ---- dequantisation: thread = key ---------------------------------------------------------------------------------
        const int x = tid - 128;
        const uint32_t lut_lane = base + kWwOffLut + 8 * (lane & 15);
        const uint32_t at = (uint32_t)(x >> 3) * kWwSbo + (uint32_t)(x & 7) * 16, at_sign = 2 * kWwBytesV + (uint32_t)(x >> 3) * kWwSboSign + (uint32_t)(x & 7) * 16;
        uint4 nib[4];
        uint2 sign = make_uint2(0u, 0u);
        float norm = 0.f;
        auto fetch = [&](int t) {                                        // keys past the end repeat the last one
            const int k = k_begin + t * kWwTile + x;
            const int64_t row = bh * a.S + (k < k_end ? k : k_end - 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) nib[i] = __ldg(reinterpret_cast<const uint4*>(a.k_nib + row * kNibBytes) + i);
            if (a.with_qjl) {
                sign = __ldg(reinterpret_cast<const uint2*>(a.k_qjl + row * kQjlBytes));
                norm = __ldg(a.k_norms + row);
            }
        };
        fetch(0);
        for (int t = 0; t < n_tiles; ++t) {
            if (t > 1) ok = ww_bar_wait(bar_empty + 8 * (t & 1), ((t >> 1) - 1) & 1);
            if (!ok) break;
            const uint32_t kv = base + (t & 1) * kWwBuf;
#pragma unroll
            for (int i = 0; i < 4; ++i) {                                // sixteen lookups, then their eight stores
                const uint32_t w[4] = {nib[i].x, nib[i].y, nib[i].z, nib[i].w};
                uint2 v[4][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[j][k] = ww_lut(lut_lane, w[j], k);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    ww_sts16(kv + at + (uint32_t)(4 * i + j) * kWwLbo, v[j][0].x, v[j][1].x, v[j][2].x, v[j][3].x);
                    ww_sts16(kv + kWwBytesV + at + (uint32_t)(4 * i + j) * kWwLbo, v[j][0].y, v[j][1].y, v[j][2].y, v[j][3].y);
                }
            }
            if (a.with_qjl) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t bits = (i < 4 ? sign.x : sign.y) >> (8 * (i & 3));
                    ww_sts16(kv + at_sign + (uint32_t)i * kWwLbo, ws_signs2(bits), ws_signs2(bits >> 2), ws_signs2(bits >> 4), ws_signs2(bits >> 6));
                }
            }
            norm_s[(t & 3) * kWwTile + x] = norm;
            if (t + 1 < n_tiles) fetch(t + 1);
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) ww_bar_arrive(bar_full + 8 * (t & 1));
        }
    } else if (ok) {
        // ---- scores: thread = column ------------------------------------------------------------------------------------
        const float f_a = a.scale * kWsLog2e / q_mul / cb_mul, f_b = a.with_qjl ? a.scale * kWsLog2e * kQjlCoef / q_mul / p_mul : 0.f;
        const int last = col_on ? (a.causal ? len - a.T + col % a.T : len - 1) : -1;    // newest key of the column
        const int open_to = a.causal ? len - a.T : len - 1;              // newest key that every column sees
        float m = -INFINITY, l = 0.f, lse = 0.f;
        if (PASS == 2 && col_on) {
            const int n = (int)((len + a.chunk_keys - 1) / a.chunk_keys);
            const float2* p = a.partial + bh * a.chunks * cols + col;
            for (int i = 0; i < n; ++i) m = fmaxf(m, p[(int64_t)i * cols].x);
            const float ref = m == -INFINITY ? 0.f : m;
            for (int i = 0; i < n; ++i) l += p[(int64_t)i * cols].y * exp2f(p[(int64_t)i * cols].x - ref);
            lse = m == -INFINITY && l == 0.f ? 0.f : ref + log2f(l);     // no open key: its scores are -inf
        }
        for (int t = 0; t < n_tiles; ++t) {
            // after a wait that ran out the warp still goes through the barriers it shares with the others, storing nothing
            if (ok) ok = ww_bar_wait(bar_s, (ph_s + t) & 1);
            ww_fence_after();
            const float* nrm = norm_s + (t & 3) * kWwTile;
            float s[128];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t u[32], v[32];
                ww_ld32(t_lane + kWwColA + 32 * j, u);
                if (a.with_qjl) ww_ld32(t_lane + kWwColB + 32 * j, v);
                ww_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) s[32 * j + i] = __uint_as_float(u[i]) * f_a;
                if (a.with_qjl) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 n4 = *reinterpret_cast<const float4*>(nrm + 32 * j + i);
                        s[32 * j + i] = fmaf(__uint_as_float(v[i]) * f_b, n4.x, s[32 * j + i]);
                        s[32 * j + i + 1] = fmaf(__uint_as_float(v[i + 1]) * f_b, n4.y, s[32 * j + i + 1]);
                        s[32 * j + i + 2] = fmaf(__uint_as_float(v[i + 2]) * f_b, n4.z, s[32 * j + i + 2]);
                        s[32 * j + i + 3] = fmaf(__uint_as_float(v[i + 3]) * f_b, n4.w, s[32 * j + i + 3]);
                    }
                }
            }
            ww_fence_before();
            __syncwarp();
            if (lane == 0) ww_bar_arrive(bar_free);                      // the accumulators may be overwritten
            const int k0 = k_begin + t * kWwTile;
            if (k0 + kWwTile - 1 > open_to || k0 + kWwTile > k_end || cols - col0 < kWwTile) {
                const int lim = (last < k_end - 1 ? last : k_end - 1) - k0;
#pragma unroll
                for (int i = 0; i < 128; ++i) s[i] = i <= lim ? s[i] : -INFINITY;
            }
            if (PASS == 1) {
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 128; ++i) mx[i & 3] = fmaxf(mx[i & 3], s[i]);
                const float m_new = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
                const float ref = m_new == -INFINITY ? 0.f : m_new;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 128; ++i) sum[i & 3] += ws_ex2(s[i] - ref);
                l = fmaf(l, ws_ex2(m - ref), (sum[0] + sum[1]) + (sum[2] + sum[3]));
                m = m_new;
            } else {
#pragma unroll
                for (int i = 0; i < 128; ++i) s[i] = ws_ex2(s[i] - lse);
                // sum over the warp's 32 columns: lanes trade halves of their keys until each has the total of four
#pragma unroll
                for (int n = 64, x = 16; n >= 4; n >>= 1, x >>= 1) {
                    const bool up = (lane & x) != 0;
#pragma unroll
                    for (int i = 0; i < 64; ++i) {
                        if (i < n) {
                            const float mine = up ? s[i + n] : s[i], other = up ? s[i] : s[i + n];
                            s[i] = mine + __shfl_xor_sync(kFullMask, other, x);
                        }
                    }
                }
                *reinterpret_cast<float4*>(red_s + warp * kWwTile + 4 * lane) = make_float4(s[0], s[1], s[2], s[3]);
                asm volatile("bar.sync 1, 128;\n" ::: "memory");
                const float total = (red_s[tid] + red_s[kWwTile + tid]) + (red_s[2 * kWwTile + tid] + red_s[3 * kWwTile + tid]);
                if (ok && k0 + tid < k_end) {
                    if (a.accumulate || col0 > 0) sums[k0 + tid] += total;
                    else sums[k0 + tid] = total;
                }
                asm volatile("bar.sync 1, 128;\n" ::: "memory");
            }
        }
        if (PASS == 1 && ok && col_on) a.partial[(bh * a.chunks + chunk) * cols + col] = make_float2(m, l);
        if (PASS == 2 && !a.accumulate && col0 == 0)                     // the rest of the chunk lies behind the length
            for (int64_t s = k_end + tid; s < a.S && s < k_begin64 + a.chunk_keys; s += 128) sums[s] = 0.f;
    }
    if (!ok && status) atomicExch(status, OMNI_STATUS_WAIT_EXPIRED);
    __syncwarp();
    ww_fence_before();
    __syncthreads();
    if (warp == 8) {
        ww_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" :: "r"(tmem), "r"(kWwTmemCols) : "memory");
    }
}

// Keys of a chunk: about three rounds of one CTA per SM, at least 512 (a CTA's prologue costs about as much as two tiles)
static int64_t ww_chunk_keys(int64_t heads, int64_t S) {
    const int64_t per = (heads * S + 148 * 3 - 1) / (148 * 3);
    const int64_t keys = per < 512 ? 512 : (per > 8192 ? 8192 : per);
    return (keys + kWwTile - 1) / kWwTile * kWwTile;
}

size_t weight_window_workspace(int64_t B, int Hq, int Hkv, int T, int64_t S) {
    const int64_t keys = ww_chunk_keys(B * Hkv, S);
    return (size_t)B * Hq * T * ((S + keys - 1) / keys) * sizeof(float2);
}

template <int DT, bool QLO>
static int32_t launch_weight_window_t(const WeightArgs& a, int32_t* status, cudaStream_t st) {
    const int cols = a.Hq / a.Hkv * a.T;
    const unsigned grid = (unsigned)(a.B * a.Hkv * a.chunks);
    OMNI_CUDA(cudaFuncSetAttribute(weight_window_kernel<DT, QLO, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, kWwSmem));
    OMNI_CUDA(cudaFuncSetAttribute(weight_window_kernel<DT, QLO, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, kWwSmem));
    for (int pass = 1; pass <= 2; ++pass) {
        for (int col0 = 0; col0 < cols; col0 += kWwTile) {
            if (pass == 1) weight_window_kernel<DT, QLO, 1><<<grid, kWwThreads, kWwSmem, st>>>(a, col0, status);
            else weight_window_kernel<DT, QLO, 2><<<grid, kWwThreads, kWwSmem, st>>>(a, col0, status);
            OMNI_CUDA(cudaGetLastError());
        }
    }
    return OMNI_OK;
}

int32_t launch_weight_window(WeightArgs a, int q_dtype, int32_t* status, cudaStream_t st) {
    a.chunk_keys = ww_chunk_keys(a.B * a.Hkv, a.S);
    a.chunks = (a.S + a.chunk_keys - 1) / a.chunk_keys;
    OMNI_REQUIRE(a.B * a.Hkv * a.chunks <= 0x7fffffffLL, OMNI_ERR_UNSUPPORTED, "omni_attn_weight_sums: too many keys");
    switch (q_dtype) {
        case OMNI_F32:  return launch_weight_window_t<OMNI_F32, true>(a, status, st);
        case OMNI_BF16: return a.rotate_q ? launch_weight_window_t<OMNI_BF16, true>(a, status, st) : launch_weight_window_t<OMNI_BF16, false>(a, status, st);
        default:        return a.rotate_q ? launch_weight_window_t<OMNI_F16, true>(a, status, st) : launch_weight_window_t<OMNI_F16, false>(a, status, st);
    }
}

}  // namespace omni

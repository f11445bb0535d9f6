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
// A warp works alone on a unit of one head's keys.  Lane (g, c) = (lane / 4, lane % 4) reads bytes 16c .. 16c + 15 of the rows of keys
// g and g + 8: k-step ks takes its bytes 2ks and 2ks + 1, i.e. dims 32c + 4ks .. + 3, and the query fragments are laid out in that order.
// 64 users x 1,500 keys take 37 us, of them 24 here, bound by issue slots (330 instructions per 16 keys, 24 of them products); the keys'
// bytes alone would take 6.  (A product per column in fp32: 310 us.)
#include "weight_sums.cuh"

namespace omni {

constexpr int kWmWarps = 8;
constexpr int kWmLutBytes = 256 * 32 * 8;

// wm_mma into a fresh accumulator
__device__ __forceinline__ void wm_mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// +-1 as fp16 for bits i and i + 16 of z (1 = +1): what an operand register pairs, at two instructions
__device__ __forceinline__ uint32_t wm_sign_pair(uint32_t z, int i) { return ((z << (15 - i)) & 0x80008000u) ^ 0xBC00BC00u; }

struct WmKeys { uint4 n0, n1; uint32_t s0, s1; float r0, r1; };          // this lane's part of keys g and g + 8 of a block of 16

// A warp per (user, head): the query and projection fragments of every lane and the score factors of its two result columns, as
// kWmPieces<QLO> 16-byte pieces [piece][lane].
template <bool QLO> constexpr int kWmPieces = QLO ? 13 : 9;
constexpr int kWmPrepWarps = 4;
template <int DT, bool QLO>
__global__ void __launch_bounds__(kWmPrepWarps * 32) weight_fragments_kernel(const __grid_constant__ WeightArgs a) {
    __shared__ __align__(16) float c_s[kWmPrepWarps][kWsStepCols][kQjlDim + 4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    follow_me_early();
    if (blockIdx.x == gridDim.x - 1) {
        ws_tiles_before<kWmPrepWarps>(a, tid);
        return;
    }
    const int64_t bh = (int64_t)blockIdx.x * kWmPrepWarps + warp;
    if (bh >= a.B * a.Hkv) return;
    const int64_t b = bh / a.Hkv;
    const int h = (int)(bh % a.Hkv), G = a.Hq / a.Hkv, cols = G * a.T;
    float cb_top = fabsf(__ldg(a.codebooks + (a.cb_per_head ? h * 16 : 0) + (lane & 15)));
#pragma unroll
    for (int x = 8; x >= 1; x >>= 1) cb_top = fmaxf(cb_top, __shfl_xor_sync(kFullMask, cb_top, x));
    const float cb_mul = ws_pow2(cb_top);

    uint32_t qv[8][2], qr[QLO ? 8 : 1][2];
    float p[16];
    const float q_mul = ws_columns8<DT, QLO>(a, b, h, g < cols ? g : -1, 1.f, c_s[warp], lane, qv, qr, p);
    // ---- G . q of the head's 64 projections -------------------------------------------------------------------------------------
    uint32_t pv[4][2], pr[4][2];
    float p_mul = 1.f;
    if (a.with_qjl) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(p[i]));
        top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 1));
        top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 2));
        p_mul = ws_pow2(top);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {                            // a register pairs projections i and i + 8 (see wm_sign_pair)
                const float u = p[2 * s + x] * p_mul, v = p[2 * s + x + 8] * p_mul;
                pv[s][x] = ws_half2(u, v);
                pr[s][x] = ws_rest2(u, v, pv[s][x]);
            }
        }
    }
    // factors of this lane's two result columns (they are lanes 8c and 8c + 4's columns); powers of two divide exactly
    float f_cb[2], f_sg[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const float qm = __shfl_sync(kFullMask, q_mul, 8 * c + 4 * x), pm = __shfl_sync(kFullMask, p_mul, 8 * c + 4 * x);
        f_cb[x] = a.scale * kWsLog2e / qm / cb_mul;
        f_sg[x] = a.scale * kWsLog2e * kQjlCoef / qm / pm;
    }
    uint4* out = reinterpret_cast<uint4*>(a.prepared) + bh * (kWmPieces<QLO> * 32) + lane;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        out[32 * k] = make_uint4(qv[2 * k][0], qv[2 * k][1], qv[2 * k + 1][0], qv[2 * k + 1][1]);
        if (a.with_qjl) out[32 * (4 + k)] = make_uint4(pv[k][0], pv[k][1], pr[k][0], pr[k][1]);
        if constexpr (QLO) out[32 * (9 + k)] = make_uint4(qr[2 * k][0], qr[2 * k][1], qr[2 * k + 1][0], qr[2 * k + 1][1]);
    }
    out[32 * 8] = make_uint4(__float_as_uint(f_cb[0]), __float_as_uint(f_cb[1]), __float_as_uint(f_sg[0]), __float_as_uint(f_sg[1]));
}

// A CTA's share of the row of tiles, heads first (kv head, user, tile), so that its centroid table rarely changes.  Warp w takes keys
// 16 w .. 16 w + 15 of every tile; its maximum and sum of a span are entry w of span (head number, CTA) = head number + CTA.
template <bool QLO>
__global__ void __launch_bounds__(kWmWarps * 32, 2) weight_step_kernel(const __grid_constant__ WeightArgs a, int pad) {
    extern __shared__ __align__(128) unsigned char wm_smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int cols = a.Hq / a.Hkv * a.T;
    int table = -1;                                                      // head whose table is in shared memory
    if (!a.cb_per_head) {
        ws_build_lut<32>(wm_smem, a.codebooks, tid);
        table = 0;
    }
    after_predecessor();
    __syncthreads();
    const int64_t per_head = *(volatile const int32_t*)(a.tiles_before + a.B), all = per_head * a.Hkv;
    const int64_t sharers = ws_sharers(gridDim.x, all);
    if (blockIdx.x >= sharers) return;
    const int64_t x0 = blockIdx.x * all / sharers, x1 = (blockIdx.x + 1) * all / sharers;
    int left = (int)(x1 - x0);                                           // tiles still to come, this span's among them
    int h = (int)(x0 / per_head), b = ws_user_of(a, x0 % per_head, 1, lane);
    int tile = (int)(x0 % per_head) - a.tiles_before[b];
    const uint32_t lane8 = 8 * lane;
    // entry of byte k of word u, this lane's copy: the address is (byte << 8) | lane8
    auto look = [&](uint32_t u, int k) { return *reinterpret_cast<const uint2*>(wm_smem + __byte_perm(u, lane8, 0x5504 | (k << 4))); };
    while (left > 0) {
        const int64_t bh = (int64_t)b * a.Hkv + h, row0 = bh * a.S;
        const int len = ws_len(a, b), tiles = (len + kWsTile - 1) / kWsTile;
        const int n_span = tiles - tile < left ? tiles - tile : left;
        const int k_end = len < (tile + n_span) * kWsTile ? len : (tile + n_span) * kWsTile;
        int k0 = tile * kWsTile + 16 * warp;
        const uint4* nib = reinterpret_cast<const uint4*>(a.k_nib + row0 * kNibBytes) + c;
        const uint16_t* sgn = reinterpret_cast<const uint16_t*>(a.k_qjl + row0 * kQjlBytes) + c;
        const float* nrm = a.k_norms + row0;
        auto load = [&](WmKeys& x) {
            int ka = k0 + g, kb = k0 + g + 8;
            if (k0 + 16 > k_end) {                                       // keys past the end repeat the last one
                ka = ka < k_end ? ka : k_end - 1;
                kb = kb < k_end ? kb : k_end - 1;
            }
            x.n0 = __ldg(nib + 4 * (int64_t)ka);
            x.n1 = __ldg(nib + 4 * (int64_t)kb);
            if (a.with_qjl) {
                x.s0 = __ldg(sgn + 4 * (int64_t)ka);
                x.s1 = __ldg(sgn + 4 * (int64_t)kb);
                x.r0 = __ldg(nrm + ka);
                x.r1 = __ldg(nrm + kb);
            }
        };
        WmKeys next;
        next.s0 = next.s1 = 0; next.r0 = next.r1 = 0.f;
        if (k0 < k_end) load(next);
        uint32_t qv[8][2], qr[QLO ? 8 : 1][2], pv[4][2], pr[4][2];
        float f_cb[2], f_sg[2];
        {
            const uint4* in = reinterpret_cast<const uint4*>(a.prepared) + bh * (kWmPieces<QLO> * 32) + lane;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint4 v = in[32 * k];
                qv[2 * k][0] = v.x; qv[2 * k][1] = v.y; qv[2 * k + 1][0] = v.z; qv[2 * k + 1][1] = v.w;
                uint4 u = make_uint4(0u, 0u, 0u, 0u);
                if (a.with_qjl) u = in[32 * (4 + k)];
                pv[k][0] = u.x; pv[k][1] = u.y; pr[k][0] = u.z; pr[k][1] = u.w;
                if constexpr (QLO) {
                    const uint4 r = in[32 * (9 + k)];
                    qr[2 * k][0] = r.x; qr[2 * k][1] = r.y; qr[2 * k + 1][0] = r.z; qr[2 * k + 1][1] = r.w;
                }
            }
            const uint4 f = in[32 * 8];
            f_cb[0] = __uint_as_float(f.x); f_cb[1] = __uint_as_float(f.y); f_sg[0] = __uint_as_float(f.z); f_sg[1] = __uint_as_float(f.w);
        }
        if (table != (a.cb_per_head ? h : 0)) {                          // (the same for the whole CTA)
            __syncthreads();
            table = a.cb_per_head ? h : 0;
            ws_build_lut<32>(wm_smem, a.codebooks + 16 * table, tid);
            __syncthreads();
        }
        int last[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int col = 2 * c + x;
            last[x] = col < cols ? (a.causal ? len - a.T + col % a.T : len - 1) : -1;
            last[x] = last[x] < k_end - 1 ? last[x] : k_end - 1;
        }
        // keys below this are open to every column; with columns to spare, none are
        const int open_to = cols < kWsStepCols ? 0 : (a.causal && len - a.T + 1 < k_end ? len - a.T + 1 : k_end);

        // ---- keys -------------------------------------------------------------------------------------------------------
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        auto block = [&](const WmKeys& x, int at) {                      // keys at .. at + 15
            float* dst = a.scores + (row0 + at + g) * pad + 2 * c;
            // rows g and g + 8 of a product: value and remainder of key g (d), of key g + 8 (e); a lookup's two words are then neighbouring
            // operand registers (with keys as all sixteen rows, 64 register moves per block)
            float d[4], e[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const uint32_t u0 = w == 0 ? x.n0.x : w == 1 ? x.n0.y : w == 2 ? x.n0.z : x.n0.w;
                const uint32_t u1 = w == 0 ? x.n1.x : w == 1 ? x.n1.y : w == 2 ? x.n1.z : x.n1.w;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int ks = 2 * w + k;
                    const uint2 t0 = look(u0, 2 * k), t1 = look(u0, 2 * k + 1), t2 = look(u1, 2 * k), t3 = look(u1, 2 * k + 1);
                    if (ks == 0) {
                        wm_mma0(d, t0.x, t0.y, t1.x, t1.y, qv[ks][0], qv[ks][1]);
                        wm_mma0(e, t2.x, t2.y, t3.x, t3.y, qv[ks][0], qv[ks][1]);
                    } else {
                        wm_mma(d, t0.x, t0.y, t1.x, t1.y, qv[ks][0], qv[ks][1]);
                        wm_mma(e, t2.x, t2.y, t3.x, t3.y, qv[ks][0], qv[ks][1]);
                    }
                    if (QLO) {
                        wm_mma(d, t0.x, t0.y, t1.x, t1.y, qr[ks][0], qr[ks][1]);
                        wm_mma(e, t2.x, t2.y, t3.x, t3.y, qr[ks][0], qr[ks][1]);
                    }
                }
            }
            d[0] = (d[0] + d[2]) * f_cb[0];
            d[1] = (d[1] + d[3]) * f_cb[1];
            d[2] = (e[0] + e[2]) * f_cb[0];
            d[3] = (e[1] + e[3]) * f_cb[1];
            if (a.with_qjl) {
                float s[4], t[4];
                const uint32_t z0 = __byte_perm(x.s0, 0, 0x4140), z1 = __byte_perm(x.s1, 0, 0x4140);    // bits 0-7 and 8-15 to the halves
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t a0 = wm_sign_pair(z0, 2 * i), a1 = wm_sign_pair(z1, 2 * i), a2 = wm_sign_pair(z0, 2 * i + 1), a3 = wm_sign_pair(z1, 2 * i + 1);
                    if (i == 0) {
                        wm_mma0(s, a0, a1, a2, a3, pv[i][0], pv[i][1]);
                        wm_mma0(t, a0, a1, a2, a3, pr[i][0], pr[i][1]);
                    } else {
                        wm_mma(s, a0, a1, a2, a3, pv[i][0], pv[i][1]);
                        wm_mma(t, a0, a1, a2, a3, pr[i][0], pr[i][1]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) d[i] = fmaf((s[i] + t[i]) * f_sg[i & 1], i < 2 ? x.r0 : x.r1, d[i]);
            }
            if (at + 16 > open_to) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (at + g + (i < 2 ? 0 : 8) > last[i & 1]) d[i] = -INFINITY;
            }
            if (2 * c < cols) {
                if (at + g < k_end) *reinterpret_cast<float2*>(dst) = make_float2(d[0], d[1]);
                if (at + g + 8 < k_end) *reinterpret_cast<float2*>(dst + 8 * pad) = make_float2(d[2], d[3]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // NaN scores: fmaxf drops them, the sum keeps them
                const float m_new = fmaxf(m[i], fmaxf(d[i], d[i + 2]));
                const float ref = m_new == -INFINITY ? 0.f : m_new;
                l[i] = l[i] * ws_ex2(m[i] - ref) + (ws_ex2(d[i] - ref) + ws_ex2(d[i + 2] - ref));
                m[i] = m_new;
            }
        };
        WmKeys other;
        other.s0 = other.s1 = 0; other.r0 = other.r1 = 0.f;
        while (k0 < k_end) {                                             // two sets of registers in turn: copying one costs a dozen moves
            k0 += kWsTile;
            if (k0 < k_end) load(other);
            block(next, k0 - kWsTile);
            if (k0 >= k_end) break;
            k0 += kWsTile;
            if (k0 < k_end) load(next);
            block(other, k0 - kWsTile);
        }
        // ---- this warp's maximum and sum per column of the span -----------------------------------------------------------------
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float top = m[i];
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, s));
            const float ref = top == -INFINITY ? 0.f : top;
            float sum = l[i] * ws_ex2(m[i] - ref);
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) sum += __shfl_xor_sync(kFullMask, sum, s);
            if (g == 0 && 2 * c + i < cols)
                a.partial[(((int64_t)h * a.B + b + blockIdx.x) * kWmWarps + warp) * cols + 2 * c + i] = make_float2(top, sum);
        }
        left -= n_span;
        tile = 0;
        if (left > 0) {                                                  // the next user with keys, or the next head's first one
            do {
                if (++b == a.B) { b = 0; ++h; }
            } while (ws_len(a, b) == 0);
        }
    }
}

// weights of the kept scores: sums[s] (+)= sum_c 2^(score_c - max_c) / sum_c
constexpr int kWfThreads = 256, kWfKeys = 2;       // keys per thread
__global__ void __launch_bounds__(kWfThreads) weight_finish_kernel(const __grid_constant__ WeightArgs a, int pad, int64_t segments, int64_t ctas) {
    __shared__ float2 norm[kWsStepCols];                                 // the columns' maxima and reciprocal sums
    const int tid = threadIdx.x;
    const int64_t bh = blockIdx.x / segments, s0 = blockIdx.x % segments * (kWfKeys * kWfThreads);
    const int64_t b = bh / a.Hkv, h = bh % a.Hkv;
    const int cols = a.Hq / a.Hkv * a.T;
    const bool ordered = a.causal && a.T > 1;                            // a column may see fewer keys than there are
    after_predecessor();
    const int len = ws_len(a, b);
    float2 v[kWfKeys][kWsStepCols / 2];                                  // the scores, requested before the normalisers are known
#pragma unroll
    for (int k = 0; k < kWfKeys; ++k) {
        const int64_t s = s0 + k * kWfThreads + tid;
#pragma unroll
        for (int i = 0; i < kWsStepCols / 2; ++i)
            v[k][i] = s < len && 2 * i < cols ? *(reinterpret_cast<const float2*>(a.scores + (bh * a.S + s) * pad) + i) : make_float2(-INFINITY, -INFINITY);
    }
    if (s0 < len) {
        // the entries of the head's spans: of the CTAs whose shares hold its first and its last tile, and those between
        const int64_t per_head = a.tiles_before[a.B], all = per_head * a.Hkv;
        const int64_t first = h * per_head + a.tiles_before[b], c0 = ws_cta_of(first, ctas, all);
        const int n = (int)(ws_cta_of(first + (len + kWsTile - 1) / kWsTile - 1, ctas, all) - c0 + 1) * kWmWarps;
        const int warp = tid >> 5, lane = tid & 31;                      // a warp per column
        if (warp < cols) {
            const float2* p = a.partial + (h * a.B + b + c0) * kWmWarps * cols + warp;
            float m = -INFINITY, l = 0.f;
            for (int i = lane; i < n; i += 32) m = fmaxf(m, p[(int64_t)i * cols].x);
#pragma unroll
            for (int x = 16; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, x));
            const float ref = m == -INFINITY ? 0.f : m;
            for (int i = lane; i < n; i += 32) l += p[(int64_t)i * cols].y * exp2f(p[(int64_t)i * cols].x - ref);
#pragma unroll
            for (int x = 16; x >= 1; x >>= 1) l += __shfl_xor_sync(kFullMask, l, x);
            if (lane == 0) norm[warp] = make_float2(ref, m == -INFINITY && l == 0.f ? 0.f : 1.f / l);   // no open key: its scores are -inf
        }
        __syncthreads();
    } else if (a.accumulate) {
        return;
    }
#pragma unroll
    for (int k = 0; k < kWfKeys; ++k) {
        const int64_t s = s0 + k * kWfThreads + tid;
        if (s >= a.S) break;
        float total = 0.f;
        if (s < len) {
#pragma unroll
            for (int i = 0; i < kWsStepCols / 2; ++i) {
                if (2 * i < cols) total = fmaf(ws_ex2(v[k][i].x - norm[2 * i].x), norm[2 * i].y, total);
                if (2 * i + 1 < cols) total = fmaf(ws_ex2(v[k][i].y - norm[2 * i + 1].x), norm[2 * i + 1].y, total);
            }
            if (ordered && total != total) {                             // keys behind a column's token add nothing, not zero times a NaN query's normaliser
                total = 0.f;
#pragma unroll
                for (int i = 0; i < kWsStepCols; ++i)
                    if (i < cols && s <= len - a.T + i % a.T) total = fmaf(ws_ex2(((i & 1) ? v[k][i / 2].y : v[k][i / 2].x) - norm[i].x), norm[i].y, total);
            }
        }
        float* d = a.sums + bh * a.S + s;
        if (!a.accumulate) *d = total;
        else if (s < len) *d += total;
    }
}

// The CTAs of a call: two per SM, or one per tile where there are fewer
static int64_t wm_ctas(int64_t heads, int64_t S) {
    const int64_t tiles = heads * ((S + kWsTile - 1) / kWsTile);
    return tiles < 148 * 2 ? tiles : 148 * 2;
}
static size_t wm_prep_bytes(int64_t heads, bool split) { return (size_t)heads * (split ? kWmPieces<true> : kWmPieces<false>) * 32 * 16; }
static size_t wm_partial_bytes(int64_t heads, int64_t S, int64_t cols) { return (size_t)(heads + wm_ctas(heads, S)) * kWmWarps * cols * sizeof(float2); }

template <int DT, bool QLO>
static int32_t launch_weight_step(WeightArgs a, cudaStream_t st) {
    const int64_t heads = a.B * a.Hkv, segments = (a.S + kWfKeys * kWfThreads - 1) / (kWfKeys * kWfThreads), ctas = wm_ctas(heads, a.S), cols = (int64_t)(a.Hq / a.Hkv) * a.T;
    const int pad = (int)((cols + 1) & ~1);
    OMNI_REQUIRE(heads * segments <= 0x7fffffffLL && a.B * ((a.S + kWsTile - 1) / kWsTile) <= 0x7fffffffLL, OMNI_ERR_UNSUPPORTED, "omni_attn_weight_sums: too many keys");
    unsigned char* ws = reinterpret_cast<unsigned char*>(a.partial);     // prepared columns, tiles in front of every user, partial states, scores
    a.prepared = ws;
    ws += wm_prep_bytes(heads, QLO);
    a.tiles_before = reinterpret_cast<int32_t*>(ws);
    ws += ws_before_bytes(a.B);
    a.partial = reinterpret_cast<float2*>(ws);
    a.scores = reinterpret_cast<float*>(ws + wm_partial_bytes(heads, a.S, cols));
    weight_fragments_kernel<DT, QLO><<<(unsigned)((heads + kWmPrepWarps - 1) / kWmPrepWarps + 1), kWmPrepWarps * 32, 0, st>>>(a);
    OMNI_CUDA(cudaGetLastError());
    OMNI_ALLOW_SMEM((weight_step_kernel<QLO>), kWmLutBytes);
    OMNI_CUDA(launch_early(weight_step_kernel<QLO>, dim3((unsigned)ctas), kWmWarps * 32, kWmLutBytes, st, a, pad));
    return check_cuda(launch_early(weight_finish_kernel, dim3((unsigned)(heads * segments)), kWfThreads, 0, st, a, pad, segments, ctas), "weight_finish_kernel launch");
}

}  // namespace omni

using namespace omni;

extern "C" size_t omni_attn_weight_sums_workspace_bytes(int64_t B, int32_t Hq, int32_t Hkv, int32_t T, int64_t S) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || T <= 0 || S <= 0) return 0;
    const size_t heads = (size_t)B * Hkv, cols = (size_t)(Hq / Hkv) * T;
    if (cols > kWsStepCols) return weight_window_workspace(B, Hq, Hkv, T, S);
    return wm_prep_bytes((int64_t)heads, true) + ws_before_bytes(B) + wm_partial_bytes((int64_t)heads, S, (int64_t)cols) +
           heads * S * ((cols + 1) & ~(size_t)1) * sizeof(float);
}

extern "C" int32_t omni_attn_weight_sums(const omni_weight_sums_t* call, void* stream) {
    OMNI_REQUIRE(call != nullptr, OMNI_ERR_ARG, "omni_attn_weight_sums: NULL call");
    const omni_weight_sums_t& p = *call;
    const int64_t B = p.B, S = p.S;
    const int32_t Hq = p.Hq, Hkv = p.Hkv, T = p.T, q_dtype = p.q_dtype, with_qjl = p.with_qjl, rotate_q = p.rotate_q;
    OMNI_REQUIRE(B >= 0 && S >= 0 && T >= 0 && Hq > 0 && Hkv > 0, OMNI_ERR_ARG, "omni_attn_weight_sums: bad extent");
    OMNI_REQUIRE(Hq % Hkv == 0, OMNI_ERR_ARG, "omni_attn_weight_sums: Hq=%d is not a multiple of Hkv=%d", Hq, Hkv);
    OMNI_REQUIRE(Hkv <= kSeeds, OMNI_ERR_UNSUPPORTED, "omni_attn_weight_sums: Hkv=%d exceeds %d heads", Hkv, kSeeds);
    OMNI_REQUIRE(q_dtype >= 0 && q_dtype <= 2, OMNI_ERR_ARG, "omni_attn_weight_sums: unknown dtype code %d", q_dtype);
    if (B == 0 || S == 0) return OMNI_OK;
    OMNI_REQUIRE(p.sums != nullptr, OMNI_ERR_ARG, "omni_attn_weight_sums: NULL buffer");
    cudaStream_t st = (cudaStream_t)stream;
    if (T == 0) {
        if (!p.accumulate) OMNI_CUDA(cudaMemsetAsync(p.sums, 0, (size_t)(B * Hkv * S) * sizeof(float), st));
        return OMNI_OK;
    }
    OMNI_REQUIRE(p.q && p.k_nib && p.codebooks && (!with_qjl || (p.k_qjl && p.k_norms)), OMNI_ERR_ARG, "omni_attn_weight_sums: NULL buffer");
    OMNI_REQUIRE((((uintptr_t)p.q | (uintptr_t)p.k_nib) & 15) == 0 && ((uintptr_t)p.k_qjl & 7) == 0, OMNI_ERR_ARG, "omni_attn_weight_sums: misaligned buffer");
    OMNI_REQUIRE(p.workspace && p.workspace_bytes >= omni_attn_weight_sums_workspace_bytes(B, Hq, Hkv, T, S) && ((uintptr_t)p.workspace & 15) == 0,
                 OMNI_ERR_ARG, "omni_attn_weight_sums: workspace too small or misaligned");
    const DeviceTables* tab = tables_for_current_device();
    if (!tab) return OMNI_ERR_NOT_INIT;
    WeightArgs a{};
    a.q = p.q; a.k_nib = p.k_nib; a.k_qjl = p.k_qjl; a.k_norms = p.k_norms; a.codebooks = p.codebooks; a.cb_per_head = p.cb_per_head;
    a.user_ids = p.user_ids; a.user_id = p.user_id; a.seq_lens = p.seq_lens; a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.T = T; a.S = S;
    a.scale = p.scale; a.with_qjl = with_qjl; a.rotate_q = rotate_q; a.causal = p.causal; a.accumulate = p.accumulate;
    a.g_rows = tab->rows; a.partial = reinterpret_cast<float2*>(p.workspace); a.sums = p.sums;
    OMNI_REQUIRE(S <= 0x7fffff00LL && B * Hkv <= 0x7fffffffLL && (int64_t)(Hq / Hkv) * T <= 0x7fffffffLL, OMNI_ERR_UNSUPPORTED, "omni_attn_weight_sums: too many keys");
    if (Hq / Hkv * (int64_t)T > kWsStepCols) return launch_weight_window(a, q_dtype, p.status_word, st);
    switch (q_dtype) {
        case OMNI_F32:  return launch_weight_step<OMNI_F32, true>(a, st);
        case OMNI_BF16: return rotate_q ? launch_weight_step<OMNI_BF16, true>(a, st) : launch_weight_step<OMNI_BF16, false>(a, st);
        default:        return rotate_q ? launch_weight_step<OMNI_F16, true>(a, st) : launch_weight_step<OMNI_F16, false>(a, st);
    }
}

// Key weights of many columns (a prompt's last tokens): tcgen05 products in two passes over the keys.
//
// Query columns are the rows of the product (128 at a time), keys its columns:  S[col, key] = Q'[col, :] . K'[key, :].  Q' is made
// once by a launch of its own (rotation, scaling, G . q, fp16 values and remainders) and lives in tensor memory for a span, K' is
// dequantised tile by tile (128 keys) into shared memory, twice: values and what they leave of the centroids, plus the signs.  Two
// accumulators, since a key's norm multiplies the sign product alone and would have to be split as well to ride in it:
//   A = Qhi Khi + Qhi Klo (+ Qlo Khi),   B = Chi sign + Clo sign,   s = f_A A + f_B norm B.
//
// The tiles of all (user, head) lie in one row, cut into equal shares, one per CTA: lengths differ, and only the device knows
// them.  A run of tiles of one head inside a share is a span; span (head, CTA) is number head + CTA, which no other span has.
// Pass 1: thread = column, running maximum and sum over a span's keys, one pair per (span, column) into the workspace.
// Pass 2: the same scores again (cheaper than 4 bytes per key and column written and read), weights 2^(s - max) / sum, and their sum over
// the columns.  There a thread reads four columns of 16 keys (the 16-row form of the tensor-memory load), so that most of the sum is its
// own: eight lanes trade halves, then the four warps' parts in order (one column of 64 keys per thread: 62 instead of 14 exchanges).
//
// Warps 0-7: scores, two threads per column with 64 of a tile's keys each.  (One thread per column and key left each scheduler two
// warps, which issued an instruction every third cycle: 135 us for a pass of 16 users x 8,192 keys x 128 columns.)  Warps 8-15:
// dequantisation, two threads per key, up to two buffers ahead of the products; with a span's first tile they bring its columns (the
// score warps doing so between two spans had the products wait: 210 us instead of 190 for 16 users x 8 heads x up to 8,192 keys x 128
// columns).  Warp 16 issues the products.
// Shared memory bounds a tile: 64 lookups of 8 bytes and 40 stores of 16 bytes per key, and the products' reads of K', about 1,900 cycles
// against 1,536 of the tensor pipe.  Measured, a tile takes 2,400 cycles in pass 1 and 3,200 in pass 2, and the call 150 us, 18.7 of which
// its products would need alone.
#include "weight_sums.cuh"

namespace omni {

constexpr int kWwTile = kWsTile;                   // keys per tile, columns per CTA
constexpr int kWwThreads = 640;                    // warps 17-19 only complete the last warpgroup
// Registers: launched with 96 per thread (61,440); scores go up to 144, dequantisation down to 72, the rest to 48
// (256 * 144 + 256 * 72 + 128 * 48 = 61,440).
constexpr int kWwScoreRegs = 144, kWwKeyRegs = 72, kWwOtherRegs = 48;
// Prepared columns: per (head, 128 columns) 48 rows of 128 16-byte pieces -- 16 of Q' values, 16 of what they leave, 8 of G . q values,
// 8 of what those leave -- and the columns' 128 score factors.
constexpr int kWwPrepRows = 48;
constexpr size_t kWwPrepBytes = (size_t)kWwPrepRows * kWwTile * 16 + kWwTile * 4;
// G . q is at most 128 times the query's scaled maximum (below 2^14), so 2^-7 keeps it inside fp16, and the same factor for every
// column lets it ride, with the coefficient and the table's factor, in the keys' norms.
constexpr float kWwProjMul = 1.f / 128.f;
constexpr uint32_t kWwLbo = 128;                   // K-major operands: bytes between the two 8-element chunks of a k-step
constexpr uint32_t kWwSbo = 16 * 128, kWwSboSign = 8 * 128;         // ... and between groups of eight keys
constexpr uint32_t kWwBytesV = 128 * 128 * 2, kWwBytesSign = 128 * 64 * 2;
constexpr uint32_t kWwLutBytes = 256 * 16 * 8;
constexpr uint32_t kWwBuf = 2 * kWwBytesV + kWwBytesSign;           // values, remainders, signs
constexpr uint32_t kWwOffLut = 2 * kWwBuf, kWwOffNorm = kWwOffLut + kWwLutBytes, kWwOffRed = kWwOffNorm + 4 * kWwTile * 4,
                   kWwOffBar = kWwOffRed + 2 * 4 * kWwTile * 4, kWwSmem = kWwOffBar + 128;
// Tensor memory: accumulators, then Q'.  Without remainders two sets of it fit, and the next head's columns are written while products
// read this head's.
constexpr uint32_t kWwColA = 0, kWwColB = 128, kWwColQ = 256, kWwTmemCols = 512;
template <bool QLO> struct WwSet {
    static constexpr uint32_t kQlo = 64, kChi = QLO ? 128 : 64, kClo = QLO ? 160 : 96;   // columns behind those of Q' values
    static constexpr uint32_t kNext = QLO ? 0 : 128;                     // columns from one set to the other
};
constexpr uint32_t kWwWaitLimit = 1u << 22;

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
__device__ __forceinline__ void ww_ld32(uint32_t taddr, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                   "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
                   "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
                   "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(taddr) : "memory");
}
// 16 rows x 64 columns: v[4 i ..] holds columns 8 i + 2 (lane % 4) and the next one of rows lane / 4 and lane / 4 + 8
__device__ __forceinline__ void ww_ld16x64(uint32_t taddr, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
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
__device__ __forceinline__ void ww_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n"
                 :: "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                    "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
// two fp32 operations in one instruction
__device__ __forceinline__ uint64_t ww_pack2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 ww_unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t ww_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t ww_add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
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

// Eight columns per warp: rotation, power-of-two scaling, G . q, and all of it as fp16 values and remainders.  (A column per warp with
// sums in fp32 and pieces of 16 bytes every 2 KiB: 25 us for 16,384 columns; four columns: 18 us.)
constexpr int kWpWarps = 4, kWpCols = 8;
template <int DT, bool QLO>
__global__ void __launch_bounds__(kWpWarps * 32) weight_prepare_kernel(const __grid_constant__ WeightArgs a, int64_t col_groups) {
    __shared__ __align__(16) float hand_s[kWpWarps][kWpCols][kQjlDim + 4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    follow_me_early();
    if (blockIdx.x == gridDim.x - 1) {
        ws_tiles_before<kWpWarps>(a, tid);
        return;
    }
    const int64_t bh = blockIdx.x / col_groups, b = bh / a.Hkv;
    const int h = (int)(bh % a.Hkv), cols = a.Hq / a.Hkv * a.T;
    const int col = ((int)(blockIdx.x % col_groups) * kWpWarps + warp) * kWpCols + g;
    if (col - g >= cols) return;
    float cb_top = fabsf(__ldg(a.codebooks + (a.cb_per_head ? h * 16 : 0) + (lane & 15)));
#pragma unroll
    for (int x = 8; x >= 1; x >>= 1) cb_top = fmaxf(cb_top, __shfl_xor_sync(kFullMask, cb_top, x));
    uint32_t qv[8][2], qr[QLO ? 8 : 1][2];
    float p[16];
    // a negative scale goes into the queries, so that the largest product is the largest score
    const float q_mul = ws_columns8<DT, QLO>(a, b, h, col < cols ? col : -1, a.scale, hand_s[warp], lane, qv, qr, p);
    if (col >= cols) return;
    unsigned char* out = reinterpret_cast<unsigned char*>(a.prepared) + (bh * ((cols + kWwTile - 1) / kWwTile) + col / kWwTile) * kWwPrepBytes;
    uint4* piece = reinterpret_cast<uint4*>(out) + col % kWwTile;         // a warp's stores fill whole sectors: eight columns side by side
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        piece[(4 * c + i) * kWwTile] = make_uint4(qv[2 * i][0], qv[2 * i][1], qv[2 * i + 1][0], qv[2 * i + 1][1]);
        if constexpr (QLO) piece[(16 + 4 * c + i) * kWwTile] = make_uint4(qr[2 * i][0], qr[2 * i][1], qr[2 * i + 1][0], qr[2 * i + 1][1]);
    }
    if (a.with_qjl) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t v[4], r[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float x = p[8 * i + 2 * k] * kWwProjMul, y = p[8 * i + 2 * k + 1] * kWwProjMul;
                v[k] = ws_half2(x, y);
                r[k] = ws_rest2(x, y, v[k]);
            }
            piece[(32 + 2 * c + i) * kWwTile] = make_uint4(v[0], v[1], v[2], v[3]);
            piece[(40 + 2 * c + i) * kWwTile] = make_uint4(r[0], r[1], r[2], r[3]);
        }
    }
    // never zero, as zero times a masked score's -inf is NaN; the factor of tiny queries and centroids is below 1e-37
    if (c == 0) reinterpret_cast<float*>(out + (size_t)kWwPrepRows * kWwTile * 16)[col % kWwTile] = fmaxf(a.scale * kWsLog2e / q_mul / ws_pow2(cb_top), 1.401298464e-45f);
}

// Position in the row of tiles: user, kv head, tile of that head.  Users without keys have no place in it.
struct WwPlace {
    int b, h, tile, len, n_tiles;                     // the user's length and its tiles per head
    __device__ __forceinline__ void user(const WeightArgs& a) { len = ws_len(a, b); n_tiles = (len + kWwTile - 1) / kWwTile; }
    // the place of tile x, by a warp
    __device__ __forceinline__ void find(const WeightArgs& a, int64_t x, int lane) {
        b = ws_user_of(a, x, a.Hkv, lane);
        user(a);
        const int64_t in = x - (int64_t)a.tiles_before[b] * a.Hkv;
        h = (int)(in / n_tiles);
        tile = (int)(in % n_tiles);
    }
    // behind the last tile of this head
    __device__ __forceinline__ void next_head(const WeightArgs& a) {
        tile = 0;
        if (++h < a.Hkv) return;
        h = 0;
        do { ++b; user(a); } while (n_tiles == 0);
    }
};

template <bool QLO, int PASS>
__global__ void __launch_bounds__(kWwThreads, 1) weight_window_kernel(const __grid_constant__ WeightArgs a, int col0, int32_t* status) {
    extern __shared__ __align__(1024) unsigned char ww_smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int cols = a.Hq / a.Hkv * a.T;
    follow_me_early();
    after_predecessor();
    if (PASS == 2 && !a.accumulate && col0 == 0) {                       // zeros behind the lengths
        for (int64_t bh = blockIdx.x; bh < a.B * a.Hkv; bh += gridDim.x)
            for (int64_t s = ws_len(a, bh / a.Hkv) + tid; s < a.S; s += kWwThreads) a.sums[bh * a.S + s] = 0.f;
    }
    const int64_t all = (int64_t)a.tiles_before[a.B] * a.Hkv;    // this CTA's share: tiles x0 .. x1 - 1
    const int64_t sharers = ws_sharers(gridDim.x, all);
    if (blockIdx.x >= sharers) return;
    const int64_t x0 = blockIdx.x * all / sharers, x1 = (blockIdx.x + 1) * all / sharers;
    const int n_share = (int)(x1 - x0);
    WwPlace at;
    at.find(a, x0, lane);
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(ww_smem);
    float* norm_s = reinterpret_cast<float*>(ww_smem + kWwOffNorm);      // ring of four tiles' norms
    float* red_s = reinterpret_cast<float*>(ww_smem + kWwOffRed);
    const uint32_t bar_full = base + kWwOffBar, bar_empty = bar_full + 16, bar_s = bar_empty + 16, bar_free = bar_s + 16, tmem_at = bar_free + 16;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            ww_bar_init(bar_full + 8 * i, 8);
            ww_bar_init(bar_empty + 8 * i, 1);
            // The products of one part of a tile go on while the other's are taken out.  Pass 1: values, then signs, of all keys (128 keys per
            // instruction; 64 take longer by a third: 171 us for the call instead of 156, when this was measured).  Pass 2: both, of keys 0-63 and then of 64-127, since its
            // four columns' factors leave no registers to keep a tile's values until the signs are there.
            ww_bar_init(bar_s + 8 * i, 1);
            ww_bar_init(bar_free + 8 * i, PASS == 1 ? 8 : 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" :: "r"(tmem_at), "r"(kWwTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    ww_fence_before();
    __syncthreads();
    ww_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(tmem) : "r"(tmem_at));
    const uint32_t t_lane = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    const int half = (warp >> 2) & 1;                                    // which half of a column's keys, of a key's dims
    const int row = tid & 127;
    bool ok = true;

    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" :: "n"(kWwOtherRegs));
        // ---- products ---------------------------------------------------------------------------------------------------
        using Set = WwSet<QLO>;
        int span_end = 0;
        uint32_t tq = tmem + kWwColQ + Set::kNext;                       // this span's columns
        for (int t = 0; warp == 16 && ok && t < n_share; ++t) {
            if (t == span_end) {                                         // another head's columns
                tq = tmem + kWwColQ + (tq == tmem + kWwColQ ? Set::kNext : 0);
                span_end += at.n_tiles - at.tile;
                if (span_end < n_share) at.next_head(a);
            }
            const uint32_t kv = base + (t & 1) * kWwBuf;
            ok = ww_bar_wait(bar_full + 8 * (t & 1), (t >> 1) & 1);
            if constexpr (PASS == 1) {                                   // all keys, values and then signs
                if (ok && t > 0) ok = ww_bar_wait(bar_free, (t - 1) & 1);
                if (!ok) break;
                ww_fence_after();
                const bool one = ww_elect();
                if (one) {
                    // the remainders' products first: added to an accumulator that already holds the values', each would cost it a rounding
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) ww_mma(tmem + kWwColA, tq + 8 * ks, kv + kWwBytesV + ks * 2 * kWwLbo, kWwSbo, kWwTile, ks > 0);
                    if (QLO) {
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks) ww_mma(tmem + kWwColA, tq + Set::kQlo + 8 * ks, kv + ks * 2 * kWwLbo, kWwSbo, kWwTile, 1);
                    }
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) ww_mma(tmem + kWwColA, tq + 8 * ks, kv + ks * 2 * kWwLbo, kWwSbo, kWwTile, 1);
                    if (!a.with_qjl) ww_commit(bar_empty + 8 * (t & 1));
                    ww_commit(bar_s);
                }
                __syncwarp();
                if (!a.with_qjl) continue;
                if (t > 0) ok = ww_bar_wait(bar_free + 8, (t - 1) & 1);
                if (!ok) break;
                ww_fence_after();
                if (one) {
                    const uint32_t sx = kv + 2 * kWwBytesV;
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) ww_mma(tmem + kWwColB, tq + Set::kClo + 8 * ks, sx + ks * 2 * kWwLbo, kWwSboSign, kWwTile, ks > 0);
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) ww_mma(tmem + kWwColB, tq + Set::kChi + 8 * ks, sx + ks * 2 * kWwLbo, kWwSboSign, kWwTile, 1);
                    ww_commit(bar_empty + 8 * (t & 1));
                    ww_commit(bar_s + 8);
                }
                __syncwarp();
            }
#pragma unroll 1
            for (int x = PASS == 1 ? 2 : 0; ok && x < 2; ++x) {
                if (t > 0) ok = ww_bar_wait(bar_free + 8 * x, (t - 1) & 1);
                if (!ok) break;
                ww_fence_after();
                if (ww_elect()) {
                    const uint32_t kx = kv + x * 8 * kWwSbo, sx = kv + 2 * kWwBytesV + x * 8 * kWwSboSign, da = tmem + kWwColA + 64 * x, db = tmem + kWwColB + 64 * x;
                    // the remainders' products first: added to an accumulator that already holds the values', each would cost it a rounding
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) ww_mma(da, tq + 8 * ks, kx + kWwBytesV + ks * 2 * kWwLbo, kWwSbo, 64, ks > 0);
                    if (QLO) {
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks) ww_mma(da, tq + Set::kQlo + 8 * ks, kx + ks * 2 * kWwLbo, kWwSbo, 64, 1);
                    }
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) ww_mma(da, tq + 8 * ks, kx + ks * 2 * kWwLbo, kWwSbo, 64, 1);
                    if (a.with_qjl) {
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks) ww_mma(db, tq + Set::kClo + 8 * ks, sx + ks * 2 * kWwLbo, kWwSboSign, 64, ks > 0);
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks) ww_mma(db, tq + Set::kChi + 8 * ks, sx + ks * 2 * kWwLbo, kWwSboSign, 64, 1);
                    }
                    if (x == 1) ww_commit(bar_empty + 8 * (t & 1));
                    ww_commit(bar_s + 8 * x);
                }
                __syncwarp();
            }
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" :: "n"(kWwKeyRegs));
        // ---- dequantisation: 64 dims of key x and 32 of its signs per thread --------------------------------------------------
        const int x = row;
        const uint32_t lut_lane = base + kWwOffLut + 8 * (lane & 15);
        const uint32_t row_at = (uint32_t)(x >> 3) * kWwSbo + (uint32_t)(x & 7) * 16 + 8 * half * kWwLbo;
        const uint32_t sign_at = 2 * kWwBytesV + (uint32_t)(x >> 3) * kWwSboSign + (uint32_t)(x & 7) * 16 + 4 * half * kWwLbo;
        float norm_mul = 1.f;                                            // the sign product in units of the value product
        uint4 nib[2];
        uint32_t sign = 0;
        float norm = 0.f;
        auto fetch = [&]() {                                             // keys past the end repeat the last one
            const int k = at.tile * kWwTile + x;
            const int64_t r = ((int64_t)at.b * a.Hkv + at.h) * a.S + (k < at.len ? k : at.len - 1);
#pragma unroll
            for (int i = 0; i < 2; ++i) nib[i] = __ldg(reinterpret_cast<const uint4*>(a.k_nib + r * kNibBytes) + 2 * half + i);
            if (a.with_qjl) {
                sign = __ldg(reinterpret_cast<const uint32_t*>(a.k_qjl + r * kQjlBytes) + half);
                norm = __ldg(a.k_norms + r);
            }
        };
        fetch();
        bool new_table = true, new_span = true;
        uint32_t tq = t_lane + kWwColQ + WwSet<QLO>::kNext;
        for (int t = 0; t < n_share; ++t) {
            // the next tile's rows are requested first: their way from DRAM takes a third of a tile's time
            const bool table_now = new_table, span_now = new_span;
            const int h_now = at.h;
            const int64_t bh_now = (int64_t)at.b * a.Hkv + at.h;
            const uint4 nib_now[2] = {nib[0], nib[1]};
            const uint32_t sign_now = sign;
            const float norm_now = norm;
            if (t + 1 < n_share) {
                new_span = ++at.tile == at.n_tiles;
                if (new_span) at.next_head(a);
                new_table = a.cb_per_head && at.h != h_now;
                fetch();
            }
            if (table_now) {                                             // no lookup of the previous table is still to come
                asm volatile("bar.sync 2, 256;\n" ::: "memory");
                norm_mul = kQjlCoef / kWwProjMul * ws_build_lut<16>(ww_smem + kWwOffLut, a.codebooks + (a.cb_per_head ? h_now * 16 : 0), tid - 256);
                asm volatile("bar.sync 2, 256;\n" ::: "memory");
            }
            if (ok && t > 1) ok = ww_bar_wait(bar_empty + 8 * (t & 1), ((t >> 1) - 1) & 1);
            // (a warp whose wait ran out stays for the barriers of the others and leaves behind the loop)
            if (span_now) {
                // Q' of another head's columns into tensor memory, half of each part per thread: it comes with the span's first tile.  Two
                // sets: that wait was for the second tile back, so no product reads the set of the span before the last one any more.
                tq = t_lane + kWwColQ + (tq == t_lane + kWwColQ ? WwSet<QLO>::kNext : 0);
                if (QLO && ok && t > 0) ok = ww_bar_wait(bar_empty + 8 * ((t - 1) & 1), ((t - 1) >> 1) & 1);
                if (ok) {
                    ww_fence_after();
                    const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned char*>(a.prepared) + (bh_now * ((cols + kWwTile - 1) / kWwTile) + col0 / kWwTile) * kWwPrepBytes) + row;
                    const bool col_on = col0 + row < cols;
                    // four pieces at a time: 64 values, their remainders, 32 values of G . q, their remainders (the warp has 72 registers)
#pragma unroll 1
                    for (int part = 0; part < 6; ++part) {
                        const bool of_q = part < 4;
                        if (of_q ? !QLO && part > 1 : !a.with_qjl) continue;
                        const uint4* from = src + (size_t)(of_q ? 16 * (part >> 1) + 8 * half + 4 * (part & 1) : 32 + 8 * (part - 4) + 4 * half) * kWwTile;
                        uint32_t v[16];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint4 x4 = col_on ? from[i * kWwTile] : make_uint4(0u, 0u, 0u, 0u);
                            v[4 * i] = x4.x; v[4 * i + 1] = x4.y; v[4 * i + 2] = x4.z; v[4 * i + 3] = x4.w;
                        }
                        ww_st16(tq + (of_q ? WwSet<QLO>::kQlo * (part >> 1) + 32 * half + 16 * (part & 1)
                                           : (part == 4 ? WwSet<QLO>::kChi : WwSet<QLO>::kClo) + 16 * half), v);
                    }
                    ww_wait_st();
                    ww_fence_before();
                }
            }
            const uint32_t kv = base + (t & 1) * kWwBuf;
#pragma unroll
            for (int i = 0; i < 2; ++i) {                                // sixteen lookups, then their eight stores
                const uint32_t w[4] = {nib_now[i].x, nib_now[i].y, nib_now[i].z, nib_now[i].w};
                uint2 v[4][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[j][k] = ww_lut(lut_lane, w[j], k);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    ww_sts16(kv + row_at + (uint32_t)(4 * i + j) * kWwLbo, v[j][0].x, v[j][1].x, v[j][2].x, v[j][3].x);
                    ww_sts16(kv + kWwBytesV + row_at + (uint32_t)(4 * i + j) * kWwLbo, v[j][0].y, v[j][1].y, v[j][2].y, v[j][3].y);
                }
            }
            if (a.with_qjl) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t bits = sign_now >> (8 * i);
                    ww_sts16(kv + sign_at + (uint32_t)i * kWwLbo, ws_signs2(bits), ws_signs2(bits >> 2), ws_signs2(bits >> 4), ws_signs2(bits >> 6));
                }
            }
            if (half == 0) norm_s[(t & 3) * kWwTile + x] = norm_now * norm_mul;
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) ww_bar_arrive(bar_full + 8 * (t & 1));
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" :: "n"(kWwScoreRegs));
        // ---- scores: 64 keys of a tile per thread -----------------------------------------------------------------------------
        const int col = col0 + row;
        const bool col_on = col < cols;
        int done = 0;                                                    // tiles behind this one
        while (done < n_share) {
            const int64_t bh = (int64_t)at.b * a.Hkv + at.h;
            const int len = at.len;
            const int n_span = at.n_tiles - at.tile < n_share - done ? at.n_tiles - at.tile : n_share - done;
            float* sums = a.sums + bh * a.S;
            const unsigned char* prep = reinterpret_cast<const unsigned char*>(a.prepared) + (bh * ((cols + kWwTile - 1) / kWwTile) + col0 / kWwTile) * kWwPrepBytes;
            const float f = col_on ? reinterpret_cast<const float*>(prep + (size_t)kWwPrepRows * kWwTile * 16)[row] : 1.f;
            const int last = col_on ? (a.causal ? len - a.T + col % a.T : len - 1) : -1;    // newest key of the column
            const int open_to = a.causal ? len - a.T : len - 1;          // newest key that every column sees
            float m = -INFINITY, l = 0.f, top_all = 0.f, inv = 0.f;          // pass 2: the column's maximum and reciprocal sum
            if (PASS == 2 && col_on) {
                // the head's spans: the CTAs whose shares hold its first and its last tile, and those between
                const int64_t first = ((int64_t)a.tiles_before[at.b]) * a.Hkv + (int64_t)at.h * at.n_tiles;
                const int64_t c0 = ws_cta_of(first, gridDim.x, all), c1 = ws_cta_of(first + at.n_tiles - 1, gridDim.x, all);
                const float2* p = a.partial + (bh + c0) * cols + col;
                for (int64_t i = 0; i <= c1 - c0; i += 4) {              // seldom more than three
                    float2 e[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) e[k] = i + k <= c1 - c0 ? p[(i + k) * cols] : make_float2(-INFINITY, 0.f);
                    const float top = fmaxf(fmaxf(fmaxf(m, e[0].x), fmaxf(e[1].x, e[2].x)), e[3].x), ref = top == -INFINITY ? 0.f : top;
                    l *= exp2f(m - ref);
#pragma unroll
                    for (int k = 0; k < 4; ++k) l += e[k].y * exp2f(e[k].x - ref);
                    m = top;
                }
                top_all = m == -INFINITY ? INFINITY : m;                  // no open key, or given up in pass 1: every weight is zero
                inv = m == -INFINITY && l == 0.f ? 0.f : 1.f / l;
            }
            // pass 2: a thread has four columns, rows lane / 4 + 8 r of its warp's 32
            uint64_t f4[PASS == 2 ? 4 : 1], top4[PASS == 2 ? 4 : 1], inv4[PASS == 2 ? 4 : 1];
            int last4[PASS == 2 ? 4 : 1];
            if constexpr (PASS == 2) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int from = 8 * r + (lane >> 2);
                    const float fr = __shfl_sync(kFullMask, f, from), tr = -__shfl_sync(kFullMask, top_all, from), ir = __shfl_sync(kFullMask, inv, from);
                    f4[r] = ww_pack2(fr, fr); top4[r] = ww_pack2(tr, tr); inv4[r] = ww_pack2(ir, ir);
                    last4[r] = __shfl_sync(kFullMask, last, from);
                }
            }
            for (int t = done; t < done + n_span; ++t) {
                // after a wait that ran out the warp still goes through the barriers it shares with the others; its columns add nothing
                if (ok) ok = ww_bar_wait(bar_s + (PASS == 1 ? 0 : 8 * half), t & 1);
                ww_fence_after();
                const int k0 = (at.tile + t - done) * kWwTile;
                const bool masked = k0 + kWwTile - 1 > open_to || k0 + kWwTile > len || cols - col0 < kWwTile;
                if constexpr (PASS == 2) {
                    // keys 8 i + 2 (lane % 4) and the next one of the half's 64: weights summed over the thread's four columns
                    uint64_t sum[8];
                    const float* nrm = norm_s + (t & 3) * kWwTile + 64 * half + 2 * (lane & 3);
#pragma unroll
                    for (int rb = 0; rb < 2; ++rb) {
                        const uint32_t at16 = t_lane + ((uint32_t)(16 * rb) << 16) + 64 * half;
                        uint32_t s[32], v[32];                           // products of the values, then the scores / f; of the signs
                        ww_ld16x64(at16 + kWwColA, s);
                        if (a.with_qjl) ww_ld16x64(at16 + kWwColB, v);
                        ww_wait_ld();
                        if (rb == 1) {
                            ww_fence_before();
                            __syncwarp();
                            if (lane == 0) ww_bar_arrive(bar_free + 8 * half);   // the accumulators may be overwritten
                        }
                        if (a.with_qjl) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float2 n2 = *reinterpret_cast<const float2*>(nrm + 8 * i);
#pragma unroll
                                for (int r = 0; r < 4; r += 2) {
                                    const float2 y = ww_unpack2(ww_fma2(ww_pack2(__uint_as_float(v[4 * i + r]), __uint_as_float(v[4 * i + r + 1])), ww_pack2(n2.x, n2.y),
                                                                        ww_pack2(__uint_as_float(s[4 * i + r]), __uint_as_float(s[4 * i + r + 1]))));
                                    s[4 * i + r] = __float_as_uint(y.x);
                                    s[4 * i + r + 1] = __float_as_uint(y.y);
                                }
                            }
                        }
                        uint64_t n2[2] = {inv4[2 * rb], inv4[2 * rb + 1]};
                        if (masked) {
                            const int l0 = (last4[2 * rb] < len - 1 ? last4[2 * rb] : len - 1) - k0 - 64 * half - 2 * (lane & 3);
                            const int l1 = (last4[2 * rb + 1] < len - 1 ? last4[2 * rb + 1] : len - 1) - k0 - 64 * half - 2 * (lane & 3);
                            // a NaN column's normaliser goes into the scores that it sees: a masked key's zero times it would be NaN
                            const float z0 = ww_unpack2(n2[0]).x, z1 = ww_unpack2(n2[1]).x;
                            n2[0] = z0 == z0 ? n2[0] : 0;
                            n2[1] = z1 == z1 ? n2[1] : 0;
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                s[i] = 8 * (i >> 2) + (i & 1) <= ((i & 2) ? l1 : l0) ? __float_as_uint(__uint_as_float(s[i]) + ((i & 2) ? z1 - z1 : z0 - z0)) : 0xff800000u;
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const float2 e = ww_unpack2(ww_fma2(ww_pack2(__uint_as_float(s[4 * i + 2 * r]), __uint_as_float(s[4 * i + 2 * r + 1])), f4[2 * rb + r], top4[2 * rb + r]));
                                sum[i] = ww_fma2(ww_pack2(ws_ex2(e.x), ws_ex2(e.y)), n2[r], rb + r ? sum[i] : ww_pack2(0.f, 0.f));
                            }
                        }
                    }
                    // and over the eight lanes with other columns: they trade halves of their keys until each has the totals of two
#pragma unroll
                    for (int n = 4, x = 16; n >= 1; n >>= 1, x >>= 1) {
                        const bool up = (lane & x) != 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (i < n) {
                                const float2 mine = ww_unpack2(up ? sum[i + n] : sum[i]), other = ww_unpack2(up ? sum[i] : sum[i + n]);
                                sum[i] = ww_pack2(mine.x + __shfl_xor_sync(kFullMask, other.x, x), mine.y + __shfl_xor_sync(kFullMask, other.y, x));
                            }
                        }
                    }
                    // two of [four warps of a half][128 keys], so one barrier per tile; the halves do not wait for one another
                    float* red = red_s + (t & 1) * 4 * kWwTile + 64 * half;
                    *reinterpret_cast<float2*>(red + (warp & 3) * kWwTile + 2 * lane) = ok ? ww_unpack2(sum[0]) : make_float2(0.f, 0.f);
                    asm volatile("bar.sync %0, 128;\n" :: "r"(3 + half) : "memory");
                    if (row < 64) {
                        const float total = (red[row] + red[kWwTile + row]) + (red[2 * kWwTile + row] + red[3 * kWwTile + row]);
                        const int key = k0 + 64 * half + row;
                        if (key < len) {
                            if (a.accumulate || col0 > 0) sums[key] += total;
                            else sums[key] = total;
                        }
                    }
                    continue;
                }
                uint32_t s[64];                                          // products of the values, then the scores / f
                ww_ld32(t_lane + kWwColA + 64 * half, s);
                ww_ld32(t_lane + kWwColA + 64 * half + 32, s + 32);
                ww_wait_ld();
                ww_fence_before();
                __syncwarp();
                if (lane == 0) ww_bar_arrive(bar_free);                  // the accumulator may be overwritten
                if (a.with_qjl) {
                    if (ok) ok = ww_bar_wait(bar_s + 8, t & 1);
                    ww_fence_after();
                    const float* nrm = norm_s + (t & 3) * kWwTile + 64 * half;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint32_t v[32];                                  // products of the signs
                        ww_ld32(t_lane + kWwColB + 64 * half + 32 * j, v);
                        ww_wait_ld();
                        if (j == 1) {
                            ww_fence_before();
                            __syncwarp();
                            if (lane == 0) ww_bar_arrive(bar_free + 8);
                        }
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 n4 = *reinterpret_cast<const float4*>(nrm + 32 * j + i);
#pragma unroll
                            for (int k = 0; k < 4; k += 2) {
                                uint32_t* d = s + 32 * j + i + k;
                                const float2 r = ww_unpack2(ww_fma2(ww_pack2(__uint_as_float(v[i + k]), __uint_as_float(v[i + k + 1])),
                                                                    k ? ww_pack2(n4.z, n4.w) : ww_pack2(n4.x, n4.y),
                                                                    ww_pack2(__uint_as_float(d[0]), __uint_as_float(d[1]))));
                                d[0] = __float_as_uint(r.x);
                                d[1] = __float_as_uint(r.y);
                            }
                        }
                    }
                }
                if (masked) {
                    const int lim = (last < len - 1 ? last : len - 1) - k0 - 64 * half;
#pragma unroll
                    for (int i = 0; i < 64; ++i) s[i] = i <= lim ? s[i] : 0xff800000u;
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 64; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(s[i]));
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                const float m_new = fmaxf(m, top * f);
                const float ref = m_new == -INFINITY ? 0.f : m_new;
                const uint64_t f2 = ww_pack2(f, f), r2 = ww_pack2(-ref, -ref);
                uint64_t sum[2] = {ww_pack2(0.f, 0.f), ww_pack2(0.f, 0.f)};
#pragma unroll
                for (int i = 0; i < 64; i += 2) {
                    const float2 e = ww_unpack2(ww_fma2(ww_pack2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), f2, r2));
                    sum[(i >> 1) & 1] = ww_add2(sum[(i >> 1) & 1], ww_pack2(ws_ex2(e.x), ws_ex2(e.y)));
                }
                const float2 total = ww_unpack2(ww_add2(sum[0], sum[1]));
                l = fmaf(l, ws_ex2(m - ref), total.x + total.y);
                m = m_new;
            }
            if (PASS == 1) {                                             // the column's halves
                float2* hand = reinterpret_cast<float2*>(red_s);
                if (!ok) { m = -INFINITY; l = 0.f; }                     // given up: a state that pass 2 ignores, not what the memory held
                if (half == 1) hand[row] = make_float2(m, l);
                asm volatile("bar.sync 1, 256;\n" ::: "memory");
                if (half == 0 && col_on) {
                    const float2 o = hand[row];
                    const float top = fmaxf(m, o.x), ref = top == -INFINITY ? 0.f : top;
                    a.partial[(bh + blockIdx.x) * cols + col] = make_float2(top, l * ws_ex2(m - ref) + o.y * ws_ex2(o.x - ref));
                }
                asm volatile("bar.sync 1, 256;\n" ::: "memory");
            }
            done += n_span;
            if (done < n_share) at.next_head(a);
        }
    }
    if (!ok && status) atomicExch(status, OMNI_STATUS_WAIT_EXPIRED);
    __syncwarp();
    ww_fence_before();
    __syncthreads();
    if (warp == 16) {
        ww_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" :: "r"(tmem), "r"(kWwTmemCols) : "memory");
    }
}

// The CTAs of a call: one per SM, or one per tile where there are fewer
static int64_t ww_ctas(int64_t heads, int64_t S) {
    const int64_t tiles = heads * ((S + kWwTile - 1) / kWwTile);
    return tiles < 148 ? tiles : 148;
}

size_t weight_window_workspace(int64_t B, int Hq, int Hkv, int T, int64_t S) {
    const int64_t heads = B * Hkv, cols = (int64_t)(Hq / Hkv) * T, col_tiles = (cols + kWwTile - 1) / kWwTile;
    return (size_t)(heads * col_tiles) * kWwPrepBytes + ws_before_bytes(B) + (size_t)(heads + ww_ctas(heads, S)) * cols * sizeof(float2);
}

template <bool QLO>
static int32_t launch_weight_window_t(const WeightArgs& a, unsigned grid, int32_t* status, cudaStream_t st) {
    const int cols = a.Hq / a.Hkv * a.T;
    OMNI_ALLOW_SMEM((weight_window_kernel<QLO, 1>), kWwSmem);
    OMNI_ALLOW_SMEM((weight_window_kernel<QLO, 2>), kWwSmem);
    for (int pass = 1; pass <= 2; ++pass) {
        for (int col0 = 0; col0 < cols; col0 += kWwTile) {
            if (pass == 1) OMNI_CUDA(launch_early(weight_window_kernel<QLO, 1>, dim3(grid), kWwThreads, kWwSmem, st, a, col0, status));
            else OMNI_CUDA(launch_early(weight_window_kernel<QLO, 2>, dim3(grid), kWwThreads, kWwSmem, st, a, col0, status));
        }
    }
    return OMNI_OK;
}

int32_t launch_weight_window(WeightArgs a, int q_dtype, int32_t* status, cudaStream_t st) {
    const int64_t heads = a.B * a.Hkv, cols = (int64_t)(a.Hq / a.Hkv) * a.T, col_groups = (cols + kWpWarps * kWpCols - 1) / (kWpWarps * kWpCols);
    const int64_t ctas = ww_ctas(heads, a.S);
    OMNI_REQUIRE(heads * col_groups < 0x7fffffffLL && a.B * ((a.S + kWwTile - 1) / kWwTile) <= 0x7fffffffLL, OMNI_ERR_UNSUPPORTED, "omni_attn_weight_sums: too many keys");
    unsigned char* ws = reinterpret_cast<unsigned char*>(a.partial);     // prepared columns, tiles in front of every user, the spans' partial states
    a.prepared = ws;
    ws += (size_t)(heads * ((cols + kWwTile - 1) / kWwTile)) * kWwPrepBytes;
    a.tiles_before = reinterpret_cast<int32_t*>(ws);
    a.partial = reinterpret_cast<float2*>(ws + ws_before_bytes(a.B));
    const unsigned grid = (unsigned)(heads * col_groups) + 1;
    const bool qlo = q_dtype == OMNI_F32 || a.rotate_q;                  // a query of a 16-bit type, not rotated, is exact in its fp16 values
    switch (q_dtype) {
        case OMNI_F32:  weight_prepare_kernel<OMNI_F32, true><<<grid, kWpWarps * 32, 0, st>>>(a, col_groups); break;
        case OMNI_BF16: if (qlo) weight_prepare_kernel<OMNI_BF16, true><<<grid, kWpWarps * 32, 0, st>>>(a, col_groups);
                        else weight_prepare_kernel<OMNI_BF16, false><<<grid, kWpWarps * 32, 0, st>>>(a, col_groups);
                        break;
        default:        if (qlo) weight_prepare_kernel<OMNI_F16, true><<<grid, kWpWarps * 32, 0, st>>>(a, col_groups);
                        else weight_prepare_kernel<OMNI_F16, false><<<grid, kWpWarps * 32, 0, st>>>(a, col_groups);
    }
    OMNI_CUDA(cudaGetLastError());
    return qlo ? launch_weight_window_t<true>(a, (unsigned)ctas, status, st) : launch_weight_window_t<false>(a, (unsigned)ctas, status, st);
}

}  // namespace omni

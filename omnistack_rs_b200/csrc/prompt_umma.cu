// Attention of whole prompts over themselves on the fifth-generation tensor cores, bf16 and fp16.
//
// One CTA takes two tiles of 128 rows (row = token and query head of one kv head's group) and walks over the keys of their
// prompt in blocks of 128:   S_t = Q_t K^T  ->  P_t = exp2(c S_t - m)  ->  O_t += P_t V     (t = 0, 1;  c = scale * log2 e)
// Q, K and V tiles come by TMA (128-byte swizzle); S, P and O live in tensor memory (512 columns: S0 S1 O0 O1, each P in the
// columns of its S, which the softmax threads have read by then).  Roles: warps 0-3 and 4-7 are the softmax of tile 0 and 1,
// thread = row; warp 8 issues every product; warp 9 every copy; warp 10 finds the work; warp 11 clears rows of no prompt.  While the
// softmax of one tile runs, the products of the other do.
//
// A pair of tiles of one head group is a work item, one per launched CTA.  A CTA that runs takes over items of CTAs that are not yet
// placed (cluster launch control), so the items are handed out as SMs become free, and the copies and first products of the next item
// run under the last softmax and the output of this one.
//
// A block's maximum only replaces the running one when it exceeds it by 2^slack, so O is rescaled rarely; the softmax threads
// do it themselves: S_t of a block is issued behind P_t V of the block before, so its arrival says that O_t is complete.
//
// What bounds it: the chain of one tile, scores (512 cycles) - softmax (about 1,900) - product (512), two tiles deep, and on long prompts
// the board's power: 16,384 tokens of 32 heads in fp16 take 1.82 to 1.99 ms on different boards, 1,100 to 1,210 TFLOP/s at about 1.62 GHz
// under the 1,000 W cap, 68 to 74 % of the measured burst rate of a plain matrix product and 79 to 86 % of its sustained one.  A quarter of the
// exponentials as a polynomial on the FP32 units (1.84 ms against 1.80 on one board) or a third (1.90 ms) gained nothing.
//
// The tensor pipe takes both operands in 16 bits, so weights are rounded to the type (their sum is not): relative to 64 bits a ragged bf16
// batch is off by 2.1e-3 and 16,384 fp16 tokens by 2.7e-4, of which 1.6e-3 and 2.1e-4 are the rounding of the result alone.
//
// A zero weight times an infinite or NaN value of a masked key is NaN.  Rows that come out NaN although no score of theirs is, in dims
// that the values they see do not account for (prompt_unexplained), are formed again from global memory over their own keys alone.
#include "prompt.cuh"
#include <cuda.h>
#include <mutex>

namespace omni {

constexpr int kPuThreads = 384;
// Registers: 384 threads are launched with 168 each (64,512); the softmax warpgroups go up to 224, the third down to 56
// (256 * 224 + 128 * 56 = 64,512).
constexpr int kPuSoftmaxRegs = 224, kPuOtherRegs = 56;
constexpr int kPuStages = 5;                       // ring of K and V tiles, 32 KiB each, in the order K0 V0 K1 V1 ...
constexpr uint32_t kPuTile = 128 * 128 * 2;        // bytes of a 128-row tile: two halves of 64 dims, 128 bytes a row
constexpr uint32_t kPuHalf = kPuTile / 2;
constexpr uint32_t kPuOffK = 2 * kPuTile;
constexpr uint32_t kPuOffBar = kPuOffK + kPuStages * kPuTile;
constexpr int kPuItems = 2;                        // ring of work items
constexpr int kPuCu = 256;                         // prompt bounds kept in shared memory (more are read from global memory)
constexpr uint32_t kPuOffCu = kPuOffBar + 256;
constexpr uint32_t kPuOffItem = kPuOffCu + kPuCu * 4;           // item: batch, first row, length, first token, kv head, first query head, valid
constexpr uint32_t kPuSmem = kPuOffItem + kPuItems * 32 + 16 + 1024;   // items, a stolen CTA's handle, and room to start on a 1,024-byte boundary
constexpr uint32_t kPuColS = 0, kPuColO = 256, kPuTmemCols = 512;
// A poll that fails lasts 4 us, so a wait runs out after 4 s (and one for the next item after 16 s: it outlasts the waits of the warp that
// publishes it).  Waits last as long as a CTA's item does; rows formed again over a million keys take a tenth of a second.
constexpr uint32_t kPuWaitLimit = 1u << 20, kPuItemWaitLimit = 1u << 22;
constexpr float kPuLog2e = 1.4426950408889634f;
// Past 2^22 a step of fp32 is half a power of two or more.  The roundings of the reference, of its bias and of the slack's comparison add up to a
// whole power there, and an fp16 weight of 2^(8 + 7) would not hold twice that.  Rows that get there are formed again (prompt_rows_again
// subtracts before it adds a bias); a second form of the loop below that does so costs every call 2 %.
constexpr float kPuFar = 4194304.f;

// ---- PTX wrappers --------------------------------------------------------------------------------
__device__ __forceinline__ void pu_bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" :: "r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void pu_bar_arrive(uint32_t bar) {
    asm volatile("{\n .reg .b64 t;\n mbarrier.arrive.shared::cta.b64 t, [%0];\n}\n" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void pu_bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("{\n .reg .b64 t;\n mbarrier.arrive.expect_tx.shared::cta.b64 t, [%0], %1;\n}\n" :: "r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool pu_bar_wait(uint32_t bar, uint32_t parity, uint32_t limit = kPuWaitLimit) {
    for (uint32_t i = 0; i < limit; ++i) {
        uint32_t ok;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
    }
    return false;
}
// by all lanes of a warp, with one answer
__device__ __forceinline__ bool pu_bar_wait_warp(uint32_t bar, uint32_t parity, uint32_t limit = kPuWaitLimit) {
    return __all_sync(kFullMask, pu_bar_wait(bar, parity, limit));
}
__device__ __forceinline__ void pu_tma_load(uint32_t dst, const CUtensorMap* map, int d, int t, int h, int b, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n"
                 :: "r"(dst), "l"(map), "r"(d), "r"(t), "r"(h), "r"(b), "r"(bar) : "memory");
}
__device__ __forceinline__ void pu_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void pu_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void pu_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void pu_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void pu_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" :: "r"(bar) : "memory");
}
__device__ __forceinline__ bool pu_elect() {
    uint32_t is;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(is));
    return is != 0;
}
// Shared-memory matrix descriptors, 128-byte swizzle.  Low word: start address (>> 4) and, for an MN-major operand, the distance
// (>> 4) between its runs of 64 elements along MN.  High word: 1,024 bytes between groups of eight rows, version, swizzle mode.
constexpr uint32_t kPuDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t pu_desc(uint32_t saddr, uint32_t lbo) { return (saddr >> 4) | ((lbo >> 4) << 16); }
// D[tmem] (+)= A[smem] B[smem]
__device__ __forceinline__ void pu_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n .reg .b64 x, y;\n setp.ne.b32 p, %4, 0;\n mov.b64 x, {%1, %5};\n mov.b64 y, {%2, %5};\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n"
                 :: "r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kPuDescHi) : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void pu_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n .reg .b64 y;\n setp.ne.b32 p, %4, 0;\n mov.b64 y, {%2, %5};\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}\n"
                 :: "r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kPuDescHi) : "memory");
}
__device__ __forceinline__ void pu_ld32(uint32_t taddr, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                   "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
                   "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
                   "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void pu_st32(uint32_t taddr, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n"
                 :: "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                    "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
                    "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
                    "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
                 : "memory");
}
template <int DT>
__device__ __forceinline__ constexpr uint32_t pu_idesc(bool b_mn_major) {
    return (1u << 4) | (DT == OMNI_BF16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn_major ? (1u << 16) : 0u) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ float pu_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void pu_store32(void* p, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" :: "l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7]) : "memory");
}
// two fp32 operations in one instruction, on register pairs
__device__ __forceinline__ uint64_t pu_pair(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 pu_parts(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t pu_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t pu_add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float pu_max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
template <int DT> __device__ __forceinline__ uint32_t pu_pack(float lo, float hi) {
    uint32_t r;
    if constexpr (DT == OMNI_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// D += A B of one warp: 16 rows x 16 x 8 columns
template <int DT>
__device__ __forceinline__ void pu_warp_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (DT == OMNI_BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <int DT> __device__ __forceinline__ float2 pu_unpack(uint32_t w) {
    if constexpr (DT == OMNI_BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Output rows of one kv head over their own keys alone, by a warp.  Lane l brings a row: token t of query head `head`, keys 0 .. lim, wanted
// where bit l of `again` is set.  Sixteen rows at a time: lane (g, c) = (lane / 4, lane % 4) holds dims 32 c .. 32 c + 31 of rows g and g + 8.
// Keys that all wanted rows see go through warp-level products, sixteen at a time, with the weights rounded to the type as everywhere; the
// others, fewer than 16 + 127, one by one, skipped where they are masked.
// 4,096 tokens of 8 heads, 64 us: 385 us with a NaN value at token 2,000 in a tile of earlier rows (21 ms with a row and a key at a time).
template <int DT>
__device__ __forceinline__ void prompt_rows_again(const PromptArgs& a, int64_t b, int64_t row0, int hkv, int t, int lim, int head, uint32_t again, int lane) {
    constexpr float kBias = DT == OMNI_F16 ? 14.f : 0.f;                 // fp16 weights end at 2^-24
    constexpr float kLeast = DT == OMNI_F16 ? 5.9604644775390625e-8f : 1.17549435e-38f;        // a visible infinity times a weight is not NaN
    using E = typename Elem<DT>::T;
    const int g = lane >> 2, c = lane & 3;
    const E* kp = reinterpret_cast<const E*>(a.k) + b * a.ks[0] + (int64_t)hkv * a.ks[1] + row0 * a.ks[2];
    const E* vp = reinterpret_cast<const E*>(a.v) + b * a.vs[0] + (int64_t)hkv * a.vs[1] + row0 * a.vs[2];
    const float scale = a.scale * kPuLog2e;
    auto load8w = [](const E* p, uint32_t* w) {                          // eight elements
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
        w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
    };
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += 16) {
        const uint32_t wanted = (again >> r0) & 0xffffu;
        if (!wanted) continue;
        const bool mine = (lane & 16) == r0 && ((again >> lane) & 1);
        const int n_common = __reduce_min_sync(kFullMask, mine ? lim : 0x7ffffffe) + 1, last = __reduce_max_sync(kFullMask, mine ? lim : -1);
        bool on[2];
        int64_t out_at[2];
        int lims[2];
        uint32_t q[2][16];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int from = r0 + g + 8 * r;
            const int tr = __shfl_sync(kFullMask, t, from), hr = __shfl_sync(kFullMask, head, from);
            lims[r] = __shfl_sync(kFullMask, lim, from);
            on[r] = (again >> from) & 1;
            out_at[r] = ((b * a.Hq + hr) * a.T + row0 + tr) * kHeadDim + 32 * c;
#pragma unroll
            for (int i = 0; i < 16; ++i) q[r][i] = 0u;
            if (on[r]) {
                const E* qp = reinterpret_cast<const E*>(a.q) + b * a.qs[0] + (int64_t)hr * a.qs[1] + (row0 + tr) * a.qs[2] + 32 * c;
#pragma unroll
                for (int i = 0; i < 4; ++i) load8w(qp + 8 * i, q[r] + 4 * i);
            }
        }
        float o[16][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};        // o[i]: dims 32 c + i and 32 c + 16 + i of row g, then of row g + 8
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        auto raise = [&](int r, float top) {                             // the row's new reference
            const float m_new = fmaxf(m[r], top), alpha = exp2f(m[r] - (m_new == -INFINITY ? 0.f : m_new));
            m[r] = m_new;
            l[r] *= alpha;
#pragma unroll
            for (int i = 0; i < 16; ++i) { o[i][2 * r] *= alpha; o[i][2 * r + 1] *= alpha; }
        };
        int j0 = 0;
#pragma unroll 1
        for (; j0 + 16 <= n_common; j0 += 16) {
            uint32_t k[2][16], v[4][8];                                  // keys g and g + 8, this lane's dims; keys 2c, 2c + 1, 2c + 8, 2c + 9, dims 16 g ..
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int x = 0; x < 4; ++x) load8w(kp + (int64_t)(j0 + g + 8 * i) * a.ks[2] + 32 * c + 8 * x, k[i] + 4 * x);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int x = 0; x < 2; ++x) load8w(vp + (int64_t)(j0 + 2 * c + (i & 1) + 8 * (i >> 1)) * a.vs[2] + 16 * g + 8 * x, v[i] + 4 * x);
            }
            float s[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) pu_warp_mma<DT>(s[i], q[0][2 * ks], q[1][2 * ks], q[0][2 * ks + 1], q[1][2 * ks + 1], k[i][2 * ks], k[i][2 * ks + 1]);
            }
            uint32_t p[2][2];                                            // [row][keys 2c and 2c + 1, then 2c + 8 and 2c + 9]
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float x[4] = {s[0][2 * r] * scale, s[0][2 * r + 1] * scale, s[1][2 * r] * scale, s[1][2 * r + 1] * scale};
                float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 1));
                top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 2));
                if (__any_sync(kFullMask, top > m[r])) raise(r, top);
                const float ref = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool seen = x[i] > -INFINITY;
                    x[i] = exp2f(x[i] - ref + kBias);
                    l[r] += x[i];
                    if (seen) x[i] = fmaxf(x[i], kLeast);
                }
                p[r][0] = pu_pack<DT>(x[0], x[1]);
                p[r][1] = pu_pack<DT>(x[2], x[3]);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t half = (i & 1) ? 0x7632u : 0x5410u;
                pu_warp_mma<DT>(o[i], p[0][0], p[1][0], p[0][1], p[1][1], __byte_perm(v[0][i >> 1], v[1][i >> 1], half), __byte_perm(v[2][i >> 1], v[3][i >> 1], half));
            }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(kFullMask, l[r], 1);
            l[r] += __shfl_xor_sync(kFullMask, l[r], 2);
        }
#pragma unroll 1
        for (; j0 <= last; ++j0) {
            uint32_t k[16], v[16];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                load8w(kp + (int64_t)j0 * a.ks[2] + 32 * c + 8 * x, k + 4 * x);
                load8w(vp + (int64_t)j0 * a.vs[2] + 32 * c + 8 * x, v + 4 * x);
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 x = pu_unpack<DT>(q[r][i]), y = pu_unpack<DT>(k[i]);
                    s = fmaf(x.x, y.x, fmaf(x.y, y.y, s));
                }
                s += __shfl_xor_sync(kFullMask, s, 1);
                s += __shfl_xor_sync(kFullMask, s, 2);
                s = j0 <= lims[r] ? s * scale : -INFINITY;
                if (__any_sync(kFullMask, s > m[r])) raise(r, s);
                const float e = exp2f(s - (m[r] == -INFINITY ? 0.f : m[r]) + kBias);
                l[r] += e;
                if (j0 <= lims[r]) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 y = pu_unpack<DT>(v[i]);            // dims 32 c + 2 i, + 1
                        float& u = o[(2 * i) & 15][2 * r + (i >> 3)];
                        float& w = o[(2 * i + 1) & 15][2 * r + (i >> 3)];
                        u = fmaf(e, y.x, u);
                        w = fmaf(e, y.y, w);
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if (!on[r]) continue;
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                float y[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) y[x] = o[(i + x) & 15][2 * r + (i >> 4)] / l[r];
                Elem<DT>::store4(a.out, out_at[r] + i, y);
            }
        }
    }
}

// Of the rows `again` (one per lane) whose sums over the values came out NaN in the dims `dims` (bit i of word w: dim 32 w + i), those that
// the values 0 .. first, which all of them see, do not account for: a NaN there, or infinities of both signs, whatever the weights.
template <int DT>
__device__ __forceinline__ uint32_t prompt_unexplained(const PromptArgs& a, int64_t b, int64_t row0, int hkv, int first, uint32_t again,
                                                       const uint32_t (&dims)[4], int lane) {
    constexpr uint32_t kExp = DT == OMNI_BF16 ? 0x7f807f80u : 0x7c007c00u, kOne = DT == OMNI_BF16 ? 0x00800080u : 0x04000400u;
    using E = typename Elem<DT>::T;
    const int half = lane >> 4, d = lane & 15;                           // dims 8 d .. 8 d + 7 of every other key
    const E* vp = reinterpret_cast<const E*>(a.v) + b * a.vs[0] + (int64_t)hkv * a.vs[1] + row0 * a.vs[2] + 8 * d;
    uint32_t is_nan = 0, up = 0, down = 0;                               // bit i: dim 8 d + i
#pragma unroll 1
    for (int j0 = 0; j0 <= first && again; j0 += 32) {
        uint4 v[16];
        uint32_t hit = 0;                                                // an exponent of ones carries into its sign's place
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = __ldg(reinterpret_cast<const uint4*>(vp + (int64_t)(j0 + 2 * i + half < first ? j0 + 2 * i + half : first) * a.vs[2]));
#pragma unroll
        for (int i = 0; i < 16; ++i) hit |= ((v[i].x & kExp) + kOne) | ((v[i].y & kExp) + kOne) | ((v[i].z & kExp) + kOne) | ((v[i].w & kExp) + kOne);
        if (!__any_sync(kFullMask, (hit & 0x80008000u) != 0)) continue;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float2 y = pu_unpack<DT>(w[x]);
                is_nan |= (y.x != y.x ? 1u << (2 * x) : 0u) | (y.y != y.y ? 2u << (2 * x) : 0u);
                up |= (y.x == INFINITY ? 1u << (2 * x) : 0u) | (y.y == INFINITY ? 2u << (2 * x) : 0u);
                down |= (y.x == -INFINITY ? 1u << (2 * x) : 0u) | (y.y == -INFINITY ? 2u << (2 * x) : 0u);
            }
        }
        is_nan |= __shfl_xor_sync(kFullMask, is_nan, 16);                // the other keys
        up |= __shfl_xor_sync(kFullMask, up, 16);
        down |= __shfl_xor_sync(kFullMask, down, 16);
        const uint32_t known = (is_nan | (up & down)) << (8 * (lane & 3));
        uint32_t left = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) left |= dims[w] & ~__reduce_or_sync(kFullMask, d >> 2 == w ? known : 0u);
        again &= __ballot_sync(kFullMask, left != 0);
    }
    return again;
}

// Zeros in a row whose work is given up.
template <int DT>
__device__ __forceinline__ void prompt_leave_row(const PromptArgs& a, int64_t b, int64_t row, int head, int at, int step) {
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = at; i < kHeadDim / 4; i += step) Elem<DT>::store4(a.out, ((b * a.Hq + head) * a.T + row) * kHeadDim + 4 * i, zero);
}

// A work item: two tiles (32-bit: a prompt's rows and a call's slots are).
struct PuItem {
    int b, row0, len, t0, hkv, head0, slot;
    int n[2];                                      // key blocks of each tile (0: no rows)
    __device__ __forceinline__ void blocks(const PromptArgs& a, int tt) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int first = t0 + x * tt, last = first + tt - 1 < len ? first + tt - 1 : len - 1;
            n[x] = first >= len ? 0 : ((a.causal ? last + 1 : len) + 127) / 128;
        }
    }
    __device__ __forceinline__ int all() const { return n[0] > n[1] ? n[0] : n[1]; }
};

template <int DT>
__global__ void __launch_bounds__(kPuThreads, 1)
prompt_umma_kernel(const __grid_constant__ PromptArgs a, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v) {
    extern __shared__ unsigned char pu_smem[];
    // fp16 weights carry 2^bias: the type ends at 2^-24, and weights far below the row's largest would lose their bits there
    constexpr float kBias = DT == OMNI_F16 ? 8.f : 0.f, kSlack = DT == OMNI_F16 ? 7.f : 8.f;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int tt = a.tpt / 2;                                            // tokens of one tile

    const uint32_t base = ((uint32_t)__cvta_generic_to_shared(pu_smem) + 1023u) & ~1023u;
    const uint32_t sQ = base, sKV = base + kPuOffK, bars = base + kPuOffBar;
    const uint32_t bar_q = bars, bar_full = bars + 16, bar_empty = bar_full + 8 * kPuStages, bar_s = bar_empty + 8 * kPuStages, bar_p = bar_s + 16,
                   bar_h = bar_p + 16, bar_o = bar_h + 16, bar_qe = bar_o + 16, bar_item = bar_qe + 16, bar_taken = bar_item + 8 * kPuItems,
                   bar_steal = bar_taken + 8 * kPuItems, bar_want = bar_steal + 8, tmem_at = bar_want + 8;
    const uint32_t items = base + kPuOffItem, handle = items + kPuItems * 32;
    if (tid == 0) {
        for (int x = 0; x < 2; ++x) {
            pu_bar_init(bar_q + 8 * x, 1);
            pu_bar_init(bar_s + 8 * x, 1);
            pu_bar_init(bar_p + 8 * x, 4);
            pu_bar_init(bar_h + 8 * x, 4);
            pu_bar_init(bar_o + 8 * x, 1);
            pu_bar_init(bar_qe + 8 * x, 1);
        }
        for (int i = 0; i < kPuItems; ++i) {
            pu_bar_init(bar_item + 8 * i, 1);
            pu_bar_init(bar_taken + 8 * i, 11);                          // every warp but the one that finds the work
        }
        pu_bar_init(bar_steal, 1);
        pu_bar_init(bar_want, 1);
        for (int i = 0; i < kPuStages; ++i) {
            pu_bar_init(bar_full + 8 * i, 1);
            pu_bar_init(bar_empty + 8 * i, 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" :: "r"(tmem_at), "r"(kPuTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    pu_fence_before();
    __syncthreads();
    pu_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(tmem) : "r"(tmem_at));
    bool ok = true;                                                      // false once a bounded wait has run out

    // the k-th item of this CTA, by a warp; false when there is none (or a wait ran out)
    PuItem it;
    auto next_item = [&](int k) {
        const int at = k % kPuItems;
        ok = pu_bar_wait_warp(bar_item + 8 * at, (k / kPuItems) & 1, kPuItemWaitLimit);
        if (!ok) return false;
        uint32_t v[7];
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(items + 32 * at) : "memory");
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%3+16];\n ld.shared.u32 %2, [%3+24];\n" : "=r"(v[4]), "=r"(v[5]), "=r"(v[6]) : "r"(items + 32 * at) : "memory");
        __syncwarp();
        if (lane == 0) pu_bar_arrive(bar_taken + 8 * at);
        it.b = (int)v[0]; it.row0 = (int)v[1]; it.len = (int)v[2]; it.t0 = (int)v[3]; it.hkv = (int)v[4]; it.head0 = (int)v[5]; it.slot = (int)v[6];
        it.blocks(a, tt);
        return it.slot >= 0;
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" :: "n"(kPuOtherRegs));
        if (warp == 10) {
            // ---- work: this CTA's own item, then those of CTAs that have not been placed ---------------------------------
            uint32_t bx = blockIdx.x, by = blockIdx.y, valid = 1;
            PromptArgs near = a;                                         // the same, with the bounds at hand
            if (a.cu && a.n_seqs < kPuCu) {
                int32_t* cu = reinterpret_cast<int32_t*>(pu_smem + (base - (uint32_t)__cvta_generic_to_shared(pu_smem)) + kPuOffCu);
                for (int i = lane; i <= a.n_seqs; i += 32) cu[i] = __ldg(a.cu + i);
                __syncwarp();
                near.cu = cu;
            }
            for (int k = 0;; ++k) {
                const int at = k % kPuItems;
                if (k >= kPuItems) ok = pu_bar_wait_warp(bar_taken + 8 * at, (k / kPuItems - 1) & 1);
                const int64_t slot = (int64_t)gridDim.x - 1 - bx;        // a prompt's last tiles have the most keys: first
                PromptTile w{};
                if (valid) w = prompt_tile(near, slot, lane);
                const uint32_t hkv = by / a.n_hg, head0 = hkv * (uint32_t)(a.Hq / a.Hkv) + by % a.n_hg * a.gp;
                if (!ok) {                                               // an item that no other CTA will take up: zeros
                    if (valid) {
                        prompt_zero_rows<DT>(a, w, slot, (int)head0, lane, 32);
                        for (int r = 0; r < a.tpt * a.gp; ++r)
                            if (w.t0 + r % a.tpt < w.len)
                                prompt_leave_row<DT>(a, w.b, w.row0 + w.t0 + r % a.tpt, (int)head0 + r / a.tpt, lane, 32);
                    }
                    break;
                }
                if (lane == 0) {
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};\n" :: "r"(items + 32 * at), "r"((uint32_t)w.b), "r"((uint32_t)w.row0), "r"(w.len), "r"(w.t0) : "memory");
                    asm volatile("st.shared.v2.u32 [%0+16], {%1,%2};\n st.shared.u32 [%0+24], %3;\n" :: "r"(items + 32 * at), "r"(hkv), "r"(head0),
                                 "r"(valid ? (uint32_t)slot : 0xffffffffu) : "memory");
                    pu_bar_arrive(bar_item + 8 * at);
                }
                __syncwarp();
                if (!valid) break;
                // the next item is taken when the copies of this one have been issued, no sooner: what a busy CTA holds, an idle one cannot get
                ok = pu_bar_wait_warp(bar_want, k & 1);
                if (!ok) break;
                if (lane == 0) {
                    pu_bar_expect(bar_steal, 16);
                    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];\n" :: "r"(handle), "r"(bar_steal) : "memory");
                }
                ok = pu_bar_wait_warp(bar_steal, k & 1);
                if (!ok) break;
                asm volatile("{\n .reg .pred p;\n .reg .b128 h;\n ld.shared.b128 h, [%3];\n clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n"
                             " selp.u32 %0, 1, 0, p;\n mov.u32 %1, 0;\n mov.u32 %2, 0;\n"
                             " @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n @p clusterlaunchcontrol.query_cancel.get_first_ctaid::y.b32.b128 %2, h;\n}\n"
                             : "=r"(valid), "=r"(bx), "=r"(by) : "r"(handle) : "memory");
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");       // the handle has been read before the next one is written
                __syncwarp();
            }
        } else if (warp == 11) {
            for (int k = 0; next_item(k); ++k) {
                PromptTile w;
                w.b = it.b; w.row0 = it.row0; w.len = it.len; w.t0 = it.t0;
                prompt_zero_rows<DT>(a, w, it.slot, it.head0, lane, 32);
            }
        } else if (warp == 9) {
            // ---- copies -----------------------------------------------------------------------------------------------
            const uint32_t q_bytes = (uint32_t)(tt * a.gp) * 256u;
            int i = 0;                                                   // tiles of the ring so far
            int used[2] = {0, 0};                                        // items so far whose first, second tile had rows
            for (int k = 0; next_item(k); ++k) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    if (!ok || it.n[x] == 0) continue;
                    // the products of the previous item have read the tile's queries
                    if (used[x] > 0) ok = pu_bar_wait_warp(bar_qe + 8 * x, (used[x] - 1) & 1);
                    if (!ok) continue;
                    ++used[x];
                    if (lane == 0) {
                        pu_bar_expect(bar_q + 8 * x, q_bytes);
                        for (int h = 0; h < 2; ++h)
                            pu_tma_load(sQ + x * kPuTile + h * kPuHalf, &map_q, 64 * h, it.row0 + it.t0 + x * tt, it.head0, it.b, bar_q + 8 * x);
                    }
                }
                const int n_tiles = 2 * it.all();                        // K and V in turn
                for (int n = 0; ok && n < n_tiles; ++n, ++i) {
                    const int st = i % kPuStages, round = i / kPuStages;
                    if (round > 0) ok = pu_bar_wait_warp(bar_empty + 8 * st, (round - 1) & 1);
                    if (!ok) break;
                    if (lane == 0) {
                        const uint32_t dst = sKV + st * kPuTile, bar = bar_full + 8 * st;
                        pu_bar_expect(bar, kPuTile);
                        const CUtensorMap* map = (n & 1) ? &map_v : &map_k;
                        for (int h = 0; h < 2; ++h) pu_tma_load(dst + h * kPuHalf, map, 64 * h, it.row0 + 128 * (n >> 1), it.hkv, it.b, bar);
                    }
                    __syncwarp();
                }
                if (!ok) break;
                if (lane == 0) pu_bar_arrive(bar_want);
            }
            // no copy may still be under way when the CTA ends (they all are complete unless a wait ran out)
            if (!ok) {
                for (int k = i < kPuStages ? 0 : i - kPuStages; k < i; ++k) pu_bar_wait(bar_full + 8 * (k % kPuStages), (k / kPuStages) & 1);
                for (int x = 0; x < 2; ++x)
                    if (used[x] > 0) pu_bar_wait(bar_q + 8 * x, (used[x] - 1) & 1);
            }
        } else {
            // ---- products: the whole warp waits, one thread issues ----------------------------------------------------------
            auto issue_s = [&](int x, uint32_t sK, bool last) {
                if (pu_elect()) {
                    const uint32_t da = pu_desc(sQ + x * kPuTile, 16), db = pu_desc(sK, 16);
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        const uint32_t off = ((ks >> 2) * kPuHalf + (ks & 3) * 32) >> 4;
                        pu_mma_ss(tmem + kPuColS + 128 * x, da + off, db + off, pu_idesc<DT>(false), ks > 0);
                    }
                    pu_commit(bar_s + 8 * x);
                    if (last) pu_commit(bar_qe + 8 * x);
                }
                __syncwarp();
            };
            int st = 0;                                                  // ring stage of the next tile, and the parity of its round
            uint32_t ph = 0;
            uint32_t done[2] = {0u, 0u}, used[2] = {0u, 0u};             // per tile: blocks and items so far (their parities are the barriers')
            for (int k = 0; next_item(k); ++k) {
                const int n_all = it.all();
                if (n_all == 0) continue;
                int stk = st;                                            // stage of K_j
                ok = pu_bar_wait_warp(bar_full + 8 * st, ph);
                if (++st == kPuStages) { st = 0; ph ^= 1u; }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    if (!ok || it.n[x] == 0) continue;
                    ok = pu_bar_wait_warp(bar_q + 8 * x, used[x] & 1);
                    if (!ok) continue;
                    ++used[x];
                    pu_fence_after();
                    issue_s(x, sKV + stk * kPuTile, it.n[x] == 1);
                }
                if (ok && pu_elect()) pu_commit(bar_empty + 8 * stk);
                __syncwarp();
                for (int j = 0; ok && j < n_all; ++j) {
                    const int stv = st;                                  // V_j
                    ok = pu_bar_wait_warp(bar_full + 8 * st, ph);
                    if (++st == kPuStages) { st = 0; ph ^= 1u; }
                    const bool more = j + 1 < n_all;
                    if (more) {                                          // K_{j+1}
                        stk = st;
                        if (ok) ok = pu_bar_wait_warp(bar_full + 8 * st, ph);
                        if (++st == kPuStages) { st = 0; ph ^= 1u; }
                    }
                    const uint32_t sV = sKV + stv * kPuTile, sK = sKV + stk * kPuTile;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (!ok || j >= it.n[x]) continue;
                        // the weights come in halves: the product over keys 0-63 runs while the softmax works on the rest
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            if (ok) ok = pu_bar_wait_warp((half ? bar_p : bar_h) + 8 * x, done[x] & 1);
                            if (!ok) break;
                            pu_fence_after();
                            if (pu_elect()) {
                                const uint32_t db = pu_desc(sV, kPuHalf), dd = tmem + kPuColO + 128 * x, da = tmem + kPuColS + 128 * x;
#pragma unroll
                                for (int ks = 4 * half; ks < 4 * half + 4; ++ks)
                                    pu_mma_ts(dd, da + 8 * ks, db + ks * (2048 >> 4), pu_idesc<DT>(true), (j > 0 || ks > 0) ? 1u : 0u);
                                if (half == 1 && j + 1 >= it.n[x]) pu_commit(bar_o + 8 * x);
                            }
                            __syncwarp();
                        }
                        if (!ok) continue;
                        ++done[x];
                        if (j + 1 < it.n[x]) issue_s(x, sK, j + 2 >= it.n[x]);
                    }
                    if (ok && pu_elect()) {
                        pu_commit(bar_empty + 8 * stv);
                        if (more) pu_commit(bar_empty + 8 * stk);
                    }
                    __syncwarp();
                }
                if (!ok) break;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" :: "n"(kPuSoftmaxRegs));
        // ---- softmax of tile x, thread = row ------------------------------------------------------------------------
        const int x = warp >> 2, row = tid & 127;
        const uint32_t t_lane = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const uint32_t t_s = t_lane + kPuColS + 128 * x, t_o = t_lane + kPuColO + 128 * x;
        const int g = row / tt, t_in = row % tt;
        const float c = a.scale * kPuLog2e;
        uint32_t done = 0, used = 0;                                     // blocks and items of this tile so far
        bool left = false;                                               // a wait ran out in the middle of an item
        int k = 0;
        for (; next_item(k); ++k) {
            const int n_mine = x ? it.n[1] : it.n[0];
            if (n_mine == 0) continue;
            const int t = it.t0 + x * tt + t_in;
            const bool live = g < a.gp && t < it.len;
            // newest key of the row; rows without a query go through the motions on whatever their operands hold
            const int lim = live ? (a.causal ? t : it.len - 1) : it.len - 1;
            const int n_free = a.causal ? it.t0 + x * tt + 1 : it.len;       // keys below this are open to every row of the tile
            float m = -INFINITY, l = 0.f;                                    // m: in units of c * score
            bool far = false;                                                // m has been past kPuFar
            for (int j = 0; j < n_mine; ++j) {
                ok = pu_bar_wait_warp(bar_s + 8 * x, done & 1);
                if (!ok) break;
                pu_fence_after();
                uint32_t s[128];
#pragma unroll
                for (int i = 0; i < 4; ++i) pu_ld32(t_s + 32 * i, s + 32 * i);
                pu_wait_ld();
                if (128 * j + 128 > n_free) {
                    const int open = lim - 128 * j;                          // columns 0 .. open of the block are seen
#pragma unroll
                    for (int i = 0; i < 128; ++i) s[i] = i <= open ? s[i] : 0xff800000u;
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 128; i += 8) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) mx[k] = pu_max3(mx[k], __uint_as_float(s[i + 2 * k]), __uint_as_float(s[i + 2 * k + 1]));
                }
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
                const bool raise = top > m + kSlack;                         // never while every score so far is -inf
                if (__any_sync(kFullMask, raise)) {
                    const float m_new = raise ? top : m;
                    const float alpha = raise ? pu_ex2(m - m_new) : 1.f;
                    m = m_new;
                    far = far || (raise && fabsf(m) > kPuFar);
                    l *= alpha;
                    if (j > 0) {
#pragma unroll 1
                        for (int i = 0; i < 4; ++i) {
                            uint32_t o[32];
                            pu_ld32(t_o + 32 * i, o);
                            pu_wait_ld();
#pragma unroll
                            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                            pu_st32(t_o + 32 * i, o);
                        }
                    }
                }
                const float shift = kBias - (m == -INFINITY ? 0.f : m);      // scores of -inf then weigh zero
                const uint64_t c2 = pu_pair(c, c), neg2 = pu_pair(shift, shift);
                uint64_t sum[2] = {pu_pair(0.f, 0.f), pu_pair(0.f, 0.f)};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t p[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float2 v = pu_parts(pu_fma2(pu_pair(__uint_as_float(s[64 * h + 2 * i]), __uint_as_float(s[64 * h + 2 * i + 1])), c2, neg2));
                        const float2 e = make_float2(pu_ex2(v.x), pu_ex2(v.y));
                        sum[i & 1] = pu_add2(sum[i & 1], pu_pair(e.x, e.y));
                        p[i] = pu_pack<DT>(e.x, e.y);
                    }
                    pu_st32(t_s + 32 * h, p);
                    pu_wait_st();
                    pu_fence_before();
                    __syncwarp();
                    if (lane == 0) pu_bar_arrive((h ? bar_p : bar_h) + 8 * x);
                }
                const float2 both = pu_parts(pu_add2(sum[0], sum[1]));
                l += both.x + both.y;
                ++done;
            }
            // ---- result rows ---------------------------------------------------------------------------------------------
            if (ok) ok = pu_bar_wait_warp(bar_o + 8 * x, used & 1);
            ++used;
            if (!ok) { left = true; break; }
            pu_fence_after();
            const float inv = 1.f / l;
            uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) +
                                                  (((int64_t)it.b * a.Hq + it.head0 + (live ? g : 0)) * a.T + it.row0 + (live ? t : it.t0)) * kHeadDim);
            bool bad = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t o[32];
                pu_ld32(t_o + 32 * i, o);
                pu_wait_ld();
                uint32_t r[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const float u = __uint_as_float(o[2 * k]) * inv, v = __uint_as_float(o[2 * k + 1]) * inv;
                    bad = bad || u != u || v != v;
                    r[k] = pu_pack<DT>(u, v);
                }
                if (live) {                                              // a thread's row, whole 32-byte sectors at a time
                    pu_store32(dst + 4 * i, r);
                    pu_store32(dst + 4 * i + 2, r + 8);
                }
            }
            // A sum l that is NaN comes from the row's own scores (masked ones are -inf before their use), one of zero from scores that are
            // all -inf: such rows are NaN, and done.  What is left has NaN among its values, visible or masked.
            far = far && live && m < INFINITY;                               // (an infinite score makes its row NaN)
            uint32_t again = __ballot_sync(kFullMask, live && bad && !far && l > 0.f);
            if (again) {
                uint32_t dims[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t o[32];
                    pu_ld32(t_o + 32 * i, o);
                    pu_wait_ld();
                    dims[i] = 0;
#pragma unroll
                    for (int k = 0; k < 32; ++k) dims[i] |= __uint_as_float(o[k]) != __uint_as_float(o[k]) ? 1u << k : 0u;
                }
                const int first = __reduce_min_sync(kFullMask, (again >> lane) & 1 ? lim : 0x7fffffff);
                again = prompt_unexplained<DT>(a, it.b, it.row0, it.hkv, first, again, dims, lane);
            }
            again |= __ballot_sync(kFullMask, far);
            if (again) prompt_rows_again<DT>(a, it.b, it.row0, it.hkv, t, lim, it.head0 + g, again, lane);
        }
        if (left) {                                                      // zeros for its rows and those of the items still to come
            do {
                const int t = it.t0 + x * tt + t_in;
                if (g < a.gp && t < it.len) prompt_leave_row<DT>(a, it.b, (int64_t)it.row0 + t, it.head0 + g, 0, 1);
            } while (next_item(++k));
            ok = false;
        }
    }
    if (!ok && a.status) atomicExch(a.status, OMNI_STATUS_WAIT_EXPIRED);
    __syncwarp();
    pu_fence_before();
    __syncthreads();
    if (warp == 8) {
        pu_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" :: "r"(tmem), "r"(kPuTmemCols) : "memory");
    }
}

// ---- host side ---------------------------------------------------------------------------------------------
typedef CUresult (*PuEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static PuEncodeFn pu_encode_fn() {
    static std::mutex mu;
    static PuEncodeFn fn = nullptr;
    std::lock_guard<std::mutex> lk(mu);
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult res;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &res) == cudaSuccess && res == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PuEncodeFn>(p);
    }
    return fn;
}

// view (dims, tokens, heads, users) of 16-bit rows, boxes of 64 dims x `tokens` x `heads`
static int32_t pu_map(CUtensorMap* map, const void* base, int dtype, const int64_t* strides, int64_t T, int64_t H, int64_t B, int tokens, int heads) {
    PuEncodeFn fn = pu_encode_fn();
    OMNI_REQUIRE(fn != nullptr, OMNI_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[4] = {(cuuint64_t)kHeadDim, (cuuint64_t)T, (cuuint64_t)H, (cuuint64_t)B};
    cuuint64_t st[3];
    const int64_t by[3] = {strides[2], strides[1], strides[0]}, n[3] = {T, H, B};
    for (int i = 0; i < 3; ++i) {
        st[i] = n[i] > 1 ? (cuuint64_t)(2 * by[i]) : (cuuint64_t)(2 * kHeadDim);          // an extent of one is never stepped over
        OMNI_REQUIRE(st[i] > 0 && st[i] % 16 == 0 && st[i] < (1ull << 40), OMNI_ERR_UNSUPPORTED, "omni_prompt_attn: stride of %lld elements", (long long)by[i]);
    }
    const cuuint32_t box[4] = {64u, (cuuint32_t)tokens, (cuuint32_t)heads, 1u}, one[4] = {1u, 1u, 1u, 1u};
    const CUresult r = fn(map, dtype == OMNI_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, st,
                          box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    OMNI_REQUIRE(r == CUDA_SUCCESS, OMNI_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return OMNI_OK;
}

template <int DT>
static int32_t launch_prompt_umma_t(const PromptArgs& a, cudaStream_t st) {
    CUtensorMap mq, mk, mv;
    int32_t rc = pu_map(&mq, a.q, DT, a.qs, a.T, a.Hq, a.B, a.tpt / 2, a.gp);
    if (rc == OMNI_OK) rc = pu_map(&mk, a.k, DT, a.ks, a.T, a.Hkv, a.B, 128, 1);
    if (rc == OMNI_OK) rc = pu_map(&mv, a.v, DT, a.vs, a.T, a.Hkv, a.B, 128, 1);
    if (rc != OMNI_OK) return rc;
    OMNI_ALLOW_SMEM((prompt_umma_kernel<DT>), kPuSmem);
    prompt_umma_kernel<DT><<<dim3((unsigned)a.slots, (unsigned)(a.Hkv * a.n_hg)), kPuThreads, kPuSmem, st>>>(a, mq, mk, mv);
    return check_cuda(cudaGetLastError(), "prompt_umma_kernel launch");
}

int32_t launch_prompt_umma(PromptArgs a, int dtype, cudaStream_t st) {
    a.tpt = 2 * (128 / a.gp);
    a.slots = a.cu ? a.T / a.tpt + a.n_seqs : a.B * ((a.T + a.tpt - 1) / a.tpt);
    OMNI_REQUIRE(a.slots <= 0x7fffffffLL && (int64_t)a.Hkv * a.n_hg <= 65535, OMNI_ERR_UNSUPPORTED, "omni_prompt_attn: too many tiles");
    return dtype == OMNI_BF16 ? launch_prompt_umma_t<OMNI_BF16>(a, st) : launch_prompt_umma_t<OMNI_F16>(a, st);
}

}  // namespace omni

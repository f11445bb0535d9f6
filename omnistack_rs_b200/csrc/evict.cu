// Eviction from the packed cache: which keys of a (user, head) stay, and their rows gathered into a smaller cache.
//
// Selection.  Keys ordered by (sum descending, position ascending); the budget - recent first of the positions below
// len - recent stay, and the `recent` last positions.  One CTA per (user, head): the sums become order-preserving 32-bit
// numbers, four histogram passes of eight bits find the value of the last one that stays, a scan over the positions emits
// the kept ones in order.
//
// Gather.  A warp moves a group of eight kept rows.  Rows are moved, never recomputed, so the new cache holds the same bits;
// V's pair layout mixes the nibbles of two keys per row, which the lanes take apart for the old pairs and join for the new.
#include "common.cuh"

namespace omni {

constexpr int kSelThreads = 1024;

// ascending unsigned order = ascending sum; +0 = -0, NaN above everything
__device__ __forceinline__ uint32_t sum_key(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ int clamp_len(const int32_t* seq_lens, int64_t b, int64_t S) {
    if (!seq_lens) return (int)S;
    const int64_t n = __ldg(seq_lens + b);
    return (int)(n < 0 ? 0 : (n > S ? S : n));
}

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const __grid_constant__ omni_evict_t a) {
    __shared__ uint32_t hist[256];
    __shared__ uint32_t s_value, s_need;
    __shared__ int warp_cnt[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t bh = blockIdx.x, b = bh / a.H;
    const int len = clamp_len(a.seq_lens, b, a.S);
    const int budget = (int)a.budget, recent = (int)a.recent;
    int32_t* index = a.index + bh * a.budget;
    if (bh % a.H == 0 && tid == 0) a.new_lens[b] = len < budget ? len : budget;
    if (len <= budget) {
        for (int i = tid; i < budget; i += kSelThreads) index[i] = i < len ? i : -1;
        return;
    }
    const float* sums = a.sums + bh * a.S;
    const int n = len - recent;                                  // candidates; budget - recent of them stay (fewer than n)
    if (tid == 0) { s_value = 0; s_need = (uint32_t)(budget - recent); }
    uint32_t known = 0;                                          // mask of the bits of the threshold found so far
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        const uint32_t value = s_value;
        for (int i = tid; i < n; i += kSelThreads) {
            const uint32_t key = sum_key(sums[i]);
            if ((key & known) == value) atomicAdd(&hist[(key >> shift) & 255], 1u);
        }
        __syncthreads();
        if (warp == 0) {                                         // the digit in which the running count from above reaches the need
            const uint32_t need = s_need;
            uint32_t c[8], mine = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) { c[k] = hist[255 - (8 * lane + k)]; mine += c[k]; }
            uint32_t upto = mine;
#pragma unroll
            for (int x = 1; x < 32; x <<= 1) {
                const uint32_t o = __shfl_up_sync(kFullMask, upto, x);
                if (lane >= x) upto += o;
            }
            uint32_t before = upto - mine;
            const bool here = need > 0 ? (before < need && upto >= need) : lane == 0;
            if (here) {
                uint32_t digit = 255 - 8 * lane;
                if (need > 0) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        if (before < need && before + c[k] >= need) { digit = 255 - (8 * lane + k); s_need = need - before; }
                        before += c[k];
                    }
                }
                s_value = value | (digit << shift);
            }
        }
        known |= 255u << shift;
        __syncthreads();
    }
    const uint32_t value = s_value;
    const int ties = (int)s_need;                                // this many of the keys equal to the threshold stay, lowest first
    int kept = 0, tied = 0;                                      // of the chunks so far
    for (int i0 = 0; i0 < len; i0 += kSelThreads) {
        const int i = i0 + tid;
        const bool last = i >= n && i < len;
        const uint32_t key = i < n ? sum_key(sums[i]) : 0;
        const bool above = i < n && budget > recent && key > value;
        const bool tie = i < n && budget > recent && key == value;
        const uint32_t tie_ballot = __ballot_sync(kFullMask, tie);
        // positions of the ties first, then of the kept keys
        if (lane == 0) warp_cnt[warp] = __popc(tie_ballot);
        __syncthreads();
        int v = lane < 32 ? warp_cnt[lane] : 0;
        int scan = v;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const int o = __shfl_up_sync(kFullMask, scan, x);
            if (lane >= x) scan += o;
        }
        const int tie_total = __shfl_sync(kFullMask, scan, 31);
        const int tie_base = __shfl_sync(kFullMask, scan - v, warp);
        const int tie_rank = tied + tie_base + __popc(tie_ballot & ((1u << lane) - 1u));
        const bool keep = last || above || (tie && tie_rank < ties);
        const uint32_t keep_ballot = __ballot_sync(kFullMask, keep);
        __syncthreads();
        if (lane == 0) warp_cnt[warp] = __popc(keep_ballot);
        __syncthreads();
        v = warp_cnt[lane];
        scan = v;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const int o = __shfl_up_sync(kFullMask, scan, x);
            if (lane >= x) scan += o;
        }
        const int keep_total = __shfl_sync(kFullMask, scan, 31);
        const int keep_base = __shfl_sync(kFullMask, scan - v, warp);
        const int at = kept + keep_base + __popc(keep_ballot & ((1u << lane) - 1u));
        if (keep && at < budget) index[at] = i;
        kept += keep_total;
        tied += tie_total;
        __syncthreads();
    }
}

constexpr int kGatherWarps = 8;

__global__ void __launch_bounds__(kGatherWarps * 32) evict_gather_kernel(const __grid_constant__ omni_evict_t a, int64_t groups_per_head, int64_t n_groups) {
    const int lane = threadIdx.x & 31;
    const int64_t g = (int64_t)blockIdx.x * kGatherWarps + (threadIdx.x >> 5);
    if (g >= n_groups) return;
    const int64_t bh = g / groups_per_head, b = bh / a.H;
    const int64_t row0 = (g % groups_per_head) * 8;              // first kept row of the group
    const int len = clamp_len(a.seq_lens, b, a.S);
    const int64_t new_len = len < a.budget ? len : a.budget;
    const int64_t src0 = bh * a.S, dst0 = bh * a.capacity;
    // old position of row r of the group in lane r (-1: no key)
    int from = -1;
    if (lane < 8 && row0 + lane < new_len) from = __ldg(a.index + bh * a.budget + row0 + lane);
    {   // K nibbles: four lanes per row
        const int r = lane >> 2, c = lane & 3;
        const int p = __shfl_sync(kFullMask, from, r);
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (p >= 0) v = __ldg(reinterpret_cast<const uint4*>(a.k_nib + (src0 + p) * kNibBytes) + c);
        if (row0 + r < a.capacity) *(reinterpret_cast<uint4*>(a.k_nib_out + (dst0 + row0 + r) * kNibBytes) + c) = v;
    }
    if (lane < 8 && row0 + lane < a.capacity) {
        const int64_t s = src0 + from, d = dst0 + row0 + lane;
        const uint2 none = make_uint2(0u, 0u);
        *reinterpret_cast<uint2*>(a.k_qjl_out + d * kQjlBytes) = from >= 0 ? __ldg(reinterpret_cast<const uint2*>(a.k_qjl + s * kQjlBytes)) : none;
        a.k_norms_out[d] = from >= 0 ? __ldg(a.k_norms + s) : 0.f;
        a.sums_out[d] = from >= 0 ? __ldg(a.sums + s) : 0.f;
        if (a.v_qjl) {
            *reinterpret_cast<uint2*>(a.v_qjl_out + d * kQjlBytes) = from >= 0 ? __ldg(reinterpret_cast<const uint2*>(a.v_qjl + s * kQjlBytes)) : none;
            a.v_norms_out[d] = from >= 0 ? __ldg(a.v_norms + s) : 0.f;
        }
    }
    {   // V nibbles: a lane has eight bytes of the rows of a pair (first, first ^ 3)
        const int pair = lane >> 3, c = lane & 7;
        const int r1 = pair < 2 ? pair : pair + 2, r2 = r1 ^ 3;
        const int whole_old = a.v_paired ? (len & ~7) : 0;
        uint2 row[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int p = __shfl_sync(kFullMask, from, x ? r2 : r1);
            row[x] = make_uint2(0u, 0u);
            if (p < 0) continue;
            const uint2 mine = __ldg(reinterpret_cast<const uint2*>(a.v_nib + (src0 + p) * kNibBytes) + c);
            if (p < whole_old) {
                // the key's own nibbles: low halves of both rows for a pair's first key, high halves for its second
                const uint2 other = __ldg(reinterpret_cast<const uint2*>(a.v_nib + (src0 + (p ^ 3)) * kNibBytes) + c);
                if (p & 2) {
                    row[x].x = ((other.x >> 4) & 0x0f0f0f0fu) | (mine.x & 0xf0f0f0f0u);
                    row[x].y = ((other.y >> 4) & 0x0f0f0f0fu) | (mine.y & 0xf0f0f0f0u);
                } else {
                    row[x].x = (mine.x & 0x0f0f0f0fu) | ((other.x << 4) & 0xf0f0f0f0u);
                    row[x].y = (mine.y & 0x0f0f0f0fu) | ((other.y << 4) & 0xf0f0f0f0u);
                }
            } else {
                row[x] = mine;
            }
        }
        if (a.v_paired && row0 + 8 <= new_len) {                 // a whole group: into the pair layout
            const uint2 p = row[0], q = row[1];
            row[0].x = (p.x & 0x0f0f0f0fu) | ((q.x << 4) & 0xf0f0f0f0u);
            row[0].y = (p.y & 0x0f0f0f0fu) | ((q.y << 4) & 0xf0f0f0f0u);
            row[1].x = ((p.x >> 4) & 0x0f0f0f0fu) | (q.x & 0xf0f0f0f0u);
            row[1].y = ((p.y >> 4) & 0x0f0f0f0fu) | (q.y & 0xf0f0f0f0u);
        }
        if (row0 + r1 < a.capacity) *(reinterpret_cast<uint2*>(a.v_nib_out + (dst0 + row0 + r1) * kNibBytes) + c) = row[0];
        if (row0 + r2 < a.capacity) *(reinterpret_cast<uint2*>(a.v_nib_out + (dst0 + row0 + r2) * kNibBytes) + c) = row[1];
    }
}

}  // namespace omni

using namespace omni;

extern "C" int32_t omni_evict_keys(const omni_evict_t* call, void* stream) {
    OMNI_REQUIRE(call != nullptr, OMNI_ERR_ARG, "omni_evict_keys: NULL call");
    const omni_evict_t& a = *call;
    OMNI_REQUIRE(a.B >= 0 && a.H >= 0 && a.S >= 0, OMNI_ERR_ARG, "omni_evict_keys: negative extent");
    OMNI_REQUIRE(a.budget >= 1 && a.recent >= 0 && a.recent <= a.budget && a.capacity >= a.budget, OMNI_ERR_ARG,
                 "omni_evict_keys: need 0 <= recent <= budget <= capacity and budget >= 1");
    OMNI_REQUIRE(a.S <= 0x7fffff00LL && a.budget <= 0x7fffff00LL && a.B * a.H <= 0x7fffffffLL, OMNI_ERR_UNSUPPORTED, "omni_evict_keys: extent past 2^31");
    if (a.B == 0 || a.H == 0) return OMNI_OK;
    OMNI_REQUIRE((a.S == 0 || (a.sums && a.k_nib && a.k_qjl && a.k_norms && a.v_nib)) && a.sums_out && a.k_nib_out && a.k_qjl_out && a.k_norms_out &&
                 a.v_nib_out && a.index && a.new_lens, OMNI_ERR_ARG, "omni_evict_keys: NULL buffer");
    OMNI_REQUIRE((a.v_qjl == nullptr) == (a.v_norms == nullptr) && (!a.v_qjl || (a.v_qjl_out && a.v_norms_out)), OMNI_ERR_ARG,
                 "omni_evict_keys: v_qjl and v_norms must both be given or both be NULL");
    OMNI_REQUIRE((((uintptr_t)a.k_nib | (uintptr_t)a.v_nib | (uintptr_t)a.k_nib_out | (uintptr_t)a.v_nib_out) & 15) == 0 &&
                 (((uintptr_t)a.k_qjl | (uintptr_t)a.v_qjl | (uintptr_t)a.k_qjl_out | (uintptr_t)a.v_qjl_out) & 7) == 0, OMNI_ERR_ARG,
                 "omni_evict_keys: misaligned buffer");
    const int64_t groups_per_head = (a.capacity + 7) / 8, n_groups = a.B * a.H * groups_per_head;
    OMNI_REQUIRE((n_groups + kGatherWarps - 1) / kGatherWarps <= 0x7fffffffLL, OMNI_ERR_UNSUPPORTED, "omni_evict_keys: too many rows");
    cudaStream_t st = (cudaStream_t)stream;
    evict_select_kernel<<<(unsigned)(a.B * a.H), kSelThreads, 0, st>>>(a);
    OMNI_CUDA(cudaGetLastError());
    evict_gather_kernel<<<(unsigned)((n_groups + kGatherWarps - 1) / kGatherWarps), kGatherWarps * 32, 0, st>>>(a, groups_per_head, n_groups);
    return check_cuda(cudaGetLastError(), "evict_gather_kernel launch");
}

// Eviction from the packed cache: which keys of a (user, head) stay, and their rows gathered into a smaller cache.
//
// Selection.  Keys ordered by (sum descending, position ascending); the budget - recent first of the positions below
// len - recent stay, and the `recent` last positions.  One CTA per (user, head): the sums become order-preserving 32-bit
// numbers in shared memory, three histogram passes find the value of the last one that stays digit by digit, and two scans over
// the positions (which of its equals stay, and where a kept position goes) emit the kept ones in order.
//
// Gather.  A warp moves a group of eight kept rows.  Rows are moved, never recomputed, so the new cache holds the same bits;
// V's pair layout mixes the nibbles of two keys per row, which the lanes take apart for the old pairs and join for the new.
//
// 64 users x 8 heads, up to 8,192 keys to 1,024: 65 us, selection 18 (shared-memory atomics and three passes over the keys) and gather 42
// (5.2 TB/s of sectors: kept rows lie apart, and a sector of signs or norms holds neighbours that go).  The selecting CTA moving its rows
// itself saves a launch and takes 76 us, too few warps to cover the rows' way.
#include "common.cuh"

namespace omni {

constexpr int kSelThreads = 512;
constexpr int kSelKeys = 16;                       // consecutive positions per thread
constexpr int kSelSpan = kSelThreads * kSelKeys;   // positions a CTA holds at a time: a longer cache is read again for every digit
constexpr int kSelKeyBytes = kSelThreads * (kSelKeys + 4) * 4;
constexpr int kSelBins = 2048;

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

// sum over the threads in front of this one, and over all of them (every thread calls this; `part` holds one value per warp)
__device__ __forceinline__ uint32_t sel_scan(uint32_t v, uint32_t* part, uint32_t& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t upto = v;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const uint32_t o = __shfl_up_sync(kFullMask, upto, x);
        if (lane >= x) upto += o;
    }
    __syncthreads();                                             // the previous use of `part` is over
    if (lane == 31) part[warp] = upto;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kSelThreads / 32; ++w) {
        const uint32_t n = part[w];
        if (w < warp) before += n;
        total += n;
    }
    return before + upto - v;
}

__global__ void __launch_bounds__(kSelThreads, 4) evict_select_kernel(const __grid_constant__ omni_evict_t a) {
    __shared__ uint32_t hist[kSelBins];
    __shared__ uint32_t part[kSelThreads / 32];
    __shared__ uint32_t s_value, s_need;
    // this thread's keys, positions base + kSelKeys * tid ..; no candidate: 0.  (Registers for them would halve the CTAs per SM;
    // 20 words apart, the 16-byte accesses of neighbouring threads meet in no bank.)
    extern __shared__ __align__(16) uint32_t sel_keys[];
    const int tid = threadIdx.x;
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
    const bool one_span = n <= kSelSpan;
    const bool aligned = ((reinterpret_cast<uintptr_t>(sums) & 15) == 0);
    uint4* mine4 = reinterpret_cast<uint4*>(sel_keys + (kSelKeys + 4) * tid);
    auto load = [&](int base) {
        const int p = base + kSelKeys * tid;
#pragma unroll
        for (int k = 0; k < kSelKeys; k += 4) {
            uint32_t key[4];
            if (aligned && p + k + 4 <= n) {
                const float4 v = __ldg(reinterpret_cast<const float4*>(sums + p + k));
                key[0] = sum_key(v.x); key[1] = sum_key(v.y); key[2] = sum_key(v.z); key[3] = sum_key(v.w);
            } else {
#pragma unroll
                for (int x = 0; x < 4; ++x) key[x] = p + k + x < n ? sum_key(__ldg(sums + p + k + x)) : 0u;
            }
            mine4[k / 4] = make_uint4(key[0], key[1], key[2], key[3]);
        }
    };
    if (one_span) load(0);
    uint32_t need = (uint32_t)(budget - recent);                 // this many of the keys that agree with `value` so far stay, the largest
    uint32_t value = 0;
    // digits of 11, 11 and 10 bits: the first spans sign, exponent and two bits of the fraction, so that sums of a few binary orders
    // already spread over dozens of counters
#pragma unroll 1
    for (int digit = 0; digit < 3 && need > 0; ++digit) {
        const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
        const uint32_t mask = digit == 2 ? 1023u : 2047u;
        const uint32_t known = digit == 0 ? 0u : digit == 1 ? 0xffe00000u : 0xfffffc00u;
        for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        for (int base = 0; base < n; base += kSelSpan) {
            if (!one_span) load(base);
            if (base + kSelKeys * tid >= n) continue;
#pragma unroll
            for (int k = 0; k < kSelKeys; k += 4) {
                const uint4 v = mine4[k / 4];
                const uint32_t key[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    // no candidate's key is 0 (that of -infinity is 0x007fffff), and from the second digit on `value` is not
                    if ((key[x] & known) == value && key[x] != 0u) atomicAdd(&hist[(key[x] >> shift) & mask], 1u);
            }
        }
        __syncthreads();
        constexpr int kPer = kSelBins / kSelThreads;             // this thread's counters, from the largest down
        uint32_t c[kPer], mine = 0, all;
#pragma unroll
        for (int k = 0; k < kPer; ++k) { c[k] = hist[kSelBins - 1 - (kPer * tid + k)]; mine += c[k]; }
        uint32_t before = sel_scan(mine, part, all);
        if (before < need && before + mine >= need) {
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                if (before < need && before + c[k] >= need) {
                    s_value = value | ((uint32_t)(kSelBins - 1 - (kPer * tid + k)) << shift);
                    s_need = need - before;
                }
                before += c[k];
            }
        }
        __syncthreads();
        value = s_value;
        need = s_need;
    }
    const bool some = budget > recent;                           // `need` of the keys equal to `value` stay, lowest positions first
    uint32_t kept = 0, tied = 0;                                 // of the spans so far
    for (int base = 0; base < len; base += kSelSpan) {
        if (!one_span || base > 0) load(base);
        uint32_t above = 0, equal = 0, total;                    // bit k: the thread's key k
#pragma unroll
        for (int k = 0; k < kSelKeys; k += 4) {
            const uint4 v = mine4[k / 4];
            const uint32_t key[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                above |= key[x] > value ? 1u << (k + x) : 0u;
                equal |= key[x] == value ? 1u << (k + x) : 0u;
            }
        }
        if (!some) above = equal = 0;
        const uint32_t rank = tied + sel_scan(__popc(equal), part, total);
        tied += total;
        uint32_t stay = rank < need ? need - rank : 0;           // the first `stay` of the thread's equals
        uint32_t keep = above;
        for (; equal && stay; --stay) {
            keep |= equal & (0u - equal);
            equal &= equal - 1;
        }
        const int p0 = base + kSelKeys * tid;
#pragma unroll
        for (int k = 0; k < kSelKeys; ++k) keep |= p0 + k >= n && p0 + k < len ? 1u << k : 0u;
        uint32_t at = kept + sel_scan(__popc(keep), part, total);
        kept += total;
        while (keep) {
            const int k = __ffs(keep) - 1;
            keep &= keep - 1;
            if (at < (uint32_t)budget) index[at] = base + kSelKeys * tid + k;
            ++at;
        }
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
    after_predecessor();                                         // the lengths above are older than the selection
    // old position of row r of the group in lane r (-1: no key)
    int from = -1;
    if (lane < 8 && row0 + lane < new_len) from = a.index[bh * a.budget + row0 + lane];
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

// sums of the T keys per (user, head) that come next
__global__ void clear_new_sums_kernel(float* sums, const int64_t* lens, int64_t n, int H, int64_t S, int64_t T) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t bh = i / T, s = __ldg(lens + bh / H) + i % T;
        if (s >= 0 && s < S) sums[bh * S + s] = 0.f;
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
    OMNI_REQUIRE(a.S <= 0x7fff0000LL && a.budget <= 0x7fff0000LL && a.B * a.H <= 0x7fffffffLL, OMNI_ERR_UNSUPPORTED, "omni_evict_keys: extent past 2^31");
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
    OMNI_ALLOW_SMEM((evict_select_kernel), kSelKeyBytes);
    evict_select_kernel<<<(unsigned)(a.B * a.H), kSelThreads, kSelKeyBytes, st>>>(a);
    OMNI_CUDA(cudaGetLastError());
    // The selection lets nobody start early (waiting CTAs take up its places: 9 us); behind its last CTA the gap to the gather is still shorter
    // this way: 12.4 us for 5 users x 2,047 keys against 12.5, and 1 us of host time.
    return check_cuda(launch_early(evict_gather_kernel, dim3((unsigned)((n_groups + kGatherWarps - 1) / kGatherWarps)), kGatherWarps * 32, 0, st, a, groups_per_head, n_groups),
                      "evict_gather_kernel launch");
}

extern "C" int32_t omni_clear_new_sums(float* sums, const int64_t* lens, int64_t B, int32_t H, int64_t S, int64_t T, void* stream) {
    OMNI_REQUIRE(B >= 0 && H >= 0 && S >= 0 && T >= 0, OMNI_ERR_ARG, "omni_clear_new_sums: negative extent");
    if (B == 0 || H == 0 || S == 0 || T == 0) return OMNI_OK;
    OMNI_REQUIRE(sums && lens, OMNI_ERR_ARG, "omni_clear_new_sums: NULL buffer");
    const int64_t n = B * H * T, blocks = (n + 255) / 256;
    clear_new_sums_kernel<<<(unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, (cudaStream_t)stream>>>(sums, lens, n, H, S, T);
    return check_cuda(cudaGetLastError(), "clear_new_sums_kernel launch");
}

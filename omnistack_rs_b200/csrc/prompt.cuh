// Declarations shared by the prompt-attention translation units.
#pragma once
#include "common.cuh"

namespace omni {

// Attention of whole prompts over themselves.  Rows of q / k / v are (b, h, t) with element strides; a prompt is a run of rows
// of one b:  packed:  b = 0, rows cu[i] .. cu[i + 1] - 1;   padded:  b = i, rows 0 .. seq_lens[i] - 1 (or T - 1).
// A tile holds `gp` query heads of one kv head next to each other (row r = head r / tpt of the group, token t0 + r % tpt), so
// that short prompts still fill it and every key is read once for all of them.
struct PromptArgs {
    const void* q; const void* k; const void* v; void* out;
    int64_t qs[3], ks[3], vs[3];                   // element strides of (b, h, t)
    const int32_t* cu; const int32_t* seq_lens;
    int64_t B, T, n_seqs;
    int Hq, Hkv, gp, n_hg;                         // gp heads per tile, n_hg = Hq / Hkv / gp tiles of heads per kv head
    int tpt;                                       // tokens per tile
    int64_t slots;                                 // tile slots per head group (an upper bound where lengths are on the device)
    float scale;
    int causal;
    int32_t* status;
};

struct PromptTile {
    int64_t b, row0;                               // first row of the prompt
    int len, t0;                                   // its length; first token of the tile (>= len: nothing to do)
};

// The prompt and tile behind a slot.  Padded: slots are (b, tile).  Packed: prompt i owns the slots from cu[i] / tpt + i up to
// those of prompt i + 1, which are at least ceil(len / tpt) of them; a warp finds the prompt with 32 probes a step.
// All 32 lanes of a warp call this together.
__device__ __forceinline__ PromptTile prompt_tile(const PromptArgs& a, int64_t slot64, int lane) {
    PromptTile r;
    const uint32_t slot = (uint32_t)slot64, tpt = (uint32_t)a.tpt;       // rows, slots and prompts of a call are below 2^31
    if (!a.cu) {
        const uint32_t per = (uint32_t)a.slots / (uint32_t)a.n_seqs;
        r.b = slot / per;
        r.row0 = 0;
        const int64_t len = a.seq_lens ? (int64_t)__ldg(a.seq_lens + r.b) : a.T;
        r.len = (int)(len < 0 ? 0 : (len > a.T ? a.T : len));
        r.t0 = (int)(slot % per * tpt);
        return r;
    }
    // the last prompt whose first slot is at or below `slot` (first slots ascend strictly; that of prompt 0 counts as 0)
    const int T = (int)a.T;
    uint32_t lo = 0, n = (uint32_t)a.n_seqs;       // the answer lies in [lo, lo + n)
    while (n > 1) {
        const uint32_t step = (n + 31) / 32;
        const uint32_t i = lo + lane * step;
        bool below = lane == 0;
        if (lane > 0 && i < lo + n) {
            int c = a.cu[i];
            c = c < 0 ? 0 : (c > T ? T : c);
            below = (uint32_t)c / tpt + i <= slot;
        }
        const uint32_t next = lo + (31 - __clz((int)__ballot_sync(kFullMask, below))) * step;
        n = lo + n - next < step ? lo + n - next : step;
        lo = next;
    }
    int c0 = a.cu[lo], c1 = a.cu[lo + 1];
    c0 = c0 < 0 ? 0 : (c0 > T ? T : c0);
    c1 = c1 < c0 ? c0 : (c1 > T ? T : c1);
    r.b = 0;
    r.row0 = c0;
    r.len = c1 - c0;
    const uint32_t first = (uint32_t)c0 / tpt + lo;
    const int64_t t0 = ((int64_t)slot - first) * tpt;
    r.t0 = slot < first || t0 > r.len ? r.len : (int)t0;
    return r;
}

// Zeros in the rows that belong to no prompt.  Padded: the rows of the slot's tokens at and behind the length.  Packed: slot i
// looks after rows i * tpt .. (i + 1) * tpt - 1 of the one user (there are more slots than such runs).
template <int DT>
__device__ __forceinline__ void prompt_zero_rows(const PromptArgs& a, const PromptTile& w, int64_t slot, int head0, int tid, int threads) {
    int64_t z0 = slot * a.tpt, zb = 0, live0 = 0, live1 = 0;
    if (a.cu) {
        live0 = __ldg(a.cu);
        live1 = __ldg(a.cu + a.n_seqs);
    } else {
        z0 = w.t0; zb = w.b; live1 = w.len;
    }
    if (z0 >= a.T || (z0 >= live0 && z0 + a.tpt <= live1)) return;
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    for (int at = tid; at < a.tpt * a.gp * 32; at += threads) {
        const int64_t t = z0 + (at >> 5) % a.tpt;
        const int head = head0 + (at >> 5) / a.tpt;
        if (t < a.T && (t < live0 || t >= live1))
            Elem<DT>::store4(a.out, ((zb * a.Hq + head) * a.T + t) * kHeadDim + 4 * (at & 31), zero);
    }
}

// Tensor-core kernel for bf16 and fp16 (prompt_umma.cu)
int32_t launch_prompt_umma(PromptArgs a, int dtype, cudaStream_t st);

}  // namespace omni

// Shared host/device helpers of the omni_b200 library.
#pragma once
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include <stdio.h>
#include <stdarg.h>
#include <atomic>
#include <vector>
#include "../../include/omni_b200.h"

namespace omni {

constexpr int kHeadDim = OMNI_HEAD_DIM;
constexpr int kQjlDim = OMNI_QJL_DIM;
constexpr int kNibBytes = OMNI_NIB_BYTES;
constexpr int kQjlBytes = OMNI_QJL_BYTES;
constexpr int kSeeds = OMNI_N_SEEDS;
constexpr int kMaxDevices = 16;
constexpr unsigned kFullMask = 0xffffffffu;

// fp32 value of 1/sqrt(128): the single multiply that ends the rotation.
#define OMNI_WHT_SCALE_BITS 0x3DB504F3u
// fp32 value of sqrt(2/pi)/128: the QJL reconstruction coefficient.
constexpr float kQjlCoef = (float)(0.7978845608028654 / 128.0);

// Per-device Rademacher tables (device memory owned by the library).
//   rows : [1024 seeds][64 projections][4 words]  bit d of projection i -> word d/32, bit d%32
//   cols : [1024 seeds][128 dims] uint64          bit i of entry d = G[i][d]
struct DeviceTables {
    uint32_t* rows = nullptr;
    uint64_t* cols = nullptr;
};

const DeviceTables* tables_for_current_device();   // nullptr (and error set) if not initialised
const uint32_t* host_rows_table();                 // host copy, built on first use
// Tables of the aligned seed block [1024 * block, 1024 * block + 1024), block >= 1, with at least the seeds
// 1024 * block + j for j in `slots` filled in (generated on the host and uploaded on demand; one block is resident
// per device at a time, and switching blocks synchronises the device).
int32_t extended_tables_for_block(int64_t block, const std::vector<int>& slots, DeviceTables* out);

int32_t set_error(int32_t code, const char* fmt, ...);
int32_t check_cuda(cudaError_t e, const char* what);

#define OMNI_CUDA(call)                                         \
    do {                                                        \
        int32_t _st = ::omni::check_cuda((call), #call);        \
        if (_st != OMNI_OK) return _st;                         \
    } while (0)

#define OMNI_REQUIRE(cond, code, ...)                           \
    do {                                                        \
        if (!(cond)) return ::omni::set_error((code), __VA_ARGS__); \
    } while (0)

// The dynamic shared memory a kernel may be launched with, set once per device (`done`: one bit each).
static inline cudaError_t allow_smem(const void* kernel, int bytes, std::atomic<uint32_t>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint32_t bit = 1u << (dev & 31);
    if (dev < 32 && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 32) done.fetch_or(bit, std::memory_order_release);
    return e;
}
#define OMNI_ALLOW_SMEM(kernel, bytes)                                                          \
    do {                                                                                        \
        static std::atomic<uint32_t> _done{0};                                                  \
        OMNI_CUDA(::omni::allow_smem(reinterpret_cast<const void*>(kernel), (int)(bytes), _done)); \
    } while (0)

// Launch behind a kernel of the same call that lets its successors start early (follow_me_early): the successor's CTAs are placed while the
// last ones of its predecessor run, and wait (after_predecessor) before they touch what it wrote.
template <typename... Params, typename... Args>
static cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t st, Args&&... args) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid; cfg.blockDim = dim3((unsigned)threads); cfg.dynamicSmemBytes = smem; cfg.stream = st; cfg.attrs = &attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

// ---- device helpers ----------------------------------------------------------

__device__ __forceinline__ void follow_me_early() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }
__device__ __forceinline__ void after_predecessor() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

// 128-point normalised Walsh-Hadamard transform of one row spread over a warp:
// lane l holds elements 4l..4l+3.  Stage order h = 1, 2, 4, ..., 64, every add and
// subtract rounded to fp32 on its own, one final multiply -- the reference order.
__device__ __forceinline__ void wht128_warp(float (&v)[4], int lane) {
    float a0 = __fadd_rn(v[0], v[1]), a1 = __fsub_rn(v[0], v[1]);
    float a2 = __fadd_rn(v[2], v[3]), a3 = __fsub_rn(v[2], v[3]);
    v[0] = __fadd_rn(a0, a2); v[2] = __fsub_rn(a0, a2);
    v[1] = __fadd_rn(a1, a3); v[3] = __fsub_rn(a1, a3);
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const bool lower = (lane & m) != 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float o = __shfl_xor_sync(kFullMask, v[k], m);
            v[k] = lower ? __fsub_rn(o, v[k]) : __fadd_rn(v[k], o);
        }
    }
    const float s = __uint_as_float(OMNI_WHT_SCALE_BITS);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = __fmul_rn(v[k], s);
}

// Load 4 consecutive elements of a row as fp32 (lane-owned quarter of a 16-float group).
template <int DT> struct Elem;
template <> struct Elem<OMNI_F32> {
    using T = float;
    static __device__ __forceinline__ void load4(const void* p, int64_t i, float (&v)[4]) {
        float4 t = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
    }
    static __device__ __forceinline__ void store4(void* p, int64_t i, const float (&v)[4]) {
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
    }
    static __device__ __forceinline__ float round(float x) { return x; }
};
template <> struct Elem<OMNI_BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ void load4(const void* p, int64_t i, float (&v)[4]) {
        uint2 t = *reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(p) + i);
        v[0] = __uint_as_float(t.x << 16); v[1] = __uint_as_float(t.x & 0xffff0000u);
        v[2] = __uint_as_float(t.y << 16); v[3] = __uint_as_float(t.y & 0xffff0000u);
    }
    static __device__ __forceinline__ void store4(void* p, int64_t i, const float (&v)[4]) {
        __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]);
        __nv_bfloat162 hi = __floats2bfloat162_rn(v[2], v[3]);
        uint2 t;
        t.x = *reinterpret_cast<uint32_t*>(&lo);
        t.y = *reinterpret_cast<uint32_t*>(&hi);
        *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p) + i) = t;
    }
    static __device__ __forceinline__ float round(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }
};
template <> struct Elem<OMNI_F16> {
    using T = __half;
    static __device__ __forceinline__ void load4(const void* p, int64_t i, float (&v)[4]) {
        uint2 t = *reinterpret_cast<const uint2*>(reinterpret_cast<const __half*>(p) + i);
        __half2 lo = *reinterpret_cast<__half2*>(&t.x), hi = *reinterpret_cast<__half2*>(&t.y);
        float2 a = __half22float2(lo), b = __half22float2(hi);
        v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    }
    static __device__ __forceinline__ void store4(void* p, int64_t i, const float (&v)[4]) {
        __half2 lo = __floats2half2_rn(v[0], v[1]);
        __half2 hi = __floats2half2_rn(v[2], v[3]);
        uint2 t;
        t.x = *reinterpret_cast<uint32_t*>(&lo);
        t.y = *reinterpret_cast<uint32_t*>(&hi);
        *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(p) + i) = t;
    }
    static __device__ __forceinline__ float round(float x) { return __half2float(__float2half_rn(x)); }
};

// Load 8 consecutive elements of a row as fp32 (16-byte loads).
template <int DT> __device__ __forceinline__ void load8(const void* p, int64_t i, float (&v)[8]) {
    if constexpr (DT == OMNI_F32) {
        const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
        const float4 b = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 t = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
        const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (DT == OMNI_BF16) {
                v[2 * k] = __uint_as_float(w[k] << 16);
                v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
                v[2 * k] = f.x;
                v[2 * k + 1] = f.y;
            }
        }
    }
}

__device__ __forceinline__ int seed_of(int32_t user_id, int head) { return ((user_id & 1023) ^ head) & 1023; }

}  // namespace omni

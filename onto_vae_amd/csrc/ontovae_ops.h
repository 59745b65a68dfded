// Shared by the dense-block operators (ontovae_ops.hip): element types, 8-element loads, wave and block reductions.
#ifndef ONTOVAE_OPS_H
#define ONTOVAE_OPS_H

#include "ontovae_device.h"
#include "ontovae_internal.h"

#define OV_OPS_LAUNCH_CHECK(what)                                                                                     \
    do {                                                                                                              \
        hipError_t e_ = hipGetLastError();                                                                            \
        if (e_ != hipSuccess) { ontovae_set_error("%s: %s", what, hipGetErrorString(e_)); return ONTOVAE_EHIP; }      \
    } while (0)

// one launch takes less than 2^32 threads along x
static inline bool ov_ops_fits(int64_t workgroups, int threads) { return workgroups <= (int64_t)UINT32_MAX / threads; }

typedef __bf16 ov_bf;
typedef _Float16 ov_hf;

// one rounding to the element type, to the nearest even
template <typename T> __device__ __forceinline__ T ov_from_f(float v) { return (T)v; }
template <typename T> __device__ __forceinline__ float ov_to_f(T v) { return (float)v; }

template <int N> struct OvBytes { int8_t b[N]; };

// 16 bytes of elements, loaded and stored at any element's address (unaligned 16-B accesses are one instruction here)
template <typename T>
struct OvVec {
    static constexpr int N = 16 / sizeof(T);
    T e[N];
    __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(e, p, 16); }
    __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(p, e, 16); }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < N; ++j) e[j] = (T)0.f;
    }
};

// waits until at most N vector-memory operations of the wave are outstanding, and its LDS operations are done
template <int N>
__device__ __forceinline__ void ov_wait_vm() {
    static_assert(N < 64, "the counter holds 63");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint32_t ov_wave_max_u(uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
    return v;
}

// sum over the workgroup (a multiple of 64 threads, every thread calls); red: 16 floats of LDS
__device__ __forceinline__ float ov_block_sum(float v, float* red) {
    v = ov_wave_sum(v);
    __syncthreads();
    if (ov_lane() == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) s += red[w];
    return s;
}

#endif

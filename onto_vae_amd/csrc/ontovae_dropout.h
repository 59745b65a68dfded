// Dropout of a sample-major matrix whose mask is drawn again wherever it is needed, never stored.
//
// Element c of row r belongs to block r * ceil(C / 8) + c / 8; one Philox4x32-10 call (key = seed, counter = block, stream,
// offset) gives the block's eight 16-bit draws, element c % 8 takes half-word c % 8.  Kept iff draw >= t, t = rint(65536 p), scaled by
// 65536 / (65536 - t): p is taken at a resolution of 2^-16, and the factor belongs to the p that is really drawn, so the
// expectation is exact.  16 bits and not 32: a 32-bit draw per element needs twice the integer products, and those, not the
// memory, would bound the 16-bit types.
// A dropped element is a select, not a product: an infinity or a NaN in a dropped place gives 0.
#ifndef ONTOVAE_DROPOUT_H
#define ONTOVAE_DROPOUT_H

#include "ontovae_ops.h"

#define OV_RNG_OP 6u

struct OvDrop {
    uint64_t seed, offset;
    uint32_t t;            // drop iff draw < t; 0: nothing is dropped
    float scale;
};

static inline int ov_drop_from(float p, uint64_t seed, uint64_t offset, OvDrop* d) {
    if (!(p >= 0.f && p <= 1.f)) return -1;
    d->seed = seed;
    d->offset = offset;
    d->t = (uint32_t)__builtin_rint((double)p * 65536.0);
    d->scale = d->t < 65536u ? (float)(65536.0 / (double)(65536u - d->t)) : 0.f;
    return 0;
}

// bit j: element j of the block is kept
__device__ __forceinline__ uint32_t ov_drop_bits(const OvDrop& d, uint64_t block) {
    const OvPhilox r = ov_philox(d.seed, d.offset, OV_RNG_OP, block);
    uint32_t m = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        m |= ((r.c[w] & 0xFFFFu) >= d.t ? 1u : 0u) << (2 * w);
        m |= ((r.c[w] >> 16) >= d.t ? 1u : 0u) << (2 * w + 1);
    }
    return m;
}

template <typename T>
__global__ __launch_bounds__(256) void ov_dropout_kernel(const T* __restrict__ x, int64_t ldx, const int32_t* __restrict__ rows, int n_src,
                                                         int R, int C, OvDrop d, T* __restrict__ y) {
    const int nb = (C + 7) / 8;
    const int64_t total = (int64_t)R * nb;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / nb;
        const int c0 = (int)(i - r * nb) * 8;
        int64_t src = r;
        bool ok = true;
        if (rows) { src = rows[r]; ok = src >= 0 && src < n_src; }
        const uint32_t m = ov_drop_bits(d, (uint64_t)i);
        for (int j = 0; j < 8 && c0 + j < C; ++j) {
            float v = __builtin_nanf("");
            if (ok) v = (m >> j) & 1 ? ov_to_f<T>(x[src * ldx + c0 + j]) * d.scale : 0.f;
            y[r * C + c0 + j] = ov_from_f<T>(v);
        }
    }
}

extern "C" int ontovae_dropout(const void* x, int32_t dtype, int64_t ldx, const int32_t* rows, int32_t n_src, int32_t R, int32_t C, float p,
                               uint64_t seed, uint64_t offset, void* y, void* stream) {
    OvDrop d;
    if (R < 0 || C < 0 || n_src < 0 || ldx < C || (!rows && n_src < R)) {
        ontovae_set_error("dropout: R = %d, C = %d, n_src = %d, ldx = %lld", R, C, n_src, (long long)ldx);
        return ONTOVAE_EINVAL;
    }
    if (ov_drop_from(p, seed, offset, &d)) { ontovae_set_error("dropout: p = %g outside [0, 1]", (double)p); return ONTOVAE_EINVAL; }
    if (dtype < ONTOVAE_F32 || dtype > ONTOVAE_F16) { ontovae_set_error("dropout: unknown element type %d", dtype); return ONTOVAE_EINVAL; }
    if (R == 0 || C == 0) return ONTOVAE_OK;
    if (!x || !y) { ontovae_set_error("dropout: NULL argument"); return ONTOVAE_EINVAL; }
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int64_t total = (int64_t)R * ((C + 7) / 8);
    const dim3 grid((unsigned)std::min<int64_t>((total + 255) / 256, 8192));
    switch (dtype) {
        case ONTOVAE_F32: hipLaunchKernelGGL(ov_dropout_kernel<float>, grid, dim3(256), 0, st, (const float*)x, ldx, rows, n_src, R, C, d, (float*)y); break;
        case ONTOVAE_BF16: hipLaunchKernelGGL(ov_dropout_kernel<ov_bf>, grid, dim3(256), 0, st, (const ov_bf*)x, ldx, rows, n_src, R, C, d, (ov_bf*)y); break;
        default: hipLaunchKernelGGL(ov_dropout_kernel<ov_hf>, grid, dim3(256), 0, st, (const ov_hf*)x, ldx, rows, n_src, R, C, d, (ov_hf*)y); break;
    }
    OV_OPS_LAUNCH_CHECK("dropout");
    return ONTOVAE_OK;
}

#endif

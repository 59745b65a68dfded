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

// The block's draws.  ov_philox with the two 32 x 32-bit products of a round as one 64-bit multiply each.
__device__ __forceinline__ OvPhilox ov_drop_draw(const OvDrop& d, uint64_t block) {
    uint32_t k0 = (uint32_t)d.seed, k1 = (uint32_t)(d.seed >> 32);
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32) ^ (OV_RNG_OP << 24), c2 = (uint32_t)d.offset, c3 = (uint32_t)(d.offset >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    OvPhilox o;
    o.c[0] = c0; o.c[1] = c1; o.c[2] = c2; o.c[3] = c3;
    return o;
}

// draw j of the block decides element j
__device__ __forceinline__ bool ov_drop_kept(const OvDrop& d, const OvPhilox& r, int j) {
    return ((j & 1) ? r.c[j >> 1] >> 16 : r.c[j >> 1] & 0xFFFFu) >= d.t;
}

__device__ __forceinline__ float ov_drop_apply(const OvDrop& d, const OvPhilox& r, int j, float v) {
    return ov_drop_kept(d, r, j) ? v * d.scale : 0.f;
}

// One block of 8 elements per thread, 16 B a load whatever the alignment.  Its place in the matrix is one 64-bit division per
// workgroup and a small one per thread.  Bound by memory: 16384 x 20000 bf16 in 274 us (4.8 TB/s where a copy runs at
// 4.9; the draws take 2 % of it), 16384 x 10000 float32 in 230.  Two, four or eight blocks in flight per thread are 3 to 15 % slower in
// bf16 and 14 to 20 % in float32: more waves hide the latency better than more loads.
template <typename T>
__global__ __launch_bounds__(256) void ov_dropout_kernel(const T* __restrict__ x, int64_t ldx, const int32_t* __restrict__ rows, int n_src,
                                                         int R, int C, uint32_t nb, OvDrop d, T* __restrict__ y) {
    constexpr int VE = 16 / sizeof(T), NV = 8 / VE;
    const int64_t first = (int64_t)blockIdx.x * 256, row0 = first / nb;
    const uint32_t t = (uint32_t)(first - row0 * nb) + threadIdx.x, dr = t / nb, c0 = (t - dr * nb) * 8;
    const int64_t row = row0 + dr;
    if (row >= R) return;
    int64_t src = row;
    bool ok = true;
    if (rows) { src = rows[src]; ok = src >= 0 && src < n_src; }
    const T* xr = x + (ok ? src : 0) * ldx + c0;
    T* yr = y + row * C + c0;
    const bool whole = c0 + 8 <= (uint32_t)C;
    OvVec<T> v[NV];
    if (whole && ok) {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i].load(xr + i * VE);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j / VE].e[j % VE] = ok && c0 + j < (uint32_t)C ? xr[j] : (T)0.f;
    }
    const OvPhilox r = ov_drop_draw(d, (uint64_t)first + threadIdx.x);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        T& e = v[j / VE].e[j % VE];
        e = ov_from_f<T>(ok ? ov_drop_apply(d, r, j, ov_to_f<T>(e)) : __builtin_nanf(""));
    }
    if (whole) {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i].store(yr + i * VE);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c0 + j < (uint32_t)C) yr[j] = v[j / VE].e[j % VE];
    }
}

template <typename T>
static int ov_dropout_launch(const void* x, int64_t ldx, const int32_t* rows, int n_src, int R, int C, const OvDrop& d, void* y, hipStream_t st) {
    const uint32_t nb = ((uint32_t)C + 7) / 8;
    const int64_t wg = ((int64_t)R * nb + 255) / 256;
    if (!ov_ops_fits(wg, 256)) { ontovae_set_error("dropout: %d x %d elements are too many for one launch", R, C); return ONTOVAE_EINVAL; }
    hipLaunchKernelGGL(ov_dropout_kernel<T>, dim3((unsigned)wg), dim3(256), 0, st, static_cast<const T*>(x), ldx, rows, n_src, R, C, nb, d, static_cast<T*>(y));
    return ONTOVAE_OK;
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
    int rc;
    switch (dtype) {
        case ONTOVAE_F32: rc = ov_dropout_launch<float>(x, ldx, rows, n_src, R, C, d, y, st); break;
        case ONTOVAE_BF16: rc = ov_dropout_launch<ov_bf>(x, ldx, rows, n_src, R, C, d, y, st); break;
        default: rc = ov_dropout_launch<ov_hf>(x, ldx, rows, n_src, R, C, d, y, st); break;
    }
    if (rc) return rc;
    OV_OPS_LAUNCH_CHECK("dropout");
    return ONTOVAE_OK;
}

#endif

// Group norm with an activation and dropout in one operator, channels last: x [N, S, C], groups of C / groups channels.
//
//   per sample and group (S rows x C / groups channels): mu, biased var, r = 1 / sqrt(var + eps)
//   v = (x - mu) r gamma_c + beta_c,   y = D act(v),   D = keep / (1 - p) as in ontovae_dropout.h over the rows [N S, C]
// Backward: dv = dy D act'(v), dgamma_c = sum dv xhat, dbeta_c = sum dv, e = dv gamma,
//   dx = r (e - mean(e) - xhat mean(e xhat)), the means over the group.
// Statistics and every sum are held in 32 bits, and a large mean costs no digits: a float32 mean alone would be off by half a step of
// its own magnitude, a shift common to the whole group (1e-3 of the spread at a mean of 1e4 spreads).  Every form takes the sum of
// x - mean about a mean it has, and with it the REST that the float32 mean leaves; x - mean - rest is what is normalised.  The
// variance is the second moment about the mean (two passes over what is held or cached).  The saved mean is the nearest float32;
// the backward pass finds the rest again from x, where it counts (ov_gn_far).
#ifndef ONTOVAE_GROUPNORM_H
#define ONTOVAE_GROUPNORM_H

#include "ontovae_dropout.h"

// 8 neighbours of a row: one Philox block of dropout where they start on a multiple of 8, else two
template <typename T>
struct OvGnPiece {
    static constexpr int N = 8;
    T e[8];
    __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(e, p, sizeof(e)); }
    __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(p, e, sizeof(e)); }
};

struct OvGn {
    int N, S, C, groups, cg;
    const void* w;
    const void* b;
    int wtype;               // element type of w and b
    float eps;
    int act;
    OvDrop drop;
};

__device__ __forceinline__ float ov_gn_param(const void* p, int wtype, int c, float none) {
    if (!p) return none;
    if (wtype == ONTOVAE_F32) return static_cast<const float*>(p)[c];
    if (wtype == ONTOVAE_BF16) return (float)static_cast<const ov_bf*>(p)[c];
    return (float)static_cast<const ov_hf*>(p)[c];
}

// E neighbours of a parameter vector from channel c on, cnt of them valid (the rest 0)
template <int E>
__device__ __forceinline__ void ov_gn_params(const void* p, int wtype, int c, int cnt, float none, float (&f)[E]) {
#pragma unroll
    for (int j = 0; j < E; ++j) f[j] = j < cnt ? none : 0.f;
    if (!p) return;
    if (wtype == ONTOVAE_F32 && cnt >= E) {
        __builtin_memcpy(f, static_cast<const float*>(p) + c, sizeof(f));
    } else if (wtype == ONTOVAE_F32) {
#pragma unroll
        for (int j = 0; j < E; ++j) f[j] = static_cast<const float*>(p)[c + min(j, max(cnt - 1, 0))];
    } else if (wtype == ONTOVAE_BF16) {
#pragma unroll
        for (int j = 0; j < E; ++j) f[j] = (float)static_cast<const ov_bf*>(p)[c + min(j, max(cnt - 1, 0))];
    } else {
#pragma unroll
        for (int j = 0; j < E; ++j) f[j] = (float)static_cast<const ov_hf*>(p)[c + min(j, max(cnt - 1, 0))];
    }
}

// sigma(v) and what silu and gelu and their slopes need of exp and erf
__device__ __forceinline__ float ov_sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + __expf(-v)); }

// act over E values: the switch stands outside the loop (act is uniform)
template <int E>
__device__ __forceinline__ void ov_act(float (&v)[E], int act) {
    if (act == ONTOVAE_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = v[j] < 0.f ? 0.f : v[j];                    // NaN stays NaN
    } else if (act == ONTOVAE_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = v[j] * ov_sigmoid(v[j]);
    } else if (act == ONTOVAE_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = 0.5f * v[j] * (1.f + erff(v[j] * 0.70710678118654752f));
    }
}

// d act / d v
template <int E>
__device__ __forceinline__ void ov_act_grad(float (&v)[E], int act) {
    if (act == ONTOVAE_ACT_NONE) {
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = 1.f;
    } else if (act == ONTOVAE_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = v[j] > 0.f ? 1.f : (v[j] <= 0.f ? 0.f : v[j]);
    } else if (act == ONTOVAE_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const float s = ov_sigmoid(v[j]);
            v[j] = s * (1.f + v[j] * (1.f - s));
        }
    } else if (act == ONTOVAE_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < E; ++j)
            v[j] = 0.5f * (1.f + erff(v[j] * 0.70710678118654752f)) + v[j] * __expf(-0.5f * v[j] * v[j]) * 0.39894228040143268f;
    }
}

// the kept ones of E neighbours of a row from column c on (E <= 8: at most two of the row's blocks of eight), bit j = element j
template <int E>
__device__ __forceinline__ uint32_t ov_gn_kept(const OvGn& p, int64_t row, int c) {
    const uint64_t block = (uint64_t)row * ((p.C + 7) / 8) + (c >> 3);
    const int o = c & 7;
    OvPhilox r = ov_drop_draw(p.drop, block);
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m |= (ov_drop_kept(p.drop, r, j) ? 1u : 0u) << j;
    if (o + E > 8) {
        r = ov_drop_draw(p.drop, block + 1);
#pragma unroll
        for (int j = 0; j < 8; ++j) m |= (ov_drop_kept(p.drop, r, j) ? 1u : 0u) << (8 + j);
    }
    return m >> o;
}
template <int E>
__device__ __forceinline__ void ov_gn_drop(const OvGn& p, int64_t row, int c, float (&v)[E]) {
    if (p.drop.t == 0) return;
    const uint32_t m = ov_gn_kept<E>(p, row, c);
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = (m >> j) & 1 ? v[j] * p.drop.scale : 0.f;
}
// dv = dy D act'(v): v comes in, dv goes out; a dropped place gives 0 whatever dy and act' are
template <int E>
__device__ __forceinline__ void ov_gn_dv(const OvGn& p, int64_t row, int c, const float (&dy)[E], float (&v)[E]) {
    ov_act_grad<E>(v, p.act);
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] *= dy[j];
    ov_gn_drop<E>(p, row, c, v);
}

// 8 elements from `off` on of x [total], whatever of them belongs to the reader: a piece that ends inside the 8 reads
// on into its neighbour.  The load is unconditional (a branch around it would make the compiler wait for every load by itself);
// the last pieces of the tensor, which have no neighbour, are read from further in front, and ov_gn_floats fetches their
// elements one by one.
template <typename T>
__device__ __forceinline__ void ov_gn_raw(const T* x, int64_t total, int64_t off, OvGnPiece<T>& v) {
    v.load(x + min(off, total - OvGnPiece<T>::N));
}
template <typename T>
__device__ __forceinline__ void ov_gn_floats(const T* x, int64_t total, int64_t off, const OvGnPiece<T>& v, float (&f)[OvGnPiece<T>::N]) {
    constexpr int E = OvGnPiece<T>::N;
#pragma unroll
    for (int j = 0; j < E; ++j) f[j] = ov_to_f<T>(v.e[j]);
    if (off > total - E) {
#pragma unroll
        for (int j = 0; j < E; ++j) f[j] = off + j < total ? ov_to_f<T>(x[off + j]) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void ov_gn_store(T* y, int cnt, const float (&f)[OvGnPiece<T>::N]) {
    constexpr int E = OvGnPiece<T>::N;
    OvGnPiece<T> v;
#pragma unroll
    for (int j = 0; j < E; ++j) v.e[j] = ov_from_f<T>(f[j]);
    if (cnt >= E) v.store(y);
    else {
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (j < cnt) y[j] = v.e[j];
    }
}

template <int E>
__device__ __forceinline__ void ov_gn_store_f(float* y, int cnt, const float (&f)[E]) {
#pragma unroll
    for (int j = 0; j < E; ++j)
        if (j < cnt) y[j] = f[j];
}

// LIGHT kernels: no dropout and no gelu, whose code (two Philox draws, erff) sets the register count of the others
template <bool LIGHT>
__device__ __forceinline__ OvGn ov_gn_light(OvGn p) {
    if (LIGHT) {
        p.drop.t = 0;
        p.act = min(p.act, (int)ONTOVAE_ACT_SILU);
    }
    return p;
}

// sum over the LPG threads of a group, in every one of them: lanes of a wave (DPP moves inside 16 lanes), or the workgroup
template <int LPG>
__device__ __forceinline__ float ov_gn_sum(float v, float* red) {
    if (LPG > 64) return ov_block_sum(v, red);
    v += ov_dpp<0xB1, 0xF>(v);                           // quad_perm [1,0,3,2]
    v += ov_dpp<0x4E, 0xF>(v);                           // quad_perm [2,3,0,1]
    v += ov_dpp<0x141, 0xF>(v);                          // row_half_mirror: 8 lanes
    if (LPG >= 16) v += ov_dpp<0x140, 0xF>(v);           // row_mirror: 16 lanes
    if (LPG >= 32) v += __shfl_xor(v, 16, 64);
    if (LPG >= 64) v += __shfl_xor(v, 32, 64);
    return v;
}

// the same for two values
template <int LPG>
__device__ __forceinline__ float2 ov_gn_sum2(float a, float b, float* red) {
    if (LPG <= 64) return make_float2(ov_gn_sum<LPG>(a, red), ov_gn_sum<LPG>(b, red));
    a = ov_wave_sum(a);
    b = ov_wave_sum(b);
    __syncthreads();
    if (ov_lane() == 0) { red[threadIdx.x >> 6] = a; red[16 + (threadIdx.x >> 6)] = b; }
    __syncthreads();
    a = b = 0.f;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) { a += red[w]; b += red[16 + w]; }
    return make_float2(a, b);
}

// Whether the backward pass looks for the rest of a group: the saved mean is off by at most 2^-24 |mean|, xhat by that times rstd.
// Up to 4 spreads that is less than what the rounding of x - mean itself does to the group's outer values.
__device__ __forceinline__ bool ov_gn_far(float mean, float rstd) { return fabsf(mean) * rstd > 4.f; }

// a + b as the nearest float32 and what that leaves
__device__ __forceinline__ float ov_gn_two(float a, float b, float* rest) {
    const float s = a + b, t = s - a;
    *rest = (a - (s - t)) + (b - t);
    return s;
}
// a variance from a second moment about a mean that is off by `rest` (NaN stays)
__device__ __forceinline__ float ov_gn_var(float m2, float rest) {
    const float v = m2 - rest * rest;
    return v < 0.f ? 0.f : v;
}

// ---------------------------------------------------------------- S = 1: a group is one contiguous run of cg elements
// LPG threads hold a group in registers, NV pieces of 8 elements each; a slot of LPG threads keeps its group and walks the
// samples rs, rs + RS, ...: weight and bias (and the sums of their gradients) stay in registers.  Neighbouring slots take
// neighbouring groups, so a workgroup reads contiguous memory.  One read of x (and dy), one write: bound by memory.
// The next sample is requested before the current one is reduced.
template <typename T, int LPG, int NV, bool LIGHT>
__global__ __launch_bounds__(LPG < 256 ? 256 : LPG) void ov_gn_row_fwd_kernel(const T* __restrict__ x, const OvGn p_, int RS, T* __restrict__ y,
                                                                             float* __restrict__ mean, float* __restrict__ rstd) {
    const OvGn p = ov_gn_light<LIGHT>(p_);
    constexpr int E = OvGnPiece<T>::N, BLOCK = LPG < 256 ? 256 : LPG;
    __shared__ float red[32];
    const int64_t slot = ((int64_t)blockIdx.x * BLOCK + threadIdx.x) / LPG;
    const int j = threadIdx.x % LPG, rs = (int)(slot / p.groups), g = (int)(slot - (int64_t)rs * p.groups);
    if (rs >= RS) return;
    const int64_t gc = (int64_t)g * p.cg, step = (int64_t)RS * p.C;
    const int64_t total = (int64_t)p.N * p.C;
    const bool ragged = p.cg % E != 0;
    int64_t at = (int64_t)rs * p.C + gc;
    OvGnPiece<T> raw[NV];
    int cnt[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int o = (j + i * LPG) * E;
        cnt[i] = min(p.cg - o, E);
        ov_gn_raw<T>(x, total, at + o, raw[i]);
    }
    float w[NV][E], b[NV][E];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (cnt[i] > 0) {
            ov_gn_params<E>(p.w, p.wtype, (int)gc + (j + i * LPG) * E, cnt[i], 1.f, w[i]);
            ov_gn_params<E>(p.b, p.wtype, (int)gc + (j + i * LPG) * E, cnt[i], 0.f, b[i]);
        }
    const float len = (float)p.cg;
    for (int n = rs; n < p.N; n += RS) {
        float v[NV][E];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            ov_gn_floats<T>(x, total, at + (j + i * LPG) * E, raw[i], v[i]);
            if (ragged || NV > 1 || LPG * E > p.cg) {     // not every piece is whole
#pragma unroll
                for (int k = 0; k < E; ++k) v[i][k] = k < cnt[i] ? v[i][k] : 0.f;
            }
#pragma unroll
            for (int k = 0; k < E; ++k) s += v[i][k];
        }
        const int64_t here = at;
        at += step;
        if (n + RS < p.N) {
#pragma unroll
            for (int i = 0; i < NV; ++i) ov_gn_raw<T>(x, total, at + (j + i * LPG) * E, raw[i]);
        }
        const float mu = ov_gn_sum<LPG>(s, red) / len;
        s = 0.f;
        float left = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < E; ++k) {
                v[i][k] = k < cnt[i] ? v[i][k] - mu : 0.f;
                s += v[i][k] * v[i][k];
                left += v[i][k];
            }
        const float2 sl = ov_gn_sum2<LPG>(s, left, red);
        const float rest = sl.y / len, r = 1.f / sqrtf(ov_gn_var(sl.x / len, rest) + p.eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (cnt[i] <= 0) continue;
            const int o = (j + i * LPG) * E;
#pragma unroll
            for (int k = 0; k < E; ++k) v[i][k] = (v[i][k] - rest) * r * w[i][k] + b[i][k];
            ov_act<E>(v[i], p.act);
            ov_gn_drop<E>(p, n, (int)gc + o, v[i]);
            ov_gn_store<T>(y + here + o, cnt[i], v[i]);
        }
        if (j == 0) {
            mean[(int64_t)n * p.groups + g] = mu + rest;
            rstd[(int64_t)n * p.groups + g] = r;
        }
    }
}

// part: [2][R][C]: sums of dv xhat, then of dv.  A slot's sums, or, where whole samples fit a workgroup (wgs of them at a time), the
// workgroup's: fewer rows to write and to add up again.
template <typename T, int LPG, int NV, bool LIGHT>
__global__ __launch_bounds__(LPG < 256 ? 256 : LPG) void ov_gn_row_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const OvGn p_, int RS, int wgs,
                                                                             const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                             T* __restrict__ dx, float* __restrict__ part) {
    const OvGn p = ov_gn_light<LIGHT>(p_);
    constexpr int E = OvGnPiece<T>::N, BLOCK = LPG < 256 ? 256 : LPG;
    __shared__ float red[32];
    __shared__ float sums[LPG < 256 ? 256 * 8 : 8];
    const int64_t slot = ((int64_t)blockIdx.x * BLOCK + threadIdx.x) / LPG;
    const int j = threadIdx.x % LPG, rs = (int)(slot / p.groups), g = (int)(slot - (int64_t)rs * p.groups);
    const int64_t gc = (int64_t)g * p.cg, step = (int64_t)RS * p.C;
    const int64_t total = (int64_t)p.N * p.C;
    const int first = min(rs, p.N - 1);                  // a slot past the last (rs >= RS) walks no sample
    int64_t at = (int64_t)first * p.C + gc;
    OvGnPiece<T> rx[NV], rd[NV];
    int cnt[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int o = (j + i * LPG) * E;
        cnt[i] = min(p.cg - o, E);
        ov_gn_raw<T>(x, total, at + o, rx[i]);
        ov_gn_raw<T>(dy, total, at + o, rd[i]);
    }
    float mu = mean[(int64_t)first * p.groups + g], r = rstd[(int64_t)first * p.groups + g];
    float w[NV][E], b[NV][E], sw[NV][E], sb[NV][E];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int k = 0; k < E; ++k) w[i][k] = b[i][k] = sw[i][k] = sb[i][k] = 0.f;
        if (cnt[i] > 0) {
            ov_gn_params<E>(p.w, p.wtype, (int)gc + (j + i * LPG) * E, cnt[i], 1.f, w[i]);
            ov_gn_params<E>(p.b, p.wtype, (int)gc + (j + i * LPG) * E, cnt[i], 0.f, b[i]);
        }
    }
    const float len = (float)p.cg;
    for (int n = rs < RS ? rs : p.N; n < p.N; n += RS) {
        const int64_t here = at;
        const float mu0 = mu, r0 = r;
        float v[NV][E], d[NV][E];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            ov_gn_floats<T>(x, total, at + (j + i * LPG) * E, rx[i], v[i]);
            ov_gn_floats<T>(dy, total, at + (j + i * LPG) * E, rd[i], d[i]);
        }
        at += step;
        if (n + RS < p.N) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                ov_gn_raw<T>(x, total, at + (j + i * LPG) * E, rx[i]);
                ov_gn_raw<T>(dy, total, at + (j + i * LPG) * E, rd[i]);
            }
            mu = mean[(int64_t)(n + RS) * p.groups + g];
            r = rstd[(int64_t)(n + RS) * p.groups + g];
        }
        float s1 = 0.f, s2 = 0.f, rest = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < E; ++k) {
                v[i][k] -= mu0;
                if (k >= cnt[i]) v[i][k] = 0.f;
            }
        if (ov_gn_far(mu0, r0)) {                        // the same in every thread of the group
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int k = 0; k < E; ++k) rest += v[i][k];
            rest = ov_gn_sum<LPG>(rest, red) / len;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float a[E];
#pragma unroll
            for (int k = 0; k < E; ++k) {
                v[i][k] = (v[i][k] - rest) * r0;
                a[k] = v[i][k] * w[i][k] + b[i][k];
            }
            ov_gn_dv<E>(p, n, (int)gc + (j + i * LPG) * E, d[i], a);
#pragma unroll
            for (int k = 0; k < E; ++k) {
                if (k >= cnt[i]) a[k] = v[i][k] = 0.f;
                sw[i][k] += a[k] * v[i][k];
                sb[i][k] += a[k];
                d[i][k] = a[k] * w[i][k];
                s1 += d[i][k];
                s2 += d[i][k] * v[i][k];
            }
        }
        const float2 sg = ov_gn_sum2<LPG>(s1, s2, red);
        s1 = sg.x / len;
        s2 = sg.y / len;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (cnt[i] <= 0) continue;
#pragma unroll
            for (int k = 0; k < E; ++k) d[i][k] = r0 * (d[i][k] - s1 - v[i][k] * s2);
            ov_gn_store<T>(dx + here + (j + i * LPG) * E, cnt[i], d[i]);
        }
    }
    if (!part) return;
    const int64_t R = wgs > 1 ? gridDim.x : RS, row = wgs > 1 ? blockIdx.x : rs;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (LPG < 256 && wgs > 1) {                      // uniform; 256 = wgs * groups * LPG
            const int lane = threadIdx.x, per = p.groups * LPG;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                __syncthreads();
#pragma unroll
                for (int k = 0; k < E; ++k) sums[k * 256 + lane] = h ? sb[i][k] : sw[i][k];
                __syncthreads();
                if (lane < per)
                    for (int o = per; o < 256; o += per) {
#pragma unroll
                        for (int k = 0; k < E; ++k) (h ? sb[i][k] : sw[i][k]) += sums[k * 256 + lane + o];
                    }
            }
            if (lane >= per) continue;
        } else if (rs >= RS) {
            continue;
        }
        const int64_t o = row * p.C + gc + (j + i * LPG) * E;
        ov_gn_store_f<E>(part + o, cnt[i], sw[i]);
        ov_gn_store_f<E>(part + R * p.C + o, cnt[i], sb[i]);
    }
}

// A thread's sum of any number of terms in three levels of 64: a path of 64 + 64 + n / 4096 additions instead of n.
struct OvGnLong {
    float a = 0.f, b = 0.f, c = 0.f;
    int n = 0;
    __device__ __forceinline__ void add(float v) {
        a += v;
        if ((++n & 63) == 0) {
            b += a;
            a = 0.f;
            if ((n & 4095) == 0) { c += b; b = 0.f; }
        }
    }
    __device__ __forceinline__ float sum() const { return (a + b) + c; }
};
// column sums of part [2][R][C] in a fixed order: 16 channels x 64 rows at a time per workgroup, 8 loads in flight per thread
__global__ __launch_bounds__(1024) void ov_gn_param_kernel(const float* __restrict__ part, int64_t R, int C, float* __restrict__ dw,
                                                           float* __restrict__ db) {
    __shared__ float red[64][17];
    float* out = blockIdx.y ? db : dw;
    if (!out) return;
    const float* src = part + (blockIdx.y ? R * C : 0);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, c = blockIdx.x * 16 + tx;
    OvGnLong s;
    if (c < C) {
        int64_t r = ty;
        for (; r + 7 * 64 < R; r += 8 * 64) {
            float t[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) t[u] = src[(r + 64 * u) * C + c];
            s.add(((t[0] + t[4]) + (t[1] + t[5])) + ((t[2] + t[6]) + (t[3] + t[7])));
        }
        for (; r < R; r += 64) s.add(src[r * C + c]);
    }
    red[ty][tx] = s.sum();
    __syncthreads();
    if (ty < 8) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) t += red[ty * 8 + k][tx];
        red[ty * 8][tx] = t;                              // read by this thread only, until the barrier
    }
    __syncthreads();
    if (ty == 0 && c < C) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) t += red[k * 8][tx];
        out[c] = t;
    }
}

// ---------------------------------------------------------------- S > 1: tiles of rows x channels
// A workgroup takes a run of a sample's rows and a block of whole groups (all channels if they fit): 256 threads as TX pieces
// of 8 channels x TY rows, a thread's channels fixed, so that weight, bias and the per-channel sums stay in registers; channel
// sums meet in LDS, group sums are sums of channel sums (a piece may hold parts of several groups).
//   MODE 0: sums of the tile only      MODE 1: the output, from the sums of the sample's tiles
//   MODE 2: the tile is the whole sample; both in one launch, the second read from the cache
// Modes 0 and 1 read x (and dy) once each; mode 1 takes the tiles in the opposite order, so that what the last-level cache still
// holds of mode 0's reads is taken first.
struct OvGnTile {
    int gb, nblk;            // groups of a channel block, channel blocks
    int tx, ty;              // pieces of a block's row, rows at a time
    int chunks, rows;        // tiles along S, rows of one
    float* part;             // per tile and group, [N][chunks][groups].  Forward: float4 (mean, rest, M2, -).  Backward: float2 sums
    float* far;              // backward: sums of x - mean, the same order
};

struct OvGnPlace { int n, chunk, c0, cb, g0, ng, r0, r1; };
// rows of tile k
__device__ __forceinline__ int ov_gn_tile_rows(const OvGn& p, const OvGnTile& t, int k) { return min(t.rows, p.S - k * t.rows); }
// of these, the rows of thread row ty
__device__ __forceinline__ int ov_gn_thread_rows(const OvGnTile& t, int rows, int ty) { return (rows - ty + t.ty - 1) / t.ty; }
__device__ __forceinline__ OvGnPlace ov_gn_place(const OvGn& p, const OvGnTile& t, bool reverse) {
    OvGnPlace q;
    int id = reverse ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
    const int blk = id % t.nblk;
    id /= t.nblk;
    q.chunk = id % t.chunks;
    q.n = id / t.chunks;
    q.g0 = blk * t.gb;
    q.ng = min(t.gb, p.groups - q.g0);
    q.c0 = q.g0 * p.cg;
    q.cb = q.ng * p.cg;
    q.r0 = q.chunk * t.rows;
    q.r1 = q.r0 + ov_gn_tile_rows(p, t, q.chunk);
    return q;
}

// lanes of a wave that share one of ng groups of n terms: a power of two, all groups in one round of 256 threads if they fit
__device__ __forceinline__ int ov_gn_lanes(int ng, int n) {
    int lg = 64;
    while (lg > 1 && (lg > n || lg * ng > 256)) lg >>= 1;
    return lg;
}

__device__ __forceinline__ float ov_gn_lanes_sum(float v, int lg) {
    for (int o = lg / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Joins n parts of a group, part k = (mean, rest, M2) of cnt(k) values, by Chan's formula; lanes l of lg share them out.  Means are
// taken relative to the first part's, so that their differences are of the spread's size and the rests count.  (Not relative to a
// single value: one that stands alone is up to sqrt(n) spreads away from the others, and the differences would be rounded at that size;
// the mean of a part that holds it is at most 45 away in any tile.)
template <typename P, typename CNT>
__device__ __forceinline__ float3 ov_gn_join(int n, int l, int lg, float total, P&& part, CNT&& cnt) {
    const float3 first = part(0);
    const float m = first.x + first.y;
    float a = 0.f, m2 = 0.f;
    for (int k = l; k < n; k += lg) {
        const float3 v = part(k);
        a += ((v.x - m) + v.y) * cnt(k);
    }
    a = ov_gn_lanes_sum(a, lg) / total;
    for (int k = l; k < n; k += lg) {
        const float3 v = part(k);
        const float d = ((v.x - m) + v.y) - a;
        m2 += v.z + d * (d * cnt(k));                    // a part of no values: d may be anything
    }
    float3 o;
    o.z = ov_gn_lanes_sum(m2, lg);
    o.x = ov_gn_two(m, a, &o.y);
    return o;
}

// a sample's statistics from its tiles' -> gs = (mean, rstd), rest.  Up to 8 tiles a lane are read at once, so that their latency
// counts once.
__device__ __forceinline__ void ov_gn_gather_fwd(const OvGn& p, const OvGnTile& t, const OvGnPlace& q, float2* gs, float* rest) {
    constexpr int NP = 8;
    const int lg = ov_gn_lanes(q.ng, t.chunks), l = threadIdx.x % lg;
    const float total = (float)((int64_t)p.S * p.cg);
    auto count = [&](int k) { return (float)ov_gn_tile_rows(p, t, k) * (float)p.cg; };
    for (int g = threadIdx.x / lg; g < q.ng; g += 256 / lg) {
        const float4* src = reinterpret_cast<const float4*>(t.part) + ((int64_t)q.n * t.chunks * p.groups + q.g0 + g);
        float3 o;
        if (t.chunks <= NP * lg) {                       // ov_gn_join on registers
            float4 v[NP];
#pragma unroll
            for (int i = 0; i < NP; ++i) v[i] = src[(int64_t)min(l + i * lg, t.chunks - 1) * p.groups];
            const float m = __shfl(v[0].x + v[0].y, ov_lane() - l, 64);
            float a = 0.f, m2 = 0.f;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                v[i].w = l + i * lg < t.chunks ? count(l + i * lg) : 0.f;
                v[i].x = (v[i].x - m) + v[i].y;
                a += v[i].x * v[i].w;
            }
            a = ov_gn_lanes_sum(a, lg) / total;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const float d = v[i].x - a;
                if (l + i * lg < t.chunks) m2 += v[i].z + d * (d * v[i].w);
            }
            o.z = ov_gn_lanes_sum(m2, lg);
            o.x = ov_gn_two(m, a, &o.y);
        } else {
            o = ov_gn_join(t.chunks, l, lg, total, [&](int k) { const float4 v = src[(int64_t)k * p.groups]; return make_float3(v.x, v.y, v.z); }, count);
        }
        if (l == 0) { gs[g] = make_float2(o.x, 1.f / sqrtf(o.z / total + p.eps)); rest[g] = o.y; }
    }
    __syncthreads();
}

// backward: the tiles' sums of (dv gamma, dv gamma xhat) / count -> gs
__device__ __forceinline__ void ov_gn_gather_bwd(const OvGn& p, const OvGnTile& t, const OvGnPlace& q, float2* gs) {
    const int lg = ov_gn_lanes(q.ng, t.chunks), l = threadIdx.x % lg;
    const float total = (float)((int64_t)p.S * p.cg);
    for (int g = threadIdx.x / lg; g < q.ng; g += 256 / lg) {
        const float2* src = reinterpret_cast<const float2*>(t.part) + ((int64_t)q.n * t.chunks * p.groups + q.g0 + g);
        float a = 0.f, b = 0.f;
        for (int k = l; k < t.chunks; k += lg) {
            const float2 v = src[(int64_t)k * p.groups];
            a += v.x;
            b += v.y;
        }
        a = ov_gn_lanes_sum(a, lg);
        b = ov_gn_lanes_sum(b, lg);
        if (l == 0) gs[g] = make_float2(a / total, b / total);
    }
    __syncthreads();
}

#define OV_GN_MAX_CB(E) (256 * (E))

template <typename T, int MODE, bool LIGHT>
__global__ __launch_bounds__(256) void ov_gn_tile_fwd_kernel(const T* __restrict__ x, const OvGn p_, const OvGnTile t, T* __restrict__ y,
                                                             float* __restrict__ mean, float* __restrict__ rstd) {
    const OvGn p = ov_gn_light<LIGHT>(p_);
    constexpr int E = OvGnPiece<T>::N, RB = 16 / (int)sizeof(T);
    __shared__ float2 cs[OV_GN_MAX_CB(E)];               // (rest, M2) of a thread's rows of a channel, of a channel; then (mu, r) of a group
    __shared__ float ks[OV_GN_MAX_CB(E)];                // the mean that belongs to it; then the group's rest
    const OvGnPlace q = ov_gn_place(p, t, MODE == 1);
    const int tid = threadIdx.x, ty = tid / t.tx, tx = tid - ty * t.tx;
    const bool on = ty < t.ty;
    const int cnt = on ? min(q.cb - tx * E, E) : 0;      // <= 0: no channel of the block
    const int64_t row0 = (int64_t)q.n * p.S, col = q.c0 + tx * E, all = (int64_t)p.N * p.S * p.C;
    constexpr int RA = 8;
    OvGnPiece<T> raw[RA];
    auto fetch = [&](int r) {
#pragma unroll
        for (int i = 0; i < RA; ++i) ov_gn_raw<T>(x, all, (row0 + min(r + i * t.ty, q.r1 - 1)) * p.C + col, raw[i]);
    };
    if (MODE != 1) {
        // sums relative to the first value that the thread meets of a channel
        float k0[E], m[E], m2[E];
#pragma unroll
        for (int k = 0; k < E; ++k) k0[k] = m[k] = m2[k] = 0.f;
        int have = 0;
        if (cnt > 0)
            for (int r = q.r0 + ty; r < q.r1; r += RB * t.ty) {
                OvGnPiece<T> v[RB];
                const int nb = min(ov_gn_thread_rows(t, q.r1 - r, 0), RB);
#pragma unroll
                for (int i = 0; i < RB; ++i) ov_gn_raw<T>(x, all, (row0 + min(r + i * t.ty, q.r1 - 1)) * p.C + col, v[i]);
                if ((row0 + min(r + (RB - 1) * t.ty, q.r1 - 1)) * p.C + col > all - E) {      // the tensor's last pieces
#pragma unroll
                    for (int i = 0; i < RB; ++i) {
                        const int64_t o = (row0 + min(r + i * t.ty, q.r1 - 1)) * p.C + col;
                        float f[E];
                        ov_gn_floats<T>(x, all, o, v[i], f);
#pragma unroll
                        for (int k = 0; k < E; ++k) v[i].e[k] = ov_from_f<T>(f[k]);
                    }
                }
                if (have == 0)
#pragma unroll
                    for (int k = 0; k < E; ++k) k0[k] = ov_to_f<T>(v[0].e[k]);
                // mean and second moment of these rows, then Chan's combination with the ones before
                const float fb = (float)nb, ft = (float)(have + nb), wgt = fb / ft, cross = (float)have * wgt, rb = 1.f / fb;
                auto merge = [&](auto whole) {
#pragma unroll
                    for (int k = 0; k < E; ++k) {
                        float s = 0.f, s2 = 0.f, u[RB];
#pragma unroll
                        for (int i = 0; i < RB; ++i) {
                            u[i] = ov_to_f<T>(v[i].e[k]) - k0[k];
                            s += whole || i < nb ? u[i] : 0.f;
                        }
                        const float mb = s * rb;
#pragma unroll
                        for (int i = 0; i < RB; ++i) {
                            const float d = u[i] - mb;
                            s2 += whole || i < nb ? d * d : 0.f;
                        }
                        const float d = mb - m[k];
                        m[k] += d * wgt;
                        m2[k] += s2 + d * (d * cross);         // no rows before: d is the mean itself, its square may pass the type
                    }
                };
                if (nb == RB) merge(std::true_type{});
                else merge(std::false_type{});
                have += nb;
            }
        if (on)
#pragma unroll
            for (int k = 0; k < E; ++k) {
                const int at = ty * t.tx * E + tx * E + k;
                cs[at] = make_float2(m[k], m2[k]);
                ks[at] = k0[k];
            }
        __syncthreads();
        // a channel's over the ty's (their row counts follow from ty), into the place of ty = 0: the lanes that read a column write it
        const int rows = q.r1 - q.r0, lc = ov_gn_lanes(q.cb, t.ty);
        for (int c = tid / lc; c < q.cb; c += 256 / lc) {
            const float3 o = ov_gn_join(t.ty, tid % lc, lc, (float)rows,
                                        [&](int k) { const int at = k * t.tx * E + c; return make_float3(ks[at], cs[at].x, cs[at].y); },
                                        [&](int k) { return (float)ov_gn_thread_rows(t, rows, k); });
            if (tid % lc == 0) {
                ks[c] = o.x;
                cs[c] = make_float2(o.y, o.z);
            }
        }
        __syncthreads();
        // a group's over its channels, into the place of channel g, whose own group has been read in this round or before
        const int lg = ov_gn_lanes(q.ng, p.cg), l = tid % lg;
        const float total = (float)((int64_t)rows * p.cg);
        for (int g0 = 0; g0 < q.ng; g0 += 256 / lg) {
            const int g = g0 + tid / lg;
            float3 o = make_float3(0.f, 0.f, 0.f);
            if (g < q.ng)
                o = ov_gn_join(p.cg, l, lg, total, [&](int k) { const int c = g * p.cg + k; return make_float3(ks[c], cs[c].x, cs[c].y); },
                               [&](int) { return (float)rows; });
            if (MODE == 0) {
                if (g < q.ng && l == 0)
                    reinterpret_cast<float4*>(t.part)[((int64_t)q.n * t.chunks + q.chunk) * p.groups + q.g0 + g] = make_float4(o.x, o.y, o.z, 0.f);
            } else {
                __syncthreads();
                if (g < q.ng && l == 0) {
                    cs[g] = make_float2(o.x, 1.f / sqrtf(o.z / total + p.eps));
                    ks[g] = o.y;
                }
            }
        }
        if (MODE == 0) return;
        __syncthreads();
    } else {
        if (cnt > 0) fetch(q.r0 + ty);                    // under the gather's latency
        ov_gn_gather_fwd(p, t, q, cs, ks);
    }
    if (q.chunk == 0)
        for (int g = tid; g < q.ng; g += 256) {
            mean[(int64_t)q.n * p.groups + q.g0 + g] = cs[g].x;
            rstd[(int64_t)q.n * p.groups + q.g0 + g] = cs[g].y;
        }
    if (cnt <= 0) return;
    if (MODE == 2) fetch(q.r0 + ty);
    float mu[E], rw[E], b[E];
    ov_gn_params<E>(p.w, p.wtype, q.c0 + tx * E, cnt, 1.f, rw);
    ov_gn_params<E>(p.b, p.wtype, q.c0 + tx * E, cnt, 0.f, b);
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const int g = min(tx * E + k, q.cb - 1) / p.cg;
        const float2 v = cs[g];
        mu[k] = v.x;
        rw[k] *= v.y;
        b[k] -= ks[g] * rw[k];                            // (x - mu - rest) rw + b
    }
    for (int r = q.r0 + ty; r < q.r1; r += RA * t.ty) {
        if (r > q.r0 + ty) fetch(r);
#pragma unroll
        for (int i = 0; i < RA; ++i) {
            const int rr = r + i * t.ty;
            if (rr >= q.r1) break;
            float v[E];
            ov_gn_floats<T>(x, all, (row0 + rr) * p.C + col, raw[i], v);
#pragma unroll
            for (int k = 0; k < E; ++k) v[k] = (v[k] - mu[k]) * rw[k] + b[k];
            ov_act<E>(v, p.act);
            ov_gn_drop<E>(p, row0 + rr, q.c0 + tx * E, v);
            ov_gn_store<T>(y + (row0 + rr) * p.C + col, cnt, v);
        }
    }
}

// chan: [2][N chunks][C]: the tiles' sums of dv xhat, then of dv, per channel.
// Rests (ov_gn_far) of a float32 x: MODE 3, in front of the others, takes the sums of x - mean of the tiles that hold such a group and
// ends at once where there is none (2.5 us: 4 x 1024 x 320 27 -> 29.5; 53 where every group has one).  A rest enters v through
// beta, the sums and dx after their loops: those are the same with and without it.  A 16-bit x goes without (64 x 16 x 320 in bf16
// would be 18 -> 21 us): the rounding of its values, 2^-12 |x| at least, has moved the mean of n of them by 2^-12 |mean| / sqrt(n), more
// than the 2^-24 |mean| in question up to n = 2^24.
template <typename T, int MODE, bool LIGHT>
__global__ __launch_bounds__(256) void ov_gn_tile_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const OvGn p_, const OvGnTile t,
                                                             const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx,
                                                             float* __restrict__ chan) {
    const OvGn p = ov_gn_light<LIGHT>(p_);
    constexpr int E = OvGnPiece<T>::N, RA = 8 / (int)sizeof(T);
    __shared__ float2 cs[OV_GN_MAX_CB(E)];
    __shared__ float2 st[OV_GN_MAX_CB(E)];
    const OvGnPlace q = ov_gn_place(p, t, MODE == 1);
    const int tid = threadIdx.x, ty = tid / t.tx, tx = tid - ty * t.tx;
    const bool on = ty < t.ty;
    const int cnt = on ? min(q.cb - tx * E, E) : 0;
    const int64_t row0 = (int64_t)q.n * p.S, col = q.c0 + tx * E, total = (int64_t)p.N * p.S * p.C;
    // x - mu, then v = (x - mu) (r gamma) + beta
    float mu[E], rw[E], b[E];
    OvGnPiece<T> rx[RA], rd[RA];
    auto fetch = [&](int r) {
#pragma unroll
        for (int i = 0; i < RA; ++i) {
            const int64_t o = (row0 + min(r + i * t.ty, q.r1 - 1)) * p.C + col;
            ov_gn_raw<T>(x, total, o, rx[i]);
            ov_gn_raw<T>(dy, total, o, rd[i]);
        }
    };
    auto group = [&](int k) { return min(tx * E + k, q.cb - 1) / p.cg; };
    if (MODE == 3) {
        bool any = false;
        for (int g = ov_lane(); g < q.ng; g += 64) any |= ov_gn_far(mean[(int64_t)q.n * p.groups + q.g0 + g], rstd[(int64_t)q.n * p.groups + q.g0 + g]);
        if (!__any(any)) return;                         // the same in every wave of the workgroup
    }
    bool far = false;                                    // one of the thread's groups
    if (cnt > 0) {
        ov_gn_params<E>(p.w, p.wtype, q.c0 + tx * E, cnt, 1.f, rw);
        ov_gn_params<E>(p.b, p.wtype, q.c0 + tx * E, cnt, 0.f, b);
#pragma unroll
        for (int k = 0; k < E; ++k) {
            const int64_t gi = (int64_t)q.n * p.groups + q.g0 + group(k);
            mu[k] = mean[gi];
            rw[k] *= rstd[gi];
            far |= sizeof(T) == 4 && ov_gn_far(mu[k], rstd[gi]);
        }
    }
    if (MODE == 3) {
        float d[E];
#pragma unroll
        for (int k = 0; k < E; ++k) d[k] = 0.f;
        if (cnt > 0)
            for (int r = q.r0 + ty; r < q.r1; r += RA * t.ty) {
#pragma unroll
                for (int i = 0; i < RA; ++i) ov_gn_raw<T>(x, total, (row0 + min(r + i * t.ty, q.r1 - 1)) * p.C + col, rx[i]);
#pragma unroll
                for (int i = 0; i < RA; ++i) {
                    if (r + i * t.ty >= q.r1) break;
                    float f[E];
                    ov_gn_floats<T>(x, total, (row0 + r + i * t.ty) * p.C + col, rx[i], f);
#pragma unroll
                    for (int k = 0; k < E; ++k) d[k] += f[k] - mu[k];
                }
            }
        if (on)
#pragma unroll
            for (int k = 0; k < E; ++k) cs[ty * t.tx * E + tx * E + k].x = d[k];
        __syncthreads();
        for (int c = tid; c < q.cb; c += 256) {
            float a = 0.f;
            for (int k = 0; k < t.ty; ++k) a += cs[k * t.tx * E + c].x;
            st[c].x = a;
        }
        __syncthreads();
        const int lg = ov_gn_lanes(q.ng, p.cg), l = tid % lg;
        for (int g = tid / lg; g < q.ng; g += 256 / lg) {
            float a = 0.f;
            for (int k = l; k < p.cg; k += lg) a += st[g * p.cg + k].x;
            a = ov_gn_lanes_sum(a, lg);
            if (l == 0) t.far[((int64_t)q.n * t.chunks + q.chunk) * p.groups + q.g0 + g] = a;
        }
        return;
    }
    // the rests of the thread's channels; mode 3 has written the sums of every such group
    auto rests = [&](float (&d)[E]) {
#pragma unroll
        for (int k = 0; k < E; ++k) {
            d[k] = k > 0 ? d[max(k - 1, 0)] : 0.f;
            if (k > 0 && group(k) == group(k - 1)) continue;
            const int64_t gi = (int64_t)q.n * p.groups + q.g0 + group(k);
            float a = 0.f;
            if (ov_gn_far(mean[gi], rstd[gi])) {
                const float* src = t.far + ((int64_t)q.n * t.chunks * p.groups + q.g0 + group(k));
#pragma unroll 8
                for (int i = 0; i < t.chunks; ++i) a += src[(int64_t)i * p.groups];
            }
            d[k] = a / (float)((int64_t)p.S * p.cg);
        }
    };
    if (far) {
        float d[E];
        rests(d);
#pragma unroll
        for (int k = 0; k < E; ++k) b[k] -= d[k] * rw[k];
    }
    auto grad = [&](int64_t row, const OvGnPiece<T>& vx, const OvGnPiece<T>& vd, float (&xm)[E], float (&dv)[E]) {
        float d[E];
        ov_gn_floats<T>(x, total, row * p.C + col, vx, xm);
        ov_gn_floats<T>(dy, total, row * p.C + col, vd, d);
#pragma unroll
        for (int k = 0; k < E; ++k) {
            xm[k] -= mu[k];
            dv[k] = xm[k] * rw[k] + b[k];
        }
        ov_gn_dv<E>(p, row, q.c0 + tx * E, d, dv);
    };
    if (MODE != 1) {
        float sb[E], sw[E];
#pragma unroll
        for (int k = 0; k < E; ++k) sb[k] = sw[k] = 0.f;
        if (cnt > 0) {
            for (int r = q.r0 + ty; r < q.r1; r += RA * t.ty) {
                fetch(r);
#pragma unroll
                for (int i = 0; i < RA; ++i) {
                    if (r + i * t.ty >= q.r1) break;
                    float xm[E], dv[E];
                    grad(row0 + r + i * t.ty, rx[i], rd[i], xm, dv);
#pragma unroll
                    for (int k = 0; k < E; ++k) {
                        sb[k] += dv[k];
                        sw[k] += dv[k] * xm[k];
                    }
                }
            }
            if (far) {
                float d[E];
                rests(d);
#pragma unroll
                for (int k = 0; k < E; ++k) sw[k] -= d[k] * sb[k];
            }
#pragma unroll
            for (int k = 0; k < E; ++k) sw[k] *= rstd[(int64_t)q.n * p.groups + q.g0 + group(k)];
        }
        if (on)
#pragma unroll
            for (int k = 0; k < E; ++k) cs[ty * t.tx * E + tx * E + k] = make_float2(sb[k], sw[k]);
        __syncthreads();
        const int64_t R = (int64_t)p.N * t.chunks, ro = (int64_t)q.n * t.chunks + q.chunk;
        for (int c = tid; c < q.cb; c += 256) {
            float a = 0.f, e = 0.f;
            for (int k = 0; k < t.ty; ++k) {
                const float2 v = cs[k * t.tx * E + c];
                a += v.x;
                e += v.y;
            }
            if (chan) {
                chan[ro * p.C + q.c0 + c] = e;
                chan[(R + ro) * p.C + q.c0 + c] = a;
            }
            const float wc = ov_gn_param(p.w, p.wtype, q.c0 + c, 1.f);
            st[c] = make_float2(a * wc, e * wc);
        }
        __syncthreads();
        const int lg = ov_gn_lanes(q.ng, p.cg), l = tid % lg;
        for (int g = tid / lg; g < q.ng; g += 256 / lg) {
            float a = 0.f, e = 0.f;
            for (int k = l; k < p.cg; k += lg) {
                const float2 v = st[g * p.cg + k];
                a += v.x;
                e += v.y;
            }
            a = ov_gn_lanes_sum(a, lg);
            e = ov_gn_lanes_sum(e, lg);
            if (l != 0) continue;
            if (MODE == 0) reinterpret_cast<float2*>(t.part)[ro * p.groups + q.g0 + g] = make_float2(a, e);
            else {
                const float total = (float)((int64_t)p.S * p.cg);
                cs[g] = make_float2(a / total, e / total);
            }
        }
        if (MODE == 0) return;
        __syncthreads();
    } else {
        ov_gn_gather_bwd(p, t, q, cs);
    }
    if (cnt <= 0) return;
    // dx = r (dv gamma - s1 - xhat s2) = dv (r gamma) - r s1 - (x - mu - rest) r^2 s2
    float k1[E], k2[E];
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const float2 v = cs[group(k)];
        const float rs = rstd[(int64_t)q.n * p.groups + q.g0 + group(k)];
        k1[k] = rs * v.x;
        k2[k] = rs * rs * v.y;
    }
    if (far) {
        float d[E];
        rests(d);
#pragma unroll
        for (int k = 0; k < E; ++k) k1[k] -= d[k] * k2[k];
    }
    for (int r = q.r0 + ty; r < q.r1; r += RA * t.ty) {
        fetch(r);
#pragma unroll
        for (int i = 0; i < RA; ++i) {
            const int rr = r + i * t.ty;
            if (rr >= q.r1) break;
            float xm[E], dv[E];
            grad(row0 + rr, rx[i], rd[i], xm, dv);
#pragma unroll
            for (int k = 0; k < E; ++k) dv[k] = dv[k] * rw[k] - k1[k] - xm[k] * k2[k];
            ov_gn_store<T>(dx + (row0 + rr) * p.C + col, cnt, dv);
        }
    }
}

// ---------------------------------------------------------------- any shape: groups too wide for the forms above
// (more than 2048 channels over several rows, more than 16384 in one), and tensors of less than 8 elements.  One workgroup per
// (sample, group), everything re-read from the cache, however long the sample: 4 x 1024 x 4096 bf16 of one group 4.9 ms forward and 7.4
// backward where 0.014 and 0.020 would be the memory's time.
template <typename T>
__global__ __launch_bounds__(1024) void ov_gn_any_fwd_kernel(const T* __restrict__ x, const OvGn p, T* __restrict__ y, float* __restrict__ mean,
                                                             float* __restrict__ rstd) {
    __shared__ float red[32];
    const int64_t n = blockIdx.x / p.groups;
    const int g = blockIdx.x % p.groups;
    const float cnt = (float)((int64_t)p.S * p.cg);
    const int64_t base = n * p.S * p.C + (int64_t)g * p.cg;
    OvGnLong s, s2, left;
    for (int r = 0; r < p.S; ++r)
        for (int c = threadIdx.x; c < p.cg; c += 1024) s.add(ov_to_f<T>(x[base + (int64_t)r * p.C + c]));
    const float mu = ov_block_sum(s.sum(), red) / cnt;
    for (int r = 0; r < p.S; ++r)
        for (int c = threadIdx.x; c < p.cg; c += 1024) {
            const float d = ov_to_f<T>(x[base + (int64_t)r * p.C + c]) - mu;
            s2.add(d * d);
            left.add(d);
        }
    const float2 sl = ov_gn_sum2<1024>(s2.sum(), left.sum(), red);
    const float rest = sl.y / cnt, rs = 1.f / sqrtf(ov_gn_var(sl.x / cnt, rest) + p.eps);
    for (int r = 0; r < p.S; ++r)
        for (int c = threadIdx.x; c < p.cg; c += 1024) {
            const int64_t o = base + (int64_t)r * p.C + c;
            const int ch = g * p.cg + c;
            float v[1] = {((ov_to_f<T>(x[o]) - mu) - rest) * rs * ov_gn_param(p.w, p.wtype, ch, 1.f) + ov_gn_param(p.b, p.wtype, ch, 0.f)};
            ov_act<1>(v, p.act);
            ov_gn_drop<1>(p, n * p.S + r, ch, v);
            y[o] = ov_from_f<T>(v[0]);
        }
    if (threadIdx.x == 0) { mean[blockIdx.x] = mu + rest; rstd[blockIdx.x] = rs; }
}

template <typename T>
__device__ __forceinline__ float ov_gn_any_dv(const OvGn& p, const T* x, const T* dy, int64_t row, int c, float mu, float rest, float r, float* xhat) {
    const int64_t o = row * p.C + c;
    *xhat = ((ov_to_f<T>(x[o]) - mu) - rest) * r;
    float d[1] = {ov_to_f<T>(dy[o])}, a[1] = {*xhat * ov_gn_param(p.w, p.wtype, c, 1.f) + ov_gn_param(p.b, p.wtype, c, 0.f)};
    ov_gn_dv<1>(p, row, c, d, a);
    return a[0];
}

// rests [N][groups]: what the parameters' kernel below takes off as well
template <typename T>
__global__ __launch_bounds__(1024) void ov_gn_any_dx_kernel(const T* __restrict__ dy, const T* __restrict__ x, const OvGn p,
                                                            const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx,
                                                            float* __restrict__ rests) {
    __shared__ float red[32];
    const int64_t n = blockIdx.x / p.groups;
    const int g = blockIdx.x % p.groups;
    const float cnt = (float)((int64_t)p.S * p.cg);
    const float mu = mean[blockIdx.x], rs = rstd[blockIdx.x];
    float rest = 0.f;
    if (ov_gn_far(mu, rs)) {
        OvGnLong left;
        for (int r = 0; r < p.S; ++r)
            for (int c = g * p.cg + threadIdx.x; c < (g + 1) * p.cg; c += 1024) left.add(ov_to_f<T>(x[(n * p.S + r) * p.C + c]) - mu);
        rest = ov_block_sum(left.sum(), red) / cnt;
    }
    if (threadIdx.x == 0) rests[blockIdx.x] = rest;
    float xh;
    OvGnLong l1, l2;
    for (int r = 0; r < p.S; ++r)
        for (int c = g * p.cg + threadIdx.x; c < (g + 1) * p.cg; c += 1024) {
            const float e = ov_gn_any_dv(p, x, dy, n * p.S + r, c, mu, rest, rs, &xh) * ov_gn_param(p.w, p.wtype, c, 1.f);
            l1.add(e);
            l2.add(e * xh);
        }
    const float2 sg = ov_gn_sum2<1024>(l1.sum(), l2.sum(), red);
    const float s1 = sg.x / cnt, s2 = sg.y / cnt;
    for (int r = 0; r < p.S; ++r)
        for (int c = g * p.cg + threadIdx.x; c < (g + 1) * p.cg; c += 1024) {
            const float e = ov_gn_any_dv(p, x, dy, n * p.S + r, c, mu, rest, rs, &xh) * ov_gn_param(p.w, p.wtype, c, 1.f);
            dx[(n * p.S + r) * p.C + c] = ov_from_f<T>(rs * (e - s1 - xh * s2));
        }
}

// sums over the rows for 64 channels: a wave's lanes along the channels, 16 waves along the rows
template <typename T>
__global__ __launch_bounds__(1024) void ov_gn_any_param_kernel(const T* __restrict__ dy, const T* __restrict__ x, const OvGn p,
                                                               const float* __restrict__ mean, const float* __restrict__ rstd,
                                                               const float* __restrict__ rests, float* __restrict__ dw, float* __restrict__ db) {
    __shared__ float2 red[16][64];
    const int lane = ov_lane(), wave = ov_wave_id(), c = blockIdx.x * 64 + lane;
    OvGnLong sw, sb;
    if (c < p.C)
        for (int64_t row = wave; row < (int64_t)p.N * p.S; row += 16) {
            const int64_t k = row / p.S * p.groups + c / p.cg;
            float xh;
            const float dv = ov_gn_any_dv(p, x, dy, row, c, mean[k], rests[k], rstd[k], &xh);
            sw.add(dv * xh);
            sb.add(dv);
        }
    float2 s = make_float2(sw.sum(), sb.sum());
    red[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < p.C) {
        for (int k = 1; k < 16; ++k) { s.x += red[k][lane].x; s.y += red[k][lane].y; }
        if (dw) dw[c] = s.x;
        if (db) db[c] = s.y;
    }
}

#define OV_GN_MOST (INT32_MAX - 65536)                    // indexes run past a size by up to a tile

static int ov_gn_check(const char* what, int32_t dtype, int32_t N, int32_t S, int32_t C, int32_t groups, const void* w, const void* b, int32_t wdtype,
                       float eps, int32_t act, float drop, uint64_t seed, uint64_t offset, OvGn* p) {
    if (N < 0 || S < 0 || C < 0 || std::max({N, S, C}) > OV_GN_MOST || groups < 1 || C % groups || (C > 0 && C < groups)) {
        ontovae_set_error("%s: N = %d, S = %d, C = %d, groups = %d (groups must divide C)", what, N, S, C, groups);
        return ONTOVAE_EINVAL;
    }
    if (dtype < ONTOVAE_F32 || dtype > ONTOVAE_F16 || wdtype < ONTOVAE_F32 || wdtype > ONTOVAE_F16) {
        ontovae_set_error("%s: unknown element type %d / %d", what, dtype, wdtype);
        return ONTOVAE_EINVAL;
    }
    if (act < ONTOVAE_ACT_NONE || act > ONTOVAE_ACT_GELU) { ontovae_set_error("%s: unknown activation %d", what, act); return ONTOVAE_EINVAL; }
    if (!(eps >= 0.f)) { ontovae_set_error("%s: eps = %g", what, (double)eps); return ONTOVAE_EINVAL; }
    if (ov_drop_from(drop, seed, offset, &p->drop)) { ontovae_set_error("%s: drop = %g outside [0, 1]", what, (double)drop); return ONTOVAE_EINVAL; }
    p->N = N; p->S = S; p->C = C; p->groups = groups; p->cg = C / groups;
    p->w = w; p->b = b; p->wtype = wdtype; p->eps = eps; p->act = act;
    return ONTOVAE_OK;
}

// ---------------------------------------------------------------- host
enum { OV_GN_ROW, OV_GN_TILE, OV_GN_TILE1, OV_GN_ANY };
struct OvGnPlan {
    int form;
    int lpg, nv, RS, wgs;    // OV_GN_ROW
    OvGnTile t;              // OV_GN_TILE (two launches), OV_GN_TILE1 (one)
    int64_t part_floats, far_floats, chan_floats, chan_rows;
};
static int64_t ov_gn_up(int64_t floats) { return (floats + 63) / 64 * 64; }

static OvGnPlan ov_gn_plan(int dtype, int N, int S, int C, int groups, bool backward) {
    OvGnPlan q{};
    const int E = 8, cg = C / groups;
    const int pieces = (cg + E - 1) / E;
    if ((int64_t)N * S * C < E) {                         // not one piece
        q.form = OV_GN_ANY;
        q.far_floats = backward ? (int64_t)N * groups : 0;
        return q;
    }
    if (S == 1 && pieces <= 2048) {
        q.form = OV_GN_ROW;
        if (pieces <= 64) {
            q.nv = 1;
            q.lpg = 8;
            while (q.lpg < pieces) q.lpg *= 2;
        } else {
            q.lpg = pieces <= 128 ? 64 : pieces <= 512 ? 256 : 1024;
            q.nv = pieces > 512 && pieces <= 1024 ? 1 : 2;        // two pieces of 1024 threads spill a few registers backward
        }
        // enough slots for four workgroups of 256 threads per CU.  Each row of gradient sums (a workgroup's where whole samples
        // fit it, else a slot's) is written and read once more: at most one to 8 samples
        const int64_t per = (int64_t)groups * q.lpg;          // threads of a sample, up to 2^34
        q.wgs = q.lpg < 256 && per <= 128 && 256 % per == 0 ? 256 / (int)per : 1;
        const int64_t want = std::max<int64_t>(262144 / per, 1);
        const int64_t most = std::max<int64_t>(((int64_t)N + 7) / 8, std::min<int64_t>(N, 65536 / std::min<int64_t>(per * q.wgs, 65536))) * q.wgs;
        q.RS = (int)std::min<int64_t>(want, backward ? std::min<int64_t>(most, N) : N);
        q.chan_rows = q.wgs > 1 ? (q.RS + q.wgs - 1) / q.wgs : q.RS;
        q.chan_floats = backward ? 2 * q.chan_rows * C : 0;
        return q;
    }
    const int max_cb = 256 * E;
    if (S > 1 && cg <= max_cb) {
        OvGnTile& t = q.t;
        t.gb = std::min(groups, max_cb / cg);
        t.nblk = (groups + t.gb - 1) / t.gb;
        t.gb = (groups + t.nblk - 1) / t.nblk;
        t.nblk = (groups + t.gb - 1) / t.gb;
        t.tx = (t.gb * cg + E - 1) / E;
        t.ty = std::min(256 / t.tx, S);
        const int64_t bytes = (int64_t)S * t.gb * cg * (dtype == ONTOVAE_F32 ? 4 : 2);
        const int64_t wg = (int64_t)N * t.nblk;
        t.chunks = 1;
        t.rows = S;
        q.form = OV_GN_TILE1;
        if (bytes > 65536) {
            q.form = OV_GN_TILE;
            // up to 768 workgroups, three a CU as the backward kernels' registers allow, of 16 rows a thread or more (32 x 4096 x 512 bf16
            // trained: 230 us; 5 % more with 1024, 11 % with 2048); where the samples are few, 256 of 4 rows or more, at most 128 a
            // sample (4 x 1024 x 320 float32 with gelu: 31 -> 18 us forward, 54 -> 30 backward; 60 x 3000 x 40 lost a fifth
            // with 900 workgroups of 4 rows, 1 x 4096 x 512 a fifth with 256 a sample)
            const int64_t few = std::min<int64_t>((S + t.ty * 4 - 1) / (t.ty * 4), std::min<int64_t>((256 + wg - 1) / wg, 128));
            const int64_t many = std::min<int64_t>((S + t.ty * 16 - 1) / (t.ty * 16), (768 + wg - 1) / wg);
            t.chunks = (int)std::max<int64_t>(1, std::max(few, many));
            t.rows = (S + t.chunks - 1) / t.chunks;
            t.chunks = (S + t.rows - 1) / t.rows;
            q.part_floats = (backward ? 2LL : 4LL) * N * t.chunks * groups;
        }
        q.far_floats = backward && dtype == ONTOVAE_F32 ? (int64_t)N * t.chunks * groups : 0;
        q.chan_rows = (int64_t)N * t.chunks;
        q.chan_floats = backward ? 2 * q.chan_rows * C : 0;
        return q;
    }
    q.form = OV_GN_ANY;
    q.far_floats = backward ? (int64_t)N * groups : 0;
    return q;
}

static int64_t ov_gn_ws(const OvGnPlan& q) { return (ov_gn_up(q.part_floats) + ov_gn_up(q.far_floats) + q.chan_floats) * 4; }

extern "C" int64_t ontovae_group_norm_act_workspace_bytes(int32_t dtype, int32_t N, int32_t S, int32_t C, int32_t groups, int32_t backward) {
    if (N < 1 || S < 1 || C < 1 || std::max({N, S, C}) > OV_GN_MOST || groups < 1 || C % groups || dtype < ONTOVAE_F32 || dtype > ONTOVAE_F16) return 0;
    return ov_gn_ws(ov_gn_plan(dtype, N, S, C, groups, backward != 0));
}

// sums: the gradients of weight or bias are wanted
static int ov_gn_ready(const char* what, const OvGn& p, const OvGnPlan& q, bool sums, const void* ws, int64_t bytes) {
    const int64_t need = ov_gn_ws(q);
    if (need > 0 && (!ws || bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255))) {
        ontovae_set_error("%s: workspace of %lld bytes, 256-B aligned, needed", what, (long long)need);
        return ONTOVAE_EINVAL;
    }
    const int threads = q.form == OV_GN_ROW ? std::max(q.lpg, 256) : q.form == OV_GN_ANY ? 1024 : 256;
    const int64_t wg = q.form == OV_GN_ROW ? ((int64_t)q.RS * p.groups * q.lpg + threads - 1) / threads
                       : q.form == OV_GN_ANY ? (int64_t)p.N * p.groups : (int64_t)p.N * q.t.chunks * q.t.nblk;
    const int64_t sum_wg = !sums ? 0 : q.form == OV_GN_ANY ? ((int64_t)p.C + 63) / 64 : ((int64_t)p.C + 15) / 16;
    if (!ov_ops_fits(wg, threads) || !ov_ops_fits(sum_wg, 1024)) {
        ontovae_set_error("%s: N = %d, S = %d, C = %d with %d groups are too many for one launch", what, p.N, p.S, p.C, p.groups);
        return ONTOVAE_EINVAL;
    }
    return ONTOVAE_OK;
}

#define OV_GN_ROW_SWITCH(GO)                                                                   \
    switch (q.lpg) {                                                                           \
        case 8: GO(8, 1); break;                                                               \
        case 16: GO(16, 1); break;                                                             \
        case 32: GO(32, 1); break;                                                             \
        case 64: if (q.nv == 1) { GO(64, 1); } else { GO(64, NVX); } break;                    \
        case 256: GO(256, NVX); break;                                                         \
        default: if (q.nv == 1) { GO(1024, 1); } else { GO(1024, NVX); } break;                                                         \
    }

template <typename T, bool LIGHT>
static void ov_gn_fwd_go(const void* x, const OvGn& p, OvGnPlan q, void* y, float* mean, float* rstd, void* ws, hipStream_t st) {
    const T* xt = static_cast<const T*>(x);
    T* yt = static_cast<T*>(y);
    q.t.part = static_cast<float*>(ws);
    constexpr int NVX = 16 / OvGnPiece<T>::N;
    if (q.form == OV_GN_ROW) {
#define OV_GO(L, V)                                                                                                                              \
    hipLaunchKernelGGL((ov_gn_row_fwd_kernel<T, L, V, LIGHT>), dim3((unsigned)(((int64_t)q.RS * p.groups * L + (L < 256 ? 256 : L) - 1) / (L < 256 ? 256 : L))), \
                       dim3(L < 256 ? 256 : L), 0, st, xt, p, q.RS, yt, mean, rstd)
        OV_GN_ROW_SWITCH(OV_GO)
#undef OV_GO
    } else if (q.form == OV_GN_ANY) {
        hipLaunchKernelGGL(ov_gn_any_fwd_kernel<T>, dim3((unsigned)((int64_t)p.N * p.groups)), dim3(1024), 0, st, xt, p, yt, mean, rstd);
    } else {
        const dim3 grid((unsigned)((int64_t)p.N * q.t.chunks * q.t.nblk));
        if (q.form == OV_GN_TILE1) hipLaunchKernelGGL((ov_gn_tile_fwd_kernel<T, 2, LIGHT>), grid, dim3(256), 0, st, xt, p, q.t, yt, mean, rstd);
        else {
            hipLaunchKernelGGL((ov_gn_tile_fwd_kernel<T, 0, true>), grid, dim3(256), 0, st, xt, p, q.t, yt, mean, rstd);
            hipLaunchKernelGGL((ov_gn_tile_fwd_kernel<T, 1, LIGHT>), grid, dim3(256), 0, st, xt, p, q.t, yt, mean, rstd);
        }
    }
}

static bool ov_gn_is_light(const OvGn& p) { return p.drop.t == 0 && p.act <= ONTOVAE_ACT_SILU; }
template <typename T>
static void ov_gn_fwd_launch(const void* x, const OvGn& p, const OvGnPlan& q, void* y, float* mean, float* rstd, void* ws, hipStream_t st) {
    if (ov_gn_is_light(p)) ov_gn_fwd_go<T, true>(x, p, q, y, mean, rstd, ws, st);
    else ov_gn_fwd_go<T, false>(x, p, q, y, mean, rstd, ws, st);
}

extern "C" int ontovae_group_norm_act(const void* x, int32_t dtype, int32_t N, int32_t S, int32_t C, int32_t groups, const void* weight,
                                      const void* bias, int32_t wdtype, float eps, int32_t act, float drop, uint64_t seed, uint64_t offset, void* y,
                                      float* mean, float* rstd, void* workspace, int64_t workspace_bytes, void* stream) {
    OvGn p;
    int rc = ov_gn_check("group_norm_act", dtype, N, S, C, groups, weight, bias, wdtype, eps, act, drop, seed, offset, &p);
    if (rc) return rc;
    if (N == 0 || S == 0 || C == 0) return ONTOVAE_OK;
    if (!x || !y || !mean || !rstd) { ontovae_set_error("group_norm_act: NULL argument"); return ONTOVAE_EINVAL; }
    const OvGnPlan q = ov_gn_plan(dtype, N, S, C, groups, false);
    if ((rc = ov_gn_ready("group_norm_act", p, q, false, workspace, workspace_bytes))) return rc;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    switch (dtype) {
        case ONTOVAE_F32: ov_gn_fwd_launch<float>(x, p, q, y, mean, rstd, workspace, st); break;
        case ONTOVAE_BF16: ov_gn_fwd_launch<ov_bf>(x, p, q, y, mean, rstd, workspace, st); break;
        default: ov_gn_fwd_launch<ov_hf>(x, p, q, y, mean, rstd, workspace, st); break;
    }
    OV_OPS_LAUNCH_CHECK("group_norm_act");
    return ONTOVAE_OK;
}

template <typename T, bool LIGHT>
static void ov_gn_bwd_go(const void* dy, const void* x, const OvGn& p, OvGnPlan q, const float* mean, const float* rstd, void* dx, float* dw,
                             float* db, void* ws, hipStream_t st) {
    const T* xt = static_cast<const T*>(x);
    const T* dt = static_cast<const T*>(dy);
    T* dxt = static_cast<T*>(dx);
    q.t.part = static_cast<float*>(ws);
    q.t.far = q.t.part + ov_gn_up(q.part_floats);
    float* chan = dw || db ? q.t.far + ov_gn_up(q.far_floats) : nullptr;
    constexpr int NVX = 16 / OvGnPiece<T>::N;
    if (q.form == OV_GN_ANY) {
        hipLaunchKernelGGL(ov_gn_any_dx_kernel<T>, dim3((unsigned)((int64_t)p.N * p.groups)), dim3(1024), 0, st, dt, xt, p, mean, rstd, dxt, q.t.far);
        if (dw || db) hipLaunchKernelGGL(ov_gn_any_param_kernel<T>, dim3((p.C + 63) / 64), dim3(1024), 0, st, dt, xt, p, mean, rstd, q.t.far, dw, db);
        return;
    }
    if (q.form == OV_GN_ROW) {
#define OV_GO(L, V)                                                                                                                              \
    hipLaunchKernelGGL((ov_gn_row_bwd_kernel<T, L, V, LIGHT>), dim3((unsigned)(((int64_t)q.RS * p.groups * L + (L < 256 ? 256 : L) - 1) / (L < 256 ? 256 : L))), \
                       dim3(L < 256 ? 256 : L), 0, st, dt, xt, p, q.RS, q.wgs, mean, rstd, dxt, chan)
        OV_GN_ROW_SWITCH(OV_GO)
#undef OV_GO
    } else {
        const dim3 grid((unsigned)((int64_t)p.N * q.t.chunks * q.t.nblk));
        if constexpr (sizeof(T) == 4) hipLaunchKernelGGL((ov_gn_tile_bwd_kernel<T, 3, true>), grid, dim3(256), 0, st, dt, xt, p, q.t, mean, rstd, dxt, chan);
        if (q.form == OV_GN_TILE1) hipLaunchKernelGGL((ov_gn_tile_bwd_kernel<T, 2, LIGHT>), grid, dim3(256), 0, st, dt, xt, p, q.t, mean, rstd, dxt, chan);
        else {
            hipLaunchKernelGGL((ov_gn_tile_bwd_kernel<T, 0, LIGHT>), grid, dim3(256), 0, st, dt, xt, p, q.t, mean, rstd, dxt, chan);
            hipLaunchKernelGGL((ov_gn_tile_bwd_kernel<T, 1, LIGHT>), grid, dim3(256), 0, st, dt, xt, p, q.t, mean, rstd, dxt, chan);
        }
    }
    if (chan) hipLaunchKernelGGL(ov_gn_param_kernel, dim3((p.C + 15) / 16, 2), dim3(1024), 0, st, chan, q.chan_rows, p.C, dw, db);
}

template <typename T>
static void ov_gn_bwd_launch(const void* dy, const void* x, const OvGn& p, const OvGnPlan& q, const float* mean, const float* rstd, void* dx, float* dw,
                             float* db, void* ws, hipStream_t st) {
    if (ov_gn_is_light(p)) ov_gn_bwd_go<T, true>(dy, x, p, q, mean, rstd, dx, dw, db, ws, st);
    else ov_gn_bwd_go<T, false>(dy, x, p, q, mean, rstd, dx, dw, db, ws, st);
}

__global__ __launch_bounds__(256) void ov_gn_zero_kernel(float* dw, float* db, int C) {
    for (int c = blockIdx.x * 256 + threadIdx.x; c < C; c += gridDim.x * 256) {
        if (dw) dw[c] = 0.f;
        if (db) db[c] = 0.f;
    }
}

extern "C" int ontovae_group_norm_act_backward(const void* dy, const void* x, int32_t dtype, int32_t N, int32_t S, int32_t C, int32_t groups,
                                               const void* weight, const void* bias, int32_t wdtype, const float* mean, const float* rstd,
                                               int32_t act, float drop, uint64_t seed, uint64_t offset, void* dx, float* dweight, float* dbias,
                                               void* workspace, int64_t workspace_bytes, void* stream) {
    OvGn p;
    int rc = ov_gn_check("group_norm_act_backward", dtype, N, S, C, groups, weight, bias, wdtype, 0.f, act, drop, seed, offset, &p);
    if (rc) return rc;
    if (C == 0) return ONTOVAE_OK;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (N == 0 || S == 0) {
        if (dweight || dbias) hipLaunchKernelGGL(ov_gn_zero_kernel, dim3(std::min((C + 255) / 256, 256)), dim3(256), 0, st, dweight, dbias, C);
        OV_OPS_LAUNCH_CHECK("group_norm_act_backward");
        return ONTOVAE_OK;
    }
    if (!dy || !x || !mean || !rstd || !dx) { ontovae_set_error("group_norm_act_backward: NULL argument"); return ONTOVAE_EINVAL; }
    const OvGnPlan q = ov_gn_plan(dtype, N, S, C, groups, true);
    if ((rc = ov_gn_ready("group_norm_act_backward", p, q, dweight || dbias, workspace, workspace_bytes))) return rc;
    switch (dtype) {
        case ONTOVAE_F32: ov_gn_bwd_launch<float>(dy, x, p, q, mean, rstd, dx, dweight, dbias, workspace, st); break;
        case ONTOVAE_BF16: ov_gn_bwd_launch<ov_bf>(dy, x, p, q, mean, rstd, dx, dweight, dbias, workspace, st); break;
        default: ov_gn_bwd_launch<ov_hf>(dy, x, p, q, mean, rstd, dx, dweight, dbias, workspace, st); break;
    }
    OV_OPS_LAUNCH_CHECK("group_norm_act_backward");
    return ONTOVAE_OK;
}

#endif

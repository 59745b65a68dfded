// Group norm with an activation and dropout in one operator, channels last: x [N, S, C], groups of C / groups channels.
//
//   per sample and group (S rows x C / groups channels): mu, biased var, r = 1 / sqrt(var + eps)
//   v = (x - mu) r gamma_c + beta_c,   y = D act(v),   D = keep / (1 - p) as in ontovae_dropout.h over the rows [N S, C]
// Backward: dv = dy D act'(v), dgamma_c = sum dv xhat, dbeta_c = sum dv, e = dv gamma,
//   dx = r (e - mean(e) - xhat mean(e xhat)), the means over the group.
// Statistics and every sum are held in 32 bits; the variance is the second moment about the mean (two passes over what is held
// or cached), so a large mean costs no digits.
#ifndef ONTOVAE_GROUPNORM_H
#define ONTOVAE_GROUPNORM_H

#include "ontovae_dropout.h"

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

__device__ __forceinline__ float ov_act(float v, int act) {
    if (act == ONTOVAE_ACT_RELU) return v > 0.f ? v : (v <= 0.f ? 0.f : v);          // NaN stays NaN
    if (act == ONTOVAE_ACT_SILU) return v / (1.f + __expf(-v));
    if (act == ONTOVAE_ACT_GELU) return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
    return v;
}

__device__ __forceinline__ float ov_act_grad(float v, int act) {
    if (act == ONTOVAE_ACT_RELU) return v > 0.f ? 1.f : (v <= 0.f ? 0.f : v);
    if (act == ONTOVAE_ACT_SILU) {
        const float s = 1.f / (1.f + __expf(-v));
        return s * (1.f + v * (1.f - s));
    }
    if (act == ONTOVAE_ACT_GELU)
        return 0.5f * (1.f + erff(v * 0.70710678118654752f)) + v * __expf(-0.5f * v * v) * 0.39894228040143268f;
    return 1.f;
}

__device__ __forceinline__ bool ov_gn_kept(const OvGn& p, int64_t row, int c) {
    if (p.drop.t == 0) return true;
    return ov_drop_kept(p.drop, ov_drop_draw(p.drop, (uint64_t)row * ((p.C + 7) / 8) + (c >> 3)), c & 7);
}

// one workgroup per (sample, group)
template <typename T>
__global__ __launch_bounds__(256) void ov_gn_fwd_kernel(const T* __restrict__ x, const OvGn p, T* __restrict__ y, float* __restrict__ mean,
                                                        float* __restrict__ rstd) {
    __shared__ float red[16];
    const int64_t n = blockIdx.x / p.groups;
    const int g = blockIdx.x % p.groups;
    const int64_t cnt = (int64_t)p.S * p.cg;
    const T* xb = x + n * p.S * p.C + g * p.cg;
    float s = 0.f;
    for (int64_t i = threadIdx.x; i < cnt; i += 256) s += ov_to_f<T>(xb[i / p.cg * p.C + i % p.cg]);
    const float mu = ov_block_sum(s, red) / (float)cnt;
    s = 0.f;
    for (int64_t i = threadIdx.x; i < cnt; i += 256) {
        const float d = ov_to_f<T>(xb[i / p.cg * p.C + i % p.cg]) - mu;
        s += d * d;
    }
    const float r = 1.f / sqrtf(ov_block_sum(s, red) / (float)cnt + p.eps);
    for (int64_t i = threadIdx.x; i < cnt; i += 256) {
        const int64_t row = n * p.S + i / p.cg;
        const int c = g * p.cg + (int)(i % p.cg);
        const float v = (ov_to_f<T>(x[row * p.C + c]) - mu) * r * ov_gn_param(p.w, p.wtype, c, 1.f) + ov_gn_param(p.b, p.wtype, c, 0.f);
        y[row * p.C + c] = ov_from_f<T>(ov_gn_kept(p, row, c) ? ov_act(v, p.act) * p.drop.scale : 0.f);
    }
    if (threadIdx.x == 0) { mean[blockIdx.x] = mu; rstd[blockIdx.x] = r; }
}

template <typename T>
__device__ __forceinline__ float ov_gn_dv(const OvGn& p, const T* x, const T* dy, int64_t row, int c, float mu, float r, float* xhat) {
    *xhat = (ov_to_f<T>(x[row * p.C + c]) - mu) * r;
    if (!ov_gn_kept(p, row, c)) return 0.f;
    const float v = *xhat * ov_gn_param(p.w, p.wtype, c, 1.f) + ov_gn_param(p.b, p.wtype, c, 0.f);
    return ov_to_f<T>(dy[row * p.C + c]) * p.drop.scale * ov_act_grad(v, p.act);
}

template <typename T>
__global__ __launch_bounds__(256) void ov_gn_bwd_dx_kernel(const T* __restrict__ dy, const T* __restrict__ x, const OvGn p,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx) {
    __shared__ float red[16];
    const int64_t n = blockIdx.x / p.groups;
    const int g = blockIdx.x % p.groups;
    const int64_t cnt = (int64_t)p.S * p.cg;
    const float mu = mean[blockIdx.x], r = rstd[blockIdx.x];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t i = threadIdx.x; i < cnt; i += 256) {
        const int c = g * p.cg + (int)(i % p.cg);
        float xh;
        const float e = ov_gn_dv(p, x, dy, n * p.S + i / p.cg, c, mu, r, &xh) * ov_gn_param(p.w, p.wtype, c, 1.f);
        s1 += e;
        s2 += e * xh;
    }
    s1 = ov_block_sum(s1, red) / (float)cnt;
    s2 = ov_block_sum(s2, red) / (float)cnt;
    for (int64_t i = threadIdx.x; i < cnt; i += 256) {
        const int64_t row = n * p.S + i / p.cg;
        const int c = g * p.cg + (int)(i % p.cg);
        float xh;
        const float e = ov_gn_dv(p, x, dy, row, c, mu, r, &xh) * ov_gn_param(p.w, p.wtype, c, 1.f);
        dx[row * p.C + c] = ov_from_f<T>(r * (e - s1 - xh * s2));
    }
}

// one workgroup per channel
template <typename T>
__global__ __launch_bounds__(256) void ov_gn_bwd_param_kernel(const T* __restrict__ dy, const T* __restrict__ x, const OvGn p,
                                                              const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ dw,
                                                              float* __restrict__ db) {
    __shared__ float red[16];
    const int c = blockIdx.x, g = c / p.cg;
    float s1 = 0.f, s2 = 0.f;
    for (int64_t row = threadIdx.x; row < (int64_t)p.N * p.S; row += 256) {
        const int64_t k = row / p.S * p.groups + g;
        float xh;
        const float dv = ov_gn_dv(p, x, dy, row, c, mean[k], rstd[k], &xh);
        s1 += dv;
        s2 += dv * xh;
    }
    s1 = ov_block_sum(s1, red);
    s2 = ov_block_sum(s2, red);
    if (threadIdx.x == 0) {
        if (dw) dw[c] = s2;
        if (db) db[c] = s1;
    }
}

static int ov_gn_check(const char* what, int32_t dtype, int32_t N, int32_t S, int32_t C, int32_t groups, const void* w, const void* b, int32_t wdtype,
                       float eps, int32_t act, float drop, uint64_t seed, uint64_t offset, OvGn* p) {
    if (N < 0 || S < 0 || C < 0 || groups < 1 || C % groups || (C > 0 && C < groups)) {
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

extern "C" int64_t ontovae_group_norm_act_workspace_bytes(int32_t dtype, int32_t N, int32_t S, int32_t C, int32_t groups, int32_t backward) {
    (void)dtype; (void)N; (void)S; (void)C; (void)groups; (void)backward;
    return 0;
}

extern "C" int ontovae_group_norm_act(const void* x, int32_t dtype, int32_t N, int32_t S, int32_t C, int32_t groups, const void* weight,
                                      const void* bias, int32_t wdtype, float eps, int32_t act, float drop, uint64_t seed, uint64_t offset, void* y,
                                      float* mean, float* rstd, void* workspace, int64_t workspace_bytes, void* stream) {
    OvGn p;
    int rc = ov_gn_check("group_norm_act", dtype, N, S, C, groups, weight, bias, wdtype, eps, act, drop, seed, offset, &p);
    if (rc) return rc;
    if (N == 0 || S == 0 || C == 0) return ONTOVAE_OK;
    if (!x || !y || !mean || !rstd) { ontovae_set_error("group_norm_act: NULL argument"); return ONTOVAE_EINVAL; }
    (void)workspace; (void)workspace_bytes;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)(N * groups));
    switch (dtype) {
        case ONTOVAE_F32: hipLaunchKernelGGL(ov_gn_fwd_kernel<float>, grid, dim3(256), 0, st, (const float*)x, p, (float*)y, mean, rstd); break;
        case ONTOVAE_BF16: hipLaunchKernelGGL(ov_gn_fwd_kernel<ov_bf>, grid, dim3(256), 0, st, (const ov_bf*)x, p, (ov_bf*)y, mean, rstd); break;
        default: hipLaunchKernelGGL(ov_gn_fwd_kernel<ov_hf>, grid, dim3(256), 0, st, (const ov_hf*)x, p, (ov_hf*)y, mean, rstd); break;
    }
    OV_OPS_LAUNCH_CHECK("group_norm_act");
    return ONTOVAE_OK;
}

template <typename T>
static void ov_gn_bwd_launch(const void* dy, const void* x, const OvGn& p, const float* mean, const float* rstd, void* dx, float* dw, float* db,
                             hipStream_t st) {
    if (p.N > 0)
        hipLaunchKernelGGL(ov_gn_bwd_dx_kernel<T>, dim3((unsigned)(p.N * p.groups)), dim3(256), 0, st, (const T*)dy, (const T*)x, p, mean, rstd, (T*)dx);
    if (dw || db) hipLaunchKernelGGL(ov_gn_bwd_param_kernel<T>, dim3(p.C), dim3(256), 0, st, (const T*)dy, (const T*)x, p, mean, rstd, dw, db);
}

extern "C" int ontovae_group_norm_act_backward(const void* dy, const void* x, int32_t dtype, int32_t N, int32_t S, int32_t C, int32_t groups,
                                               const void* weight, const void* bias, int32_t wdtype, const float* mean, const float* rstd,
                                               int32_t act, float drop, uint64_t seed, uint64_t offset, void* dx, float* dweight, float* dbias,
                                               void* workspace, int64_t workspace_bytes, void* stream) {
    OvGn p;
    int rc = ov_gn_check("group_norm_act_backward", dtype, N, S, C, groups, weight, bias, wdtype, 0.f, act, drop, seed, offset, &p);
    if (rc) return rc;
    if (C == 0) return ONTOVAE_OK;
    const bool none = N == 0 || S == 0;
    if (!none && (!dy || !x || !mean || !rstd || !dx)) { ontovae_set_error("group_norm_act_backward: NULL argument"); return ONTOVAE_EINVAL; }
    (void)workspace; (void)workspace_bytes;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (none) p.N = 0;
    switch (dtype) {
        case ONTOVAE_F32: ov_gn_bwd_launch<float>(dy, x, p, mean, rstd, dx, dweight, dbias, st); break;
        case ONTOVAE_BF16: ov_gn_bwd_launch<ov_bf>(dy, x, p, mean, rstd, dx, dweight, dbias, st); break;
        default: ov_gn_bwd_launch<ov_hf>(dy, x, p, mean, rstd, dx, dweight, dbias, st); break;
    }
    OV_OPS_LAUNCH_CHECK("group_norm_act_backward");
    return ONTOVAE_OK;
}

#endif

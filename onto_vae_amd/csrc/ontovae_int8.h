// Products in 8-bit integers with one scale per row of each operand.
//
//   s_m = max_k |x_mk| / 127,  q_mk = rint(x_mk / s_m)          (ov_q8_rows_kernel)
//   y_mn = s_m t_n sum_k q_mk w_nk + b_n                        (ov_q8_gemm_kernel), the sum exact in 32-bit integers
#ifndef ONTOVAE_INT8_H
#define ONTOVAE_INT8_H

#include "ontovae_ops.h"

#define OV_Q8_MAX_K 131071          // 128 * 128 * K < 2^31

// A row's scale from the bits of its largest magnitude: NaN if the row holds an infinity or a NaN.
__device__ __forceinline__ float ov_q8_scale(uint32_t amax_bits) {
    return amax_bits >= 0x7f800000u ? __builtin_nanf("") : __builtin_bit_cast(float, amax_bits) / 127.0f;
}

// Rounding of the TRUE quotient x / s to the nearest integer, ties to even: x * (1 / s) is off by two roundings, so its
// integer may be one off next to a border; the residual x - n s is exact in one fma (|r| <= 1.5 s, a multiple of the finer of
// the two ulps), and settles it.  (A bf16 row has exact ties: its largest element's half.)
struct OvQ8 {
    float s, h, inv, up;
    __device__ __forceinline__ explicit OvQ8(float scale) {
        up = scale < 0x1p-60f ? 0x1p80f : 1.0f;      // s / 2 and 1 / s stay normal
        s = scale * up;
        h = 0.5f * s;
        inv = scale > 0.f ? 1.0f / s : 0.f;          // zero row and NaN scale: every q is 0
    }
    __device__ __forceinline__ int operator()(float x) const {
        if (!(inv > 0.f)) return 0;
        x *= up;
        float n = rintf(x * inv);
        const float r = fmaf(-n, s, x);
        const bool odd = ((int)n) & 1;
        if (r > h || (r == h && odd)) n += 1.f;
        else if (r < -h || (r == -h && odd)) n -= 1.f;
        return (int)fminf(fmaxf(n, -127.f), 127.f);
    }
};

template <typename T>
__global__ __launch_bounds__(256) void ov_q8_rows_kernel(const T* __restrict__ x, int64_t ldx, const int32_t* __restrict__ rows, int n_src,
                                                         int K, int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale) {
    __shared__ uint32_t red[4];
    const int64_t m = blockIdx.x;
    int64_t src = m;
    bool ok = true;
    if (rows) { src = rows[m]; ok = src >= 0 && src < n_src; }
    const T* xr = x + (ok ? src : 0) * ldx;
    uint32_t a = ok ? 0u : 0x7fffffffu;
    if (ok)
        for (int k = threadIdx.x; k < K; k += 256) a = max(a, __builtin_bit_cast(uint32_t, ov_to_f<T>(xr[k])) & 0x7fffffffu);
    a = ov_wave_max_u(a);
    if (ov_lane() == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    const float s = ov_q8_scale(max(max(red[0], red[1]), max(red[2], red[3])));
    const OvQ8 f(s);
    for (int64_t k = threadIdx.x; k < ldq; k += 256) q[m * ldq + k] = k < K && ok ? (int8_t)f(ov_to_f<T>(xr[k])) : (int8_t)0;
    if (threadIdx.x == 0) scale[m] = s;
}

template <typename T>
__global__ __launch_bounds__(256) void ov_q8_gemm_kernel(const int8_t* __restrict__ A, int64_t lda, const float* __restrict__ sa,
                                                         const int8_t* __restrict__ B, int64_t ldb, const float* __restrict__ sb,
                                                         const float* __restrict__ bias, int M, int N, int K, T* __restrict__ y, int64_t ldy) {
    __shared__ int8_t As[16][68], Bs[16][68];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t m0 = (int64_t)blockIdx.y * 16, n0 = (int64_t)blockIdx.x * 16;
    int acc = 0;
    for (int k0 = 0; k0 < K; k0 += 64) {
        for (int e = threadIdx.x; e < 1024; e += 256) {
            const int r = e >> 6, k = e & 63;
            As[r][k] = m0 + r < M && k0 + k < K ? A[(m0 + r) * lda + k0 + k] : (int8_t)0;
            Bs[r][k] = n0 + r < N && k0 + k < K ? B[(n0 + r) * ldb + k0 + k] : (int8_t)0;
        }
        __syncthreads();
        for (int k = 0; k < 64; ++k) acc += (int)As[ty][k] * (int)Bs[tx][k];
        __syncthreads();
    }
    const int64_t m = m0 + ty, n = n0 + tx;
    if (m < M && n < N) y[m * ldy + n] = ov_from_f<T>((float)acc * sa[m] * sb[n] + (bias ? bias[n] : 0.f));
}

extern "C" int ontovae_quantize_rows(const void* x, int32_t dtype, int64_t ldx, const int32_t* rows, int32_t n_src, int32_t M, int32_t K,
                                     int8_t* q, int64_t ldq, float* scale, void* stream) {
    if (M < 0 || K < 0 || n_src < 0 || ldx < K || ldq < K || (!rows && n_src < M)) {
        ontovae_set_error("quantize_rows: M = %d, K = %d, n_src = %d, ldx = %lld, ldq = %lld", M, K, n_src, (long long)ldx, (long long)ldq);
        return ONTOVAE_EINVAL;
    }
    if (dtype < ONTOVAE_F32 || dtype > ONTOVAE_F16) { ontovae_set_error("quantize_rows: unknown element type %d", dtype); return ONTOVAE_EINVAL; }
    if (M == 0) return ONTOVAE_OK;
    if (!scale || (K > 0 && (!x || !q))) { ontovae_set_error("quantize_rows: NULL argument"); return ONTOVAE_EINVAL; }
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    switch (dtype) {
        case ONTOVAE_F32: hipLaunchKernelGGL(ov_q8_rows_kernel<float>, dim3(M), dim3(256), 0, st, (const float*)x, ldx, rows, n_src, K, q, ldq, scale); break;
        case ONTOVAE_BF16: hipLaunchKernelGGL(ov_q8_rows_kernel<ov_bf>, dim3(M), dim3(256), 0, st, (const ov_bf*)x, ldx, rows, n_src, K, q, ldq, scale); break;
        default: hipLaunchKernelGGL(ov_q8_rows_kernel<ov_hf>, dim3(M), dim3(256), 0, st, (const ov_hf*)x, ldx, rows, n_src, K, q, ldq, scale); break;
    }
    OV_OPS_LAUNCH_CHECK("quantize_rows");
    return ONTOVAE_OK;
}

extern "C" int64_t ontovae_int8_matmul_workspace_bytes(int32_t M, int32_t N, int32_t K) {
    (void)M; (void)N; (void)K;
    return 0;
}

extern "C" int ontovae_int8_matmul(const int8_t* a, int64_t lda, const float* sa, const int8_t* b, int64_t ldb, const float* sb,
                                   const float* bias, int32_t M, int32_t N, int32_t K, void* y, int32_t dtype, int64_t ldy, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
    if (M < 0 || N < 0 || K < 0 || lda < K || ldb < K || ldy < N) {
        ontovae_set_error("int8_matmul: M = %d, N = %d, K = %d, lda = %lld, ldb = %lld, ldy = %lld", M, N, K, (long long)lda, (long long)ldb,
                          (long long)ldy);
        return ONTOVAE_EINVAL;
    }
    if (K > OV_Q8_MAX_K) { ontovae_set_error("int8_matmul: K = %d, the sums are exact in 32 bits up to %d", K, OV_Q8_MAX_K); return ONTOVAE_EINVAL; }
    if (dtype < ONTOVAE_F32 || dtype > ONTOVAE_F16) { ontovae_set_error("int8_matmul: unknown element type %d", dtype); return ONTOVAE_EINVAL; }
    if (M == 0 || N == 0) return ONTOVAE_OK;
    if (!sa || !sb || !y || (K > 0 && (!a || !b))) { ontovae_set_error("int8_matmul: NULL argument"); return ONTOVAE_EINVAL; }
    if (workspace_bytes < ontovae_int8_matmul_workspace_bytes(M, N, K)) {
        ontovae_set_error("int8_matmul: workspace of %lld bytes needed", (long long)ontovae_int8_matmul_workspace_bytes(M, N, K));
        return ONTOVAE_EINVAL;
    }
    (void)workspace;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const dim3 grid((N + 15) / 16, (M + 15) / 16);
    switch (dtype) {
        case ONTOVAE_F32: hipLaunchKernelGGL(ov_q8_gemm_kernel<float>, grid, dim3(256), 0, st, a, lda, sa, b, ldb, sb, bias, M, N, K, (float*)y, ldy); break;
        case ONTOVAE_BF16: hipLaunchKernelGGL(ov_q8_gemm_kernel<ov_bf>, grid, dim3(256), 0, st, a, lda, sa, b, ldb, sb, bias, M, N, K, (ov_bf*)y, ldy); break;
        default: hipLaunchKernelGGL(ov_q8_gemm_kernel<ov_hf>, grid, dim3(256), 0, st, a, lda, sa, b, ldb, sb, bias, M, N, K, (ov_hf*)y, ldy); break;
    }
    OV_OPS_LAUNCH_CHECK("int8_matmul");
    return ONTOVAE_OK;
}

#endif

// Products in 8-bit integers with one scale per row of each operand.
//
//   s_m = max_k |x_mk| * (1 / 127),  q_mk = rint(x_mk / s_m)      (ov_q8_rows_kernel)
//   y_mn = s_m t_n sum_k q_mk w_nk + b_n                        (ov_q8_gemm_kernel), the sum exact in 32-bit integers
//
// Integer sums are exact in any order, so the K axis may be cut into slabs (ov_q8_combine_kernel) without a rounding.
#ifndef ONTOVAE_INT8_H
#define ONTOVAE_INT8_H

#include "ontovae_ops.h"

#define OV_Q8_MAX_K 131071          // 128 * 128 * K < 2^31
#define OV_Q8_MAX_MN (INT32_MAX - 1024)        // row and column indexes run past M and N by up to a tile

typedef int ov_i32x4 __attribute__((ext_vector_type(4)));
typedef int ov_i32x16 __attribute__((ext_vector_type(16)));

// A row's scale from the bits of its largest magnitude: NaN if the row holds an infinity or a NaN.  A product with the float32
// nearest to 1 / 127, as tensor libraries divide by a constant: a weight that such a program quantised has the same scale, bit for bit.
__device__ __forceinline__ float ov_q8_scale(uint32_t amax_bits) {
    return amax_bits >= 0x7f800000u ? __builtin_nanf("") : __builtin_bit_cast(float, amax_bits) * (1.0f / 127.0f);
}

// Rounding of the TRUE quotient x / s to the nearest integer, ties to even: x * (1 / s) is off by two roundings, so its
// integer may be one off next to a border; the residual r = x - n s is exact in one fma (|r| <= 1.5 s, a multiple of the finer
// of the two ulps), and settles it: |r| < s / 2 is right, else the neighbour on r's side, or the even one on a tie.  (A bf16
// row has exact ties: its largest element's half.)
struct OvQ8 {
    float s, h, inv, up;
    bool plain;
    __device__ __forceinline__ explicit OvQ8(float scale) {
        up = scale < 0x1p-60f ? 0x1p80f : 1.0f;      // s / 2 and 1 / s stay normal
        s = scale * up;
        h = 0.5f * s;
        inv = scale > 0.f ? 1.0f / s : 0.f;          // zero row and NaN scale: every q is 0
        plain = scale >= 0x1p-60f;
    }
    __device__ __forceinline__ int one(float x) const {
        if (!(inv > 0.f)) return 0;
        x *= up;
        float n = rintf(x * inv);
        const float r = fmaf(-n, s, x);
        const bool odd = ((int)n) & 1;
        if (r > h || (r == h && odd)) n += 1.f;
        else if (r < -h || (r == -h && odd)) n -= 1.f;
        return (int)fminf(fmaxf(n, -127.f), 127.f);
    }
    // V values at once: the sum with 1.5 2^23 rounds and leaves the integer in the low byte; the careful form only where some
    // value of the wave stands next to a border
    template <int V>
    __device__ __forceinline__ void many(const float (&x)[V], uint32_t (&q)[V / 4]) const {
        bool near = !plain;
        uint32_t b[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float t = fmaf(x[j], inv, 12582912.0f), n = t - 12582912.0f;
            near |= fabsf(fmaf(-n, s, x[j])) >= h;
            b[j] = __builtin_bit_cast(uint32_t, t);
        }
        if (near) {
#pragma unroll
            for (int j = 0; j < V; ++j) b[j] = (uint32_t)one(x[j]);
        }
#pragma unroll
        for (int j = 0; j < V; j += 4)
            q[j / 4] = __builtin_amdgcn_perm(b[j + 1], b[j], 0x0c0c0400u) | __builtin_amdgcn_perm(b[j + 3], b[j + 2], 0x04000c0cu);
    }
};

// the epilogue of every variant, bit for bit: the float32 result is pinned before its rounding to the output type (which the
// compiler otherwise merges into the fma for float16 where it can see both)
__device__ __forceinline__ float ov_q8_out(int acc, float sa, float sb, float bias) {
    float v = fmaf((float)acc * sa, sb, bias);
    asm("" : "+v"(v));
    return v;
}

__device__ __forceinline__ uint32_t ov_abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

// One row per group of THREADS threads (a wave: 4 rows per workgroup; else one), the row held in registers between the search
// for its maximum and the rounding, 16 B per lane and load: x is read once.  Bound by that read and the write of a quarter
// or half of it.  Rows of more than THREADS * NV pieces re-read the rest, from the cache.  Rows may start at any element:
// the loads are not assumed aligned.  Column k of row m goes to q[(k / 128) kst + m ldq + k % 128]: kst = 128 is the plain matrix.
template <typename T, int THREADS, int NV>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void ov_q8_rows_kernel(const T* __restrict__ x, int64_t ldx,
                                                                                    const int32_t* __restrict__ rows, int n_src, int M, int K,
                                                                                    int8_t* __restrict__ q, int64_t ldq, int64_t kst, int64_t kpad,
                                                                                    float* __restrict__ scale) {
    constexpr int VE = 16 / sizeof(T);
    __shared__ uint32_t red[16];
    const int tid = THREADS < 256 ? ov_lane() : (int)threadIdx.x;
    const int64_t m = THREADS < 256 ? (int64_t)blockIdx.x * 4 + ov_wave_id() : (int64_t)blockIdx.x;
    if (THREADS < 256 && m >= M) return;
    int64_t src = m;
    bool ok = true;
    if (rows) { src = rows[m]; ok = src >= 0 && src < n_src; }
    const T* xr = x + (ok ? src : 0) * ldx;
    const int nfull = ok ? K / VE : 0, kt = nfull * VE;      // whole 16-B pieces; the rest of the row goes element by element
    OvVec<T> v[NV];
    uint32_t a = ok ? 0u : 0x7fffffffu;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int p = tid + i * THREADS;
        if (p < nfull) v[i].load(xr + (int64_t)p * VE);
        else v[i].zero();
    }
    T t = (T)0.f;
    if (ok && kt + tid < K) t = xr[kt + tid];                // fewer than VE elements
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VE; ++j) a = max(a, ov_abs_bits(ov_to_f<T>(v[i].e[j])));
    a = max(a, ov_abs_bits(ov_to_f<T>(t)));
    for (int p = tid + NV * THREADS; p < nfull; p += THREADS) {
        OvVec<T> w;
        w.load(xr + (int64_t)p * VE);
#pragma unroll
        for (int j = 0; j < VE; ++j) a = max(a, ov_abs_bits(ov_to_f<T>(w.e[j])));
    }
    a = ov_wave_max_u(a);
    if (THREADS >= 256) {
        if (ov_lane() == 0) red[threadIdx.x >> 6] = a;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) a = max(a, red[w]);
    }
    const float s = ov_q8_scale(a);
    const OvQ8 f(s);
    int8_t* qr = q + m * ldq;
    const bool qal = ((reinterpret_cast<uintptr_t>(q) | (uintptr_t)ldq | (uintptr_t)kst) & 7) == 0;
    auto put = [&](int p, const OvVec<T>& w) {
        const int k = p * VE;
        int8_t* dst = qr + (int64_t)(k >> 7) * kst + (k & 127);
        uint32_t o[VE / 4] = {};
        if (s > 0.f) {                                       // else a zero row or one without a scale
            float e[VE];
#pragma unroll
            for (int j = 0; j < VE; ++j) e[j] = ov_to_f<T>(w.e[j]);
            f.many<VE>(e, o);
        }
        if (qal) {
#pragma unroll
            for (int j = 0; j < VE / 4; ++j) reinterpret_cast<uint32_t*>(dst)[j] = o[j];
        } else {
#pragma unroll
            for (int j = 0; j < VE; ++j) dst[j] = (int8_t)(o[j / 4] >> (8 * (j % 4)));
        }
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int p = tid + i * THREADS;
        if (p < nfull) put(p, v[i]);
    }
    for (int p = tid + NV * THREADS; p < nfull; p += THREADS) {
        OvVec<T> w;
        w.load(xr + (int64_t)p * VE);
        put(p, w);
    }
    for (int64_t k = kt + tid; k < kpad; k += THREADS) qr[(k >> 7) * kst + (k & 127)] = k < K && ok ? (int8_t)f.one(ov_to_f<T>(t)) : (int8_t)0;
    if (tid == 0) scale[m] = s;
}

struct OvQ8Gemm {
    const int8_t* A; int64_t lda, ast;   // [M, K]: column k of row m at (k / 128) ast + m lda + k % 128 (ast = 128: a plain matrix)
    const int8_t* B; int64_t ldb;        // [N, K]
    const float* sa; const float* sb; const float* bias;
    int M, N, K, kchunk;                 // kchunk % 128 == 0: K range of a slab
    int nm, nn;                          // tiles
    int32_t* slab;                       // split: [splits][M][N]
    void* y; int64_t ldy;
};

// Tile BM x BN of the product, waves of WM x WN on v_mfma_i32_32x32x32_i8, K in steps of BK bytes through a ring of ST LDS
// stages, one barrier a step.  DIRECT: the pieces go from memory to LDS without passing registers, and the wait before the
// barrier leaves the ST - 2 youngest stages in flight.  A row of a stage is BK / 16 pieces of 16 B, stored with the piece
// index xor-ed with bits of the row (the source address is permuted, LDS is written in lane order): a wave's 16-B fragment
// reads then spread over all 64 banks.  Rows beyond M / N repeat the last one, their results are dropped.  The last, partial step
// of K is loaded with its bytes masked, so nothing is assumed of what stands behind column K.
// !DIRECT: operands whose rows do not start on 16 B; the same loads through registers, unaligned, in tiles of 64 x 64 with the slabs of the
// tile that aligned rows would get (8192 x 4096 x 4096 390 us where aligned rows take 146; few rows alike, 16 us).
// T = int32_t: the raw sums to slab blockIdx.y.
template <int BM, int BN, int WM, int WN, int BK, int ST, bool DIRECT, typename T>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void ov_q8_gemm_kernel(const OvQ8Gemm g) {
    constexpr int THREADS = (BM / WM) * (BN / WN) * 64, ROWS = BM + BN, STAGE = ROWS * BK, PC = BK / 16, NL = ROWS * PC / THREADS;
    constexpr int FM = WM / 32, FN = WN / 32, NLA = BM * PC / THREADS, RSTEP = THREADS / PC;
    static_assert(ROWS * PC % THREADS == 0 && BM * PC % THREADS == 0 && RSTEP % 16 == 0 && (BK == 64 || BK == 128), "whole loads per thread");
    // the permutation of a row's pieces: 16 neighbouring rows put piece p into 16 different 16-B slots of 256 B
    auto swz = [](int row) { return BK == 128 ? (row >> 1) & 7 : (row >> 2) & 3; };
    extern __shared__ __attribute__((aligned(16))) int8_t ov_q8_lds[];
    // workgroups are dealt to the 8 XCDs round-robin: XCD x takes a contiguous run of tiles, in which the tiles of up to 8
    // neighbouring row panels share their B panels (and the column panels their A) in that XCD's L2
    int tm, tn;
    {
        const int nt = g.nm * g.nn;
        int id = blockIdx.x;
        const int per = nt >> 3, rem = nt & 7, x = id & 7, j = id >> 3;
        id = x * per + min(x, rem) + j;
        const int gs = 8 * g.nn, gid = id / gs, first = gid * 8, rows = min(g.nm - first, 8), r = id - gid * gs;
        tm = first + r % rows;
        tn = r / rows;
    }
    const int m0 = tm * BM, n0 = tn * BN;
    const int kbeg = blockIdx.y * g.kchunk, kend = min(g.K, kbeg + g.kchunk);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / (BN / WN) * WM, wn = wave % (BN / WN) * WN;
    const int8_t* Ab = g.A + (int64_t)m0 * g.lda + (int64_t)(kbeg >> 7) * g.ast;
    const int8_t* Bb = g.B + (int64_t)n0 * g.ldb + kbeg;
    const int len = max(kend - kbeg, 0), full = len / BK;

    ov_i32x16 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

    // piece i of this thread: row tid / PC + i RSTEP of the stage (A rows, then B rows), LDS piece tid % PC
    const int piece = (tid % PC) ^ swz(tid / PC);                         // RSTEP is a multiple of 16: the same for every i
    auto row_of = [&](int i) { return tid / PC + i * RSTEP; };
    uint32_t off[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int r = row_of(i);
        off[i] = (i < NLA ? (uint32_t)min(r, g.M - 1 - m0) * (uint32_t)g.lda : (uint32_t)min(r - BM, g.N - 1 - n0) * (uint32_t)g.ldb) +
                 (uint32_t)piece * 16u;
    }
    auto acol = [&](int k) { return (int64_t)(k >> 7) * g.ast + (k & 127); };
    auto dma = [&](int step, int stage) {
        int8_t* dst = ov_q8_lds + stage * STAGE + wave * 1024;
        const int8_t* sa = Ab + acol(step * BK);
        const int8_t* sb = Bb + step * BK;
#pragma unroll
        for (int i = 0; i < NL; ++i)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)((i < NLA ? sa : sb) + off[i]),
                                             (__attribute__((address_space(3))) void*)(dst + i * (THREADS * 16)), 16, 0, 0);
    };
    // the fragments of the next 32 columns are read while the products of the current ones run
    auto compute = [&](int stage) {
        const int8_t* sA = ov_q8_lds + stage * STAGE + (wm + (lane & 31)) * BK;
        const int8_t* sB = ov_q8_lds + stage * STAGE + (BM + wn + (lane & 31)) * BK;
        const int sw = swz(lane & 31);                                    // the fragment rows differ by multiples of 32
        ov_i32x4 a[2][FM], b[2][FN];
        auto frag = [&](int kk) {
            const int p = ((kk * 2 + (lane >> 5)) ^ sw) * 16;
#pragma unroll
            for (int j = 0; j < FN; ++j) b[kk & 1][j] = *reinterpret_cast<const ov_i32x4*>(sB + j * 32 * BK + p);
#pragma unroll
            for (int i = 0; i < FM; ++i) a[kk & 1][i] = *reinterpret_cast<const ov_i32x4*>(sA + i * 32 * BK + p);
        };
        frag(0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk) {
            if (kk + 1 < BK / 32) frag(kk + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[kk & 1][j], a[kk & 1][i], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // a 16-B piece of a row through registers: bytes from kend on are 0 and not read
    auto masked = [&](int i, int k0) {
        const int r = row_of(i);
        const int8_t* base = (i < NLA ? Ab + (int64_t)min(r, g.M - 1 - m0) * g.lda + acol(k0)
                                                   : Bb + (int64_t)min(r - BM, g.N - 1 - n0) * g.ldb + k0) + piece * 16;
        const int n = len - k0 - piece * 16;
        OvBytes<16> v = {};
        if (n >= 16) __builtin_memcpy(&v, base, 16);
        else
#pragma unroll
            for (int j = 0; j < 15; ++j)
                if (j < n) v.b[j] = base[j];
        return __builtin_bit_cast(ov_i32x4, v);
    };
    auto put = [&](int stage, int i, ov_i32x4 v) {
        *reinterpret_cast<ov_i32x4*>(ov_q8_lds + stage * STAGE + tid * 16 + i * (THREADS * 16)) = v;
    };

    if (DIRECT) {
        // step `full`, if there is one, is the partial one.  ONE call of compute: a second copy of it would move the accumulators
        const int steps = (len + BK - 1) / BK;
        auto fill = [&](int step, int stage) {
            if (step < full) dma(step, stage);
            else if (step < steps) {
#pragma unroll 1
                for (int i = 0; i < NL; ++i) put(stage, i, masked(i, step * BK));
            }
        };
#pragma unroll
        for (int s = 0; s < ST - 1; ++s) fill(s, s);
        int cur = 0;
        for (int s = 0; s < steps; ++s) {
            // the stage of this step has landed when at most the younger stages' loads are outstanding
            if (s + ST - 2 < full) ov_wait_vm<NL * (ST - 2)>();
            else ov_wait_vm<0>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            int nx = cur + ST - 1;
            nx -= nx >= ST ? ST : 0;
            fill(s + ST - 1, nx);                                         // read by nobody since the barrier above
            compute(cur);
            cur = cur + 1 == ST ? 0 : cur + 1;
        }
    } else {
        const int steps = (len + BK - 1) / BK;
        ov_i32x4 v[NL];
        if (steps > 0) {
#pragma unroll
            for (int i = 0; i < NL; ++i) v[i] = masked(i, 0);
        }
        for (int s = 0; s < steps; ++s) {
            const int st = s & 1;
#pragma unroll
            for (int i = 0; i < NL; ++i) put(st, i, v[i]);
            __syncthreads();
            if (s + 1 < steps) {
#pragma unroll
                for (int i = 0; i < NL; ++i) v[i] = masked(i, (s + 1) * BK);
            }
            compute(st);
        }
    }

    // A 32 x 32 tile of the TRANSPOSED product: column (lane & 31) is the row m of y, row (e & 3) + 8 (e >> 2) + 4 (lane >> 5) its
    // column n.  A lane then holds 4 neighbours of a row of y; a wave collects 32 rows x WN columns in LDS and writes whole
    // 16-B pieces of rows (single elements straight from the registers took 75 of 195 us of an 8192 x 4096 x 4096 product: a
    // scale to load and a store to issue for each).
    constexpr int TS = sizeof(T), LDW = WN * TS + 16, WAVES = THREADS / 64, EV = 16 / TS;
    static_assert(WAVES * 32 * LDW + 2 * BN * 4 <= (DIRECT ? ST : 2) * STAGE, "the epilogue fits the stages' LDS");
    float* sbl = reinterpret_cast<float*>(ov_q8_lds + WAVES * 32 * LDW);
    __syncthreads();                                                      // every stage is free
    if (!__is_same(T, int32_t)) {
        for (int i = tid; i < BN; i += THREADS) {
            const int n = min(n0 + i, g.N - 1);
            sbl[i] = g.sb[n];
            sbl[BN + i] = g.bias ? g.bias[n] : 0.f;
        }
        __syncthreads();
    }
    int8_t* wl = ov_q8_lds + wave * 32 * LDW;
    T* yb;
    int64_t ldy;
    if constexpr (__is_same(T, int32_t)) { yb = g.slab + (int64_t)blockIdx.y * g.M * g.N; ldy = g.N; }
    else { yb = static_cast<T*>(g.y); ldy = g.ldy; }
    const bool al = ((reinterpret_cast<uintptr_t>(yb) | (uintptr_t)(ldy * TS)) & 15) == 0;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        float sam = 0.f;
        if (!__is_same(T, int32_t)) sam = g.sa[min(m0 + wm + 32 * i + (lane & 31), g.M - 1)];
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4) {
                const int c = 32 * j + 8 * e4 + 4 * (lane >> 5);
                T o[4];
                if constexpr (__is_same(T, int32_t)) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = acc[i][j][4 * e4 + e];
                } else {
                    const f32x4 tb = *reinterpret_cast<const f32x4*>(sbl + wn + c), bi = *reinterpret_cast<const f32x4*>(sbl + BN + wn + c);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = ov_from_f<T>(ov_q8_out(acc[i][j][4 * e4 + e], sam, tb[e], bi[e]));
                }
                __builtin_memcpy(__builtin_assume_aligned(wl + (lane & 31) * LDW + c * TS, 4 * TS), o, sizeof(o));
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();                                  // the buffer is the wave's own
        constexpr int PR = WN / EV;                                       // 16-B pieces of a row
#pragma unroll
        for (int q = 0; q < 32 * PR / 64; ++q) {
            const int id = q * 64 + lane, r = id / PR, pc = id % PR;
            const int m = m0 + wm + 32 * i + r, n = n0 + wn + pc * EV;
            OvVec<T> v;
            __builtin_memcpy(v.e, __builtin_assume_aligned(wl + r * LDW + pc * 16, 16), 16);
            if (m >= g.M || n >= g.N) continue;
            T* dst = yb + m * ldy + n;
            if (al && n + EV <= g.N) __builtin_memcpy(__builtin_assume_aligned(dst, 16), v.e, 16);
            else {
#pragma unroll
                for (int e = 0; e < EV; ++e)
                    if (n + e < g.N) dst[e] = v.e[e];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// sum of the slabs, scales, bias: one element per thread and trip
template <typename T>
__global__ __launch_bounds__(256) void ov_q8_combine_kernel(const OvQ8Gemm g, int splits) {
    const int64_t total = (int64_t)g.M * g.N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int m = (int)(i / g.N), n = (int)(i - (int64_t)m * g.N);
        int a = 0;
#pragma unroll 8
        for (int z = 0; z < splits; ++z) a += g.slab[z * total + i];
        static_cast<T*>(g.y)[(int64_t)m * g.ldy + n] = ov_from_f<T>(ov_q8_out(a, g.sa[m], g.sb[n], g.bias ? g.bias[n] : 0.f));
    }
}

// One to four rows of x against a layer, rows quantised on the way: the latency of one launch instead of three.  Every
// workgroup reads the MT rows of x (from the L2 after the first), rounds its threads' pieces of 16 elements into registers and
// walks weight rows blockIdx, + gridDim, ... with them: a thread meets the same 16 columns of every row, so neither operand
// passes LDS.  Bound by the read of the weights.  The next weight row is requested before the current one is reduced.
template <typename T, int MT, int NP>
__global__ __launch_bounds__(256) void ov_q8_few_kernel(const T* __restrict__ x, int64_t ldx, const int32_t* __restrict__ rows, int n_src, int M,
                                                        const OvQ8Gemm g, int ytype) {
    constexpr int VE = 16 / sizeof(T);
    __shared__ uint32_t redu[4][MT];
    __shared__ int redi[2][4][MT];
    const int tid = threadIdx.x, lane = ov_lane(), wave = ov_wave_id();
    ov_i32x4 w[NP];
    auto wload = [&](int n) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int k = (tid + i * 256) * 16;
            w[i] = ov_i32x4{0, 0, 0, 0};
            const int8_t* src = g.B + (int64_t)n * g.ldb + k;
            if (k + 16 <= g.K) __builtin_memcpy(&w[i], src, 16);
            else if (k < g.K) {
                OvBytes<16> b = {};
#pragma unroll
                for (int j = 0; j < 15; ++j)
                    if (k + j < g.K) b.b[j] = src[j];
                w[i] = __builtin_bit_cast(ov_i32x4, b);
            }
        }
    };
    wload(blockIdx.x);
    ov_i32x4 q[MT][NP];
    float s[MT];
    {
        T v[NP][16];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            int64_t src = m;
            bool ok = m < M;
            if (ok && rows) { src = rows[m]; ok = src >= 0 && src < n_src; }
            const T* xr = x + (ok ? src : 0) * ldx;
            uint32_t a = ok ? 0u : 0x7fffffffu;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int k = (tid + i * 256) * 16;
                if (ok && k + 16 <= g.K) {
#pragma unroll
                    for (int c = 0; c < 16 / VE; ++c) __builtin_memcpy(&v[i][c * VE], xr + k + c * VE, 16);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[i][j] = ok && k + j < g.K ? xr[k + j] : (T)0.f;
                }
            }
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) a = max(a, ov_abs_bits(ov_to_f<T>(v[i][j])));
            a = ov_wave_max_u(a);
            if (lane == 0) redu[wave][m] = a;
            __syncthreads();
            s[m] = ov_q8_scale(max(max(redu[0][m], redu[1][m]), max(redu[2][m], redu[3][m])));
            const OvQ8 f(s[m]);
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                q[m][i] = ov_i32x4{0, 0, 0, 0};
                if (s[m] > 0.f) {
                    float e[16];
                    uint32_t o[4];
#pragma unroll
                    for (int j = 0; j < 16; ++j) e[j] = ov_to_f<T>(v[i][j]);
                    f.many<16>(e, o);
#pragma unroll
                    for (int j = 0; j < 4; ++j) q[m][i][j] = (int)o[j];
                }
            }
        }
    }
    int buf = 0;
    for (int n = blockIdx.x; n < g.N; n += gridDim.x, buf ^= 1) {
        int acc[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            acc[m] = 0;
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[m] = __builtin_amdgcn_sdot4(q[m][i][c], w[i][c], acc[m], false);
        }
        if (n + (int)gridDim.x < g.N) wload(n + gridDim.x);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) acc[m] += __shfl_xor(acc[m], o, 64);
            if (lane == 0) redi[buf][wave][m] = acc[m];
        }
        __syncthreads();                     // two buffers: the next row's sums go to the other one
        if (tid < MT && tid < M) {
            const int a = (redi[buf][0][tid] + redi[buf][1][tid]) + (redi[buf][2][tid] + redi[buf][3][tid]);
            float sm = s[0];
#pragma unroll
            for (int m = 1; m < MT; ++m) sm = tid == m ? s[m] : sm;
            const float v = ov_q8_out(a, sm, g.sb[n], g.bias ? g.bias[n] : 0.f);
            const int64_t o = (int64_t)tid * g.ldy + n;
            if (ytype == ONTOVAE_F32) static_cast<float*>(g.y)[o] = v;
            else if (ytype == ONTOVAE_BF16) static_cast<ov_bf*>(g.y)[o] = ov_from_f<ov_bf>(v);
            else static_cast<ov_hf*>(g.y)[o] = ov_from_f<ov_hf>(v);
        }
    }
}

// ---------------------------------------------------------------- host
// threads that share a row of p pieces; 64: four rows a workgroup
static int ov_q8_row_threads(int p, int M) {
    if (p <= 256) return 64;
    if (p <= 1024) return 256;
    if (p <= 2048) return 512;
    return p <= 5120 && M > 512 ? 512 : 1024;                 // up to 512 rows, one round of workgroups: fewer pieces one behind the other
}
static bool ov_q8_rows_fit(int dtype, int M, int K) {
    const int ve = dtype == ONTOVAE_F32 ? 4 : 8, th = ov_q8_row_threads((K + ve - 1) / ve, M);
    return th < 256 ? ov_ops_fits(((int64_t)M + 3) / 4, 256) : ov_ops_fits(M, th);
}

template <typename T>
static void ov_q8_rows_launch(const void* x, int64_t ldx, const int32_t* rows, int n_src, int M, int K, int8_t* q, int64_t ldq, int64_t kst,
                              int64_t kpad, float* scale, hipStream_t st) {
    constexpr int VE = 16 / sizeof(T);
    const int p = (K + VE - 1) / VE;
    const T* xt = static_cast<const T*>(x);
#define OV_Q8_ROWS(TH, NV) \
    hipLaunchKernelGGL((ov_q8_rows_kernel<T, TH, NV>), dim3((unsigned)(TH < 256 ? ((int64_t)M + 3) / 4 : (int64_t)M)), dim3(TH < 256 ? 256 : TH), 0, st, xt, ldx, rows, n_src, M, K, q, \
                       ldq, kst, kpad, scale)
    switch (ov_q8_row_threads(p, M)) {
        case 64: if (p <= 64) { OV_Q8_ROWS(64, 1); } else { OV_Q8_ROWS(64, 4); } break;
        case 256: OV_Q8_ROWS(256, 4); break;
        case 512: if (p <= 2048) { OV_Q8_ROWS(512, 4); } else { OV_Q8_ROWS(512, 10); } break;
        default: if (p <= 5120) { OV_Q8_ROWS(1024, 5); } else { OV_Q8_ROWS(1024, 16); } break;
    }
#undef OV_Q8_ROWS
}

static int ov_q8_rows_any(const void* x, int dtype, int64_t ldx, const int32_t* rows, int n_src, int M, int K, int8_t* q, int64_t ldq, int64_t kst,
                          int64_t kpad, float* scale, hipStream_t st) {
    switch (dtype) {
        case ONTOVAE_F32: ov_q8_rows_launch<float>(x, ldx, rows, n_src, M, K, q, ldq, kst, kpad, scale, st); break;
        case ONTOVAE_BF16: ov_q8_rows_launch<ov_bf>(x, ldx, rows, n_src, M, K, q, ldq, kst, kpad, scale, st); break;
        default: ov_q8_rows_launch<ov_hf>(x, ldx, rows, n_src, M, K, q, ldq, kst, kpad, scale, st); break;
    }
    OV_OPS_LAUNCH_CHECK("quantize_rows");
    return ONTOVAE_OK;
}

extern "C" int ontovae_quantize_rows(const void* x, int32_t dtype, int64_t ldx, const int32_t* rows, int32_t n_src, int32_t M, int32_t K,
                                     int8_t* q, int64_t ldq, float* scale, void* stream) {
    if (M < 0 || K < 0 || n_src < 0 || ldx < K || ldq < K || (!rows && n_src < M)) {
        ontovae_set_error("quantize_rows: M = %d, K = %d, n_src = %d, ldx = %lld, ldq = %lld", M, K, n_src, (long long)ldx, (long long)ldq);
        return ONTOVAE_EINVAL;
    }
    if (K > (1 << 30)) { ontovae_set_error("quantize_rows: K = %d, rows of up to 2^30 elements", K); return ONTOVAE_EINVAL; }
    if (dtype < ONTOVAE_F32 || dtype > ONTOVAE_F16) { ontovae_set_error("quantize_rows: unknown element type %d", dtype); return ONTOVAE_EINVAL; }
    if (!ov_q8_rows_fit(dtype, M, K)) { ontovae_set_error("quantize_rows: %d rows of %d are too many for one launch", M, K); return ONTOVAE_EINVAL; }
    if (M == 0) return ONTOVAE_OK;
    if (!scale || (K > 0 && (!x || !q))) { ontovae_set_error("quantize_rows: NULL argument"); return ONTOVAE_EINVAL; }
    return ov_q8_rows_any(x, dtype, ldx, rows, n_src, M, K, q, ldq, 128, ldq, scale, reinterpret_cast<hipStream_t>(stream));
}

// Tile and split of a product.
struct OvQ8Plan { int cfg, splits, kchunk; };
enum { OV_Q8_T32 = 0, OV_Q8_T64 = 1, OV_Q8_T128 = 2, OV_Q8_T192 = 3, OV_Q8_T256 = 4 };
static const int ov_q8_bm[5] = {32, 64, 128, 128, 256}, ov_q8_bn[5] = {128, 64, 128, 192, 256};

// The form with the least estimated time: rounds of 256 workgroups at the share of the matrix rate that each tile reaches
// (measured over 128 <= M, N <= 16384, 2048 <= K <= 20000), plus what cutting K costs: the slabs written and read, and a launch.
// 8192^3: 256 x 256 518 us, 128 x 192 656, 128 x 128 684, 64 x 64 905; 16384 x 360 x 20000: 128 x 192 167 us, 256 x 256 in slabs 191,
// 128 x 128 229; 4096 x 360 x 20000: 128 x 192 in 4 slabs 55 us, 64 x 64 uncut 76; 2048^3: 128 x 128 18.2 us, 128 x 192 19.0, 64 x 64 19.7.
static OvQ8Plan ov_q8_plan(int64_t M, int64_t N, int K) {
    static const double share[5] = {0.15, 0.24, 0.32, 0.33, 0.45};
    const int steps = std::max((K + 127) / 128, 1);
    OvQ8Plan best{};
    double least = 1e300;
    for (int c = M <= 32 ? OV_Q8_T32 : OV_Q8_T64; c <= (M <= 32 ? OV_Q8_T32 : OV_Q8_T256); ++c) {
        const int64_t t = ((M + ov_q8_bm[c] - 1) / ov_q8_bm[c]) * ((N + ov_q8_bn[c] - 1) / ov_q8_bn[c]);
        const int cut = (int)std::min<int64_t>((256 + t - 1) / t, std::max(steps / 4, 1));      // a slab has 4 steps at least
        for (int s : {1, cut}) {
            const int per = (steps + s - 1) / s, n = (steps + per - 1) / per;
            const double us = (double)((t * n + 255) / 256) * ov_q8_bm[c] * ov_q8_bn[c] * per * 128 / (9.8e6 * share[c]) +
                              (n > 1 ? 4.0 + (double)n * M * N * 8 / 5e6 : 0.0);
            if (us < least) { least = us; best = OvQ8Plan{c, n, per * 128}; }
        }
    }
    return best;
}

template <int BM, int BN, int WM, int WN, int BK, int ST, bool DIRECT, typename T>
static int ov_q8_gemm_go(const OvQ8Gemm& g, int splits, hipStream_t st) {
    constexpr int THREADS = (BM / WM) * (BN / WN) * 64, LDS = (DIRECT ? ST : 2) * (BM + BN) * BK;
    auto* fn = ov_q8_gemm_kernel<BM, BN, WM, WN, BK, ST, DIRECT, T>;
    static std::atomic<uint64_t> raised{0};                               // bit = device: the limit is raised once
    int dev = 0;
    if (LDS > 65536 && (hipGetDevice(&dev) != hipSuccess || dev > 63 || !(raised.load() >> dev & 1))) {
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) { ontovae_set_error("int8_matmul: %d bytes of LDS: %s", LDS, hipGetErrorString(e)); return ONTOVAE_EHIP; }
        if (dev >= 0 && dev < 64) raised |= 1ull << dev;
    }
    hipLaunchKernelGGL(fn, dim3(g.nm * g.nn, splits), dim3(THREADS), LDS, st, g);
    return ONTOVAE_OK;
}

template <typename T>
static int ov_q8_gemm_launch(OvQ8Gemm g, const OvQ8Plan& p, bool direct, hipStream_t st) {
    g.nm = (g.M + ov_q8_bm[p.cfg] - 1) / ov_q8_bm[p.cfg];
    g.nn = (g.N + ov_q8_bn[p.cfg] - 1) / ov_q8_bn[p.cfg];
    g.kchunk = p.kchunk;
    if (!direct) {
        g.nm = (g.M + 63) / 64;
        g.nn = (g.N + 63) / 64;
        return ov_q8_gemm_go<64, 64, 32, 32, 128, 2, false, T>(g, p.splits, st);
    }
    switch (p.cfg) {
        case OV_Q8_T32: return ov_q8_gemm_go<32, 128, 32, 32, 128, 4, true, T>(g, p.splits, st);
        case OV_Q8_T64: return ov_q8_gemm_go<64, 64, 32, 32, 128, 4, true, T>(g, p.splits, st);
        case OV_Q8_T128: return ov_q8_gemm_go<128, 128, 64, 64, 64, 4, true, T>(g, p.splits, st);
        case OV_Q8_T192: return ov_q8_gemm_go<128, 192, 32, 96, 128, 3, true, T>(g, p.splits, st);
        default: return ov_q8_gemm_go<256, 256, 128, 64, 64, 4, true, T>(g, p.splits, st);
    }
}

extern "C" int64_t ontovae_int8_matmul_workspace_bytes(int32_t M, int32_t N, int32_t K) {
    if (M <= 0 || N <= 0 || K < 0 || K > OV_Q8_MAX_K || std::max(M, N) > OV_Q8_MAX_MN) return 0;
    const OvQ8Plan p = ov_q8_plan(M, N, K);
    return p.splits > 1 ? (int64_t)p.splits * M * N * 4 : 0;
}

// operands whose rows start on 16 B, at 32-bit offsets inside a tile
static bool ov_q8_direct(const int8_t* a, int64_t lda, const int8_t* b, int64_t ldb) {
    return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | (uintptr_t)lda | (uintptr_t)ldb) & 15) == 0 &&
           std::max(lda, ldb) < (1 << 23);
}
// more tiles than one launch takes (tiles of 64 x 64 by 256 threads where the operands are not direct)
static bool ov_q8_too_many(int64_t M, int64_t N, int K, bool direct) {
    if (std::max(M, N) > OV_Q8_MAX_MN) return true;
    const int cfg = direct ? ov_q8_plan(M, N, K).cfg : OV_Q8_T64;
    return !ov_ops_fits(((M + ov_q8_bm[cfg] - 1) / ov_q8_bm[cfg]) * ((N + ov_q8_bn[cfg] - 1) / ov_q8_bn[cfg]), cfg >= OV_Q8_T192 ? 512 : 256);
}

// the product on checked arguments; column k of row m of a at (k / 128) ast + m lda + k % 128
static int ov_q8_matmul(const int8_t* a, int64_t lda, int64_t ast, const float* sa, const int8_t* b, int64_t ldb, const float* sb, const float* bias,
                        int M, int N, int K, void* y, int dtype, int64_t ldy, void* workspace, hipStream_t st) {
    const OvQ8Plan p = ov_q8_plan(M, N, K);
    const bool direct = ov_q8_direct(a, lda, b, ldb);
    OvQ8Gemm g{a, lda, ast, b, ldb, sa, sb, bias, M, N, K, 0, 0, 0, static_cast<int32_t*>(workspace), y, ldy};
    int rc;
    if (p.splits > 1) {
        if ((rc = ov_q8_gemm_launch<int32_t>(g, p, direct, st))) return rc;
        const dim3 grid((unsigned)std::min<int64_t>(((int64_t)M * N + 255) / 256, 4096));
        switch (dtype) {
            case ONTOVAE_F32: hipLaunchKernelGGL(ov_q8_combine_kernel<float>, grid, dim3(256), 0, st, g, p.splits); break;
            case ONTOVAE_BF16: hipLaunchKernelGGL(ov_q8_combine_kernel<ov_bf>, grid, dim3(256), 0, st, g, p.splits); break;
            default: hipLaunchKernelGGL(ov_q8_combine_kernel<ov_hf>, grid, dim3(256), 0, st, g, p.splits); break;
        }
    } else {
        switch (dtype) {
            case ONTOVAE_F32: rc = ov_q8_gemm_launch<float>(g, p, direct, st); break;
            case ONTOVAE_BF16: rc = ov_q8_gemm_launch<ov_bf>(g, p, direct, st); break;
            default: rc = ov_q8_gemm_launch<ov_hf>(g, p, direct, st); break;
        }
        if (rc) return rc;
    }
    OV_OPS_LAUNCH_CHECK("int8_matmul");
    return ONTOVAE_OK;
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
    if (ov_q8_too_many(M, N, K, ov_q8_direct(a, lda, b, ldb))) { ontovae_set_error("int8_matmul: M = %d, N = %d: too many tiles", M, N); return ONTOVAE_EINVAL; }
    const int64_t need = ontovae_int8_matmul_workspace_bytes(M, N, K);
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255))) {
        ontovae_set_error("int8_matmul: workspace of %lld bytes, 256-B aligned, needed", (long long)need);
        return ONTOVAE_EINVAL;
    }
    return ov_q8_matmul(a, lda, 128, sa, b, ldb, sb, bias, M, N, K, y, dtype, ldy, workspace, reinterpret_cast<hipStream_t>(stream));
}

// ---- linear layer with its input quantised on the way
// The rows in 8 bits live in the workspace in blocks of 128 columns, [K / 128][M][128]: a step of a tile then reads one
// contiguous run instead of one cache line from each of its rows (16384 x 20000 against 360 columns: 12 % of the
// product).
static int64_t ov_q8_blocks(int K) { return std::max<int64_t>(((int64_t)K + 127) / 128, 1); }
// few rows: the fused kernel.  Up to 4 rows and 8 pieces of 16 columns per thread (K <= 32768), 32 registers a row
static bool ov_q8_few(int M, int K) { return M <= 4 && K <= 32768 && (M <= 2 || K <= 20480); }

extern "C" int64_t ontovae_int8_linear_workspace_bytes(int32_t M, int32_t N, int32_t K) {
    if (M <= 0 || N <= 0 || K < 0 || K > OV_Q8_MAX_K || std::max(M, N) > OV_Q8_MAX_MN || ov_q8_few(M, K)) return 0;
    const int64_t head = (M * ov_q8_blocks(K) * 128 + 255) / 256 * 256 + ((int64_t)M * 4 + 255) / 256 * 256;
    return head + ontovae_int8_matmul_workspace_bytes(M, N, K);
}

// K is cut only where a form has t < 256 tiles, into at most 256 / t + 1 slabs of at most t whole tiles, and never below 4 steps
int64_t ov_int8_linear_bytes_upto(int max_M, int N, int K) {
    int64_t slabs = 0;
    for (int c = 0; c < 5; ++c) {
        const int64_t t = std::min<int64_t>((((int64_t)max_M + ov_q8_bm[c] - 1) / ov_q8_bm[c]) * (((int64_t)N + ov_q8_bn[c] - 1) / ov_q8_bn[c]), 255);
        slabs = std::max(slabs, (256 + t) * ov_q8_bm[c] * ov_q8_bn[c]);
    }
    const int64_t cuts = std::min<int64_t>(256, std::max((K + 127) / 128 / 4, 1));
    const int64_t one = std::min<int64_t>((int64_t)max_M * N, slabs);        // `slabs` stays below 2^26: no product wraps
    slabs = std::min(slabs, cuts * one);
    return (max_M * ov_q8_blocks(K) * 128 + 255) / 256 * 256 + ((int64_t)max_M * 4 + 255) / 256 * 256 + slabs * 4;
}

template <typename T, int MT>
static void ov_q8_few_go(const void* x, int64_t ldx, const int32_t* rows, int n_src, int M, const OvQ8Gemm& g, int ytype, hipStream_t st) {
    const T* xt = static_cast<const T*>(x);
    const dim3 grid((unsigned)std::min(g.N, 512));
    const int np = (g.K + 4095) / 4096;
    if (np <= 1) hipLaunchKernelGGL((ov_q8_few_kernel<T, MT, 1>), grid, dim3(256), 0, st, xt, ldx, rows, n_src, M, g, ytype);
    else if (np <= 2) hipLaunchKernelGGL((ov_q8_few_kernel<T, MT, 2>), grid, dim3(256), 0, st, xt, ldx, rows, n_src, M, g, ytype);
    else if (np <= 5) hipLaunchKernelGGL((ov_q8_few_kernel<T, MT, 5>), grid, dim3(256), 0, st, xt, ldx, rows, n_src, M, g, ytype);
    else if constexpr (MT <= 2) hipLaunchKernelGGL((ov_q8_few_kernel<T, MT, 8>), grid, dim3(256), 0, st, xt, ldx, rows, n_src, M, g, ytype);
}
template <typename T>
static void ov_q8_few_launch(const void* x, int64_t ldx, const int32_t* rows, int n_src, int M, const OvQ8Gemm& g, int ytype, hipStream_t st) {
    if (M == 1) ov_q8_few_go<T, 1>(x, ldx, rows, n_src, M, g, ytype, st);
    else if (M == 2) ov_q8_few_go<T, 2>(x, ldx, rows, n_src, M, g, ytype, st);
    else ov_q8_few_go<T, 4>(x, ldx, rows, n_src, M, g, ytype, st);
}

extern "C" int ontovae_int8_linear(const void* x, int32_t dtype, int64_t ldx, const int32_t* rows, int32_t n_src, const int8_t* w, int64_t ldw,
                                   const float* sw, const float* bias, int32_t M, int32_t N, int32_t K, void* y, int32_t ydtype, int64_t ldy,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
    if (M < 0 || N < 0 || K < 0 || n_src < 0 || ldx < K || ldw < K || ldy < N || (!rows && n_src < M)) {
        ontovae_set_error("int8_linear: M = %d, N = %d, K = %d, n_src = %d, ldx = %lld, ldw = %lld, ldy = %lld", M, N, K, n_src, (long long)ldx,
                          (long long)ldw, (long long)ldy);
        return ONTOVAE_EINVAL;
    }
    if (K > OV_Q8_MAX_K) { ontovae_set_error("int8_linear: K = %d, the sums are exact in 32 bits up to %d", K, OV_Q8_MAX_K); return ONTOVAE_EINVAL; }
    if (dtype < ONTOVAE_F32 || dtype > ONTOVAE_F16 || ydtype < ONTOVAE_F32 || ydtype > ONTOVAE_F16) {
        ontovae_set_error("int8_linear: unknown element type %d / %d", dtype, ydtype);
        return ONTOVAE_EINVAL;
    }
    if (M == 0 || N == 0) return ONTOVAE_OK;
    if (!sw || !y || (K > 0 && (!x || !w))) { ontovae_set_error("int8_linear: NULL argument"); return ONTOVAE_EINVAL; }
    // the few-row form has its own, small grid; for the others the rows in 8 bits are laid out in the workspace for the direct form
    const bool few = ov_q8_few(M, K);
    if (std::max(M, N) > OV_Q8_MAX_MN || (!few && (ov_q8_too_many(M, N, K, ov_q8_direct(nullptr, 128, w, ldw)) || !ov_q8_rows_fit(dtype, M, K)))) {
        ontovae_set_error("int8_linear: M = %d, N = %d, K = %d are too many for one launch", M, N, K);
        return ONTOVAE_EINVAL;
    }
    const int64_t need = ontovae_int8_linear_workspace_bytes(M, N, K);
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255))) {
        ontovae_set_error("int8_linear: workspace of %lld bytes, 256-B aligned, needed", (long long)need);
        return ONTOVAE_EINVAL;
    }
    if (few) {
        hipStream_t st = reinterpret_cast<hipStream_t>(stream);
        OvQ8Gemm g{nullptr, 0, 0, w, ldw, nullptr, sw, bias, M, N, K, 0, 0, 0, nullptr, y, ldy};
        if (dtype == ONTOVAE_F32) ov_q8_few_launch<float>(x, ldx, rows, n_src, M, g, ydtype, st);
        else if (dtype == ONTOVAE_BF16) ov_q8_few_launch<ov_bf>(x, ldx, rows, n_src, M, g, ydtype, st);
        else ov_q8_few_launch<ov_hf>(x, ldx, rows, n_src, M, g, ydtype, st);
        OV_OPS_LAUNCH_CHECK("int8_linear");
        return ONTOVAE_OK;
    }
    const int64_t nb = ov_q8_blocks(K), kst = (int64_t)M * 128;
    char* p = static_cast<char*>(workspace);
    int8_t* q = reinterpret_cast<int8_t*>(p);
    p += (M * nb * 128 + 255) / 256 * 256;
    float* s = reinterpret_cast<float*>(p);
    p += ((int64_t)M * 4 + 255) / 256 * 256;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    int rc = ov_q8_rows_any(x, dtype, ldx, rows, n_src, M, K, q, 128, kst, nb * 128, s, st);
    if (rc) return rc;
    return ov_q8_matmul(q, 128, kst, s, w, ldw, sw, bias, M, N, K, y, ydtype, ldy, p, st);
}

#endif

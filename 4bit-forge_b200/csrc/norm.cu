// Root-mean-square norm of a row, with the residual's addition in front of it and, optionally, an 8-bit output:
//   h = x + residual (fp32),   y = h * rsqrt(mean(h^2) + eps) * weight,   r = round(h)
//   quantised form, per 128 consecutive channels of a row:  s = max(max|y|, 1e-12) / 448,  q = e4m3(y / s)
// and its backward pass at the stored stream r:
//   n = r * rstd,  t = dy * weight,  dx = rstd * (t - n * mean(t n)) + dresidual,  dweight = sum over rows of dy * n
//
// Bound by HBM: a row is read once, kept in registers across the reduction, and written once.  One row belongs to a warp
// (up to 512 channels) or to a CTA, eight or sixteen channels a thread.
// Rows of more than 16384 channels (backward: 8192), not of a multiple of 8 of them, or not 16-byte aligned take the strided
// kernels below, which read a row twice (the second time from cache); so do some rows of fp32 (launch_fwd).
// Backward: 5003 x 2048 with dresidual (82 MB) 17 us, and 4 us for the column sums.
// dweight: every CTA walks rows and keeps its columns' sums in registers; one fp32 partial row per CTA, summed in a
// fixed order by a second launch, so results do not depend on scheduling.
#include "common.cuh"
#include "column_sum.cuh"
#include "elem.cuh"
#include "tcgen05.cuh"

using namespace forge;

namespace {

constexpr int kQGroup = 128;
constexpr float kF8Max = 448.0f, kAmaxFloor = 1e-12f;

struct NormParams {
    const void *x, *res, *w;
    int64_t ldx, ldres, T, C;
    int w_f32;
    float eps;
    void *y;             // element type, [T, C]; or e4m3 when scales is given
    float *scales;       // [T, ceil(C/128)]
    void *r;             // [T, C], written when res is given
};
struct NormBwdParams {
    const void *dy, *x, *w, *dres;
    int64_t lddy, ldx, lddres, T, C;
    int w_f32;
    float eps;
    void *dx;
    float *partial;      // [n_partial, C]
    float *stats;        // [2, T]: rstd, mean(t n) (strided form only)
    int n_partial;
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

// Sum over the threads of a row: every thread gets it.  `slot` holds one float per warp and is used once per call site
// and row (two slots alternate where a kernel walks several rows).
template <bool CTA> __device__ __forceinline__ float row_sum(float v, float *slot) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (CTA) {
        const int lane = threadIdx.x & 31;
        if (lane == 0) slot[threadIdx.x >> 5] = v;
        __syncthreads();
        v = lane < (int)(blockDim.x >> 5) ? slot[lane] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}

template <typename T> __device__ __forceinline__ float load_w(const void *w, int w_f32, int64_t c) {
    return w_f32 ? ((const float *)w)[c] : Elem<T>::to_f(((const T *)w)[c]);
}

// CTAs of as many warps as a row's vectors fill walk the rows (WARP: a warp a row, eight a CTA) with the next four rows on
// their way into shared memory.  A row is a chain of load, reduction and store of about a microsecond, so what keeps HBM
// busy is the bytes in flight beside it: 8192 x 7168 with residual to e4m3 (413 MB) took 87 us with one row a CTA and
// two CTAs an SM, and takes 77 us this way (5.4 TB/s, 0.82 of the measured copy rate).  A thread copies (cp.async) and reads
// its own vectors only, so the ring needs no barrier.
// A thread takes two vectors of rows that are longer than a CTA of 1024 threads of one (512 in fp32); those rows are large
// enough to keep HBM busy with three under way, and 128 KB of fp32 with one.
constexpr int ring_depth(int es, bool warp, int nv, int threads) { return warp || nv == 1 ? 4 : es * threads <= 2048 ? 3 : 1; }
constexpr int ring_bytes(int es, int nv, int threads, int deep, int arrays) { return deep * arrays * nv * es / 2 * threads * 16; }

// TMAX: most threads of a CTA
template <typename T, bool WARP, int NV, int TMAX>
__global__ void __launch_bounds__(TMAX) rmsnorm_kernel(const NormParams P) {
    constexpr int kQ = sizeof(T) / 2;                     // 16-byte pieces of a vector
    constexpr int kDeep = ring_depth(sizeof(T), WARP, NV, TMAX);
    extern __shared__ uint4 ring[];                       // [kDeep][x, residual][NV][kQ][threads]
    __shared__ float slot[2][32];
    const int TPR = WARP ? 32 : (int)blockDim.x, t = WARP ? threadIdx.x % 32 : threadIdx.x, C = (int)P.C;
    const int64_t step = WARP ? (int64_t)gridDim.x * 8 : gridDim.x;
    const int64_t row0 = WARP ? (int64_t)blockIdx.x * 8 + threadIdx.x / 32 : blockIdx.x;
    const int arrays = P.res ? 2 : 1;
    const auto place = [&](int s, int a, int i, int k) -> uint4 * {
        return ring + ((((s * arrays + a) * NV + i) * kQ + k) * (int)blockDim.x + (int)threadIdx.x);
    };
    const auto fetch = [&](int64_t row, int s) {
        if (row < P.T)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (t + i * TPR) * 8;
                if (c < C)
#pragma unroll
                    for (int k = 0; k < kQ; ++k) {
                        tc::cp_async16_zfill(tc::smem_u32(place(s, 0, i, k)),
                                             reinterpret_cast<const uint4 *>((const T *)P.x + row * P.ldx + c) + k, true);
                        if (P.res)
                            tc::cp_async16_zfill(tc::smem_u32(place(s, 1, i, k)),
                                                 reinterpret_cast<const uint4 *>((const T *)P.res + row * P.ldres + c) + k, true);
                    }
            }
        tc::cp_async_commit();
    };
    const auto take = [&](int s, int a, int i, float (&v)[8]) {
        Raw8<T> r;
        if ((t + i * TPR) * 8 < C)
#pragma unroll
            for (int k = 0; k < kQ; ++k) r.q[k] = *place(s, a, i, k);
        else
            r.zero();
        r.get(v);
    };
    Raw8<T> hw[NV];
#pragma unroll
    for (int a = 0; a < kDeep; ++a) fetch(row0 + a * step, a);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * 8;
        hw[i].zero();
        if (c < C && !P.w_f32) hw[i].load((const T *)P.w + c);
    }
    int flip = 0, s = 0;
    for (int64_t row = row0; row < P.T; row += step, s = (s + 1) % kDeep) {
        tc::cp_async_wait<kDeep - 1>();
        float h[NV][8], ss = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * 8;
            take(s, 0, i, h[i]);
            if (P.res) {
                float v[8];
                take(s, 1, i, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) h[i][e] += v[e];
                if (c < C) store8((T *)P.r + row * P.C + c, h[i]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(h[i][e], h[i][e], ss);
        }
        fetch(row + kDeep * step, s);
        const float rstd = rsqrtf(row_sum<!WARP>(ss, slot[flip]) / (float)C + P.eps);
        flip ^= 1;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * 8;
            float w[8] = {}, amax = kAmaxFloor;
            if (!P.w_f32) hw[i].get(w);
            else if (c < C) load8((const float *)P.w + c, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                h[i][e] = h[i][e] * rstd * w[e];
                if (c < C) amax = max_nan(amax, fabsf(h[i][e]));   // channels past the row are not part of its group
            }
            if (!P.scales) {
                if (c < C) store8((T *)P.y + row * P.C + c, h[i]);
                continue;
            }
            // 16 neighbouring threads hold a group of 128 channels
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            const float sc = amax / kF8Max, inv = 1.0f / sc;       // (a division a value: 100 us in place of 77)
            if (c < C) {
                uint2 out;
                out.x = e4m3x4(h[i][0] * inv, h[i][1] * inv, h[i][2] * inv, h[i][3] * inv);
                out.y = e4m3x4(h[i][4] * inv, h[i][5] * inv, h[i][6] * inv, h[i][7] * inv);
                *reinterpret_cast<uint2 *>((uint8_t *)P.y + row * P.C + c) = out;
                if ((t & 15) == 0) P.scales[row * cdiv(P.C, (int64_t)kQGroup) + c / kQGroup] = sc;
            }
        }
    }
    tc::cp_async_wait<0>();
}

// Any length, stride and alignment: the row is read twice.
template <typename T> __global__ void __launch_bounds__(256) rmsnorm_strided_kernel(const NormParams P) {
    __shared__ float slot[32];
    const int64_t row = blockIdx.x;
    const T *x = (const T *)P.x + row * P.ldx;
    const T *res = P.res ? (const T *)P.res + row * P.ldres : nullptr;
    float ss = 0.0f;
    for (int64_t c = threadIdx.x; c < P.C; c += 256) {
        float h = Elem<T>::to_f(x[c]);
        if (res) {
            h += Elem<T>::to_f(res[c]);
            ((T *)P.r)[row * P.C + c] = Elem<T>::from_f(h);
        }
        ss = fmaf(h, h, ss);
    }
    const float rstd = rsqrtf(row_sum<true>(ss, slot) / (float)P.C + P.eps);
    if (!P.scales) {
        for (int64_t c = threadIdx.x; c < P.C; c += 256) {
            float h = Elem<T>::to_f(x[c]);
            if (res) h += Elem<T>::to_f(res[c]);
            ((T *)P.y)[row * P.C + c] = Elem<T>::from_f(h * rstd * load_w<T>(P.w, P.w_f32, c));
        }
        return;
    }
    const int64_t G = cdiv(P.C, (int64_t)kQGroup);
    const int lane = threadIdx.x & 31;
    for (int64_t g = threadIdx.x >> 5; g < G; g += 8) {      // a warp per group of 128 channels
        float v[4], amax = kAmaxFloor;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t c = g * kQGroup + k * 32 + lane;
            v[k] = 0.0f;
            if (c < P.C) {
                float h = Elem<T>::to_f(x[c]);
                if (res) h += Elem<T>::to_f(res[c]);
                v[k] = h * rstd * load_w<T>(P.w, P.w_f32, c);
                amax = max_nan(amax, fabsf(v[k]));
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const float s = amax / kF8Max, inv = 1.0f / s;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t c = g * kQGroup + k * 32 + lane;
            if (c < P.C)
                ((uint8_t *)P.y)[row * P.C + c] = __nv_cvt_float_to_fp8(v[k] * inv, __NV_SATFINITE, __NV_E4M3);
        }
        if (lane == 0) P.scales[row * G + g] = s;
    }
}

// Backward: every CTA (or warp, TPR = 32) walks rows; column sums of dy * n stay in registers.
// CTAs on an SM, as many as the registers hold (16-bit rows of 257 to 512 channels, two vectors a lane: 64000 x 512 take 48 us
// with two and took 106 with three, which spilled 370 bytes a thread)
constexpr int bwd_per_sm(int tpr, int nv) { return tpr == 128 ? 6 : tpr == 32 && nv == 2 ? 2 : tpr <= 256 ? 3 : 1; }
template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, sizeof(T) == 2 ? bwd_per_sm(TPR, NV) : 1)
rmsnorm_bwd_kernel(const NormBwdParams P) {
    constexpr int kRows = TPR == 32 ? 8 : 1;
    __shared__ float slot[2][2][32];
    const int t = threadIdx.x % TPR;
    const int C = (int)P.C;
    const int64_t unit = (int64_t)blockIdx.x * kRows + (TPR == 32 ? threadIdx.x / 32 : 0);
    const int64_t units = (int64_t)gridDim.x * kRows;
    float w[NV][8], dw[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) w[i][e] = dw[i][e] = 0.0f;
        if (c < C) {
            if (P.w_f32) load8((const float *)P.w + c, w[i]);
            else load8((const T *)P.w + c, w[i]);
        }
    }
    Raw8<T> rx[NV], rg[NV], rd[NV];
    const auto fetch = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * 8;
            rx[i].zero(); rg[i].zero();
            if (c < C && row < P.T) {
                rx[i].load((const T *)P.x + row * P.ldx + c);
                rg[i].load((const T *)P.dy + row * P.lddy + c);
            }
        }
    };
    fetch(unit);
    int flip = 0;
    for (int64_t row = unit; row < P.T; row += units, flip ^= 1) {
        float r[NV][8], g[NV][8];
        float ss = 0.0f, dot = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * 8;
            rx[i].get(r[i]);
            rg[i].get(g[i]);
            if (P.dres && c < C) rd[i].load((const T *)P.dres + row * P.lddres + c);
        }
        fetch(row + units);                       // under way while this row is reduced
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                ss = fmaf(r[i][e], r[i][e], ss);
                dot = fmaf(g[i][e] * w[i][e], r[i][e], dot);
            }
        ss = row_sum<(TPR > 32)>(ss, slot[flip][0]);
        dot = row_sum<(TPR > 32)>(dot, slot[flip][1]);
        const float rstd = rsqrtf(ss / (float)C + P.eps);
        const float c1 = dot * rstd / (float)C;                 // mean(t n)
        T *dx = (T *)P.dx + row * P.C;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * 8;
            if (c < C) {
                float o[8], d[8] = {};
                if (P.dres) rd[i].get(d);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float n = r[i][e] * rstd;
                    dw[i][e] = fmaf(g[i][e], n, dw[i][e]);
                    o[e] = rstd * (g[i][e] * w[i][e] - n * c1) + d[e];
                }
                store8(dx + c, o);
            }
        }
    }
    float *part = P.partial + unit * P.C;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * 8;
        if (c < C) store8(part + c, dw[i]);
    }
}

template <typename T> __global__ void __launch_bounds__(256) rmsnorm_bwd_strided_kernel(const NormBwdParams P) {
    __shared__ float slot[2][32];
    const int64_t row = blockIdx.x;
    const T *x = (const T *)P.x + row * P.ldx, *dy = (const T *)P.dy + row * P.lddy;
    float ss = 0.0f, dot = 0.0f;
    for (int64_t c = threadIdx.x; c < P.C; c += 256) {
        const float r = Elem<T>::to_f(x[c]);
        ss = fmaf(r, r, ss);
        dot = fmaf(Elem<T>::to_f(dy[c]) * load_w<T>(P.w, P.w_f32, c), r, dot);
    }
    ss = row_sum<true>(ss, slot[0]);
    dot = row_sum<true>(dot, slot[1]);
    const float rstd = rsqrtf(ss / (float)P.C + P.eps), c1 = dot * rstd / (float)P.C;
    if (threadIdx.x == 0) P.stats[row] = rstd;
    for (int64_t c = threadIdx.x; c < P.C; c += 256) {
        float o = rstd * (Elem<T>::to_f(dy[c]) * load_w<T>(P.w, P.w_f32, c) - Elem<T>::to_f(x[c]) * rstd * c1);
        if (P.dres) o += Elem<T>::to_f(((const T *)P.dres)[row * P.lddres + c]);
        ((T *)P.dx)[row * P.C + c] = Elem<T>::from_f(o);
    }
}
// column sums for the strided form: partial row blockIdx.y covers its share of the rows
template <typename T> __global__ void __launch_bounds__(256) rmsnorm_dw_strided_kernel(const NormBwdParams P) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= P.C) return;
    const int64_t per = cdiv(P.T, (int64_t)P.n_partial);
    const int64_t r0 = blockIdx.y * per, r1 = imin64(P.T, r0 + per);
    float s = 0.0f;
#pragma unroll 4
    for (int64_t row = r0; row < r1; ++row)
        s = fmaf(Elem<T>::to_f(((const T *)P.dy)[row * P.lddy + c]),
                 Elem<T>::to_f(((const T *)P.x)[row * P.ldx + c]) * P.stats[row], s);
    P.partial[(int64_t)blockIdx.y * P.C + c] = s;
}

constexpr int64_t kMaxRows = 0x7fffffffLL;       // one CTA per row at most
// CTAs that walk the rows in the backward pass: as many as the SMs hold
int bwd_cap(int tpr, int nv) { return 148 * bwd_per_sm(tpr, nv); }

bool vec_ok(const void *p, int64_t ld, size_t es) { return ((uintptr_t)p % 16 == 0) && (ld * (int64_t)es) % 16 == 0; }
// The row-in-registers backward kernels: (threads per row, vectors per thread) by length; 0 = strided form.  1024 threads of two
// vectors have no room for a longer row: 2048 x 8200 took 127 us so (fp32 189) and takes 58 (89) in the strided form, 16384
// channels 155 against 137 (268 against 200); 8192 channels take 27 us in registers and 57 strided.
struct RowShape { int tpr, nv; };
RowShape row_shape(int64_t C) {
    if (C <= 256) return {32, 1};
    if (C <= 512) return {32, 2};
    if (C <= 1024) return {128, 1};
    if (C <= 2048) return {256, 1};
    if (C <= 4096) return {512, 1};
    if (C <= 8192) return {512, 2};
    return {0, 0};
}

template <typename T, bool WARP, int NV, int TMAX> int launch_rows(const NormParams &P, int threads, cudaStream_t st) {
    constexpr int kDeep = ring_depth(sizeof(T), WARP, NV, TMAX), kMost = ring_bytes(sizeof(T), NV, TMAX, kDeep, 2);
    static_assert(kMost <= 192 * 1024, "the ring fits an SM");
    const int smem = ring_bytes(sizeof(T), NV, threads, kDeep, P.res ? 2 : 1);
    const auto kernel = rmsnorm_kernel<T, WARP, NV, TMAX>;
    // one limit for every launch of the kernel: another thread's call may set it between this one's two steps
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (e != cudaSuccess) {
        set_error("forge_rmsnorm: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
        return FORGE_ERR_LAUNCH;
    }
    const int64_t per_sm = 1024 / threads;                 // CTAs on an SM: 1024 threads, 192 KB of ring at most
    const int64_t rows = WARP ? cdiv(P.T, (int64_t)8) : P.T;
    kernel<<<(unsigned)imin64(rows, 148 * per_sm), threads, smem, st>>>(P);
    return FORGE_OK;
}
template <typename T> int launch_fwd(const NormParams &P, bool vec, cudaStream_t st) {
    constexpr int kRow = sizeof(T) == 2 ? 1024 : 512;      // threads of a row of one vector each
    const int64_t vecs = P.C / 8;
    const auto warps = [](int64_t v) { return (int)((v + 31) / 32 * 32); };
    if (vec && P.C <= 256) return launch_rows<T, true, 1, 256>(P, 256, st);
    if (vec && P.C <= 512) return launch_rows<T, true, 2, 256>(P, 256, st);
    if (vec && vecs <= kRow) return launch_rows<T, false, 1, kRow>(P, warps(vecs), st);
    // Two vectors a thread.  4096 rows of 16-bit elements, ring against rows read twice: 8200 channels 37 against 48 us, with
    // residual 53 against 138; 16384 channels 53 against 97, 99 against 321.  fp32: with residual 7168 channels 115 against
    // 144 us, 16384 channels 272 against 411, but 4608 channels 95 against 89; without one 8192 channels 73 against 63.
    if (vec && (sizeof(T) == 2 || (P.res && P.C >= 5120))) {
        if (vecs <= 2 * kRow) return launch_rows<T, false, 2, kRow>(P, warps((vecs + 1) / 2), st);
        if (vecs <= 2 * 1024) return launch_rows<T, false, 2, 1024>(P, warps((vecs + 1) / 2), st);
    }
    rmsnorm_strided_kernel<T><<<(unsigned)P.T, 256, 0, st>>>(P);
    return FORGE_OK;
}

int bwd_ctas(int64_t T, RowShape s) {
    const int64_t rows = s.tpr == 32 ? 8 : 1;
    return (int)imin64(cdiv(T, rows), bwd_cap(s.tpr, s.nv));
}
int strided_partials(int64_t T) { return (int)imin64(cdiv(T, (int64_t)16), 64); }

template <typename T> void launch_bwd(NormBwdParams &P, RowShape s, cudaStream_t st) {
#define FORGE_NORM_CASE(TPR, NV)                                                                             \
    if (s.tpr == TPR && s.nv == NV) {                                                                        \
        const int ctas = bwd_ctas(P.T, s);                                                                   \
        P.n_partial = ctas * (TPR == 32 ? 8 : 1);                                                            \
        rmsnorm_bwd_kernel<T, TPR, NV><<<ctas, TPR == 32 ? 256 : TPR, 0, st>>>(P); FORGE_NOTE_LAUNCH();       \
        return;                                                                                              \
    }
    FORGE_NORM_CASE(32, 1) FORGE_NORM_CASE(32, 2) FORGE_NORM_CASE(128, 1) FORGE_NORM_CASE(256, 1)
    FORGE_NORM_CASE(512, 1) FORGE_NORM_CASE(512, 2)
#undef FORGE_NORM_CASE
    P.n_partial = strided_partials(P.T);
    rmsnorm_bwd_strided_kernel<T><<<(unsigned)P.T, 256, 0, st>>>(P); FORGE_NOTE_LAUNCH();
    rmsnorm_dw_strided_kernel<T><<<dim3((unsigned)cdiv(P.C, (int64_t)256), P.n_partial), 256, 0, st>>>(P);
    FORGE_NOTE_LAUNCH();
}

size_t elem_size(int dtype) { return dtype == FORGE_DTYPE_F32 ? 4 : 2; }
bool known_dtype(int d) { return d == FORGE_DTYPE_F32 || d == FORGE_DTYPE_BF16 || d == FORGE_DTYPE_F16; }

}  // namespace

extern "C" int forge_rmsnorm(const void *x, int64_t ldx, const void *residual, int64_t ldres, const void *weight,
                             int w_dtype, int dtype, int64_t T, int64_t C, float eps, void *y, float *scales,
                             void *residual_out, void *stream) {
    FORGE_REQUIRE(T >= 0 && T <= kMaxRows && C > 0 && C <= kMaxRows, "bad sizes");
    FORGE_REQUIRE(known_dtype(dtype), "dtype must be fp32, bf16 or fp16");
    FORGE_REQUIRE(w_dtype == dtype || w_dtype == FORGE_DTYPE_F32, "weight must be fp32 or of x's type");
    if (T == 0) return FORGE_OK;
    FORGE_REQUIRE(x && weight && y, "null pointer");
    FORGE_REQUIRE(!residual == !residual_out, "residual and residual_out go together");
    FORGE_REQUIRE((T == 1 || ldx >= C) && (!residual || T == 1 || ldres >= C), "row stride below the row length");
    NormParams P{x, residual, weight, ldx, ldres, T, C, w_dtype == FORGE_DTYPE_F32, eps, y, scales, residual_out};
    const size_t es = elem_size(dtype), ws = elem_size(w_dtype);
    const bool vec = C % 8 == 0 && vec_ok(x, ldx, es) && (!residual || (vec_ok(residual, ldres, es) &&
                     vec_ok(residual_out, C, es))) && vec_ok(weight, 0, ws) && (uintptr_t)y % 16 == 0;
    cudaStream_t st = (cudaStream_t)stream;
    const int rc = dtype == FORGE_DTYPE_F32    ? launch_fwd<float>(P, vec, st)
                   : dtype == FORGE_DTYPE_BF16 ? launch_fwd<__nv_bfloat16>(P, vec, st)
                                               : launch_fwd<__half>(P, vec, st);
    if (rc != FORGE_OK) return rc;
    FORGE_NOTE_LAUNCH();
    return check_launch("forge_rmsnorm");
}

extern "C" int64_t forge_rmsnorm_backward_workspace_bytes(int64_t T, int64_t C) {
    if (T <= 0 || C <= 0 || T > kMaxRows || C > kMaxRows) return 16;
    const RowShape s = row_shape(C);
    const int64_t a = s.tpr ? (int64_t)bwd_ctas(T, s) * (s.tpr == 32 ? 8 : 1) * C * 4 : 0;
    const int64_t b = (int64_t)strided_partials(T) * C * 4 + T * 4 + 16;
    return a > b ? a : b;
}

extern "C" int forge_rmsnorm_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, const void *weight,
                                      int w_dtype, int dtype, const void *dresidual, int64_t lddres, int64_t T,
                                      int64_t C, float eps, void *dx, void *dweight, void *ws, void *stream) {
    FORGE_REQUIRE(T >= 0 && T <= kMaxRows && C > 0 && C <= kMaxRows, "bad sizes");
    FORGE_REQUIRE(known_dtype(dtype), "dtype must be fp32, bf16 or fp16");
    FORGE_REQUIRE(w_dtype == dtype || w_dtype == FORGE_DTYPE_F32, "weight must be fp32 or of x's type");
    FORGE_REQUIRE(dweight, "null pointer");
    cudaStream_t st = (cudaStream_t)stream;
    NormBwdParams P{dy, x, weight, dresidual, lddy, ldx, lddres, T, C, w_dtype == FORGE_DTYPE_F32, eps, dx,
                    (float *)ws, nullptr, 0};
    if (T > 0) {
        FORGE_REQUIRE(dy && x && weight && dx && ws, "null pointer");
        FORGE_REQUIRE((uintptr_t)ws % 16 == 0, "workspace must be 16-byte aligned");
        FORGE_REQUIRE(T == 1 || (lddy >= C && ldx >= C && (!dresidual || lddres >= C)), "row stride below the row length");
        const size_t es = elem_size(dtype), wsz = elem_size(w_dtype);
        const bool vec = C % 8 == 0 && vec_ok(x, ldx, es) && vec_ok(dy, lddy, es) &&
                         (!dresidual || vec_ok(dresidual, lddres, es)) && vec_ok(weight, 0, wsz) && (uintptr_t)dx % 16 == 0;
        const RowShape s = vec ? row_shape(C) : RowShape{0, 0};
        P.stats = P.partial + (int64_t)strided_partials(T) * C;
        if (dtype == FORGE_DTYPE_F32) launch_bwd<float>(P, s, st);
        else if (dtype == FORGE_DTYPE_BF16) launch_bwd<__nv_bfloat16>(P, s, st);
        else launch_bwd<__half>(P, s, st);
    }
    launch_column_sum(P.partial, P.n_partial, C, dweight, w_dtype, st);
    return check_launch("forge_rmsnorm_backward");
}

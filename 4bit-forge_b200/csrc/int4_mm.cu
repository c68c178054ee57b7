// Entry points and the elementwise part of the products with packed int4 weights (the layout of forge_pack_int4, symmetric codes):
//   W[r, c] = (nibble(r, c) - 8) * scale[r, c / gs]
//   linear:  y = act(x W^T + bias) + residual            gated:  h = act(x Wg^T) * (x Wu^T)
// and their backward passes for frozen weights:
//   linear:  dz = dy * act'(z),  dx = dz W,  dbias = sum over rows of dz
//   gated:   dg = dh * u * act'(g),  du = dh * act(g),  dx = dg Wg + du Wu
//
// Backward operand: dz is the K operand of the second product and has to be a 16-bit matrix.  It is written as fp16
// (11 bits, against bf16's 8) times a power of two per token row that puts the row's largest entry just below 2^15;
// the product is multiplied by the inverse power at the end, so nothing but the rounding (2^-11 relative, half a step)
// remains.  For fp16 gradients that would be as much as their own rounding, so a second fp16 matrix holds what the first
// rounds off (22 bits together), unless dz is dy itself or zero (no activation, relu), and exact.  The weights' scales are
// split the same way, see scale_prep_kernel.
#include <cooperative_groups.h>
#include <type_traits>
#include <utility>
#include "column_sum.cuh"
#include "common.cuh"
#include "elem.cuh"
#include "int4_mm.cuh"

using namespace forge;

namespace {

// ---- backward preparation ------------------------------------------------------------------------------------------

// Scales of the backward operand.  K is the weight rows (gate and up one after the other), in blocks of kKBlock.
//   f[k]     = 2^floor(log2 max_g |s[k, g]|)                            a row's power, moved into dz
//   e        = floor(log2 max over the block's k of |s[k, g]| / f[k])   a channel group's, one per block of rows
//   s'[k, g] = s[k, g] / f[k] 2^(11 - e) <= 2^12                        as an fp16 pair (hi, lo)
//   group[block, g] = 2^(e - 11)                                        undone where the block's sums are added up
// Both are powers of two, so they cost no bits.  With 2^12 at the top a product (nibble - 8) s' stays below 2^15, and it is a
// normal fp16 number down to 2^-25 of its block's largest scale: only a scale that far below its row's AND below its block's
// group loses bits.  A cluster takes a block, a CTA of it 64 rows and a warp four: the rows' powers stay in the warp, the
// groups' maxima meet in shared memory.  Nothing but latency: 2048 rows of 16 groups take 3.7 us, 2 x 2048 rows of 56 groups
// 4.8 us (every scale read three times: 4.6 and 7.5 us; without the groups' powers, a warp a row: 2.2 and 3.8 us).
constexpr int kPrepCtas = 8, kPrepRows = 4, kPrepGroups = 1024;      // a cluster's CTAs, a warp's rows, groups at a time
constexpr int kPrepKept = 2;                  // a lane's groups whose scales stay in registers, read once
static_assert(kPrepCtas * 16 * kPrepRows == kKBlock, "a cluster of 16 warps a CTA covers a block");
__device__ __forceinline__ int exponent_of(float v) { return (int)((__float_as_uint(v) >> 23) & 255u) - 127; }
__device__ __forceinline__ float finite_abs(float v) { return isfinite(v) ? fabsf(v) : 0.0f; }
__device__ __forceinline__ float pow2_any(int e) {      // -149 <= e <= 127
    return __uint_as_float(e < -126 ? 1u << (e + 149) : (uint32_t)(e + 127) << 23);
}

__global__ void __cluster_dims__(kPrepCtas) __launch_bounds__(512)
scale_prep_kernel(const float *__restrict__ s0, const float *__restrict__ s1, int64_t R, int64_t K, int64_t G,
                  __half2 *__restrict__ pairs, float *__restrict__ f, float *__restrict__ group) {
    __shared__ int top[kPrepGroups];          // largest s / f, as the bits of a float that is not negative
    __shared__ float power[kPrepGroups];      // 2^(11 - e)
    const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t k0 = (int64_t)blockIdx.x * (16 * kPrepRows) + warp * kPrepRows, block = blockIdx.x / kPrepCtas;
    const float *row[kPrepRows];
    float kept[kPrepKept][kPrepRows], m[kPrepRows], inv[kPrepRows];
#pragma unroll
    for (int i = 0; i < kPrepRows; ++i) {
        const int64_t k = k0 + i < K ? k0 + i : K - 1;
        row[i] = k < R ? s0 + k * G : s1 + (k - R) * G;
        m[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < kPrepKept; ++j) kept[j][i] = lane + 32 * j < G ? row[i][lane + 32 * j] : 0.0f;
    }
    const int top_n = (int)imin64(G, kPrepGroups);
    for (int g = threadIdx.x; g < top_n; g += 512) top[g] = 0;
    for (int64_t g = lane + 32 * kPrepKept; g < G; g += 32)
#pragma unroll
        for (int i = 0; i < kPrepRows; ++i) m[i] = fmaxf(m[i], finite_abs(row[i][g]));
#pragma unroll
    for (int i = 0; i < kPrepRows; ++i) {
#pragma unroll
        for (int j = 0; j < kPrepKept; ++j) m[i] = fmaxf(m[i], finite_abs(kept[j][i]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m[i] = fmaxf(m[i], __shfl_xor_sync(0xffffffffu, m[i], o));
        const int e = m[i] > 0.0f ? exponent_of(m[i]) : 0;
        inv[i] = k0 + i < K ? pow2_any(-e) : 0.0f;            // (rows past the last one are no part of a maximum)
        if (lane == 0 && k0 + i < K) f[k0 + i] = pow2_any(e);
    }
    for (int64_t g0 = 0; g0 < G; g0 += kPrepGroups) {
        const int n = (int)imin64(G - g0, kPrepGroups);
        if (g0 > 0)
            for (int g = threadIdx.x; g < n; g += 512) top[g] = 0;
        __syncthreads();
        const auto raise = [&](int g, const float (&v)[kPrepRows]) {
            float t = 0.0f;
#pragma unroll
            for (int i = 0; i < kPrepRows; ++i) t = fmaxf(t, finite_abs(v[i]) * inv[i]);
            atomicMax(top + g, __float_as_int(t));
        };
        const auto write = [&](int g, const float (&v)[kPrepRows]) {
#pragma unroll
            for (int i = 0; i < kPrepRows; ++i)
                if (k0 + i < K) {
                    const float x = v[i] * inv[i] * power[g];
                    const __half hi = __float2half_rn(x);
                    pairs[(k0 + i) * G + g0 + g] = __halves2half2(hi, __float2half_rn(x - __half2float(hi)));
                }
        };
        // the groups of this turn, those in registers first
        const auto each = [&](const auto &what) {
            if (g0 == 0)
#pragma unroll
                for (int j = 0; j < kPrepKept; ++j)
                    if (lane + 32 * j < n) what(lane + 32 * j, kept[j]);
            for (int g = lane + (g0 == 0 ? 32 * kPrepKept : 0); g < n; g += 32) {
                float v[kPrepRows];
#pragma unroll
                for (int i = 0; i < kPrepRows; ++i) v[i] = row[i][g0 + g];
                what(g, v);
            }
        };
        each(raise);
        cluster.sync();
        for (int g = threadIdx.x; g < n; g += 512) {
            int t = 0;
#pragma unroll
            for (int r = 0; r < kPrepCtas; ++r) t = max(t, *cluster.map_shared_rank(top + g, r));
            const int e = t == 0 ? 0 : max(exponent_of(__int_as_float(t)), -100);      // 2^(e - 11) stays a normal number
            power[g] = pow2_any(11 - e);
            if (cluster.block_rank() == 0) group[block * G + g0 + g] = pow2_any(e - 11);
        }
        auto read = cluster.barrier_arrive();
        __syncthreads();
        each(write);
        cluster.barrier_wait(std::move(read));        // nobody clears or leaves its maxima while they are read
    }
}

struct DzParams {
    const void *dy, *z, *u;     // z NULL: act is none; u given: gated
    int64_t lddy, T, R, K, ldk; // ldk: columns of a, a multiple of 64; K = used columns
    int64_t lo;                 // 0, or ldk: what a rounds off goes lo columns behind it (the row stride is ldk + lo)
    const float *f;
    __half *a;
    float *unscale;
};
__device__ __forceinline__ float pow2_of(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127
// the largest entry of a row becomes 2^14 .. 2^15; rows of zeros and of infinities keep the factor 1
__device__ __forceinline__ int row_exponent(float amax) {
    const int e = (amax > 0.0f && isfinite(amax)) ? 14 - ilogbf(amax) : 0;
    return e > 126 ? 126 : (e < -126 ? -126 : e);
}

// One CTA per token row: the row of the K operand, its power of two, and zeros up to the padded length.
template <typename T, int ACT, bool GATED> __global__ void __launch_bounds__(256) dz_kernel(const DzParams P) {
    __shared__ float slot[8];
    const int64_t t = blockIdx.x;
    const T *dy = (const T *)P.dy + t * P.lddy;
    const T *z = (const T *)P.z + t * P.R, *u = (const T *)P.u + t * P.R;
    __half *a = P.a + t * (P.ldk + P.lo);
    const auto put = [&](int64_t k, float v) {
        const __half hi = __float2half_rn(v);
        a[k] = hi;
        if (P.lo) a[P.lo + k] = __float2half_rn(v - __half2float(hi));
    };
    float scale = 1.0f;
    for (int pass = 0; pass < 2; ++pass) {
        float amax = 0.0f;
        for (int64_t r = threadIdx.x; r < P.R; r += 256) {
            const float d = Elem<T>::to_f(dy[r]);
            const float zv = (ACT == FORGE_ACT_NONE && !GATED) ? 0.0f : Elem<T>::to_f(z[r]);
            if constexpr (GATED) {
                const float vg = d * Elem<T>::to_f(u[r]) * act_bwd<ACT>(zv) * P.f[r];
                const float vu = d * act_fwd<ACT>(zv) * P.f[P.R + r];
                if (pass == 0) amax = fmaxf(amax, fmaxf(fabsf(vg), fabsf(vu)));
                else {
                    put(r, vg * scale);
                    put(P.R + r, vu * scale);
                }
            } else {
                const float v = d * act_bwd<ACT>(zv) * P.f[r];
                if (pass == 0) amax = fmaxf(amax, fabsf(v));
                else put(r, v * scale);
            }
        }
        if (pass == 0) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = amax;
            __syncthreads();
            amax = slot[0];
#pragma unroll
            for (int w = 1; w < 8; ++w) amax = fmaxf(amax, slot[w]);
            const int e = row_exponent(amax);
            scale = pow2_of(e);
            if (threadIdx.x == 0) P.unscale[t] = pow2_of(-e);
        }
    }
    for (int64_t k = P.K + threadIdx.x; k < P.ldk; k += 256) put(k, 0.0f);
}

// The same with a row in registers (R a multiple of 8, 16-byte aligned rows, R <= 8 TPR NV): dz is computed once, rows are
// read 16 bytes at a time, and a CTA that walks several rows keeps the column sums of dz (linear form) on the way:
// partial[blockIdx.x, R] when wanted.
template <typename T, int ACT, bool GATED, int TPR, int NV>
__global__ void __launch_bounds__(TPR) dz_rows_kernel(const DzParams P, float *partial) {
    constexpr int M = GATED ? 2 : 1, W = TPR / 32;
    constexpr bool kLow = std::is_same<T, __half>::value && (GATED || (ACT != FORGE_ACT_NONE && ACT != FORGE_ACT_RELU));
    __shared__ float slot[2][W];
    const int R = (int)P.R, tid = threadIdx.x;
    float db[NV][8];
    if (!GATED)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) db[i][e] = 0.0f;
    Raw8<T> rd[NV], rz[NV], ru[NV];
    const auto fetch = [&](int64_t t) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int r = (tid + i * TPR) * 8;
            rd[i].zero(); rz[i].zero(); ru[i].zero();
            if (r < R && t < P.T) {
                rd[i].load((const T *)P.dy + t * P.lddy + r);
                if (GATED || ACT != FORGE_ACT_NONE) rz[i].load((const T *)P.z + t * P.R + r);
                if (GATED) ru[i].load((const T *)P.u + t * P.R + r);
            }
        }
    };
    fetch(blockIdx.x);
    int flip = 0;
    for (int64_t t = blockIdx.x; t < P.T; t += gridDim.x, flip ^= 1) {
        float v[M][NV][8], amax = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int r = (tid + i * TPR) * 8;
            float d[8], z[8], u[8], f[8] = {};
            rd[i].get(d);
            rz[i].get(z);
            ru[i].get(u);
            if (r < R) load8(P.f + r, f);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if constexpr (GATED) {
                    v[0][i][e] = d[e] * u[e] * act_bwd<ACT>(z[e]) * f[e];
                    v[M - 1][i][e] = d[e] * act_fwd<ACT>(z[e]);
                } else {
                    const float dz = d[e] * act_bwd<ACT>(z[e]);
                    db[i][e] += dz;
                    v[0][i][e] = dz * f[e];
                }
            }
            if constexpr (GATED) {
                if (r < R) load8(P.f + R + r, f);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[M - 1][i][e] *= f[e];
            }
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(v[m][i][e]));
        }
        fetch(t + gridDim.x);                    // under way while this row is scaled
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if ((tid & 31) == 0) slot[flip][tid >> 5] = amax;
        __syncthreads();
        amax = (tid & 31) < W ? slot[flip][tid & 31] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const int e2 = row_exponent(amax);
        const float scale = pow2_of(e2);
        if (tid == 0) P.unscale[t] = pow2_of(-e2);
        __half *a = P.a + t * (P.ldk + P.lo);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int r = (tid + i * TPR) * 8;
            if (r < R)
#pragma unroll
                for (int m = 0; m < M; ++m) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[m][i][e] *= scale;
                    store8(a + m * R + r, v[m][i]);
                    if (kLow && P.lo) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[m][i][e] -= __half2float(__float2half_rn(v[m][i][e]));
                        store8(a + P.lo + m * R + r, v[m][i]);
                    }
                }
        }
        for (int64_t k = P.K + tid; k < P.ldk; k += TPR) {
            a[k] = __float2half_rn(0.0f);
            if (kLow && P.lo) a[P.lo + k] = __float2half_rn(0.0f);
        }
    }
    if (!GATED && partial)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int r = (tid + i * TPR) * 8;
            if (r < R) store8(partial + (int64_t)blockIdx.x * R + r, db[i]);
        }
}

// Partial column sums of dz: CTA (column block, row share)
template <typename T, int ACT>
__global__ void __launch_bounds__(256) dbias_kernel(const T *__restrict__ dy, int64_t lddy, const T *__restrict__ z,
                                                    int64_t n, int64_t R, float *__restrict__ partial) {
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r >= R) return;
    const int64_t per = cdiv(n, (int64_t)gridDim.y);
    const int64_t t0 = blockIdx.y * per, t1 = imin64(n, t0 + per);
    float s = 0.0f;
#pragma unroll 4
    for (int64_t t = t0; t < t1; ++t) {
        const float d = Elem<T>::to_f(dy[t * lddy + r]);
        s = fmaf(d, ACT == FORGE_ACT_NONE ? 1.0f : act_bwd<ACT>(Elem<T>::to_f(z[t * R + r])), s);
    }
    partial[(int64_t)blockIdx.y * R + r] = s;
}
// ---- host side -------------------------------------------------------------------------------------------------------
constexpr int64_t kMaxDim = 1ll << 24;        // rows and columns of a weight matrix
constexpr int64_t kMaxTokens = 0x7fffffffLL;
constexpr int kBiasParts = 64;            // row shares of the column sums of dz, strided form
constexpr int kRowCtas = 296;             // CTAs that walk rows in the row-in-registers form, two per SM

int check_sizes(const char *who, int dtype, int64_t T, int64_t C, int64_t R, int gs, int act) {
    const char *msg = nullptr;
    if (T < 0 || T > kMaxTokens || C <= 0 || C > kMaxDim || R <= 0 || R > kMaxDim) msg = "bad sizes";
    else if (dtype != FORGE_DTYPE_BF16 && dtype != FORGE_DTYPE_F16) msg = "dtype must be bf16 or fp16";
    else if (C % 8 != 0) msg = "in_features must be a multiple of 8 (whole packed words)";
    else if (gs != 32 && gs != 64 && gs != 128) msg = "group size must be 32, 64 or 128";
    else if (act < FORGE_ACT_NONE || act > FORGE_ACT_GELU) msg = "unknown activation";
    if (!msg) return FORGE_OK;
    set_error("%s: %s", who, msg);
    return FORGE_ERR_INVALID;
}
bool rows_ok(const void *p, int64_t ld, int64_t n, int64_t T) {
    return (uintptr_t)p % 16 == 0 && (T <= 1 || (ld >= n && ld % 8 == 0));
}

struct BwdLayout {       // byte offsets into the workspace of a backward pass
    int64_t ldk, lo, a, unscale, pairs, f, group, partial, total;
};
// whether dz has bits below its fp16 rounding that the gradient's type can see
bool dz_has_low(int dtype, int act, int mats) {
    return dtype == FORGE_DTYPE_F16 && (mats == 2 || (act != FORGE_ACT_NONE && act != FORGE_ACT_RELU));
}
BwdLayout bwd_layout(int64_t T, int64_t C, int64_t R, int gs, int mats, bool low) {
    BwdLayout L{};
    const auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    L.ldk = cdiv(mats * R, (int64_t)64) * 64;
    L.lo = low ? L.ldk : 0;
    L.a = 0;
    L.unscale = up(T * (L.ldk + L.lo) * 2);
    L.pairs = L.unscale + up(T * 4);
    L.f = L.pairs + up(mats * R * cdiv(C, (int64_t)gs) * 4);
    L.group = L.f + up(mats * R * 4);
    L.partial = L.group + up(cdiv(mats * R, (int64_t)kKBlock) * cdiv(C, (int64_t)gs) * 4);
    L.total = L.partial + up((T < kRowCtas ? (T < kBiasParts ? kBiasParts : T) : kRowCtas) * R * 4);
    return L;
}

// Partial column sums of dz where the pass that writes dz did not leave them; returns their number of rows
template <typename T> int launch_dbias(const void *dy, int64_t lddy, const void *z, int act, int64_t n, int64_t R, float *partial,
                                       cudaStream_t st) {
    const int parts = (int)imin64(n, kBiasParts);
    if (parts == 0) return 0;
    const dim3 grid((unsigned)cdiv(R, (int64_t)256), parts);
    switch (act) {
        case FORGE_ACT_RELU: dbias_kernel<T, FORGE_ACT_RELU><<<grid, 256, 0, st>>>((const T *)dy, lddy, (const T *)z, n, R, partial); break;
        case FORGE_ACT_SILU: dbias_kernel<T, FORGE_ACT_SILU><<<grid, 256, 0, st>>>((const T *)dy, lddy, (const T *)z, n, R, partial); break;
        case FORGE_ACT_GELU: dbias_kernel<T, FORGE_ACT_GELU><<<grid, 256, 0, st>>>((const T *)dy, lddy, (const T *)z, n, R, partial); break;
        default: dbias_kernel<T, FORGE_ACT_NONE><<<grid, 256, 0, st>>>((const T *)dy, lddy, (const T *)z, n, R, partial);
    }
    FORGE_NOTE_LAUNCH();
    return parts;
}
// The row-in-registers form of dz where it fits; the number of partial rows written, or 0 when the call is not for it.
template <typename T, int ACT, bool GATED> int launch_dz_rows(const DzParams &P, float *partial, cudaStream_t st) {
    if (P.R % 8 != 0 || P.R > 8192 || (uintptr_t)P.dy % 16 != 0 || P.lddy % 8 != 0 || (uintptr_t)P.z % 16 != 0 ||
        (uintptr_t)P.u % 16 != 0)
        return 0;
    const int ctas = (int)imin64(P.T, kRowCtas);
    if (P.R <= 2048) dz_rows_kernel<T, ACT, GATED, 256, 1><<<ctas, 256, 0, st>>>(P, partial);
    else if (P.R <= 4096) dz_rows_kernel<T, ACT, GATED, 512, 1><<<ctas, 512, 0, st>>>(P, partial);
    else dz_rows_kernel<T, ACT, GATED, 512, 2><<<ctas, 512, 0, st>>>(P, partial);
    FORGE_NOTE_LAUNCH();
    return ctas;
}

// dz into the K operand; returns the partial rows of its column sums that were written on the way (0: none)
template <typename T, bool GATED, int ACT> int launch_dz_act(const DzParams &P, float *partial, cudaStream_t st) {
    if (const int parts = launch_dz_rows<T, ACT, GATED>(P, partial, st)) return parts;
    dz_kernel<T, ACT, GATED><<<(unsigned)P.T, 256, 0, st>>>(P);
    FORGE_NOTE_LAUNCH();
    return 0;
}
template <typename T, bool GATED> int launch_dz(const DzParams &P, int act, float *partial, cudaStream_t st) {
    switch (act) {
        case FORGE_ACT_RELU: return launch_dz_act<T, GATED, FORGE_ACT_RELU>(P, partial, st);
        case FORGE_ACT_SILU: return launch_dz_act<T, GATED, FORGE_ACT_SILU>(P, partial, st);
        case FORGE_ACT_GELU: return launch_dz_act<T, GATED, FORGE_ACT_GELU>(P, partial, st);
        default: return launch_dz_act<T, GATED, FORGE_ACT_NONE>(P, partial, st);
    }
}
int run_fwd(Int4Fwd &P, int dtype, bool gated, cudaStream_t st) {
    const uintptr_t a = (uintptr_t)P.packed[0] | (uintptr_t)P.packed[1];
    P.vec8 = P.C % 16 == 0 && a % 8 == 0;
    P.vec16 = P.C % 32 == 0 && a % 16 == 0;
    const bool bf16 = dtype == FORGE_DTYPE_BF16;
    return P.T <= kDecodeTokens ? int4_decode(P, bf16, gated, st) : int4_fwd_tc(P, bf16, gated, st);
}

}  // namespace

extern "C" int forge_int4_linear(const void *x, int64_t ldx, int dtype, const int32_t *packed, const float *scales, int gs,
                                 int64_t T, int64_t C, int64_t R, const void *bias, int act, const void *residual,
                                 int64_t ldres, void *y, void *preact, int32_t *status, void *stream) {
    if (int rc = check_sizes(__func__, dtype, T, C, R, gs, act)) return rc;
    if (T == 0) return FORGE_OK;
    FORGE_REQUIRE(x && packed && scales && y, "null pointer");
    FORGE_REQUIRE(rows_ok(x, ldx, C, T), "x must be 16-byte aligned with a row stride >= C that is a multiple of 8");
    FORGE_REQUIRE(!residual || T == 1 || ldres >= R, "residual row stride below R");
    FORGE_REQUIRE((uintptr_t)y % 16 == 0 && (uintptr_t)preact % 16 == 0, "outputs must be 16-byte aligned");
    Int4Fwd P{x, ldx, {(const uint32_t *)packed, nullptr}, {scales, nullptr}, gs, T, C, R, cdiv(C, (int64_t)gs), bias, act,
              residual, ldres, y, preact, nullptr, status, false, false};
    return run_fwd(P, dtype, false, (cudaStream_t)stream);
}

extern "C" int forge_int4_gated(const void *x, int64_t ldx, int dtype, const int32_t *gate_packed, const float *gate_scales,
                                const int32_t *up_packed, const float *up_scales, int gs, int64_t T, int64_t C, int64_t R,
                                int act, void *h, void *g, void *u, int32_t *status, void *stream) {
    if (int rc = check_sizes(__func__, dtype, T, C, R, gs, act)) return rc;
    FORGE_REQUIRE(!g == !u, "g and u go together");
    if (T == 0) return FORGE_OK;
    FORGE_REQUIRE(x && gate_packed && gate_scales && up_packed && up_scales && h, "null pointer");
    FORGE_REQUIRE(rows_ok(x, ldx, C, T), "x must be 16-byte aligned with a row stride >= C that is a multiple of 8");
    FORGE_REQUIRE((uintptr_t)h % 16 == 0 && (uintptr_t)g % 16 == 0 && (uintptr_t)u % 16 == 0, "outputs must be 16-byte aligned");
    Int4Fwd P{x, ldx, {(const uint32_t *)gate_packed, (const uint32_t *)up_packed}, {gate_scales, up_scales}, gs, T, C, R,
              cdiv(C, (int64_t)gs), nullptr, act, nullptr, 0, h, g, u, status, false, false};
    return run_fwd(P, dtype, true, (cudaStream_t)stream);
}

static int64_t workspace_bytes(int64_t T, int64_t C, int64_t R, int gs, int mats, bool low) {
    if (T < 0 || C <= 0 || R <= 0 || gs <= 0 || mats < 1 || mats > 2 || T > kMaxTokens || C > kMaxDim || R > kMaxDim) return 0;
    return bwd_layout(T, C, R, gs, mats, low).total;
}
extern "C" int64_t forge_int4_backward_workspace_bytes(int64_t T, int64_t C, int64_t R, int gs, int mats) {
    return workspace_bytes(T, C, R, gs, mats, true);
}
extern "C" int64_t forge_int4_backward_workspace_bytes_for(int dtype, int act, int64_t T, int64_t C, int64_t R, int gs, int mats) {
    return workspace_bytes(T, C, R, gs, mats, dz_has_low(dtype, act, mats));
}

static int backward(const char *who, const void *dy, int64_t lddy, int dtype, const int32_t *p0, const float *s0,
                    const int32_t *p1, const float *s1, int gs, int64_t T, int64_t C, int64_t R, const void *z, const void *u,
                    int act, void *dx, void *dbias, void *ws, int32_t *status, cudaStream_t st) {
    const int mats = p1 ? 2 : 1;
    const bool bf16 = dtype == FORGE_DTYPE_BF16;
    const BwdLayout L = bwd_layout(T, C, R, gs, mats, dz_has_low(dtype, act, mats));
    uint8_t *base = (uint8_t *)ws;
    float *partial = (float *)(base + L.partial);
    int parts = 0;
    const int64_t G = cdiv(C, (int64_t)gs);
    if (dx && T > 0) {
        scale_prep_kernel<<<(unsigned)cdiv(mats * R, (int64_t)kKBlock) * kPrepCtas, 512, 0, st>>>(
            s0, s1, R, mats * R, G, (__half2 *)(base + L.pairs), (float *)(base + L.f), (float *)(base + L.group));
        FORGE_NOTE_LAUNCH();
        DzParams D{dy, z, u, lddy, T, R, mats * R, L.ldk, L.lo, (const float *)(base + L.f), (__half *)(base + L.a),
                   (float *)(base + L.unscale)};
        float *pp = dbias ? partial : nullptr;
        if (mats == 2) parts = bf16 ? launch_dz<__nv_bfloat16, true>(D, act, pp, st) : launch_dz<__half, true>(D, act, pp, st);
        else parts = bf16 ? launch_dz<__nv_bfloat16, false>(D, act, pp, st) : launch_dz<__half, false>(D, act, pp, st);
    }
    if (dbias) {
        if (parts == 0)
            parts = bf16 ? launch_dbias<__nv_bfloat16>(dy, lddy, z, act, T, R, partial, st)
                         : launch_dbias<__half>(dy, lddy, z, act, T, R, partial, st);
        launch_column_sum(partial, parts, R, dbias, dtype, st);
    }
    if (!dx || T == 0) return check_launch(who);
    Int4Dgrad P{(const __half *)(base + L.a), L.ldk, L.lo, (const float *)(base + L.unscale),
                {(const uint32_t *)p0, (const uint32_t *)p1}, (const __half2 *)(base + L.pairs), (const float *)(base + L.group),
                gs, mats, T, C, R, G, dx, status,
                C % 16 == 0 && ((uintptr_t)p0 | (uintptr_t)p1) % 8 == 0};
    return int4_dgrad_tc(P, dtype == FORGE_DTYPE_BF16, who, st);
}

extern "C" int forge_int4_linear_backward(const void *dy, int64_t lddy, int dtype, const int32_t *packed, const float *scales,
                                          int gs, int64_t T, int64_t C, int64_t R, const void *preact, int act, void *dx,
                                          void *dbias, void *ws, int32_t *status, void *stream) {
    if (int rc = check_sizes(__func__, dtype, T, C, R, gs, act)) return rc;
    FORGE_REQUIRE(T == 0 || dx || dbias, "nothing to compute");     // (no tokens: dx is empty and may be null)
    FORGE_REQUIRE(T == 0 || (dy && (!dx || (packed && scales)) && (act == FORGE_ACT_NONE || preact)), "null pointer");
    FORGE_REQUIRE(ws && (uintptr_t)ws % 256 == 0, "workspace must be 256-byte aligned");
    FORGE_REQUIRE(T <= 1 || lddy >= R, "dy row stride below R");
    FORGE_REQUIRE((uintptr_t)dx % 16 == 0, "dx must be 16-byte aligned");
    return backward(__func__, dy, lddy, dtype, packed, scales, nullptr, nullptr, gs, T, C, R, act == FORGE_ACT_NONE ? nullptr : preact,
                    nullptr, act, dx, dbias, ws, status, (cudaStream_t)stream);
}

extern "C" int forge_int4_gated_backward(const void *dh, int64_t lddh, int dtype, const void *g, const void *u,
                                         const int32_t *gate_packed, const float *gate_scales, const int32_t *up_packed,
                                         const float *up_scales, int gs, int64_t T, int64_t C, int64_t R, int act, void *dx,
                                         void *ws, int32_t *status, void *stream) {
    if (int rc = check_sizes(__func__, dtype, T, C, R, gs, act)) return rc;
    if (T == 0) return FORGE_OK;
    FORGE_REQUIRE(dh && g && u && gate_packed && gate_scales && up_packed && up_scales && dx, "null pointer");
    FORGE_REQUIRE(ws && (uintptr_t)ws % 256 == 0, "workspace must be 256-byte aligned");
    FORGE_REQUIRE(T <= 1 || lddh >= R, "dh row stride below R");
    FORGE_REQUIRE((uintptr_t)dx % 16 == 0, "dx must be 16-byte aligned");
    return backward(__func__, dh, lddh, dtype, gate_packed, gate_scales, up_packed, up_scales, gs, T, C, R, g, u, act, dx,
                    nullptr, ws, status, (cudaStream_t)stream);
}

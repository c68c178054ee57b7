// int4 products for many tokens on the tensor cores (tcgen05, accumulators in tensor memory), forward and backward.
//
// Forward (linear, gated), per 128-token x 256-weight-row tile:
//   acc[t, r] = sum over chunks  scale[r, g] * ( sum over the chunk's channels  x[t, c] * (nibble(r, c) - 8) )
// A chunk is a scale group (gs channels).  The inner sum is one accumulation in tensor memory whose operands are exact
// (nibble - 8 is an integer of four bits); the scale is applied in fp32 when the chunk's accumulator is added to the
// running sums, which live in registers.  So nothing is rounded before the result, and the tensor core's truncating
// accumulation covers 128 terms at most.  Gated form: 128 gate rows and the 128 up rows of the same channels make the 256.
//
// Backward (dx = dz W):  the K axis is the weight rows, so a chunk has many scales and they have to be in the operand:
// W' = fp16((nibble - 8) * s'), s' the scale without its row's power of two (which dz carries exactly), from an fp16 pair
// (hi, lo) so that W' is rounded once.  W is read along its rows, which are the N side here: an MN-major operand.
// Chunks of 512 weight rows are added up in registers.
//
// A CTA (one per SM, 512 threads): warps 0-7 add finished chunks to the sums and run the epilogue, warps 8-11 turn packed
// words into 16-bit operand tiles (read two stages ahead into registers, written with the 128-byte swizzle), warp 12
// brings the token tile in with TMA, warp 13 owns tensor memory and issues the MMAs.  Four 48 KB stages of 64 channels,
// two 256-column accumulators.  Registers move from the loading warps to the summing ones (setmaxnreg; 2 x 192 + 88 + 40
// is the 4 x 128 that the CTA starts with).
//
// With fewer tiles than SMs the K axis is shared by the CTAs of a cluster: each leaves its sums in its shared memory and
// every CTA adds up a slice of the columns from all of them, in rank order, over distributed shared memory.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>
#include "common.cuh"
#include "elem.cuh"
#include "int4_mm.cuh"
#include "tcgen05.cuh"

using namespace forge;
using namespace forge::tc;

namespace {

constexpr int kLinear = 0, kGated = 1, kDgrad = 2;

constexpr int kMT = 128, kNT = 256, kKT = 64;
constexpr int kABytes = kMT * 128, kBBytes = kNT * 128;
constexpr int kStageBytes = kABytes + kBBytes;
constexpr int kStages = 4;
constexpr int kSlots = 8;                       // scale ring: one slot of 256 scales per chunk
constexpr int kThreads = 512;
constexpr int kRegsSum = 192, kRegsLoad = 88, kRegsMisc = 40;
static_assert(2 * kRegsSum + kRegsLoad + kRegsMisc <= 4 * 128, "register shares within the launch's total");
constexpr int kOffScales = kStages * kStageBytes;
constexpr int kOffBars = kOffScales + kSlots * kNT * 4;
constexpr size_t kSmemBytes = kOffBars + 256 + 1024;

struct TcParams {
    Int4Fwd f;
    Int4Dgrad d;
    int64_t T, N;        // token rows, output columns (weight rows, or channels in the backward form)
    int mt, nt;          // tiles
    int nst;             // 64-wide k stages in all
    int split, per;      // cluster size along K, stages per member (a multiple of 2)
    int32_t *status;
};

// K-major operand, 128-byte swizzle: 8-row groups 1 KB apart
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// MN-major operand, 128-byte swizzle: blocks of 64 MN elements x 64 K rows, 8 KB apart; groups of 8 K rows 1 KB apart
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(8192 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}
template <int MODE, bool BF16> constexpr uint32_t idesc() {
    return (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (MODE == kDgrad ? 1u << 16 : 0u) | ((kNT >> 3) << 17) |
           ((kMT >> 4) << 24);
}
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}"
        :
        : "r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
    return d;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    uint32_t lo, hi;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v));
    return make_float2(__uint_as_float(lo), __uint_as_float(hi));
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster(uint32_t addr, uint32_t rank) {
    uint32_t a;
    float4 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// eight codes of a word as (nibble - 8) in the 16-bit type, in channel order
template <bool BF16> __device__ __forceinline__ uint4 word_to_half(uint32_t w) {
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t v = ((w >> (4 * i)) & 0x000F000Fu) | (BF16 ? 0x43004300u : 0x64006400u);
        if constexpr (BF16) {
            const __nv_bfloat162 h = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&v), __floats2bfloat162_rn(136.0f, 136.0f));
            p[i] = *reinterpret_cast<const uint32_t *>(&h);
        } else {
            const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&v), __floats2half2_rn(1032.0f, 1032.0f));
            p[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
    }
    return make_uint4(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[2], p[3], 0x5410), __byte_perm(p[0], p[1], 0x7632),
                      __byte_perm(p[2], p[3], 0x7632));
}
__device__ __forceinline__ uint32_t scaled(uint32_t v, __half2 hi, __half2 lo) {
    const __half2 q = *reinterpret_cast<const __half2 *>(&v);
    const __half2 r = __hfma2(q, hi, __hmul2(q, lo));
    return *reinterpret_cast<const uint32_t *>(&r);
}

constexpr uint32_t kZeroWord = 0x88888888u;

// where the four 32-column blocks of a summing warp lie in the tile: its half of the columns; in the gated form two
// blocks of gate and the same two of up
template <int MODE> __device__ __forceinline__ int block_col(int half, int j) {
    return MODE == kGated ? (j >> 1) * 128 + half * 64 + (j & 1) * 32 : half * 128 + j * 32;
}

// Eight neighbouring outputs of one token row, starting at column c (a multiple of 8); u: the up projections (gated).
template <typename T, int MODE, int W>
__device__ __forceinline__ void emit(const TcParams &P, int64_t t, int64_t c, const float (&v)[W], const float (&u)[W]) {
    const int64_t N = P.N;
    if (c >= N) return;
    const int64_t o = t * N + c;
    float y[W];
    if constexpr (MODE == kDgrad) {
        const float s = P.d.unscale[t];
#pragma unroll
        for (int i = 0; i < W; ++i) y[i] = v[i] * s;
    } else {
        const T *bias = (const T *)P.f.bias, *res = (const T *)P.f.res;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            float z = v[i];
            if (MODE == kLinear && bias && c + i < N) z += Elem<T>::to_f(bias[c + i]);
            y[i] = z;
        }
        if (P.f.pre0) {
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (c + i < N) {
                    ((T *)P.f.pre0)[o + i] = Elem<T>::from_f(y[i]);
                    if (MODE == kGated) ((T *)P.f.pre1)[o + i] = Elem<T>::from_f(u[i]);
                }
        }
#pragma unroll
        for (int i = 0; i < W; ++i) {
            y[i] = act_fwd_rt(P.f.act, y[i]);
            if (MODE == kGated) y[i] *= u[i];
            if (MODE == kLinear && res && c + i < N) y[i] += Elem<T>::to_f(res[t * P.f.ldres + c + i]);
        }
    }
    T *out = (T *)(MODE == kDgrad ? P.d.dx : P.f.y) + o;
    if (W == 8 && N % 8 == 0) {
        float w8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w8[i] = y[i % W];
        store8(out, w8);
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (c + i < N) out[i] = Elem<T>::from_f(y[i]);
    }
}

// T: output type; MODE; CH: channels per chunk (forward: the group size; backward: 512 weight rows)
template <typename T, int MODE, int CH>
__global__ void __launch_bounds__(kThreads, 1) int4_tc_kernel(const __grid_constant__ TcParams P,
                                                              const __grid_constant__ CUtensorMap tmap) {
    constexpr bool kBf16 = MODE != kDgrad && std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_al = smem_raw + (smem_base - smem_u32(smem_raw));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem_al + kOffBars);
    const uint32_t b_full = smem_u32(bars), b_empty = b_full + 8 * kStages, b_afull = b_empty + 8 * kStages,
                   b_aempty = b_afull + 16, b_sfull = b_aempty + 16, b_sempty = b_sfull + 8 * kSlots;
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(bars + 2 * kStages + 4 + 2 * kSlots);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_holder + 1);
    static_assert((2 * kStages + 4 + 2 * kSlots) * 8 + 8 <= 256, "barrier block");

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(b_full + 8 * s, 1 + 128);
            mbar_init(b_empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(b_afull + 8 * a, 1);
            mbar_init(b_aempty + 8 * a, 8);
        }
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(b_sfull + 8 * s, 128);
            mbar_init(b_sempty + 8 * s, 8);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 13) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_holder;

    const int rank = P.split > 1 ? (int)(blockIdx.x % P.split) : 0;
    const int st0 = rank * P.per, st1 = min(P.nst, st0 + P.per);      // may be empty
    const int ntiles = P.mt * P.nt;
    const int tile0 = P.split > 1 ? (int)(blockIdx.x / P.split) : (int)blockIdx.x;
    const int tile_step = P.split > 1 ? ntiles : (int)gridDim.x;
    constexpr int kRowsN = MODE == kGated ? 128 : kNT;                // output columns of a tile

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSum));
        const int quarter = warp & 3, half = warp >> 2;
        const uint32_t tlane = tmem_base + ((uint32_t)(quarter * 32) << 16);
        uint32_t chunk = 0;
        bool ok = true;
        for (int tile = tile0; tile < ntiles && ok; tile += tile_step) {
            const int64_t m0 = (int64_t)(tile / P.nt) * kMT, n0 = (int64_t)(tile % P.nt) * kRowsN;
            uint64_t acc[4][16];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[j][i] = 0ull;
            constexpr int kPerStage = CH < kKT ? kKT / CH : 1, kStagesPer = CH > kKT ? CH / kKT : 1;
            const int nch = (st1 - st0 + kStagesPer - 1) / kStagesPer * kPerStage;
            for (int ch = 0; ch < nch; ++ch, ++chunk) {
                const uint32_t buf = chunk & 1u, slot = chunk % kSlots;
                ok = mbar_wait(b_afull + 8 * buf, (chunk >> 1) & 1u, abort_flag);
                if (MODE != kDgrad) ok = ok && mbar_wait(b_sfull + 8 * slot, (chunk / kSlots) & 1u, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint8_t *sc = smem_al + kOffScales + slot * (kNT * 4);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int col = block_col<MODE>(half, j >> 1) + (j & 1) * 16;
                    uint32_t v[16];
                    tmem_ld16(tlane + buf * kNT + col, v);
                    tmem_ld_wait();
                    if (j == 7) {      // the accumulator is free once everything is in registers
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(b_aempty + 8 * buf);
                    }
                    uint64_t *a = acc[j >> 1] + (j & 1) * 8;
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        if constexpr (MODE == kDgrad) {
                            a[i] = add2(a[i], pack2(v[2 * i], v[2 * i + 1]));
                            a[i + 1] = add2(a[i + 1], pack2(v[2 * i + 2], v[2 * i + 3]));
                        } else {
                            const ulonglong2 s = *reinterpret_cast<const ulonglong2 *>(sc + (col + 2 * i) * 4);
                            a[i] = fma2(pack2(v[2 * i], v[2 * i + 1]), s.x, a[i]);
                            a[i + 1] = fma2(pack2(v[2 * i + 2], v[2 * i + 3]), s.y, a[i + 1]);
                        }
                    }
                }
                if (MODE != kDgrad) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(b_sempty + 8 * slot);
                }
            }
            if (!ok) break;
            if (P.split == 1) {
                const int64_t t = m0 + quarter * 32 + lane;
                if (t < P.T) {
#pragma unroll
                    for (int j = 0; j < (MODE == kGated ? 2 : 4); ++j)
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            float a[8], b[8];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float2 p = unpack2(acc[j][i + e]);
                                a[2 * e] = p.x; a[2 * e + 1] = p.y;
                                const float2 r = unpack2(acc[MODE == kGated ? j + 2 : j][i + e]);
                                b[2 * e] = r.x; b[2 * e + 1] = r.y;
                            }
                            emit<T, MODE, 8>(P, t, n0 + block_col<MODE>(half, j) + 2 * i, a, b);
                        }
                }
            } else {
                // sums to shared memory (every MMA of this CTA is complete, the stages are free): [column / 4][row] float4
                const int row = quarter * 32 + lane;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const int c4 = (block_col<MODE>(half, j) + 2 * i) >> 2;
                        const float2 p = unpack2(acc[j][i]), r = unpack2(acc[j][i + 1]);
                        sts128(smem_base + (uint32_t)(c4 * kMT + row) * 16u,
                               make_uint4(__float_as_uint(p.x), __float_as_uint(p.y), __float_as_uint(r.x), __float_as_uint(r.y)));
                    }
            }
        }
        if (P.split > 1) {
            cluster_sync();
            const int64_t m0 = (int64_t)(tile0 / P.nt) * kMT, n0 = (int64_t)(tile0 % P.nt) * kRowsN;
            const int per4 = kRowsN / 4 / P.split;                    // column quads of this CTA's slice
            for (int i = tid; i < per4 * kMT && ok; i += 256) {
                const int c4 = rank * per4 + i / kMT, row = i % kMT;
                const int64_t t = m0 + row;
                if (t >= P.T) continue;
                float a[4] = {0.0f, 0.0f, 0.0f, 0.0f}, b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                for (int r = 0; r < P.split; ++r) {
                    const float4 v = ld_cluster(smem_base + (uint32_t)(c4 * kMT + row) * 16u, r);
                    a[0] += v.x; a[1] += v.y; a[2] += v.z; a[3] += v.w;
                    if constexpr (MODE == kGated) {
                        const float4 w = ld_cluster(smem_base + (uint32_t)((c4 + 32) * kMT + row) * 16u, r);
                        b[0] += w.x; b[1] += w.y; b[2] += w.z; b[3] += w.w;
                    }
                }
                emit<T, MODE, 4>(P, t, n0 + c4 * 4, a, b);
            }
        }
    } else if (warp < 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLoad));
        const int lt = tid - 256;                                     // 0..127
        uint32_t it = 0, chunk = 0;
        bool ok = true;
        if constexpr (MODE != kDgrad) {
            const int CP = (int)(P.f.C / 8);
            const bool vec = P.f.vec8;
            const int q = lt & 3, r0 = lt >> 2;                       // words 2q, 2q+1 of rows r0 + 32 p
            for (int tile = tile0; tile < ntiles && ok; tile += tile_step) {
                const int64_t n0 = (int64_t)(tile % P.nt) * kRowsN;
                uint2 w[2][8];
                const auto row_of = [&](int p, const uint32_t *&base) -> int64_t {
                    const int r = r0 + 32 * p;
                    const bool second = MODE == kGated && r >= 128;
                    base = P.f.packed[second ? 1 : 0];
                    const int64_t row = n0 + (second ? r - 128 : r);
                    return row < P.f.R ? row : P.f.R - 1;             // rows past the matrix: computed, never stored
                };
                const auto fetch = [&](int st, uint2 (&d)[8]) {
                    const int word = st * 8 + 2 * q;
#pragma unroll
                    for (int p = 0; p < 8; ++p) {
                        const uint32_t *base;
                        const int64_t row = row_of(p, base);
                        const uint32_t *src = base + row * CP + word;
                        if (vec && word < CP) {
                            d[p] = __ldg(reinterpret_cast<const uint2 *>(src));
                        } else {
                            d[p].x = word < CP ? __ldg(src) : kZeroWord;
                            d[p].y = word + 1 < CP ? __ldg(src + 1) : kZeroWord;
                        }
                    }
                };
                if (st0 < st1) fetch(st0, w[0]);
                if (st0 + 1 < st1) fetch(st0 + 1, w[1]);
                const auto stage_work = [&](int st, uint2 (&d)[8]) {
                    const uint32_t s = it % kStages;
                    // the chunk's scales (rows lt and lt + 128 of the tile)
                    constexpr int kPerStage = CH < kKT ? kKT / CH : 1, kStagesPer = CH > kKT ? CH / kKT : 1;
                    if ((st - st0) % kStagesPer == 0) {
#pragma unroll
                        for (int e = 0; e < kPerStage; ++e, ++chunk) {
                            const int64_t g = (int64_t)st * kKT / CH + e;
                            float v[2];
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const bool second = MODE == kGated && h == 1;
                                int64_t row = n0 + lt + (MODE == kGated ? 0 : h * 128);
                                row = row < P.f.R ? row : P.f.R - 1;
                                v[h] = g < P.f.G ? __ldg(P.f.scales[second ? 1 : 0] + row * P.f.G + g) : 0.0f;
                            }
                            const uint32_t slot = chunk % kSlots;
                            ok = ok && mbar_wait(b_sempty + 8 * slot, ((chunk / kSlots) & 1u) ^ 1u, abort_flag);
                            if (!ok) return;
                            float *dst = reinterpret_cast<float *>(smem_al + kOffScales + slot * (kNT * 4));
                            dst[lt] = v[0];
                            dst[lt + 128] = v[1];
                            mbar_arrive(b_sfull + 8 * slot);
                        }
                    }
                    ok = mbar_wait(b_empty + 8 * s, ((it / kStages) & 1u) ^ 1u, abort_flag);
                    if (!ok) return;
                    const uint32_t tileb = smem_base + s * kStageBytes + kABytes;
#pragma unroll
                    for (int p = 0; p < 8; ++p) {
                        const int r = r0 + 32 * p;
                        const uint32_t rowb = tileb + (uint32_t)((r >> 3) * 1024 + (r & 7) * 128);
                        sts128(rowb + (uint32_t)(((2 * q) ^ (r & 7)) << 4), word_to_half<kBf16>(d[p].x));
                        sts128(rowb + (uint32_t)(((2 * q + 1) ^ (r & 7)) << 4), word_to_half<kBf16>(d[p].y));
                    }
                    fence_proxy_async();
                    mbar_arrive(b_full + 8 * s);
                    ++it;
                    if (st + 2 < st1) fetch(st + 2, d);
                };
                for (int st = st0; st < st1 && ok; st += 2) {
                    stage_work(st, w[0]);
                    if (ok && st + 1 < st1) stage_work(st + 1, w[1]);
                }
            }
        } else {
            const int CP = (int)(P.d.C / 8);
            const int l8 = lt & 7, k0 = lt >> 3;                      // words l8 + 8 i of K rows k0 + 16 p
            const int64_t K = (int64_t)P.d.mats * P.d.R;
            for (int tile = tile0; tile < ntiles && ok; tile += tile_step) {
                const int64_t n0 = (int64_t)(tile % P.nt) * kNT;
                uint32_t w[4][4];
                __half2 sc[4][4];
                const auto fetch = [&](int st) {
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        const int64_t k = (int64_t)st * kKT + k0 + 16 * p;
                        const bool second = k >= P.d.R;
                        const uint32_t *src = P.d.packed[second ? 1 : 0] + (k - (second ? P.d.R : 0)) * CP;
                        const __half2 *ss = P.d.pairs + k * P.d.G;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int64_t word = n0 / 8 + l8 + 8 * i;
                            const bool in = k < K && word < CP;
                            w[p][i] = in ? __ldg(src + word) : kZeroWord;
                            sc[p][i] = in ? ss[(word * 8) / P.d.gs] : __half2(__ushort_as_half(0), __ushort_as_half(0));
                        }
                    }
                };
                if (st0 < st1) fetch(st0);
                for (int st = st0; st < st1; ++st) {
                    const uint32_t s = it % kStages;
                    ok = mbar_wait(b_empty + 8 * s, ((it / kStages) & 1u) ^ 1u, abort_flag);
                    if (!ok) break;
                    const uint32_t tileb = smem_base + s * kStageBytes + kABytes;
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        const int k = k0 + 16 * p;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint4 v = word_to_half<false>(w[p][i]);
                            const __half2 hi = __low2half2(sc[p][i]), lo = __high2half2(sc[p][i]);
                            sts128(tileb + (uint32_t)(i * 8192 + (k >> 3) * 1024 + (k & 7) * 128 + ((l8 ^ (k & 7)) << 4)),
                                   make_uint4(scaled(v.x, hi, lo), scaled(v.y, hi, lo), scaled(v.z, hi, lo), scaled(v.w, hi, lo)));
                        }
                    }
                    fence_proxy_async();
                    mbar_arrive(b_full + 8 * s);
                    ++it;
                    if (st + 1 < st1) fetch(st + 1);
                }
            }
        }
        if (P.split > 1) { __syncwarp(); cluster_sync(); }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsMisc));
        if (warp == 12) {
            // ------------------------------ token tile by TMA ------------------------------
            uint32_t it = 0;
            bool ok = true;
            if (lane == 0) {
                for (int tile = tile0; tile < ntiles && ok; tile += tile_step) {
                    const int m0 = (tile / P.nt) * kMT;
                    for (int st = st0; st < st1; ++st, ++it) {
                        const uint32_t s = it % kStages;
                        ok = mbar_wait(b_empty + 8 * s, ((it / kStages) & 1u) ^ 1u, abort_flag);
                        if (!ok) break;
                        mbar_arrive_expect_tx(b_full + 8 * s, kABytes);
                        tma_load_2d(smem_base + s * kStageBytes, &tmap, st * kKT, m0, b_full + 8 * s);
                    }
                }
            }
            __syncwarp();
        } else if (warp == 13) {
            // ------------------------------ MMA issuer ------------------------------
            uint32_t it = 0, chunk = 0;
            bool ok = true;
            constexpr int kStepsPer = (CH < kKT ? CH : kKT) / 16;     // k-steps of a chunk inside a stage
            constexpr int kStagesPer = CH > kKT ? CH / kKT : 1;
            if (lane == 0) {
                for (int tile = tile0; tile < ntiles && ok; tile += tile_step) {
                    for (int st = st0; st < st1 && ok; ++st, ++it) {
                        const uint32_t s = it % kStages;
                        ok = mbar_wait(b_full + 8 * s, (it / kStages) & 1u, abort_flag);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t abase = smem_base + s * kStageBytes, bbase = abase + kABytes;
                        const bool first_stage = (st - st0) % kStagesPer == 0;
                        const bool last_stage = (st - st0) % kStagesPer == kStagesPer - 1 || st + 1 == st1;
#pragma unroll
                        for (int kk = 0; kk < kKT / 16; ++kk) {
                            const bool starts = kk % kStepsPer == 0 && first_stage;
                            if (starts) {
                                ok = mbar_wait(b_aempty + 8 * (chunk & 1u), ((chunk >> 1) & 1u) ^ 1u, abort_flag);
                                if (!ok) break;
                                tc_fence_after();
                            }
                            umma_f16(tmem_base + (chunk & 1u) * kNT, desc_kmajor(abase + kk * 32),
                                     MODE == kDgrad ? desc_mnmajor(bbase + kk * 2048) : desc_kmajor(bbase + kk * 32),
                                     idesc<MODE, kBf16>(), starts ? 0u : 1u);
                            if (kk % kStepsPer == kStepsPer - 1 && last_stage) {
                                umma_commit(b_afull + 8 * (chunk & 1u));
                                ++chunk;
                            }
                        }
                        if (!ok) break;
                        umma_commit(b_empty + 8 * s);
                    }
                }
            }
            __syncwarp();
        }
        if (P.split > 1) cluster_sync();
    }
    // ------------------------------ teardown ------------------------------
    if (P.split > 1) {
        __syncwarp();
        cluster_sync();          // nobody leaves while its sums are being read
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {           // gave up: let copies and MMAs in flight land before shared and tensor memory are given back
        const long long t0 = clock64();
        while (clock64() - t0 < 200000) __nanosleep(1000);
        if (tid == 0 && P.status) atomicExch(P.status, FORGE_ERR_TIMEOUT);
        __syncthreads();
    }
    if (warp == 13) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                             const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
    static EncodeFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return (EncodeFn)p;
    }();
    return fn;
}
// [rows, cols] of 16-bit elements, row stride ld elements; box of 64 columns x 128 rows, 128-byte swizzle, zero fill
bool make_map(CUtensorMap *m, const void *base, bool bf16, int64_t rows, int64_t cols, int64_t ld) {
    EncodeFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
    const cuuint32_t box[2] = {kKT, kMT}, es[2] = {1, 1};
    return fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(base), dims,
              strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int MODE, int CH> int launch(TcParams &P, const CUtensorMap &map, const char *who, cudaStream_t st) {
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const int64_t tiles = (int64_t)P.mt * P.nt;
    if (tiles > 0x3fffffff) {
        set_error("%s: more than 2^30 output tiles", who);
        return FORGE_ERR_UNSUPPORTED;
    }
    const int units = (P.nst + 1) / 2;                                 // 128-wide pieces of K
    P.split = 1;
    while (P.split < 8 && tiles * P.split * 2 <= sms && units >= P.split * 4) P.split *= 2;
    P.per = (units + P.split - 1) / P.split * 2;
    const auto kernel = int4_tc_kernel<T, MODE, CH>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)(P.split > 1 ? tiles * P.split : imin64(tiles, sms)));
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = kSmemBytes;
        cfg.stream = st;
        cudaLaunchAttribute at{};
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = (unsigned)P.split;
        at.val.clusterDim.y = at.val.clusterDim.z = 1;
        cfg.attrs = &at;
        cfg.numAttrs = 1;
        e = cudaLaunchKernelEx(&cfg, kernel, P, map);
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        set_error("%s: %s", who, cudaGetErrorString(e));
        return FORGE_ERR_LAUNCH;
    }
    FORGE_NOTE_LAUNCH();
    return FORGE_OK;
}
template <typename T, int MODE> int launch_gs(TcParams &P, const CUtensorMap &map, const char *who, cudaStream_t st) {
    if (P.f.gs == 32) return launch<T, MODE, 32>(P, map, who, st);
    if (P.f.gs == 64) return launch<T, MODE, 64>(P, map, who, st);
    return launch<T, MODE, 128>(P, map, who, st);
}

}  // namespace

namespace forge {

int int4_fwd_tc(const Int4Fwd &F, bool bf16, bool gated, cudaStream_t st) {
    const char *who = gated ? "forge_int4_gated" : "forge_int4_linear";
    TcParams P{};
    P.f = F; P.T = F.T; P.N = F.R; P.status = F.status;
    P.mt = (int)cdiv(F.T, (int64_t)kMT);
    P.nt = (int)cdiv(F.R, (int64_t)(gated ? 128 : kNT));
    P.nst = (int)cdiv(F.C, (int64_t)kKT);
    alignas(64) CUtensorMap map;
    if (!make_map(&map, F.x, bf16, F.T, F.C, F.ldx)) {
        set_error("%s: no tensor map could be made", who);
        return FORGE_ERR_LAUNCH;
    }
    if (bf16) return gated ? launch_gs<__nv_bfloat16, kGated>(P, map, who, st) : launch_gs<__nv_bfloat16, kLinear>(P, map, who, st);
    return gated ? launch_gs<__half, kGated>(P, map, who, st) : launch_gs<__half, kLinear>(P, map, who, st);
}

int int4_dgrad_tc(const Int4Dgrad &D, bool bf16, const char *who, cudaStream_t st) {
    TcParams P{};
    P.d = D; P.T = D.T; P.N = D.C; P.status = D.status;
    P.mt = (int)cdiv(D.T, (int64_t)kMT);
    P.nt = (int)cdiv(D.C, (int64_t)kNT);
    P.nst = (int)(D.ldk / kKT);
    alignas(64) CUtensorMap map;
    if (!make_map(&map, D.a, false, D.T, D.ldk, D.ldk)) {
        set_error("%s: no tensor map could be made", who);
        return FORGE_ERR_LAUNCH;
    }
    return bf16 ? launch<__nv_bfloat16, kDgrad, 512>(P, map, who, st) : launch<__half, kDgrad, 512>(P, map, who, st);
}

}  // namespace forge

// int4 products for many tokens on the tensor cores (tcgen05, accumulators in tensor memory), forward and backward.
//
// Forward (linear, gated): the weight rows are the M side (a row of the accumulator is a lane of tensor memory), the tokens
// the N side:
//   acc[r, t] = sum over chunks  scale[r, g] * ( sum over the chunk's channels  (nibble(r, c) - 8) * x[t, c] )
// A chunk is a scale group (gs channels).  The inner sum is one accumulation in tensor memory whose operands are exact
// (nibble - 8 is an integer of four bits); a thread then adds its row's chunk to running sums in registers, times ONE
// scale, since a thread sees one row only.  So nothing is rounded before the result, and the tensor core's truncating
// accumulation covers 128 terms at most.  Gated form: a block of 32 rows is 16 gate rows and the 16 up rows of the same
// channels, so both halves of a product meet in one warp.
//
// Backward (dx = dz W): M is the channels, read along the rows of W (an MN-major operand), K the weight rows.  A chunk has
// many scales there, so they have to be in the operand: W' = fp16((nibble - 8) * s'), s' the scale without its row's power
// of two (which dz carries exactly) and without that of its channel group in the chunk, kept as an fp16 pair (hi, lo).  Chunks
// of 512 weight rows are added up in registers, times the group's power: again one factor for a thread, which has one channel.
// fp16 gradients have 11 bits themselves, and dz and W' rounded to 11 bits would nearly double their error (4.0e-4 against
// 2.1e-4).  For them both are pairs of fp16 numbers (22 bits), and a stage is 64 weight rows: their high parts in the upper half
// of its W' tile and their low parts in the lower one, dz's high and low parts in its two sub-tiles, and three products, high x
// high, low x high, high x low (two where dz is dy itself, whose low part is zero): dx of 4096 x 7168 <- 2 x 2048 467 us.
//
// A CTA (one per SM, 640 threads): warps 0-7 add finished chunks to the sums and run the epilogue, warps 8-11 and 12-15
// turn packed words into 16-bit operand tiles, one stage each in turn (words read ahead into registers, tiles written with
// the 128-byte swizzle), warp 16 brings the token tile in with TMA, warp 17 owns tensor memory and issues the MMAs.  Stages
// of 128 channels, two accumulators.  Registers move from the loading warps to the summing ones (setmaxnreg).
//
// Two CTAs of a pair share a tile of 256 rows x 256 tokens (cta_group::2): each turns its own 128 weight rows and loads
// half of the tokens, the even one issues the MMAs for both.  One CTA alone moves 192 KB through its shared memory per
// 128-channel step (operands written and read), 1.5 times what the 1024 cycles of the MMAs allow; a pair's CTA moves 128.
//
// Measured (burst clocks): gated 8192 x 7168 -> 2048 352 us (1.37 PFLOP/s, 0.84 of the measured cuBLAS burst rate; 416 us,
// 1.16 PFLOP/s, when the power limit holds the clock down), 4096 x 2048 -> 7168 with residual 124 us (0.97 PFLOP/s), dx of
// 4096 x 7168 <- 2 x 2048 (gated) 198 us (1.21 PFLOP/s), without the 19 us of dz and the 5 us of the scales.  ncu on the
// gated kernel at 4096 tokens: tensor pipe 72 % active (84 % on the SMs that have four tiles), shared memory 84 %: what bounds
// it is the shared-memory port, which carries both operands in and out.  The smaller products end on a partly filled round of
// tiles (448 tiles on 74 pairs).
//
// With fewer tiles than SMs the K axis is shared by the CTAs of a cluster: each leaves its sums in its shared memory and
// every CTA adds up a slice of the tokens from all of them, in rank order, over distributed shared memory.
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

constexpr int kMT = 128, kKT = 128;             // rows of a CTA tile, channels of a stage
constexpr int kSubA = kMT * 128, kABytes = 2 * kSubA;   // K-major: two sub-tiles of 64 channels (128 bytes a row)
constexpr int kThreads = 640;
// Registers a thread of the summing, loading and other warps, out of 5 x 96, as measured for each form (4096 x 2048 -> 7168:
// 130 us with 176 for the sums, 190 with 160; gated 8192 x 7168 -> 2048: 371 us with 64 for the loads, 454 with 48; dx of 4096 x
// 7168 <- 2 x 2048: 198 us with 160 and 64, 204 with 152 and 72).  ptxas still spills 112 bytes in the paired backward form, 16
// to 40 in the linear and the backward form of a single CTA, nothing in the others.
template <int MODE> struct Regs {
    static constexpr int kSum = MODE == kLinear ? 176 : 160, kLoad = MODE == kLinear ? 48 : 64, kMisc = 32;
    static_assert(2 * kSum + 2 * kLoad + kMisc <= 5 * 96, "register shares within the launch's total");
};
constexpr int kOutBytes = 32 * 128;             // a summing warp's block: 32 tokens x 32 rows, fp32
constexpr int kRing = 196608;                   // operand stages
constexpr int kOffOut = kRing;
constexpr int kOffBars = kOffOut + 8 * kOutBytes;
constexpr size_t kSmemBytes = kOffBars + 256 + 1024;

struct TcParams {
    Int4Fwd f;
    Int4Dgrad d;
    int64_t T, N;        // token rows, output columns (weight rows; channels in the backward form)
    int rt, tt;          // row tiles, token tiles
    int nst;             // k stages in all
    int split, per;      // cluster size along K, stages per member
    bool res_vec;        // residual rows start on 16 bytes
    bool simple;         // linear: no bias, activation or pre-activation, and 16-byte rows throughout
    int32_t *status;
};

// K-major operand, 128-byte swizzle: 8-row groups 1 KB apart
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// MN-major operand, 128-byte swizzle: blocks of 64 MN elements x 128 K rows, 16 KB apart; groups of 8 K rows 1 KB apart
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(16384 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}
// D fp32, A and B both bf16 or both fp16; the backward form's A is MN-major
template <int MODE, bool BF16> constexpr uint32_t idesc(int m, int n) {
    return (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (MODE == kDgrad ? 1u << 15 : 0u) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
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
// the same over a pair: M = 256, each CTA holds its half of A's rows, of B's rows and of the accumulator's lanes
__device__ __forceinline__ void umma_f16_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}"
        :
        : "r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u)
        : "memory");
}
// arrives on the barrier at the same place of both CTAs of the pair
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ uint32_t even_cta(uint32_t addr) {       // the same shared-memory place in the pair's even CTA
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(addr));
    return a;
}
__device__ __forceinline__ void arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// completes on the barrier of the even CTA
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t even_bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"(map), "r"(x), "r"(y), "r"(even_bar)
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
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
    return d;
}
__device__ __forceinline__ void unpack2(uint64_t v, uint32_t &lo, uint32_t &hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v));
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
__device__ __forceinline__ float4 lds_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void sts32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// eight codes of a word as (nibble - 8) in the 16-bit type, in channel order: a byte of w has the even code in its low
// nibble, the same byte of w >> 4 the odd one; the pair goes into the low mantissa bits of 128 (bf16) or 1024 (fp16)
template <bool BF16> __device__ __forceinline__ uint4 word_to_half(uint32_t w) {
    const uint32_t w4 = w >> 4;
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t v = __byte_perm(w, w4, ((4 + i) << 8) | i) & 0x000F000Fu;
        const uint32_t m = v | (BF16 ? 0x43004300u : 0x64006400u);
        if constexpr (BF16) {
            const __nv_bfloat162 h = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&m), __floats2bfloat162_rn(136.0f, 136.0f));
            p[i] = *reinterpret_cast<const uint32_t *>(&h);
        } else {
            const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&m), __floats2half2_rn(1032.0f, 1032.0f));
            p[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
    }
    return make_uint4(p[0], p[1], p[2], p[3]);
}
// W' of the backward form, from both halves of the scale and rounded once (2^-11).
__device__ __forceinline__ uint32_t scaled(uint32_t v, __half2 hi, __half2 lo) {
    const __half2 q = *reinterpret_cast<const __half2 *>(&v);
    const __half2 r = __hfma2(q, hi, __hmul2(q, lo));
    return *reinterpret_cast<const uint32_t *>(&r);
}

// What `scaled` rounds off, itself rounded to fp16: (nibble - 8) hi - W' is exact, so 2^-22 of W' is left.
__device__ __forceinline__ uint32_t scaled_low(uint32_t v, __half2 hi, __half2 lo, uint32_t w) {
    const __half2 q = *reinterpret_cast<const __half2 *>(&v);
    const __half2 r = __hfma2(q, lo, __hfma2(q, hi, __hneg2(*reinterpret_cast<const __half2 *>(&w))));
    return *reinterpret_cast<const uint32_t *>(&r);
}

constexpr uint32_t kZeroWord = 0x88888888u;

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// Polls without a pause first: the partner is a few hundred cycles away.  Then with pauses, within the time limit.
__device__ __forceinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    while (true) {
        if (mbar_try_wait(bar, parity)) return true;
        __nanosleep(64);
        if (*abort_flag) return false;
        if (clock64() - t0 > kWaitBudget) {
            *abort_flag = 1;
            return false;
        }
    }
}

// Eight neighbouring outputs of token t, columns c .. c + 7 (c a multiple of 8); u: the up projections (gated).
template <typename T, int MODE>
__device__ __forceinline__ void emit8(const TcParams &P, int64_t t, int64_t c, float (&z)[8], const float (&u)[8]) {
    const int64_t N = P.N, o = t * N + c;
    if (t >= P.T || c >= N) return;
    const bool vec = N % 8 == 0;
    const auto put = [&](void *base, const float (&v)[8]) {
        T *dst = (T *)base + o;
        if (vec) {
            store8(dst, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < N) dst[i] = Elem<T>::from_f(v[i]);
        }
    };
    if constexpr (MODE == kDgrad) {
        const float s = __ldg(P.d.unscale + t);
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] *= s;
        put(P.d.dx, z);
    } else {
        float r[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (MODE == kLinear && P.f.res) {
            const T *res = (const T *)P.f.res + t * P.f.ldres + c;
            if (P.res_vec && vec) {
                load8(res, r);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c + i < N) r[i] = Elem<T>::to_f(res[i]);
            }
        }
        if (MODE == kLinear && P.f.bias)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < N) z[i] += Elem<T>::to_f(((const T *)P.f.bias)[c + i]);
        if (P.f.pre0) {
            put(P.f.pre0, z);
            if (MODE == kGated) put(P.f.pre1, u);
        }
        switch (P.f.act) {
            case FORGE_ACT_RELU:
#pragma unroll
                for (int i = 0; i < 8; ++i) z[i] = act_fwd<FORGE_ACT_RELU>(z[i]);
                break;
            case FORGE_ACT_SILU:
#pragma unroll
                for (int i = 0; i < 8; ++i) z[i] = act_fwd<FORGE_ACT_SILU>(z[i]);
                break;
            case FORGE_ACT_GELU:
#pragma unroll
                for (int i = 0; i < 8; ++i) z[i] = act_fwd<FORGE_ACT_GELU>(z[i]);
                break;
            default: break;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = MODE == kGated ? z[i] * u[i] : z[i] + r[i];
        put(P.f.y, z);
    }
}

// A summing warp's block of 32 tokens x 32 rows in shared memory: [token][row] fp32, the 16-byte piece index XORed with the
// token, so lanes (rows) write one token and 4-lane groups read eight rows of a token without bank conflicts.
__device__ __forceinline__ uint32_t blk(uint32_t buf, int token, int row) {
    return buf + (uint32_t)(token * 128 + ((((row >> 2) ^ (token & 7)) << 4) | ((row & 3) << 2)));
}
__device__ __forceinline__ void rows8(uint32_t buf, int token, int row, float (&v)[8]) {
    const float4 a = lds_f4(blk(buf, token, row)), b = lds_f4(blk(buf, token, row + 4));
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// T: output type; MODE; CH: channels per chunk (forward: the group size; backward: kKBlock weight rows); NT: tokens per tile;
// PAIR: two CTAs per tile
template <typename T, int MODE, int CH, int NT, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) int4_tc_kernel(const __grid_constant__ TcParams P,
                                                              const __grid_constant__ CUtensorMap tmap) {
    constexpr bool kBf16 = MODE != kDgrad && std::is_same<T, __nv_bfloat16>::value;
    constexpr bool kSplit = MODE == kDgrad && std::is_same<T, __half>::value;     // both operands in high and low parts
    constexpr int kStageK = kSplit ? kKT / 2 : kKT;                   // K rows of a stage
    constexpr int kBRows = PAIR ? NT / 2 : NT;                        // tokens that this CTA loads
    constexpr int kSubB = kBRows * 128, kBBytes = 2 * kSubB, kStageBytes = kABytes + kBBytes;
    constexpr int kStages = kRing / kStageBytes < 8 ? kRing / kStageBytes : 8;
    constexpr int kCols = NT / 2;                                     // tokens of a summing warp
    constexpr int kTileCols = MODE == kGated ? 64 : kMT;              // output columns of a tile
    constexpr int kPerStage = CH < kKT ? kKT / CH : 1, kStagesPer = CH > kKT ? CH / kStageK : 1;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_al = smem_raw + (smem_base - smem_u32(smem_raw));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem_al + kOffBars);
    const uint32_t b_full = smem_u32(bars), b_empty = b_full + 8 * kStages, b_afull = b_empty + 8 * kStages, b_aempty = b_afull + 16;
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(bars + 2 * kStages + 4);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_holder + 1);
    static_assert((2 * kStages + 4) * 8 + 8 <= 256, "barrier block");

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(b_full + 8 * s, 1 + 8);   // the TMA issuer and the loading warps: four of each CTA of a pair, or all eight
            mbar_init(b_empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(b_afull + 8 * a, 1);
            mbar_init(b_aempty + 8 * a, PAIR ? 16 : 8);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 17) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                         "r"(2u * NT) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                         "r"(2u * NT) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();        // the partner's barriers exist before anything arrives on them
    tc_fence_after();
    const uint32_t tmem_base = *tmem_holder;

    // PAIR: the cluster is the pair; else the cluster (if any) shares the K axis
    const int member = (int)(blockIdx.x % (PAIR ? 2 : P.split));
    const int rank = PAIR ? 0 : member;
    const int st0 = rank * P.per, st1 = min(P.nst, st0 + P.per);      // may be empty
    const int ntiles = P.rt * P.tt;
    const int tile0 = (int)blockIdx.x / (PAIR ? 2 : P.split);
    const int tile_step = PAIR ? (int)gridDim.x / 2 : P.split > 1 ? ntiles : (int)gridDim.x;
    const auto tile_col = [&](int tile) -> int {                      // first output column of this CTA's rows
        return PAIR ? ((tile % P.rt) * 2 + member) * kTileCols : (tile % P.rt) * kTileCols;
    };

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Regs<MODE>::kSum));
        const int quarter = warp & 3, half = warp >> 2;
        const uint32_t tlane = tmem_base + ((uint32_t)(quarter * 32) << 16) + half * kCols;
        uint32_t chunk = 0;
        bool ok = true;
        for (int tile = tile0; tile < ntiles && ok; tile += tile_step) {
            uint64_t acc[kCols / 2];
#pragma unroll
            for (int i = 0; i < kCols / 2; ++i) acc[i] = 0ull;
            const float *sp = nullptr;                                // this lane's next scale
            int left = 0;                                             // scales of the row from there on
            float s_next = 0.0f;
            if constexpr (MODE != kDgrad) {
                const int c = tile_col(tile) + (MODE == kGated ? quarter * 16 + (lane & 15) : quarter * 32 + lane);
                const int row = c < (int)P.f.R ? c : (int)P.f.R - 1, g = st0 * (kKT / CH);
                sp = P.f.scales[MODE == kGated && lane >= 16 ? 1 : 0] + (int64_t)row * P.f.G + g;
                left = (int)P.f.G - g;
                s_next = left > 0 ? __ldg(sp) : 0.0f;
            } else {
                const int c = min(tile_col(tile) + quarter * 32 + lane, (int)P.d.C - 1);
                sp = P.d.group + (int64_t)(st0 / kStagesPer) * P.d.G + c / P.d.gs;
                s_next = __ldg(sp);
            }
            if (MODE == kLinear && P.split == 1 && P.f.res) {         // the residual's lines, long before the epilogue reads them
#pragma unroll
                for (int j = 0; j < kCols / 32; ++j) {
                    const int64_t t = (int64_t)(tile / P.rt) * NT + half * kCols + j * 32 + lane, c = tile_col(tile) + quarter * 32;
                    if (t < P.T && c < P.N)
                        asm volatile("prefetch.global.L2 [%0];" ::"l"((const T *)P.f.res + t * P.f.ldres + c));
                }
            }
            // chunks end at multiples of kStagesPer stages, wherever this CTA's share of them begins
            const int nch = st1 > st0 ? ((st1 - 1) / kStagesPer - st0 / kStagesPer + 1) * kPerStage : 0;
            for (int ch = 0; ch < nch; ++ch, ++chunk) {
                const uint32_t buf = chunk & 1u;
                const float sc = s_next;
                if constexpr (MODE != kDgrad) {
                    ++sp;
                    s_next = --left > 0 ? __ldg(sp) : 0.0f;
                } else if (ch + 1 < nch) {
                    sp += P.d.G;
                    s_next = __ldg(sp);
                }
                ok = wait_on(b_afull + 8 * buf, (chunk >> 1) & 1u, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint64_t sc2 = pack2(__float_as_uint(sc), __float_as_uint(sc));
#pragma unroll
                for (int j = 0; j < kCols / 16; ++j) {
                    uint32_t v[16];
                    tmem_ld16(tlane + buf * NT + j * 16, v);
                    tmem_ld_wait();
                    if (j == kCols / 16 - 1) {      // the accumulator is free once everything is in registers
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            if (PAIR) arrive_cluster(even_cta(b_aempty + 8 * buf));
                            else mbar_arrive(b_aempty + 8 * buf);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[j * 8 + i] = fma2(pack2(v[2 * i], v[2 * i + 1]), sc2, acc[j * 8 + i]);
                }
            }
            if (!ok) break;
            if (P.split == 1) {
                const int64_t t0 = (int64_t)(tile / P.rt) * NT, c0 = tile_col(tile);
                const uint32_t buf = smem_base + kOffOut + warp * kOutBytes;
                const uint32_t wb = blk(buf, 0, lane) - buf;          // piece index without the token's bits
#pragma unroll
                for (int j = 0; j < kCols / 32; ++j) {
                    const int64_t tb = t0 + half * kCols + j * 32;
                    if (tb >= P.T) break;
                    // what the outputs need from memory is requested before the block goes through shared memory
                    const int64_t cl = c0 + quarter * 32 + (lane & 3) * 8;
                    const bool simple = MODE == kDgrad || (MODE == kLinear && P.simple);
                    uint4 rv[4];
                    float us[4];
                    if (MODE == kLinear && simple && P.f.res)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int64_t t = tb + k * 8 + (lane >> 2);
                            rv[k] = t < P.T && cl < P.N ? __ldg(reinterpret_cast<const uint4 *>((const T *)P.f.res + t * P.f.ldres + cl))
                                                        : make_uint4(0u, 0u, 0u, 0u);
                        }
                    if (MODE == kDgrad)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int64_t t = tb + k * 8 + (lane >> 2);
                            us[k] = t < P.T ? __ldg(P.d.unscale + t) : 0.0f;
                        }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        uint32_t lo, hi;
                        unpack2(acc[j * 16 + i], lo, hi);
                        sts32(buf + (2 * i) * 128 + (wb ^ (((2 * i) & 7) << 4)), lo);
                        sts32(buf + (2 * i + 1) * 128 + (wb ^ (((2 * i + 1) & 7) << 4)), hi);
                    }
                    __syncwarp();
                    if constexpr (MODE == kGated) {
#pragma unroll 1
                        for (int k = 0; k < 2; ++k) {
                            const int tok = k * 16 + (lane >> 1), p = (lane & 1) * 8;
                            float z[8], u[8];
                            rows8(buf, tok, p, z);
                            rows8(buf, tok, 16 + p, u);
                            emit8<T, MODE>(P, tb + tok, c0 + quarter * 16 + p, z, u);
                        }
                    } else if (simple) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int tok = k * 8 + (lane >> 2);
                            const int64_t t = tb + tok;
                            float z[8];
                            rows8(buf, tok, (lane & 3) * 8, z);
                            if constexpr (MODE == kDgrad) {
#pragma unroll
                                for (int i = 0; i < 8; ++i) z[i] *= us[k];
                            } else if (P.f.res) {
                                const T *e = reinterpret_cast<const T *>(&rv[k]);
#pragma unroll
                                for (int i = 0; i < 8; ++i) z[i] += Elem<T>::to_f(e[i]);
                            }
                            if (t < P.T && cl < P.N) store8((T *)(MODE == kDgrad ? P.d.dx : P.f.y) + t * P.N + cl, z);
                        }
                    } else {
#pragma unroll 1
                        for (int k = 0; k < 4; ++k) {
                            const int tok = k * 8 + (lane >> 2);
                            float z[8];
                            rows8(buf, tok, (lane & 3) * 8, z);
                            emit8<T, MODE>(P, tb + tok, cl, z, z);
                        }
                    }
                }
            } else {
                // sums to shared memory (every MMA of this CTA is complete, the stages are free): [token][row] fp32
#pragma unroll
                for (int i = 0; i < kCols / 2; ++i) {
                    uint32_t lo, hi;
                    unpack2(acc[i], lo, hi);
                    const uint32_t a = smem_base + (uint32_t)((half * kCols + 2 * i) * kMT + quarter * 32 + lane) * 4u;
                    sts32(a, lo);
                    sts32(a + kMT * 4, hi);
                }
            }
        }
        if (P.split > 1) {
            cluster_sync();
            const int64_t t0 = (int64_t)(tile0 / P.rt) * NT, c0 = tile_col(tile0);
            constexpr int kGroups = kTileCols / 8;
            for (int i = rank * 256 + tid; i < NT * kGroups && ok; i += 256 * P.split) {
                const int tok = i / kGroups, cg = i % kGroups;
                if (t0 + tok >= P.T) break;                           // tokens only grow
                // gated: channels cg * 8 .. are gate rows of the 32-row block cg / 2, the up rows 16 further
                const int row = MODE == kGated ? (cg >> 1) * 32 + (cg & 1) * 8 : cg * 8;
                float z[8] = {}, u[8] = {};
                for (int r = 0; r < P.split; ++r) {
                    const uint32_t a = smem_base + (uint32_t)(tok * kMT + row) * 4u;
                    const float4 v = ld_cluster(a, r), w = ld_cluster(a + 16, r);
                    z[0] += v.x; z[1] += v.y; z[2] += v.z; z[3] += v.w;
                    z[4] += w.x; z[5] += w.y; z[6] += w.z; z[7] += w.w;
                    if constexpr (MODE == kGated) {
                        const float4 v2 = ld_cluster(a + 64, r), w2 = ld_cluster(a + 80, r);
                        u[0] += v2.x; u[1] += v2.y; u[2] += v2.z; u[3] += v2.w;
                        u[4] += w2.x; u[5] += w2.y; u[6] += w2.z; u[7] += w2.w;
                    }
                }
                emit8<T, MODE>(P, t0 + tok, c0 + cg * 8, z, u);
            }
            __syncwarp();
        }
    } else if (warp < 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Regs<MODE>::kLoad));
        // Two groups of four warps.  Pairs (long runs of stages): the groups take the stages in turn.  Else (few stages, where
        // the time to the first products counts): both work on every stage, one 64-channel half each.
        const int lt = tid & 127, group = (warp >> 2) & 1;
        constexpr int kTurn = PAIR ? 2 : 1;
        int base = 0;                                                 // stages before this tile
        bool ok = true;
        const auto publish = [&](uint32_t s) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) arrive_cluster(even_cta(b_full + 8 * s));
                else mbar_arrive(b_full + 8 * s);
            }
        };
        if constexpr (MODE != kDgrad) {
            // four lanes share a row of the stage: words 2q, 2q+1 of rows r0 + 32 p
            const int CP = (int)(P.f.C / 8), q = lt & 3, r0 = lt >> 2;
            const uint32_t d0 = (uint32_t)((r0 >> 3) * 1024 + (r0 & 7) * 128), x0 = (uint32_t)(((2 * q) ^ (r0 & 7)) << 4),
                           x1 = (uint32_t)(((2 * q + 1) ^ (r0 & 7)) << 4);
            for (int tile = tile0; tile < ntiles && ok; tile += tile_step, base += st1 - st0) {
                const int c0 = tile_col(tile) + (MODE == kGated ? r0 & 15 : r0), R = (int)P.f.R;
                constexpr int kStep = MODE == kGated ? 16 : 32;       // matrix rows between this thread's rows
                const uint32_t *rp = P.f.packed[MODE == kGated && r0 >= 16 ? 1 : 0] + (int64_t)c0 * CP + 2 * q;
                // [half][row] words of one stage, or [row] words of this group's half; rows past the matrix are zeros
                constexpr int kWords = PAIR ? 8 : 4, kDeep = PAIR ? 1 : 2;
                const int h0 = PAIR ? 0 : group;
                uint2 w[kDeep][kWords];
                const auto fetch = [&](int st, uint2 (&d)[kWords]) {
                    const int word = st * 16 + h0 * 8;
                    if (P.f.vec8 && st * 16 + 16 <= CP && c0 + 3 * kStep < R) {
                        const uint32_t *src = rp + word;
#pragma unroll
                        for (int p = 0; p < 4; ++p, src += kStep * CP) {
                            d[p] = __ldg(reinterpret_cast<const uint2 *>(src));
                            if (PAIR) d[kWords - 4 + p] = __ldg(reinterpret_cast<const uint2 *>(src + 8));
                        }
                    } else {
#pragma unroll
                        for (int p = 0; p < kWords; ++p) {
                            const int j = word + (p >> 2) * 8 + 2 * q;
                            const bool in = c0 + (p & 3) * kStep < R;
                            const uint32_t *src = rp + (int64_t)(p & 3) * kStep * CP + word + (p >> 2) * 8;
                            d[p].x = in && j < CP ? __ldg(src) : kZeroWord;
                            d[p].y = in && j + 1 < CP ? __ldg(src + 1) : kZeroWord;
                        }
                    }
                };
                const int first = st0 + (PAIR ? (group + base) & 1 : 0);
#pragma unroll
                for (int a = 0; a < kDeep; ++a)
                    if (first + a < st1) fetch(first + a, w[a]);
                for (int stb = first; stb < st1 && ok; stb += kTurn * kDeep) {
#pragma unroll
                    for (int a = 0; a < kDeep; ++a) {
                        const int st = stb + a;
                        if (st >= st1) break;
                        const uint32_t it = (uint32_t)(base + st - st0), s = it % kStages;
                        ok = wait_on(b_empty + 8 * s, ((it / kStages) & 1u) ^ 1u, abort_flag);
                        if (!ok) break;
                        const uint32_t tileb = smem_base + s * kStageBytes + h0 * kSubA + d0;
#pragma unroll
                        for (int p = 0; p < kWords; ++p) {
                            sts128(tileb + (p >> 2) * kSubA + (p & 3) * 4096 + x0, word_to_half<kBf16>(w[a][p].x));
                            sts128(tileb + (p >> 2) * kSubA + (p & 3) * 4096 + x1, word_to_half<kBf16>(w[a][p].y));
                        }
                        publish(s);
                        if (st + kTurn * kDeep < st1) fetch(st + kTurn * kDeep, w[a]);
                    }
                }
            }
        } else {
            // Eight lanes read the 16 words (128 channels) of a K row, two each; K rows k0 + 16 p of a 64-row half.  The upper
            // four lanes, whose words lie in the second 64-channel block, store their two pieces in the other order: eight
            // lanes then write eight different pieces of 16 bytes.
            const int CP = (int)(P.d.C / 8), l8 = lt & 7, k0 = lt >> 3, K = (int)(P.d.mats * P.d.R), R = (int)P.d.R;
            const int G = (int)P.d.G, sh = P.d.gs == 32 ? 5 : P.d.gs == 64 ? 6 : 7;
            const bool swap = l8 >= 4;
            const uint32_t d0 = (uint32_t)((l8 >> 2) * 16384 + (k0 >> 3) * 1024 + (k0 & 7) * 128);
            const uint32_t xa = (uint32_t)((((2 * l8 + (swap ? 1 : 0)) & 7) ^ (k0 & 7)) << 4),
                           xb = (uint32_t)((((2 * l8 + (swap ? 0 : 1)) & 7) ^ (k0 & 7)) << 4);
            struct Half {
                uint2 w[4];
                __half2 s[4];
            };
            for (int tile = tile0; tile < ntiles && ok; tile += tile_step, base += st1 - st0) {
                const int c = tile_col(tile) + l8 * 16, word = c / 8;
                const bool in0 = word < CP, in1 = word + 1 < CP;
                const uint32_t *w0 = P.d.packed[0] + word, *w1 = P.d.mats == 2 ? P.d.packed[1] + word : w0;
                const __half2 *sp = P.d.pairs + (c >> sh);            // 16 channels lie in one group
                // whole halves inside one matrix, and a tile inside its columns: no test and little address work per load
                const bool whole = P.d.vec8 && tile_col(tile) + kMT <= (int)P.d.C;
                const auto fetch = [&](int st, int h, Half &H) {
                    const int kb = st * kStageK + h * 64;
                    if (whole && kb + 64 <= K && (kb + 64 <= R || kb >= R)) {
                        const uint32_t *src = (kb >= R ? w1 : w0) + (int64_t)((kb >= R ? kb - R : kb) + k0) * CP;
                        const __half2 *ss = sp + (int64_t)(kb + k0) * G;
#pragma unroll
                        for (int p = 0; p < 4; ++p, src += 16 * CP, ss += 16 * G) {
                            H.w[p] = __ldg(reinterpret_cast<const uint2 *>(src));
                            H.s[p] = __ldg(ss);
                        }
                        return;
                    }
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        const int k = kb + k0 + 16 * p;
                        const uint32_t *src = (k < R ? w0 : w1) + (int64_t)(k < R ? k : k - R) * CP;
                        uint2 v = make_uint2(kZeroWord, kZeroWord);
                        if (P.d.vec8) {
                            if (k < K && in0) v = __ldg(reinterpret_cast<const uint2 *>(src));
                        } else {
                            if (k < K && in0) v.x = __ldg(src);
                            if (k < K && in1) v.y = __ldg(src + 1);
                        }
                        H.w[p] = v;
                        H.s[p] = k < K && in0 ? __ldg(sp + (int64_t)k * G) : __half2(__ushort_as_half(0), __ushort_as_half(0));
                    }
                };
                // the parts that are asked for, the low one 64 K rows behind the high one
                const auto unpack = [&](uint32_t at, const Half &H, bool high, bool low) {
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        const __half2 hi = __low2half2(H.s[p]), lo = __high2half2(H.s[p]);
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint4 v = word_to_half<false>((e == 0) != swap ? H.w[p].x : H.w[p].y);
                            const uint4 w = make_uint4(scaled(v.x, hi, lo), scaled(v.y, hi, lo), scaled(v.z, hi, lo), scaled(v.w, hi, lo));
                            const uint32_t dst = at + p * 2048 + (e == 0 ? xa : xb);
                            if (high) sts128(dst, w);
                            if (low)
                                sts128(dst + 8192, make_uint4(scaled_low(v.x, hi, lo, w.x), scaled_low(v.y, hi, lo, w.y),
                                                              scaled_low(v.z, hi, lo, w.z), scaled_low(v.w, hi, lo, w.w)));
                        }
                    }
                };
                const int first = st0 + (PAIR ? (group + base) & 1 : 0);
                constexpr bool kBoth = PAIR && !kSplit;               // b: both halves of a stage, or one of two stages
                constexpr int kAhead = kBoth ? 1 : 2;
                const int half = PAIR || kSplit ? 0 : group;
                Half b[2];
                if (first < st1) fetch(first, half, b[0]);
                if (kBoth ? first < st1 : first + kTurn < st1) fetch(kBoth ? first : first + kTurn, kBoth ? 1 : half, b[1]);
                for (int stb = first; stb < st1 && ok; stb += kTurn * kAhead) {
#pragma unroll
                    for (int a = 0; a < kAhead; ++a) {
                        const int st = stb + a * kTurn;
                        if (st >= st1) break;
                        const uint32_t it = (uint32_t)(base + st - st0), s = it % kStages;
                        ok = wait_on(b_empty + 8 * s, ((it / kStages) & 1u) ^ 1u, abort_flag);
                        if (!ok) break;
                        const uint32_t at = smem_base + s * kStageBytes + d0;
                        if constexpr (kBoth) {
                            unpack(at, b[0], true, false);
                            unpack(at + 8192, b[1], true, false);
                        } else if constexpr (!kSplit) {
                            unpack(at + group * 8192, b[a], true, false);
                        } else if constexpr (PAIR) {
                            unpack(at, b[a], true, true);
                        } else {                                      // one group the high parts, the other the low ones
                            if (group == 0) unpack(at, b[a], true, false);
                            else unpack(at, b[a], false, true);
                        }
                        publish(s);
                        if (st + kTurn * kAhead < st1) {
                            fetch(st + kTurn * kAhead, half, b[a]);
                            if constexpr (kBoth) fetch(st + kTurn * kAhead, 1, b[1]);
                        }
                    }
                }
            }
        }
        __syncwarp();
        if (P.split > 1) cluster_sync();
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Regs<MODE>::kMisc));
        if (warp == 16) {
            // ------------------------------ token tile by TMA ------------------------------
            uint32_t it = 0;
            bool ok = true;
            if (lane == 0) {
                for (int tile = tile0; tile < ntiles && ok; tile += tile_step) {
                    const int t0 = (tile / P.rt) * NT + (PAIR ? member * kBRows : 0);
                    for (int st = st0; st < st1; ++st, ++it) {
                        const uint32_t s = it % kStages;
                        ok = wait_on(b_empty + 8 * s, ((it / kStages) & 1u) ^ 1u, abort_flag);
                        if (!ok) break;
                        const uint32_t dst = smem_base + s * kStageBytes + kABytes;
                        const int x0 = st * kStageK, x1 = kSplit ? (int)P.d.lo + x0 : x0 + 64;    // dz's low parts lie behind its high ones
                        const bool both = !kSplit || P.d.lo != 0;
                        if constexpr (PAIR) {
                            if (member == 0) mbar_arrive_expect_tx(b_full + 8 * s, both ? 2 * kBBytes : kBBytes);
                            tma_load_2d_pair(dst, &tmap, x0, t0, even_cta(b_full + 8 * s));
                            if (both) tma_load_2d_pair(dst + kSubB, &tmap, x1, t0, even_cta(b_full + 8 * s));
                        } else {
                            mbar_arrive_expect_tx(b_full + 8 * s, both ? kBBytes : kSubB);
                            tma_load_2d(dst, &tmap, x0, t0, b_full + 8 * s);
                            if (both) tma_load_2d(dst + kSubB, &tmap, x1, t0, b_full + 8 * s);
                        }
                    }
                }
            }
        } else if (warp == 17) {
            // ------------------------------ MMA issuer ------------------------------
            // the whole warp walks the loop and one elected lane issues, so addresses and descriptors stay uniform
            uint32_t s = 0, phase = 0, chunk = 0;
            bool ok = !PAIR || member == 0;
            constexpr int kStepsPer = kSplit ? 12 : (CH < kKT ? CH : kKT) / 16;       // k-steps of a chunk inside a stage
            const int steps = kSplit && P.d.lo == 0 ? 8 : kStepsPer;
            const uint64_t ad0 = MODE == kDgrad ? desc_mnmajor(smem_base) : desc_kmajor(smem_base);
            const uint64_t bd0 = desc_kmajor(smem_base + kABytes);
            for (int tile = tile0; tile < ntiles && ok; tile += tile_step) {
                for (int st = st0; st < st1; ++st) {
                    ok = wait_on(b_full + 8 * s, phase, abort_flag);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after();
                    const bool first_stage = st % kStagesPer == 0 || st == st0;
                    const bool last_stage = st % kStagesPer == kStagesPer - 1 || st + 1 == st1;
                    const uint64_t ad = ad0 + (uint64_t)(s * (kStageBytes >> 4)), bd = bd0 + (uint64_t)(s * (kStageBytes >> 4));
#pragma unroll
                    for (int e = 0; e < kPerStage; ++e) {
                        if (first_stage) {
                            ok = wait_on(b_aempty + 8 * (chunk & 1u), ((chunk >> 1) & 1u) ^ 1u, abort_flag);
                            ok = __all_sync(0xffffffffu, ok);
                            if (!ok) break;
                            tc_fence_after();
                        }
                        if (elect_one()) {
                            const uint32_t d = tmem_base + (chunk & 1u) * NT;
#pragma unroll
                            for (int i = 0; i < kStepsPer; ++i) {
                                if (kSplit && i >= steps) break;
                                // split: high x high, low x high, high x low, four k-steps each
                                const int kk = e * kStepsPer + i, ka = kSplit && i >= 8 ? i - 8 : kk;
                                const int kb = !kSplit ? kk : i >= 8 ? i - 4 : i & 3;
                                const uint64_t a = ad + (MODE == kDgrad ? ka * 2048 : (ka >> 2) * kSubA + (ka & 3) * 32) / 16;
                                const uint64_t bb = bd + ((kb >> 2) * kSubB + (kb & 3) * 32) / 16;
                                const uint32_t more = (i == 0 && first_stage) ? 0u : 1u;
                                if constexpr (PAIR) umma_f16_pair(d, a, bb, idesc<MODE, kBf16>(2 * kMT, NT), more);
                                else umma_f16(d, a, bb, idesc<MODE, kBf16>(kMT, NT), more);
                            }
                            if (last_stage) {
                                if (PAIR) umma_commit_pair(b_afull + 8 * (chunk & 1u));
                                else umma_commit(b_afull + 8 * (chunk & 1u));
                            }
                            if (e == kPerStage - 1) {
                                if (PAIR) umma_commit_pair(b_empty + 8 * s);
                                else umma_commit(b_empty + 8 * s);
                            }
                        }
                        __syncwarp();
                        if (last_stage) ++chunk;
                    }
                    if (!ok) break;
                    if (++s == kStages) { s = 0; phase ^= 1u; }
                }
            }
        }
        __syncwarp();
        if (P.split > 1) cluster_sync();
    }
    // ------------------------------ teardown ------------------------------
    if (PAIR || P.split > 1) {
        __syncwarp();
        cluster_sync();          // nobody leaves while its sums or operands are being read, or its barriers arrived on
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {           // gave up: let copies and MMAs in flight land before shared and tensor memory are given back
        const long long c0 = clock64();
        while (clock64() - c0 < 200000) __nanosleep(1000);
        if (tid == 0 && P.status) atomicExch(P.status, FORGE_ERR_TIMEOUT);
        __syncthreads();
    }
    if (warp == 17) {
        tc_fence_after();
        if constexpr (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2u * NT) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2u * NT) : "memory");
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
// [rows, cols] of 16-bit elements, row stride ld elements; box of 64 columns x box_rows rows, 128-byte swizzle, zero fill
bool make_map(CUtensorMap *m, const void *base, bool bf16, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
    EncodeFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, es[2] = {1, 1};
    return fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(base), dims,
              strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct TokenSource {
    const void *base;
    bool bf16;
    int64_t rows, cols, ld;
};

template <typename T, int MODE, int CH, int NT, bool PAIR>
int launch(TcParams &P, const TokenSource &src, const char *who, cudaStream_t st) {
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const int64_t rt = cdiv(P.N, (int64_t)(MODE == kGated ? 64 : kMT) * (PAIR ? 2 : 1)), tt = cdiv(P.T, (int64_t)NT), tiles = rt * tt;
    if (tiles > 0x0fffffff) {
        set_error("%s: more than 2^28 output tiles", who);
        return FORGE_ERR_UNSUPPORTED;
    }
    alignas(64) CUtensorMap map;
    if (!make_map(&map, src.base, src.bf16, src.rows, src.cols, src.ld, PAIR ? NT / 2 : NT)) {
        set_error("%s: no tensor map could be made", who);
        return FORGE_ERR_LAUNCH;
    }
    P.rt = (int)rt;
    P.tt = (int)tt;
    // Clusters of this size that a B200 runs at once with one such CTA per SM (cudaOccupancyMaxActiveClusters): the largest
    // share of the K axis whose clusters all run together and that leaves a member two stages of work.
    static const int kResident[9] = {0, 148, 74, 45, 33, 26, 22, 15, 15};
    P.split = 1;
    if (!PAIR)
        for (int c = 8; c > 1; --c)
            if (tiles <= kResident[c] && P.nst >= 2 * c) {
                P.split = c;
                break;
            }
    P.per = (P.nst + P.split - 1) / P.split;
    P.split = (P.nst + P.per - 1) / P.per;                             // no member without stages
    const auto kernel = int4_tc_kernel<T, MODE, CH, NT, PAIR>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)(PAIR ? 2 * imin64(tiles, sms / 2) : P.split > 1 ? tiles * P.split : imin64(tiles, sms)));
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = kSmemBytes;
        cfg.stream = st;
        cudaLaunchAttribute at{};
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = (unsigned)(PAIR ? 2 : P.split);
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
// Token tiles of 64 or 128 for one CTA; pairs with 256 as soon as their tiles keep more than half of the SMs busy (below
// that, sharing the K axis among more CTAs counts for more).
template <typename T, int MODE, int CH> int launch_nt(TcParams &P, const TokenSource &src, const char *who, cudaStream_t st) {
    if (P.T <= 64) return launch<T, MODE, CH, 64, false>(P, src, who, st);
    const int64_t pairs = cdiv(P.N, (int64_t)(MODE == kGated ? 128 : 2 * kMT)) * cdiv(P.T, (int64_t)256);
    if (pairs > 37) return launch<T, MODE, CH, 256, true>(P, src, who, st);
    return launch<T, MODE, CH, 128, false>(P, src, who, st);
}
template <typename T, int MODE> int launch_gs(TcParams &P, const TokenSource &src, const char *who, cudaStream_t st) {
    if (P.f.gs == 32) return launch_nt<T, MODE, 32>(P, src, who, st);
    if (P.f.gs == 64) return launch_nt<T, MODE, 64>(P, src, who, st);
    return launch_nt<T, MODE, 128>(P, src, who, st);
}

}  // namespace

namespace forge {

int int4_fwd_tc(const Int4Fwd &F, bool bf16, bool gated, cudaStream_t st) {
    const char *who = gated ? "forge_int4_gated" : "forge_int4_linear";
    TcParams P{};
    P.f = F; P.T = F.T; P.N = F.R; P.status = F.status;
    P.nst = (int)cdiv(F.C, (int64_t)kKT);
    P.res_vec = F.ldres % 8 == 0 && (uintptr_t)F.res % 16 == 0;
    P.simple = !F.bias && !F.pre0 && F.act == FORGE_ACT_NONE && F.R % 8 == 0 && (!F.res || P.res_vec);
    const TokenSource src{F.x, bf16, F.T, F.C, F.ldx};
    if (bf16) return gated ? launch_gs<__nv_bfloat16, kGated>(P, src, who, st) : launch_gs<__nv_bfloat16, kLinear>(P, src, who, st);
    return gated ? launch_gs<__half, kGated>(P, src, who, st) : launch_gs<__half, kLinear>(P, src, who, st);
}

int int4_dgrad_tc(const Int4Dgrad &D, bool bf16, const char *who, cudaStream_t st) {
    TcParams P{};
    P.d = D; P.T = D.T; P.N = D.C; P.status = D.status;
    P.nst = (int)cdiv(D.ldk, (int64_t)(bf16 ? kKT : kKT / 2));
    const TokenSource src{D.a, false, D.T, D.ldk + D.lo, D.ldk + D.lo};
    return bf16 ? launch_nt<__nv_bfloat16, kDgrad, kKBlock>(P, src, who, st) : launch_nt<__half, kDgrad, kKBlock>(P, src, who, st);
}

}  // namespace forge

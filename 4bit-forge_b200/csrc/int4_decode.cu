// int4 products for few tokens (up to 16): the weights are streamed once, from global memory straight into the operand
// registers of warp-level m16n8k16 matrix instructions; 16 weight rows are the M side, the tokens the N side.
//
//   acc[r, t] = sum over groups  scale[r, g] * ( sum over the group's channels  (nibble - 8) * x[t, c] )
//
// The inner sum has exact operands (nibble - 8 is an integer of four bits, x is as given) and runs in the instruction's
// fp32 accumulator over gs channels at most; the scale enters in fp32, once per group.  A sum over k does not care about
// the order of k, so a thread gives the instruction's k slots to the eight channels of one packed word, four per
// instruction, and takes the same channels of x: neither side is shuffled between threads.
//
// Bound by the weights' bytes (0.5 B per weight and 4 B of scale per group) once there is enough of them, below that by
// latency.  A CTA owns 16 rows; its warps share the K axis in blocks of 128 channels and join through shared memory in a
// fixed order, so there is one launch and no second pass.  One token, 2048 -> 7168: 5.5 us (7.8 MB); one token through
// gate and up, 7168 -> 2048: 7.5 us (15.7 MB, 2.1 TB/s).  Both are chains of a launch, two to four loads and a join; the
// next block's loads are under way while a block is multiplied.  Wide matrices, one token, 7168 -> 18432: 27.4 us (2.6 TB/s),
// gate and up 48.6 us (2.9 TB/s).  Above kDecodeTokens, where every CTA's reading all of x weighs, the tensor-memory kernel is
// the faster one.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"
#include "elem.cuh"
#include "int4_mm.cuh"

using namespace forge;

namespace {

template <typename T> struct Mma;
template <> struct Mma<__nv_bfloat16> {
    static constexpr uint32_t kMagic = 0x43004300u;      // 128.0: a nibble in the low mantissa bits adds its value
    static __device__ __forceinline__ uint32_t minus8(uint32_t v) {
        __nv_bfloat162 h = *reinterpret_cast<__nv_bfloat162 *>(&v);
        h = __hsub2(h, __floats2bfloat162_rn(136.0f, 136.0f));
        return *reinterpret_cast<uint32_t *>(&h);
    }
    static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                               uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
};
template <> struct Mma<__half> {
    static constexpr uint32_t kMagic = 0x64006400u;      // 1024.0
    static __device__ __forceinline__ uint32_t minus8(uint32_t v) {
        __half2 h = *reinterpret_cast<__half2 *>(&v);
        h = __hsub2(h, __floats2half2_rn(1032.0f, 1032.0f));
        return *reinterpret_cast<uint32_t *>(&h);
    }
    static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                               uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
};

// channels (0,4), (1,5), (2,6), (3,7) of a packed word as pairs of the 16-bit type
template <typename T> __device__ __forceinline__ void unpack(uint32_t w, uint32_t (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = Mma<T>::minus8(((w >> (4 * i)) & 0x000F000Fu) | Mma<T>::kMagic);
}

constexpr uint32_t kZeroWord = 0x88888888u;    // eight codes of value zero

// LW consecutive words of a row from word index j on; words past the row are zeros.  `vec`: rows start on LW words
template <int LW> __device__ __forceinline__ void load_words(const uint32_t *row, int j, int CP, bool vec, uint32_t (&w)[LW]) {
    if (vec && j < CP) {
        if constexpr (LW == 4) {
            const uint4 v = __ldg(reinterpret_cast<const uint4 *>(row + j));
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else if constexpr (LW == 2) {
            const uint2 v = __ldg(reinterpret_cast<const uint2 *>(row + j));
            w[0] = v.x; w[1] = v.y;
        } else {
            w[0] = __ldg(row + j);
        }
    } else {
#pragma unroll
        for (int i = 0; i < LW; ++i) w[i] = (j + i < CP) ? __ldg(row + j + i) : kZeroWord;
    }
}

// CTAs of eight warps on an SM: three where 80 registers hold two blocks of words, scales and tokens, two for gate and up and
// for groups of 32.  Held to three, those spilled up to 364 bytes a thread: gated, 1 token, 7168 -> 18432 took 64 us at groups
// of 128 and 149 us at groups of 32, and takes 49 and 80; linear at groups of 32 43 and 40.
constexpr int ctas_per_sm(bool gated, int gs, int nt, int warps) { return warps == 8 && nt == 1 ? (gated || gs == 32 ? 2 : 3) : 1; }

// GS: group size; NT: blocks of 8 tokens; W: warps
template <typename T, bool GATED, int GS, int NT, int W>
__global__ void __launch_bounds__(W * 32, ctas_per_sm(GATED, GS, NT, W)) decode_kernel(const Int4Fwd P) {
    constexpr int M = GATED ? 2 : 1;
    constexpr int LW = GS / 32;            // packed words of a group that one thread takes
    constexpr int NG = 128 / GS;           // groups in a block of 128 channels
    extern __shared__ float part[];        // [W][M][8 NT tokens][16 rows + 1]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int q = lane & 3, r8 = lane >> 2;
    const int64_t row0 = (int64_t)blockIdx.x * 16;
    const int CP = (int)(P.C / 8), nblk = (int)cdiv(P.C, (int64_t)128);
    const bool vec = P.vec16 || LW == 1 || (LW == 2 && P.vec8);
    const int64_t ra = row0 + r8 < P.R ? row0 + r8 : P.R - 1, rb = row0 + r8 + 8 < P.R ? row0 + r8 + 8 : P.R - 1;
    const uint32_t *wa[M], *wb[M];
    const float *sa[M], *sb[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
        wa[m] = P.packed[m] + ra * CP; wb[m] = P.packed[m] + rb * CP;
        sa[m] = P.scales[m] + ra * P.G; sb[m] = P.scales[m] + rb * P.G;
    }
    float acc[M][NT][4] = {};

    // one block of 128 channels: the words and scales of this thread's two rows, and (one token block) its channels of x;
    // the next block's are under way while a block is multiplied
    struct Block {
        uint32_t a[M][NG][LW], b[M][NG][LW];
        float fa[M][NG], fb[M][NG];
        uint4 x[NT == 1 ? 4 : 1];
    };
    const auto fetch_x = [&](int kb, int j, int i, int n) {
        const int word = kb * 16 + j * (GS / 8) + q * LW + i, t = n * 8 + r8;
        return t < (int)P.T && word < CP ? __ldg(reinterpret_cast<const uint4 *>((const T *)P.x + t * P.ldx + word * 8))
                                         : make_uint4(0u, 0u, 0u, 0u);
    };
    const auto fetch = [&](int kb, Block &B) {
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                const int word = kb * 16 + j * (GS / 8) + q * LW, g = kb * NG + j;
                load_words<LW>(wa[m], word, CP, vec, B.a[m][j]);
                load_words<LW>(wb[m], word, CP, vec, B.b[m][j]);
                B.fa[m][j] = g < (int)P.G ? __ldg(sa[m] + g) : 0.0f;
                B.fb[m][j] = g < (int)P.G ? __ldg(sb[m] + g) : 0.0f;
            }
        if constexpr (NT == 1)
#pragma unroll
            for (int k = 0; k < 4; ++k) B.x[k] = fetch_x(kb, k / LW, k % LW, 0);
    };
    Block next;
    if (warp < nblk) fetch(warp, next);
    for (int kb = warp; kb < nblk; kb += W) {
        const Block B = next;
        if (kb + W < nblk) fetch(kb + W, next);
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            float d[M][NT][4] = {};
#pragma unroll
            for (int i = 0; i < LW; ++i) {
                uint32_t b[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint4 v;
                    if constexpr (NT == 1) v = B.x[j * LW + i];
                    else v = fetch_x(kb, j, i, n);
                    b[n][0] = __byte_perm(v.x, v.z, 0x5410);   // channels 0, 4
                    b[n][1] = __byte_perm(v.x, v.z, 0x7632);   // 1, 5
                    b[n][2] = __byte_perm(v.y, v.w, 0x5410);   // 2, 6
                    b[n][3] = __byte_perm(v.y, v.w, 0x7632);   // 3, 7
                }
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    uint32_t a[4], c[4];
                    unpack<T>(B.a[m][j][i], a);
                    unpack<T>(B.b[m][j][i], c);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        Mma<T>::mma(d[m][n], a[0], c[0], a[1], c[1], b[n][0], b[n][1]);
                        Mma<T>::mma(d[m][n], a[2], c[2], a[3], c[3], b[n][2], b[n][3]);
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    acc[m][n][0] = fmaf(B.fa[m][j], d[m][n][0], acc[m][n][0]);
                    acc[m][n][1] = fmaf(B.fa[m][j], d[m][n][1], acc[m][n][1]);
                    acc[m][n][2] = fmaf(B.fb[m][j], d[m][n][2], acc[m][n][2]);
                    acc[m][n][3] = fmaf(B.fb[m][j], d[m][n][3], acc[m][n][3]);
                }
        }
    }
    // a thread holds rows r8, r8 + 8 and tokens 2q, 2q + 1 of every 8-token block
    constexpr int kTok = NT * 8;
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float *p = part + ((warp * M + m) * kTok + n * 8 + 2 * q) * 17 + r8;
            p[0] = acc[m][n][0]; p[17] = acc[m][n][1]; p[8] = acc[m][n][2]; p[25] = acc[m][n][3];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < kTok * 16; i += W * 32) {
        const int t = i >> 4, r = i & 15;
        const int64_t row = row0 + r;
        if (t >= P.T || row >= P.R) continue;
        float z = 0.0f, u = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            z += part[((w * M) * kTok + t) * 17 + r];
            if constexpr (GATED) u += part[((w * M + 1) * kTok + t) * 17 + r];
        }
        const int64_t o = t * P.R + row;
        if (!GATED && P.bias) z += Elem<T>::to_f(((const T *)P.bias)[row]);
        if (P.pre0) ((T *)P.pre0)[o] = Elem<T>::from_f(z);
        float y = act_fwd_rt(P.act, z);
        if constexpr (GATED) {
            if (P.pre1) ((T *)P.pre1)[o] = Elem<T>::from_f(u);
            y *= u;
        } else if (P.res) {
            y += Elem<T>::to_f(((const T *)P.res)[t * P.ldres + row]);
        }
        ((T *)P.y)[o] = Elem<T>::from_f(y);
    }
}

template <typename T, bool GATED, int GS, int NT, int W> int launch_w(const Int4Fwd &P, cudaStream_t st) {
    constexpr int smem = W * (GATED ? 2 : 1) * NT * 8 * 17 * 4;
    static_assert(smem <= 48 * 1024, "fits the default shared memory");
    decode_kernel<T, GATED, GS, NT, W><<<(unsigned)cdiv(P.R, (int64_t)16), W * 32, smem, st>>>(P);
    FORGE_NOTE_LAUNCH();
    return check_launch(GATED ? "forge_int4_gated" : "forge_int4_linear");
}
// Sixteen warps share the K axis where a CTA has an SM to itself, eight where several are resident.
template <typename T, bool GATED, int GS, int NT> int launch(const Int4Fwd &P, cudaStream_t st) {
    if (P.R <= 148 * 16 && P.C > 1024) return launch_w<T, GATED, GS, NT, 16>(P, st);
    return launch_w<T, GATED, GS, NT, 8>(P, st);
}
template <typename T, bool GATED, int GS> int launch_nt(const Int4Fwd &P, cudaStream_t st) {
    if (P.T <= 8) return launch<T, GATED, GS, 1>(P, st);
    return launch<T, GATED, GS, 2>(P, st);
}
template <typename T, bool GATED> int launch_gs(const Int4Fwd &P, cudaStream_t st) {
    if (P.gs == 32) return launch_nt<T, GATED, 32>(P, st);
    if (P.gs == 64) return launch_nt<T, GATED, 64>(P, st);
    return launch_nt<T, GATED, 128>(P, st);
}

}  // namespace

namespace forge {
int int4_decode(const Int4Fwd &P, bool bf16, bool gated, cudaStream_t st) {
    if (bf16) return gated ? launch_gs<__nv_bfloat16, true>(P, st) : launch_gs<__nv_bfloat16, false>(P, st);
    return gated ? launch_gs<__half, true>(P, st) : launch_gs<__half, false>(P, st);
}
}  // namespace forge

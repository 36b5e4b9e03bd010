// mm_tiles.hpp — matrix products of the item scores (scores.hip) and of the
// softmax loss (softmax.hip) on the matrix cores.
//
// Two forms, both with f32 (bf16 operands) or int32 (int8 operands) sums:
//   k_nt   Y[i][j] = sum_k A[i][k] B[j][k]     (rows against rows)
//   k_kn   Y[m][n] = sum_k A(m,k) B[k][n]      (A [m][k] or [k][m])
// An epilogue object takes each wave's accumulators.
//
// f32 operands come as three bf16 planes x = h + m + l (8 + 8 + 8 significant
// bits: exact but for subnormal tails).  Their product is the sum of six bf16
// products (hh, hm, mh, hl, lh, mm); what is left out (ml, lm, ll) is below
// 2^-25 of |x||y|, the rounding of one f32 product.  The small ones are added
// first.
#pragma once
#include "common.hpp"

namespace mn {
namespace mm {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

constexpr int KBY = 64;  // bytes of a row in one k-step: 32 bf16 or 64 int8

// planes of A and B in the six products, smallest first
__device__ __forceinline__ int seg_a(int s) { return (0x001021 >> (4 * s)) & 3; }
__device__ __forceinline__ int seg_b(int s) { return (0x010201 >> (4 * s)) & 3; }

struct Bf16 {
    typedef f32x4 acc_t;
    static __device__ __forceinline__ acc_t mma(uint4 a, uint4 b, acc_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
struct Int8 {
    typedef i32x4 acc_t;
    static __device__ __forceinline__ acc_t mma(uint4 a, uint4 b, acc_t c) {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a),
                                                     __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
    }
};

struct NtArgs {
    const char *A;      // [nplane][m][lda], rows zero from their end to nk * KBY
    const char *B;      // [nplane][n][ldb]; bytes past bmax + 16 are never read
    int64_t lda, ldb;   // bytes
    int64_t planeA, planeB;
    int64_t m, n;
    int nk;             // k-steps of KBY bytes
    int nseg;           // 1, or 6 (f32 planes)
    int bmax;           // last 16-byte piece of a row of B
};

// 128 x 128 tile, four waves of 64 x 64.
template <class OP, class EPI>
__global__ __launch_bounds__(256) void k_nt(NtArgs a, EPI epi, int64_t tiles_j) {
    __shared__ uint4 sA[128][5], sB[128][5];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int64_t bi = blockIdx.x / tiles_j, bj = blockIdx.x % tiles_j;
    const int64_t i0 = bi * 128, j0 = bj * 128;
    typename OP::acc_t acc[4][4];
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int g = 0; g < 4; ++g) acc[f][g] = (typename OP::acc_t)(0);
    for (int sg = 0; sg < a.nseg; ++sg) {
        const char *A = a.A + (a.nseg == 1 ? 0 : seg_a(sg) * a.planeA);
        const char *B = a.B + (a.nseg == 1 ? 0 : seg_b(sg) * a.planeB);
        for (int k = 0; k < a.nk; ++k) {
#pragma unroll
            for (int e = tid; e < 512; e += 256) {
                const int r = e >> 2, c = e & 3;
                const int64_t ra = min(i0 + r, a.m - 1), rb = min(j0 + r, a.n - 1);
                sA[r][c] = *reinterpret_cast<const uint4 *>(A + ra * a.lda + k * KBY + 16 * c);
                sB[r][c] = *reinterpret_cast<const uint4 *>(B + rb * a.ldb + min(k * KBY + 16 * c, a.bmax));
            }
            __syncthreads();
            uint4 fa[4], fb[4];
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                fa[f] = sA[64 * (w & 1) + 16 * f + (lane & 15)][lane >> 4];
                fb[f] = sB[64 * (w >> 1) + 16 * f + (lane & 15)][lane >> 4];
            }
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int g = 0; g < 4; ++g) acc[f][g] = OP::mma(fb[g], fa[f], acc[f][g]);
            __syncthreads();
        }
    }
    // acc[f][g][r] = Y[i0w + 16 f + (lane & 15)][j0w + 16 g + 4 (lane >> 4) + r]
    epi(acc, i0 + 64 * (w & 1), j0 + 64 * (w >> 1), lane);
}

struct KnArgs {
    const uint16_t *A;  // [nplane][m][lda] (A_T false) or [nplane][k][lda] (A_T true)
    const uint16_t *B;  // [nplane][k][ldb]
    int64_t lda, ldb, planeA, planeB;
    int64_t m, n, k;    // rows / columns past m, n, k are not used
    int64_t kpart;      // k's per grid z
    int nseg;
};

// 128 x 128 tile, four waves of 64 x 64; blockIdx.z takes k's [z kpart, +kpart).
template <bool A_T, class EPI>
__global__ __launch_bounds__(256) void k_kn(KnArgs a, EPI epi) {
    __shared__ uint16_t sA[128][40], sB[128][40];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int64_t m0 = (int64_t)blockIdx.x * 128, n0 = (int64_t)blockIdx.y * 128;
    const int64_t kb = blockIdx.z * a.kpart, ke = min(a.k, kb + a.kpart);
    f32x4 acc[4][4];
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int g = 0; g < 4; ++g) acc[f][g] = (f32x4)(0.f);
    for (int sg = 0; sg < a.nseg; ++sg) {
        const uint16_t *A = a.A + (a.nseg == 1 ? 0 : seg_a(sg) * a.planeA);
        const uint16_t *B = a.B + (a.nseg == 1 ? 0 : seg_b(sg) * a.planeB);
        for (int64_t k0 = kb; k0 < ke; k0 += 32) {
            for (int e = tid; e < 128 * 32; e += 256) {
                const int kk = e >> 7, c = e & 127;
                const int64_t k = k0 + kk;
                sB[c][kk] = k < ke && n0 + c < a.n ? B[k * a.ldb + n0 + c] : (uint16_t)0;
                if (A_T) {
                    sA[c][kk] = k < ke && m0 + c < a.m ? A[k * a.lda + m0 + c] : (uint16_t)0;
                } else {
                    const int r = e >> 5, q = e & 31;
                    sA[r][q] = k0 + q < ke && m0 + r < a.m ? A[(m0 + r) * a.lda + k0 + q] : (uint16_t)0;
                }
            }
            __syncthreads();
            uint4 fa[4], fb[4];
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                fa[f] = *reinterpret_cast<const uint4 *>(&sA[64 * (w & 1) + 16 * f + (lane & 15)][8 * (lane >> 4)]);
                fb[f] = *reinterpret_cast<const uint4 *>(&sB[64 * (w >> 1) + 16 * f + (lane & 15)][8 * (lane >> 4)]);
            }
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int g = 0; g < 4; ++g) acc[f][g] = Bf16::mma(fb[g], fa[f], acc[f][g]);
            __syncthreads();
        }
    }
    // acc[f][g][r] = Y[m0w + 16 f + (lane & 15)][n0w + 16 g + 4 (lane >> 4) + r]
    epi(acc, m0 + 64 * (w & 1), n0 + 64 * (w >> 1), lane, (int)blockIdx.z);
}

__device__ __forceinline__ uint16_t bf16_bits(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
__device__ __forceinline__ float bf16_value(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }

// x = h + m + l.  A finite x whose nearest bf16 is infinite takes the one
// below; m and l of a non-finite x are 0.
__device__ __forceinline__ void split3(float x, uint16_t (&p)[3]) {
    uint16_t h = bf16_bits(x);
    const bool finite = (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
    if (finite && (h & 0x7f80u) == 0x7f80u) h = (uint16_t)(__float_as_uint(x) >> 16);
    const float r = finite ? x - bf16_value(h) : 0.f;
    p[0] = h;
    p[1] = bf16_bits(r);
    p[2] = bf16_bits(r - bf16_value(p[1]));
}

}  // namespace mm
}  // namespace mn

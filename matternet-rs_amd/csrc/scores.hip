// scores.hip — rows in 8 bits with a scale per row, and the scores of
// quantised queries against a quantised item table:
//
//     a_i = max_k |x_ik|,  scale_i = a_i / 127,  code_ik = rint(x_ik (127 (1 / a_i)))
//     y_ij = (sum_k qcode_ik ccode_jk) qscale_i cscale_j
//
// The sums are exact (int32: 128 * 128 * d < 2^31 for d <= 131071); y is the
// sum rounded to f32, times the query's scale, times the item's.
#include <algorithm>
#include <climits>

#include "common.hpp"
#include "mm_tiles.hpp"

namespace mn {
namespace i8 {

// A row's largest |x| as bits: NaN > inf > every finite value, so one integer
// maximum also tells whether the row holds something that is not finite.
template <typename T>
__device__ __forceinline__ float load_x(const T *X, int64_t e);
template <>
__device__ __forceinline__ float load_x<float>(const float *X, int64_t e) { return X[e]; }
template <>
__device__ __forceinline__ float load_x<uint16_t>(const uint16_t *X, int64_t e) { return mm::bf16_value(X[e]); }

// Below 2^-100 the reciprocal 1 / a could overflow, above 2^100 be subnormal:
// such a row is multiplied by 2^64 or 2^-64 first (exact where it matters).  A row of zeros has scale 0 and codes 0; a row that
// holds an infinity or a NaN has scale NaN, which every score with it shows.
template <typename T>
__global__ __launch_bounds__(256) void k_quantize(const T *__restrict__ X, int64_t n, int d,
                                                  int8_t *__restrict__ codes, int64_t ld,
                                                  float *__restrict__ scale) {
    const int lane = threadIdx.x & 63;
    for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += (int64_t)gridDim.x * 4) {
        uint32_t top = 0;
        for (int k = lane; k < d; k += 64) top = max(top, __float_as_uint(load_x(X, i * d + k)) & 0x7fffffffu);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
        float a = __uint_as_float(top);
        const bool finite = top < 0x7f800000u;
        const float up = a < 0x1p-100f ? 0x1p64f : a > 0x1p100f ? 0x1p-64f : 1.f;
        const float inv = finite && top != 0 ? 1.f / (a * up) * 127.f : 0.f;
        for (int k = lane; k < ld; k += 64) {
            float v = 0.f;
            if (k < d && finite) v = __builtin_rintf(load_x(X, i * d + k) * up * inv);
            codes[i * ld + k] = (int8_t)(int)fminf(fmaxf(v, -127.f), 127.f);
        }
        if (lane == 0) scale[i] = finite ? a / 127.f : __builtin_nanf("");
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_dequantize(const int8_t *__restrict__ codes, int64_t ld,
                                                    const float *__restrict__ scale, int64_t n, int d,
                                                    T *__restrict__ X) {
    const int lane = threadIdx.x & 63;
    for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += (int64_t)gridDim.x * 4) {
        const float s = scale[i];
        for (int k = lane; k < d; k += 64) {
            const float v = (float)codes[i * ld + k] * s;
            if constexpr (sizeof(T) == 4) X[i * d + k] = v;
            else X[i * d + k] = mm::bf16_bits(v);
        }
    }
}

// the queries' codes with zeros up to whole k-steps
__global__ __launch_bounds__(256) void k_pad_codes(const int8_t *__restrict__ Q, int64_t ldq, int64_t m,
                                                   int d, int ldp, int8_t *__restrict__ out) {
    const int64_t total = m * ldp, stride = (int64_t)gridDim.x * 256;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += stride) {
        const int64_t i = e / ldp;
        const int k = (int)(e - i * ldp);
        out[e] = k < d ? Q[i * ldq + k] : (int8_t)0;
    }
}

template <typename T>
struct ScoreEpi {
    struct Shared {
        float cs[2][mm::TILE];  // the items' scales of a tile, two tiles in turn
    };
    static constexpr bool FETCH = true;
    const float *qs, *cs;
    T *Y;
    int64_t m, n;
    float q[4];
    int64_t i0_;
    __device__ __forceinline__ void init(Shared &, int64_t i0, int lane) {
        i0_ = i0;
#pragma unroll
        for (int f = 0; f < 4; ++f) q[f] = qs[min(i0 + 16 * f + (lane & 15), m - 1)];
    }
    __device__ __forceinline__ void fetch(Shared &sh, int64_t j0, int tid, int par) {
        const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
        if (w < 4)
            mm::dma4((const char *)(cs + j0), 4 * (int)min<int64_t>(tid, n - 1 - j0), mm::lds_addr(&sh.cs[par][64 * w]));
    }
    __device__ __forceinline__ void tile(Shared &sh, mm::i32x4 (&acc)[4][8], int64_t j0, int lane, int par) {
        const int jl = 8 * (lane >> 4);
#pragma unroll
        for (int g = 0; g < 8; g += 2) {
            const int64_t j = j0 + jl + 16 * g;
            float c[8];
#pragma unroll
            for (int q8 = 0; q8 < 8; ++q8) c[q8] = sh.cs[par][(int)(j0 & (mm::TILE - 1)) + jl + 16 * g + q8];
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                const int64_t i = i0_ + 16 * f + (lane & 15);
                float x[8];
#pragma unroll
                for (int q8 = 0; q8 < 8; ++q8) x[q8] = (float)acc[f][g + (q8 >> 2)][q8 & 3] * q[f] * c[q8];
                if (i >= m) continue;
                T *p = Y + i * n + j;
                if constexpr (sizeof(T) == 4) {
                    if (j + 8 <= n) {
                        __builtin_memcpy(p, x, 32);
                    } else {
#pragma unroll
                        for (int q8 = 0; q8 < 8; ++q8)
                            if (j + q8 < n) p[q8] = x[q8];
                    }
                } else {
                    if (j + 8 <= n) {
                        const uint4 y = make_uint4(mm::bf16_pair(x[0], x[1]), mm::bf16_pair(x[2], x[3]),
                                                   mm::bf16_pair(x[4], x[5]), mm::bf16_pair(x[6], x[7]));
                        __builtin_memcpy(p, &y, 16);
                    } else {
#pragma unroll
                        for (int q8 = 0; q8 < 8; ++q8)
                            if (j + q8 < n) p[q8] = mm::bf16_bits(x[q8]);
                    }
                }
            }
        }
    }
    __device__ __forceinline__ void finish(Shared &, int64_t, int, int) {}
};

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
inline int padded(int d) { return (d + mm::KBY - 1) / mm::KBY * mm::KBY; }

}  // namespace i8
}  // namespace mn

extern "C" int mn_quantize_rows_i8(const void *X, int32_t x_type, int64_t n, int32_t d,
                                   int8_t *codes, int64_t ld, float *scale, void *stream) {
    using namespace mn::i8;
    mn::clear_error();
    MN_REQUIRE(n >= 0 && d >= 1 && ld >= d && ld % 16 == 0 && ld <= INT_MAX, MN_EINVAL,
               "mn_quantize_rows_i8: n >= 0, d >= 1, ld >= d and a multiple of 16 needed");
    MN_REQUIRE(x_type == MN_F32 || x_type == MN_BF16, MN_ENOTSUP, "mn_quantize_rows_i8: MN_F32 or MN_BF16");
    if (n == 0) return MN_OK;
    MN_REQUIRE(X && codes && scale, MN_EINVAL, "mn_quantize_rows_i8: NULL pointer");
    MN_REQUIRE(aligned16(codes), MN_EINVAL, "mn_quantize_rows_i8: codes not 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    const unsigned grid = (unsigned)std::min<int64_t>((n + 3) / 4, 1 << 20);
    if (x_type == MN_F32)
        hipLaunchKernelGGL(k_quantize<float>, dim3(grid), dim3(256), 0, s, (const float *)X, n, d, codes, ld, scale);
    else
        hipLaunchKernelGGL(k_quantize<uint16_t>, dim3(grid), dim3(256), 0, s, (const uint16_t *)X, n, d, codes, ld, scale);
    MN_KCHECK(s, "k_quantize");
    return MN_OK;
}

extern "C" int mn_dequantize_rows_i8(const int8_t *codes, int64_t ld, const float *scale, int64_t n,
                                     int32_t d, void *X, int32_t x_type, void *stream) {
    using namespace mn::i8;
    mn::clear_error();
    MN_REQUIRE(n >= 0 && d >= 1 && ld >= d && ld % 16 == 0 && ld <= INT_MAX, MN_EINVAL,
               "mn_dequantize_rows_i8: n >= 0, d >= 1, ld >= d and a multiple of 16 needed");
    MN_REQUIRE(x_type == MN_F32 || x_type == MN_BF16, MN_ENOTSUP, "mn_dequantize_rows_i8: MN_F32 or MN_BF16");
    if (n == 0) return MN_OK;
    MN_REQUIRE(X && codes && scale, MN_EINVAL, "mn_dequantize_rows_i8: NULL pointer");
    MN_REQUIRE(aligned16(codes), MN_EINVAL, "mn_dequantize_rows_i8: codes not 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    const unsigned grid = (unsigned)std::min<int64_t>((n + 3) / 4, 1 << 20);
    if (x_type == MN_F32)
        hipLaunchKernelGGL(k_dequantize<float>, dim3(grid), dim3(256), 0, s, codes, ld, scale, n, d, (float *)X);
    else
        hipLaunchKernelGGL(k_dequantize<uint16_t>, dim3(grid), dim3(256), 0, s, codes, ld, scale, n, d, (uint16_t *)X);
    MN_KCHECK(s, "k_dequantize");
    return MN_OK;
}

extern "C" int mn_scores_i8_workspace(int64_t m, int32_t d, size_t *bytes) {
    mn::clear_error();
    MN_REQUIRE(bytes && m >= 0 && d >= 1 && d <= 131071, MN_EINVAL, "mn_scores_i8_workspace: bad args");
    *bytes = d % mn::mm::KBY == 0 ? 0 : (size_t)m * mn::i8::padded(d);
    return MN_OK;
}

extern "C" int mn_scores_i8(const int8_t *Q, int64_t ldq, const float *q_scale, int64_t m,
                            const int8_t *C, int64_t ldc, const float *c_scale, int64_t n, int32_t d,
                            void *Y, int32_t y_type, void *ws, size_t ws_bytes, void *stream) {
    using namespace mn;
    using namespace mn::i8;
    clear_error();
    MN_REQUIRE(m >= 0 && n >= 0 && d >= 1, MN_EINVAL, "mn_scores_i8: m >= 0, n >= 0, d >= 1 needed");
    MN_REQUIRE(m <= INT_MAX - 1024 && n <= INT_MAX - 1024 && (m + 255) / 256 * ((n + 255) / 256) < (1 << 30), MN_ENOTSUP,
               "mn_scores_i8: too many scores for one call");
    MN_REQUIRE(d <= 131071, MN_ENOTSUP, "mn_scores_i8: d > 131071 (an int32 sum could overflow)");
    MN_REQUIRE(ldq >= d && ldc >= d && ldq % 16 == 0 && ldc % 16 == 0, MN_EINVAL,
               "mn_scores_i8: row strides need to be >= d and multiples of 16");
    MN_REQUIRE(y_type == MN_F32 || y_type == MN_BF16, MN_ENOTSUP, "mn_scores_i8: MN_F32 or MN_BF16 scores");
    if (m == 0 || n == 0) return MN_OK;
    MN_REQUIRE(Q && q_scale && C && c_scale && Y, MN_EINVAL, "mn_scores_i8: NULL pointer");
    MN_REQUIRE(aligned16(Q) && aligned16(C), MN_EINVAL, "mn_scores_i8: codes not 16-byte aligned");
    const int ldp = padded(d);
    const size_t need = d % mm::KBY == 0 ? 0 : (size_t)m * ldp;
    MN_REQUIRE(need == 0 || (ws && ws_bytes >= need && aligned16(ws)), MN_ECAP,
               "mn_scores_i8: workspace of %zu bytes (16-byte aligned) needed", need);
    hipStream_t s = (hipStream_t)stream;
    const int8_t *A = Q;
    int64_t lda = ldq;
    if (need) {
        const unsigned grid = (unsigned)std::min<int64_t>((m * ldp + 255) / 256, 8192);
        hipLaunchKernelGGL(k_pad_codes, dim3(grid), dim3(256), 0, s, Q, ldq, m, d, ldp, (int8_t *)ws);
        MN_KCHECK(s, "k_pad_codes");
        A = (const int8_t *)ws;
        lda = ldp;
    }
    mm::NtArgs a = {};
    a.A = (const char *)A;
    a.B = (const char *)C;
    a.lda = lda;
    a.ldb = ldc;
    a.m = m;
    a.n = n;
    a.nk = ldp / mm::KBY;
    a.nseg = 1;
    a.bmax = (d + 15) / 16 * 16 - 16;
    mm::plan_runs(a);
    const dim3 grid((unsigned)(a.panels * a.slices));
    if (y_type == MN_F32) {
        ScoreEpi<float> epi = {};
        epi.qs = q_scale;
        epi.cs = c_scale;
        epi.Y = (float *)Y;
        epi.m = m;
        epi.n = n;
        hipLaunchKernelGGL((mm::k_nt<mm::Int8, ScoreEpi<float>>), grid, dim3(mm::NT), 0, s, a, epi);
    } else {
        ScoreEpi<uint16_t> epi = {};
        epi.qs = q_scale;
        epi.cs = c_scale;
        epi.Y = (uint16_t *)Y;
        epi.m = m;
        epi.n = n;
        hipLaunchKernelGGL((mm::k_nt<mm::Int8, ScoreEpi<uint16_t>>), grid, dim3(mm::NT), 0, s, a, epi);
    }
    MN_KCHECK(s, "k_nt");
    return MN_OK;
}

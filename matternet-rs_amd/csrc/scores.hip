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
#include <type_traits>

#include "common.hpp"
#include "mm_tiles.hpp"

namespace mn {
namespace i8 {

// 8 values of a row from column k (a multiple of 8), zeros past column d.
// vec: rows start on 16-byte borders.  NT: past the caches.
template <bool NT, typename T>
__device__ __forceinline__ void load8(const T *row, int k, int d, bool vec, float (&v)[8]) {
    if (vec && k + 8 <= d) {
        if constexpr (sizeof(T) == 4) {
            const mm::f32x4 *p = reinterpret_cast<const mm::f32x4 *>(row + k);
            const mm::f32x4 a = NT ? __builtin_nontemporal_load(p) : p[0], b = NT ? __builtin_nontemporal_load(p + 1) : p[1];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = e < 4 ? a[e] : b[e - 4];
        } else {
            const mm::u32x4 *p = reinterpret_cast<const mm::u32x4 *>(row + k);
            const mm::u32x4 w = NT ? __builtin_nontemporal_load(p) : *p;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = mm::bf16_value((uint16_t)(w[e >> 1] >> (16 * (e & 1))));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool in = k + e < d;
            if constexpr (sizeof(T) == 4) v[e] = in ? row[k + e] : 0.f;
            else v[e] = in ? mm::bf16_value(row[k + e]) : 0.f;
        }
    }
}

// threads a block, whole rows of L lanes
constexpr int quantize_block(int L) { return L > 64 ? L : 256; }

// L lanes take a row, 8 values a lane at a time; up to 16 values a lane stay in
// registers between the two passes: such rows are read once, past the caches
// (262144 x 768 f32 and back: 314 us, 5.8 TB/s; 339 with ordinary loads); longer
// ones are read again, from L2.  A row's largest |x| is folded as bits: NaN > inf
// > every finite value, so one integer maximum also tells whether the row holds
// something that is not finite.
// Below 2^-100 the reciprocal 1 / a could overflow, above 2^100 be subnormal:
// such a row is multiplied by 2^64 or 2^-64 first (exact where it matters).  A
// row of zeros has scale 0 and codes 0; a row that holds an infinity or a NaN
// has scale NaN, which every score with it shows.
template <typename T, int L>
__global__ __launch_bounds__(quantize_block(L)) void k_quantize(const T *__restrict__ X, int64_t n, int d, bool vec,
                                                  int8_t *__restrict__ codes, int64_t ld,
                                                  float *__restrict__ scale) {
    const int l = threadIdx.x % L;
    const int64_t i = (int64_t)blockIdx.x * (quantize_block(L) / L) + threadIdx.x / L;
    if (i >= n) return;  // whole groups of L lanes
    const T *row = X + i * d;
    float v[2][8];
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int k = 8 * (L * u + l);
        if (k < d && d <= 16 * L) load8<true>(row, k, d, vec, v[u]);
        else if (k < d) load8<false>(row, k, d, vec, v[u]);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) v[u][e] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[u][e]) & 0x7fffffffu);
    }
    for (int k = 8 * (2 * L + l); k < d; k += 8 * L) {
        float x[8];
        load8<false>(row, k, d, vec, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
    }
#pragma unroll
    for (int o = std::min(L, 64) / 2; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    if constexpr (L > 64) {  // a row a block
        __shared__ uint32_t tops[L / 64];
        if (l % 64 == 0) tops[l / 64] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < L / 64; ++w) top = max(top, tops[w]);
    }
    const float a = __uint_as_float(top);
    const bool finite = top < 0x7f800000u;
    const float up = a < 0x1p-100f ? 0x1p64f : a > 0x1p100f ? 0x1p-64f : 1.f;
    const float inv = finite && top != 0 ? 1.f / (a * up) * 127.f : 0.f;
    int8_t *out = codes + i * ld;
    for (int u = 0; 8 * (L * u + l) < ld; ++u) {
        const int k = 8 * (L * u + l);
        float x[8];
        if (u < 2) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = u == 0 ? v[0][e] : v[1][e];
        } else {
            load8<false>(row, k, d, vec, x);
        }
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float c = finite ? __builtin_rintf(x[e] * up * inv) : 0.f;
            w[e >> 2] |= ((uint32_t)(int)fminf(fmaxf(c, -127.f), 127.f) & 255u) << (8 * (e & 3));
        }
        *reinterpret_cast<uint2 *>(out + k) = make_uint2(w[0], w[1]);
    }
    if (l == 0) scale[i] = finite ? a / 127.f : __builtin_nanf("");
}

// 16 bytes of values (4 f32 or 8 bf16) a thread at a time, so that a wave's
// store is 1 KB in a row; a block takes U x 256 pieces, all loads first.  From
// 2^21 pieces (32 MB of values) on U is 4 and the stores pass the caches by:
// quantise + dequantise of 262144 x 768 f32 took 339 us so, 361 with ordinary
// stores, 398 with U 1 (U 2 and 8: 361, 366).
template <typename T, int U>
__global__ __launch_bounds__(256) void k_dequantize(const int8_t *__restrict__ codes, int64_t ld,
                                                    const float *__restrict__ scale, int64_t n, int d, bool vec,
                                                    T *__restrict__ X) {
    constexpr int P = 16 / sizeof(T);
    const uint32_t np = (uint32_t)(d + P - 1) / P;
    const int64_t base = (int64_t)blockIdx.x * (256 * U), total = n * np;
    const int64_t row0 = base / np;
    const uint32_t rem = (uint32_t)(base - row0 * np);
    const uint32_t left = (uint32_t)min<int64_t>(256 * U, total - base);
    uint32_t q[U], c[U][2];
    int k[U];
    float s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t l = min(256 * u + threadIdx.x, left - 1), x = rem + l;
        q[u] = x / np;
        k[u] = P * (int)(x - q[u] * np);
        s[u] = scale[row0 + q[u]];
        __builtin_memcpy(c[u], codes + (row0 + q[u]) * ld + k[u], P);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (256 * u + threadIdx.x >= left) return;
        float v[P];
#pragma unroll
        for (int e = 0; e < P; ++e) v[e] = (float)(int8_t)(c[u][e >> 2] >> (8 * (e & 3))) * s[u];
        T *out = X + (row0 + q[u]) * d + k[u];
        if (vec && k[u] + P <= d) {
            mm::u32x4 y;
            if constexpr (P == 4)
                y = (mm::u32x4){__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
            else
                y = (mm::u32x4){mm::bf16_pair(v[0], v[1]), mm::bf16_pair(v[2], v[3]), mm::bf16_pair(v[4], v[5]),
                                mm::bf16_pair(v[6], v[7])};
            if constexpr (U > 1) __builtin_nontemporal_store(y, reinterpret_cast<mm::u32x4 *>(out));
            else *reinterpret_cast<mm::u32x4 *>(out) = y;
        } else {
#pragma unroll
            for (int e = 0; e < P; ++e)
                if (k[u] + e < d) {
                    if constexpr (P == 4) out[e] = v[e];
                    else out[e] = mm::bf16_bits(v[e]);
                }
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
    static constexpr int STORES = 4 * sizeof(T) * 2, STAGE = 16 * 272;
    const float *qs, *cs;
    T *Y;
    int64_t m, n;
    float q[4];
    int64_t i0_;
    bool counted;
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
    // 16 rows by 256 bytes at a time through LDS (272 bytes a row), so that a
    // store of the wave is 256 bytes of each of four rows; rows of Y on 16-byte
    // borders or not (a store may start anywhere).  4096 x 131072 x 768 takes 566 us
    // to bf16, 798 to f32.  On a card where it took 560: 605 with 128 bytes of each
    // of 8 rows, 830 with 64 of each of 16 (D of the softmax loss, whose row stride
    // is ours, takes the same time with all three); without any store 475, without
    // this whole step 337.
    __device__ __forceinline__ void tile(Shared &sh, char *stage, mm::i32x4 (&acc)[4][8], int64_t j0, int lane, int par) {
        constexpr int E = 16 / sizeof(T), PASS = sizeof(T) / 2;  // values of a piece; passes of 128 / PASS columns
        const int jl = 8 * (lane >> 4);
        const bool inside = i0_ + 64 <= m && j0 + 128 <= n;
        counted = inside;
        const float *c = &sh.cs[par][(int)(j0 & (mm::TILE - 1)) + jl];
        char *put = stage + (lane & 15) * 272 + jl * (int)sizeof(T);
        const char *get = stage + (lane >> 4) * 272 + 16 * (lane & 15);
        const int64_t row = i0_ + (lane >> 4), col = j0 + E * (lane & 15);
        T *to = Y + row * n + col;
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
            for (int p = 0; p < PASS; ++p) {
#pragma unroll
                for (int g2 = 0; g2 < 4 / PASS; ++g2) {
                    const int g = 2 * (g2 + p * (4 / PASS));
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = (float)acc[f][g + (e >> 2)][e & 3] * q[f] * c[16 * g + e];
                    uint4 *o = reinterpret_cast<uint4 *>(put + 32 * g2 * sizeof(T));
                    if constexpr (sizeof(T) == 4) {
                        o[0] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
                        o[1] = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
                    } else {
                        o[0] = make_uint4(mm::bf16_pair(x[0], x[1]), mm::bf16_pair(x[2], x[3]),
                                          mm::bf16_pair(x[4], x[5]), mm::bf16_pair(x[6], x[7]));
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const uint4 y = *reinterpret_cast<const uint4 *>(get + 4 * u * 272);
                    T *dst = to + (int64_t)(16 * f + 4 * u) * n + p * (128 / PASS);
                    if (inside) {
                        __builtin_memcpy(dst, &y, 16);
                    } else if (row + 16 * f + 4 * u < m) {
                        const int64_t left = n - col - p * (128 / PASS);
                        T e[E];
                        __builtin_memcpy(e, &y, 16);
#pragma unroll
                        for (int k = 0; k < E; ++k)
                            if (k < left) dst[k] = e[k];
                    }
                }
            }
    }
    __device__ __forceinline__ void finish(Shared &, int64_t, int, int) {}
};

// As ScoreEpi, for mm::k_few
template <typename T, int MF>
struct FewScoreEpi {
    const float *qs, *cs;
    T *Y;
    int64_t n;
    int m, q0_;
    float q[MF], c[4];
    __device__ __forceinline__ bool takes(int) const { return true; }
    __device__ __forceinline__ void init(int q0, int lane) {
        q0_ = q0;
#pragma unroll
        for (int f = 0; f < MF; ++f) q[f] = qs[min(q0 + 16 * f + (lane & 15), m - 1)];
    }
    __device__ __forceinline__ void fetch(int64_t j0, int lane) {
        const int64_t j = j0 + 4 * (lane >> 4);
#pragma unroll
        for (int r = 0; r < 4; ++r) c[r] = cs[min(j + r, n - 1)];
    }
    __device__ __forceinline__ void group(mm::i32x4 (&acc)[MF], int64_t j0, int lane) {
        const int64_t j = j0 + 4 * (lane >> 4);
#pragma unroll
        for (int f = 0; f < MF; ++f) {
            const int i = q0_ + 16 * f + (lane & 15);
            if (i >= m || j >= n) continue;
            mm::f32x4 x;
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = (float)acc[f][r] * q[f] * c[r];
            mm::store4<sizeof(T) == 4>(Y, i * n + j, (int)min<int64_t>(4, n - j), x);
        }
    }
    __device__ __forceinline__ void finish(char *, int, int) {}
};

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// lanes a row: the power of two that takes ld in one turn, 2 to 64, and a block
// of 128, 256 or 1024 for rows that do not fit a wave's registers (8 x 65536 f32:
// 62 us with a wave a row, 8.5 so; 65536 x 1536 bf16: 55 and 57)
template <typename T>
void quantize(const T *X, int64_t n, int d, int8_t *codes, int64_t ld, float *scale, hipStream_t s) {
    const bool vec = (d * sizeof(T)) % 16 == 0 && aligned16(X);
    auto go = [&](auto L) {
        constexpr int l = decltype(L)::value, block = quantize_block(l), per = block / l;
        for (int64_t i = 0, m; i < n; i += m) {
            m = std::min<int64_t>(n - i, mm::LAUNCH / l);
            hipLaunchKernelGGL((k_quantize<T, l>), dim3((unsigned)((m + per - 1) / per)), dim3(block), 0, s, X + i * d, m, d,
                               vec, codes + i * ld, ld, scale + i);
        }
    };
    if (ld <= 16) go(std::integral_constant<int, 2>());
    else if (ld <= 32) go(std::integral_constant<int, 4>());
    else if (ld <= 64) go(std::integral_constant<int, 8>());
    else if (ld <= 128) go(std::integral_constant<int, 16>());
    else if (ld <= 256) go(std::integral_constant<int, 32>());
    else if (ld <= 1024) go(std::integral_constant<int, 64>());
    else if (ld <= 2048) go(std::integral_constant<int, 128>());
    else if (ld <= 4096) go(std::integral_constant<int, 256>());
    else go(std::integral_constant<int, 1024>());
}

inline int padded(int d) { return (d + mm::KBY - 1) / mm::KBY * mm::KBY; }

// Up to 64 queries that fit LDS go to k_few, which needs no workspace; more where
// it is the faster by the time of both (mm::few_faster).
inline bool fits_few(mm::FewArgs &a, int64_t m, int d) {
    a.m = (int)m;
    a.qbytes = d;
    return m <= 64 && mm::plan_few(a, false);
}
inline bool few_args(mm::FewArgs &a, const mm::NtArgs &nt, int64_t m, int d) {
    return fits_few(a, m, d) || (mm::plan_few(a, true) && mm::few_faster(a, nt, 10));
}
inline size_t workspace(int64_t m, int d) {
    mm::FewArgs few = {};
    return d % mm::KBY == 0 || fits_few(few, m, d) ? 0 : (size_t)m * padded(d);
}

}  // namespace i8
}  // namespace mn

extern "C" int mn_quantize_rows_i8(const void *X, int32_t x_type, int64_t n, int32_t d,
                                   int8_t *codes, int64_t ld, float *scale, void *stream) {
    using namespace mn::i8;
    mn::clear_error();
    MN_REQUIRE(n >= 0 && d >= 1 && ld >= d && ld % 16 == 0 && ld <= INT_MAX - 16384, MN_EINVAL,
               "mn_quantize_rows_i8: n >= 0, d >= 1, ld >= d, a multiple of 16 and < 2^31 - 16384 needed");
    MN_REQUIRE(n < INT_MAX && n * ((d + 3) / 4) / 256 < INT_MAX && d < INT_MAX - 4096, MN_ENOTSUP,
               "mn_quantize_rows_i8: n < 2^31 - 1 rows and n d < 2^40 needed");
    MN_REQUIRE(x_type == MN_F32 || x_type == MN_BF16, MN_ENOTSUP, "mn_quantize_rows_i8: MN_F32 or MN_BF16");
    if (n == 0) return MN_OK;
    MN_REQUIRE(X && codes && scale, MN_EINVAL, "mn_quantize_rows_i8: NULL pointer");
    MN_REQUIRE(aligned16(codes), MN_EINVAL, "mn_quantize_rows_i8: codes not 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    if (x_type == MN_F32) quantize((const float *)X, n, d, codes, ld, scale, s);
    else quantize((const uint16_t *)X, n, d, codes, ld, scale, s);
    MN_KCHECK(s, "k_quantize");
    return MN_OK;
}

extern "C" int mn_dequantize_rows_i8(const int8_t *codes, int64_t ld, const float *scale, int64_t n,
                                     int32_t d, void *X, int32_t x_type, void *stream) {
    using namespace mn::i8;
    mn::clear_error();
    MN_REQUIRE(n >= 0 && d >= 1 && ld >= d && ld % 16 == 0 && ld <= INT_MAX - 16384, MN_EINVAL,
               "mn_dequantize_rows_i8: n >= 0, d >= 1, ld >= d, a multiple of 16 and < 2^31 - 16384 needed");
    MN_REQUIRE(n < INT_MAX && n * ((d + 3) / 4) / 256 < INT_MAX && d < INT_MAX - 4096, MN_ENOTSUP,
               "mn_dequantize_rows_i8: n < 2^31 - 1 rows and n d < 2^40 needed");
    MN_REQUIRE(x_type == MN_F32 || x_type == MN_BF16, MN_ENOTSUP, "mn_dequantize_rows_i8: MN_F32 or MN_BF16");
    if (n == 0) return MN_OK;
    MN_REQUIRE(X && codes && scale, MN_EINVAL, "mn_dequantize_rows_i8: NULL pointer");
    MN_REQUIRE(aligned16(codes), MN_EINVAL, "mn_dequantize_rows_i8: codes not 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    const int64_t row = x_type == MN_F32 ? (d + 3) / 4 : (d + 7) / 8, pieces = n * row;
    auto go = [&](auto U, auto *x) {
        typedef std::remove_pointer_t<decltype(x)> T;
        constexpr int u = decltype(U)::value;
        for (int64_t i = 0, m; i < n; i += m) {
            m = std::min<int64_t>(n - i, std::max<int64_t>(1, mn::mm::LAUNCH * u / row));
            hipLaunchKernelGGL((k_dequantize<T, u>), dim3((unsigned)((m * row + 256 * u - 1) / (256 * u))), dim3(256), 0, s,
                               codes + i * ld, ld, scale + i, m, d, (d * sizeof(T)) % 16 == 0 && aligned16(X), x + i * d);
        }
    };
    auto size = [&](auto *x) {
        if (pieces >= 1 << 21) go(std::integral_constant<int, 4>(), x);
        else go(std::integral_constant<int, 1>(), x);
    };
    if (x_type == MN_F32) size((float *)X);
    else size((uint16_t *)X);
    MN_KCHECK(s, "k_dequantize");
    return MN_OK;
}

extern "C" int mn_scores_i8_workspace(int64_t m, int32_t d, size_t *bytes) {
    mn::clear_error();
    MN_REQUIRE(bytes && m >= 0 && d >= 1 && d <= 131071, MN_EINVAL, "mn_scores_i8_workspace: bad args");
    *bytes = mn::i8::workspace(m, d);
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
    MN_REQUIRE(ldq <= 1 << 23 && ldc <= 1 << 23, MN_ENOTSUP,  // offsets in a tile of 256 rows are 32 bits
               "mn_scores_i8: row strides above 2^23 bytes");
    MN_REQUIRE(y_type == MN_F32 || y_type == MN_BF16, MN_ENOTSUP, "mn_scores_i8: MN_F32 or MN_BF16 scores");
    if (m == 0 || n == 0) return MN_OK;
    MN_REQUIRE(Q && q_scale && C && c_scale && Y, MN_EINVAL, "mn_scores_i8: NULL pointer");
    MN_REQUIRE(aligned16(Q) && aligned16(C), MN_EINVAL, "mn_scores_i8: codes not 16-byte aligned");
    const size_t need = workspace(m, d);
    MN_REQUIRE(need == 0 || (ws && ws_bytes >= need && aligned16(ws)), MN_ECAP,
               "mn_scores_i8: workspace of %zu bytes (16-byte aligned) needed", need);
    const int ldp = padded(d);
    hipStream_t s = (hipStream_t)stream;
    mm::NtArgs a = {};
    a.B = (const char *)C;
    a.ldb = ldc;
    a.m = m;
    a.n = n;
    a.nk = ldp / mm::KBY;
    a.bmax = (d + 15) / 16 * 16 - 16;
    mm::plan_runs(a);
    mm::FewArgs few = {};
    few.Q = (const char *)Q;
    few.B = (const char *)C;
    few.ldq = ldq;
    few.ldb = ldc;
    few.n = n;
    if (few_args(few, a, m, d)) {
        auto go = [&](auto out, auto MF) {
            typedef decltype(out) T;
            FewScoreEpi<T, decltype(MF)::value> epi = {};
            epi.qs = q_scale;
            epi.cs = c_scale;
            epi.Y = (T *)Y;
            epi.n = n;
            epi.m = (int)m;
            mm::launch_few<mm::Int8, decltype(MF)::value>(few, epi, s);
        };
        auto size = [&](auto out) {
            if (few.mf == 1) go(out, std::integral_constant<int, 1>());
            else if (few.mf == 2) go(out, std::integral_constant<int, 2>());
            else go(out, std::integral_constant<int, 4>());
        };
        if (y_type == MN_F32) size(float());
        else size(uint16_t());
        MN_KCHECK(s, "k_few");
        return MN_OK;
    }
    a.A = (const char *)Q;
    a.lda = ldq;
    if (need) {
        const unsigned grid = (unsigned)std::min<int64_t>((m * ldp + 255) / 256, 8192);
        hipLaunchKernelGGL(k_pad_codes, dim3(grid), dim3(256), 0, s, Q, ldq, m, d, ldp, (int8_t *)ws);
        MN_KCHECK(s, "k_pad_codes");
        a.A = (const char *)ws;
        a.lda = ldp;
    }
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

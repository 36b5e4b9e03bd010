// softmax.hip — softmax cross entropy of queries over the rows of an item
// table, and its gradients, in pieces of the table: no [t][v] matrix of logits
// is kept.
//
//     z_ij = scale q_i . c_j          t(i) = targets[i] (< 0: row i has no part)
//     rest_i = log sum_{j != t(i)} exp z_ij,   zt_i = z_i,t(i)
//     loss_i = log(1 + exp(rest_i - zt_i)),    lse_i = zt_i + loss_i
//     D_ij = g_i (exp(z_ij - lse_i) - [j = t(i)]),  D_i,t(i) = -g_i exp(rest_i - lse_i)
//     dQ = scale D C,   dC = scale D^T Q
//
// Keeping the target's logit out of the sum gives a loss near 0 (and 1 - p of
// the target) its full relative precision: as lse - z it would be the
// difference of two numbers near 10.  rest and zt of row ranges of the table
// join: rest by log-sum-exp, zt by maximum (-inf where the target is not).
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "common.hpp"
#include "mm_f32.hpp"

namespace mn {
namespace sm {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

// Per row for the gradients.  rel = g_i / max |g| (of the finite g), so that D =
// rel (p - [t]) is rounded to bf16 without the common factor; a g that is not
// finite gives NaN and leaves the other rows' factor alone.  dt = rel times the
// target's entry; resid = dt less its rounding (bf16 operands: added to dQ in f32
// and to dC in bf16, where a target's entry is the largest of its item: without it
// dC is off by 2.3e-3 of its norm and not the 1.66e-3 of its own rounding).
struct Row {
    float rel, lse2, dt, resid;
};

// A matrix [rows][d] on its way to rows of kp values, zero past d, whole k-steps.
// Rows whose target is < 0 become zeros, so that what they hold (a NaN, say)
// reaches no sum.  A thread takes 16 bytes at a time, all loads first.
struct Pack {
    const void *X;
    char *out;               // or NULL
    char *planes;            // or NULL: f32 as three planes of bf16 of rows * kp values
    const int64_t *targets;  // or NULL
    int64_t rows;
    int d, kp, per, blocks;  // per: pieces a thread, 1 or kPackPer
    bool vec;                // rows start on 16-byte borders
};
constexpr int kPackPer = 4;  // of a large matrix

template <bool F32, int U>
__device__ __forceinline__ void pack(const Pack &p, int block) {
    constexpr int E = F32 ? 4 : 8;  // values of a piece
    const uint32_t np = p.kp / E;
    const int64_t base = (int64_t)block * (256 * U), total = p.rows * np;
    const int64_t row0 = base / np;
    const uint32_t rem = (uint32_t)(base - row0 * np), left = (uint32_t)min<int64_t>(256 * U, total - base);
    mm::u32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t x = rem + min(256 * u + threadIdx.x, left - 1), q = x / np;
        const int c = E * (int)(x - q * np);
        const int64_t i = row0 + q;
        const bool has = !p.targets || p.targets[i] >= 0;
        if (p.vec && has && c + E <= p.d) {
            v[u] = *reinterpret_cast<const mm::u32x4 *>((const char *)p.X + (i * p.d + c) * (16 / E));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (F32) {
                    v[u][e] = has && c + e < p.d ? ((const uint32_t *)p.X)[i * p.d + c + e] : 0u;
                } else {
                    const uint16_t *src = (const uint16_t *)p.X + i * p.d + c + 2 * e;
                    const uint32_t lo = has && c + 2 * e < p.d ? src[0] : 0u, hi = has && c + 2 * e + 1 < p.d ? src[1] : 0u;
                    v[u][e] = lo | (hi << 16);
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t l = 256 * u + threadIdx.x;
        if (l >= left) return;
        if (p.out) *reinterpret_cast<mm::u32x4 *>(p.out + 16 * (base + l)) = v[u];
        if (F32 && p.planes) {
            uint2 s[3];
            mm::split4(v[u], s);
#pragma unroll
            for (int k = 0; k < 3; ++k) *reinterpret_cast<uint2 *>(p.planes + k * p.rows * p.kp * 2 + 8 * (base + l)) = s[k];
        }
    }
}

// As StatsEpi, for k_few: 16 items at a time, MF groups of 16 queries.
template <int MF>
struct FewStatsEpi {
    float2 *part;  // [slices][t]
    const int64_t *targets;
    int64_t c_offset, v;
    int t, q0_;
    float scale2;
    int at[MF];
    float m2[MF], sum[MF];
    __device__ __forceinline__ bool takes(int i) const { return targets[i] >= 0; }
    __device__ __forceinline__ void init(int q0, int lane) {
        q0_ = q0;
#pragma unroll
        for (int f = 0; f < MF; ++f) {
            const int i = q0 + 16 * f + (lane & 15);
            const int64_t x = i < t ? targets[i] : -1;
            at[f] = x >= c_offset && x - c_offset < v ? (int)(x - c_offset) : -1;
            m2[f] = -__builtin_inff();
            sum[f] = 0.f;
        }
    }
    __device__ __forceinline__ void fetch(int64_t, int) {}
    __device__ __forceinline__ void group(mm::f32x4 (&acc)[MF], int64_t j0, int lane) {
        const int j = (int)j0 + 4 * (lane >> 4);
#pragma unroll
        for (int f = 0; f < MF; ++f) {
            float z[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) z[r] = j + r >= v || j + r == at[f] ? -__builtin_inff() : acc[f][r];
            const float m = fmaxf(m2[f], fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])) * scale2);
            const float mz = m == -__builtin_inff() ? 0.f : m;
            float s = 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) s += __builtin_amdgcn_exp2f(__builtin_fmaf(z[r], scale2, -mz));
            sum[f] = sum[f] * __builtin_amdgcn_exp2f(m2[f] - mz) + s;
            m2[f] = m;
        }
    }
    // joined over the lanes, then over the block's waves
    __device__ __forceinline__ void finish(char *lds, int slice, int tid) {
        float2 *sh = reinterpret_cast<float2 *>(lds);
        const int lane = tid & 63, w = tid >> 6;
        auto join = [](float &m, float &s, float mo, float so) {
            const float x = fmaxf(m, mo), z = x == -__builtin_inff() ? 0.f : x;
            s = s * __builtin_amdgcn_exp2f(m - z) + so * __builtin_amdgcn_exp2f(mo - z);
            m = x;
        };
        __syncthreads();
#pragma unroll
        for (int f = 0; f < MF; ++f) {
#pragma unroll
            for (int o = 16; o <= 32; o <<= 1) {
                const float mo = __shfl_xor(m2[f], o), so = __shfl_xor(sum[f], o);
                join(m2[f], sum[f], mo, so);
            }
            if (lane < 16) sh[w * 16 * MF + 16 * f + lane] = make_float2(m2[f], sum[f]);
        }
        __syncthreads();
        if (tid < 16 * MF && q0_ + tid < t) {
            float2 x = sh[tid];
#pragma unroll
            for (int k = 1; k < mm::NT / 64; ++k) join(x.x, x.y, sh[k * 16 * MF + tid].x, sh[k * 16 * MF + tid].y);
            part[(int64_t)slice * t + q0_ + tid] = x;
        }
    }
};

// |g|, 0 where it is not finite; the factor that the rows are relative to
__device__ __forceinline__ float finite_abs(float g) { return fabsf(g) < __builtin_inff() ? fabsf(g) : 0.f; }
__device__ __forceinline__ float grad_top(float most) { return most > 0.f ? most : 1.f; }

__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))); }

// What the rows need before the products: forward the targets' logits (a wave
// a row: f32 sums of the d products); backward Row and the target within the
// rows of C here.
struct Rows {
    int64_t t, tp, v, c_offset;
    const int64_t *targets;
    const void *Q, *C;
    int d;
    float *zt_out;         // forward
    const float *rest, *zt;  // backward (rest not NULL)
    const float *grad, *grad_scale;
    int64_t grad_n;
    float scale;
    float *gs;             // [0] the factor of every gradient, [1] the largest finite |g| (grad_n > 1: of k_grad_max)
    Row *row;
    int32_t *at;
};

template <bool F32>
__device__ __forceinline__ void rows(const Rows &p, int block) {
    if (!p.rest) {
        const int lane = threadIdx.x & 63;
        const int64_t i = (int64_t)block * 4 + (threadIdx.x >> 6);
        if (i >= p.t) return;
        const int64_t at = p.targets[i] - p.c_offset;
        if (p.targets[i] < 0 || at < 0 || at >= p.v) {
            if (lane == 0) p.zt_out[i] = -__builtin_inff();
            return;
        }
        float z = 0.f;
        for (int k = lane; k < p.d; k += 64) {
            if constexpr (F32)
                z = __builtin_fmaf(((const float *)p.Q)[i * p.d + k], ((const float *)p.C)[at * p.d + k], z);
            else
                z = __builtin_fmaf(mm::bf16_value(((const uint16_t *)p.Q)[i * p.d + k]),
                                   mm::bf16_value(((const uint16_t *)p.C)[at * p.d + k]), z);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) z += __shfl_xor(z, o);
        if (lane == 0) p.zt_out[i] = z * p.scale;
        return;
    }
    const int64_t i = (int64_t)block * 256 + threadIdx.x;
    if (i >= p.tp) return;
    const float top = grad_top(p.grad_n == 1 ? finite_abs(p.grad[0]) : p.gs[1]);
    if (i == 0) p.gs[0] = (p.grad_scale ? top * p.grad_scale[0] : top) * p.scale;
    // no part (or only there to fill a tile, where the last query's logits of any
    // size are computed again): exp(z - inf) = 0
    Row r = {0.f, __builtin_inff(), 0.f, 0.f};
    int32_t a = -1;
    if (i < p.t && p.targets[i] >= 0) {
        const int64_t tl = p.targets[i] - p.c_offset;
        const float g = p.grad_n == 1 ? p.grad[0] : p.grad[i];
        const float inf = __builtin_inff();
        const float re = p.rest[i], z = p.zt[i];
        r.rel = fabsf(g) < inf ? g / top : __builtin_nanf("");
        const float lse = re == -inf ? z : z == -inf ? re : z + softplus(re - z);
        r.lse2 = lse * kLog2e;
        r.dt = re == -inf ? 0.f * r.rel : -r.rel / (1.f + expf(z - re));
        if (tl >= 0 && tl < p.v) {
            a = (int32_t)tl;
            if (!F32) r.resid = r.dt - mm::bf16_value(mm::bf16_bits(r.dt));
        }
    }
    p.row[i] = r;
    p.at[i] = a;
}

// One launch for all that comes before the products.
template <bool F32>
__global__ __launch_bounds__(256) void k_prep(Pack q, Pack c, Rows r) {
    int b = (int)blockIdx.x;
    if (b < q.blocks) return q.per == 1 ? pack<F32, 1>(q, b) : pack<F32, kPackPer>(q, b);
    b -= q.blocks;
    if (b < c.blocks) return c.per == 1 ? pack<F32, 1>(c, b) : pack<F32, kPackPer>(c, b);
    rows<F32>(r, b - c.blocks);
}

// Per lane and row the largest logit so far (m2, base 2, rounded: the number
// that every exponent is taken from) and the sum of exp of the rest, the
// target's left out; joined over the lanes and written per run of tiles and
// half of the columns.  An element costs a max, an fma, an exp and an add: 667 to
// 694 us for 4096 x 131072 x 768 in bf16, 618 without.
struct StatsEpi {
    struct Shared {};
    static constexpr bool FETCH = false;
    static constexpr int STORES = 0, STAGE = 0;
    static constexpr bool counted = false;
    float2 *part;
    const int64_t *targets;
    int64_t c_offset, t;
    int v;
    float scale2;  // scale log2(e)
    int at[4];
    float m2[4], sum[4];
    int64_t row0;
    __device__ __forceinline__ void init(Shared &, int64_t i0, int lane) {
        row0 = i0 + (lane & 15);
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const int64_t i = row0 + 16 * f, x = i < t ? targets[i] : -1;
            at[f] = x >= c_offset && x - c_offset < v ? (int)(x - c_offset) : -1;
            m2[f] = -__builtin_inff();
            sum[f] = 0.f;
        }
    }
    __device__ __forceinline__ void fetch(Shared &, int64_t, int, int) {}
    template <int G>
    __device__ __forceinline__ void tile(Shared &, mm::f32x4 (&acc)[4][G], int64_t j0, int lane) {
        const int jw = (int)j0, jl = jw + 8 * (lane >> 4);
        bool hit = jw + 16 * G > v;
#pragma unroll
        for (int f = 0; f < 4; ++f) hit = hit || (unsigned)(at[f] - jw) < 16u * G;
        if (__ballot(hit)) {
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int f = 0; f < 4; ++f) {
                        const int j = jl + 32 * (g >> 1) + 4 * (g & 1) + r;
                        acc[f][g][r] = j >= v || j == at[f] ? -__builtin_inff() : acc[f][g][r];
                    }
        }
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            float top = acc[f][0][0];
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, acc[f][g][r]);
            const float m = fmaxf(m2[f], top * scale2);
            const float mz = m == -__builtin_inff() ? 0.f : m;
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int g = 0; g < G; g += 2)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s0 += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[f][g][r], scale2, -mz));
                    s1 += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[f][g + 1][r], scale2, -mz));
                }
            sum[f] = sum[f] * __builtin_amdgcn_exp2f(m2[f] - mz) + (s0 + s1);
            m2[f] = m;
        }
    }
    __device__ __forceinline__ void finish(Shared &, int64_t, int piece, int lane) {
#pragma unroll
        for (int f = 0; f < 4; ++f) {
#pragma unroll
            for (int o = 16; o <= 32; o <<= 1) {
                const float mo = __shfl_xor(m2[f], o), so = __shfl_xor(sum[f], o);
                const float m = fmaxf(m2[f], mo), mz = m == -__builtin_inff() ? 0.f : m;
                sum[f] = sum[f] * __builtin_amdgcn_exp2f(m2[f] - mz) + so * __builtin_amdgcn_exp2f(mo - mz);
                m2[f] = m;
            }
            const int64_t i = row0 + 16 * f;
            if (lane < 16 && i < t) part[piece * t + i] = make_float2(m2[f], sum[f]);
        }
    }
};

// loss of a row from (rest, zt); -inf for zt: no target in any range (loss +inf)
__device__ __forceinline__ float row_loss(float rest, float zt) {
    if (zt != zt) return zt;
    if (rest == -__builtin_inff()) return zt == rest ? __builtin_inff() : 0.f;
    return zt == -__builtin_inff() ? __builtin_inff() : softplus(rest - zt);
}

// maximum, NaN if either is
__device__ __forceinline__ float fmax_nan(float x, float y) { return x != x || x > y ? x : y; }

template <class F>
__device__ __forceinline__ float block_fold(float x, float *sh, F f) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = f(x, __shfl_xor(x, o));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
    __syncthreads();
    x = sh[0];
    for (int w = 1; w < (int)blockDim.x / 64; ++w) x = f(x, sh[w]);
    __syncthreads();
    return x;
}

// The mean of the losses of the rows that take part and 1 / their number; no
// such row: 0 and 1.  One block and a fixed order.  (As the last act of k_join's
// last block it took 85 us longer at 4096 rows: every block's fence writes its
// L2 back.)
__global__ __launch_bounds__(1024) void k_mean(const float *__restrict__ loss, const int64_t *__restrict__ targets,
                                               int64_t t, float *__restrict__ mean, float *__restrict__ share) {
    __shared__ float sh[16];
    float sum = 0.f, num = 0.f;
    for (int64_t i = threadIdx.x; i < t; i += 1024) {
        const bool has = targets[i] >= 0;
        sum += has ? loss[i] : 0.f;
        num += has ? 1.f : 0.f;
    }
    auto add = [](float a, float b) { return a + b; };
    sum = block_fold(sum, sh, add);
    num = fmaxf(block_fold(num, sh, add), 1.f);
    if (threadIdx.x == 0) {
        *mean = sum / num;
        *share = 1.f / num;
    }
}

// One wave a row: joins n (maximum, sum) pairs (base 2), or with `rests` n
// values of rest and zt (the ranges of a table).
__global__ __launch_bounds__(256) void k_join(const float2 *__restrict__ part, const float *__restrict__ rests,
                                              const float *__restrict__ zts, int64_t n, int64_t t,
                                              const int64_t *__restrict__ targets, float *__restrict__ rest,
                                              float *__restrict__ zt, float *__restrict__ loss) {
    const int lane = threadIdx.x & 63;
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= t) return;
    float top = -__builtin_inff(), sum = 0.f, z = -__builtin_inff();
    for (int64_t k = lane; k < n; k += 64) {
        float2 p;
        if (part) {
            p = part[k * t + i];
        } else {
            const float r = rests[k * t + i];
            p = make_float2(r * kLog2e, r == -__builtin_inff() ? 0.f : r == r ? 1.f : r);
        }
        const float m = fmaxf(top, p.x);
        if (m != -__builtin_inff())
            sum = sum * __builtin_amdgcn_exp2f(top - m) + p.y * __builtin_amdgcn_exp2f(p.x - m);
        else
            sum += p.y;  // nothing yet, or a NaN
        top = m;
        if (zts) z = fmax_nan(z, zts[k * t + i]);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float m2 = __shfl_xor(top, o), s2 = __shfl_xor(sum, o);
        const float m = fmaxf(top, m2);
        if (m != -__builtin_inff())
            sum = sum * __builtin_amdgcn_exp2f(top - m) + s2 * __builtin_amdgcn_exp2f(m2 - m);
        else
            sum += s2;
        top = m;
        z = fmax_nan(z, __shfl_xor(z, o));
    }
    if (lane == 0) {
        const float r = sum == 0.f ? -__builtin_inff() : (top == -__builtin_inff() ? sum : (top + log2f(sum)) * kLn2);
        if (!zts) z = zt[i];
        else zt[i] = z;
        rest[i] = r;
        loss[i] = targets[i] < 0 ? 0.f : row_loss(r, z);
    }
}

// k_join and k_mean in one block of a thread a row, for few rows and pieces:
// a launch less (4 us of the host) where the rows are not what takes the time
__global__ __launch_bounds__(1024) void k_join_few(const float2 *__restrict__ part, int n, int t,
                                                   const int64_t *__restrict__ targets, float *__restrict__ rest,
                                                   const float *__restrict__ zt, float *__restrict__ loss,
                                                   float *__restrict__ mean, float *__restrict__ share) {
    __shared__ float sh[16];
    const int i = threadIdx.x;
    float l = 0.f, num = 0.f;
    if (i < t) {
        float top = -__builtin_inff(), sum = 0.f;
        for (int k0 = 0; k0 < n; k0 += 8) {
            float2 p[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) p[k] = k0 + k < n ? part[(k0 + k) * t + i] : make_float2(-__builtin_inff(), 0.f);
            float m = top;
#pragma unroll
            for (int k = 0; k < 8; ++k) m = fmaxf(m, p[k].x);
            const float mz = m == -__builtin_inff() ? 0.f : m;
            sum *= __builtin_amdgcn_exp2f(top - mz);
#pragma unroll
            for (int k = 0; k < 8; ++k) sum += p[k].y * __builtin_amdgcn_exp2f(p[k].x - mz);
            top = m;
        }
        const float r = sum == 0.f ? -__builtin_inff() : (top == -__builtin_inff() ? sum : (top + log2f(sum)) * kLn2);
        const bool has = targets[i] >= 0;
        l = has ? row_loss(r, zt[i]) : 0.f;
        num = has ? 1.f : 0.f;
        rest[i] = r;
        loss[i] = l;
    }
    if (!mean) return;
    auto add = [](float a, float b) { return a + b; };
    l = block_fold(l, sh, add);
    num = fmaxf(block_fold(num, sh, add), 1.f);
    if (i == 0) {
        *mean = l / num;
        *share = 1.f / num;
    }
}

// gs[1] = the largest finite |g| of the rows that take part
__global__ __launch_bounds__(1024) void k_grad_max(const float *__restrict__ grad, int64_t t,
                                                   const int64_t *__restrict__ targets, float *__restrict__ gs) {
    __shared__ float sh[16];
    float top = 0.f;
    for (int64_t i = threadIdx.x; i < t; i += 1024) top = fmaxf(top, targets[i] >= 0 ? finite_abs(grad[i]) : 0.f);
    top = block_fold(top, sh, [](float a, float b) { return fmaxf(a, b); });
    if (threadIdx.x == 0) gs[1] = top;
}

// D of a piece of the table, [tp][ldd], f32 or rounded to bf16; zeros in the
// rows and columns that only fill tiles.  4096 x 32768 x 768 in bf16 220 us, 158
// without this (the exp, and 268 MB to the last-level cache).
template <bool F32>
struct DlogitsEpi {
    struct Shared {};
    static constexpr bool FETCH = false;
    static constexpr int STORES = 16, STAGE = 0;  // (k_nt; k_nt32 counts nothing)
    static constexpr bool counted = true;
    char *D;
    int64_t ldd;
    int v;  // columns of this piece that exist
    const Row *row;
    const int32_t *at_;
    int64_t j_first;
    float scale2;
    int at[4];
    float rel[4], lse2[4], dt[4];
    int64_t i0_;
    __device__ __forceinline__ void init(Shared &, int64_t i0, int lane) {
        i0_ = i0;
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const int64_t i = i0_ + 16 * f + (lane & 15);
            const Row r = row[i];
            rel[f] = r.rel;
            lse2[f] = r.lse2;
            dt[f] = r.dt;
            const int64_t a = at_[i] - j_first;
            at[f] = at_[i] >= 0 && a >= 0 && a < v ? (int)a : -1;
        }
    }
    __device__ __forceinline__ void fetch(Shared &, int64_t, int, int) {}
    template <int G>
    __device__ __forceinline__ void tile(Shared &, mm::f32x4 (&acc)[4][G], int64_t j0, int lane) {
        constexpr int SZ = F32 ? 4 : 2;
        const int jw = (int)j0, jl = 8 * (lane >> 4);
        bool hit = jw + 16 * G > v;
#pragma unroll
        for (int f = 0; f < 4; ++f) hit = hit || (unsigned)(at[f] - jw) < 16u * G;
        const bool slow = __ballot(hit) != 0;
        char *base = D + SZ * (i0_ * ldd + j0);
        const int to = SZ * ((lane & 15) * (int)ldd + jl);
#pragma unroll
        for (int f = 0; f < 4; ++f) {
#pragma unroll
            for (int g = 0; g < G; g += 2) {
                float x[8];
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    x[q] = rel[f] * __builtin_amdgcn_exp2f(__builtin_fmaf(acc[f][g + (q >> 2)][q & 3], scale2, -lse2[f]));
                if (slow) {
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const int j = jw + jl + 16 * g + q;
                        const float y = j == at[f] ? dt[f] : x[q];
                        x[q] = j >= v ? 0.f : y;
                    }
                }
                const int off = to + SZ * (16 * f * (int)ldd + 16 * g);
                if constexpr (F32) {
                    mm::store16(base, off, make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                                                      __float_as_uint(x[3])));
                    mm::store16(base, off + 16, make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]),
                                                           __float_as_uint(x[6]), __float_as_uint(x[7])));
                } else {
                    mm::store16(base, off, make_uint4(mm::bf16_pair(x[0], x[1]), mm::bf16_pair(x[2], x[3]),
                                                      mm::bf16_pair(x[4], x[5]), mm::bf16_pair(x[6], x[7])));
                }
            }
        }
    }
    __device__ __forceinline__ void finish(Shared &, int64_t, int, int) {}
};

// partial sums of dQ: [splits][m][ld] f32 (ld a multiple of 4) of a piece of
// the table, or added to those of the pieces before
struct PartEpi {
    float *part;
    int64_t m, ld;
    bool first;
    template <int NF>
    __device__ __forceinline__ void operator()(mm::f32x4 (&acc)[4][NF], int64_t m0, int64_t n0, int lane, int z) const {
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const int64_t i = m0 + 16 * f + (lane & 15);
            if (i >= m) continue;
#pragma unroll
            for (int g = 0; g < NF; ++g) {
                const int64_t c = n0 + 16 * g + 4 * (lane >> 4);
                if (c >= ld) continue;
                mm::f32x4 *p = reinterpret_cast<mm::f32x4 *>(part + ((int64_t)z * m + i) * ld + c);
                *p = first ? acc[f][g] : *p + acc[f][g];
            }
        }
    }
};

// dC of a piece, or partial sums of it (part not NULL)
template <bool F32>
struct GradEpi {
    void *out;
    int64_t m, n;
    const float *gs;
    float *part;
    int64_t ld;
    template <int NF>
    __device__ __forceinline__ void operator()(mm::f32x4 (&acc)[4][NF], int64_t m0, int64_t n0, int lane, int z) const {
        if (part) {
            const PartEpi e = {part, m, ld, true};
            e(acc, m0, n0, lane, z);
            return;
        }
        const float s = gs[0];
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const int64_t i = m0 + 16 * f + (lane & 15);
            if (i >= m) continue;
#pragma unroll
            for (int g = 0; g < NF; ++g) {
                const int64_t c = n0 + 16 * g + 4 * (lane >> 4);
                if (c < n) mm::store4<F32>(out, i * n + c, (int)min<int64_t>(4, n - c), acc[f][g] * s);
            }
        }
    }
};

// Joins partial sums: out = factor (their sum + resid c_target), a thread 4
// columns; the second part only for dQ.
struct Sums {
    const float *part;       // [n][rows][ldp]
    int n, blocks;
    int64_t rows;
    void *out;
    const int64_t *targets;  // dQ: rows that have a part; NULL: dC
};
template <bool F32>
__device__ __forceinline__ void reduce(const Sums &p, int block, int ldp, int d, const uint16_t *C, const Row *row,
                                       const int32_t *at, const float *gs) {
    const uint32_t n4 = ldp / 4;
    const int64_t total = p.rows * n4, e = (int64_t)block * 256 + threadIdx.x;
    if (e >= total) return;
    const int64_t i = total <= 0xffffffffll ? (int64_t)((uint32_t)e / n4) : e / n4;
    const int c = 4 * (int)(e - i * n4);
    mm::f32x4 x = (mm::f32x4)(0.f);
    if (!p.targets || p.targets[i] >= 0) {
        const mm::f32x4 *src = reinterpret_cast<const mm::f32x4 *>(p.part) + e;
#pragma unroll 8
        for (int s = 0; s < p.n; ++s) x += src[s * total];
        if (!F32 && p.targets && at[i] >= 0) {
            const float r = row[i].resid;
            const uint16_t *y = C + (int64_t)at[i] * d + c;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (c + q < d) x[q] += r * mm::bf16_value(y[q]);
        }
        x *= gs[0];
    }
    mm::store4<F32>(p.out, i * d + c, min(4, d - c), x);
}
template <bool F32>
__global__ __launch_bounds__(256) void k_reduce(Sums dq, Sums dc, int first, int ldp, int d, const uint16_t *__restrict__ C,
                                                const Row *__restrict__ row, const int32_t *__restrict__ at,
                                                const float *__restrict__ gs) {
    const int b = first + (int)blockIdx.x;
    if (b < dq.blocks) reduce<F32>(dq, b, ldp, d, C, row, at, gs);
    else reduce<F32>(dc, b - dq.blocks, ldp, d, C, row, at, gs);
}

inline size_t up(size_t x) { return (x + 255) / 256 * 256; }
inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// Sizes of one call and where its workspace holds what.
struct Plan {
    int64_t t, v, tp;   // tp: t in whole tiles
    int d, kp, ldp;     // values of a packed row, of a row of dQ's partial sums
    int size;           // bytes of a value
    bool pack_c;        // C's rows start off 16-byte borders
    int64_t ldc;        // bytes of a row of C as the products read it
    int tile;           // items of a tile of logits
    mm::NtArgs nt;      // the whole table's logits
    mm::FewArgs few;    // the same for few queries; slices 0: not so
    bool few_q;         // on the queries as they are
    int64_t ldd;        // row stride of D
    int64_t vc, vmax;   // items per piece (backward), of the longest piece, in whole tiles
    int nf;             // 32 nf columns a tile of dQ and dC
    int splits;         // of dQ's sum over a piece
    int splits_c;       // of dC's sum over the queries
    int pieces, parts;  // of the table; partial sums of dQ in all
    bool apart;         // a piece's partial sums are its own
    size_t q, planes, c, part, row, at, gs, D, dq, dc, bytes;
};

inline Plan make_plan(int64_t t, int64_t v, int d, bool f32, bool backward) {
    Plan p = {};
    p.t = t;
    p.v = v;
    p.d = d;
    p.size = f32 ? 4 : 2;
    p.kp = (d + 31) / 32 * 32;
    p.ldp = (d + 3) / 4 * 4;
    p.pack_c = (d * p.size) % 16 != 0;
    p.ldc = (int64_t)(p.pack_c ? p.kp : d) * p.size;
    p.tp = (t + mm::TILE - 1) / mm::TILE * mm::TILE;
    p.tile = f32 ? mm::COLS32 : mm::TILE;
    p.nt.lda = (int64_t)p.kp * 2;
    p.nt.ldb = p.ldc;
    p.nt.m = t;
    p.nt.n = v;
    p.nt.nk = p.kp / 32;
    p.nt.bmax = (int)p.ldc - 16;
    size_t o = 0;
    auto take = [&](size_t b) { const size_t at = o; o += up(b); return at; };
    p.c = take(p.pack_c ? (size_t)v * p.kp * p.size : 0);
    if (!backward) {
        // few queries: items straight to registers
        p.few.m = (int)t;
        p.few.n = v;
        p.few_q = !p.pack_c;
        p.few.ldq = p.few.ldb = p.ldc;
        p.few.qbytes = (int)p.ldc;
        mm::plan_runs(p.nt, p.tile);
        if (!mm::plan_few(p.few, f32 || t > 64)) {
            p.few.slices = 0;
        } else if (t > 64 && !f32) {
            if (!mm::few_faster(p.few, p.nt, 7)) p.few.slices = 0;
        } else if (t > 64) {
            // where there are too few tiles for the processors, by the rate of
            // k_few's products (85 TFLOP/s) and the time of a step of k_nt32
            // (2.3 us, 256 blocks at a time), and 8 blocks a group
            // have a processor each: 192 queries on 3000 x 768 take 31 us so,
            // 58 by k_nt32, 1024 on 1500 x 2048 (64 groups) 155 and 138
            const double few_us = 16.0 * p.few.mf * p.few.groups * v * p.kp * 2 / 85e6;
            const double nt_us = 2.3 * p.nt.nk * p.nt.run * (((int64_t)p.nt.panels * p.nt.slices + 255) / 256);
            if (p.few.groups > 32 || few_us > 0.8 * nt_us) p.few.slices = 0;
        }
        const bool few = p.few.slices > 0;
        p.q = take(few ? (p.few_q ? 0 : (size_t)t * p.kp * p.size) : f32 ? 0 : (size_t)t * p.kp * 2);
        p.planes = take(f32 && !few ? (size_t)t * p.kp * 6 : 0);
        p.part = take((size_t)std::max(p.nt.slices * 2, p.few.slices) * t * 8);
    } else {
        p.q = take((size_t)t * p.kp * p.size);
        p.planes = take(f32 ? (size_t)t * p.kp * 6 : 0);
        // Pieces whose D stays below 256 MB (the last-level cache; 128, 512 and
        // 1024 MB take 3.22, 3.05 and 3.06 ms for 4096 x 131072 x 768, 256 MB
        // 3.05) and whose tiles fill whole rounds of 256 blocks; a short
        // rest joins the last piece where it fits.
        const int64_t all = (v + mm::TILE - 1) / mm::TILE, panels = p.tp / mm::TILE;
        const int64_t most = std::max<int64_t>(1, std::min<int64_t>(4096, ((int64_t)256 << 20) / (p.tp * mm::TILE * p.size)));
        const int64_t unit = std::max<int64_t>(1, 256 / panels);
        const int64_t piece = most >= unit ? most / unit * unit : most;
        const int64_t rest = all % piece;
        int64_t longest = std::min(piece, all);
        if (all > piece && rest > 0 && piece + rest <= most) longest = piece + rest;
        p.vc = std::min(piece, all) * mm::TILE;
        p.vmax = longest * mm::TILE;
        // The runs of k of both products: the cuts with the least time for
        // their blocks on 256 processors, dQ's first, in steps: a block that
        // writes partial sums costs its run and 20 (256 KB to memory), one that
        // writes dC itself 10 (f32, whose steps take longer: 6 and 4).  Free
        // processors take the next block: dC's done by a time are counted from
        // the two times at which dQ's blocks end.  dC's sum over the queries is
        // only cut where its tiles do not fill the processors (3630 queries,
        // 1384 x 64 items: 214 us without, 47 with in f32, 70 and 39 in bf16).
        p.nf = f32 ? (d > 64 ? 4 : 2) : d > 128 ? 8 : d > 64 ? 4 : 2;
        const int64_t cols = (d + 32 * p.nf - 1) / (32 * p.nf), tiles = panels * cols, sum = f32 ? 6 : 20;
        const int64_t steps = p.vc / 32, steps_c = (t + 31) / 32, nc1 = p.vc / mm::TILE * cols;
        int64_t best = INT64_MAX;
        for (int64_t sc = 1; sc == 1 || (sc * nc1 <= 256 && sc * 4 <= steps_c); sc *= 2) {
            const int64_t nc = sc * nc1, b = (steps_c + sc - 1) / sc + (sc > 1 ? sum : f32 ? 4 : 10);
            for (int64_t s = 1; s <= std::min<int64_t>(steps / 4 + 1, std::max<int64_t>(1, 512 / tiles)); ++s) {
                const int64_t a = (steps + s - 1) / s + sum, nq = tiles * s, full = nq / 256 * a, more = nq % 256;
                int64_t end = full + (more ? a : 0);
                for (int64_t k = (nc + 255) / 256;; ++k) {
                    const int64_t e1 = full + k * b, e2 = std::max<int64_t>(0, e1 - full - a) / b;
                    if ((256 - more) * k + more * e2 >= nc) {
                        end = std::max(end, e1);
                        break;
                    }
                }
                if (end < best) {
                    best = end;
                    p.splits = (int)s;
                    p.splits_c = (int)sc;
                }
            }
        }
        // every piece's partial sums apart (written once, read once) while
        // they stay below 256 MB, else added up
        p.pieces = 1;
        for (int64_t j = 0; v - j > p.vmax; j += p.vc) ++p.pieces;
        p.apart = (int64_t)p.pieces * p.splits * t * p.ldp * 4 <= ((int64_t)256 << 20);
        p.parts = p.apart ? p.pieces * p.splits : p.splits;
        p.row = take(sizeof(Row) * p.tp);
        p.at = take(4 * p.tp);
        p.gs = take(8);
        p.ldd = p.vmax + 128 / p.size;  // an odd number of 128-byte lines: rows on different memory channels
        p.D = take((size_t)p.tp * p.ldd * p.size);
        p.dq = take((size_t)p.parts * t * p.ldp * 4);
        p.dc = take(p.splits_c > 1 ? (size_t)p.splits_c * p.vmax * p.ldp * 4 : 0);
    }
    p.bytes = o;
    return p;
}

template <bool F32>
int prep(const Plan &p, const void *Q, const void *C, const int64_t *targets, char *w, const Rows &r, int64_t row_blocks,
         hipStream_t s) {
    // f32 queries: planes for the logits, as they are for k_few and for dC
    const bool few = p.few.slices > 0, planes = F32 && !few;
    auto one = [&](const void *X, char *out, char *pl, int64_t n, const int64_t *tg) {
        const int64_t pieces = n * (p.kp * p.size / 16);
        const int per = pieces >= kPackPer * 256 * 1024 ? kPackPer : 1;
        const int blocks = (int)((pieces + 256 * per - 1) / (256 * per));
        return Pack{X, out, pl, tg, n, p.d, p.kp, per, blocks, !p.pack_c};
    };
    const Pack q = few && p.few_q ? Pack{} : one(Q, planes && !r.rest ? nullptr : w + p.q, planes ? w + p.planes : nullptr, p.t, targets);
    const Pack c = p.pack_c ? one(C, w + p.c, nullptr, p.v, nullptr) : Pack{};
    hipLaunchKernelGGL(k_prep<F32>, dim3((unsigned)(q.blocks + c.blocks + row_blocks)), dim3(256), 0, s, q, c, r);
    MN_KCHECK(s, "k_prep");
    return MN_OK;
}

static mm::NtArgs nt_args(const Plan &p, const void *C, char *ws) {
    mm::NtArgs a = p.nt;
    a.A = ws + (p.size == 4 ? p.planes : p.q);
    a.B = p.pack_c ? ws + p.c : (const char *)C;
    return a;
}

template <bool F32, class EPI>
void launch_nt(const mm::NtArgs &a, const EPI &epi, hipStream_t s) {
    const dim3 grid((unsigned)(a.panels * a.slices));
    if constexpr (F32) hipLaunchKernelGGL((mm::k_nt32<EPI>), grid, dim3(mm::NT), 0, s, a, a.m * a.lda, epi);
    else hipLaunchKernelGGL((mm::k_nt<mm::Bf16, EPI>), grid, dim3(mm::NT), 0, s, a, epi);
}

template <bool F32>
int stats_impl(const void *Q, const void *C, int64_t t, int64_t v, int32_t d, const int64_t *targets, int64_t c_offset,
               float scale, float *rest, float *zt, float *loss, float *mean, float *share, void *ws, hipStream_t s) {
    const Plan p = make_plan(t, v, d, F32, false);
    char *w = (char *)ws;
    Rows r = {};
    r.t = t;
    r.v = v;
    r.c_offset = c_offset;
    r.targets = targets;
    r.Q = Q;
    r.C = C;
    r.d = d;
    r.zt_out = zt;
    r.scale = scale;
    const int rc = prep<F32>(p, Q, C, targets, w, r, (t + 3) / 4, s);
    if (rc != MN_OK) return rc;
    float2 *part = (float2 *)(w + p.part);
    int64_t pieces;
    if (p.few.slices) {
        mm::FewArgs a = p.few;
        a.Q = p.few_q ? (const char *)Q : w + p.q;
        a.B = p.pack_c ? w + p.c : (const char *)C;
        pieces = a.slices;
        auto go = [&](auto MF) {
            FewStatsEpi<decltype(MF)::value> epi = {};
            epi.part = part;
            epi.targets = targets;
            epi.c_offset = c_offset;
            epi.v = v;
            epi.t = (int)t;
            epi.scale2 = scale * kLog2e;
            mm::launch_few<std::conditional_t<F32, mm::F32, mm::Bf16>, decltype(MF)::value>(a, epi, s);
        };
        if (a.mf == 1) go(std::integral_constant<int, 1>());
        else if (a.mf == 2) go(std::integral_constant<int, 2>());
        else go(std::integral_constant<int, 4>());
        MN_KCHECK(s, "k_few");
    } else {
        const mm::NtArgs a = nt_args(p, C, w);
        pieces = (int64_t)a.slices * 2;
        StatsEpi epi = {};
        epi.part = part;
        epi.targets = targets;
        epi.c_offset = c_offset;
        epi.t = t;
        epi.v = (int)v;
        epi.scale2 = scale * kLog2e;
        launch_nt<F32>(a, epi, s);
        MN_KCHECK(s, "k_nt");
    }
    if (t <= 1024 && pieces <= 64) {
        hipLaunchKernelGGL(k_join_few, dim3(1), dim3(1024), 0, s, part, (int)pieces, (int)t, targets, rest, zt, loss, mean,
                           share);
        MN_KCHECK(s, "k_join_few");
        return MN_OK;
    }
    hipLaunchKernelGGL(k_join, dim3((unsigned)((t + 3) / 4)), dim3(256), 0, s, part, (const float *)nullptr,
                       (const float *)nullptr, pieces, t, targets, rest, zt, loss);
    MN_KCHECK(s, "k_join");
    if (mean) {
        hipLaunchKernelGGL(k_mean, dim3(1), dim3(1024), 0, s, loss, targets, t, mean, share);
        MN_KCHECK(s, "k_mean");
    }
    return MN_OK;
}

template <bool F32>
int backward_impl(const void *Q, const void *C, int64_t t, int64_t v, int32_t d, const int64_t *targets,
                  int64_t c_offset, float scale, const float *rest, const float *zt, const float *grad,
                  int64_t grad_n, const float *grad_scale, void *dQ, void *dC, void *ws, hipStream_t s) {
    const Plan p = make_plan(t, v, d, F32, true);
    char *w = (char *)ws;
    float *gs = (float *)(w + p.gs);
    Row *row = (Row *)(w + p.row);
    int32_t *at = (int32_t *)(w + p.at);
    if (grad_n != 1) {
        hipLaunchKernelGGL(k_grad_max, dim3(1), dim3(1024), 0, s, grad, t, targets, gs);
        MN_KCHECK(s, "k_grad_max");
    }
    Rows r = {};
    r.t = t;
    r.tp = p.tp;
    r.v = v;
    r.c_offset = c_offset;
    r.targets = targets;
    r.rest = rest;
    r.zt = zt;
    r.grad = grad;
    r.grad_scale = grad_scale;
    r.grad_n = grad_n;
    r.scale = scale;
    r.gs = gs;
    r.row = row;
    r.at = at;
    const int rc = prep<F32>(p, Q, C, targets, w, r, p.tp / 256, s);
    if (rc != MN_OK) return rc;
    const char *Cp = p.pack_c ? w + p.c : (const char *)C;
    const int row_tiles = (int)(p.tp / mm::TILE), col_tiles = (d + 32 * p.nf - 1) / (32 * p.nf);
    int64_t vn = 0;
    int piece = 0;
    for (int64_t j0 = 0; j0 < v; j0 += vn, ++piece) {
        vn = v - j0 <= p.vmax ? v - j0 : p.vc;  // items of this piece
        mm::NtArgs a = nt_args(p, C, w);
        a.B += j0 * a.ldb;
        a.n = vn;
        mm::plan_runs(a, p.tile);
        DlogitsEpi<F32> epi = {};
        epi.D = w + p.D;
        epi.ldd = p.ldd;
        epi.v = (int)vn;
        epi.row = row;
        epi.at_ = at;
        epi.j_first = j0;
        epi.scale2 = scale * kLog2e;
        launch_nt<F32>(a, epi, s);
        MN_KCHECK(s, "k_nt");
        mm::KnArgs g = {};
        g.A = w + p.D;
        g.lda = p.size * p.ldd;
        mm::KnArgs gq = g, gc = g;
        gq.ldb = p.ldc;
        gq.B = Cp + j0 * p.ldc;
        gq.k = vn;
        gq.steps_all = (int)((vn + 31) / 32);
        gq.steps = (gq.steps_all + p.splits - 1) / p.splits;
        gc.ldb = (int64_t)p.kp * p.size;
        gc.B = w + p.q;
        gc.k = t;
        gc.steps_all = (int)((t + 31) / 32);
        gc.steps = (gc.steps_all + p.splits_c - 1) / p.splits_c;
        const mm::KnGrid nq = {dQ ? col_tiles : 0, row_tiles, p.splits};
        const mm::KnGrid nc = {dC ? col_tiles : 0, (int)((vn + mm::TILE - 1) / mm::TILE), p.splits_c};
        const PartEpi pe = {(float *)(w + p.dq) + (p.apart ? (int64_t)piece * p.splits * t * p.ldp : 0), t, p.ldp,
                            p.apart || piece == 0};
        char *out = (char *)dC + j0 * d * (F32 ? 4 : 2);
        const GradEpi<F32> ge = {out, vn, d, gs, p.splits_c > 1 ? (float *)(w + p.dc) : nullptr, p.ldp};
        [[maybe_unused]] const mm::KnExtra extra = {at, &row->resid, (int)(sizeof(Row) / sizeof(float)), j0};
        auto go = [&](auto NF) {
            constexpr int n = decltype(NF)::value;
            const dim3 grid((unsigned)(nq.blocks() + nc.blocks()));
            if constexpr (F32)
                hipLaunchKernelGGL((mm::k_kn2_32<n, PartEpi, GradEpi<F32>>), grid, dim3(mm::NT), 0, s, gq, pe, nq, gc, ge, nc);
            else
                hipLaunchKernelGGL((mm::k_kn2<n, PartEpi, GradEpi<F32>>), grid, dim3(mm::NT), 0, s, gq, pe, nq, gc, ge, nc,
                                   extra);
        };
        if (p.nf == 4) go(std::integral_constant<int, 4>());
        else if (p.nf == 2) go(std::integral_constant<int, 2>());
        else if constexpr (!F32) go(std::integral_constant<int, 8>());
        MN_KCHECK(s, "k_kn2");
        const bool last = j0 + vn >= v;
        auto sums = [&](size_t part, int n, int64_t rows, void *to, const int64_t *tg) {
            return Sums{(const float *)(w + part), n, (int)((rows * (p.ldp / 4) + 255) / 256), rows, to, tg};
        };
        const Sums sq = dQ && last ? sums(p.dq, p.parts, t, dQ, targets) : Sums{};
        const Sums sd = dC && p.splits_c > 1 ? sums(p.dc, p.splits_c, vn, out, nullptr) : Sums{};
        for (int b = 0, n; b < sq.blocks + sd.blocks; b += n) {
            n = (int)std::min<int64_t>(sq.blocks + sd.blocks - b, mm::LAUNCH / 256);
            hipLaunchKernelGGL(k_reduce<F32>, dim3((unsigned)n), dim3(256), 0, s, sq, sd, b, p.ldp, d, (const uint16_t *)C, row,
                               at, gs);
            MN_KCHECK(s, "k_reduce");
        }
    }
    return MN_OK;
}

// what every entry point checks
static int check_args(const char *who, int32_t x_type, int64_t t, int64_t v, int32_t d, float scale) {
    MN_REQUIRE(t >= 0 && v >= 1 && d >= 1, MN_EINVAL, "%s: t >= 0, v >= 1, d >= 1 needed", who);
    MN_REQUIRE(x_type == MN_F32 || x_type == MN_BF16, MN_ENOTSUP, "%s: MN_F32 or MN_BF16", who);
    MN_REQUIRE(std::isfinite(scale) && scale > 0.f, MN_EINVAL, "%s: scale has to be positive and finite", who);
    MN_REQUIRE(t <= (1 << 24) && v < INT_MAX - 1024 && d <= 65536, MN_ENOTSUP,
               "%s: t <= 2^24, v < 2^31 - 1025, d <= 65536", who);
    MN_REQUIRE(v * ((d + 31) / 32) / 512 < (1 << 30), MN_ENOTSUP, "%s: v d too large for one call", who);
    MN_REQUIRE((t + 255) / 256 * ((v + 255) / 256) < (1 << 30), MN_ENOTSUP, "%s: t v too large for one call", who);
    // what k_prep copies, 64 bytes a thread: 2^31 of them and a wave for each of t rows
    const int64_t size = x_type == MN_F32 ? 4 : 2, copied = t + (d * size % 16 ? v : 0);
    MN_REQUIRE(copied * ((d + 31) / 32 * 32) * size <= (int64_t)1 << 37, MN_ENOTSUP,
               "%s: more than 128 GB of queries and of items whose rows start off 16-byte borders", who);
    return MN_OK;
}

}  // namespace sm
}  // namespace mn

extern "C" int mn_softmax_workspace(int64_t t, int64_t v, int32_t d, int32_t x_type, int32_t backward,
                                    size_t *bytes) {
    using namespace mn::sm;
    mn::clear_error();
    MN_REQUIRE(bytes, MN_EINVAL, "mn_softmax_workspace: NULL pointer");
    const int rc = check_args("mn_softmax_workspace", x_type, t, v, d, 1.f);
    if (rc != MN_OK) return rc;
    *bytes = t == 0 ? 0 : make_plan(t, v, d, x_type == MN_F32, backward != 0).bytes;
    return MN_OK;
}

extern "C" int mn_softmax_stats(const void *Q, const void *C, int32_t x_type, int64_t t, int64_t v, int32_t d,
                                const int64_t *targets, int64_t c_offset, float scale, float *rest, float *zt,
                                float *loss, float *mean, float *share, void *ws, size_t ws_bytes, void *stream) {
    using namespace mn::sm;
    mn::clear_error();
    const int rc = check_args("mn_softmax_stats", x_type, t, v, d, scale);
    if (rc != MN_OK) return rc;
    MN_REQUIRE(c_offset >= 0, MN_EINVAL, "mn_softmax_stats: c_offset >= 0 needed");
    MN_REQUIRE(!mean || share, MN_EINVAL, "mn_softmax_stats: mean without share");
    hipStream_t s = (hipStream_t)stream;
    if (t == 0) {
        if (mean) {
            hipLaunchKernelGGL(k_mean, dim3(1), dim3(1024), 0, s, loss, targets, t, mean, share);
            MN_KCHECK(s, "k_mean");
        }
        return MN_OK;
    }
    MN_REQUIRE(Q && C && targets && rest && zt && loss, MN_EINVAL, "mn_softmax_stats: NULL pointer");
    MN_REQUIRE(aligned16(Q) && aligned16(C), MN_EINVAL, "mn_softmax_stats: Q or C not 16-byte aligned");
    const size_t need = make_plan(t, v, d, x_type == MN_F32, false).bytes;
    MN_REQUIRE(ws && ws_bytes >= need && aligned16(ws), MN_ECAP,
               "mn_softmax_stats: workspace of %zu bytes (16-byte aligned) needed", need);
    return x_type == MN_F32 ? stats_impl<true>(Q, C, t, v, d, targets, c_offset, scale, rest, zt, loss, mean, share, ws, s)
                            : stats_impl<false>(Q, C, t, v, d, targets, c_offset, scale, rest, zt, loss, mean, share, ws, s);
}

extern "C" int mn_softmax_merge(const float *rests, const float *zts, int64_t parts, int64_t t,
                                const int64_t *targets, float *rest, float *zt, float *loss, float *mean,
                                float *share, void *stream) {
    using namespace mn::sm;
    mn::clear_error();
    MN_REQUIRE(parts >= 1 && t >= 0 && t <= (1 << 24), MN_EINVAL, "mn_softmax_merge: parts >= 1, 0 <= t <= 2^24 needed");
    MN_REQUIRE(t == 0 || (rests && zts && targets && rest && zt && loss), MN_EINVAL, "mn_softmax_merge: NULL pointer");
    MN_REQUIRE(!mean || share, MN_EINVAL, "mn_softmax_merge: mean without share");
    hipStream_t s = (hipStream_t)stream;
    if (t > 0) {
        hipLaunchKernelGGL(k_join, dim3((unsigned)((t + 3) / 4)), dim3(256), 0, s, (const float2 *)nullptr, rests, zts,
                           parts, t, targets, rest, zt, loss);
        MN_KCHECK(s, "k_join");
    }
    if (mean) {
        hipLaunchKernelGGL(k_mean, dim3(1), dim3(1024), 0, s, loss, targets, t, mean, share);
        MN_KCHECK(s, "k_mean");
    }
    return MN_OK;
}

extern "C" int mn_softmax_backward(const void *Q, const void *C, int32_t x_type, int64_t t, int64_t v, int32_t d,
                                   const int64_t *targets, int64_t c_offset, float scale, const float *rest,
                                   const float *zt, const float *grad, int64_t grad_n, const float *grad_scale,
                                   void *dQ, void *dC, void *ws, size_t ws_bytes, void *stream) {
    using namespace mn::sm;
    mn::clear_error();
    const int rc = check_args("mn_softmax_backward", x_type, t, v, d, scale);
    if (rc != MN_OK) return rc;
    MN_REQUIRE(c_offset >= 0, MN_EINVAL, "mn_softmax_backward: c_offset >= 0 needed");
    MN_REQUIRE(grad_n == 1 || grad_n == t, MN_EINVAL, "mn_softmax_backward: grad_n has to be 1 or t");
    MN_REQUIRE(t >= 1, MN_EINVAL, "mn_softmax_backward: t >= 1 needed");
    MN_REQUIRE(Q && C && targets && rest && zt && grad, MN_EINVAL, "mn_softmax_backward: NULL pointer");
    MN_REQUIRE(dQ || dC, MN_EINVAL, "mn_softmax_backward: no gradient asked for");
    MN_REQUIRE(aligned16(Q) && aligned16(C), MN_EINVAL, "mn_softmax_backward: Q or C not 16-byte aligned");
    const bool f32 = x_type == MN_F32;
    const size_t need = make_plan(t, v, d, f32, true).bytes;
    MN_REQUIRE(ws && ws_bytes >= need && aligned16(ws), MN_ECAP,
               "mn_softmax_backward: workspace of %zu bytes (16-byte aligned) needed", need);
    hipStream_t s = (hipStream_t)stream;
    return f32 ? backward_impl<true>(Q, C, t, v, d, targets, c_offset, scale, rest, zt, grad, grad_n, grad_scale, dQ,
                                     dC, ws, s)
               : backward_impl<false>(Q, C, t, v, d, targets, c_offset, scale, rest, zt, grad, grad_n, grad_scale, dQ,
                                      dC, ws, s);
}

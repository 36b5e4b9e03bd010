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

#include "common.hpp"
#include "mm_tiles.hpp"

namespace mn {
namespace sm {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

// Per row for the gradients.  rel = g_i / max |g|, so that D = rel (p - [t])
// is rounded to bf16 without the common factor; dt = rel times the target's
// entry; resid = dt less its rounding (bf16 operands: added to dQ in f32).
struct Row {
    float rel, lse2, dt, resid;
};

// [rows][d] to `P` planes of [rows][kp] bf16, zero past d; rows whose target
// is < 0 become zeros, so that what they hold (a NaN, say) reaches no sum.
template <bool F32>
__global__ __launch_bounds__(256) void k_pack(const void *__restrict__ X, int64_t rows, int d, int kp,
                                              const int64_t *__restrict__ targets,
                                              uint16_t *__restrict__ out) {
    const int64_t total = rows * kp, stride = (int64_t)gridDim.x * 256;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += stride) {
        const int64_t i = e / kp;
        const int k = (int)(e - i * kp);
        const bool has = k < d && (!targets || targets[i] >= 0);
        if constexpr (F32) {
            uint16_t p[3];
            mm::split3(has ? ((const float *)X)[i * d + k] : 0.f, p);
#pragma unroll
            for (int q = 0; q < 3; ++q) out[q * total + e] = p[q];
        } else {
            out[e] = has ? ((const uint16_t *)X)[i * d + k] : (uint16_t)0;
        }
    }
}

// Per lane and row the largest logit so far (m2, base 2, rounded: the number
// that every exponent is taken from) and the sum of exp of the rest, the
// target's left out; joined over the lanes and written per run of tiles and
// half of the columns.  An element costs a max, an fma, an exp and an add: for
// 768 columns of operands about a seventh of its time on the matrix pipe.
struct StatsEpi {
    struct Shared {};
    static constexpr bool FETCH = false;
    float2 *part;
    float *zt;
    const int64_t *targets;
    int64_t c_offset, t;
    int v;
    float scale, scale2;  // scale2 = scale log2(e)
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
    __device__ __forceinline__ void tile(Shared &, mm::f32x4 (&acc)[4][8], int64_t j0, int lane, int) {
        const int jw = (int)j0, jl = jw + 8 * (lane >> 4);
        bool hit = jw + 128 > v;
#pragma unroll
        for (int f = 0; f < 4; ++f) hit = hit || (unsigned)(at[f] - jw) < 128u;
        if (__ballot(hit)) {
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                float z = 0.f;
                bool mine = false;
#pragma unroll
                for (int g = 0; g < 8; ++g)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int j = jl + 32 * (g >> 1) + 4 * (g & 1) + r;
                        z = j == at[f] ? acc[f][g][r] : z;
                        mine = mine || j == at[f];
                        acc[f][g][r] = j >= v || j == at[f] ? -__builtin_inff() : acc[f][g][r];
                    }
                if (mine) zt[row0 + 16 * f] = z * scale;
            }
        }
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            float top = acc[f][0][0];
#pragma unroll
            for (int g = 0; g < 8; ++g)
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, acc[f][g][r]);
            const float m = fmaxf(m2[f], top * scale2);
            const float mz = m == -__builtin_inff() ? 0.f : m;
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int g = 0; g < 8; g += 2)
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

__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))); }

// loss of a row from (rest, zt); -inf for zt: no target in any range (loss +inf)
__device__ __forceinline__ float row_loss(float rest, float zt) {
    if (rest == -__builtin_inff()) return zt == rest ? __builtin_inff() : 0.f;
    return zt == -__builtin_inff() ? __builtin_inff() : softplus(rest - zt);
}

// one wave a row: joins n (maximum, sum) pairs (base 2), or with `rests` n
// values of rest and zt (the ranges of a table)
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
        if (zts) z = fmaxf(z, zts[k * t + i]);
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
        z = fmaxf(z, __shfl_xor(z, o));
    }
    if (lane == 0) {
        const float r = sum == 0.f ? -__builtin_inff() : (top == -__builtin_inff() ? sum : (top + log2f(sum)) * kLn2);
        if (!zts) z = zt[i];
        else zt[i] = z;
        rest[i] = r;
        if (loss) loss[i] = targets[i] < 0 ? 0.f : row_loss(r, z);
    }
}

__global__ __launch_bounds__(256) void k_fill(float *__restrict__ p, int64_t n, float v) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = v;
}

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

// out = (mean of the losses of the rows that take part, 1 / their number);
// no such row: (0, 1).  One block: the order of the sum is fixed.
__global__ __launch_bounds__(1024) void k_mean(const float *__restrict__ loss, const int64_t *__restrict__ targets,
                                               int64_t t, float *__restrict__ out) {
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
        out[0] = sum / num;
        out[1] = 1.f / num;
    }
}

// gs[0] = the factor of every gradient (scale, max |g|, *grad_scale), gs[1] = max |g|
__global__ __launch_bounds__(1024) void k_grad_scale(const float *__restrict__ grad, int64_t grad_n,
                                                     const float *__restrict__ grad_scale,
                                                     const int64_t *__restrict__ targets, float scale,
                                                     float *__restrict__ gs) {
    __shared__ float sh[16];
    float top = 0.f;
    if (grad_n == 1) {
        top = fabsf(grad[0]);
    } else {
        for (int64_t i = threadIdx.x; i < grad_n; i += 1024)
            top = fmaxf(top, targets[i] >= 0 ? fabsf(grad[i]) : 0.f);
        top = block_fold(top, sh, [](float a, float b) { return fmaxf(a, b); });
    }
    if (threadIdx.x == 0) {
        gs[0] = (grad_scale ? top * grad_scale[0] : top) * scale;
        gs[1] = top;
    }
}

__global__ __launch_bounds__(256) void k_rows(const float *__restrict__ rest, const float *__restrict__ zt,
                                              const int64_t *__restrict__ targets, int64_t c_offset, int64_t t,
                                              int64_t tp, int64_t v, const float *__restrict__ grad, int64_t grad_n,
                                              const float *__restrict__ gs, bool f32, Row *__restrict__ row,
                                              int32_t *__restrict__ at) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= tp) return;
    Row r = {0.f, 0.f, 0.f, 0.f};
    int32_t a = -1;
    if (i < t && targets[i] >= 0) {
        const int64_t tl = targets[i] - c_offset;
        const float top = gs[1], g = grad_n == 1 ? grad[0] : grad[i];
        const float inf = __builtin_inff();
        const float re = rest[i], z = zt[i];
        r.rel = top == 0.f ? 0.f : g / top;
        const float lse = re == -inf ? z : z == -inf ? re : z + softplus(re - z);
        r.lse2 = lse * kLog2e;
        r.dt = re == -inf ? 0.f : -r.rel / (1.f + expf(z - re));
        if (tl >= 0 && tl < v) {
            a = (int32_t)tl;
            if (!f32) r.resid = r.dt - mm::bf16_value(mm::bf16_bits(r.dt));
        }
    }
    row[i] = r;
    at[i] = a;
}

// D of a piece of the table, [tp][ldd] (three planes for f32 operands); zeros
// in the rows and columns that only fill tiles.
template <int PLANES>
struct DlogitsEpi {
    struct Shared {};
    static constexpr bool FETCH = false;
    uint16_t *D;
    int64_t ldd, plane;
    int v;  // columns of this piece that exist
    const Row *row;
    const int32_t *at_;
    int64_t j_first;
    float scale2;
    int at[4];
    float rel[4], lse2[4], dt[4];
    bool any;
    int64_t i0_;
    __device__ __forceinline__ void init(Shared &, int64_t i0, int lane) {
        any = false;
        i0_ = i0;
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const int64_t i = i0 + 16 * f + (lane & 15);
            const Row r = row[i];
            rel[f] = r.rel;
            lse2[f] = r.lse2;
            dt[f] = r.dt;
            const int64_t a = at_[i] - j_first;
            at[f] = at_[i] >= 0 && a >= 0 && a < v ? (int)a : -1;
            any = any || r.rel != 0.f;
        }
        any = __ballot(any) != 0;
    }
    __device__ __forceinline__ void fetch(Shared &, int64_t, int, int) {}
    __device__ __forceinline__ void tile(Shared &, mm::f32x4 (&acc)[4][8], int64_t j0, int lane, int) {
        const int jw = (int)j0, jl = 8 * (lane >> 4);
        bool hit = jw + 128 > v || !any;
#pragma unroll
        for (int f = 0; f < 4; ++f) hit = hit || (unsigned)(at[f] - jw) < 128u;
        const bool slow = __ballot(hit) != 0;
        uint16_t *base = D + i0_ * ldd + j0;
        const int lrow = (lane & 15) * (int)ldd + jl;
#pragma unroll
        for (int f = 0; f < 4; ++f) {
#pragma unroll
            for (int g = 0; g < 8; g += 2) {
                float x[8];
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    x[q] = rel[f] * __builtin_amdgcn_exp2f(__builtin_fmaf(acc[f][g + (q >> 2)][q & 3], scale2, -lse2[f]));
                if (slow) {
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const int j = jw + jl + 16 * g + q;
                        if (j == at[f]) x[q] = dt[f];
                        if (j >= v || !any) x[q] = 0.f;
                    }
                }
                uint16_t *p = base + (int64_t)16 * f * ldd + (lrow + 16 * g);
                if constexpr (PLANES == 1) {
                    *reinterpret_cast<uint4 *>(p) = make_uint4(mm::bf16_pair(x[0], x[1]), mm::bf16_pair(x[2], x[3]),
                                                               mm::bf16_pair(x[4], x[5]), mm::bf16_pair(x[6], x[7]));
                } else {
                    uint32_t o[3][4];
#pragma unroll
                    for (int q = 0; q < 8; q += 2) {
                        uint16_t a[3], b[3];
                        mm::split3(x[q], a);
                        mm::split3(x[q + 1], b);
#pragma unroll
                        for (int s = 0; s < 3; ++s) o[s][q / 2] = (uint32_t)a[s] | ((uint32_t)b[s] << 16);
                    }
#pragma unroll
                    for (int s = 0; s < 3; ++s)
                        *reinterpret_cast<uint4 *>(p + s * plane) = make_uint4(o[s][0], o[s][1], o[s][2], o[s][3]);
                }
            }
        }
    }
    __device__ __forceinline__ void finish(Shared &, int64_t, int, int) {}
};

// partial sums of dQ: [splits][m][ld] f32 (ld a multiple of 4), added up over
// the pieces of the table
struct PartEpi {
    float *part;
    int64_t m, ld;
    bool first;
    __device__ __forceinline__ void operator()(mm::f32x4 (&acc)[4][8], int64_t m0, int64_t n0, int lane, int z) const {
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const int64_t i = m0 + 16 * f + (lane & 15);
            if (i >= m) continue;
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                const int64_t c = n0 + 16 * g + 4 * (lane >> 4);
                if (c >= ld) continue;
                mm::f32x4 *p = reinterpret_cast<mm::f32x4 *>(part + ((int64_t)z * m + i) * ld + c);
                *p = first ? acc[f][g] : *p + acc[f][g];
            }
        }
    }
};

template <bool F32>
struct GradEpi {
    void *out;
    int64_t m, n;
    const float *gs;
    __device__ __forceinline__ void operator()(mm::f32x4 (&acc)[4][8], int64_t m0, int64_t n0, int lane, int) const {
        const float s = gs[0];
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const int64_t i = m0 + 16 * f + (lane & 15);
            if (i >= m) continue;
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                const int64_t c = n0 + 16 * g + 4 * (lane >> 4);
                const mm::f32x4 x = acc[f][g] * s;
                if constexpr (F32) {
                    float *p = (float *)out + i * n + c;
                    if (c + 4 <= n) {
                        __builtin_memcpy(p, &x, 16);
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            if (c + q < n) p[q] = x[q];
                    }
                } else {
                    uint16_t *p = (uint16_t *)out + i * n + c;
                    if (c + 4 <= n) {
                        const uint2 y = make_uint2(mm::bf16_pair(x[0], x[1]), mm::bf16_pair(x[2], x[3]));
                        __builtin_memcpy(p, &y, 8);
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            if (c + q < n) p[q] = mm::bf16_bits(x[q]);
                    }
                }
            }
        }
    }
};

// dQ = factor (sum of the partials + resid c_target)
template <bool F32>
__global__ __launch_bounds__(256) void k_reduce_dq(const float *__restrict__ part, int splits, int ldp, int64_t t, int d,
                                                   const uint16_t *__restrict__ C, const Row *__restrict__ row,
                                                   const int32_t *__restrict__ at,
                                                   const int64_t *__restrict__ targets,
                                                   const float *__restrict__ gs, void *__restrict__ dQ) {
    const int64_t total = t * d, stride = (int64_t)gridDim.x * 256;
    const float s = gs[0];
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += stride) {
        const int64_t i = e / d;
        float x = 0.f;
        if (targets[i] >= 0) {
            for (int p = 0; p < splits; ++p) x += part[(p * t + i) * ldp + (e - i * d)];
            if (!F32 && at[i] >= 0)
                x += row[i].resid * mm::bf16_value(C[(int64_t)at[i] * d + (e - i * d)]);
            x *= s;
        }
        if constexpr (F32) ((float *)dQ)[e] = x;
        else ((uint16_t *)dQ)[e] = mm::bf16_bits(x);
    }
}

inline size_t up(size_t x) { return (x + 255) / 256 * 256; }
inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
inline unsigned grid1(int64_t n, int per, int64_t most = 1 << 20) {
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>((n + per - 1) / per, most));
}

// Sizes of one call and where its workspace holds what.
struct Plan {
    int64_t t, v, tp;   // tp: t in whole tiles
    int d, kp, ldp, planes;
    bool pack_c;
    mm::NtArgs nt;      // the whole table's logits: how its tiles are cut
    int64_t vc;         // items per piece (backward), in whole tiles
    int splits;         // of dQ's sum over a piece
    size_t q, c, part, row, at, gs, D, dq, bytes;
};

inline Plan make_plan(int64_t t, int64_t v, int d, bool f32, bool backward) {
    Plan p = {};
    p.t = t;
    p.v = v;
    p.d = d;
    p.kp = (d + 31) / 32 * 32;
    p.ldp = (d + 3) / 4 * 4;
    p.planes = f32 ? 3 : 1;
    p.pack_c = f32 || p.kp != d;
    p.tp = (t + mm::TILE - 1) / mm::TILE * mm::TILE;
    p.nt.lda = p.nt.ldb = p.kp * 2;
    p.nt.planeA = t * p.kp * 2;
    p.nt.planeB = v * p.kp * 2;
    p.nt.m = t;
    p.nt.n = v;
    p.nt.nk = p.kp / 32;
    p.nt.nseg = f32 ? 6 : 1;
    p.nt.bmax = p.kp * 2 - 16;
    size_t o = 0;
    auto take = [&](size_t b) { const size_t at = o; o += up(b); return at; };
    p.q = take((size_t)p.planes * t * p.kp * 2);
    p.c = take(p.pack_c ? (size_t)p.planes * v * p.kp * 2 : 0);
    if (!backward) {
        mm::plan_runs(p.nt);
        p.part = take((size_t)p.nt.slices * 2 * t * 8);
    } else {
        // pieces of equal size whose D (read twice after it is written) stays
        // below 192 MB, most of the last-level cache
        const int64_t all = (v + mm::TILE - 1) / mm::TILE;
        const int64_t most = std::max<int64_t>(1, std::min<int64_t>(4096, ((int64_t)192 << 20) / (p.tp * mm::TILE * 2 * p.planes)));
        const int64_t pieces = (all + most - 1) / most;
        p.vc = (all + pieces - 1) / pieces * mm::TILE;
        const int64_t tiles = p.tp / mm::TILE * ((d + mm::TILE - 1) / mm::TILE);
        p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(256 / tiles, p.vc / mm::TILE));
        p.row = take(sizeof(Row) * p.tp);
        p.at = take(4 * p.tp);
        p.gs = take(8);
        p.D = take((size_t)p.planes * p.tp * p.vc * 2);
        p.dq = take((size_t)p.splits * t * p.ldp * 4);
    }
    p.bytes = o;
    return p;
}

template <bool F32>
int pack(const void *X, int64_t rows, int d, int kp, const int64_t *targets, void *out, hipStream_t s) {
    hipLaunchKernelGGL(k_pack<F32>, dim3(grid1(rows * kp, 256, 65536)), dim3(256), 0, s, X, rows, d, kp, targets,
                       (uint16_t *)out);
    MN_KCHECK(s, "k_pack");
    return MN_OK;
}

static int operands(const Plan &p, const void *Q, const void *C, bool f32, const int64_t *zero_rows, char *ws,
                    hipStream_t s) {
    int rc = f32 ? pack<true>(Q, p.t, p.d, p.kp, zero_rows, ws + p.q, s)
                 : pack<false>(Q, p.t, p.d, p.kp, zero_rows, ws + p.q, s);
    if (rc == MN_OK && p.pack_c)
        rc = f32 ? pack<true>(C, p.v, p.d, p.kp, nullptr, ws + p.c, s)
                 : pack<false>(C, p.v, p.d, p.kp, nullptr, ws + p.c, s);
    return rc;
}

static mm::NtArgs nt_args(const Plan &p, const void *C, char *ws) {
    mm::NtArgs a = p.nt;
    a.A = ws + p.q;
    a.B = p.pack_c ? ws + p.c : (const char *)C;
    return a;
}

static int stats_impl(const void *Q, const void *C, int32_t x_type, int64_t t, int64_t v, int32_t d,
                      const int64_t *targets, int64_t c_offset, float scale, float *rest, float *zt, float *loss,
                      float *mean, void *ws, hipStream_t s) {
    const bool f32 = x_type == MN_F32;
    const Plan p = make_plan(t, v, d, f32, false);
    char *w = (char *)ws;
    const int rc = operands(p, Q, C, f32, nullptr, w, s);
    if (rc != MN_OK) return rc;
    hipLaunchKernelGGL(k_fill, dim3(grid1(t, 256)), dim3(256), 0, s, zt, t, -__builtin_inff());
    MN_KCHECK(s, "k_fill");
    const mm::NtArgs a = nt_args(p, C, w);
    StatsEpi epi = {};
    epi.part = (float2 *)(w + p.part);
    epi.zt = zt;
    epi.targets = targets;
    epi.c_offset = c_offset;
    epi.t = t;
    epi.v = (int)v;
    epi.scale = scale;
    epi.scale2 = scale * kLog2e;
    hipLaunchKernelGGL((mm::k_nt<mm::Bf16, StatsEpi>), dim3((unsigned)(a.panels * a.slices)), dim3(mm::NT), 0, s, a, epi);
    MN_KCHECK(s, "k_nt");
    hipLaunchKernelGGL(k_join, dim3((unsigned)((t + 3) / 4)), dim3(256), 0, s, epi.part, (const float *)nullptr,
                       (const float *)nullptr, (int64_t)a.slices * 2, t, targets, rest, zt, loss);
    MN_KCHECK(s, "k_join");
    if (mean) {
        hipLaunchKernelGGL(k_mean, dim3(1), dim3(1024), 0, s, loss, targets, t, mean);
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
    const int rc = operands(p, Q, C, F32, targets, w, s);
    if (rc != MN_OK) return rc;
    float *gs = (float *)(w + p.gs);
    Row *row = (Row *)(w + p.row);
    int32_t *at = (int32_t *)(w + p.at);
    hipLaunchKernelGGL(k_grad_scale, dim3(1), dim3(1024), 0, s, grad, grad_n, grad_scale, targets, scale, gs);
    MN_KCHECK(s, "k_grad_scale");
    hipLaunchKernelGGL(k_rows, dim3(grid1(p.tp, 256)), dim3(256), 0, s, rest, zt, targets, c_offset, t, p.tp, v, grad,
                       grad_n, gs, F32, row, at);
    MN_KCHECK(s, "k_rows");
    constexpr int PL = F32 ? 3 : 1;
    const char *Cp = p.pack_c ? w + p.c : (const char *)C;
    const int row_tiles = (int)(p.tp / mm::TILE), col_tiles = (d + mm::TILE - 1) / mm::TILE;
    for (int64_t j0 = 0; j0 < v; j0 += p.vc) {
        const int64_t vn = std::min(p.vc, v - j0);           // items of this piece
        mm::NtArgs a = nt_args(p, C, w);
        a.B += j0 * a.ldb;
        a.n = vn;
        mm::plan_runs(a);
        DlogitsEpi<PL> epi = {};
        epi.D = (uint16_t *)(w + p.D);
        epi.ldd = p.vc;
        epi.plane = p.tp * p.vc;
        epi.v = (int)vn;
        epi.row = row;
        epi.at_ = at;
        epi.j_first = j0;
        epi.scale2 = scale * kLog2e;
        hipLaunchKernelGGL((mm::k_nt<mm::Bf16, DlogitsEpi<PL>>), dim3((unsigned)(a.panels * a.slices)), dim3(mm::NT), 0, s,
                           a, epi);
        MN_KCHECK(s, "k_nt");
        mm::KnArgs g = {};
        g.A = w + p.D;
        g.lda = 2 * p.vc;
        g.ldb = 2 * p.kp;
        g.planeA = 2 * p.tp * p.vc;
        g.nseg = F32 ? 6 : 1;
        if (dQ) {
            g.B = Cp + j0 * g.ldb;
            g.planeB = v * g.ldb;
            g.k = vn;
            g.steps_all = (int)((vn + 31) / 32);
            g.steps = (g.steps_all + p.splits - 1) / p.splits;
            PartEpi pe = {(float *)(w + p.dq), t, p.ldp, j0 == 0};
            hipLaunchKernelGGL((mm::k_kn<false, PartEpi>), dim3(col_tiles, row_tiles, p.splits), dim3(mm::NT), 0, s, g, pe);
            MN_KCHECK(s, "k_kn");
        }
        if (dC) {
            g.B = w + p.q;
            g.planeB = t * g.ldb;
            g.k = t;
            g.steps_all = g.steps = (int)((t + 31) / 32);
            GradEpi<F32> ge = {(char *)dC + j0 * d * (F32 ? 4 : 2), vn, d, gs};
            hipLaunchKernelGGL((mm::k_kn<true, GradEpi<F32>>), dim3(col_tiles, (unsigned)((vn + mm::TILE - 1) / mm::TILE), 1),
                               dim3(mm::NT), 0, s, g, ge);
            MN_KCHECK(s, "k_kn");
        }
    }
    if (dQ) {
        hipLaunchKernelGGL(k_reduce_dq<F32>, dim3(grid1(t * d, 256, 65536)), dim3(256), 0, s, (const float *)(w + p.dq),
                           p.splits, p.ldp, t, d, (const uint16_t *)C, row, at, targets, gs, dQ);
        MN_KCHECK(s, "k_reduce_dq");
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
    MN_REQUIRE((t + 255) / 256 * ((v + 255) / 256) < (1 << 30), MN_ENOTSUP, "%s: t v too large for one call", who);
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
                                float *loss, float *mean, void *ws, size_t ws_bytes, void *stream) {
    using namespace mn::sm;
    mn::clear_error();
    const int rc = check_args("mn_softmax_stats", x_type, t, v, d, scale);
    if (rc != MN_OK) return rc;
    MN_REQUIRE(c_offset >= 0, MN_EINVAL, "mn_softmax_stats: c_offset >= 0 needed");
    hipStream_t s = (hipStream_t)stream;
    if (t == 0) {
        if (mean) {
            hipLaunchKernelGGL(k_mean, dim3(1), dim3(1024), 0, s, loss, targets, t, mean);
            MN_KCHECK(s, "k_mean");
        }
        return MN_OK;
    }
    MN_REQUIRE(Q && C && targets && rest && zt, MN_EINVAL, "mn_softmax_stats: NULL pointer");
    MN_REQUIRE(!mean || loss, MN_EINVAL, "mn_softmax_stats: the mean needs loss");
    MN_REQUIRE(aligned16(Q) && aligned16(C), MN_EINVAL, "mn_softmax_stats: Q or C not 16-byte aligned");
    const size_t need = make_plan(t, v, d, x_type == MN_F32, false).bytes;
    MN_REQUIRE(ws && ws_bytes >= need && aligned16(ws), MN_ECAP,
               "mn_softmax_stats: workspace of %zu bytes (16-byte aligned) needed", need);
    return stats_impl(Q, C, x_type, t, v, d, targets, c_offset, scale, rest, zt, loss, mean, ws, s);
}

extern "C" int mn_softmax_merge(const float *rests, const float *zts, int64_t parts, int64_t t,
                                const int64_t *targets, float *rest, float *zt, float *loss, float *mean,
                                void *stream) {
    using namespace mn::sm;
    mn::clear_error();
    MN_REQUIRE(parts >= 1 && t >= 0 && t <= (1 << 24), MN_EINVAL, "mn_softmax_merge: parts >= 1, 0 <= t <= 2^24 needed");
    MN_REQUIRE(t == 0 || (rests && zts && targets && rest && zt), MN_EINVAL, "mn_softmax_merge: NULL pointer");
    MN_REQUIRE(!mean || loss || t == 0, MN_EINVAL, "mn_softmax_merge: the mean needs loss");
    hipStream_t s = (hipStream_t)stream;
    if (t > 0) {
        hipLaunchKernelGGL(k_join, dim3((unsigned)((t + 3) / 4)), dim3(256), 0, s, (const float2 *)nullptr, rests, zts,
                           parts, t, targets, rest, zt, loss);
        MN_KCHECK(s, "k_join");
    }
    if (mean) {
        hipLaunchKernelGGL(k_mean, dim3(1), dim3(1024), 0, s, loss, targets, t, mean);
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

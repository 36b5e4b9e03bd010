// mm_f32.hpp — the products of mm_tiles.hpp for f32 operands, on the bf16
// matrix cores.
//
// x = h + m + l, 8 + 8 + 8 significant bits cut off one after the other (exact
// but for subnormal tails), and a product is six bf16 products, mm, lh, hl, mh,
// hm, hh; what is left out (ml, lm, ll) is below 2^-23 |x||y| and mostly far
// below: the size of an f32 product's rounding.  Six at the bf16 rate are 2.7
// times the f32 matrix rate.
//
// A block has a tile of 256 x 128 (or 64 columns), eight waves of 64 x 64 = 4 x
// 4 tiles of 16 x 16.  A step is 32 k's.  Each thread loads 24 values of a step
// to registers, two steps ahead, splits them (44 vector instructions for 8
// values) and writes three times 8 bf16 to LDS: every value is split once, and a
// matrix with k in its rows is turned on the way (a thread's 8 values are 8 k's
// of one column).  LDS holds the three planes of two steps, 144 KB.
//
// Waves w and w + 4 share a SIMD and run one barrier window apart: while one
// issues its 96 matrix instructions, the other reads its 24 fragments, splits
// and writes its part of the next step and starts the loads of the third.  A
// plane buffer is written in the windows after those in which both halves have
// read it (lgkmcnt(0) before every barrier).
//
// 1024 x 100000 x 768: logits with the loss's sums 770 us (1.22 PFLOP/s of bf16
// products, 204 TFLOP/s of f32 ones; the f32 matrix rate of a large library
// product is 154), the gradients' two products 770 us for 65536 rows and their
// rest.  Bound by the window of the half that reads, splits and writes: it takes
// longer than the other half's 96 matrix instructions (53% of the matrix pipe);
// without loads, splits, writes or five of the six products each 20% less.
// Splitting between the matrix instructions instead spills registers.
//
// LDS rows: 64 bytes (32 k's of a plane), piece c of row r at c ^ f(r's quad),
// f = 0, 2, 3, 1: writes of 16 rows and reads of a fragment (16 rows by 4
// pieces) are free of bank conflicts.  A quad is 4 rows of a fragment's 16.
#pragma once
#include "mm_tiles.hpp"

namespace mn {
namespace mm {

constexpr int COLS32 = 128;                     // columns of a tile of k_nt32
constexpr int PLANE = (TILE + COLS32) * KBY;    // a plane of a step, 24 KB

struct alignas(1024) Planes {
    char b[2][3][PLANE];  // [step & 1][h, m, l][rows of i, rows of j]
};

__device__ __forceinline__ int quad_swizzle(int a) { return ((a & 1) << 1) ^ ((a >> 1) & 1) * 3; }

// 8 values to three times 8 bf16: the upper halves of x, x - h, x - h - m
__device__ __forceinline__ void split8(const float (&v)[8], u32x4 (&s)[3]) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        auto upper = [](float u, float w) __attribute__((always_inline)) {  // w's, u's upper halves
            return __builtin_amdgcn_perm(__float_as_uint(w), __float_as_uint(u), 0x07060302u);
        };
        auto rest = [](float u) __attribute__((always_inline)) {
            return u - __uint_as_float(__float_as_uint(u) & 0xffff0000u);
        };
        const float x = v[2 * p], y = v[2 * p + 1], x1 = rest(x), y1 = rest(y);
        s[0][p] = upper(x, y);
        s[1][p] = upper(x1, y1);
        s[2][p] = upper(rest(x1), rest(y1));
    }
}

// 8 values of a row of k: two 16-byte pieces
__device__ __forceinline__ void load_row(float (&v)[8], const char *base, uint32_t lo, uint32_t hi) {
    const f32x4 a = *reinterpret_cast<const f32x4 *>(base + lo), b = *reinterpret_cast<const f32x4 *>(base + hi);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
}
// 8 values of a column: rows k0 .. k0 + 7, at most `last`
__device__ __forceinline__ void load_col(float (&v)[8], const char *base, uint32_t col, int k0, uint32_t ld, int last) {
    if (last >= 31) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = *reinterpret_cast<const float *>(base + e * (uint64_t)ld + (k0 * ld + col));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = *reinterpret_cast<const float *>(base + (min(k0 + e, last) * ld + col));
    }
}

// The loop of both kernels.  load(set): the next step's values (a thread's
// pieces: two of i, one of j); put[k]: where in a plane piece k goes; start(n):
// before step n (a tile's end, zeroed accumulators), false ends the loop.
template <int NJ, class LOAD, class START>
__device__ __forceinline__ void steps32(Planes &pl, f32x4 (&acc)[4][NJ], int nstep, const int (&put)[3], bool j_half,
                                        int ri, int rj, int jstep0, int jstep1, LOAD load, START start) {
    const int wj = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    float v[2][3][8];
    auto write = [&](float (&x)[3][8], int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            if (k == 2 && !j_half) break;
            u32x4 s[3];
            split8(x[k], s);
#pragma unroll
            for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x4 *>(&pl.b[buf][p][put[k]]) = s[p];
        }
    };
    auto lds_end = []() __attribute__((always_inline)) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        window_end();
    };
    if (nstep == 0) {
        start(0);
        return;
    }
    load(v[0]);
    if (nstep > 1) load(v[1]);
    write(v[0], 0);
    if (nstep > 2) load(v[0]);
    lds_end();
    if (wj) window_end();
    u32x4 fi[4][3], fj[NJ][3];
    auto step = [&](int n, int buf, float (&x)[3][8]) __attribute__((always_inline)) {
        const char *b = &pl.b[buf][0][0];
#pragma unroll
        for (int p = 0; p < 3; ++p) {
#pragma unroll
            for (int f = 0; f < 4; ++f) fi[f][p] = *reinterpret_cast<const u32x4 *>(b + p * PLANE + ri + 16 * f * KBY);
#pragma unroll
            for (int g = 0; g < NJ; ++g)
                fj[g][p] = *reinterpret_cast<const u32x4 *>(b + p * PLANE + rj + (g >> 1) * jstep1 + (g & 1) * jstep0);
        }
        if (n + 1 < nstep) write(x, buf ^ 1);
        if (n + 3 < nstep) load(x);
        lds_end();
        constexpr int PI[6] = {1, 0, 2, 0, 1, 0}, PJ[6] = {1, 2, 0, 1, 0, 0};  // smallest first
#pragma unroll
        for (int q = 0; q < 6; ++q)
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int g = 0; g < NJ; ++g) acc[f][g] = Bf16::mma(fj[g][PJ[q]], fi[f][PI[q]], acc[f][g]);
        window_end();
    };
    for (int n = 0;; n += 2) {
        if (!start(n)) break;
        step(n, 0, v[1]);
        if (!start(n + 1)) break;
        step(n + 1, 1, v[0]);
    }
    if (!wj) window_end();  // the other half's last products
}

// k_nt of f32: a tile has 128 rows of B; nk counts steps of 32 k's, bmax is the
// last 16-byte piece of a row of B.  Accumulators as k_nt's, a wave's 64 columns.
template <class EPI>
__global__ __launch_bounds__(NT, 2) void k_nt32(NtArgs a, EPI epi) {
    __shared__ Planes pl;
    __shared__ typename EPI::Shared sh;
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wi = w & 3, wj = w >> 2;
    const int fr = lane & 15, fk = lane >> 4;
    int slice, panel;
    block_of(a, (int)blockIdx.x, (int)gridDim.x, panel, slice);
    const int64_t i0 = (int64_t)panel * TILE;
    const int t0 = slice * a.run, t1 = min(a.tiles, t0 + a.run);
    const int nstep = a.nk * (t1 - t0);

    // pieces: rows tid / 4 and 128 more of i, tid / 4 of j, 32 bytes at 32 (tid & 3)
    const int row = tid >> 2, c = tid & 3;
    const int ilast = (int)min<int64_t>(TILE - 1, a.m - 1 - i0);
    const uint32_t vi0 = min(row, ilast) * (uint32_t)a.lda + 32 * c, vi1 = min(row + 128, ilast) * (uint32_t)a.lda + 32 * c;
    const int ci = 16 * (c ^ quad_swizzle((row >> 2) & 3)), cj = 16 * (c ^ quad_swizzle((row >> 3) & 3));
    const int put[3] = {row * KBY + ci, (row + 128) * KBY + ci, (TILE + row) * KBY + cj};
    int st = t0, sk = 0;  // of the next load
    auto load = [&](float (&v)[3][8]) __attribute__((always_inline)) {
        const int ko = sk * 128;
        const char *pa = a.A + i0 * a.lda + ko, *pb = a.B + (int64_t)st * COLS32 * a.ldb;
        const int jlast = (int)min<int64_t>(COLS32 - 1, a.n - 1 - (int64_t)st * COLS32);
        const uint32_t vj = min(row, jlast) * (uint32_t)a.ldb;
        load_row(v[0], pa, vi0, vi0 + 16);
        load_row(v[1], pa, vi1, vi1 + 16);
        load_row(v[2], pb, vj + min(ko + 32 * c, a.bmax), vj + min(ko + 32 * c + 16, a.bmax));
        if (++sk == a.nk) {
            sk = 0;
            ++st;
        }
    };
    f32x4 acc[4][4];
    epi.init(sh, i0 + 64 * wi, lane);
    int k = 0, t = t0;
    auto start = [&](int n) __attribute__((always_inline)) {
        if (k == 0) {
            if (n) epi.tile(sh, acc, (int64_t)(t - 1) * COLS32 + 64 * wj, lane);
            if (n == nstep) return false;
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int g = 0; g < 4; ++g) acc[f][g] = (f32x4)(0.f);
        }
        if (++k == a.nk) {
            k = 0;
            ++t;
        }
        return true;
    };
    const int q = fk ^ quad_swizzle(fr >> 2);
    // row of fragment g: 32 (g >> 1) + 4 (g & 1) + 8 (fr >> 2) + (fr & 3)
    steps32<4>(pl, acc, nstep, put, true, (64 * wi + fr) * KBY + 16 * q,
               (TILE + 64 * wj + 8 * (fr >> 2) + (fr & 3)) * KBY + 16 * q, 4 * KBY, 32 * KBY, load, start);
    epi.finish(sh, i0 + 64 * wi, slice * 2 + wj, lane);
}

// kn_tile of f32: 256 rows and 32 NJ columns, accumulators as kn_tile's, a
// wave's 16 NJ columns.
template <int NJ, bool A_T, class EPI>
__device__ __forceinline__ void kn32_tile(Planes &pl, const KnArgs &a, const EPI &epi, int64_t m0, int64_t n0, int z) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wi = w & 3, wj = w >> 2;
    const int fr = lane & 15, fk = lane >> 4;
    const int s0 = z * a.steps, s1 = min(a.steps_all, s0 + a.steps), nstep = max(0, s1 - s0);

    // pieces of i: as k_nt32, or column tid & 255, rows 8 (tid / 256) and 16
    // more; of j: column tid % (32 NJ), rows 8 (tid / (32 NJ))
    const int ri = A_T ? tid & 255 : tid >> 2, ki = A_T ? tid >> 8 : tid & 3;
    const int rj = tid % (32 * NJ), kj = tid / (32 * NJ);
    auto at = [](int r, int c) __attribute__((always_inline)) { return r * KBY + 16 * (c ^ quad_swizzle((r >> 2) & 3)); };
    const int put[3] = {at(ri, ki), A_T ? at(ri, ki + 2) : at(ri + 128, ki), TILE * KBY + at(rj, kj & 3)};
    const uint32_t vj = (uint32_t)min<int64_t>(4 * rj, a.ldb - 4 - 4 * n0);
    const char *pa = a.A + (A_T ? 4 * m0 + (int64_t)s0 * 32 * a.lda : m0 * a.lda + (int64_t)s0 * 128);
    const char *pb = a.B + 4 * n0 + (int64_t)s0 * 32 * a.ldb;
    int sk = s0;
    auto load = [&](float (&v)[3][8]) __attribute__((always_inline)) {
        const int last = (int)min<int64_t>(31, a.k - 1 - (int64_t)sk * 32);
        if constexpr (A_T) {  // whole tiles exist
            load_col(v[0], pa, 4 * ri, 8 * ki, (uint32_t)a.lda, 31);
            load_col(v[1], pa, 4 * ri, 8 * ki + 16, (uint32_t)a.lda, 31);
        } else {
            const uint32_t o = ri * (uint32_t)a.lda + 32 * ki;
            load_row(v[0], pa, o, o + 16);
            load_row(v[1], pa, o + 128 * (uint32_t)a.lda, o + 128 * (uint32_t)a.lda + 16);
        }
        if (NJ == 4 || tid < 128 * NJ) load_col(v[2], pb, vj, 8 * kj, (uint32_t)a.ldb, last);
        ++sk;
        pa += A_T ? 32 * a.lda : 128;
        pb += 32 * a.ldb;
    };
    f32x4 acc[4][NJ];
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int g = 0; g < NJ; ++g) acc[f][g] = (f32x4)(0.f);
    auto start = [&](int n) __attribute__((always_inline)) { return n < nstep; };
    const int q = 16 * (fk ^ quad_swizzle(fr >> 2));
    steps32<NJ>(pl, acc, nstep, put, NJ == 4 || tid < 128 * NJ, (64 * wi + fr) * KBY + q,
                (TILE + 16 * NJ * wj + fr) * KBY + q, 16 * KBY, 32 * KBY, load, start);
    epi(acc, m0 + 64 * wi, n0 + 16 * NJ * wj, lane, z);
}

template <int NJ, class E1, class E2>
__global__ __launch_bounds__(NT, 2) void k_kn2_32(KnArgs a1, E1 e1, KnGrid g1, KnArgs a2, E2 e2, KnGrid g2) {
    __shared__ Planes pl;
    const int b = (int)blockIdx.x, n1 = g1.blocks();
    if (b < n1) {
        const int v = xcd_range(b, n1), r = v / g1.cols;
        kn32_tile<NJ, false>(pl, a1, e1, (int64_t)(r % g1.rows) * TILE, (int64_t)(v % g1.cols) * 32 * NJ, r / g1.rows);
    } else {
        const int v = xcd_range(b - n1, g2.blocks()), r = v / g2.cols;
        kn32_tile<NJ, true>(pl, a2, e2, (int64_t)(r % g2.rows) * TILE, (int64_t)(v % g2.cols) * 32 * NJ, r / g2.rows);
    }
}

}  // namespace mm
}  // namespace mn

// mm_f32.hpp — the products of mm_tiles.hpp for f32 operands, on the bf16
// matrix cores.
//
// x = h + m + l, 8 significant bits each (exact but for subnormal tails), and a
// product is six bf16 products, mm, lh, hl, mh, hm, hh.  h is cut off (rounded, the
// largest values, which masks are made of, would become infinite), m rounded, so
// that |m| <= 2^-7 |x| and |l| <= 2^-16 |x| with either sign: what is left out (ml,
// lm, ll) is up to 2^-22 |x||y| but 0.4 2^-24 in the mean square, and has no sign of
// its own that would add up over a sum (with m cut off too: up to 2^-21, in the
// mean 0.7 2^-24 towards zero).  Six at the bf16 rate are 2.7 times the f32 matrix
// rate.
//
// A block has a tile of 256 x 128 (or 64 columns), eight waves of 64 x 64 = 4 x
// 4 tiles of 16 x 16.  A step is 32 k's.  LDS holds the three planes of two
// steps, 144 KB.  Waves w and w + 4 share a SIMD and run one barrier window
// apart: while one issues its 96 matrix instructions, the other reads its 24
// fragments and brings its part of the next steps.  A plane buffer is written in
// the windows after those in which both halves have read it (lgkmcnt(0) before
// every barrier).
//
// k_nt32 (rows against rows): the queries are split once, in memory (their
// planes stay in L2); the first half loads them to LDS directly, after its reads
// (before them: 5% slower; between its products, or by both halves: no faster)
// and waits for them when its products end.  The second half loads the items'
// rows to registers, a step ahead, splits them (44 vector instructions for 8
// values) and writes them.
//
// k_kn2_32 (rows times columns): each thread loads 24 values to registers, two
// steps ahead, splits and writes them; a matrix with k in its rows is turned on
// the way (a thread's 8 values are 8 k's of one column).  With D and the queries
// as planes in memory, loaded directly and read transposed, it took as long (4%
// longer to 2% less): half as many bytes again come from L2.
//
// 1024 x 100000 x 768: logits with the loss's sums 672 us (1.40 PFLOP/s of bf16
// products, 234 TFLOP/s of f32 ones; the f32 matrix rate of a large library
// product is 154), the gradients' two products 985 us for 65536 rows.  A step
// takes 4.4 thousand cycles on a few blocks, 5 to 5.4 on all, for 3.1 of matrix
// instructions (490 us if there were nothing else): the reading half's window is
// the longer one, and what comes from L2 slows it when all blocks run (590 us
// without those loads).
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

// 8 values to three times 8 bf16: the upper half of x, x - h rounded, x - h - m.  (The
// differences as dot products of bf16 pairs with (-1, 0) and (0, -1) are exact
// too and fewer instructions, but hold up the matrix pipe: 2.99 -> 3.28 ms for a
// step of 1024 x 100000 x 768.)
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
        const uint32_t m = bf16_pair(x1, y1);
        s[0][p] = upper(x, y);
        s[1][p] = m;
        s[2][p] = upper(x1 - __uint_as_float(m << 16), y1 - __uint_as_float(m & 0xffff0000u));
    }
}

// the same of 4 values
__device__ __forceinline__ void split4(u32x4 v, uint2 (&s)[3]) {
    float x[8] = {__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]), __uint_as_float(v[3]), 0.f, 0.f, 0.f, 0.f};
    u32x4 y[3];
    split8(x, y);
#pragma unroll
    for (int k = 0; k < 3; ++k) s[k] = make_uint2(y[k][0], y[k][1]);
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

__device__ __forceinline__ void write_split(const float (&v)[8], char *plane0) {
    u32x4 s[3];
    split8(v, s);
#pragma unroll
    for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x4 *>(plane0 + p * PLANE) = s[p];
}

// the end of a reading window
__device__ __forceinline__ void reads_end() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    window_end();
}
// the end of the products' window of the half that loads to LDS directly
__device__ __forceinline__ void loads_end() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    window_end();
}

template <int NJ>
__device__ __forceinline__ void products32(f32x4 (&acc)[4][NJ], const u32x4 (&fi)[4][3], const u32x4 (&fj)[NJ][3]) {
    constexpr int PI[6] = {1, 0, 2, 0, 1, 0}, PJ[6] = {1, 2, 0, 1, 0, 0};  // smallest first
    __builtin_amdgcn_s_setprio(1);  // before the other wave's splitting (step of 1024 x 100000 x 768: 2.99 -> 2.95 ms)
#pragma unroll
    for (int x = 0; x < 6; ++x)
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
            for (int g = 0; g < NJ; ++g) acc[f][g] = Bf16::mma(fj[g][PJ[x]], fi[f][PI[x]], acc[f][g]);
    __builtin_amdgcn_s_setprio(0);
}

// What a step's window of the loading half does for A [256][k] of planes:
// rows 64 w .. 64 w + 63 (w < 4) of each, 16 at a time.
struct RowLoads {
    const char *p;
    int64_t plane;
    int v[4];
    uint32_t to;
    __device__ __forceinline__ RowLoads(Planes &pl, const char *base, int64_t lda, int64_t plane_, int last, int w, int lane)
        : p(base), plane(plane_), to(lds_addr(&pl.b[0][0][64 * w * KBY])) {
        const int pc = 16 * ((lane & 3) ^ quad_swizzle((lane >> 4) & 3));
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = min(64 * w + 16 * u + (lane >> 2), last) * (int)lda + pc;
    }
    __device__ __forceinline__ void issue(int64_t k_bytes, int buf) const {
#pragma unroll
        for (int x = 0; x < 3; ++x)
#pragma unroll
            for (int u = 0; u < 4; ++u) dma16(p + x * plane + k_bytes, v[u], to + (buf * 3 + x) * PLANE + 16 * u * KBY);
    }
};

// fragments of rows of k (64 bytes a row in LDS): i at ri + 16 rows each, j at rj
template <int NJ>
__device__ __forceinline__ void read_rows(u32x4 (&fi)[4][3], u32x4 (&fj)[NJ][3], const char *b, int ri, int rj, int jstep0,
                                          int jstep1) {
#pragma unroll
    for (int p = 0; p < 3; ++p) {
#pragma unroll
        for (int f = 0; f < 4; ++f) fi[f][p] = *reinterpret_cast<const u32x4 *>(b + p * PLANE + ri + 16 * f * KBY);
#pragma unroll
        for (int g = 0; g < NJ; ++g)
            fj[g][p] = *reinterpret_cast<const u32x4 *>(b + p * PLANE + rj + (g >> 1) * jstep1 + (g & 1) * jstep0);
    }
}

// k_nt of f32: a tile has 128 rows of B; nk counts steps of 32 k's, bmax is the
// last 16-byte piece of a row of B.  A comes as planes (lda: bytes of a row of
// one).  Accumulators as k_nt's, a wave's 64 columns.
template <class EPI>
__global__ __launch_bounds__(NT, 2) void k_nt32(NtArgs a, int64_t plane, EPI epi) {
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

    f32x4 acc[4][4];
    epi.init(sh, i0 + 64 * wi, lane);
    const int q = fk ^ quad_swizzle(fr >> 2);
    // row of fragment g: 32 (g >> 1) + 4 (g & 1) + 8 (fr >> 2) + (fr & 3)
    const int ri = (64 * wi + fr) * KBY + 16 * q, rj = (TILE + 64 * wj + 8 * (fr >> 2) + (fr & 3)) * KBY + 16 * q;
    u32x4 fi[4][3], fj[4][3];
    int k = 0, t = t0;
    // a step's reads, before them the last tile's end
    auto begin = [&](int n) __attribute__((always_inline)) {
        if (k == 0) {
            if (n) epi.tile(sh, acc, (int64_t)(t - 1) * COLS32 + 64 * wj, lane);
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int g = 0; g < 4; ++g) acc[f][g] = (f32x4)(0.f);
        }
        if (++k == a.nk) {
            k = 0;
            ++t;
        }
        read_rows<4>(fi, fj, &pl.b[n & 1][0][0], ri, rj, 4 * KBY, 32 * KBY);
    };
    if (!wj) {
        const RowLoads rows(pl, a.A + i0 * a.lda, a.lda, plane, (int)min<int64_t>(TILE - 1, a.m - 1 - i0), w, lane);
        int sk = 0;  // of the next loads
        auto issue = [&](int buf) __attribute__((always_inline)) {
            rows.issue(sk * KBY, buf);
            sk = sk + 1 == a.nk ? 0 : sk + 1;
        };
        issue(0);
        loads_end();
        for (int n = 0; n < nstep; ++n) {
            begin(n);
            if (n + 1 < nstep) issue((n + 1) & 1);
            reads_end();
            products32<4>(acc, fi, fj);
            loads_end();
        }
        window_end();  // the other half's last products
    } else {
        // rows r and r + 64 of B, 8 values at 32 (tid & 3) bytes
        const int r = (tid & 255) >> 2, c = tid & 3;
        const int put = (TILE + r) * KBY + 16 * (c ^ quad_swizzle((r >> 3) & 3));
        int st = t0, sk = 0;  // of the next load
        float x[2][8];
        auto load = [&]() __attribute__((always_inline)) {
            const int ko = sk * 128;
            const char *pb = a.B + (int64_t)st * COLS32 * a.ldb;
            const int jlast = (int)min<int64_t>(COLS32 - 1, a.n - 1 - (int64_t)st * COLS32);
            const uint32_t v0 = min(r, jlast) * (uint32_t)a.ldb, v1 = min(r + 64, jlast) * (uint32_t)a.ldb;
            const int lo = min(ko + 32 * c, a.bmax), hi = min(ko + 32 * c + 16, a.bmax);
            load_row(x[0], pb, v0 + lo, v0 + hi);
            load_row(x[1], pb, v1 + lo, v1 + hi);
            if (++sk == a.nk) {
                sk = 0;
                ++st;
            }
        };
        auto write = [&](int buf) __attribute__((always_inline)) {
            write_split(x[0], &pl.b[buf][0][put]);
            write_split(x[1], &pl.b[buf][0][put + 64 * KBY]);
        };
        load();
        write(0);
        if (nstep > 1) load();
        reads_end();
        window_end();
        for (int n = 0; n < nstep; ++n) {
            begin(n);
            if (n + 1 < nstep) write((n + 1) & 1);
            if (n + 2 < nstep) load();
            reads_end();
            products32<4>(acc, fi, fj);
            window_end();
        }
    }
    epi.tile(sh, acc, (int64_t)(t1 - 1) * COLS32 + 64 * wj, lane);
    epi.finish(sh, i0 + 64 * wi, slice * 2 + wj, lane);
}

// The loop of kn32_tile.  load(set): the next step's values (a thread's pieces:
// two of i, one of j); put[k]: where in a plane piece k goes.
template <int NJ, class LOAD>
__device__ __forceinline__ void steps32(Planes &pl, f32x4 (&acc)[4][NJ], int nstep, const int (&put)[3], bool j_half,
                                        int ri, int rj, LOAD load) {
    const int wj = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    float v[2][3][8];
    auto write = [&](float (&x)[3][8], int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 3; ++k)
            if (k < 2 || j_half) write_split(x[k], &pl.b[buf][0][put[k]]);
    };
    if (nstep == 0) return;
    load(v[0]);
    if (nstep > 1) load(v[1]);
    write(v[0], 0);
    if (nstep > 2) load(v[0]);
    reads_end();
    if (wj) window_end();
    u32x4 fi[4][3], fj[NJ][3];
    auto step = [&](int n, int buf, float (&x)[3][8]) __attribute__((always_inline)) {
        read_rows<NJ>(fi, fj, &pl.b[buf][0][0], ri, rj, 16 * KBY, 32 * KBY);
        if (n + 1 < nstep) write(x, buf ^ 1);
        if (n + 3 < nstep) load(x);
        reads_end();
        products32<NJ>(acc, fi, fj);
        window_end();
    };
    for (int n = 0; n < nstep; n += 2) {
        step(n, 0, v[1]);
        if (n + 1 == nstep) break;
        step(n + 1, 1, v[0]);
    }
    if (!wj) window_end();  // the other half's last products
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

    // pieces of i: rows tid / 4 and 128 more, 32 bytes at 32 (tid & 3), or column
    // tid & 255, rows 8 (tid / 256) and 16 more; of j: column tid % (32 NJ), rows 8 (tid / (32 NJ))
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
    const int q = 16 * (fk ^ quad_swizzle(fr >> 2));
    steps32<NJ>(pl, acc, nstep, put, NJ == 4 || tid < 128 * NJ, (64 * wi + fr) * KBY + q,
                (TILE + 16 * NJ * wj + fr) * KBY + q, load);
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

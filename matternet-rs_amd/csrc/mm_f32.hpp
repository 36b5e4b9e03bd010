// mm_f32.hpp — the products of mm_tiles.hpp for f32 operands, on the bf16
// matrix cores.
//
// x = h + m + l, 8 + 8 + 8 significant bits cut off one after the other (exact
// but for subnormal tails), and a product is six bf16 products, mm, lh, hl, mh,
// hm, hh; what is left out (ml, lm, ll) is below 2^-23 |x||y| and mostly far
// below: the size of an f32 product's rounding.  Six at the bf16 rate are 2.7
// times the f32 matrix rate.
//
// Operands stay f32 in memory and LDS; a wave splits its fragments after it has
// read them: 44 vector instructions for 8 values a lane.  That is 2100 cycles a
// wave for a step of 32 k's next to 3070 of its 192 matrix instructions, and
// they run side by side: waves w and w + 4 share a SIMD and are one barrier
// window apart, one reads and splits while the other multiplies.  A step has
// four windows (fragments of i and half of j, products, other half, products);
// registers hold 4 + 4 split fragments beside the 128 accumulators.
//
// LDS: two slots of a step (64 KB), filled by loads that go there directly.
// Waves 0-3 issue a step's loads in their first window, 4-7 at the same time, in
// their last; both wait for them three windows later, before the barrier after
// which they are read.
// Rows of k: 128 bytes a step, piece c (16 bytes) at c ^ s, s = fr / 2 for row
// fr of a fragment's 16; a lane takes pieces lane / 16 and 4 + lane / 16 (the
// order of k is the same for both operands).  Rows of k by columns: 1 KB, the
// 64 bytes of 16 columns s of row k at s ^ ((k / 4) & 3), read a value at a
// time.  Both are free of bank conflicts.
#pragma once
#include "mm_tiles.hpp"

namespace mn {
namespace mm {

constexpr int KBY32 = 128;             // bytes of k in a step of rows of k
constexpr int HALF32 = TILE * KBY32;   // one operand's step, 32 KB

struct alignas(1024) Ring32 {
    char b[2][2][HALF32];
};

struct Split {
    u32x4 h, m, l;
};

// 8 values to three times 8 bf16 (the upper halves of x, x - h, x - h - m)
__device__ __forceinline__ Split split8(f32x4 a, f32x4 b) {
    Split s;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const float x = p < 2 ? a[2 * p] : b[2 * p - 4], y = p < 2 ? a[2 * p + 1] : b[2 * p - 3];
        auto upper = [](float u, float v) __attribute__((always_inline)) {  // v's, u's upper halves
            return __builtin_amdgcn_perm(__float_as_uint(v), __float_as_uint(u), 0x07060302u);
        };
        auto rest = [](float u) __attribute__((always_inline)) {
            return u - __uint_as_float(__float_as_uint(u) & 0xffff0000u);
        };
        s.h[p] = upper(x, y);
        const float x1 = rest(x), y1 = rest(y);
        s.m[p] = upper(x1, y1);
        s.l[p] = upper(rest(x1), rest(y1));
    }
    return s;
}

template <int NJ, int NF>
__device__ __forceinline__ void products(f32x4 (&acc)[4][NF], int g0, const Split (&fi)[4], const Split (&fj)[NJ]) {
    auto one = [&](auto pj, auto pi) __attribute__((always_inline)) {
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
            for (int g = 0; g < NJ; ++g) acc[f][g0 + g] = Bf16::mma(pj(fj[g]), pi(fi[f]), acc[f][g0 + g]);
    };
    auto h = [](const Split &s) __attribute__((always_inline)) { return s.h; };
    auto m = [](const Split &s) __attribute__((always_inline)) { return s.m; };
    auto l = [](const Split &s) __attribute__((always_inline)) { return s.l; };
    one(m, m);
    one(l, h);
    one(h, l);
    one(m, h);
    one(h, m);
    one(h, h);
}

__device__ __forceinline__ void lds_wait() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// the split belongs to the window it is written in: nothing else keeps the
// compiler from moving it next to the products that use it
template <int N>
__device__ __forceinline__ void here(Split (&s)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k) asm volatile("" : "+v"(s[k].h), "+v"(s[k].m), "+v"(s[k].l));
}
__device__ __forceinline__ void vm_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// the order of a window's reads and splits: DS LDS reads a fragment, those of
// fragment k + 2 before the split of fragment k + 1
template <int N, int DS>
__device__ __forceinline__ void read_ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * DS, 0);
#pragma unroll
    for (int k = 0; k < N; ++k) {
        __builtin_amdgcn_sched_group_barrier(0x002, 44, 0);
        if (k + 2 < N) __builtin_amdgcn_sched_group_barrier(0x100, DS, 0);
    }
}

// rows of k: fragment row fr, both pieces of the lane
__device__ __forceinline__ Split read_rows(const char *lo, const char *hi, int off) {
    return split8(*reinterpret_cast<const f32x4 *>(lo + off), *reinterpret_cast<const f32x4 *>(hi + off));
}

// k_nt of f32: nk is steps of 128 bytes, bmax the last 16-byte piece of a row of B.
template <class EPI>
__global__ __launch_bounds__(NT, 2) void k_nt32(NtArgs a, EPI epi) {
    __shared__ Ring32 rg;
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

    // ---- loads: wave w stages rows 32 w .. 32 w + 31 of both operands, 8 a piece
    const int r0 = 32 * w + (lane >> 3), l4 = lane >> 4;
    const int ilast = (int)min<int64_t>(TILE - 1, a.m - 1 - i0);
    int st = t0, sk = 0, staged = 0;
    const char *pa = a.A + i0 * a.lda;
    const uint32_t li = lds_addr(&rg.b[0][0][32 * w * KBY32]), lj = lds_addr(&rg.b[0][1][32 * w * KBY32]);
    auto issue = [&]() __attribute__((always_inline)) {  // the next step, if there is one
        if (staged >= nstep) return;
        const int ko = sk * KBY32, left = a.bmax - ko;  // pieces past a row's last one repeat it
        const int jlast = (int)min<int64_t>(TILE - 1, a.n - 1 - (int64_t)st * TILE);
        const char *pb = a.B + (int64_t)st * TILE * a.ldb;
        const uint32_t slot = (staged & 1) * 2 * HALF32;
        // (offsets worked out here: kept, they would spill)
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const int vi = (int)__umul24(min(r0 + 8 * p, ilast), (int)a.lda) + 16 * ((lane & 7) ^ ((4 * (p & 1) + l4) & 7));
            const int vj = (int)__umul24(min(r0 + 8 * p, jlast), (int)a.ldb) + min(16 * ((lane & 7) ^ (2 * p + (l4 & 1))), left);
            dma16(pa + ko, vi, li + slot + 1024 * p);
            dma16(pb + ko, vj, lj + slot + 1024 * p);
        }
        ++staged;
        if (++sk == a.nk) {
            sk = 0;
            ++st;
        }
    };

    f32x4 acc[4][8];
    Split fi[4], fj[4];
    const int pc = 16 * (fk ^ (fr >> 1));
    const char *ri = &rg.b[0][0][(64 * wi + fr) * KBY32];
    const char *rj = &rg.b[0][1][(128 * wj + 8 * (fr >> 2) + (fr & 3)) * KBY32];
    auto read_j = [&](int so, int g0) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
            fj[g] = read_rows(rj + pc, rj + (pc ^ 64), so + (32 * ((g0 + g) >> 1) + 4 * (g & 1)) * KBY32);
    };
    epi.init(sh, i0 + 64 * wi, lane);
    issue();
    vm_wait();
    window_end();
    if (wj) {
        issue();
        window_end();
    }
    int k = 0, t = t0;
    for (int n = 0;; ++n) {
        if (k == 0) {
            if (n) epi.tile(sh, acc, (int64_t)(t - 1) * TILE + 128 * wj, lane);
            if (n == nstep) break;
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int g = 0; g < 8; ++g) acc[f][g] = (f32x4)(0.f);
        }
        if (!wj) issue();
        const int so = (n & 1) * 2 * HALF32;
#pragma unroll
        for (int f = 0; f < 4; ++f) fi[f] = read_rows(ri + pc, ri + (pc ^ 64), so + 16 * f * KBY32);
        read_j(so, 0);
        here(fi);
        here(fj);
        read_ahead<8, 2>();
        lds_wait();
        window_end();
        products<4>(acc, 0, fi, fj);
        window_end();
        read_j(so, 4);
        here(fj);
        read_ahead<4, 2>();
        lds_wait();
        if (wj) vm_wait();
        window_end();
        if (wj) issue();
        products<4>(acc, 4, fi, fj);
        if (!wj) vm_wait();
        window_end();
        if (++k == a.nk) {
            k = 0;
            ++t;
        }
    }
    if (!wj) window_end();  // the other half's last products, then its last tile
    vm_wait();
    epi.finish(sh, i0 + 64 * wi, slice * 2 + wj, lane);
}

// kn_tile of f32.  NF 8: j in two halves; 4, 2: in one.
template <int NF, bool A_T, class EPI>
__device__ __forceinline__ void kn32_tile(Ring32 &rg, const KnArgs &a, const EPI &epi, int64_t m0, int64_t n0, int z) {
    constexpr int NJ = NF == 8 ? 4 : NF;
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wi = w & 3, wj = w >> 2;
    const int fr = lane & 15, fk = lane >> 4;
    const int s0 = z * a.steps, s1 = min(a.steps_all, s0 + a.steps), nstep = max(0, s1 - s0);

    // ---- loads.  [k][256]: wave w stages rows 4 w .. 4 w + 3; [256][k]: as k_nt32
    const int col = 64 * ((lane >> 2) ^ (w & 3)) + 16 * (lane & 3);
    const int cj = (int)min<int64_t>(col, a.ldb - 16 - 4 * n0);
    int vi[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        if constexpr (A_T) vi[p] = (4 * w + p) * (int)a.lda + col;
        else vi[p] = (32 * w + 8 * p + (lane >> 3)) * (int)a.lda + 16 * ((lane & 7) ^ ((4 * (p & 1) + fk) & 7));
    }
    const int64_t astep = A_T ? 32 * a.lda : KBY32, bstep = 32 * a.ldb;
    const char *pa = a.A + (A_T ? 4 * m0 : m0 * a.lda) + s0 * astep;
    const char *pb = a.B + 4 * n0 + s0 * bstep;
    const uint32_t li = lds_addr(&rg.b[0][0][4096 * w]), lj = lds_addr(&rg.b[0][1][4096 * w]);
    int staged = 0;
    auto issue = [&]() __attribute__((always_inline)) {
        if (staged >= nstep) return;
        const int last = (int)min<int64_t>(31, a.k - 1 - (int64_t)(s0 + staged) * 32);
        const uint32_t slot = (staged & 1) * 2 * HALF32;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            dma16(pa, vi[p], li + slot + 1024 * p);
            dma16(pb, min(4 * w + p, last) * (int)a.ldb + cj, lj + slot + 1024 * p);
        }
        pa += astep;
        pb += bstep;
        ++staged;
    };

    f32x4 acc[4][NF];
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int g = 0; g < NF; ++g) acc[f][g] = (f32x4)(0.f);
    Split fi[4], fj[NJ];
    const int pc = 16 * (fk ^ (fr >> 1));
    const char *ri = &rg.b[0][0][(64 * wi + fr) * KBY32];
    // columns: rows 4 fk .. + 3 and 16 on, 16-column slot s
    auto cols = [&](const char *half, int s) __attribute__((always_inline)) {
        const float *p = reinterpret_cast<const float *>(half + 4096 * fk + 64 * (s ^ fk)) + fr;
        const f32x4 x = {p[0], p[256], p[512], p[768]}, y = {p[4096], p[4352], p[4608], p[4864]};
        return split8(x, y);
    };
    auto read_j = [&](int so, int g0) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < NJ; ++g) fj[g] = cols(&rg.b[0][1][0] + so, NF * wj + g0 + g);
    };
    if (nstep > 0) {
        issue();
        vm_wait();
        window_end();
        if (wj) {
            issue();
            window_end();
        }
        for (int n = 0; n < nstep; ++n) {
            if (!wj) issue();
            const int so = (n & 1) * 2 * HALF32;
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                if constexpr (A_T) fi[f] = cols(&rg.b[0][0][0] + so, 4 * wi + f);
                else fi[f] = read_rows(ri + pc, ri + (pc ^ 64), so + 16 * f * KBY32);
            }
            read_j(so, 0);
            here(fi);
            here(fj);
            read_ahead<4 + NJ, 4>();
            lds_wait();
            window_end();
            products<NJ>(acc, 0, fi, fj);
            window_end();
            if constexpr (NF == 8) {
                read_j(so, 4);
                here(fj);
                read_ahead<NJ, 4>();
            }
            lds_wait();
            if (wj) vm_wait();
            window_end();
            if (wj) issue();
            if constexpr (NF == 8) products<NJ>(acc, 4, fi, fj);
            if (!wj) vm_wait();
            window_end();
        }
        if (!wj) window_end();
        vm_wait();
    }
    epi(acc, m0 + 64 * wi, n0 + 16 * NF * wj, lane, z);
}

template <int NF, class E1, class E2>
__global__ __launch_bounds__(NT, 2) void k_kn2_32(KnArgs a1, E1 e1, KnGrid g1, KnArgs a2, E2 e2, KnGrid g2) {
    __shared__ Ring32 rg;
    const int b = (int)blockIdx.x, n1 = g1.blocks();
    if (b < n1) {
        const int v = xcd_range(b, n1), r = v / g1.cols;
        kn32_tile<NF, false>(rg, a1, e1, (int64_t)(r % g1.rows) * TILE, (int64_t)(v % g1.cols) * 32 * NF, r / g1.rows);
    } else {
        const int v = xcd_range(b - n1, g2.blocks()), r = v / g2.cols;
        kn32_tile<NF, true>(rg, a2, e2, (int64_t)(r % g2.rows) * TILE, (int64_t)(v % g2.cols) * 32 * NF, r / g2.rows);
    }
}

}  // namespace mm
}  // namespace mn

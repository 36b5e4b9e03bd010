// mm_tiles.hpp — matrix products of the item scores (scores.hip) and of the
// softmax loss (softmax.hip) on the matrix cores.
//
//   k_nt   Y[i][j] = sum_k A[i][k] B[j][k]   (rows against rows): a block keeps
//          256 rows of A and goes through a run of 256-row tiles of B
//   k_few  the same for few rows of A, B straight to registers
//   k_kn2  Y[m][n] = sum_k A(m,k) B[k][n]    (A [m][k] or [k][m]): one 256 x 256
//          tile and run of k a block, two such products in a launch
// with f32 (bf16 operands) or int32 (int8 operands) sums; an epilogue object
// takes each wave's accumulators.  f32 operands: mm_f32.hpp.
//
// Schedule (k_nt, k_kn2).  Eight waves, each 64 (i, m) x 128 (j, n) = 4 x 8
// tiles of 16 x 16: 128 accumulator registers.  A k-step is 64 bytes of k (32
// bf16, 64 int8) of both operands, 32 KB, in a ring of four slots, filled three
// steps ahead by loads that go to LDS directly.  Waves w and w + 4 share a SIMD
// and run one barrier window apart: while one issues its 32 matrix
// instructions, the other reads the next step's fragments and issues its four
// loads, so the matrix pipe does not wait for LDS.  A slot is refilled in the
// window after the one in which its last reads ended (lgkmcnt(0) before the
// barrier); vmcnt(8) before a barrier leaves the newest two steps in flight, so
// the step read after the next barrier has landed.  Past the last step the
// loads repeat it into the slot that nobody reads any more: the count stays.
//
// What bounds it: the chip's power, then LDS.  4096 x 131072 x 768 in bf16
// without the epilogue takes 618 us, 1.33 PFLOP/s; with the softmax loss's 667, 62%
// of the matrix pipe at the 1.90 GHz that the chip then holds.  A large library
// product (8192^3, 1.33 to 1.40) fills 87% of the pipe and gets 1.60 GHz for it.
// A step's 32 matrix instructions a wave take a SIMD 512 cycles for each of its
// two waves; its fragments (96 KB a block) and the loads that land (32 KB) take LDS
// the same 1024 at 128 bytes a cycle.  An epilogue is not hidden: the other wave of
// the SIMD has one window to give.
//
// LDS layouts, free of bank conflicts.  Rows of k: a row's k-step is 64 bytes,
// piece c (16 bytes) of row r at c ^ 2 ((r >> s) & 1), s = 3 where a fragment's
// 16 rows are consecutive, 4 where its quads of rows are 8 apart.  Rows of k by
// columns ([k][256]): 512 bytes a row, read transposed (ds_read_b64_tr_b16:
// lane l of 16 gives the address of four columns of row l >> 2 and gets column
// l of the four rows); the 32-byte slot of 16 columns s of row k is at s ^
// ((k & 3) | ((k >> 3) & 1) << 2).
#pragma once
#include <algorithm>

#include "common.hpp"

namespace mn {
namespace mm {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int TILE = 256;              // rows / columns of a tile
constexpr int KBY = 64;                // bytes of k in a step
constexpr int NSLOT = 4;
constexpr int HALF = TILE * KBY;       // one operand's step, 16 KB
constexpr int NT = 512;
constexpr int GP = 8;
// Threads of one launch at most (HIP refuses 2^32); longer work is launched in parts.
constexpr int64_t LAUNCH = (int64_t)1 << 30;

__device__ __forceinline__ uint16_t bf16_bits(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
__device__ __forceinline__ float bf16_value(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
__device__ __forceinline__ uint32_t bf16_pair(float x, float y) {  // (one instruction so; two conversions took two and an or)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x, y}, bf16x2));
}

struct Bf16 {
    typedef f32x4 acc_t;
    // of k_few: matrix instructions for 16 bytes of k; k-steps of a turn
    static constexpr int PARTS = 1, AHEAD = 2;
    static __device__ __forceinline__ acc_t part(u32x4 a, u32x4 b, acc_t c, int) { return mma(a, b, c); }
    static __device__ __forceinline__ acc_t mma(u32x4 a, u32x4 b, acc_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
struct Int8 {
    typedef i32x4 acc_t;
    // of k_few: matrix instructions for 16 bytes of k; k-steps of a turn
    static constexpr int PARTS = 1, AHEAD = 2;
    static __device__ __forceinline__ acc_t part(u32x4 a, u32x4 b, acc_t c, int) { return mma(a, b, c); }
    static __device__ __forceinline__ acc_t mma(u32x4 a, u32x4 b, acc_t c) {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a),
                                                     __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
    }
};

// f32 operands as they are: 16 bytes are four k's of one product each
struct F32 {
    typedef f32x4 acc_t;
    static constexpr int PARTS = 4, AHEAD = 4;
    static __device__ __forceinline__ acc_t part(u32x4 a, u32x4 b, acc_t c, int e) {
        return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
    }
};

struct alignas(1024) Ring {
    char b[NSLOT][2][HALF];  // [.][0]: i / m, [.][1]: j / n
};

__device__ __forceinline__ uint32_t lds_addr(const void *p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)p;
}

// 16 bytes a lane from base + voff to LDS at lds + 16 lane
__device__ __forceinline__ void dma16(const char *base, int voff, uint32_t lds) {
    const uint64_t a = (uint64_t)(uintptr_t)base;
    u32x4 r;
    r.x = __builtin_amdgcn_readfirstlane((uint32_t)a);
    r.y = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xffffu);
    r.z = 0xffffffffu;
    r.w = 0x00020000u;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(r)
                 : "memory", "m0");
}
// 4 bytes a lane
__device__ __forceinline__ void dma4(const char *base, int voff, uint32_t lds) {
    const uint64_t a = (uint64_t)(uintptr_t)base;
    u32x4 r;
    r.x = __builtin_amdgcn_readfirstlane((uint32_t)a);
    r.y = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xffffu);
    r.z = 0xffffffffu;
    r.w = 0x00020000u;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(r)
                 : "memory", "m0");
}

// one 16-byte store instruction, to base + voff
__device__ __forceinline__ void store16(char *base, int voff, uint4 x) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(base, 0, 0xffffffffu, 0x00020000);
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), r, voff, 0, 0);
}

// the end of a barrier window
__device__ __forceinline__ void window_end() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// N: 8, or 8 and the stores issued since the loads of the step read next
template <int N>
__device__ __forceinline__ void read_window_end() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    window_end();
}

// block b of n so that each of the 8 XCDs (blocks go to them in turn) gets a
// contiguous range: neighbours share operands in one L2
__device__ __forceinline__ int xcd_range(int b, int n) {
    const int q = n / 8, r = n % 8, x = b % 8;
    return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + b / 8;
}

struct NtArgs {
    const char *A;      // [m][lda] bytes, rows zero from their end to the end of nk steps
    const char *B;      // [n][ldb]; bytes past bmax + 16 of a row are never read
    int64_t lda, ldb;
    int64_t m, n;
    int nk;             // k-steps of a row
    int bmax;           // last 16-byte piece of a row of B
    int panels, slices; // 256-row panels of A; runs of tiles of B
    int tiles, run;     // tiles of B, tiles of a run
};

// How many runs the tiles of B are cut into for `panels` panels: the cut with
// the least rounds of 256 blocks, a run costing its tiles and 0.3 for filling
// the ring.
inline void plan_runs(NtArgs &a, int cols = TILE) {  // cols: rows of B in a tile
    a.panels = (int)((a.m + TILE - 1) / TILE);
    a.tiles = (int)((a.n + cols - 1) / cols);
    double best = 1e300;
    a.run = a.tiles;  // panels alone are below the limit of blocks
    for (int run = 1; run <= a.tiles; run = run < 32 ? run + 1 : run + run / 16) {
        const int64_t s = (a.tiles + run - 1) / run, blocks = s * a.panels;
        const double cost = (double)((blocks + 255) / 256) * (run + 0.3);
        if (blocks * NT < ((int64_t)1 << 32) && cost < best * 0.999) {
            best = cost;
            a.run = run;
        }
    }
    a.slices = (a.tiles + a.run - 1) / a.run;
}

// A block's panel of A and run of tiles of B: GP panels by 32 / GP runs on an
// XCD at a time (1, 2, 4, 8, 16: 3.11, 3.11, 3.11, 3.09, 3.13 ms for a step of
// 4096 x 131072 x 768).
__device__ __forceinline__ void block_of(const NtArgs &a, int b, int n, int &panel, int &slice) {
    int v = xcd_range(b, n);
    const int grp = v / (GP * a.slices);
    v -= grp * GP * a.slices;
    const int gp = min(GP, a.panels - GP * grp);
    slice = v / gp;
    panel = GP * grp + v % gp;
}

// Epilogue: init (before the loop), fetch (a tile's loads to LDS; FETCH: there
// are any), tile (a tile's accumulators; stage: STAGE bytes of LDS of the
// wave's own; with `counted` set it issued at least STORES store instructions),
// finish.
// accumulator r of tile (f, g): row i = 16 f + (lane & 15) of the wave's 64,
// column j = 32 (g >> 1) + 8 (lane >> 4) + 4 (g & 1) + r of its 128, so that a
// lane holds 8 neighbours of a row in each pair of tiles
template <class OP, class EPI>
__global__ __launch_bounds__(NT, 2) void k_nt(NtArgs a, EPI epi) {
    __shared__ Ring rg;
    __shared__ typename EPI::Shared sh;
    // waves w and w + 4 write their tiles out in different windows
    __shared__ alignas(16) char stage_[EPI::STAGE ? 4 * EPI::STAGE : 16];
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wi = w & 3, wj = w >> 2;
    const int fr = lane & 15, fk = lane >> 4;
    int slice, panel;
    block_of(a, (int)blockIdx.x, (int)gridDim.x, panel, slice);
    const int64_t i0 = (int64_t)panel * TILE;
    const int t0 = slice * a.run, t1 = min(a.tiles, t0 + a.run);
    const int nstep = a.nk * (t1 - t0);

    // ---- loads: wave w stages rows 32 w .. 32 w + 31 of both operands
    const int r0 = 32 * w + (lane >> 2), r1 = r0 + 16;
    const int ilast = (int)min<int64_t>(TILE - 1, a.m - 1 - i0);
    const int pci = 16 * ((lane & 3) ^ (((r0 >> 3) & 1) << 1));  // r1: the same bit
    const int pcj0 = 16 * ((lane & 3) ^ (((r0 >> 4) & 1) << 1)), pcj1 = 16 * ((lane & 3) ^ (((r1 >> 4) & 1) << 1));
    const int vi0 = min(r0, ilast) * (int)a.lda + pci, vi1 = min(r1, ilast) * (int)a.lda + pci;
    int vj0 = 0, vj1 = 0;
    int st = t0, sk = 0;   // the staged step: tile, k
    uint32_t slot = 0;
    const char *pa = a.A + i0 * a.lda, *pb;
    auto rows_j = [&]() __attribute__((always_inline)) {
        pb = a.B + (int64_t)st * TILE * a.ldb;
        const int jlast = (int)min<int64_t>(TILE - 1, a.n - 1 - (int64_t)st * TILE);
        vj0 = min(r0, jlast) * (int)a.ldb;
        vj1 = min(r1, jlast) * (int)a.ldb;
    };
    rows_j();
    const uint32_t li = lds_addr(&rg.b[0][0][32 * w * KBY]), lj = lds_addr(&rg.b[0][1][32 * w * KBY]);
    auto issue = [&]() __attribute__((always_inline)) {
        const int ko = sk * KBY;
        const int left = a.bmax - ko;  // pieces past a row's last one repeat it
        dma16(pa + ko, vi0, li + slot);
        dma16(pa + ko, vi1, li + slot + 1024);
        dma16(pb + ko, vj0 + min(pcj0, left), lj + slot);
        dma16(pb + ko, vj1 + min(pcj1, left), lj + slot + 1024);
        slot = (slot + 2 * HALF) & (NSLOT * 2 * HALF - 1);
        if (++sk == a.nk) {
            if (st + 1 < t1) {
                sk = 0;
                ++st;
                rows_j();
            } else {  // past the end: the last step again
                sk = a.nk - 1;
            }
        }
    };

    typename OP::acc_t acc[4][8];
    u32x4 fi[4], fj[8];
    const char *ri = &rg.b[0][0][(64 * wi + fr) * KBY + 16 * (fk ^ (((fr >> 3) & 1) << 1))];
    // row of fragment g: 32 (g >> 1) + 4 (g & 1) + 8 (fr >> 2) + (fr & 3)
    char *stage = stage_ + wi * EPI::STAGE;
    const char *rj = &rg.b[0][1][(128 * wj + 8 * (fr >> 2) + (fr & 3)) * KBY + 16 * (fk ^ (((fr >> 3) & 1) << 1))];
    epi.init(sh, i0 + 64 * wi, lane);
    issue();
    issue();
    issue();
    asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    window_end();
    if (wj) window_end();
    int k = 0, t = t0;
    const int per = a.nk;
    for (int n = 0;; ++n) {
        if (k == 0) {
            if (n) {
                if constexpr (EPI::STAGE > 0) epi.tile(sh, stage, acc, (int64_t)(t - 1) * TILE + 128 * wj, lane, (t - 1) & 1);
                else epi.tile(sh, acc, (int64_t)(t - 1) * TILE + 128 * wj, lane);
            }
            if (n == nstep) break;
            epi.fetch(sh, (int64_t)t * TILE, tid, t & 1);
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int g = 0; g < 8; ++g) acc[f][g] = (typename OP::acc_t)(0);
        }
        const int so = (n & (NSLOT - 1)) * 2 * HALF;
#pragma unroll
        for (int f = 0; f < 4; ++f) fi[f] = *reinterpret_cast<const u32x4 *>(ri + so + 16 * f * KBY);
#pragma unroll
        for (int g = 0; g < 8; ++g)
            fj[g] = *reinterpret_cast<const u32x4 *>(rj + so + (32 * (g >> 1) + 4 * (g & 1)) * KBY);
        issue();
        if (EPI::FETCH && per < 4) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        // a tile's stores come between the loads of the next two steps and
        // those of the third: they have two steps to drain
        if (EPI::STORES > 0 && k < 2 && n >= per && epi.counted) read_window_end<(8 + EPI::STORES < 63 ? 8 + EPI::STORES : 63)>();
        else read_window_end<8>();
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
            for (int g = 0; g < 8; ++g) acc[f][g] = OP::mma(fj[g], fi[f], acc[f][g]);
        window_end();
        if (++k == per) {
            k = 0;
            ++t;
        }
    }
    if (!wj) window_end();  // the other half's last products, then its last tile
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    epi.finish(sh, i0 + 64 * wi, slice * 2 + wj, lane);
}

// Few queries against many rows (up to 64, or more in groups of 16 to 64 where
// that is the faster): that the bytes of B are in flight is all that counts.  The
// queries lie in LDS ([k-step][query][64 bytes], pieces at c ^ 2 ((query >> 3) & 1):
// no bank conflicts), a wave takes 16 rows of B at a time from memory to
// registers, a turn of k-steps ahead of their products (the next 16 rows' first
// turn too), and the block's waves go through B side by side.
// One query on 1M rows of 768 codes (768 MB): 132 us, 5.8 TB/s; 512 blocks (768:
// 134, 1024: 145, 256: 181), turns of two k-steps (one: 162, three: 138, four:
// 137), through the caches (past them: 150).  f32, whose products take longer
// than the bytes: turns of four (64 queries x 200000 x 512: 162 us, two: 192);
// more queries than LDS holds go in groups.
struct FewArgs {
    const char *Q, *B;
    int64_t ldq, ldb;  // bytes, multiples of 16
    int64_t n;         // rows of B
    int m;             // queries
    int qbytes;        // bytes of a query's row that count (zeros behind)
    int nk, bmax;
    int mf;            // a block has 16 mf queries in LDS
    int groups;        // of so many queries; the groups' blocks of the same rows lie side by side on an XCD
    int slices;        // blocks of a group
    bool small;        // queries take at most FEW_SMALL bytes of LDS
};
constexpr int FEW_SMALL = 40 << 10, FEW_LARGE = 144 << 10;

// false: the queries do not fit LDS (split: not even 16 of them)
inline bool plan_few(FewArgs &a, bool split) {
    a.nk = (a.qbytes + KBY - 1) / KBY;
    a.bmax = (a.qbytes + 15) / 16 * 16 - 16;
    a.mf = a.m <= 16 ? 1 : a.m <= 32 ? 2 : 4;
    auto bytes = [&]() { return (int64_t)a.mf * 16 * a.nk * KBY; };
    while (split && a.mf > 1 && bytes() > FEW_LARGE) a.mf /= 2;
    a.small = bytes() <= FEW_SMALL;
    if (bytes() > FEW_LARGE) return false;
    a.groups = (a.m + 16 * a.mf - 1) / (16 * a.mf);
    a.slices = (int)std::min<int64_t>((a.n + 127) / 128, std::max(1, (a.small ? 512 : 256) / a.groups));
    if (a.groups > 1) a.slices = (a.slices + 7) / 8 * 8;
    return true;
}

// Whether k_few takes less time than k_nt for more than 64 queries, by what both
// take, in us (int8 and bf16): few problems have tiles enough to hide a tile's
// start and end.  tile: that of a tile of k_nt beside its k-steps.  Scores of m x
// n x d to f32: 128 x 16000 x 768 9.2 us by k_few, 20.1 by k_nt; 512 x 16000 x 768
// 23.1, 22.1; 1000 x 4000 x 64 7.0, 17.2; 1000 x 64000 x 256 89, 70.
inline bool few_faster(const FewArgs &a, const NtArgs &nt, double tile) {
    const double few = 3 + 16.0 * a.mf * a.groups * a.n * (1.6e-7 * a.nk + 6e-7);
    const int64_t rounds = ((int64_t)nt.panels * nt.slices + 255) / 256;
    return a.groups <= 32 && few < 0.9 * (4 + (double)rounds * nt.run * (tile + 0.75 * nt.nk));
}

template <class OP, int MF, int LDSB, class EPI>
__global__ __launch_bounds__(NT) void k_few(FewArgs a, EPI epi) {
    __shared__ alignas(16) char qs[LDSB];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int fr = lane & 15, fk = lane >> 4;
    const int unit = (int)blockIdx.x >> 3, slice = ((int)blockIdx.x & 7) + 8 * (unit / a.groups);
    const int q0 = 16 * MF * (unit % a.groups);
    for (int p = tid; p < 64 * MF * a.nk; p += NT) {
        const int c = p & 3, r = (p >> 2) % (16 * MF), kc = (p >> 2) / (16 * MF);
        const int byte = kc * KBY + 16 * c;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (q0 + r < a.m && byte < a.qbytes && epi.takes(q0 + r)) {
            x = *reinterpret_cast<const uint4 *>(a.Q + (q0 + r) * a.ldq + byte);
            const int left = a.qbytes - byte;  // bytes of the piece that count
            if (left < 16) {
                uint32_t *q = &x.x;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int keep = left - 4 * e;
                    q[e] = keep >= 4 ? q[e] : keep <= 0 ? 0u : q[e] & ((1u << (8 * keep)) - 1u);
                }
            }
        }
        *reinterpret_cast<uint4 *>(qs + (p >> 2) * KBY + 16 * (c ^ (((r >> 3) & 1) << 1))) = x;
    }
    epi.init(q0, lane);
    __syncthreads();
    const char *qr = qs + fr * KBY + 16 * (fk ^ (((fr >> 3) & 1) << 1));
    const int64_t groups = (a.n + 15) / 16;
    const int64_t stride = (int64_t)a.slices * (NT / 64);
    int64_t g = (int64_t)slice * (NT / 64) + w;
    typename OP::acc_t acc[MF];
    constexpr int U = OP::AHEAD;
    u32x4 b[2][U];
    auto row_of = [&](int64_t x) __attribute__((always_inline)) { return a.B + min(16 * x + fr, a.n - 1) * a.ldb; };
    auto load = [&](u32x4 (&x)[U], const char *row, int kc) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const u32x4 *>(row + min((kc + u) * KBY + 16 * fk, a.bmax));
    };
    const char *row = nullptr;
    int kc = 0;
    // a turn of U k-steps: those after them on their way first, of the next rows too
    auto turn = [&](u32x4 (&x)[U], u32x4 (&next)[U]) __attribute__((always_inline)) {
        const bool last = kc + U >= a.nk;
        const int64_t gn = last ? g + stride : g;
        const int kn = last ? 0 : kc + U;
        if (kc == 0) {
            epi.fetch(16 * g, lane);
#pragma unroll
            for (int f = 0; f < MF; ++f) acc[f] = (typename OP::acc_t)(0);
        }
        if (gn < groups) {
            if (last) row = row_of(gn);
            load(next, row, kn);
        }
        auto use = [&](int u) __attribute__((always_inline)) {
            u32x4 q[MF];
#pragma unroll
            for (int f = 0; f < MF; ++f) q[f] = *reinterpret_cast<const u32x4 *>(qr + ((kc + u) * MF + f) * 16 * KBY);
#pragma unroll
            for (int e = 0; e < OP::PARTS; ++e)
#pragma unroll
                for (int f = 0; f < MF; ++f) acc[f] = OP::part(x[u], q[f], acc[f], e);
        };
        if (kc + U <= a.nk) {
#pragma unroll
            for (int u = 0; u < U; ++u) use(u);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (kc + u < a.nk) use(u);
        }
        if (last) epi.group(acc, 16 * g, lane);
        g = gn;
        kc = kn;
        return g < groups;
    };
    if (g < groups) {
        row = row_of(g);
        load(b[0], row, 0);
        while (turn(b[0], b[1]) && turn(b[1], b[0])) {
        }
    }
    epi.finish(qs, slice, tid);
}

template <class OP, int MF, class EPI>
void launch_few(const FewArgs &a, const EPI &epi, hipStream_t s) {
    if (a.small) hipLaunchKernelGGL((k_few<OP, MF, FEW_SMALL, EPI>), dim3(a.slices * a.groups), dim3(NT), 0, s, a, epi);
    else hipLaunchKernelGGL((k_few<OP, MF, FEW_LARGE, EPI>), dim3(a.slices * a.groups), dim3(NT), 0, s, a, epi);
}

struct KnArgs {
    const char *A;      // [m][lda] (A_T false) or [k][lda] (A_T true); whole tiles exist
    const char *B;      // [k][ldb]; columns past ldb and rows past k are never read
    int64_t lda, ldb;   // bytes; ldb a multiple of 16
    int64_t k;          // rows of B; A's entries past k are zero
    int steps;          // k-steps of 32 of a run (a block takes one)
    int steps_all;
};

// A fragment of [32 k][256] (16-column slot s), read transposed: row 8 fk + (fr >>
// 2) and 4 below
__device__ __forceinline__ u32x4 read_turned(const char *half, int s, int fr, int fk) {
    const char *p = half + (8 * fk + (fr >> 2)) * 512 + 8 * (fr & 3) + 32 * (s ^ ((fr >> 2) | ((fk & 1) << 2)));
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p));
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p + 4 * 512));
    const uint2 a2 = __builtin_bit_cast(uint2, x), b2 = __builtin_bit_cast(uint2, y);
    return (u32x4){a2.x, a2.y, b2.x, b2.y};
}

// One more entry for each k of A [k][m], x[k * stride] (as bf16) at column at[k] -
// first where that is among the columns; at < 0: none.
struct KnExtra {
    const int32_t *at;
    const float *x;
    int stride;
    int64_t first;
};
constexpr int EXTRA_SCAN = 8;   // entries of at that a thread looks at together
constexpr int EXTRA_GROUPS = 3; // ring slots of 32 entries; the fourth holds the list

// The extra entries of a tile, after its steps: the k's whose column is in the
// tile are listed (in their order: the sums are the same every time), and 32 of
// them are a step of their own, with gathered rows of B.  It costs a step of the
// softmax loss of 4096 x 131072 x 768 1% (3.04 -> 3.08 ms), one of 70001 x 40 x 256,
// where every k's column is in the tile, 10% (241 -> 266 us).
template <int NF>
__device__ __forceinline__ void add_extra(Ring &rg, int (&counts)[64], const KnArgs &a, const KnExtra &x, f32x4 (&acc)[4][NF],
                                          int64_t m0, int64_t n0, int s0, int s1) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wi = w & 3, wj = w >> 2;
    const int fr = lane & 15, fk = lane >> 4;
    auto turned = [](int k) __attribute__((always_inline)) { return (k & 3) | (((k >> 3) & 1) << 2); };
    uint2 *list = reinterpret_cast<uint2 *>(&rg.b[EXTRA_GROUPS][0][0]);  // k; column, value
    const int64_t first = x.first + m0, k1 = min<int64_t>(a.k, 32 * (int64_t)s1);
    const char *b = a.B + 2 * n0;
    for (int64_t c0 = 32 * (int64_t)s0; c0 < k1; c0 += EXTRA_SCAN * NT) {
        int at[EXTRA_SCAN];
#pragma unroll
        for (int u = 0; u < EXTRA_SCAN; ++u) {
            const int64_t k = c0 + NT * u + tid;
            at[u] = k < k1 ? x.at[k] : -1;
        }
#pragma unroll
        for (int u = 0; u < EXTRA_SCAN; ++u) {
            const int64_t m = at[u] - first;
            at[u] = at[u] >= 0 && m >= 0 && m < TILE ? (int)m : -1;
            const uint64_t in = __ballot(at[u] >= 0);
            if (lane == 0) counts[8 * u + w] = __popcll(in);
        }
        __syncthreads();  // the steps' loads and reads have ended too
        int sum = counts[lane];
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(sum, o);
            sum += lane >= o ? y : 0;
        }
        const int total = __builtin_amdgcn_readfirstlane(__shfl(sum, 63));
#pragma unroll
        for (int u = 0; u < EXTRA_SCAN; ++u) {
            const uint64_t in = __ballot(at[u] >= 0);
            const int end = __shfl(sum, 8 * u + w);
            if (at[u] >= 0) {
                const int64_t k = c0 + NT * u + tid;
                const uint32_t v = __builtin_bit_cast(uint16_t, (__bf16)x.x[k * x.stride]);
                list[end - __popcll(in >> lane)] = make_uint2((uint32_t)k, (uint32_t)at[u] | v << 16);
            }
        }
        __syncthreads();
        for (int e0 = 0; e0 < total; e0 += 32 * EXTRA_GROUPS) {
            const int n = min(32 * EXTRA_GROUPS, total - e0), groups = (n + 31) / 32;
            for (int h = 0; h < groups; ++h)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const int k = 4 * w + 2 * p + (lane >> 5), e = e0 + 32 * h + k;
                    const int c = 16 * ((((lane & 31) >> 1) ^ turned(k)) * 2 + (lane & 1));
                    u32x4 y = (u32x4)(0u);
                    if (e < total) y = *reinterpret_cast<const u32x4 *>(b + list[e].x * a.ldb + min<int64_t>(c, a.ldb - 16 - 2 * n0));
                    const int to = 2048 * w + 1024 * p + 16 * lane;
                    *reinterpret_cast<u32x4 *>(&rg.b[h][0][to]) = (u32x4)(0u);
                    *reinterpret_cast<u32x4 *>(&rg.b[h][1][to]) = y;
                }
            __syncthreads();
            if (tid < n) {
                const int k = tid & 31, m = list[e0 + tid].y & 0xffff;
                char *row = &rg.b[tid >> 5][0][512 * k];
                *reinterpret_cast<uint16_t *>(row + 32 * ((m >> 4) ^ turned(k)) + 2 * (m & 15)) = (uint16_t)(list[e0 + tid].y >> 16);
            }
            __syncthreads();
            for (int h = 0; h < groups; ++h) {
                u32x4 fi[4], fj[NF];
#pragma unroll
                for (int f = 0; f < 4; ++f) fi[f] = read_turned(&rg.b[h][0][0], 4 * wi + f, fr, fk);
#pragma unroll
                for (int g = 0; g < NF; ++g) fj[g] = read_turned(&rg.b[h][1][0], NF * wj + g, fr, fk);
#pragma unroll
                for (int f = 0; f < 4; ++f)
#pragma unroll
                    for (int g = 0; g < NF; ++g) acc[f][g] = Bf16::mma(fj[g], fi[f], acc[f][g]);
            }
            __syncthreads();
        }
    }
}

// One tile of 256 rows and 32 NF columns (the rest of a step's 256 columns of B
// is loaded and not used): accumulator r of (f, g) is row m = 16 f + (lane & 15)
// of the wave's 64, column n = 16 g + 4 (lane >> 4) + r of its 16 NF; z: which
// run of k-steps.  NF 8 wherever more than 128 columns are wanted, else 4 or 2.
template <int NF, bool A_T, class EPI>
__device__ __forceinline__ void kn_tile(Ring &rg, int (&counts)[64], const KnArgs &a, const KnExtra &extra, const EPI &epi,
                                        int64_t m0, int64_t n0, int z) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wi = w & 3, wj = w >> 2;
    const int fr = lane & 15, fk = lane >> 4;
    const int s0 = z * a.steps, s1 = min(a.steps_all, s0 + a.steps);
    const int nstep = max(0, s1 - s0);

    // ---- loads.  [k][256]: wave w stages rows 4 w .. 4 w + 3 in two pieces of
    // two rows; [256][k]: rows 32 w .. as k_nt
    const int kr0 = 4 * w + (lane >> 5);  // the second piece: kr0 + 2
    auto col = [&](int kr) __attribute__((always_inline)) {
        const int f = (kr & 3) | (((kr >> 3) & 1) << 2);
        return 16 * ((((lane & 31) >> 1) ^ f) * 2 + (lane & 1));
    };
    const int cj0 = (int)min<int64_t>(col(kr0), a.ldb - 16 - 2 * n0), cj1 = (int)min<int64_t>(col(kr0 + 2), a.ldb - 16 - 2 * n0);
    const int64_t kstep = 32 * a.ldb;
    int vi0, vi1;
    int64_t astep;
    if constexpr (A_T) {
        vi0 = kr0 * (int)a.lda + col(kr0);
        vi1 = (kr0 + 2) * (int)a.lda + col(kr0 + 2);
        astep = 32 * a.lda;
    } else {
        const int r0 = 32 * w + (lane >> 2);
        const int pc = 16 * ((lane & 3) ^ (((r0 >> 3) & 1) << 1));
        vi0 = r0 * (int)a.lda + pc;
        vi1 = (r0 + 16) * (int)a.lda + pc;
        astep = KBY;
    }
    int sk = s0;
    uint32_t slot = 0;
    const char *pa = a.A + (A_T ? 2 * m0 : m0 * a.lda) + sk * astep;
    const char *pb = a.B + 2 * n0 + sk * kstep;
    const uint32_t li = lds_addr(&rg.b[0][0][2048 * w]), lj = lds_addr(&rg.b[0][1][2048 * w]);
    auto issue = [&]() __attribute__((always_inline)) {
        const int last = (int)min<int64_t>(31, a.k - 1 - (int64_t)sk * 32);
        dma16(pa, vi0, li + slot);
        dma16(pa, vi1, li + slot + 1024);
        dma16(pb, min(kr0, last) * (int)a.ldb + cj0, lj + slot);
        dma16(pb, min(kr0 + 2, last) * (int)a.ldb + cj1, lj + slot + 1024);
        slot = (slot + 2 * HALF) & (NSLOT * 2 * HALF - 1);
        if (sk + 1 < s1) {  // past the end: the last step again
            ++sk;
            pa += astep;
            pb += kstep;
        }
    };

    f32x4 acc[4][NF];
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int g = 0; g < NF; ++g) acc[f][g] = (f32x4)(0.f);
    u32x4 fi[4], fj[NF];
    const char *ri = &rg.b[0][0][(64 * wi + fr) * KBY + 16 * (fk ^ (((fr >> 3) & 1) << 1))];
    if (nstep > 0) {
        issue();
        issue();
        issue();
        asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        window_end();
        if (wj) window_end();
        for (int n = 0; n < nstep; ++n) {
            const int so = (n & (NSLOT - 1)) * 2 * HALF;
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                if constexpr (A_T) fi[f] = read_turned(&rg.b[0][0][0] + so, 4 * wi + f, fr, fk);
                else fi[f] = *reinterpret_cast<const u32x4 *>(ri + so + 16 * f * KBY);
            }
#pragma unroll
            for (int g = 0; g < NF; ++g) fj[g] = read_turned(&rg.b[0][1][0] + so, NF * wj + g, fr, fk);
            read_window_end<4>();
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int g = 0; g < NF; ++g) {
                    acc[f][g] = Bf16::mma(fj[g], fi[f], acc[f][g]);
                    if (NF * f + g == 4) {  // the loads among the products: what is read next is two steps old
                        __builtin_amdgcn_sched_barrier(0);
                        issue();
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            window_end();
        }
        if (!wj) window_end();
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    if constexpr (A_T) add_extra<NF>(rg, counts, a, extra, acc, m0, n0, s0, s1);
    epi(acc, m0 + 64 * wi, n0 + 16 * NF * wj, lane, z);
}

// What a launch of k_kn2 has of one product: blocks = splits x rows x cols of
// tiles, columns fastest (they share A), then rows (they share B).
struct KnGrid {
    int cols, rows, splits;
    __host__ __device__ int blocks() const { return cols * rows * splits; }
};

// Two products in one launch, so that the tiles of the second fill the
// processors that the last round of the first leaves idle: A [m][k] first, then
// A [k][m].  Bound as k_nt, with twice the read instructions for a transposed
// fragment; the loads are issued among the products (in the reading window: 379
// us; k_nt is the faster that way): 4096 x 32768 x 768 and its transpose 351 to 373
// us, 1.1 PFLOP/s, with the extra entries of the second.
template <int NF, class E1, class E2>
__global__ __launch_bounds__(NT, 2) void k_kn2(KnArgs a1, E1 e1, KnGrid g1, KnArgs a2, E2 e2, KnGrid g2, KnExtra extra) {
    __shared__ Ring rg;
    __shared__ int counts[64];
    const int b = (int)blockIdx.x, n1 = g1.blocks();
    if (b < n1) {
        const int v = xcd_range(b, n1), r = v / g1.cols;
        kn_tile<NF, false>(rg, counts, a1, extra, e1, (int64_t)(r % g1.rows) * TILE, (int64_t)(v % g1.cols) * 32 * NF, r / g1.rows);
    } else {
        const int v = xcd_range(b - n1, g2.blocks()), r = v / g2.cols;
        kn_tile<NF, true>(rg, counts, a2, extra, e2, (int64_t)(r % g2.rows) * TILE, (int64_t)(v % g2.cols) * 32 * NF, r / g2.rows);
    }
}

// the first n (<= 4) of x to element e of an f32 or bf16 array, any alignment
template <bool F32>
__device__ __forceinline__ void store4(void *out, int64_t e, int n, f32x4 x) {
    if constexpr (F32) {
        float *p = (float *)out + e;
        if (n == 4) {
            __builtin_memcpy(p, &x, 16);
        } else {
            for (int q = 0; q < n; ++q) p[q] = q == 0 ? x[0] : q == 1 ? x[1] : x[2];
        }
    } else {
        uint16_t *p = (uint16_t *)out + e;
        const uint2 y = make_uint2(bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]));
        if (n == 4) {
            __builtin_memcpy(p, &y, 8);
        } else {
            for (int q = 0; q < n; ++q) p[q] = (uint16_t)((q < 2 ? y.x : y.y) >> (16 * (q & 1)));
        }
    }
}

}  // namespace mm
}  // namespace mn

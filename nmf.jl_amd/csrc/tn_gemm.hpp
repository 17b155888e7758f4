// tn_gemm.hpp -- D(m, n) = sum_c A(m, c) B(n, c) for operands whose contraction index c is contiguous in memory, with the consumer of D
// as an epilogue functor: the products of the softmax cross entropy (xent.hip) and their gradients, in bf16, f16 and f32, accumulated in
// f32.
//
// Bytes, not elements, are the unit: a row of an LDS tile is 128 bytes = 8 chunks of 16 (64 contraction steps of a 16-bit type, 32 of
// f32), so one address path serves all types.  Both operands see the same order of c inside a tile, so any order is right.
//
// Feeding the matrix unit (bf16, 256 x 256 tile, 2048 x 32768 x 8192 product; TFLOP/s after each step):
//   1120  32x32x16 instructions, fragments read a quarter of a tile ahead, one barrier a tile in front of its last quarter, the loads of
//         the tile after next all issued behind it (two LDS stages)
//   1212  the loads written out (to_lds), so that the compiler waits for none of them in front of a read, and a main loop without
//         conditions
//   1247  loads between the products instead of in a bunch: a bunch fills the address unit's queue and holds the wave's products back
//   1290  16x16x32 instructions.  At this rate the card runs at its power limit, and they do the same work for less: registers alone,
//         1985 TFLOP/s against 1745
//   1318  the loads spread over 20 products, 8 of them in the next tile (12: 1290, 28: 1276, 44: 1198: the last ones then come too late)
// A row stride that is a large power of two sends the rows of a tile to few memory channels (2048 x 8192 x 32768: 1137 TFLOP/s at 65536
// bytes, 1317 at 256 more): images made for these products are padded, or stored in blocks (Blocked).  Stages of 64-byte rows, 4 or 5 deep, were slower (1174-1195).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nmfx {
namespace tn {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Elem;
template <> struct Elem<__bf16> {
    static constexpr int PARTS = 1;      // matrix instructions for a chunk
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c, int) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Elem<_Float16> {
    static constexpr int PARTS = 1;
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c, int) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
// f32: a chunk is 4 contraction steps; the four quarters of the wave hold chunks 4 q .. 4 q + 3, and the e-th of four 16x16x4 instructions
// takes each one's e-th element
template <> struct Elem<float> {
    static constexpr int PARTS = 4;
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c, int e) {
        return __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, a)[e], __builtin_bit_cast(f32x4, b)[e], c, 0, 0, 0);
    }
};

constexpr int ROW = 128;   // bytes of a tile's row

struct Operand {
    const void *p;
    int64_t ld;            // bytes between rows (a multiple of 16; p is 16-byte aligned)
    int64_t block;         // bytes between blocks of 256 rows
    int rows;              // rows that exist; rows behind them read as zero (or as what is there: their results are nobody's)
    int chunks;            // 16-byte chunks of a row that exist; chunks behind them read as zero
    int kstep;             // bytes between a row's tiles of the contraction
    uint32_t width;        // bytes from a row's start to where its last chunk ends
};
inline Operand plain(const void *p, int64_t ld, int rows, int chunks) { return Operand{p, ld, 256 * ld, rows, chunks, ROW, (uint32_t)chunks * 16}; }
// An operand of this project's own making is stored in blocks, block x tile x row: what a block of 256 rows has of one tile of the contraction
// (256 x 128 bytes) lies together, so that a tile's loads go to a few pages of memory instead of one a row.  Element (row, c):
template <typename T> struct Blocked {
    static constexpr int CT = ROW / (int)sizeof(T);
    T *p;
    int ktiles;            // tiles of a row
    __device__ __forceinline__ T *at(uint32_t row, uint32_t c) const { return p + ((int64_t)(row >> 8) * ktiles + c / CT) * (256 * CT) + ((row & 255) * CT + c % CT); }
    Operand operand(int rows) const { return Operand{p, ROW, (int64_t)ktiles * 256 * ROW, rows, ktiles * (ROW / 16), 256 * ROW, (uint32_t)(ktiles - 1) * (256 * ROW) + ROW}; }
};
enum { LIMIT_NONE = 0, LIMIT_N = 1, LIMIT_C = 2 };
struct Args {
    Operand a, b;
    const int *count;   // device-side extent of n (LIMIT_N) or of the contraction in elements (LIMIT_C)
    int limit;
    int tiles_m, tiles_n, splits;
    int ktiles;         // tiles of the contraction, over all splits
};

// where a wave's part of a tile lies: element r of acc[i][j] is row m0 + 16 i + r, column n0 + 16 j
struct Geom {
    int m0, n0;         // with the lane's own share: m0 includes 4 (lane >> 4), n0 includes lane & 15
    int tile_m, tile_n, split, wm, wn, lane, tid;
};

// An epilogue functor has finish(acc, where, early, shared, st0, st1), with the LDS stages free for its use; what it reads ahead, in
// begin(where, early, shared), is kept in an Early (registers) and a Shared (LDS of its own).
struct None {};

typedef __attribute__((address_space(3))) void lds_void;

// what a row's chunk numbers are xored with to give their slots: 16 consecutive rows' slots of one chunk fill all 64 banks once
__device__ __forceinline__ int swizzle(int row) { return row >> 1 & 7; }

// 16 bytes a lane from rsrc + off into LDS at `lds` (the same for the whole wave) + 16 lane.  Written out, so that the compiler, which cannot
// tell which stage a load is for, does not wait for all of them in front of a read: the waits are walk()'s own.
__device__ __forceinline__ void to_lds(u32x4 rsrc, char *lds, uint32_t off) {
    const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void *)lds);
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"        // m0 is said to be reserved: it is written here and named for that
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(at), "v"(off), "s"(rsrc) : "memory", "m0");
#pragma clang diagnostic pop
}

// TILE_ROWS rows, by NT threads
template <int TILE_ROWS, int NT> struct Loader {
    static constexpr int LPR = ROW / 16;                   // lanes of a row
    static constexpr int PER = TILE_ROWS * LPR / NT;       // 16-byte loads of a thread per tile
    static_assert(NT / LPR % 16 == 0, "a load of the block starts at a row that is a multiple of 16");
    u32x4 rsrc;
    uint32_t off, apart, kstep;   // of the thread's first load; between one load's row and the next one's
    int chunk, chunks;
    __device__ __forceinline__ void init(const Operand &o, int row0, int tid) {
        const int here = min(TILE_ROWS, o.rows - row0);                 // >= 1: the grid covers existing rows only
        const uint64_t at = reinterpret_cast<uint64_t>(o.p) + (row0 >> 8) * o.block + (row0 & 255) * o.ld;
        rsrc = u32x4{(uint32_t)at, (uint32_t)(at >> 32), (uint32_t)((here - 1) * o.ld) + o.width, 0x00020000u};
        kstep = o.kstep;
#pragma unroll
        for (int i = 0; i < 4; ++i) rsrc[i] = __builtin_amdgcn_readfirstlane(rsrc[i]);
        const int row = tid / LPR;
        chunk = (tid & (LPR - 1)) ^ swizzle(row);
        chunks = o.chunks;
        off = (uint32_t)row * (uint32_t)o.ld + chunk * 16;
        apart = (uint32_t)(NT / LPR) * (uint32_t)o.ld;
    }
    // where tile kt's loads start; a chunk behind the row's end is asked for beyond the buffer and reads as zero
    __device__ __forceinline__ uint32_t start(int kt) const { return kt * LPR + chunk < chunks ? off + kt * kstep : 0x80000000u; }
    __device__ __forceinline__ void load(char *lds, int tid, uint32_t start, int i) const { to_lds(rsrc, lds + (i * NT + (tid & ~63)) * 16, start + i * apart); }
};

// vmcnt(n) lgkmcnt(0)
template <int N> __device__ __forceinline__ void wait_loads() {
    static_assert(N < 64, "");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0070);
}

// Tiles in columns of 8 row tiles, so that those in flight on a die share rows of A and B in its L2.
struct Place { int tile_m, tile_n, split; };
__device__ __forceinline__ Place place_at(const Args &g, int id) {
    const int tiles = g.tiles_m * g.tiles_n;
    const int split = id / tiles;
    int in = id - split * tiles;
    const int per = 8 * g.tiles_n, grp = in / per;
    in -= grp * per;
    const int gm = min(8, g.tiles_m - grp * 8);
    return Place{grp * 8 + in % gm, in / gm, split};
}
// consecutive blocks go to the 8 dies in turn: every die gets a contiguous range of tiles
__device__ __forceinline__ Place place_of(const Args &g, int bid, int nblk) {
    const int die = bid & 7, q = nblk >> 3, rest = nblk & 7;
    return place_at(g, die * q + min(die, rest) + (bid >> 3));
}

// A tile's sums, in acc; then use(acc, where), and on to the tile that next(place) gives, if any, whose first loads go out before use() runs
// (which then has to leave the stages alone).  Nothing where the tile lies behind the operand's end.  ST: LDS stages.  meanwhile(where) runs
// while the first loads are on their way: in a small product they and what the consumer reads take longer than the products.
template <typename T, int BM, int BN, int WM, int WN, int ST, typename Next, typename Mid, typename Use>
__device__ __forceinline__ void walk(const Args &g, Place at, char *const (&st)[ST], f32x4 (&acc)[BM / WM / 16][BN / WN / 16], Next &&next, Mid &&meanwhile, Use &&use) {
    constexpr int NT = WM * WN * 64, MI = BM / WM / 16, NJ = BN / WN / 16;
    int kbeg, kend;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wn = wave / WM;
    Loader<BM, NT> la;
    Loader<BN, NT> lb;
    constexpr int LA = Loader<BM, NT>::PER, LOADS = LA + Loader<BN, NT>::PER;

    // A tile is 2 halves of the contraction (64 bytes: one matrix instruction's), a half MI steps: A's fragment i times all NJ of B's.
    // A's fragments are read D steps ahead into a ring of 4 sets of registers, B's a half ahead into the other of 2.
    constexpr int STEPS = 2 * MI, D = MI < 3 ? MI : 3, MEET = STEPS - D;
    static_assert(STEPS % 4 == 0, "the ring's place of a step is the same in every tile");
    const int arow = (wm * (BM / WM) + (lane & 15)) * ROW, brow = BM * ROW + (wn * (BN / WN) + (lane & 15)) * ROW;
    const int sw = swizzle(lane & 15), hi = lane >> 4;
    const int slot0 = (hi ^ sw) * 16, slot1 = ((4 + hi) ^ sw) * 16;      // of the two halves
    u32x4 fa[4], fb[2][NJ];
    auto read_a = [&](const char *from, int s) { fa[s & 3] = *reinterpret_cast<const u32x4 *>(from + arow + (s % MI) * (16 * ROW) + (s < MI ? slot0 : slot1)); };
    auto read_b = [&](const char *from, int half, int j) { fb[half][j] = *reinterpret_cast<const u32x4 *>(from + brow + j * (16 * ROW) + (half ? slot1 : slot0)); };
    uint32_t sa = 0, sb = 0;
    auto starts = [&](int kt) { sa = la.start(kt); sb = lb.start(kt); };
    auto load = [&](char *to, int i) {
        if (i < LA) la.load(to, tid, sa, i);
        else lb.load(to + BM * ROW, tid, sb, i - LA);
    };
    // this wave's loads of the next tile are in LDS and its fragments of this one read (`later` tiles may still be on their way);
    // then all waves'
    auto meet = [&](int later) {
        if (ST == 4 && later >= 2) wait_loads<2 * LOADS>();
        else if (ST == 4 && later >= 1) wait_loads<LOADS>();
        else wait_loads<0>();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // Tile kt.  In front of step MEET all its fragments are in registers or on the way there: behind the barrier there its stage is free
    // and tile kt + ST goes into it, the loads and the reads of the next tile's first fragments between the products of the last D steps.
    // `all`: tiles up to kt + ST exist.
    // the product behind the barrier after which load l goes out: from BEHIND on in the next tile
    constexpr int BEHIND = D * NJ, WINDOW = BEHIND + 2 * NJ;
    constexpr auto place = [](int l) { return (l + 1) * WINDOW / LOADS - 1; };
    constexpr int LATE = [](auto f) { int n = 0; for (int l = 0; l < LOADS; ++l) n += f(l) >= BEHIND; return n; }(place);
    auto run = [&](char *prev, char *cur, char *nxt, int kt, bool all) {
        const bool more = all || kt + 1 < kend, fill = all || kt + ST < kend, late = all || kt - 1 + ST < kend;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int half = s / MI, i = s % MI;
            if (s == MEET && more) {
                meet(all ? ST - 2 : kend - kt - 2);
                starts(kt + ST);
            }
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                acc[i][j] = Elem<T>::mma(fa[s & 3], fb[half][j], acc[i][j], 0);
                __builtin_amdgcn_sched_barrier(0);
                if (s < MEET) {
                    if (late)
#pragma unroll
                        for (int l = 0; l < LOADS; ++l)
                            if (place(l) == BEHIND + s * NJ + j) load(prev, l);
                    if (j == 0) read_a(cur, s + D);
                    // the other half of B: in the first half, spread over its steps
                    if (half == 0)
#pragma unroll
                        for (int b = NJ * (i * NJ + j) / (MI * NJ); b < NJ * (i * NJ + j + 1) / (MI * NJ); ++b) read_b(cur, 1, b);
                } else {
                    const int e = (s - MEET) * NJ + j;
                    if (more) {
                        if (MEET >= MI) {                // (else B's first set is still in use)
#pragma unroll
                            for (int b = NJ * e / BEHIND; b < NJ * (e + 1) / BEHIND; ++b) read_b(nxt, 0, b);
                        }
                        if (j == NJ - 1) read_a(nxt, s + D - STEPS);
                    }
                    if (fill)
#pragma unroll
                        for (int l = 0; l < LOADS; ++l)
                            if (place(l) == e) load(cur, l);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int e = 1; e < Elem<T>::PARTS; ++e)
#pragma unroll
                for (int j = 0; j < NJ; ++j) acc[i][j] = Elem<T>::mma(fa[s & 3], fb[half][j], acc[i][j], e);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    static_assert(MEET >= MI, "the barrier lies in the second half");
    auto aim = [&]() {
        // the number of columns is read while loads are on their way, but where it decides what to load
        int ktiles = g.ktiles;
        if (g.limit == LIMIT_C && g.splits > 1) ktiles = min(ktiles, (int)((*g.count * (int64_t)sizeof(T) + ROW - 1) / ROW));
        kbeg = (int)((int64_t)ktiles * at.split / g.splits);
        kend = (int)((int64_t)ktiles * (at.split + 1) / g.splits);
        la.init(g.a, at.tile_m * BM, tid);
        lb.init(g.b, at.tile_n * BN, tid);
#pragma unroll
        for (int i = 0; i < ST; ++i)
            if (kbeg + i < kend) {
                starts(kbeg + i);
#pragma unroll
                for (int l = 0; l < LOADS; ++l)
                    if (i + 1 < ST || place(l) < BEHIND) load(st[i], l);
            }
    };
    aim();
    const int count = g.limit == LIMIT_NONE ? 0 : *g.count;
    if (g.limit == LIMIT_N && at.tile_n * BN >= count) {
        wait_loads<0>();
        return;
    }
    for (;;) {
        const Geom geo{at.tile_m * BM + wm * (BM / WM) + 4 * hi, at.tile_n * BN + wn * (BN / WN) + (lane & 15), at.tile_m, at.tile_n, at.split, wm, wn, lane, tid};
        meanwhile(geo);
        // (loads of tiles behind the end that the count gives are waited for, and not looked at)
        if (g.limit == LIMIT_C && g.splits == 1) kend = min(kend, (int)((count * (int64_t)sizeof(T) + ROW - 1) / ROW));
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

        if (kbeg < kend) {
            if (kbeg + ST - 1 < kend) wait_loads<(ST - 1) * LOADS - LATE>();
            else wait_loads<0>();
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
#pragma unroll
            for (int j = 0; j < NJ; ++j) read_b(st[0], 0, j);
#pragma unroll
            for (int s = 0; s < D; ++s) read_a(st[0], s);
            __builtin_amdgcn_sched_barrier(0);
            int kt = kbeg;
            for (; kt + 2 * ST <= kend; kt += ST) {
#pragma unroll
                for (int i = 0; i < ST; ++i) run(st[(i + ST - 1) % ST], st[i], st[(i + 1) % ST], kt + i, true);
            }
            for (; kt < kend; kt += ST) {
#pragma unroll
                for (int i = 0; i < ST; ++i)
                    if (kt + i < kend) run(st[(i + ST - 1) % ST], st[i], st[(i + 1) % ST], kt + i, false);
            }
        }
        wait_loads<0>();
        __syncthreads();
        const bool more = next(at);
        if (more) aim();
        use(acc, geo);
        if (!more) return;
    }
}

// (the epilogues take the first two for their own use)
#define NMFX_TN_STAGES(BM, BN, ST)                                                        \
    static_assert(ST == 2 || ST == 4, "meet()'s waits");                                  \
    constexpr int STAGE = (BM + BN) * tn::ROW;                                            \
    __shared__ __attribute__((aligned(1024))) char st0[STAGE];                            \
    __shared__ __attribute__((aligned(1024))) char st1[STAGE];                            \
    __shared__ __attribute__((aligned(1024))) char st2[ST == 4 ? STAGE : 16];             \
    __shared__ __attribute__((aligned(1024))) char st3[ST == 4 ? STAGE : 16];             \
    char *const stages[4] = {st0, st1, st2, st3};                                         \
    char *st[ST];                                                                         \
    _Pragma("unroll") for (int i = 0; i < ST; ++i) st[i] = stages[i];

// (the host pass needs the kernels' stubs only: with the bodies it drops the stubs of all but the first uses)
template <typename T, int BM, int BN, int WM, int WN, int ST, typename Epi>
__global__ __launch_bounds__(WM *WN * 64) void tn_kernel(Args g, Epi epi) {
#ifdef __HIP_DEVICE_COMPILE__
    NMFX_TN_STAGES(BM, BN, ST)
    __shared__ typename Epi::template Shared<BM, BN, WM, WN> sh;
    typename Epi::template Early<BM / WM / 16, BN / WN / 16> early;
    f32x4 acc[BM / WM / 16][BN / WN / 16];
    walk<T, BM, BN, WM, WN, ST>(g, place_of(g, blockIdx.x, gridDim.x), st, acc, [](Place &) { return false; }, [&](const Geom &at) { epi.template begin<BM, BN, WM, WN>(at, early, sh); },
                                [&](auto &sums, const Geom &at) { epi.template finish<BM, BN, WM, WN>(sums, at, early, sh, st0, st1); });
#endif
}

// The same with a block for every compute unit, which takes tile after tile of its die's range: the first loads of a tile pass under the
// epilogue of the one before.  For LIMIT_N, unsplit, and an epilogue that leaves the stages alone.
template <typename T, int BM, int BN, int WM, int WN, int ST, typename Epi>
__global__ __launch_bounds__(WM *WN * 64) void tn_stream_kernel(Args g, Epi epi) {
#ifdef __HIP_DEVICE_COMPILE__
    NMFX_TN_STAGES(BM, BN, ST)
    __shared__ typename Epi::template Shared<BM, BN, WM, WN> sh;
    typename Epi::template Early<BM / WM / 16, BN / WN / 16> early;
    f32x4 acc[BM / WM / 16][BN / WN / 16];
    g.tiles_n = min(g.tiles_n, (*g.count + BN - 1) / BN);
    const int64_t tiles = (int64_t)g.tiles_m * g.tiles_n;
    const int die = blockIdx.x & 7, last = (int)(tiles * (die + 1) / 8), step = gridDim.x / 8;
    int id = (int)(tiles * die / 8) + (blockIdx.x >> 3);
    if (id >= last) return;
    walk<T, BM, BN, WM, WN, ST>(
        g, place_at(g, id), st, acc,
        [&](Place &at) {
            id += step;
            if (id >= last) return false;
            at = place_at(g, id);
            return true;
        },
        [&](const Geom &at) { epi.template begin<BM, BN, WM, WN>(at, early, sh); }, [&](auto &sums, const Geom &at) { epi.template finish<BM, BN, WM, WN>(sums, at, early, sh, st0, st1); });
#endif
}

// The tiles of those columns of tiles that `on` names, dealt out to the blocks one by one: one column's tiles are as many blocks' work.
template <typename T, int BM, int BN, int WM, int WN, int ST, typename Epi>
__global__ __launch_bounds__(WM *WN * 64) void tn_some_kernel(Args g, Epi epi, const int *on) {
#ifdef __HIP_DEVICE_COMPILE__
    int any = 0;
    for (int t = threadIdx.x; t < g.tiles_n; t += WM * WN * 64) any |= on[t];
    if (!__syncthreads_or(any)) return;
    NMFX_TN_STAGES(BM, BN, ST)
    __shared__ typename Epi::template Shared<BM, BN, WM, WN> sh;
    typename Epi::template Early<BM / WM / 16, BN / WN / 16> early;
    f32x4 acc[BM / WM / 16][BN / WN / 16];
    for (int id = blockIdx.x; id < g.tiles_m * g.tiles_n; id += gridDim.x) {
        const int tile_n = id / g.tiles_m;
        if (!on[tile_n]) continue;
        walk<T, BM, BN, WM, WN, ST>(g, Place{id - tile_n * g.tiles_m, tile_n, 0}, st, acc, [](Place &) { return false; }, [&](const Geom &at) { epi.template begin<BM, BN, WM, WN>(at, early, sh); },
                                    [&](auto &sums, const Geom &at) { epi.template finish<BM, BN, WM, WN>(sums, at, early, sh, st0, st1); });
        __syncthreads();
    }
#endif
}

// two products in one launch: the first `first` blocks are one's, those up to `last` the other's; a block behind them runs `more`
template <typename T, int BM, int BN, int WM, int WN, int ST, typename EpiA, typename EpiB, typename More>
__global__ __launch_bounds__(WM *WN * 64) void tn_pair_kernel(Args ga, EpiA ea, Args gb, EpiB eb, int first, int last, More more) {
#ifdef __HIP_DEVICE_COMPILE__
    if ((int)blockIdx.x >= last) {
        more.template run<WM * WN * 64>();
        return;
    }
    NMFX_TN_STAGES(BM, BN, ST)
    None none;
    f32x4 acc[BM / WM / 16][BN / WN / 16];
    const bool is_a = (int)blockIdx.x < first;
    const Args g = is_a ? ga : gb;
    walk<T, BM, BN, WM, WN, ST>(g, place_of(g, blockIdx.x - (is_a ? 0 : first), is_a ? first : last - first), st, acc, [](Place &) { return false; }, [](const Geom &) {},
                                [&](auto &sums, const Geom &at) {
                                    if (is_a) ea.template finish<BM, BN, WM, WN>(sums, at, none, none, st0, st1);
                                    else eb.template finish<BM, BN, WM, WN>(sums, at, none, none, st0, st1);
                                });
#endif
}

}  // namespace tn
}  // namespace nmfx

// tn_gemm.hpp -- D(m, n) = sum_c A(m, c) B(n, c) for operands whose contraction index c is contiguous in memory, with the consumer of D
// as an epilogue functor: the products of the softmax cross entropy (xent.hip) and their gradients, in bf16, f16 and f32, accumulated in
// f32.
//
// Bytes, not elements, are the unit: a row of an LDS tile is 128 bytes = 8 chunks of 16 (64 contraction steps of a 16-bit type, 32 of
// f32), so one address path serves all types.  Chunk c of row r sits in slot c ^ (r & 7) of its row: eight consecutive rows of one
// chunk -- what the eight lanes of one LDS cycle read -- then fall into eight different 16-byte bank groups.  Tiles go from memory to LDS
// without registers (buffer_load ... lds): lane l of a wave's load writes slot l & 7 of row l >> 3, so it fetches chunk (l & 7) ^ (l >> 3);
// eight lanes read one whole 128-byte line.  Both operands see the same order of c inside a tile, so any order is right.
//
// Schedule: two LDS stages, ONE barrier per tile, placed in front of the tile's last quarter of matrix instructions: by then a wave holds
// the fragments of that quarter in registers, so behind the barrier the freed stage is refilled and the first fragments of the next tile
// are read while the matrix unit works through the quarter.  The loads of a tile have a whole tile's matrix time to arrive.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nmfx {
namespace tn {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Elem;
template <> struct Elem<__bf16> {
    static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Elem<_Float16> {
    static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
// f32: a chunk is 4 contraction steps; lanes 0-31 hold chunk 2q, lanes 32-63 chunk 2q + 1, and the e-th of four 32x32x2 instructions
// takes the pair (4 (2q) + e, 4 (2q + 1) + e)
template <> struct Elem<float> {
    static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], c, 0, 0, 0);
        return c;
    }
};

constexpr int ROW = 128;   // bytes of a tile's row

struct Operand {
    const void *p;
    int64_t ld;       // bytes between rows (a multiple of 16; p is 16-byte aligned)
    int rows;         // rows that exist; rows behind them repeat the last one
    int chunks;       // 16-byte chunks of a row that exist; chunks behind them read as zero
};
enum { LIMIT_NONE = 0, LIMIT_N = 1, LIMIT_C = 2 };
struct Args {
    Operand a, b;
    const int *count;   // device-side extent of n (LIMIT_N) or of the contraction in elements (LIMIT_C)
    int limit;
    int tiles_m, tiles_n, splits;
    int ktiles;         // tiles of the contraction, over all splits
};

// where a wave's part of a tile lies: element (i, j, r) of acc is row m0 + 32 i + 8 (r >> 2) + (r & 3), column n0 + 32 j
struct Geom {
    int m0, n0;         // with the lane's own share: m0 includes 4 (lane >> 5), n0 includes lane & 31
    int tile_m, tile_n, split, wm, wn, lane, tid;
};
__device__ __forceinline__ int acc_row(int i, int r) { return 32 * i + 8 * (r >> 2) + (r & 3); }

typedef __attribute__((address_space(3))) void lds_void;

template <int TILE_ROWS, int NT> struct Loader {
    static constexpr int PER = TILE_ROWS * 8 / NT;   // 16-byte loads of a thread per tile
    __amdgpu_buffer_rsrc_t rsrc;
    uint32_t off[PER];
    int chunk, chunks;
    __device__ __forceinline__ void init(const Operand &o, int row0, int tid) {
        const int here = min(TILE_ROWS, o.rows - row0);                 // >= 1: the grid covers existing rows only
        const char *base = static_cast<const char *>(o.p) + (int64_t)row0 * o.ld;
        rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base), 0, (int)((int64_t)(here - 1) * o.ld + (int64_t)o.chunks * 16), 0x00020000);
        const int l = tid & 63;
        chunk = (l & 7) ^ (l >> 3);
        chunks = o.chunks;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int row = (i * NT + (tid & ~63)) / 8 + (l >> 3);
            off[i] = (uint32_t)min(row, here - 1) * (uint32_t)o.ld + chunk * 16;
        }
    }
    __device__ __forceinline__ void load(char *lds, int tid, int kt) const {
        // a chunk behind the row's end is asked for beyond the buffer: such loads return zero
        const bool in = kt * 8 + chunk < chunks;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void *)(lds + (i * NT + (tid & ~63)) * 16), 16, in ? off[i] + kt * ROW : 0x80000000u, 0, 0, 0);
    }
};

template <typename T, int BM, int BN, int WM, int WN, typename Epi>
__global__ __launch_bounds__(WM *WN * 64) void tn_kernel(Args g, Epi epi) {
#ifdef __HIP_DEVICE_COMPILE__   // the host pass needs the kernel's stub only (with the body it drops the stubs of all but the first uses)
    constexpr int NT = WM * WN * 64, MI = BM / WM / 32, NJ = BN / WN / 32, STAGE = (BM + BN) * ROW;
    __shared__ __attribute__((aligned(1024))) char stage0[STAGE];
    __shared__ __attribute__((aligned(1024))) char stage1[STAGE];
    // consecutive blocks go to the 8 dies in turn: give every die a contiguous range of tiles, and walk a range in columns of 8 row
    // tiles, so that the tiles in flight on a die share rows of A and B in its L2
    int bid = blockIdx.x;
    const int nblk = gridDim.x;
    {
        const int die = bid & 7, q = nblk >> 3, rest = nblk & 7;
        bid = die * q + min(die, rest) + (bid >> 3);
    }
    const int tiles = g.tiles_m * g.tiles_n;
    const int split = bid / tiles;
    int in = bid - split * tiles;
    const int per = 8 * g.tiles_n, grp = in / per;
    in -= grp * per;
    const int gm = min(8, g.tiles_m - grp * 8);
    const int tile_m = grp * 8 + in % gm, tile_n = in / gm;
    int ktiles = g.ktiles;
    if (g.limit == LIMIT_N && tile_n * BN >= *g.count) return;
    if (g.limit == LIMIT_C) ktiles = min(ktiles, (int)((*g.count * (int64_t)sizeof(T) + ROW - 1) / ROW));
    const int kbeg = (int)((int64_t)ktiles * split / g.splits), kend = (int)((int64_t)ktiles * (split + 1) / g.splits);

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wn = wave / WM;
    Loader<BM, NT> la;
    Loader<BN, NT> lb;
    la.init(g.a, tile_m * BM, tid);
    lb.init(g.b, tile_n * BN, tid);

    f32x16 acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    // fragment addresses: row (lane & 31) of a 32-row group, chunk 2 q + (lane >> 5)
    const int arow = wm * (BM / WM) + (lane & 31), brow = wn * (BN / WN) + (lane & 31);
    const int sw = lane & 7, hi = lane >> 5;
    u32x4 fa[2][MI], fb[2][NJ];
    auto frags = [&](const char *st, int q, int set) {
        const int slot = ((2 * q + hi) ^ sw) * 16;
#pragma unroll
        for (int i = 0; i < MI; ++i) fa[set][i] = *reinterpret_cast<const u32x4 *>(st + (arow + 32 * i) * ROW + slot);
#pragma unroll
        for (int j = 0; j < NJ; ++j) fb[set][j] = *reinterpret_cast<const u32x4 *>(st + BM * ROW + (brow + 32 * j) * ROW + slot);
    };
    auto mult = [&](int set) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[i][j] = Elem<T>::mma(fa[set][i], fb[set][j], acc[i][j]);
    };
    auto fill = [&](char *st, int kt) {
        la.load(st, tid, kt);
        lb.load(st + BM * ROW, tid, kt);
    };
    // vmcnt(0) lgkmcnt(0): this wave's loads into LDS are there and its fragments read; then all waves'
    auto meet = [&]() {
        __builtin_amdgcn_s_waitcnt(0x0070);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto step = [&](char *cur, char *nxt, int kt) {
        frags(cur, 1, 1);
        __builtin_amdgcn_sched_barrier(0);
        mult(0);
        __builtin_amdgcn_sched_barrier(0);
        frags(cur, 2, 0);
        __builtin_amdgcn_sched_barrier(0);
        mult(1);
        __builtin_amdgcn_sched_barrier(0);
        frags(cur, 3, 1);
        __builtin_amdgcn_sched_barrier(0);
        mult(0);
        __builtin_amdgcn_sched_barrier(0);
        if (kt + 1 < kend) {
            meet();
            if (kt + 2 < kend) fill(cur, kt + 2);
            frags(nxt, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        mult(1);
    };
    if (kbeg < kend) {
        fill(stage0, kbeg);
        meet();
        if (kbeg + 1 < kend) fill(stage1, kbeg + 1);
        frags(stage0, 0, 0);
        int kt = kbeg;
        for (; kt + 1 < kend; kt += 2) {
            step(stage0, stage1, kt);
            step(stage1, stage0, kt + 1);
        }
        if (kt < kend) step(stage0, stage1, kt);
    }
    Geom geo{tile_m * BM + wm * (BM / WM) + 4 * hi, tile_n * BN + wn * (BN / WN) + (lane & 31), tile_m, tile_n, split, wm, wn, lane, tid};
    __syncthreads();
    epi.template finish<BM, BN, WM, WN, MI, NJ>(acc, geo, stage0);
#endif
}

}  // namespace tn
}  // namespace nmfx

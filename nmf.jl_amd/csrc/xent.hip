// xent.hip -- softmax cross entropy with logits z = W H (W p x k, H k x n, one class y_j out of p per column j), its log-sum-exp and its
// gradients, without keeping z:
//     lse_j = log sum_v exp z_vj            l_j = lse_j - (1 - eps) z_{y_j, j} - (eps / p) sum_v z_vj
//     dz_vj = g_j (exp(z_vj - lse_j) - (1 - eps) [v = y_j] - eps / p)
//     dH = W' dz        dW = dz H'
// Columns whose label is the ignored one are taken out first: a list of the others is made on the device, H is copied to a packed image
// in that order, and every later pass runs over the packed columns only (their number never leaves the device: blocks behind it return).
// So ignored columns cost nothing, and what stands in them (infinities, NaN) reaches nothing.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "device_ops.hpp"
#include "tn_gemm.hpp"

namespace nmfx {
namespace xent {

using tn::f32x4;
using tn::Geom;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

struct Info {            // written by select_kernel, read by everything behind it
    int count;           // columns that are not ignored
    float unscale;       // what products with the stored dz are multiplied by
    unsigned ticket;     // combine_kernel's blocks that are done
    int pad;
};
// What is stored of dz, in the type of W and H, is
//     f_j ((exp(z_vj - lse_j) - eps / p) / a - [v = y_j]),   a = 1 - eps (1 where eps > 1/2)
// and the products take unscale = a g / scale (one g for all columns: f_j = scale) or a / scale (a g_j for each: f_j = g_j scale).  The
// label's entry, the largest of its column while the model is unsure, is then -1 up to the column's own f_j: stored as g (p - 1 + eps), its
// rounding was the same for all columns and added up (bf16, eps = 0.1, 612 columns: gradients 2.8e-3 off instead of 1.7e-3).  scale is a
// power of two: 1, but for f16, whose range exp(z - lse) g_j leaves at its lower end.

// ---- columns: which are there, in what order, their labels and factors ------------------------------------------------------------
struct Select {
    const int64_t *labels;
    const float *gout;        // n values (no reduction), one value, or NULL for 1
    const float *lse_given;   // n values or NULL
    int64_t ignore;
    int n, p, reduction, scaled;
    float a;
    Info *info;
    int *idx, *pos, *y;       // packed -> column, column -> packed or -1, packed label (-1: not a class)
    float *f, *lse_c;         // packed: f_j, log-sum-exp
    float *loss, *lse;        // the caller's: zero in ignored columns (loss only without reduction); NULL: not written
    int *counts;              // of 2048 columns each
    float *maxima;
};

// 8 NT columns from t00 on, 8 a thread: column(e) is thread's e-th, so that a wave's loads and ranks are of 64 columns in a row.
template <int NT> struct Columns {
    int64_t lab[8];
    int rank[8];              // among the block's columns that are not ignored; -1: ignored, or none
    int all;                  // of them in the block
    static __device__ __forceinline__ int column(int t00, int e) { return t00 + (threadIdx.x >> 6) * 512 + e * 64 + (threadIdx.x & 63); }
    __device__ __forceinline__ void find(const Select &s, int t00) {
        __shared__ int wsum[NT / 64];
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const unsigned long long below = (1ull << lane) - 1;
#pragma unroll
        for (int e = 0; e < 8; ++e) lab[e] = column(t00, e) < s.n ? s.labels[column(t00, e)] : s.ignore;
        int mine = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const unsigned long long m = __ballot(lab[e] != s.ignore);
            rank[e] = lab[e] != s.ignore ? mine + __popcll(m & below) : -1;
            mine += __popcll(m);
        }
        if (lane == 0) wsum[wave] = mine;
        __syncthreads();
        all = 0;
        int before = 0;
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) {
            before += w < wave ? wsum[w] : 0;
            all += wsum[w];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) rank[e] += rank[e] >= 0 ? before : 0;
    }
};

// how many of the first `upto` columns are not ignored, and the largest |gout| among them, by a block
template <int NT> __device__ __forceinline__ int count_columns(const Select &s, int from, int upto, bool per, float &gmax) {
    __shared__ int sh[NT / 64];
    __shared__ float shm[NT / 64];
    int c = 0;
    for (int t0 = from + threadIdx.x; t0 < upto; t0 += 16 * NT) {       // 16 loads on their way at a time
        int64_t lab[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) lab[e] = t0 + e * NT < upto ? s.labels[t0 + e * NT] : s.ignore;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            c += lab[e] != s.ignore;
            if (per && lab[e] != s.ignore) gmax = fmaxf(gmax, fabsf(s.gout[t0 + e * NT]));
        }
    }
    for (int o = 32; o; o >>= 1) {
        c += __shfl_xor(c, o);
        gmax = fmaxf(gmax, __shfl_xor(gmax, o));
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { sh[threadIdx.x >> 6] = c; shm[threadIdx.x >> 6] = gmax; }
    __syncthreads();
    c = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) { c += sh[w]; gmax = fmaxf(gmax, shm[w]); }
    return c;
}

// The order of the packed columns is that of the columns: block `blk` places 8 NT of them behind those of the blocks in front, which it
// counts itself (up to 4096 columns: a few loads a thread, 23.6 -> 21.4 us for a small call) or finds counted by count_kernel (16384 columns:
// 37.4 -> 33.4 us, 200000: 285 -> 97).
constexpr int SELF = 4096;
template <int NT> __device__ __forceinline__ void select_columns(const Select &s, int blk) {
    if (!s.n) {
        if (threadIdx.x == 0) *s.info = Info{0, 0.f, 0, 0};
        return;
    }
    const int t00 = blk * 8 * NT, tid = threadIdx.x;
    const bool per = s.reduction == NMFX_REDUCE_NONE && s.gout != nullptr, range = per && s.scaled;
    const int blocks = (s.n + 8 * NT - 1) / (8 * NT);
    int base = 0;
    float gmax = 0.f;
    if (s.n > SELF) {
        for (int b = 0; b < blocks; ++b) {
            base += b < blk ? s.counts[b] : 0;
            if (range) gmax = fmaxf(gmax, s.maxima[b]);
        }
    } else {
        if (blk) base = count_columns<NT>(s, 0, t00, range, gmax);
        if (range) count_columns<NT>(s, t00, s.n, true, gmax);
    }
    float scale = 1.f;
    if (s.scaled) {
        // the largest factor becomes at most 2^14: with a >= 1/2 what is stored is below 2^15 and finite in f16, and 2^-28 of it normal
        if (!per) gmax = 1.f;
        if (gmax > 0.f && gmax < __builtin_inff()) {
            int e;
            frexpf(gmax, &e);
            scale = ldexpf(1.f, min(max(14 - e, -100), 100));
        }
    }
    Columns<NT> c;
    c.find(s, t00);
    float g8[8], l8[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int t = min(c.column(t00, e), s.n - 1);
        g8[e] = per ? s.gout[t] : 1.f;
        l8[e] = s.lse_given ? s.lse_given[t] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int t = c.column(t00, e);
        if (t >= s.n) continue;
        s.pos[t] = c.rank[e] >= 0 ? base + c.rank[e] : -1;
        if (c.rank[e] >= 0) {
            const int i = base + c.rank[e];
            const bool bad = c.lab[e] < 0 || c.lab[e] >= s.p;
            s.idx[i] = t;
            s.y[i] = bad ? -1 : (int)c.lab[e];
            if (s.lse_given) s.lse_c[i] = bad ? __builtin_nanf("") : l8[e];
            s.f[i] = g8[e] * scale;
        } else {
            if (s.lse) s.lse[t] = 0.f;
            if (s.loss && s.reduction == NMFX_REDUCE_NONE) s.loss[t] = 0.f;
        }
    }
    const int all = c.all;
    if (tid == 0 && blk == max(blocks, 1) - 1) {
        float g = 1.f;
        if (!per && s.gout) g = s.gout[0];
        if (s.reduction == NMFX_REDUCE_MEAN) g /= (float)max(base + all, 1);
        *s.info = Info{base + all, base + all ? g * s.a / scale : 0.f, 0, 0};      // (of no columns the gradients are zero whatever g is)
    }
}
__global__ __launch_bounds__(256) void count_kernel(Select s) {
    float gmax = 0.f;
    const int c = count_columns<256>(s, blockIdx.x * 2048, min(s.n, (int)(blockIdx.x + 1) * 2048), s.reduction == NMFX_REDUCE_NONE && s.gout != nullptr, gmax);
    if (threadIdx.x == 0) { s.counts[blockIdx.x] = c; s.maxima[blockIdx.x] = gmax; }
}
__global__ __launch_bounds__(256) void select_kernel(Select s) { select_columns<256>(s, blockIdx.x); }

// A patch of a matrix in 16-bit elements in LDS: rows of M elements.  The 16-byte slots of a row are xored with its number, so that 16 lanes
// at one place of 16 rows touch all banks once.  transposed() reads 8 rows of one element, by the LDS' own transposing read: of 16 lanes,
// lane l gives the address of 4 elements of row l / 4 and gets element l of the 4 rows.
template <int M, int WAVES> struct Patch {
    static constexpr int RB = 2 * M, SLOTS = RB / 16, PER = 256 / RB;       // bytes, slots of a row; rows of 256 bytes
    static __device__ __forceinline__ char *of(char *st0, char *st1, int wave, int rows) {
        return (wave < WAVES / 2 ? st0 : st1) + (wave % (WAVES / 2)) * rows * RB;
    }
    static __device__ __forceinline__ int at(int row, int slot) { return row * RB + ((slot ^ (row / PER & (SLOTS - 1))) << 4); }
    // rows row .. row + 7 of element m + (lane & 15), m a multiple of 16
    static __device__ __forceinline__ tn::u32x4 transposed(const char *patch, int row, int m, int lane) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        const int l = lane & 15;
        tn::u32x4 o;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const char *from = patch + at(row + 4 * q + (l >> 2), m / 8 + (l >> 1 & 1)) + (l & 1) * 8;
            const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)from));
            o[2 * q] = v[0];
            o[2 * q + 1] = v[1];
        }
        return o;
    }
};

// ---- packed images ----------------------------------------------------------------------------------------------------------------
// in: element (r, c) at in[r * rs + c * cs]; out1[r * ld1 + c], out2[c * ld2 + r], zero where r or c is behind the end.  64 x 64 tiles:
// 16-byte loads along the contiguous index (at any address), 16-byte stores of that order from registers and of the other one through LDS.
template <typename T> struct Pack {
    const T *in;
    int64_t rs, cs;
    int rows, cols;           // that exist
    T *out1, *out2;           // NULL: not wanted
    int64_t ld1, ld2;
    int rpad1, rpad2, cpad;   // written extent: rows of out1, of out2 (its columns), columns of out1
    int tiles_r, tiles;
};
typedef tn::u32x4 u32x4_any __attribute__((aligned(2)));
template <typename T> __device__ __forceinline__ void pack_tile(const Pack<T> &a, char *tile, const int *from, int rows, int r0, int c0) {
    constexpr int V = 16 / sizeof(T), CH = 64 / V;
    using P = Patch<64, 2>;
    const int tid = threadIdx.x, lane = tid & 63;
    const bool by_row = a.cs == 1;
    // y: the index between the contiguous runs of `in`, x: along them
    const int x0 = by_row ? c0 : r0, y0 = by_row ? r0 : c0, xs = by_row ? a.cols : rows, ys = by_row ? rows : a.cols;
    const int64_t ld = by_row ? a.rs : a.cs;
    T *same = by_row ? a.out1 : a.out2, *turn = by_row ? a.out2 : a.out1;
    const int64_t lds = by_row ? a.ld1 : a.ld2, ldt = by_row ? a.ld2 : a.ld1;
    const int same_x = by_row ? a.cpad : a.rpad2, same_y = by_row ? a.rpad1 : a.cols, turn_x = by_row ? a.cols : a.rpad1, turn_y = by_row ? a.rpad2 : a.cpad;
    float (*tf)[65] = reinterpret_cast<float (*)[65]>(tile);
#pragma unroll
    for (int i = 0; i < 64 * CH / 256; ++i) {
        const int q = i * 256 + tid, y = q / CH, xc = q % CH, x = x0 + xc * V;
        tn::u32x4 v = {0, 0, 0, 0};
        T *e = reinterpret_cast<T *>(&v);
        if (y0 + y < ys) {
            if (by_row || !from) {
                const T *src = a.in + (int64_t)(from ? from[y] : y0 + y) * ld + x;
                if (x + V <= xs) v = *reinterpret_cast<const u32x4_any *>(src);
                else
#pragma unroll
                    for (int u = 0; u < V; ++u)
                        if (x + u < xs) e[u] = src[u];
            } else
#pragma unroll
                for (int u = 0; u < V; ++u)
                    if (x + u < xs) e[u] = a.in[from[xc * V + u] + (int64_t)(y0 + y) * ld];
        }
        if (same && y0 + y < same_y && x < same_x) *reinterpret_cast<tn::u32x4 *>(same + (int64_t)(y0 + y) * lds + x) = v;
        if (turn) {
            if constexpr (sizeof(T) == 2) *reinterpret_cast<tn::u32x4 *>(tile + P::at(y, xc)) = v;
            else
#pragma unroll
                for (int u = 0; u < V; ++u) tf[y][xc * V + u] = (float)e[u];
        }
    }
    if (!turn) return;
    __syncthreads();
    if constexpr (sizeof(T) == 2) {
        const int x = 16 * (tid >> 6) + (lane & 15), rows8 = (lane >> 4) * 8;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const tn::u32x4 v = P::transposed(tile, 32 * h + rows8, 16 * (tid >> 6), lane);
            if (x0 + x < turn_x && y0 + 32 * h + rows8 < turn_y) *reinterpret_cast<tn::u32x4 *>(turn + (int64_t)(x0 + x) * ldt + y0 + 32 * h + rows8) = v;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int q = i * 256 + tid, x = q / 16, y = q % 16 * 4;
            if (x0 + x < turn_x && y0 + y < turn_y) *reinterpret_cast<f32x4 *>(turn + (int64_t)(x0 + x) * ldt + y0 + y) = f32x4{tf[y][x], tf[y + 1][x], tf[y + 2][x], tf[y + 3][x]};
        }
    }
}
// Everything the products read, in one launch: H packed (first blocks), the images of W that its own order does not serve.  Up to
// ONE_ROUND columns every block of H finds its 64 packed columns for itself (a round of 256 threads with 8 labels each: less than a launch; a
// call of 2048 columns 17.5 -> 15.9 us), and the last block leaves the lists; above, select_kernel has made them.  Bound by memory: W' of
// 131072 x 2048 bf16 with 8192 columns of H, 1.2 GB read and written in 257 us, 4.7 TB/s.
constexpr int ONE_ROUND = 2048;
template <typename T> struct Blank {           // zero in the ignored columns of a matrix with contiguous columns
    T *out;
    int64_t ld;
    int k, blocks;            // of 64 columns each
    __device__ __forceinline__ void run(const Select &s, int b) const {
        const int lane = threadIdx.x & 63;
        for (int t = b * 64 + (threadIdx.x >> 6); t < min(s.n, b * 64 + 64); t += 4)
            if (s.labels[t] == s.ignore)
                for (int c = lane; c < k; c += 64) out[t * ld + c] = (T)0.f;
    }
};
template <typename T> __global__ __launch_bounds__(256) void prepare_kernel(Select s, Pack<T> h, Pack<T> w, Blank<T> z) {
    __shared__ __attribute__((aligned(16))) char tile[sizeof(T) == 2 ? 64 * 128 : 64 * 65 * 4];
    __shared__ int from[64];
    int b = blockIdx.x;
    if (b >= h.tiles) {
        b -= h.tiles;
        if (b < w.tiles) pack_tile<T>(w, tile, nullptr, w.rows, (b % w.tiles_r) * 64, (b / w.tiles_r) * 64);
        else if (b < w.tiles + z.blocks) z.run(s, b - w.tiles);
        else select_columns<256>(s, 0);
        return;
    }
    const int r0 = (b % h.tiles_r) * 64, c0 = (b / h.tiles_r) * 64;
    int rows;
    if (s.n <= ONE_ROUND) {
        Columns<256> c;
        c.find(s, 0);
        rows = c.all;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c.rank[e] >= r0 && c.rank[e] < r0 + 64) from[c.rank[e] - r0] = c.column(0, e);
    } else {
        rows = s.info->count;
        if (threadIdx.x < 64 && r0 + (int)threadIdx.x < rows) from[threadIdx.x] = s.idx[r0 + threadIdx.x];
    }
    __syncthreads();
    pack_tile<T>(h, tile, from, rows, r0, c0);
}

// exp(z - r) with one multiply-add and one exp2 a logit: 2^(z log2(e) - x), where x is r log2(e) as it was rounded, is exp(z - r) 2^rest.  rest
// goes into the column's factor: without it exp(z - lse) of logits of 10^8 comes out e^6 and more times too large.  From BIG on rest would leave
// exp2's range: logits are then taken relative to r beforehand, and x = rest = 0 (as for a NaN, and the minus infinity of no logits).
constexpr float BIG = 0x1p26f;
__device__ __forceinline__ bool big(float r) { return !(fabsf(r) < BIG); }
struct Scaled { float x, rest; };
__device__ __forceinline__ Scaled scaled(float r) {
    const float x = big(r) ? 0.f : r * LOG2E;
    return Scaled{x, big(r) ? 0.f : __builtin_fmaf(r, LOG2E, -x)};
}

// Statistics of a set of logits: (reference r, sum of exp(z - r)), r its maximum in most places.  Of two sets: an empty one, or one of minus
// infinities, is (-inf, 0) and changes nothing; a NaN sum is not 0 and goes through.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x);
    return make_float2(m, (a.y != 0.f ? a.y * exp2_((a.x - m) * LOG2E) : 0.f) + (b.y != 0.f ? b.y * exp2_((b.x - m) * LOG2E) : 0.f));
}
// the same where the references are mostly one
__device__ __forceinline__ float2 join_same(float2 a, float2 b) { return a.x == b.x ? make_float2(a.x, a.y + b.y) : join(a, b); }
__device__ __forceinline__ float lse_of(float2 a) { return __builtin_fmaf(log2f(a.y), LN2, a.x); }

// ---- statistics of the logits: rows of D are classes, columns are packed columns ----------------------------------------------------
// Bound by the product where k is long (131072 x 8192, k = 2048: 3.26 ms, 1350 TFLOP/s); where it is short by the exponentials, which go in
// the products' shadow only between blocks (131072 x 16384, k = 256: 1.25 to 1.39 ms on several cards, 790 to 880 TFLOP/s).
struct EpiStats {
    float2 *part;         // [tile_m][npad]: reference and sum over the tile's classes
    float *zsum;          // [tile_m][npad] or NULL
    float *zy;            // packed: the label's logit
    const int *y;
    const int *count;
    int p, v0, npad;      // classes of the piece that exist; its first class
    template <int MI, int NJ> struct Early { int cnt, y[NJ]; };
    template <int BM, int BN, int WM, int WN> struct Shared { float2 s[WM * BN]; float t[WM * BN]; };
    template <int BM, int BN, int WM, int WN, typename E, typename S> __device__ __forceinline__ void begin(const Geom &g, E &early, S &) const {
        early.cnt = *count;
#pragma unroll
        for (int j = 0; j < BN / WN / 16; ++j) early.y[j] = g.n0 + 16 * j < early.cnt ? y[g.n0 + 16 * j] - v0 : -1;
    }
    template <int BM, int BN, int WM, int WN, int MI, int NJ, typename E, typename S>
    __device__ __forceinline__ void finish(f32x4 (&acc)[MI][NJ], const Geom &g, const E &early, S &sh, char *, char *) const {
        float2 *ps = sh.s;                        // [WM][BN]
        float *zs = sh.t;
        if (g.tile_m * BM + BM > p) {
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (g.m0 + 16 * i + r >= p)
#pragma unroll
                        for (int j = 0; j < NJ; ++j) acc[i][j][r] = -__builtin_inff();
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int n = g.n0 + 16 * j, col = g.wn * (BN / WN) + 16 * j + (g.lane & 15);
            if (zsum) {
                float t = 0.f;
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) t += g.m0 + 16 * i + r < p ? acc[i][j][r] : 0.f;
                t += __shfl_xor(t, 16);
                t += __shfl_xor(t, 32);
                if (g.lane < 16) zs[g.wm * BN + col] = t;
            }
            {
                const int d = early.y[j] - g.m0;           // (-1 where there is no column or no class: below every m0)
                if (d >= 0 && d < 16 * MI && (d & 15) < 4) {
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (d == 16 * i + r) zy[n] = acc[i][j][r];
                }
            }
        }
        float mx[NJ];
        bool any = false;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            mx[j] = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx[j] = fmaxf(mx[j], acc[i][j][r]);
            mx[j] = fmaxf(mx[j], __shfl_xor(mx[j], 16));
            mx[j] = fmaxf(mx[j], __shfl_xor(mx[j], 32));
            any |= big(mx[j]);
        }
        if (__any(any)) {
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[i][j][r] -= big(mx[j]) && mx[j] != -__builtin_inff() ? mx[j] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const Scaled ref = scaled(mx[j]);
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) s += exp2_(__builtin_fmaf(acc[i][j][r], LOG2E, -ref.x));
            s += __shfl_xor(s, 16);
            s += __shfl_xor(s, 32);
            if (g.lane < 16) ps[g.wm * BN + g.wn * (BN / WN) + 16 * j + g.lane] = make_float2(mx[j], s * exp2_(-ref.rest));
        }
        __syncthreads();
        if (g.tid < BN) {
            float2 a = ps[g.tid];
            float t = zsum ? zs[g.tid] : 0.f;
#pragma unroll
            for (int w = 1; w < WM; ++w) {
                const float2 b = ps[w * BN + g.tid];
                a = join(a, b);
                if (zsum) t += zs[w * BN + g.tid];
            }
            const int64_t o = (int64_t)g.tile_m * npad + g.tile_n * BN + g.tid;
            part[o] = a;
            if (zsum) zsum[o] = t;
        }
    }
};

// joins the tiles' statistics of a column and finishes it
struct Combine {
    const float2 *part;
    const float *zsum, *zy;
    const int *idx, *y;
    Info *info;
    int tiles, npad, p, reduction;
    float eps;
    float *lse_c, *loss_c, *lse, *loss;
    // tiles slice, slice + step, ...
    __device__ __forceinline__ void some(int i, int slice, int step, float2 &a, float &t) const {
        a = make_float2(-__builtin_inff(), 0.f);
        t = 0.f;
#pragma unroll 4
        for (int k = slice; k < tiles; k += step) {
            a = join(a, part[(int64_t)k * npad + i]);
            if (zsum) t += zsum[(int64_t)k * npad + i];
        }
    }
    __device__ __forceinline__ float finish(int i, float2 a, float t, bool write) const {
        const int lab = y[i];
        const float v = lab < 0 ? __builtin_nanf("") : lse_of(a);     // a label that is no class: the column's loss is NaN
        if (write) {
            float l = v - (1.f - eps) * (lab < 0 ? 0.f : zy[i]);
            if (zsum) l -= eps * (t / (float)p);
            lse_c[i] = v;
            loss_c[i] = l;
            const int col = idx[i];
            if (lse) lse[col] = v;
            if (loss && reduction == NMFX_REDUCE_NONE) loss[col] = l;
        }
        return v;
    }
};

// the losses' sum or mean, by one block: Float64, a fixed order
template <int NT> __device__ __forceinline__ void reduce_losses(const float *loss_c, int cnt, int reduction, float *loss) {
    __shared__ double sh[NT / 64];
    double s = 0.;
    for (int i = threadIdx.x; i < cnt; i += NT) s += (double)loss_c[i];
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < NT / 64; ++w) s += sh[w];
        *loss = (float)(reduction == NMFX_REDUCE_MEAN ? s / (double)max(cnt, 1) : s);
    }
}

struct Losses {          // as a block of another launch
    const float *loss_c;
    const Info *info;
    int reduction;
    float *loss;              // NULL: not wanted
    template <int NT> __device__ __forceinline__ void run() const { reduce_losses<NT>(loss_c, info->count, reduction, loss); }
};

// 256 threads share 2^lc packed columns; the block that is done last adds up the losses.
__global__ __launch_bounds__(256) void combine_kernel(Combine c, int lc, int add) {
    __shared__ float2 ps[256];
    __shared__ float ts[256];
    __shared__ unsigned done;
    const int cols = 1 << lc, step = 256 >> lc, at = threadIdx.x & (cols - 1), slice = threadIdx.x >> lc;
    const int cnt = c.info->count, i = blockIdx.x * cols + at;
    if (blockIdx.x * cols < cnt) {
        float2 a;
        float t;
        c.some(i, slice, step, a, t);
        ps[threadIdx.x] = a;
        ts[threadIdx.x] = t;
        for (int o = step / 2; o; o >>= 1) {
            __syncthreads();
            if (slice < o) {
                ps[threadIdx.x] = join(ps[threadIdx.x], ps[threadIdx.x + (o << lc)]);
                ts[threadIdx.x] += ts[threadIdx.x + (o << lc)];
            }
        }
        if (slice == 0 && i < cnt) c.finish(i, ps[at], ts[at], true);
    }
    if (!add) return;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) done = atomicAdd(&c.info->ticket, 1u);
    __syncthreads();
    if (done != gridDim.x - 1) return;
    __threadfence();
    reduce_losses<256>(c.loss_c, cnt, c.reduction, c.loss);
}

// ---- a few columns (scoring tokens): one pass over W, two launches -----------------------------------------------------------------------
// Up to 16 columns are the 16 columns of a matrix instruction.  H is in LDS, each wave streams 16 rows of W at a time from memory into the
// other operand's registers (no LDS: nobody else reads them) and keeps the running statistics of its rows; ignored columns stay, as zeros.
// Bound by reading W: 200 MB (100003 x 1000, f16) in 35.6 us, 5.6 TB/s.  Against the general way: 49.7 -> 40.6 us a call; 32768 x 512 and one
// column 15.3 -> 12.6 (the call), 16 columns of 50000 x 512 22.5 -> 18.4.
struct Score {
    const void *w, *h;
    int64_t ldw, hrs, hcs;    // bytes between rows of W; elements between components and columns of H
    const int64_t *labels;
    int64_t ignore;
    int p, n, k, steps, per;  // steps: of 4 chunks; per: groups of 16 rows of a wave
    float2 *part;             // [block][16]
    float *zsum, *zy;         // [block][16] or NULL; [16]
};
template <typename T> __global__ __launch_bounds__(512) void score_kernel(Score a) {
#ifdef __HIP_DEVICE_COMPILE__
    extern __shared__ __attribute__((aligned(16))) char hs[];        // [steps][4 chunks][16 columns] of 16 bytes
    __shared__ float2 ps[8][16];
    __shared__ float zs[8][16];
    constexpr int PER = 16 / sizeof(T), U = 8;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, hi = lane >> 4;
    const int chunks = a.k / PER, groups = (a.p + 15) / 16, parts = (a.steps + U - 1) / U;
    // a wave's work: groups of 16 rows, each in parts of U steps; a part's loads go out before the products of the part in front of it
    int g = (blockIdx.x * 8 + wave) * a.per, q = 0;
    const int last = min(groups, g + a.per);
    tn::u32x4 f[2][U];
    auto fetch = [&](int set, int gg, int qq) {
        const char *src = static_cast<const char *>(a.w) + (int64_t)min(gg * 16 + col, a.p - 1) * a.ldw + hi * 16;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            f[set][u] = tn::u32x4{0, 0, 0, 0};
            if ((qq * U + u) * 4 + hi < chunks) f[set][u] = *reinterpret_cast<const tn::u32x4 *>(src + (qq * U + u) * 64);
        }
    };
    if (g < last) fetch(0, g, 0);
    const int64_t lab = col < a.n ? a.labels[col] : a.ignore;
    for (int e = tid; e < a.steps * 64; e += 512) {                  // (e & 15 is col)
        const int chunk = e >> 4;
        tn::u32x4 v = {0, 0, 0, 0};
        T *x = reinterpret_cast<T *>(&v);
        if (lab != a.ignore) {
            const T *src = static_cast<const T *>(a.h) + col * a.hcs + (int64_t)chunk * PER * a.hrs;
            if (a.hrs == 1 && chunk < chunks) v = *reinterpret_cast<const u32x4_any *>(src);
            else
#pragma unroll
                for (int u = 0; u < PER; ++u)
                    if (chunk * PER + u < a.k) x[u] = src[u * a.hrs];
        }
        *reinterpret_cast<tn::u32x4 *>(hs + e * 16) = v;
    }
    __syncthreads();
    float top = -__builtin_inff(), sum = 0.f, zsum = 0.f, fix = 1.f;      // fix: what a group's sum is multiplied by
    Scaled ref = {0.f, 0.f};
    f32x4 z = {0.f, 0.f, 0.f, 0.f};
    auto work = [&](int set) {
        const int gn = q + 1 < parts ? g : g + 1, qn = q + 1 < parts ? q + 1 : 0;
        if (gn < last) fetch(set ^ 1, gn, qn);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (q * U + u < a.steps) {
                const tn::u32x4 b = *reinterpret_cast<const tn::u32x4 *>(hs + ((q * U + u) * 64 + lane) * 16);
#pragma unroll
                for (int e = 0; e < tn::Elem<T>::PARTS; ++e) z = tn::Elem<T>::mma(f[set][u], b, z, e);
            }
        if (qn == 0) {                                               // the group is done
            float mx = -__builtin_inff();
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int v = g * 16 + 4 * hi + r;
                if (v >= a.p) z[r] = -__builtin_inff();
                else if (a.zsum) zsum += z[r];
                if (v == lab) a.zy[col] = z[r];
                mx = fmaxf(mx, z[r]);
            }
            if (mx > top) {
                sum *= sum != 0.f ? exp2_((top - mx) * LOG2E) : 0.f;
                top = mx;
                ref = scaled(top);
                fix = exp2_(-ref.rest);
            }
            if (big(top) && top != -__builtin_inff())
#pragma unroll
                for (int r = 0; r < 4; ++r) z[r] -= top;
            float s = 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) s += exp2_(__builtin_fmaf(z[r], LOG2E, -ref.x));
            sum = __builtin_fmaf(s, fix, sum);
            z = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        g = gn;
        q = qn;
    };
    while (g < last) {
        work(0);
        if (g < last) work(1);
    }
    float2 s = make_float2(top, sum);
#pragma unroll
    for (int o = 16; o < 64; o <<= 1) {
        s = join(s, make_float2(__shfl_xor(s.x, o), __shfl_xor(s.y, o)));
        zsum += __shfl_xor(zsum, o);
    }
    if (lane < 16) { ps[wave][lane] = s; zs[wave][lane] = zsum; }
    __syncthreads();
    if (tid < 16) {
#pragma unroll
        for (int w = 1; w < 8; ++w) { s = join(s, ps[w][tid]); zsum += zs[w][tid]; }
        a.part[blockIdx.x * 16 + tid] = s;
        if (a.zsum) a.zsum[blockIdx.x * 16 + tid] = zsum;
    }
#endif
}
// one block, a wave a column
__global__ __launch_bounds__(1024) void score_join_kernel(Score a, int blocks, float eps, int reduction, float *lse, float *loss) {
    __shared__ float ls[16];
    __shared__ int on[16];
    const int col = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t lab = col < a.n ? a.labels[col] : a.ignore;
    float2 s = make_float2(-__builtin_inff(), 0.f);
    float t = 0.f;
#pragma unroll 4
    for (int b = lane; b < blocks; b += 64) {
        s = join(s, a.part[b * 16 + col]);
        if (a.zsum) t += a.zsum[b * 16 + col];
    }
    for (int o = 32; o; o >>= 1) {
        s = join(s, make_float2(__shfl_xor(s.x, o), __shfl_xor(s.y, o)));
        t += __shfl_xor(t, o);
    }
    if (lane == 0) {
        float v = 0.f, l = 0.f;
        if (lab != a.ignore) {
            const bool bad = lab < 0 || lab >= a.p;
            v = bad ? __builtin_nanf("") : lse_of(s);
            l = v - (1.f - eps) * (bad ? 0.f : a.zy[col]);
            if (a.zsum) l -= eps * (t / (float)a.p);
        }
        if (col < a.n) {
            if (lse) lse[col] = v;
            if (reduction == NMFX_REDUCE_NONE) loss[col] = l;
        }
        ls[col] = l;
        on[col] = lab != a.ignore;
    }
    __syncthreads();
    if (threadIdx.x == 0 && reduction != NMFX_REDUCE_NONE) {
        double sum = 0.;
        int cnt = 0;
        for (int c = 0; c < 16; ++c) { sum += (double)ls[c]; cnt += on[c]; }
        *loss = (float)(reduction == NMFX_REDUCE_MEAN ? sum / (double)max(cnt, 1) : sum);
    }
}

// ---- dz of a piece of the classes, in both orders -----------------------------------------------------------------------------------
// Both gradient products contract an index that has to be contiguous, so dz is written twice: 32768 x 8192, k = 2048: 995 us (1105 TFLOP/s
// with 1.07 GB of stores); 16384 x 16384, k = 256, f16: 353 us, bound by the stores (3.0 TB/s) and the exponentials.  It is rounded to the type of
// W and H there, the one rounding in front of the products: in f32 they would run at an eighth of the rate.  Both images are in blocks
// (tn::Blocked): with padded rows that case took 400 us here and the products that read them 465 instead of 326.
template <typename T> __device__ __forceinline__ T to(float x) { return (T)x; }
constexpr float SUM_MOST = 1e30f;      // of the E of a column

// KEEP (f32): the same images of E = exp(z - r_j) instead, before the log-sum-exp is known, with the tiles' statistics and the labels' logits.
// SOME (f32): dz of the columns that `only` names, the others' entries stay.
template <typename T, bool KEEP = false, bool SOME = false> struct EpiDz {
    tn::Blocked<T> dz, dzt;   // rows are packed columns, rows are classes of the piece
    const float *lse_c, *f;   // KEEP: lse_c is the reference
    const int *y, *count;
    int p, v0;                // classes that exist in the piece; its first class
    float inv, label, off;    // 1 / a, (1 - eps) / a, eps / (a p)
    int few;                  // the tiles' statistics are not joined yet: every block does it for its own columns
    Combine c;
    float2 *part;             // KEEP: [tile_m][npad], as EpiStats'
    float *zy, *zsum;         // KEEP: the labels' logits; [tile_m][npad] or NULL
    const int *only;          // SOME: of every packed column
    // per column: log-sum-exp, factor, label's class in the piece.  The large tile has no registers for them to wait in: it reads them late.
    template <int MI, int NJ> struct Early { int cnt, y[NJ]; float lse[NJ], f[NJ]; };
    template <int BM, int BN, int WM, int WN> struct Shared { float lse[BN], t[WM * WN * 64]; float2 s[WM * WN * 64]; };
    template <int BM, int BN, int WM, int WN, typename E, typename S> __device__ __forceinline__ void begin(const Geom &g, E &early, S &sh) const {
        early.cnt = *count;
        if (few) {
            constexpr int STEP = WM * WN * 64 / BN;
            const int at = g.tid % BN, slice = g.tid / BN, i = g.tile_n * BN + at;
            float2 a;
            float t;
            c.some(i, slice, STEP, a, t);
            sh.s[g.tid] = a;
            sh.t[g.tid] = t;
            __syncthreads();
            if (slice == 0) {
#pragma unroll
                for (int w = 1; w < STEP; ++w) {
                    a = join(a, sh.s[w * BN + at]);
                    t += sh.t[w * BN + at];
                }
                sh.lse[at] = i < early.cnt ? c.finish(i, a, t, g.tile_m == 0) : 0.f;
            }
            __syncthreads();
        }
        if (BM < 256) read<BN, BN / WN / 16>(g, early, sh);
    }
    template <int BN, int NJ, typename E, typename S> __device__ __forceinline__ void read(const Geom &g, E &early, S &sh) const {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int n = g.n0 + 16 * j;
            const bool on = n < early.cnt;
            early.lse[j] = few ? sh.lse[n - g.tile_n * BN] : on ? lse_c[n] : 0.f;
            early.f[j] = KEEP ? 1.f : on ? f[n] : 0.f;
            early.y[j] = on ? y[n] - v0 : -1;
        }
    }
    template <int BM, int BN, int WM, int WN, int MI, int NJ, typename E, typename S>
    __device__ __forceinline__ void finish(f32x4 (&acc)[MI][NJ], const Geom &g, E &early, S &sh, char *st0, char *st1) const {
        typedef T T4 __attribute__((ext_vector_type(4)));
        if (BM == 256) read<BN, NJ>(g, early, sh);
        const int cnt = early.cnt;
        using P = Patch<16 * MI, WM * WN>;
        const int wave = g.tid >> 6;
        char *patch = P::of(st0, st1, wave, 16 * NJ);
        // edge: some of the tile's rows or columns do not exist, and have a zero dz.  Of the columns that do not exist dz is never looked at,
        // dzt up to where the tiles of its contraction end.
        constexpr int CT = tn::ROW / (int)sizeof(T);
        const int ends = (cnt + CT - 1) / CT * CT;
        const bool edge = g.tile_m * BM + BM > p || g.tile_n * BN + BN > cnt;
        auto column = [&](int j, auto at_edge) {
            const int n = g.n0 + 16 * j;
            const bool on = n < cnt;
            if (SOME && (!on || !only[n])) return;
            const Scaled from = scaled(early.lse[j]);
            const float fac = early.f[j], mul = KEEP ? 1.f : fac * inv * exp2_(-from.rest), sub = -fac * off, ref = -from.x;
            float sum = 0.f, zs = 0.f;
            // (a wave's part lies in one block of rows either way, and begins with a tile of them)
            T *const zto = sizeof(T) == 4 ? dz.at(n, g.m0) : nullptr, *const tto = sizeof(T) == 4 ? dzt.at(g.m0, n) : nullptr;
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                T4 o;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float e = exp2_(__builtin_fmaf(acc[i][j][r], LOG2E, ref));
                    const float v = !at_edge || (on && g.m0 + 16 * i + r < p) ? (KEEP ? e : __builtin_fmaf(e, mul, sub)) : 0.f;
                    if (KEEP) {
                        sum += v;
                        if (zsum) zs += !at_edge || g.m0 + 16 * i + r < p ? acc[i][j][r] : 0.f;
                    }
                    o[r] = to<T>(v);
                }
                if constexpr (sizeof(T) == 2) *reinterpret_cast<T4 *>(patch + P::at(16 * j + (g.lane & 15), 2 * i + (g.lane >> 5)) + (g.lane >> 4 & 1) * 8) = o;
                else {
                    if (!at_edge || n < cnt) *reinterpret_cast<T4 *>(zto + i * 16 / CT * (256 * CT) + i * 16 % CT) = o;
                    if (!at_edge || n < ends)
#pragma unroll
                        for (int r = 0; r < 4; ++r) tto[(16 * i + r) * CT] = o[r];
                }
            }
            // the label's entry, where it is this lane's: written once more
            const int d = early.y[j] - g.m0;
            if (early.y[j] >= 0 && d >= 0 && d < 16 * MI && (d & 15) < 4) {
                float z = 0.f;
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) z = d == 16 * i + r ? acc[i][j][r] : z;
                if constexpr (KEEP) zy[n] = z;
                else {
                const T v = to<T>(__builtin_fmaf(exp2_(__builtin_fmaf(z, LOG2E, ref)), mul, sub - fac * label));
                if constexpr (sizeof(T) == 2) *reinterpret_cast<T *>(patch + P::at(16 * j + (g.lane & 15), 2 * (d >> 4) + (g.lane >> 5)) + (g.lane >> 4 & 1) * 8 + (d & 3) * 2) = v;
                else {
                    *dz.at(n, g.m0 + d) = v;
                    *dzt.at(g.m0 + d, n) = v;
                }
                }
            }
            if constexpr (KEEP) {
                sum += __shfl_xor(sum, 16);
                sum += __shfl_xor(sum, 32);
                zs += __shfl_xor(zs, 16);
                zs += __shfl_xor(zs, 32);
                float2 s = make_float2(early.lse[j], sum * exp2_(-from.rest));
                if (!(sum < SUM_MOST) || big(early.lse[j])) {              // (seldom) E is of no use here: the statistics with the maximum for a reference
                    auto there = [&](int i, int r) { return !at_edge || (on && g.m0 + 16 * i + r < p); };
                    float mx = -__builtin_inff();
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, there(i, r) ? acc[i][j][r] : mx);
                    mx = fmaxf(mx, __shfl_xor(mx, 16));
                    mx = fmaxf(mx, __shfl_xor(mx, 32));
                    s = make_float2(mx, 0.f);
                    const float at = mx == -__builtin_inff() ? 0.f : mx;
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s.y += there(i, r) ? exp2_((acc[i][j][r] - at) * LOG2E) : 0.f;
                    s.y += __shfl_xor(s.y, 16);
                    s.y += __shfl_xor(s.y, 32);
                }
                if (g.lane < 16) {
                    sh.s[g.wm * BN + n - g.tile_n * BN] = s;
                    sh.t[g.wm * BN + n - g.tile_n * BN] = zs;
                }
            }
        };
        if (!KEEP) {
            bool any = false;
#pragma unroll
            for (int j = 0; j < NJ; ++j) any |= big(early.lse[j]);
            if (__any(any)) {
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[i][j][r] -= big(early.lse[j]) ? early.lse[j] : 0.f;
            }
        }
        if (edge) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) column(j, std::true_type{});
        } else {
#pragma unroll
            for (int j = 0; j < NJ; ++j) column(j, std::false_type{});
        }
        if constexpr (KEEP) {
            __syncthreads();
            if (g.tid < BN) {
                float2 s = sh.s[g.tid];
                float t = sh.t[g.tid];
#pragma unroll
                for (int w = 1; w < WM; ++w) {
                    s = join_same(s, sh.s[w * BN + g.tid]);
                    t += sh.t[w * BN + g.tid];
                }
                const int64_t o = (int64_t)g.tile_m * c.npad + g.tile_n * BN + g.tid;
                part[o] = s;
                if (zsum) zsum[o] = t;
            }
        }
        if constexpr (sizeof(T) == 2) {
            // from the patch both orders go out in 16-byte stores: its rows as they are, and transposed
            const int m0 = g.m0 - 4 * (g.lane >> 4), n0 = g.n0 - (g.lane & 15);
            T *const zto = dz.at(n0 + g.lane / P::SLOTS, m0 + g.lane % P::SLOTS * 8);
#pragma unroll
            for (int e = 0; e < 16 * NJ * P::SLOTS / 64; ++e) {
                const int at = e * 64 + g.lane, row = at / P::SLOTS, slot = at % P::SLOTS;
                if (!edge || n0 + row < cnt) *reinterpret_cast<tn::u32x4 *>(zto + e * (64 / P::SLOTS) * CT) = *reinterpret_cast<const tn::u32x4 *>(patch + P::at(row, slot));
            }
            const int l = g.lane & 15, rows8 = (g.lane >> 4) * 8;
            T *const tto = dzt.at(m0 + l, n0 + rows8);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int h = 0; h < NJ / 2; ++h)
                    if (!edge || n0 + 32 * h + rows8 < ends) *reinterpret_cast<tn::u32x4 *>(tto + i * 16 * CT + 32 * h) = P::transposed(patch, 32 * h + rows8, 16 * i, g.lane);
        }
    }
};

// ---- E kept from the first pass ---------------------------------------------------------------------------------------------------------
// (Of the last piece of the classes: the first ones' E would have to wait for its sums.)
// dz_j = f_j / S_j (E_vj - S_j (1 - eps) [v = y_j] - S_j eps / p) with E_vj = exp(z_vj - r_j), S_j = sum_v E_vj, whatever r_j is.  With r_j the
// label's logit (or a little less) S_j = exp(l_j): between 1 and 10^30 for every loss that training sees.  So E is written by the pass that sums it, and the
// logits are formed once: the column's factor f_j / S_j goes on dH's result and on H's image for dW.  The other pieces'
// dz are formed to go with that: times S_j / f_j.  What smoothing takes from every entry is taken by a pass over the images (smooth_kernel).
// Where a tile's sum of E leaves its range the tile's statistics take the maximum for a reference, while the logits are in registers, and dz of
// such a column is formed again, its column of tiles by as many blocks (16384 x 2048, k = 512: 855 us, with one such column 979, with nothing
// else 1166; by one block for the whole column of tiles it was 18500).
struct Keep {
    const float2 *part;       // [tile_m][npad]: statistics of all pieces; the reference of the last one's is r_j where its sum is in range
    const float *f, *ref, *zy, *zsum;     // zsum: [tile_m][npad] of all pieces, or NULL
    const int *idx, *y;
    const Info *info;
    float eps, a;
    int p, tiles, v0, npad, reduction, k, per;   // v0: the piece's first class; per: columns of a tile of the product (what is done again)
    float *lse_c, *loss_c, *lse, *loss;
    float *scale, *again_f, *shift;   // of a column: f_j / (a S_j); what its dz is multiplied by where it is formed again; S_j eps / p
    int *again, *only;        // per tile, per column: some column's, the column's sum or factor is out of range
    tn::Blocked<float> dz, dzt;
    int64_t ldn;              // of H's image
};
// f_j / S_j too goes on H's image only where it leaves H's elements normal numbers (of 2^-78 to 2^80): below, the image would lose their last bits
// (f = 10^-30 and losses of 60: dW 3e-33 off where its rounding is 3e-34)
constexpr float FACTOR_LEAST = 0x1p-48f, FACTOR_MOST = 0x1p48f;
// r_j, by a wave a column; and no tile is to be done again
__global__ __launch_bounds__(256) void label_kernel(Keep s, const float *w, int64_t ldw, int chunks, const float *h, int64_t ldh, float *ref, int tiles_n) {
    if (blockIdx.x == 0)
        for (int t = threadIdx.x; t < tiles_n; t += 256) s.again[t] = 0;
    const int i = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (i >= s.info->count) return;
    const int v = s.y[i];
    float d = 0.f, size = 0.f;
    if (v >= 0)
        for (int q = lane; q < chunks; q += 64) {
            const f32x4 a = reinterpret_cast<const f32x4 *>(w + v * ldw)[q], b = reinterpret_cast<const f32x4 *>(h + i * ldh)[q];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                d = __builtin_fmaf(a[u], b[u], d);
                size = __builtin_fmaf(fabsf(a[u]), fabsf(b[u]), size);
            }
        }
    for (int o = 32; o; o >>= 1) {
        d += __shfl_xor(d, o);
        size += __shfl_xor(size, o);
    }
    // not above the label's logit as the product forms it, whose terms are added in another order: so S_j is at least 1.  (Both orders' errors, and
    // that of scaling by log2(e); a few thousandths for ordinary logits.)
    if (lane == 0) ref[i] = d - size * ((4 * chunks + 8) * 0x1p-23f);
}
// joins the tiles' statistics of 2^lc (at least 8) columns, finishes them, puts the label's entry right and scales H's image
__global__ __launch_bounds__(256) void keep_kernel(Keep s, float *ht, int lc) {
    __shared__ float2 ps[256];
    __shared__ float zs[256], by[256];
    const int cols = 1 << lc, step = 256 >> lc, at = threadIdx.x & (cols - 1), slice = threadIdx.x >> lc;
    const int cnt = s.info->count, i0 = blockIdx.x * cols, i = i0 + at;
    if (i0 >= cnt) return;
    float2 a = make_float2(-__builtin_inff(), 0.f);
#pragma unroll 4
    for (int q = slice; q < s.tiles; q += step) a = join_same(a, s.part[(int64_t)q * s.npad + i]);
    float t = 0.f;
    if (s.zsum)
        for (int q = slice; q < s.tiles; q += step) t += s.zsum[(int64_t)q * s.npad + i];
    ps[threadIdx.x] = a;
    zs[threadIdx.x] = t;
    for (int o = step / 2; o; o >>= 1) {
        __syncthreads();
        if (slice < o) {
            ps[threadIdx.x] = join(ps[threadIdx.x], ps[threadIdx.x + (o << lc)]);
            zs[threadIdx.x] += zs[threadIdx.x + (o << lc)];
        }
    }
    if (slice == 0) {
        by[at] = 0.f;
        if (i < cnt) {
            a = ps[at];
            const float r = s.ref[i], f = s.f[i];
            const Scaled from = scaled(r);
            const float sum = a.y * exp2_(__builtin_fmaf(a.x - r, LOG2E, from.rest));      // of E as it is stored
            const int lab = s.y[i];
            const float factor = f / (sum * s.a), size = fabsf(factor);
            const bool good = sum < SUM_MOST && !big(r) && (f == 0.f || !(size < FACTOR_LEAST || (size > FACTOR_MOST && size < __builtin_inff())));
            float v = __builtin_nanf(""), l = v, c = v;
            if (lab >= 0) {
                v = lse_of(a);
                l = v - (1.f - s.eps) * s.zy[i];
                if (s.zsum) l -= s.eps * (zs[at] / (float)s.p);
                c = good ? factor : 1.f;
                if (lab >= s.v0) {
                    const float e = exp2_(__builtin_fmaf(s.zy[i], LOG2E, -from.x)) - sum * (1.f - s.eps);
                    *s.dz.at(i, lab - s.v0) = e;
                    *s.dzt.at(lab - s.v0, i) = e;
                }
            }
            if (!good) s.again[i / s.per] = 1;
            s.only[i] = !good;
            s.lse_c[i] = v;
            s.loss_c[i] = l;
            const int col = s.idx[i];
            if (s.lse) s.lse[col] = v;
            if (s.loss && s.reduction == NMFX_REDUCE_NONE) s.loss[col] = l;
            s.scale[i] = by[at] = c;
            s.again_f[i] = good ? sum * s.a : f;
            if (s.zsum) s.shift[i] = good ? sum * (s.eps / (float)s.p) : 0.f;
        }
    }
    __syncthreads();
    const int chunks = cols / 4;
    for (int e = threadIdx.x; e < s.k * chunks; e += 256) {
        const int c = e / chunks, o = e % chunks * 4;
        f32x4 *x = reinterpret_cast<f32x4 *>(ht + c * s.ldn + i0 + o);
        *x = *x * f32x4{by[o], by[o + 1], by[o + 2], by[o + 3]};
    }
}

// what smoothing takes from every entry of the piece's images, by its column.  Read and written once each: cheaper than the logits again from
// k = 256 or so on.
__global__ __launch_bounds__(256) void smooth_kernel(Keep s, int classes, int64_t chunks) {
    const int cnt = s.info->count;
    for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < 2 * chunks; e += gridDim.x * 256ll) {
        const bool turned = e >= chunks;                  // dzt: rows are classes
        const int64_t q = turned ? e - chunks : e, tile = q >> 11;
        const int kt = turned ? s.dzt.ktiles : s.dz.ktiles, block = (int)(tile / kt);
        const int row = block * 256 + (int)(q >> 3 & 255), c = (int)(tile - (int64_t)block * kt) * 32 + (int)(q & 7) * 4;
        if (row >= (turned ? classes : cnt) || c >= (turned ? cnt : classes)) continue;
        f32x4 *x = reinterpret_cast<f32x4 *>(turned ? s.dzt.p : s.dz.p) + q;
        f32x4 v = *x;
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (c + u < (turned ? cnt : classes)) v[u] -= s.shift[turned ? c + u : row];
        *x = v;
    }
}

// ---- sums of products kept in f32: slot s of [split][n][ld], m contiguous -------------------------------------------------------------
struct EpiSlot {
    float *out;
    int64_t ld, slot;
    int nmax, add;
    template <int MI, int NJ> using Early = tn::None;
    template <int BM, int BN, int WM, int WN> using Shared = tn::None;
    template <int BM, int BN, int WM, int WN> __device__ __forceinline__ void begin(const Geom &, tn::None &, tn::None &) const {}
    template <int BM, int BN, int WM, int WN, int MI, int NJ>
    __device__ __forceinline__ void finish(f32x4 (&acc)[MI][NJ], const Geom &g, tn::None &, tn::None &, char *, char *) const {
        float *base = out + g.split * slot;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int n = g.n0 + 16 * j;
            if (n >= nmax) continue;
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                const int m = g.m0 + 16 * i;
                if (m < ld) {
                    f32x4 *to4 = reinterpret_cast<f32x4 *>(base + (int64_t)n * ld + m);
                    *to4 = add ? acc[i][j] + *to4 : acc[i][j];
                }
            }
        }
    }
};

// up to four results in the caller's type, in one store at whatever address
template <typename T> __device__ __forceinline__ void put4(T *o, f32x4 x, int there) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    typedef T4 T4_any __attribute__((aligned(sizeof(T))));
    T4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = to<T>(x[r]);
    if (there >= 4) *reinterpret_cast<T4_any *>(o) = v;
    else
#pragma unroll
        for (int r = 0; r < 3; ++r)
            if (r < there) o[r] = v[r];
}

// ---- a finished product in the caller's type: element (m, n) at out[m + n * ld] ------------------------------------------------------
template <typename T> struct EpiOut {
    T *out;
    int64_t ld;
    const Info *info;
    int mmax, nmax;
    const int *cols, *count;  // column n goes to column cols[n], for n < *count; or NULL
    const float *scale;       // of column n, or NULL
    template <int MI, int NJ> using Early = tn::None;
    template <int BM, int BN, int WM, int WN> using Shared = tn::None;
    template <int BM, int BN, int WM, int WN> __device__ __forceinline__ void begin(const Geom &, tn::None &, tn::None &) const {}
    template <int BM, int BN, int WM, int WN, int MI, int NJ>
    __device__ __forceinline__ void finish(f32x4 (&acc)[MI][NJ], const Geom &g, tn::None &, tn::None &, char *, char *) const {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            int n = g.n0 + 16 * j;
            if (n >= (cols ? *count : nmax)) continue;
            const float u = info->unscale * (scale ? scale[n] : 1.f);
            if (cols) n = cols[n];
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                const int m = g.m0 + 16 * i;
                put4(out + (int64_t)n * ld + m, acc[i][j] * u, mmax - m);
            }
        }
    }
};

// out(m, n) = unscale * sum over slots, m < mmax; n through pos where given (-1: zero)
template <typename T> struct Join {
    const float *slots;
    int64_t ld, slot;
    int nslots;
    const int *pos;
    const float *scale;       // of a packed column, or NULL
    int mmax, nmax;
    T *out;
    int64_t ms, ns;
    int blocks;
    // 2^lanes threads share four outputs' slots
    int lanes;
    __device__ __forceinline__ void run(int b, float u) const {
        const int mq = (mmax + 3) / 4, part = threadIdx.x & ((1 << lanes) - 1);
        const int64_t total = (int64_t)mq * nmax, threads = blocks * 256ll >> lanes;
        const int inner = ms == 1 ? mq : nmax;                            // of the two indexes the one that neighbouring threads step
        for (int64_t e0 = 0; e0 < total; e0 += threads) {                 // (whole waves stay together: they exchange sums)
            const int64_t e = e0 + ((b * 256ll + threadIdx.x) >> lanes);
            int m = 0, n = 0, from = -1;
            if (e < total) {
                const int o = total >> 32 ? (int)(e / inner) : (int)((uint32_t)e / (uint32_t)inner), i = (int)(e - (int64_t)o * inner);
                n = ms == 1 ? o : i;
                m = (ms == 1 ? i : o) * 4;
                from = pos ? pos[n] : n;
            }
            f32x4 s = {0.f, 0.f, 0.f, 0.f};
            if (from >= 0) {
                const float *p = slots + (int64_t)from * ld + m;
#pragma unroll 4
                for (int q = part; q < nslots; q += 1 << lanes) s += *reinterpret_cast<const f32x4 *>(p + q * slot);
            }
            for (int o = 1; o < 1 << lanes; o <<= 1)
#pragma unroll
                for (int q = 0; q < 4; ++q) s[q] += __shfl_xor(s[q], o);
            if (e < total && part == 0) {
                if (from >= 0) s *= scale ? u * scale[from] : u;            // (a zero stays one whatever u is)
                if (ms == 1) put4(out + m + n * ns, s, mmax - m);
                else
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (m + q < mmax) out[(m + q) * ms + n * ns] = to<T>(s[q]);
            }
        }
    }
};
// (blocks, lanes) of a join: the slots are shared where the outputs alone would not fill the card
struct JoinGrid { int blocks, lanes; };
inline JoinGrid join_grid(int64_t m, int64_t n, int slots) {
    const int64_t quads = (m + 3) / 4 * n;
    int lanes = 0;
    while (lanes < 6 && (2 << lanes) <= slots && (quads << lanes) < 65536) ++lanes;
    return JoinGrid{(int)std::min<int64_t>(((quads << lanes) + 255) / 256, 2048), lanes};
}
// the last launch of a call: dH, dW where it was summed in parts, and the losses' sum
template <typename T> __global__ __launch_bounds__(256) void join_kernel(Join<T> h, Join<T> w, const Info *info, const float *loss_c, int reduction, float *loss) {
    const int b = blockIdx.x;
    if (b < h.blocks) h.run(b, info->unscale);
    else if (b < h.blocks + w.blocks) w.run(b - h.blocks, info->unscale);
    else reduce_losses<256>(loss_c, info->count, reduction, loss);
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------
inline int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

struct Choice { int kind, splits; };   // of a product: its tiles (KINDS) and into how many parts its contraction is split

struct Shape {
    int64_t p, n, k;
    int es;                       // bytes of an element
    int64_t wrs, wcs;             // strides of W
    bool w_rows_direct, w_cols_direct;   // W can be read in place as [class][component], as [component][class]
    int64_t npad, kpad, ppad;     // extents as the images have them
    int64_t ldn, ldp;             // between rows of the images ht, by columns, and wt, by classes: padded (tn_gemm.hpp)
    int64_t piece, pieces;        // classes of a piece (a multiple of 256)
    int64_t ldslot;
    Choice z, h, w;               // the products Z, W' dz, dz H'
    bool w_slots, direct;         // direct: dH need not be summed from slots
    bool keep;                    // E is kept from the first pass
    // workspace offsets
    int64_t o_info, o_counts, o_idx, o_pos, o_y, o_f, o_lse, o_loss, o_zy, o_h, o_ht, o_w, o_wt, o_part, o_zsum, o_ref, o_scale, o_again_f, o_shift, o_again, o_only, o_dz, o_dzt, o_hslot, o_wslot, bytes;
};

constexpr int CUS = 256;

// Tiles of a product.  What a tile of the contraction (128 bytes of it) takes a block, in us: alone on its compute unit (lat: the loads'
// way), and of the matrix unit (mat); how many blocks a compute unit holds.  Measured on bf16 and f32 products that fill the card (mat) or
// a few units (lat).  The large tile reads the least from LDS and memory per matrix instruction; the small ones occupy the card where the
// product is small, and waste less behind its edges.
struct TileKind { int m, n, cap; double lat16, mat16, lat32, mat32; };
constexpr TileKind KINDS[3] = {{256, 256, 1, 1.2, 1.65, 7.6, 7.8}, {128, 128, 2, 0.75, 0.52, 2.0, 2.15}, {64, 64, 2, 0.35, 0.23, 0.67, 0.6}};

// The least estimated time of a product by tiles of one kind, over the numbers of splits; a split adds a slot of m x n floats, written and
// read.
struct Guess { Choice c; double us; };
Guess guess(int kind, int64_t m, int64_t n, int64_t ktiles, int es, bool split) {
    const TileKind &t = KINDS[kind];
    const double lat = es == 2 ? t.lat16 : t.lat32, mat = es == 2 ? t.mat16 : t.mat32;
    const int64_t tiles = ((m + t.m - 1) / t.m) * ((n + t.n - 1) / t.n);
    const int64_t most = split ? std::min<int64_t>(std::max<int64_t>(1, ktiles / 4), std::max<int64_t>(1, t.cap * CUS / tiles)) : 1;
    Guess best{{kind, 1}, 1e30};
    for (int64_t s = 1; s <= most; s = s < most && s * 2 > most ? most : s * 2) {
        const double kt = (double)((ktiles + s - 1) / s);
        const int64_t per = (tiles * s + CUS - 1) / CUS;              // blocks of a compute unit
        const double us = std::max(per * kt * mat, (double)((per + t.cap - 1) / t.cap) * kt * lat) + 2. * (per + t.cap - 1) / t.cap + (s > 1 ? 2. + 8e-6 * s * m * n / 4. : 0.);
        if (us < best.us) best = Guess{{kind, (int)s}, us};
    }
    return best;
}
Guess choose(int64_t m, int64_t n, int64_t ktiles, int es) {
    Guess best{{2, 1}, 1e30};
    for (int k = 0; k < 3; ++k) {
        const Guess g = guess(k, m, n, ktiles, es, false);
        if (g.us < best.us) best = g;
    }
    return best;
}
// The two gradient products: each by the kind that suits it, or both by one kind in one launch; and, where neither is split, without the
// launch that joins the slots (dH then goes straight to its columns).  A launch costs about LAUNCH us, the host's part or the gap it leaves.
constexpr double LAUNCH = 4.;
void choose_two(int64_t hm, int64_t hn, int64_t hk, int64_t wm, int64_t wn, int64_t wk, int es, bool direct, Choice &h, Choice &w) {
    double least = 1e30;
    auto take = [&](const Guess &a, const Guess &b, double more) {
        if (a.us + b.us + more < least) { least = a.us + b.us + more; h = a.c; w = b.c; }
    };
    for (int k = 0; k < 3; ++k) {
        for (int l = 0; l < 3; ++l) take(guess(k, hm, hn, hk, es, true), guess(l, wm, wn, wk, es, true), k == l ? LAUNCH - 2. : 2. * LAUNCH);
        if (direct) take(guess(k, hm, hn, hk, es, false), guess(k, wm, wn, wk, es, false), -2.);
    }
}

// E is kept from the first pass in f32, where a pass over the logits takes longer than this estimate (us) and so more than the two launches
// that come with it: 5000 x 1000, k = 100 (estimate 18): 100 -> 83 us; 2000 x 400, k = 42 (3.3): 33 -> 35 us.  (Not in 16 bits: the rounding of the
// scaled H is not small there, and shows in the rows of dW that are mostly labels: bf16, 32768 x 4096, k = 1024, 1067 -> 894 us, but
// gradients 2.9e-3 off instead of 1.7e-3.)  With smoothing a pass over the images comes on top: 20000 x 3000, k = 256: 1181 -> 1107 us,
// 32768 x 8192, k = 1024: 16.6 -> 13.1 ms (without: 14.4 -> 12.1).
constexpr double KEEP_US = 6.;
constexpr int KEEP_SMOOTHED = 256;

Shape shape_of(const nmfx_dmat &W, const nmfx_dmat &H, bool grad, bool smooth) {
    Shape s{};
    s.p = W.rows; s.k = W.cols; s.n = H.cols;
    s.es = ops::elem_bytes(W.dtype);
    s.wrs = W.rs; s.wcs = W.cs;
    const int64_t per = 16 / s.es, step = 128 / s.es;
    const bool base = (reinterpret_cast<uintptr_t>(W.data) & 15) == 0;
    s.w_rows_direct = base && W.cs == 1 && W.rs % per == 0 && s.k % per == 0;
    s.w_cols_direct = base && W.rs == 1 && W.cs % per == 0 && s.p % per == 0;
    s.npad = up(std::max<int64_t>(s.n, 1), 256);
    s.kpad = up(s.k, step);
    s.ppad = up(s.p, 256);
    // two images of dz of at most 2^28 elements each (or 256 classes), and pieces of one size
    const int64_t most = std::max<int64_t>(256, ((1ll << 28) / s.npad) / 256 * 256);
    s.pieces = (s.ppad + most - 1) / most;
    s.piece = up((s.ppad + s.pieces - 1) / s.pieces, 256);
    s.pieces = (s.ppad + s.piece - 1) / s.piece;
    s.ldslot = up(s.k, 4);
    s.ldn = s.npad + 256 / s.es; s.ldp = s.ppad + 256 / s.es;
    const int64_t n1 = std::max<int64_t>(s.n, 1);
    const int64_t pp = std::min(s.piece, s.p);
    const Guess z = choose(pp, n1, s.kpad / step, s.es);
    s.z = z.c;
    s.keep = grad && W.dtype == NMFX_F32 && z.us > KEEP_US && (!smooth || s.k >= KEEP_SMOOTHED);
    choose_two(s.k, n1, (pp + step - 1) / step, pp, s.k, (n1 + step - 1) / step, s.es, s.pieces == 1, s.h, s.w);
    s.direct = s.pieces == 1 && s.h.splits == 1 && s.w.splits == 1 && s.h.kind == s.w.kind;
    s.w_slots = s.w.splits > 1;
    int64_t at = 0;
    auto take = [&](int64_t b) { const int64_t o = at; at = up(at + b, 256); return o; };
    s.o_info = take(sizeof(Info));
    s.o_counts = take(2 * 4096);       // of 2048 columns each: at most 1024 numbers and 1024 maxima
    s.o_idx = take(s.npad * 4); s.o_pos = take(s.npad * 4); s.o_y = take(s.npad * 4);
    s.o_f = take(s.npad * 4); s.o_lse = take(s.npad * 4); s.o_loss = take(s.npad * 4); s.o_zy = take(s.npad * 4);
    s.o_h = take(s.npad * s.kpad * s.es);
    const int64_t tiles = (s.p + KINDS[s.z.kind].m - 1) / KINDS[s.z.kind].m, parts = std::max<int64_t>(tiles * s.npad, 16 * 4 * CUS);
    s.o_part = take(parts * sizeof(float2));
    s.o_zsum = smooth ? take(parts * 4) : -1;
    s.o_ref = s.o_scale = s.o_again_f = s.o_shift = s.o_again = s.o_only = -1;
    if (s.keep) { s.o_ref = take(s.npad * 4); s.o_scale = take(s.npad * 4); s.o_again_f = take(s.npad * 4); s.o_shift = take(s.npad * 4); s.o_again = take(s.npad / 64 * 4); s.o_only = take(s.npad * 4); }
    s.o_w = s.w_rows_direct ? -1 : take(s.p * s.kpad * s.es);
    s.o_ht = s.o_wt = s.o_dz = s.o_dzt = s.o_hslot = s.o_wslot = -1;
    if (grad) {
        s.o_ht = take(s.k * s.ldn * s.es);
        s.o_wt = s.w_cols_direct ? -1 : take(s.k * s.ldp * s.es);
        s.o_dz = take(s.npad * s.piece * s.es);
        s.o_dzt = take(s.npad * s.piece * s.es);
        s.o_hslot = take((int64_t)s.h.splits * s.npad * s.ldslot * 4);
        if (s.w_slots) s.o_wslot = take((int64_t)s.w.splits * std::max(up(s.piece, 4) * s.k, s.ldslot * s.piece) * 4);
    }
    s.bytes = at;
    return s;
}

inline void grid(tn::Args &a, int64_t m, int64_t n, const Choice &c) {
    a.tiles_m = (int)((m + KINDS[c.kind].m - 1) / KINDS[c.kind].m);
    a.tiles_n = (int)((n + KINDS[c.kind].n - 1) / KINDS[c.kind].n);
    a.splits = c.splits;
}
inline int blocks_of(const tn::Args &a) { return a.tiles_m * a.tiles_n * a.splits; }

template <typename T, typename Epi> void product(tn::Args a, int64_t m, int64_t n, const Choice &c, const Epi &epi, hipStream_t st) {
    grid(a, m, n, c);
    switch (c.kind) {
        case 0: tn::tn_kernel<T, 256, 256, 2, 4, 2, Epi><<<blocks_of(a), 512, 0, st>>>(a, epi); break;
        case 1: tn::tn_kernel<T, 128, 128, 2, 2, 2, Epi><<<blocks_of(a), 256, 0, st>>>(a, epi); break;
        default: tn::tn_kernel<T, 64, 64, 2, 2, 4, Epi><<<blocks_of(a), 256, 0, st>>>(a, epi); break;
    }
    ops::hip_ok(hipGetLastError(), "product");
}
// the large tile, several tiles for every compute unit: their loads pass under one another's epilogues (131072 x 16384, k = 256: 1393 -> 1300 us;
// 512 tiles of k = 1024: 68.5 -> 68.1; from fewer no gain)
template <typename T, typename Epi> void stream(tn::Args a, int64_t m, int64_t n, const Choice &c, const Epi &epi, hipStream_t st) {
    grid(a, m, n, c);
    if (c.kind != 0 || blocks_of(a) < 2 * CUS) return product<T>(a, m, n, c, epi, st);
    tn::tn_stream_kernel<T, 256, 256, 2, 4, 2, Epi><<<CUS, 512, 0, st>>>(a, epi);
    ops::hip_ok(hipGetLastError(), "product");
}
// two products at once where they go by the same kind of tile
template <typename T, typename EA, typename EB>
void products(tn::Args a, int64_t ma, int64_t na, const Choice &ca, const EA &ea, tn::Args b, int64_t mb, int64_t nb, const Choice &cb, const EB &eb, const Losses &more, hipStream_t st) {
    if (ca.kind != cb.kind) {
        product<T>(a, ma, na, ca, ea, st);
        product<T>(b, mb, nb, cb, eb, st);
        return;
    }
    grid(a, ma, na, ca);
    grid(b, mb, nb, cb);
    const int first = blocks_of(a), last = first + blocks_of(b), all = last + (more.loss != nullptr);
    switch (ca.kind) {
        case 0: tn::tn_pair_kernel<T, 256, 256, 2, 4, 2, EA, EB, Losses><<<all, 512, 0, st>>>(a, ea, b, eb, first, last, more); break;
        case 1: tn::tn_pair_kernel<T, 128, 128, 2, 2, 2, EA, EB, Losses><<<all, 256, 0, st>>>(a, ea, b, eb, first, last, more); break;
        default: tn::tn_pair_kernel<T, 64, 64, 2, 2, 4, EA, EB, Losses><<<all, 256, 0, st>>>(a, ea, b, eb, first, last, more); break;
    }
    ops::hip_ok(hipGetLastError(), "products");
}

struct Call {
    nmfx_dmat W, H, dW, dH;
    const int64_t *labels;
    nmfx_xent_opts o;
    const float *gout;
    float *loss, *lse;
    bool grad, lse_given;
    char *ws;
    hipStream_t st;
};

// The short way: few columns, W in an order and alignment that a wave can load fragments from, H small enough for LDS.
constexpr int SCORE_LDS = 65536;
inline bool scored(const Shape &s) { return s.n > 0 && s.n <= 16 && s.w_rows_direct && up(s.k * s.es, 64) * 16 <= SCORE_LDS; }
template <typename T> void score(const Call &c, const Shape &s) {
    // one round of blocks, 2 a compute unit (16 waves of up to 16 loads each), with the same number of groups for every wave
    const int steps = (int)(up(s.k * s.es, 64) / 64), groups = (int)((s.p + 15) / 16), per = (groups + 16 * CUS - 1) / (16 * CUS), blocks = (groups + 8 * per - 1) / (8 * per);
    Score a{c.W.data, c.H.data, s.wrs * s.es, c.H.rs, c.H.cs, c.labels, c.o.ignore_index, (int)s.p, (int)s.n, (int)s.k, steps, per, reinterpret_cast<float2 *>(c.ws + s.o_part),
            s.o_zsum >= 0 ? reinterpret_cast<float *>(c.ws + s.o_zsum) : nullptr, reinterpret_cast<float *>(c.ws + s.o_zy)};
    score_kernel<T><<<blocks, 512, steps * 1024, c.st>>>(a);
    ops::hip_ok(hipGetLastError(), "score");
    score_join_kernel<<<1, 1024, 0, c.st>>>(a, blocks, (float)c.o.label_smoothing, c.o.reduction, c.lse, c.loss);
    ops::hip_ok(hipGetLastError(), "score");
}

// the first pass with E kept, up to the images that the gradient products read
template <typename F, typename I>
void keep_first(const Call &c, const Shape &s, const float *w, int64_t ldw, int wchunks, const tn::Operand &hop, const float *h, float *ht, const tn::Blocked<float> &dz, const tn::Blocked<float> &dzt, const Combine &cb, float a_, float inv, float label, float off, F f32, I i32) {
    const int n = (int)s.n, es = 4, n1 = std::max(n, 1), v0 = (int)((s.pieces - 1) * s.piece), p = (int)s.p - v0, before = v0 / KINDS[s.z.kind].m, kt = (int)(s.kpad * es / 128);
    const int *count = &cb.info->count;
    float2 *part = const_cast<float2 *>(cb.part), *here = part + (int64_t)before * s.npad;      // (a piece is whole tiles)
    float *zsum = const_cast<float *>(cb.zsum), *zhere = zsum ? zsum + (int64_t)before * s.npad : nullptr;
    if (v0) stream<float>(tn::Args{tn::plain(w, ldw * es, v0, wchunks), hop, count, tn::LIMIT_N, 0, 0, 1, kt}, v0, n1, s.z, EpiStats{part, zsum, f32(s.o_zy), i32(s.o_y), count, v0, 0, (int)s.npad}, c.st);
    tn::Args a{tn::plain(w + v0 * ldw, ldw * es, p, wchunks), hop, count, tn::LIMIT_N, 0, 0, 1, kt};
    grid(a, p, n1, s.z);
    const Keep kp{part, f32(s.o_f), f32(s.o_ref), f32(s.o_zy), zsum, i32(s.o_idx), i32(s.o_y), cb.info, cb.eps, a_, (int)s.p, before + a.tiles_m, v0, (int)s.npad, c.o.reduction, (int)s.k, KINDS[s.z.kind].n,
                  f32(s.o_lse), f32(s.o_loss), c.lse, c.loss, f32(s.o_scale), f32(s.o_again_f), f32(s.o_shift), i32(s.o_again), i32(s.o_only), dz, dzt, s.ldn};
    label_kernel<<<(n1 + 3) / 4, 256, 0, c.st>>>(kp, w, ldw, wchunks, h, s.kpad, f32(s.o_ref), a.tiles_n);
    ops::hip_ok(hipGetLastError(), "label");
    product<float>(a, p, n1, s.z, EpiDz<float, true>{dz, dzt, f32(s.o_ref), nullptr, i32(s.o_y), count, p, v0, 1.f, 0.f, 0.f, 0, cb, here, f32(s.o_zy), zhere, nullptr}, c.st);
    int lc = 6;
    while (lc > 3 && (n1 >> lc) < CUS) --lc;
    keep_kernel<<<(n1 + (1 << lc) - 1) >> lc, 256, 0, c.st>>>(kp, ht, lc);
    ops::hip_ok(hipGetLastError(), "keep");
    if (zsum) {
        const int64_t chunks = s.npad * s.piece / 4;
        smooth_kernel<<<(int)std::min<int64_t>(8 * CUS, (chunks + 127) / 128), 256, 0, c.st>>>(kp, p, chunks);
        ops::hip_ok(hipGetLastError(), "smooth");
    }
    // dz of the columns whose sums or factors left the range of E, from logits formed again
    const EpiDz<float, false, true> again{dz, dzt, f32(s.o_lse), f32(s.o_again_f), i32(s.o_y), count, p, v0, inv, label, off, 0, cb, nullptr, nullptr, nullptr, i32(s.o_only)};
    const int blocks = std::min(a.tiles_m * a.tiles_n, KINDS[s.z.kind].cap * CUS);
    switch (s.z.kind) {
        case 0: tn::tn_some_kernel<float, 256, 256, 2, 4, 2, EpiDz<float, false, true>><<<blocks, 512, 0, c.st>>>(a, again, kp.again); break;
        case 1: tn::tn_some_kernel<float, 128, 128, 2, 2, 2, EpiDz<float, false, true>><<<blocks, 256, 0, c.st>>>(a, again, kp.again); break;
        default: tn::tn_some_kernel<float, 64, 64, 2, 2, 4, EpiDz<float, false, true>><<<blocks, 256, 0, c.st>>>(a, again, kp.again); break;
    }
    ops::hip_ok(hipGetLastError(), "again");
}

template <typename T> void run(const Call &c, const Shape &s) {
    if (!c.grad && scored(s)) return score<T>(c, s);
    const int es = sizeof(T), step = 128 / es, per = 16 / es;
    char *ws = c.ws;
    auto f32 = [&](int64_t o) { return reinterpret_cast<float *>(ws + o); };
    auto i32 = [&](int64_t o) { return reinterpret_cast<int *>(ws + o); };
    Info *info = reinterpret_cast<Info *>(ws + s.o_info);
    const int *count = &info->count;
    const float eps = (float)c.o.label_smoothing;
    const double a_ = c.o.label_smoothing > 0.5 ? 1. : 1. - c.o.label_smoothing;
    const int n = (int)s.n, p = (int)s.p, k = (int)s.k;

    Select sel{c.labels, c.grad ? c.gout : nullptr, c.lse_given ? c.lse : nullptr, c.o.ignore_index, n, p, c.o.reduction, c.grad && sizeof(T) == 2 && !std::is_same<T, __bf16>::value,
               (float)a_, info, i32(s.o_idx), i32(s.o_pos), i32(s.o_y), f32(s.o_f), f32(s.o_lse), c.lse_given ? nullptr : c.loss, c.lse_given ? nullptr : c.lse, i32(s.o_counts), f32(s.o_counts + 4096)};
    if (n > ONE_ROUND) {
        if (n > SELF) {
            count_kernel<<<(n + 2047) / 2048, 256, 0, c.st>>>(sel);
            ops::hip_ok(hipGetLastError(), "count");
        }
        select_kernel<<<(n + 2047) / 2048, 256, 0, c.st>>>(sel);
        ops::hip_ok(hipGetLastError(), "select");
    }

    T *h = reinterpret_cast<T *>(ws + s.o_h), *ht = c.grad ? reinterpret_cast<T *>(ws + s.o_ht) : nullptr;
    T *pw = s.o_w >= 0 ? reinterpret_cast<T *>(ws + s.o_w) : nullptr, *pwt = s.o_wt >= 0 ? reinterpret_cast<T *>(ws + s.o_wt) : nullptr;
    const T *w = static_cast<const T *>(c.W.data), *wt = w;
    const int ct = (int)(s.kpad / 64 + (s.kpad % 64 != 0)), wr = pw || pwt ? (int)(s.ppad / 64) : 0;
    Pack<T> ph{static_cast<const T *>(c.H.data), c.H.cs, c.H.rs, n, k, h, ht, s.kpad, s.ldn, (int)s.npad, (int)s.npad, (int)s.kpad, (int)(s.npad / 64), (int)(s.npad / 64) * ct};
    Pack<T> pk{w, s.wrs, s.wcs, p, k, pw, pwt, s.kpad, s.ldp, p, (int)s.ppad, (int)s.kpad, wr, wr * ct};
    const bool direct = c.grad && s.direct && c.dH.rs == 1;
    const Blank<T> blank{static_cast<T *>(c.dH.data), c.dH.cs, k, direct ? (n + 63) / 64 : 0};
    prepare_kernel<T><<<ph.tiles + pk.tiles + blank.blocks + (n <= ONE_ROUND), 256, 0, c.st>>>(sel, ph, pk, blank);
    ops::hip_ok(hipGetLastError(), "prepare");
    int64_t ldw = s.wrs, ldwt = s.wcs;
    int wchunks = (int)(s.k / per), wtpad = p;
    if (pw) { w = pw; ldw = s.kpad; wchunks = (int)(s.kpad / per); }
    if (pwt) { wt = pwt; ldwt = s.ldp; wtpad = (int)s.ppad; }

    const int kt = (int)(s.kpad / step), n1 = std::max(n, 1), tiles = (p + KINDS[s.z.kind].m - 1) / KINDS[s.z.kind].m;
    const tn::Operand hop = tn::plain(h, s.kpad * es, (int)s.npad, (int)(s.kpad / per));
    const Combine cb{reinterpret_cast<float2 *>(ws + s.o_part), s.o_zsum >= 0 ? f32(s.o_zsum) : nullptr, f32(s.o_zy), i32(s.o_idx), i32(s.o_y), info, tiles, (int)s.npad, p,
                     c.o.reduction, eps, f32(s.o_lse), f32(s.o_loss), c.lse, c.loss};
    // dz's blocks join the tiles' statistics of their columns themselves where that is a few of them: less than a launch (17 tiles, 83 columns:
    // 27.0 -> 25.3 us a call; 32 tiles, 200 columns: 30.5 -> 28.6; 63 tiles, 1000 columns: 61 -> 67, left to combine_kernel)
    const bool keep = s.keep && !c.lse_given;
    const bool few = c.grad && !c.lse_given && !keep && s.pieces == 1 && tiles <= 32 && (int64_t)tiles * ((n1 + KINDS[s.z.kind].n - 1) / KINDS[s.z.kind].n) <= 2 * CUS;
    const tn::Blocked<T> dz{c.grad ? reinterpret_cast<T *>(ws + s.o_dz) : nullptr, (int)(s.piece / step)}, dzt{c.grad ? reinterpret_cast<T *>(ws + s.o_dzt) : nullptr, (int)(s.npad / step)};
    const float inv = (float)(1. / a_), label = (float)((1. - c.o.label_smoothing) / a_), off = (float)(c.o.label_smoothing / (a_ * p));
    if (keep) {
        if constexpr (std::is_same<T, float>::value) keep_first(c, s, w, ldw, wchunks, hop, h, ht, dz, dzt, cb, (float)a_, inv, label, off, f32, i32);
    } else if (!c.lse_given) {
        tn::Args a{tn::plain(w, ldw * es, p, wchunks), hop, count, tn::LIMIT_N, 0, 0, 1, kt};
        stream<T>(a, p, n1, s.z, EpiStats{reinterpret_cast<float2 *>(ws + s.o_part), s.o_zsum >= 0 ? f32(s.o_zsum) : nullptr, f32(s.o_zy), i32(s.o_y), count, p, 0, (int)s.npad}, c.st);
        if (!few) {
            // as many threads for a column as leave every compute unit a block
            int lc = 6;
            while (lc > 0 && (n1 >> lc) < CUS) --lc;
            combine_kernel<<<(n1 + (1 << lc) - 1) >> lc, 256, 0, c.st>>>(cb, lc, !c.grad && c.o.reduction != NMFX_REDUCE_NONE);
            ops::hip_ok(hipGetLastError(), "combine");
        }
    }
    if (!c.grad) return;

    const float *scale = keep ? f32(s.o_scale) : nullptr;
    T *dw = static_cast<T *>(c.dW.data), *dh = static_cast<T *>(c.dH.data);
    const bool add = !c.lse_given && c.loss && c.o.reduction != NMFX_REDUCE_NONE;
    for (int64_t t = 0; t < s.pieces; ++t) {
        const int64_t q = keep ? s.pieces - 1 - t : t, v0 = q * s.piece;      // (the piece whose E was kept first)
        const int pv = (int)std::min(s.piece, s.p - v0), pt = (int)up(pv, step);
        const bool last = t + 1 == s.pieces;
        tn::Args a{tn::plain(w + v0 * ldw, ldw * es, pv, wchunks), hop, count, tn::LIMIT_N, 0, 0, 1, kt};
        if (!keep || t)
            product<T>(a, pv, n1, s.z, EpiDz<T>{dz, dzt, f32(s.o_lse), f32(keep ? s.o_again_f : s.o_f), i32(s.o_y), count, pv, (int)v0, inv, label, off, few, cb, nullptr, nullptr, nullptr, nullptr}, c.st);
        // dH: rows are components, columns are packed columns
        tn::Args b{tn::plain(wt + v0, ldwt * es, k, (int)std::min<int64_t>((wtpad - v0) / per, s.piece / per)), dz.operand((int)s.npad), count, tn::LIMIT_N, 0, 0, 0, pt / step};
        const EpiSlot eh{f32(s.o_hslot), s.ldslot, s.npad * s.ldslot, (int)s.npad, t > 0};
        // dW: the contiguous index of dW is the row
        const tn::Operand zop = dzt.operand(pv), top = tn::plain(ht, s.ldn * es, k, (int)(s.npad / per));
        const bool kfast = c.dW.cs == 1;
        T *out = dw + v0 * c.dW.rs;
        const int64_t ldo = kfast ? c.dW.rs : c.dW.cs;
        const int mm = kfast ? k : pv, nn = kfast ? pv : k;
        tn::Args d{kfast ? top : zop, kfast ? zop : top, count, tn::LIMIT_C, 0, 0, 0, (int)(s.npad / step)};
        Join<T> jh{}, jw{};
        const EpiOut<T> ew{out, ldo, info, mm, nn, nullptr, nullptr, nullptr};
        if (direct) {
            products<T>(b, k, n1, s.h, EpiOut<T>{dh, c.dH.cs, info, k, n, i32(s.o_idx), count, scale}, d, mm, nn, s.w, ew, Losses{f32(s.o_loss), info, c.o.reduction, add ? c.loss : nullptr}, c.st);
            return;
        }
        if (s.w_slots) {
            const int64_t ld = up(mm, 4);
            products<T>(b, k, n1, s.h, eh, d, mm, nn, s.w, EpiSlot{f32(s.o_wslot), ld, ld * nn, nn, 0}, Losses{}, c.st);
            const JoinGrid jg = join_grid(mm, nn, s.w.splits);
            jw = Join<T>{f32(s.o_wslot), ld, ld * nn, s.w.splits, nullptr, nullptr, mm, nn, out, 1, ldo, jg.blocks, jg.lanes};
        } else products<T>(b, k, n1, s.h, eh, d, mm, nn, s.w, ew, Losses{}, c.st);
        if (last && n) {
            const JoinGrid jg = join_grid(k, n, s.h.splits);
            jh = Join<T>{f32(s.o_hslot), s.ldslot, s.npad * s.ldslot, s.h.splits, i32(s.o_pos), scale, k, n, dh, c.dH.rs, c.dH.cs, jg.blocks, jg.lanes};
        }
        const int jb = jh.blocks + jw.blocks + (last && add);
        if (jb) {
            join_kernel<T><<<jb, 256, 0, c.st>>>(jh, jw, info, f32(s.o_loss), c.o.reduction, c.loss);
            ops::hip_ok(hipGetLastError(), "join");
        }
    }
}

void check_mat(const nmfx_dmat *m, const char *name) {
    const std::string s(name);
    if (!m) throw ops::OpError{NMFX_ERR_BAD_ARG, s + " is NULL"};
    if (m->reserved != 0) throw ops::OpError{NMFX_ERR_BAD_ARG, s + ".reserved must be 0"};
    if (m->rows < 0 || m->cols < 0) throw ops::OpError{NMFX_ERR_DIM_MISMATCH, s + " has a negative extent"};
    if (!m->data && m->rows && m->cols) throw ops::OpError{NMFX_ERR_BAD_ARG, s + ".data is NULL"};
    const int es = ops::elem_bytes(m->dtype);
    if (!es) throw ops::OpError{NMFX_ERR_BAD_ARG, s + ".dtype is none of NMFX_F32, NMFX_F64, NMFX_BF16, NMFX_F16"};
    if (reinterpret_cast<uintptr_t>(m->data) % es) throw ops::OpError{NMFX_ERR_BAD_ARG, s + ".data is not aligned to its element"};
    // one index contiguous, the other one's elements apart from each other: no overlap, no reversal
    const bool by_row = m->cs == 1 && (m->rs >= m->cols || m->rows <= 1), by_col = m->rs == 1 && (m->cs >= m->rows || m->cols <= 1);
    if (m->rows && m->cols && !by_row && !by_col) throw ops::OpError{NMFX_ERR_BAD_ARG, s + ": one of rs, cs must be 1 and the other at least the extent it steps over"};
}

// a stride over an extent of one says nothing: make both what the kernels take for granted
nmfx_dmat tidy(nmfx_dmat m) {
    const bool by_row = m.cs == 1 && (m.rs >= m.cols || m.rows <= 1);
    if (by_row) { if (m.rows <= 1) m.rs = up(std::max<int64_t>(m.cols, 1), 16); }
    else if (m.cols <= 1) m.cs = up(std::max<int64_t>(m.rows, 1), 16);
    return m;
}

ops::View view_of(const nmfx_dmat &m) {
    const bool by_row = m.cs == 1;
    ops::View v{static_cast<char *>(m.data), by_row ? m.rows : m.cols, by_row ? m.cols : m.rows, by_row ? m.rs : m.cs, ops::elem_bytes(m.dtype), m.dtype};
    if (!m.rows || !m.cols) v.rows = 0;
    else if (v.rows == 1 || v.ld == v.len) v = ops::View{v.p, 1, v.rows * v.len, v.rows * v.len, v.es, v.dtype};
    return v;
}

constexpr int64_t MOST = (1 << 21) - 1024;   // 256 rows of Float32, padded, stay below the 2^31 bytes from which on loads ask for zeros

void check(const nmfx_dmat *W, const nmfx_dmat *H) {
    check_mat(W, "W");
    check_mat(H, "H");
    ops::require(W->dtype == H->dtype, NMFX_ERR_BAD_ARG, "W and H must have one dtype");
    ops::require(W->dtype != NMFX_F64, NMFX_ERR_UNSUPPORTED, "softmax cross entropy takes NMFX_F32, NMFX_BF16 and NMFX_F16");
    ops::require(W->cols == H->rows, NMFX_ERR_DIM_MISMATCH, "W is p x k and H is k x n: their k differ");
    ops::require(W->rows >= 1 && W->cols >= 1, NMFX_ERR_DIM_MISMATCH, "p and k must be positive");
    ops::require(W->rows <= MOST && H->cols <= MOST && W->cols <= MOST / 2, NMFX_ERR_UNSUPPORTED, "p and n may be at most 2^21 - 1024 and k half of that");
    ops::require((W->cs == 1 ? W->rs : W->cs) <= MOST, NMFX_ERR_UNSUPPORTED, "the stride of W may be at most 2^21 - 1024 elements");
}

void check_opts(const nmfx_xent_opts *o) {
    ops::require(o != nullptr, NMFX_ERR_BAD_ARG, "opts is NULL");
    ops::require(o->reserved0 == 0, NMFX_ERR_BAD_ARG, "opts.reserved0 must be 0");
    ops::require(o->reduction >= NMFX_REDUCE_NONE && o->reduction <= NMFX_REDUCE_MEAN, NMFX_ERR_BAD_ARG, "opts.reduction is none of NMFX_REDUCE_NONE, _SUM, _MEAN");
    ops::require(o->label_smoothing >= 0. && o->label_smoothing <= 1., NMFX_ERR_BAD_ARG, "opts.label_smoothing must lie in [0, 1]");
}

void dispatch(const Call &c, const Shape &s) {
    switch (c.W.dtype) {
        case NMFX_F32: run<float>(c, s); break;
        case NMFX_BF16: run<__bf16>(c, s); break;
        default: run<_Float16>(c, s); break;
    }
}

}  // namespace xent
}  // namespace nmfx

using namespace nmfx;

extern "C" {

int nmfx_xent_workspace(const nmfx_dmat *W, const nmfx_dmat *H, const nmfx_xent_opts *opts, int grad, int64_t *bytes) {
    return ops::guarded([&] {
        ops::require(bytes != nullptr, NMFX_ERR_BAD_ARG, "bytes is NULL");
        xent::check(W, H);
        xent::check_opts(opts);
        *bytes = xent::shape_of(xent::tidy(*W), xent::tidy(*H), grad != 0, opts->label_smoothing != 0.).bytes;
    });
}

int nmfx_xent(const nmfx_dmat *W, const nmfx_dmat *H, const int64_t *labels, const nmfx_xent_opts *opts, float *loss, float *lse, void *workspace,
              int64_t workspace_bytes, int device, void *stream) {
    return ops::guarded([&] {
        xent::check(W, H);
        xent::check_opts(opts);
        ops::require(labels || !H->cols, NMFX_ERR_BAD_ARG, "labels is NULL");
        ops::require(loss || (!H->cols && opts->reduction == NMFX_REDUCE_NONE), NMFX_ERR_BAD_ARG, "loss is NULL");
        xent::Call c{xent::tidy(*W), xent::tidy(*H), {}, {}, labels, *opts, nullptr, loss, lse, false, false, static_cast<char *>(workspace), static_cast<hipStream_t>(stream)};
        const xent::Shape s = xent::shape_of(c.W, c.H, false, opts->label_smoothing != 0.);
        ops::require(workspace && workspace_bytes >= s.bytes, NMFX_ERR_BAD_ARG, "the workspace is smaller than nmfx_xent_workspace says");
        ops::require((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, NMFX_ERR_BAD_ARG, "the workspace must be aligned to 256 bytes");
        ops::OnDevice on(device);
        xent::dispatch(c, s);
    });
}

int nmfx_xent_grad(const nmfx_dmat *W, const nmfx_dmat *H, const int64_t *labels, const nmfx_xent_opts *opts, const float *gout, int lse_given, float *loss,
                   float *lse, const nmfx_dmat *dW, const nmfx_dmat *dH, void *workspace, int64_t workspace_bytes, int device, void *stream) {
    return ops::guarded([&] {
        xent::check(W, H);
        xent::check_opts(opts);
        xent::check_mat(dW, "dW");
        xent::check_mat(dH, "dH");
        ops::require(dW->dtype == W->dtype && dH->dtype == W->dtype, NMFX_ERR_BAD_ARG, "dW and dH must have the dtype of W and H");
        ops::require(dW->rows == W->rows && dW->cols == W->cols, NMFX_ERR_DIM_MISMATCH, "dW must have the shape of W");
        ops::require(dH->rows == H->rows && dH->cols == H->cols, NMFX_ERR_DIM_MISMATCH, "dH must have the shape of H");
        ops::require(labels || !H->cols, NMFX_ERR_BAD_ARG, "labels is NULL");
        ops::require(lse || !H->cols || !lse_given, NMFX_ERR_BAD_ARG, "lse is NULL, yet lse_given is set");
        xent::Call c{xent::tidy(*W), xent::tidy(*H), xent::tidy(*dW), xent::tidy(*dH), labels, *opts, gout, loss, lse, true, lse_given != 0, static_cast<char *>(workspace),
                     static_cast<hipStream_t>(stream)};
        const ops::View w = xent::view_of(c.W), h = xent::view_of(c.H), gw = xent::view_of(c.dW), gh = xent::view_of(c.dH);
        ops::require(!ops::meet(gw, gh) && !ops::meet(gw, w) && !ops::meet(gw, h) && !ops::meet(gh, w) && !ops::meet(gh, h), NMFX_ERR_BAD_ARG, "dW and dH may share no elements with each other, W or H");
        const xent::Shape s = xent::shape_of(c.W, c.H, true, opts->label_smoothing != 0.);
        ops::require(workspace && workspace_bytes >= s.bytes, NMFX_ERR_BAD_ARG, "the workspace is smaller than nmfx_xent_workspace says");
        ops::require((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, NMFX_ERR_BAD_ARG, "the workspace must be aligned to 256 bytes");
        ops::OnDevice on(device);
        xent::dispatch(c, s);
    });
}

}  // extern "C"

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

using tn::f32x16;
using tn::Geom;

constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

struct Info {            // written by select_kernel, read by everything behind it
    int count;           // columns that are not ignored
    float unscale;       // what products with the stored dz are multiplied by
    int pad[2];
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
};
// One block: the order of the packed columns is that of the columns, so it takes a running count.  It is n / 1024 rounds of a ballot
// and a 16-entry sum.
__global__ __launch_bounds__(1024) void select_kernel(Select s) {
    __shared__ int wsum[16];
    __shared__ float wmax[16];
    __shared__ float sh_scale;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int base = 0;
    float gmax = 0.f;
    const bool per = s.reduction == NMFX_REDUCE_NONE && s.gout != nullptr;
    for (int t0 = 0; t0 < s.n; t0 += 1024) {
        const int t = t0 + tid;
        const int64_t lab = t < s.n ? s.labels[t] : s.ignore;
        const bool on = t < s.n && lab != s.ignore;
        const unsigned long long m = __ballot(on);
        if (lane == 0) wsum[wave] = __popcll(m);
        __syncthreads();
        int before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            before += w < wave ? wsum[w] : 0;
            all += wsum[w];
        }
        const int i = base + before + __popcll(m & ((1ull << lane) - 1));
        if (t < s.n) s.pos[t] = on ? i : -1;
        if (on) {
            const bool bad = lab < 0 || lab >= s.p;
            s.idx[i] = t;
            s.y[i] = bad ? -1 : (int)lab;
            if (s.lse_given) s.lse_c[i] = bad ? __builtin_nanf("") : s.lse_given[t];
            if (per) {
                const float g = s.gout[t];
                s.f[i] = g;
                gmax = fmaxf(gmax, fabsf(g));
            }
        } else if (t < s.n) {
            if (s.lse) s.lse[t] = 0.f;
            if (s.loss && s.reduction == NMFX_REDUCE_NONE) s.loss[t] = 0.f;
        }
        base += all;
        __syncthreads();
    }
    float g = 1.f;
    if (!per) {
        if (s.gout) g = s.gout[0];
        if (s.reduction == NMFX_REDUCE_MEAN) g /= (float)max(base, 1);
        gmax = 1.f;
    }
    for (int o = 32; o; o >>= 1) gmax = fmaxf(gmax, __shfl_xor(gmax, o));
    if (lane == 0) wmax[wave] = gmax;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < 16; ++w) gmax = fmaxf(gmax, wmax[w]);
        float scale = 1.f;
        // the largest factor becomes at most 2^14: with a >= 1/2 what is stored is below 2^15 and finite in f16, and 2^-28 of it normal
        if (s.scaled && gmax > 0.f && gmax < __builtin_inff()) {
            int e;
            frexpf(gmax, &e);
            scale = ldexpf(1.f, min(max(14 - e, -100), 100));
        }
        sh_scale = scale;
        *s.info = Info{base, (per ? 1.f : g) * s.a / scale, {0, 0}};
    }
    __syncthreads();
    const float scale = sh_scale;
    for (int i = tid; i < base; i += 1024) s.f[i] = (per ? s.f[i] : 1.f) * scale;
}

// ---- packed images ----------------------------------------------------------------------------------------------------------------
// in: element (r, c) at in[r * rs + c * cs], r through idx where given; out1[r * ld1 + c], out2[c * ld2 + r], zero where r or c is
// behind the end.  64 x 64 tiles through LDS, so that reads follow the contiguous index of `in` and both writes are contiguous.
template <typename T> struct Pack {
    const T *in;
    int64_t rs, cs;
    const int *idx, *count;   // NULL: rows as they are
    int rows, cols;           // that exist (rows: an upper bound where count is given)
    T *out1, *out2;           // NULL: not wanted
    int64_t ld1, ld2;
    int rpad, cpad;           // written extent
};
template <typename T> __global__ __launch_bounds__(256) void pack_kernel(Pack<T> a) {
    __shared__ T tile[64][65];
    const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64, lo = threadIdx.x & 63, up = threadIdx.x >> 6;
    const int rows = a.count ? min(a.rows, *a.count) : a.rows;
    if (a.cs == 1) {
        for (int i = up; i < 64; i += 4) {
            const int r = r0 + i, c = c0 + lo;
            tile[i][lo] = r < rows && c < a.cols ? a.in[(int64_t)(a.idx ? a.idx[r] : r) * a.rs + c] : (T)0.f;
        }
    } else {
        const int r = r0 + lo;
        const T *row = a.in + (r < rows ? (int64_t)(a.idx ? a.idx[r] : r) * a.rs : 0);
        for (int i = up; i < 64; i += 4) {
            const int c = c0 + i;
            tile[lo][i] = r < rows && c < a.cols ? row[(int64_t)c * a.cs] : (T)0.f;
        }
    }
    __syncthreads();
    if (a.out1)
        for (int i = up; i < 64; i += 4)
            if (r0 + i < a.rpad && c0 + lo < a.cpad) a.out1[(int64_t)(r0 + i) * a.ld1 + c0 + lo] = tile[i][lo];
    if (a.out2)
        for (int i = up; i < 64; i += 4)
            if (c0 + i < a.cols && r0 + lo < a.rpad) a.out2[(int64_t)(c0 + i) * a.ld2 + r0 + lo] = tile[lo][i];
}

// (maximum, sum of exp(z - maximum)) of two sets.  An empty set, or one of minus infinities, is (-inf, 0) and changes nothing; a NaN sum
// is not 0 and goes through.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x);
    return make_float2(m, (a.y != 0.f ? a.y * exp2_((a.x - m) * LOG2E) : 0.f) + (b.y != 0.f ? b.y * exp2_((b.x - m) * LOG2E) : 0.f));
}

// ---- statistics of the logits: rows of D are classes, columns are packed columns ----------------------------------------------------
struct EpiStats {
    float2 *part;         // [tile_m][npad]: maximum and sum of exp(z - maximum) over the tile's classes
    float *zsum;          // [tile_m][npad] or NULL
    float *zy;            // packed: the label's logit
    const int *y;
    const int *count;
    int p, npad;
    template <int BM, int BN, int WM, int WN, int MI, int NJ>
    __device__ __forceinline__ void finish(f32x16 (&acc)[MI][NJ], const Geom &g, char *smem) const {
        float2 *ps = reinterpret_cast<float2 *>(smem);                        // [WM][BN]
        float *zs = reinterpret_cast<float *>(smem + sizeof(float2) * WM * BN);
        if (g.tile_m * BM + BM > p) {
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (g.m0 + tn::acc_row(i, r) >= p)
#pragma unroll
                        for (int j = 0; j < NJ; ++j) acc[i][j][r] = -__builtin_inff();
        }
        const int cnt = *count;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int n = g.n0 + 32 * j;
            float mx = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, acc[i][j][r]);
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float ref = mx == -__builtin_inff() ? 0.f : mx;
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) s += exp2_((acc[i][j][r] - ref) * LOG2E);
            s += __shfl_xor(s, 32);
            const int col = g.wn * (BN / WN) + 32 * j + (g.lane & 31);
            if (g.lane < 32) ps[g.wm * BN + col] = make_float2(mx, s);
            if (zsum) {
                float t = 0.f;
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) t += g.m0 + tn::acc_row(i, r) < p ? acc[i][j][r] : 0.f;
                t += __shfl_xor(t, 32);
                if (g.lane < 32) zs[g.wm * BN + col] = t;
            }
            if (n < cnt) {
                const int d = y[n] - g.m0;
                if (d >= 0 && d < 32 * MI) {
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (d == tn::acc_row(i, r)) zy[n] = acc[i][j][r];
                }
            }
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

// joins the tiles' statistics: 64 packed columns a block, 4 waves share the tiles
struct Combine {
    const float2 *part;
    const float *zsum, *zy;
    const int *idx, *y;
    const Info *info;
    int tiles, npad, p, reduction;
    float eps;
    float *lse_c, *loss_c, *lse, *loss;
};
__global__ __launch_bounds__(256) void combine_kernel(Combine c) {
    __shared__ float2 ps[4][64];
    __shared__ float zs[4][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, i = blockIdx.x * 64 + lane, cnt = c.info->count;
    if (blockIdx.x * 64 >= cnt) return;
    float2 a = make_float2(-__builtin_inff(), 0.f);
    float t = 0.f;
    for (int k = w; k < c.tiles; k += 4) {
        const float2 b = c.part[(int64_t)k * c.npad + i];
        a = join(a, b);
        if (c.zsum) t += c.zsum[(int64_t)k * c.npad + i];
    }
    ps[w][lane] = a;
    zs[w][lane] = t;
    __syncthreads();
    if (w || i >= cnt) return;
    for (int q = 1; q < 4; ++q) {
        a = join(a, ps[q][lane]);
        t += zs[q][lane];
    }
    const int y = c.y[i];
    float lse = a.x + logf(a.y);
    if (y < 0) lse = __builtin_nanf("");                        // a label that is no class: the column's loss is NaN
    float l = lse - (1.f - c.eps) * (y < 0 ? 0.f : c.zy[i]);
    if (c.zsum) l -= c.eps * (t / (float)c.p);
    c.lse_c[i] = lse;
    c.loss_c[i] = l;
    const int col = c.idx[i];
    if (c.lse) c.lse[col] = lse;
    if (c.loss && c.reduction == NMFX_REDUCE_NONE) c.loss[col] = l;
}

// one block, Float64, a fixed order
__global__ __launch_bounds__(1024) void reduce_kernel(const float *loss_c, const Info *info, int reduction, float *loss) {
    __shared__ double sh[16];
    double s = 0.;
    const int cnt = info->count;
    for (int i = threadIdx.x; i < cnt; i += 1024) s += (double)loss_c[i];
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) s += sh[w];
        *loss = (float)(reduction == NMFX_REDUCE_MEAN ? s / (double)max(cnt, 1) : s);
    }
}

// ---- dz of a piece of the classes, in both orders -----------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ T to(float x) { return (T)x; }

template <typename T> struct EpiDz {
    T *dz, *dzt;              // [npad][ldc] by packed column, [classes of the piece][npad] by class
    int64_t ldc;
    const float *lse_c, *f;
    const int *y, *count;
    int p, v0, npad;          // classes that exist in the piece; its first class
    float inv, label, off;    // 1 / a, (1 - eps) / a, eps / (a p)
    template <int BM, int BN, int WM, int WN, int MI, int NJ>
    __device__ __forceinline__ void finish(f32x16 (&acc)[MI][NJ], const Geom &g, char *) const {
        typedef T T4 __attribute__((ext_vector_type(4)));
        const int cnt = *count;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int n = g.n0 + 32 * j;
            const bool on = n < cnt;
            const float lse = on ? lse_c[n] : 0.f, fac = on ? f[n] : 0.f;
            const int d = on ? y[n] - v0 - g.m0 : -1;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    T4 o;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int m = tn::acc_row(i, 4 * q + e);
                        const float pr = exp2_((acc[i][j][4 * q + e] - lse) * LOG2E);
                        const float v = fac * (pr * inv - off - (d == m ? label : 0.f));
                        o[e] = to<T>(on && g.m0 + m < p ? v : 0.f);
                        dzt[(int64_t)(g.m0 + m) * npad + n] = o[e];
                    }
                    *reinterpret_cast<T4 *>(dz + (int64_t)n * ldc + g.m0 + tn::acc_row(i, 4 * q)) = o;
                }
        }
    }
};

// ---- sums of products kept in f32: slot s of [split][n][ld], m contiguous -------------------------------------------------------------
struct EpiSlot {
    float *out;
    int64_t ld, slot;
    int nmax, add;
    template <int BM, int BN, int WM, int WN, int MI, int NJ>
    __device__ __forceinline__ void finish(f32x16 (&acc)[MI][NJ], const Geom &g, char *) const {
        typedef float f4 __attribute__((ext_vector_type(4)));
        float *base = out + g.split * slot;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int n = g.n0 + 32 * j;
            if (n >= nmax) continue;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int m = g.m0 + tn::acc_row(i, 4 * q);
                    if (m < ld) {
                        f4 *to4 = reinterpret_cast<f4 *>(base + (int64_t)n * ld + m);
                        f4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                        if (add) v += *to4;
                        *to4 = v;
                    }
                }
        }
    }
};

// ---- a finished product in the caller's type: element (m, n) at out[m + n * ld] ------------------------------------------------------
template <typename T> struct EpiOut {
    T *out;
    int64_t ld;
    const Info *info;
    int mmax, nmax, wide;     // wide: four consecutive m go in one store
    template <int BM, int BN, int WM, int WN, int MI, int NJ>
    __device__ __forceinline__ void finish(f32x16 (&acc)[MI][NJ], const Geom &g, char *) const {
        typedef T T4 __attribute__((ext_vector_type(4)));
        const float u = info->unscale;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int n = g.n0 + 32 * j;
            if (n >= nmax) continue;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int m = g.m0 + tn::acc_row(i, 4 * q);
                    T4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = to<T>(acc[i][j][4 * q + e] * u);
                    T *o = out + (int64_t)n * ld + m;
                    if (wide && m + 3 < mmax) *reinterpret_cast<T4 *>(o) = v;
                    else
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (m + e < mmax) o[e] = v[e];
                }
        }
    }
};

// out(m, n) = unscale * sum over slots, m < mmax; n through pos where given (-1: zero)
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const float *slots, int64_t ld, int64_t slot, int nslots, const Info *info, const int *pos, int mmax, int nmax, T *out,
                                                   int64_t ms, int64_t ns) {
    const int64_t total = (int64_t)mmax * nmax;
    const float u = info->unscale;
    for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < total; e += gridDim.x * 256ll) {
        int m, n;
        if (ms == 1) { n = (int)(e / mmax); m = (int)(e - (int64_t)n * mmax); }
        else { m = (int)(e / nmax); n = (int)(e - (int64_t)m * nmax); }
        const int from = pos ? pos[n] : n;
        float s = 0.f;
        if (from >= 0)
            for (int q = 0; q < nslots; ++q) s += slots[q * slot + (int64_t)from * ld + m];
        out[m * ms + n * ns] = to<T>(s * u);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------
inline int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

struct Shape {
    int64_t p, n, k;
    int es;                       // bytes of an element
    int64_t wrs, wcs;             // strides of W
    bool w_rows_direct, w_cols_direct;   // W can be read in place as [class][component], as [component][class]
    int64_t npad, kpad, ppad;
    int64_t piece, pieces;        // classes of a piece (a multiple of 256)
    int64_t ldslot;
    int hsplits, wsplits;
    bool w_slots;
    // workspace offsets
    int64_t o_info, o_idx, o_pos, o_y, o_f, o_lse, o_loss, o_zy, o_h, o_ht, o_w, o_wt, o_part, o_zsum, o_dz, o_dzt, o_hslot, o_wslot, bytes;
};

constexpr int CUS = 256;

// the 256 x 256 tile reads half as many bytes from LDS and memory per matrix instruction as the 128 x 128 one, but needs as many tiles
// as the card has compute units to occupy them
inline bool big_tiles(int64_t m, int64_t n, int splits) { return m > 128 && n > 128 && ((m + 255) / 256) * ((n + 255) / 256) * splits >= CUS - 56; }

inline int splits_for(int64_t m, int64_t n, int64_t ktiles) {
    const int64_t big = ((m + 255) / 256) * ((n + 255) / 256), small = ((m + 127) / 128) * ((n + 127) / 128);
    // a split shorter than 8 tiles spends more on its sums than on its products
    const int64_t most = std::max<int64_t>(1, ktiles / 8);
    if (m > 128 && n > 128 && big >= 32) return (int)std::min<int64_t>(most, std::max<int64_t>(1, CUS / big));
    return (int)std::min<int64_t>(most, std::max<int64_t>(1, 2 * CUS / small));
}

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
    // two images of dz of at most 512 MiB each, and pieces of one size
    const int64_t most = std::max<int64_t>(256, ((512ll << 20) / (s.npad * s.es)) / 256 * 256);
    s.pieces = (s.ppad + most - 1) / most;
    s.piece = up((s.ppad + s.pieces - 1) / s.pieces, 256);
    s.pieces = (s.ppad + s.piece - 1) / s.piece;
    s.ldslot = up(s.k, 4);
    s.hsplits = splits_for(s.k, s.npad, s.piece / step);
    s.wsplits = splits_for(std::min(s.piece, s.p), s.k, s.npad / step);
    s.w_slots = s.wsplits > 1;
    int64_t at = 0;
    auto take = [&](int64_t b) { const int64_t o = at; at = up(at + b, 256); return o; };
    s.o_info = take(sizeof(Info));
    s.o_idx = take(s.npad * 4); s.o_pos = take(s.npad * 4); s.o_y = take(s.npad * 4);
    s.o_f = take(s.npad * 4); s.o_lse = take(s.npad * 4); s.o_loss = take(s.npad * 4); s.o_zy = take(s.npad * 4);
    s.o_h = take(s.npad * s.kpad * s.es);
    const int64_t tiles = (s.p + 127) / 128;
    s.o_part = take(tiles * s.npad * sizeof(float2));
    s.o_zsum = smooth ? take(tiles * s.npad * 4) : -1;
    s.o_w = s.w_rows_direct ? -1 : take(s.p * s.kpad * s.es);
    s.o_ht = s.o_wt = s.o_dz = s.o_dzt = s.o_hslot = s.o_wslot = -1;
    if (grad) {
        s.o_ht = take(s.k * s.npad * s.es);
        s.o_wt = s.w_cols_direct ? -1 : take(s.k * s.ppad * s.es);
        s.o_dz = take(s.npad * s.piece * s.es);
        s.o_dzt = take(s.npad * s.piece * s.es);
        s.o_hslot = take((int64_t)s.hsplits * s.npad * s.ldslot * 4);
        if (s.w_slots) s.o_wslot = take((int64_t)s.wsplits * std::max(up(s.piece, 4) * s.k, s.ldslot * s.piece) * 4);
    }
    s.bytes = at;
    return s;
}

template <typename T, typename Epi> void product(tn::Args a, int64_t m, int64_t n, const Epi &epi, hipStream_t st) {
    if (big_tiles(m, n, a.splits)) {
        a.tiles_m = (int)((m + 255) / 256); a.tiles_n = (int)((n + 255) / 256);
        tn::tn_kernel<T, 256, 256, 2, 4, Epi><<<a.tiles_m * a.tiles_n * a.splits, 512, 0, st>>>(a, epi);
    } else {
        a.tiles_m = (int)((m + 127) / 128); a.tiles_n = (int)((n + 127) / 128);
        tn::tn_kernel<T, 128, 128, 2, 2, Epi><<<a.tiles_m * a.tiles_n * a.splits, 256, 0, st>>>(a, epi);
    }
    ops::hip_ok(hipGetLastError(), "product");
}

template <typename T> void pack(const Pack<T> &a, hipStream_t st) {
    pack_kernel<T><<<dim3((a.rpad + 63) / 64, (a.cpad + 63) / 64), 256, 0, st>>>(a);
    ops::hip_ok(hipGetLastError(), "pack");
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

template <typename T> void run(const Call &c, const Shape &s) {
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
               (float)a_, info, i32(s.o_idx), i32(s.o_pos), i32(s.o_y), f32(s.o_f), f32(s.o_lse), c.lse_given ? nullptr : c.loss, c.lse_given ? nullptr : c.lse};
    select_kernel<<<1, 1024, 0, c.st>>>(sel);
    ops::hip_ok(hipGetLastError(), "select");

    T *h = reinterpret_cast<T *>(ws + s.o_h), *ht = c.grad ? reinterpret_cast<T *>(ws + s.o_ht) : nullptr;
    pack(Pack<T>{static_cast<const T *>(c.H.data), c.H.cs, c.H.rs, i32(s.o_idx), count, n, k, h, ht, s.kpad, s.npad, (int)s.npad, (int)s.kpad}, c.st);

    const T *w = static_cast<const T *>(c.W.data), *wt = w;
    int64_t ldw = s.wrs, ldwt = s.wcs;
    int wchunks = (int)(s.k / per), wtpad = p;
    if (s.o_w >= 0 || s.o_wt >= 0) {
        T *pw = s.o_w >= 0 ? reinterpret_cast<T *>(ws + s.o_w) : nullptr, *pwt = s.o_wt >= 0 ? reinterpret_cast<T *>(ws + s.o_wt) : nullptr;
        // (rows behind p are written to the transposed image only: the first has none)
        if (pw) { pack(Pack<T>{w, s.wrs, s.wcs, nullptr, nullptr, p, k, pw, nullptr, s.kpad, 0, p, (int)s.kpad}, c.st); }
        if (pwt) { pack(Pack<T>{w, s.wrs, s.wcs, nullptr, nullptr, p, k, nullptr, pwt, 0, s.ppad, (int)s.ppad, (int)s.kpad}, c.st); }
        if (pw) { w = pw; ldw = s.kpad; wchunks = (int)(s.kpad / per); }
        if (pwt) { wt = pwt; ldwt = s.ppad; wtpad = (int)s.ppad; }
    }
    const int kt = (int)(s.kpad / step);
    const tn::Operand hop{h, s.kpad * es, (int)s.npad, (int)(s.kpad / per)};
    if (!c.lse_given) {
        tn::Args a{{w, ldw * es, p, wchunks}, hop, count, tn::LIMIT_N, 0, 0, 1, kt};
        EpiStats e{reinterpret_cast<float2 *>(ws + s.o_part), s.o_zsum >= 0 ? f32(s.o_zsum) : nullptr, f32(s.o_zy), i32(s.o_y), count, p, (int)s.npad};
        product<T>(a, p, std::max(n, 1), e, c.st);
        const bool big = big_tiles(p, std::max(n, 1), 1);
        Combine cb{e.part, e.zsum, e.zy, i32(s.o_idx), i32(s.o_y), info, big ? (p + 255) / 256 : (p + 127) / 128, (int)s.npad, p, c.o.reduction, eps, f32(s.o_lse), f32(s.o_loss), c.lse, c.loss};
        combine_kernel<<<(int)(s.npad / 64), 256, 0, c.st>>>(cb);
        ops::hip_ok(hipGetLastError(), "combine");
        if (c.loss && c.o.reduction != NMFX_REDUCE_NONE) {
            reduce_kernel<<<1, 1024, 0, c.st>>>(f32(s.o_loss), info, c.o.reduction, c.loss);
            ops::hip_ok(hipGetLastError(), "reduce");
        }
    }
    if (!c.grad) return;

    T *dz = reinterpret_cast<T *>(ws + s.o_dz), *dzt = reinterpret_cast<T *>(ws + s.o_dzt);
    T *dw = static_cast<T *>(c.dW.data), *dh = static_cast<T *>(c.dH.data);
    for (int64_t q = 0; q < s.pieces; ++q) {
        const int64_t v0 = q * s.piece;
        const int pv = (int)std::min(s.piece, s.p - v0), pt = (int)up(pv, step);
        tn::Args a{{w + v0 * ldw, ldw * es, pv, wchunks}, hop, count, tn::LIMIT_N, 0, 0, 1, kt};
        product<T>(a, pv, std::max(n, 1), EpiDz<T>{dz, dzt, s.piece, f32(s.o_lse), f32(s.o_f), i32(s.o_y), count, pv, (int)v0, (int)s.npad, (float)(1. / a_), (float)((1. - c.o.label_smoothing) / a_), (float)(c.o.label_smoothing / (a_ * p))}, c.st);
        // dH: rows are components, columns are packed columns
        tn::Args b{{wt + v0, ldwt * es, k, (int)std::min<int64_t>((wtpad - v0) / per, s.piece / per)}, {dz, s.piece * es, (int)s.npad, (int)(s.piece / per)}, count, tn::LIMIT_N, 0, 0, s.hsplits, pt / step};
        product<T>(b, k, std::max(n, 1), EpiSlot{f32(s.o_hslot), s.ldslot, s.npad * s.ldslot, (int)s.npad, q > 0}, c.st);
        // dW: the contiguous index of dW is the row
        const tn::Operand zop{dzt, s.npad * es, pv, (int)(s.npad / per)}, top{ht, s.npad * es, k, (int)(s.npad / per)};
        const bool kfast = c.dW.cs == 1;
        T *out = dw + v0 * c.dW.rs;
        const int64_t ldo = kfast ? c.dW.rs : c.dW.cs;
        const int mm = kfast ? k : pv, nn = kfast ? pv : k;
        tn::Args d{kfast ? top : zop, kfast ? zop : top, count, tn::LIMIT_C, 0, 0, s.wsplits, (int)(s.npad / step)};
        if (s.w_slots) {
            const int64_t ld = up(mm, 4);
            product<T>(d, mm, nn, EpiSlot{f32(s.o_wslot), ld, ld * nn, nn, 0}, c.st);
            const int64_t blocks = std::min<int64_t>(((int64_t)mm * nn + 255) / 256, 8 * CUS);
            join_kernel<T><<<(int)blocks, 256, 0, c.st>>>(f32(s.o_wslot), ld, ld * nn, s.wsplits, info, nullptr, mm, nn, out, 1, ldo);
            ops::hip_ok(hipGetLastError(), "join");
        } else {
            const bool wide = ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & (4 * es - 1)) == 0;
            product<T>(d, mm, nn, EpiOut<T>{out, ldo, info, mm, nn, wide}, c.st);
        }
    }
    if (n > 0) {
        const int64_t blocks = std::min<int64_t>(((int64_t)k * n + 255) / 256, 8 * CUS);
        join_kernel<T><<<(int)blocks, 256, 0, c.st>>>(f32(s.o_hslot), s.ldslot, s.npad * s.ldslot, s.hsplits, info, i32(s.o_pos), k, n, dh, c.dH.rs, c.dH.cs);
        ops::hip_ok(hipGetLastError(), "join");
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

constexpr int64_t MOST = 1 << 21;   // rows of a tile must stay within the 2 GiB that a buffer descriptor spans

void check(const nmfx_dmat *W, const nmfx_dmat *H) {
    check_mat(W, "W");
    check_mat(H, "H");
    ops::require(W->dtype == H->dtype, NMFX_ERR_BAD_ARG, "W and H must have one dtype");
    ops::require(W->dtype != NMFX_F64, NMFX_ERR_UNSUPPORTED, "softmax cross entropy takes NMFX_F32, NMFX_BF16 and NMFX_F16");
    ops::require(W->cols == H->rows, NMFX_ERR_DIM_MISMATCH, "W is p x k and H is k x n: their k differ");
    ops::require(W->rows >= 1 && W->cols >= 1, NMFX_ERR_DIM_MISMATCH, "p and k must be positive");
    ops::require(W->rows <= MOST && H->cols <= MOST && W->cols <= MOST / 2, NMFX_ERR_UNSUPPORTED, "p and n may be at most 2^21 and k at most 2^20");
    ops::require((W->cs == 1 ? W->rs : W->cs) <= MOST, NMFX_ERR_UNSUPPORTED, "the stride of W may be at most 2^21 elements");
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
        const xent::Shape s = xent::shape_of(c.W, c.H, true, opts->label_smoothing != 0.);
        ops::require(workspace && workspace_bytes >= s.bytes, NMFX_ERR_BAD_ARG, "the workspace is smaller than nmfx_xent_workspace says");
        ops::require((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, NMFX_ERR_BAD_ARG, "the workspace must be aligned to 256 bytes");
        ops::OnDevice on(device);
        xent::dispatch(c, s);
    });
}

}  // extern "C"

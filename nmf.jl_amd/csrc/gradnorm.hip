// gradnorm.hip -- the norm over all elements of a list of matrices, sqrt(sum g^2) or max |g|, and clipping by it:
//     coef = min(1, max_norm / (norm + 1e-6)),   out = g * coef
// Two passes over the list: partial sums (a fixed number of blocks, each over a fixed set of chunks: the same list gives the same bits),
// and the scaling, whose every block adds up the partial sums for itself (some thousand doubles from L2: cheaper than a launch in between).
// Squares are summed in Float64: the sum of 10^9 of them loses nothing, and a gradient of 10^30 does not overflow.  (For 16-bit elements
// eight squares summed in Float32 first, where that is safe, were no faster: 416 us either way for 680 MB of bf16, clipped.)  The scaling
// walks the chunks backwards, so that it starts on what the first pass read last and the last-level cache still holds.
// Bound by memory: one read for the norm, one more and a write for the scaling.  Norm of 5.2 GB of f32: 852 us, 6.1 TB/s; 680 MB of bf16:
// the sum 154 us (4.4 TB/s: two conversions an element), the scaling 255 us (5.3 TB/s).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>
#include <vector>

#include "device_ops.hpp"

namespace nmfx {
namespace gradnorm {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));   // 16 bytes at any element's address

constexpr int NT = 256;
constexpr int CHUNK_BYTES = 16384;      // 4 loads of 16 bytes for each of 256 threads
// as many blocks as the card holds at a time (4 and 8 a compute unit, by their registers): their shares are equal, so more would only make a
// second, short round
constexpr int SUM_BLOCKS = 1024, SCALE_BLOCKS = 2048;

// The list travels as kernel arguments (an argument's bytes cost the host about a nanosecond each, a launch with 3.6 KB of them 7 us, one
// with little 2.5: hence 16 bytes an entry, 24 with a result of its own, and a short form of the table).
struct Entry {
    const char *in;
    uint32_t chunk0;        // first chunk
    uint32_t bits;          // elements of the last chunk: 14 bits; dtype: 2; place in Table::s + 1, or 0 where dense: 16
};
struct Strided {
    int64_t ldi, ldo;       // elements between rows
    int64_t cols;           // elements of a row
};
// N entries, S of them strided, OUT with results of their own
template <int N_, int S_, bool OUT> struct Table {
    static constexpr int N = N_, S = S_;
    static constexpr bool HAS_OUT = OUT;
    Entry e[N];
    char *out[OUT ? N : 1];
    Strided s[S];
    int count, strided, chunks;
};
typedef Table<8, 2, true> Short;
typedef Table<192, 16, false> Long;
typedef Table<128, 16, true> LongOut;
static_assert(sizeof(Long) <= 3600 && sizeof(LongOut) <= 3600, "a kernel's arguments");

// an entry as the kernels work with it
struct Item {
    const char *in;
    char *out;
    int64_t n;
    int chunk0, next, dtype;      // its first chunk, the next entry's
    const Strided *strided;
};

template <int INF> __device__ __forceinline__ void take(double &s, double x) {
    if (INF) {
        const double a = fabs(x);
        s = a > s || a != a ? a : s;      // a NaN stays
    } else s = __builtin_fma(x, x, s);
}
template <int INF> __device__ __forceinline__ double both(double a, double b) {
    if (INF) return a != a ? a : (b > a || b != b ? b : a);
    return a + b;
}
template <int INF> __device__ __forceinline__ double block_total(double s, double *sh, int nt) {
    for (int o = 32; o; o >>= 1) s = both<INF>(s, __shfl_xor(s, o));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    s = sh[0];
    for (int w = 1; w < nt / 64; ++w) s = both<INF>(s, sh[w]);
    __syncthreads();
    return s;
}

// the entry a chunk belongs to (the table is short and the index the same for the whole block)
template <typename Tab> __device__ __forceinline__ Item item_of(const Tab &t, int chunk) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((int)t.e[mid].chunk0 <= chunk) lo = mid;
        else hi = mid - 1;
    }
    const Entry &e = t.e[lo];
    const int next = lo + 1 < t.count ? (int)t.e[lo + 1].chunk0 : t.chunks, dtype = e.bits >> 14 & 3, place = e.bits >> 16;
    const int per = CHUNK_BYTES / (dtype == NMFX_F64 ? 8 : dtype == NMFX_F32 ? 4 : 2);
    char *out = const_cast<char *>(e.in);
    if constexpr (Tab::HAS_OUT) out = t.out[lo];
    return Item{e.in, out, (int64_t)(next - 1 - (int)e.chunk0) * per + (e.bits & 0x3fff), (int)e.chunk0, next, dtype, place ? &t.s[place - 1] : nullptr};
}

__device__ __forceinline__ int64_t at(int64_t cols, int64_t i, int64_t ld) {
    const int64_t r = i / cols;
    return r * ld + (i - r * cols);
}

// Elements beg .. end - 1 of an entry, by a block of nt threads: U loads of 16 bytes a thread on their way at a time.
template <typename T, int INF> __device__ __forceinline__ void sum_span(const Item &e, int64_t beg, int64_t end, int nt, double &s) {
    constexpr int V = 16 / sizeof(T), U = 8;
    const T *in = reinterpret_cast<const T *>(e.in);
    if (e.strided) {
        const Strided &d = *e.strided;
        for (int64_t i = beg + threadIdx.x; i < end; i += nt) take<INF>(s, (double)in[at(d.cols, i, d.ldi)]);
        return;
    }
    double part[4] = {0., 0., 0., 0.};
    auto add = [&](const u32x4 &v) {
        const T *x = reinterpret_cast<const T *>(&v);
#pragma unroll
        for (int u = 0; u < V; ++u) take<INF>(part[u & 3], (double)x[u]);
    };
    const int64_t step = (int64_t)nt * V;
    int64_t i = beg;
    for (; i + U * step <= end; i += U * step) {
        u32x4 v[U];
#pragma unroll
        for (int q = 0; q < U; ++q) v[q] = *reinterpret_cast<const u32x4_any *>(in + i + q * step + threadIdx.x * V);
#pragma unroll
        for (int q = 0; q < U; ++q) add(v[q]);
    }
    for (; i + step <= end; i += step) add(*reinterpret_cast<const u32x4_any *>(in + i + threadIdx.x * V));
    for (int64_t j = i + threadIdx.x; j < end; j += nt) take<INF>(s, (double)in[j]);
#pragma unroll
    for (int u = 0; u < 4; ++u) s = both<INF>(s, part[u]);
}

// The coefficient, and for Float32 as a product of two, the second a power of two and 1 unless the whole is no normal number (norms near Float32's
// largest): a result may be one all the same.  (One multiplication more; in Float64 instead, a branch around the loops: 10.9 -> 15.1 us for the
// short list, whose one block fetches its instructions anew in every call.)
struct Coef {
    double c;
    float c1, c2;
};
__device__ __forceinline__ Coef coef_parts(double c) {
    const bool tiny = c < 0x1p-126;      // (so c1 is below 1 either way, and x c1 does not overflow)
    return Coef{c, (float)(tiny ? c * 0x1p126 : c), tiny ? 0x1p-126f : 1.f};
}
template <typename T> __device__ __forceinline__ T scaled(T x, const Coef &c) {
    if constexpr (sizeof(T) == 8) return x * c.c;
    else return (T)((float)x * c.c1 * c.c2);
}
template <typename T> __device__ __forceinline__ void scale_span(const Item &e, int64_t beg, int64_t end, int nt, const Coef &c) {
    constexpr int V = 16 / sizeof(T), U = 4;
    const T *in = reinterpret_cast<const T *>(e.in);
    T *out = reinterpret_cast<T *>(e.out);
    if (e.strided) {
        const Strided &d = *e.strided;
        for (int64_t i = beg + threadIdx.x; i < end; i += nt) out[at(d.cols, i, d.ldo)] = scaled(in[at(d.cols, i, d.ldi)], c);
        return;
    }
    auto put = [&](u32x4 v, int64_t i) {
        T *x = reinterpret_cast<T *>(&v);
#pragma unroll
        for (int u = 0; u < V; ++u) x[u] = scaled(x[u], c);
        *reinterpret_cast<u32x4_any *>(out + i) = v;
    };
    const int64_t step = (int64_t)nt * V;
    int64_t i = beg;
    for (; i + U * step <= end; i += U * step) {
        u32x4 v[U];
#pragma unroll
        for (int q = 0; q < U; ++q) v[q] = *reinterpret_cast<const u32x4_any *>(in + i + q * step + threadIdx.x * V);
#pragma unroll
        for (int q = 0; q < U; ++q) put(v[q], i + q * step + threadIdx.x * V);
    }
    for (; i + step <= end; i += step) put(*reinterpret_cast<const u32x4_any *>(in + i + threadIdx.x * V), i + threadIdx.x * V);
    for (int64_t j = i + threadIdx.x; j < end; j += nt) out[j] = scaled(in[j], c);
}

// calls f(entry, first, last element) for the pieces of chunks c .. last - 1, entry by entry
template <typename Tab, typename F> __device__ __forceinline__ void spans(const Tab &t, int c, int last, F &&f) {
    while (c < last) {
        const Item e = item_of(t, c);
        const int upto = min(last, e.next), per = CHUNK_BYTES / (e.dtype == NMFX_F64 ? 8 : e.dtype == NMFX_F32 ? 4 : 2);
        f(e, (int64_t)(c - e.chunk0) * per, min(e.n, (int64_t)(upto - e.chunk0) * per));
        c = upto;
    }
}
template <int INF, typename Tab> __device__ __forceinline__ void sum_chunks(const Tab &t, int c, int last, int nt, double &s) {
    spans(t, c, last, [&](const Item &e, int64_t beg, int64_t end) {
        switch (e.dtype) {
            case NMFX_F32: sum_span<float, INF>(e, beg, end, nt, s); break;
            case NMFX_F64: sum_span<double, INF>(e, beg, end, nt, s); break;
            case NMFX_BF16: sum_span<__bf16, INF>(e, beg, end, nt, s); break;
            default: sum_span<_Float16, INF>(e, beg, end, nt, s); break;
        }
    });
}
template <typename Tab> __device__ __forceinline__ void scale_chunks(const Tab &t, int c, int last, int nt, double by) {
    const Coef coef = coef_parts(by);
    spans(t, c, last, [&](const Item &e, int64_t beg, int64_t end) {
        switch (e.dtype) {
            case NMFX_F32: scale_span<float>(e, beg, end, nt, coef); break;
            case NMFX_F64: scale_span<double>(e, beg, end, nt, coef); break;
            case NMFX_BF16: scale_span<__bf16>(e, beg, end, nt, coef); break;
            default: scale_span<_Float16>(e, beg, end, nt, coef); break;
        }
    });
}
template <int INF> __device__ __forceinline__ double norm_of(double s) { return INF ? s : sqrt(s); }
__device__ __forceinline__ double coef_of(double norm, double max_norm) {
    const double c = max_norm / (norm + 1e-6);
    return c >= 1. ? 1. : c;                 // a NaN norm gives a NaN coefficient
}

template <int INF, typename Tab> __global__ __launch_bounds__(NT) void partial_kernel(Tab t, double *part) {
    __shared__ double sh[NT / 64];
    double s = 0.;
    // neighbouring chunks: an entry is looked up once for all of its chunks that the block has
    sum_chunks<INF>(t, (int)((int64_t)t.chunks * blockIdx.x / gridDim.x), (int)((int64_t)t.chunks * (blockIdx.x + 1) / gridDim.x), NT, s);
    s = block_total<INF>(s, sh, NT);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}
template <int INF> __global__ __launch_bounds__(1024) void norm_kernel(const double *part, int parts, float *norm) {
    __shared__ double sh[16];
    double s = 0.;
    for (int i = threadIdx.x; i < parts; i += 1024) s = both<INF>(s, part[i]);
    s = block_total<INF>(s, sh, 1024);
    if (threadIdx.x == 0) *norm = (float)norm_of<INF>(s);
}
template <int INF, typename Tab> __global__ __launch_bounds__(NT) void scale_kernel(Tab t, const double *part, int parts, double max_norm, int in_place, float *norm) {
    __shared__ double sh[NT / 64];
    double s = 0.;
    for (int i = threadIdx.x; i < parts; i += NT) s = both<INF>(s, part[i]);
    const double nrm = norm_of<INF>(block_total<INF>(s, sh, NT)), c = coef_of(nrm, max_norm);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)nrm;
    if (c == 1. && in_place) return;
    const int b = gridDim.x - 1 - blockIdx.x;
    scale_chunks(t, (int)((int64_t)t.chunks * b / gridDim.x), (int)((int64_t)t.chunks * (b + 1) / gridDim.x), NT, c);
}
// a short list: one block does all, in one launch for two.  12000 floats: 13.5 -> 10.9 us a call, 60000 (15 chunks) 13 -> 10.3; beyond that the
// block's own time shows next to a call's.
template <int INF> __global__ __launch_bounds__(1024) void small_kernel(Short t, double max_norm, int in_place, int clip, float *norm) {
    __shared__ double sh[16];
    double s = 0.;
    sum_chunks<INF>(t, 0, t.chunks, 1024, s);
    const double nrm = norm_of<INF>(block_total<INF>(s, sh, 1024));
    if (threadIdx.x == 0) *norm = (float)nrm;
    if (!clip) return;
    const double c = coef_of(nrm, max_norm);
    if (c == 1. && in_place) return;
    scale_chunks(t, 0, t.chunks, 1024, c);
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------
constexpr int64_t SMALL_CHUNKS = 16;

using ops::View;
using ops::meet;
View view_of(const nmfx_dmat &m, const char *what) {
    auto refuse = [&](int status, const char *why) { throw ops::OpError{status, std::string(what) + why}; };
    const int es = ops::elem_bytes(m.dtype);
    if (!es) refuse(NMFX_ERR_BAD_ARG, ": dtype is none of NMFX_F32, NMFX_F64, NMFX_BF16, NMFX_F16");
    if (m.reserved != 0) refuse(NMFX_ERR_BAD_ARG, ": reserved must be 0");
    if (m.rows < 0 || m.cols < 0) refuse(NMFX_ERR_DIM_MISMATCH, ": negative extent");
    if (!m.rows || !m.cols) return View{nullptr, 0, 0, 0, es, m.dtype};
    if (!m.data) refuse(NMFX_ERR_BAD_ARG, ": data is NULL");
    if (reinterpret_cast<uintptr_t>(m.data) & (es - 1)) refuse(NMFX_ERR_BAD_ARG, ": data is not aligned to its element");
    View v{static_cast<char *>(m.data), 0, 0, 0, es, m.dtype};
    if (m.cs == 1 && (m.rs >= m.cols || m.rows == 1)) { v.rows = m.rows; v.len = m.cols; v.ld = m.rs; }
    else if (m.rs == 1 && (m.cs >= m.rows || m.cols == 1)) { v.rows = m.cols; v.len = m.rows; v.ld = m.cs; }
    else refuse(NMFX_ERR_BAD_ARG, ": one of rs, cs must be 1 and the other at least the extent it steps over");
    if (v.rows == 1 || v.ld == v.len) { v.len *= v.rows; v.rows = 1; v.ld = v.len; }
    if (v.rows > 1 && v.len > INT32_MAX) refuse(NMFX_ERR_UNSUPPORTED, ": rows of a strided matrix may have at most 2^31 - 1 elements");
    return v;
}

bool before(const View &a, const View &b) { return a.p < b.p; }
// of views in order of address
bool any_meet(const std::vector<View> &v) {
    for (size_t i = 0; i < v.size(); ++i)
        for (size_t j = i + 1; j < v.size() && v[j].p < v[i].p + v[i].bytes(); ++j)
            if (meet(v[i], v[j])) return true;
    return false;
}

int64_t chunks_of(const View &v) { return (v.rows * v.len * v.es + CHUNK_BYTES - 1) / CHUNK_BYTES; }
// a table is full with 16 strided entries at the earliest (of the short form: 2)
int64_t workspace_of(int64_t count) { return 8ll * SUM_BLOCKS * (count / Long::S + 5); }

struct Work {
    const std::vector<View> &in, &out;
    bool clip, in_place;
    double max_norm;
    float *norm;
    double *part;
    hipStream_t st;
};
template <typename Tab> std::vector<Tab> tables_of(const Work &w) {
    std::vector<Tab> ts;
    for (size_t i = 0; i < w.in.size(); ++i) {
        const View &a = w.in[i], &b = w.out[i];
        if (!a.rows) continue;
        const int64_t c = chunks_of(a);
        ops::require(c <= INT32_MAX / 2, NMFX_ERR_UNSUPPORTED, "a matrix is larger than 2^44 bytes");
        const bool dense = a.rows == 1 && b.rows == 1;
        if (ts.empty() || ts.back().count == Tab::N || (!dense && ts.back().strided == Tab::S) || ts.back().chunks + c > INT32_MAX / 2) {
            ts.emplace_back();
            ts.back().count = ts.back().strided = ts.back().chunks = 0;
        }
        Tab &t = ts.back();
        if (!dense) {
            // where only one side is dense, both go by the rows of the other
            const int64_t cols = a.rows > 1 ? a.len : b.len;
            t.s[t.strided++] = Strided{a.rows > 1 ? a.ld : cols, b.rows > 1 ? b.ld : cols, cols};
        }
        const uint32_t last = (uint32_t)(a.rows * a.len - (c - 1) * (CHUNK_BYTES / a.es));
        if constexpr (Tab::HAS_OUT) t.out[t.count] = b.p;
        t.e[t.count++] = Entry{a.p, (uint32_t)t.chunks, last | (uint32_t)a.dtype << 14 | (dense ? 0u : (uint32_t)t.strided) << 16};
        t.chunks += (int)c;
    }
    return ts;
}

template <int INF, typename Tab> void launch(const Work &w) {
    const std::vector<Tab> ts = tables_of<Tab>(w);
    int64_t chunks = 0;
    for (const Tab &t : ts) chunks += t.chunks;
    if constexpr (std::is_same<Tab, Short>::value)
        if (ts.size() == 1 && chunks <= SMALL_CHUNKS) {
            small_kernel<INF><<<1, 1024, 0, w.st>>>(ts[0], w.max_norm, w.in_place, w.clip, w.norm);
            ops::hip_ok(hipGetLastError(), "gradient norm");
            return;
        }
    int parts = 0;
    ops::require((int64_t)(SUM_BLOCKS * ts.size()) * 8 <= workspace_of((int64_t)w.in.size()), NMFX_ERR_STATE, "partial sums exceed the workspace");
    for (const Tab &t : ts) {
        const int blocks = std::min(t.chunks, SUM_BLOCKS);
        partial_kernel<INF, Tab><<<blocks, NT, 0, w.st>>>(t, w.part + parts);
        ops::hip_ok(hipGetLastError(), "gradient norm");
        parts += blocks;
    }
    if (!w.clip || ts.empty()) {
        norm_kernel<INF><<<1, 1024, 0, w.st>>>(w.part, parts, w.norm);
        ops::hip_ok(hipGetLastError(), "gradient norm");
        return;
    }
    for (size_t i = ts.size(); i-- > 0;) {
        scale_kernel<INF, Tab><<<std::min(ts[i].chunks, SCALE_BLOCKS), NT, 0, w.st>>>(ts[i], w.part, parts, w.max_norm, w.in_place, i == 0 ? w.norm : nullptr);
        ops::hip_ok(hipGetLastError(), "gradient scaling");
    }
}
template <int INF> void launch_any(const Work &w) {
    if (w.in.size() <= 8) launch<INF, Short>(w);
    else if (w.in_place) launch<INF, Long>(w);
    else launch<INF, LongOut>(w);
}

void run(int count, const nmfx_dmat *g, const nmfx_dmat *o, bool clip, double max_norm, int norm_type, float *norm, void *ws, int64_t ws_bytes, int device, void *stream) {
    ops::require(count >= 0, NMFX_ERR_BAD_ARG, "count must not be negative");
    ops::require(g || !count, NMFX_ERR_BAD_ARG, "the list of matrices is NULL");
    ops::require(norm != nullptr, NMFX_ERR_BAD_ARG, "norm is NULL");
    ops::require(norm_type == NMFX_NORM_2 || norm_type == NMFX_NORM_INF, NMFX_ERR_BAD_ARG, "norm_type is neither NMFX_NORM_2 nor NMFX_NORM_INF");
    ops::require(!clip || max_norm >= 0., NMFX_ERR_BAD_ARG, "max_norm must not be negative");
    ops::require(ws && ws_bytes >= workspace_of(count), NMFX_ERR_BAD_ARG, "the workspace is smaller than nmfx_grad_norm_workspace says");
    ops::require((reinterpret_cast<uintptr_t>(ws) & 7) == 0, NMFX_ERR_BAD_ARG, "the workspace must be aligned to 8 bytes");
    std::vector<View> in, out;
    in.reserve(count);
    out.reserve(count);
    for (int i = 0; i < count; ++i) {
        in.push_back(view_of(g[i], "a gradient"));
        out.push_back(clip && o ? view_of(o[i], "a clipped gradient") : in.back());
        if (clip && o) {
            ops::require(g[i].rows == o[i].rows && g[i].cols == o[i].cols, NMFX_ERR_DIM_MISMATCH, "a clipped gradient must have its gradient's shape");
            ops::require(g[i].dtype == o[i].dtype, NMFX_ERR_BAD_ARG, "a clipped gradient must have its gradient's dtype");
            const bool vec = g[i].rows <= 1 || g[i].cols <= 1;
            ops::require(vec || (g[i].cs == 1) == (o[i].cs == 1), NMFX_ERR_BAD_ARG, "a clipped gradient must have its gradient's contiguous index");
        }
    }
    if (clip) {
        // every element is written by one thread once: no two results may share one, and none may be another's input
        std::vector<View> w, r;
        w.reserve(count);
        for (int i = 0; i < count; ++i) {
            if (!out[i].rows) continue;
            w.push_back(out[i]);
            if (o && !(in[i].p == out[i].p && in[i].rows == out[i].rows && in[i].ld == out[i].ld)) r.push_back(in[i]);
        }
        if (!std::is_sorted(w.begin(), w.end(), before)) std::sort(w.begin(), w.end(), before);
        ops::require(!any_meet(w), NMFX_ERR_BAD_ARG, "two of the matrices to write share elements");
        if (!r.empty()) {
            std::vector<char *> reach;            // how far the written views up to this one reach
            reach.reserve(w.size());
            for (const View &v : w) reach.push_back(std::max(reach.empty() ? v.p : reach.back(), v.p + v.bytes()));
            for (const View &a : r)
                for (size_t j = std::upper_bound(reach.begin(), reach.end(), a.p) - reach.begin(); j < w.size() && w[j].p < a.p + a.bytes(); ++j)
                    ops::require(!meet(a, w[j]), NMFX_ERR_BAD_ARG, "a matrix to write shares elements with a gradient that is not its own");
        }
    }
    bool in_place = true;
    for (int i = 0; i < count; ++i) in_place = in_place && in[i].p == out[i].p && in[i].rows == out[i].rows && in[i].ld == out[i].ld;
    ops::OnDevice on(device);
    const Work w{in, out, clip, in_place, max_norm, norm, static_cast<double *>(ws), static_cast<hipStream_t>(stream)};
    if (norm_type == NMFX_NORM_2) launch_any<0>(w);
    else launch_any<1>(w);
}

}  // namespace gradnorm

namespace ops {
std::string &last_error() {
    thread_local std::string msg;
    return msg;
}
}  // namespace ops
}  // namespace nmfx

using namespace nmfx;

extern "C" {

const char *nmfx_last_op_error(void) { return ops::last_error().c_str(); }

int nmfx_grad_norm_workspace(int count, int64_t *bytes) {
    return ops::guarded([&] {
        ops::require(bytes && count >= 0, NMFX_ERR_BAD_ARG, "bytes is NULL or count negative");
        *bytes = gradnorm::workspace_of(count);
    });
}

int nmfx_grad_norm(int count, const nmfx_dmat *grads, int norm_type, float *norm, void *workspace, int64_t workspace_bytes, int device, void *stream) {
    return ops::guarded([&] { gradnorm::run(count, grads, nullptr, false, 0., norm_type, norm, workspace, workspace_bytes, device, stream); });
}

int nmfx_clip_grad_norm(int count, const nmfx_dmat *grads, const nmfx_dmat *out, double max_norm, int norm_type, float *norm, void *workspace,
                        int64_t workspace_bytes, int device, void *stream) {
    return ops::guarded([&] { gradnorm::run(count, grads, out, true, max_norm, norm_type, norm, workspace, workspace_bytes, device, stream); });
}

}  // extern "C"

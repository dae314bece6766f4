// group_norm_cl.hip — GroupNorm with an activation over channels-last tensors, forward and
// backward (stx_group_norm_cl, stx_group_norm_cl_back).
#include <algorithm>
#include <cmath>
#include <numeric>

#include "typed.hpp"

namespace stx {
namespace {

// One slice (ne3 index) is [T][C], dense. Threads move vectors of V elements; so that a
// thread meets the same channels in every vector it takes whatever C is, the slice is walked in
// super-rows of R = V / gcd(C, V) rows, which hold a whole number of vectors: vector j of a
// super-row covers channels (j V + e) mod C. Accesses may be unaligned (odd C, odd slices); only
// the slice's last super-row can be partial.
//
// A block has a tile of `cols` vector columns x `rws` super-rows at a time, and one chunk of the
// slice's super-rows. Two kernels, forward and backward alike:
//   sums:  two sums of every slot (position in the super-row) over the chunk: t, t^2 or dz, dz xhat;
//          added up to groups (backward: times w), one pair a (slice, chunk, tile, group), and in the
//          backward pass also kept per slot, for dweight and dbias;
//   apply: each block adds the pairs of its slice's groups, then streams its elements, one fused
//          multiply-add and the activation each. In the backward pass extra blocks add the
//          slots' sums to dweight and dbias.
// (slices with more than kDirect pairs have them added by a small kernel in between). t = x - the
// group's first element, and t and t^2 are summed in double: E[t^2] - E[t]^2 loses at most 2^-53 times the
// number of elements, wherever the mean lies (the element is within that number's root of deviations
// from it); sums of x itself would lose 2^-53 mean^2 / var. The backward sums in float over kHeld rows
// of a thread (64 terms drift by about 1e-7 of their sum), then in double. The first forward
// pass is bound by HBM, the second, as far as the last-level cache still holds the input, by that or by the
// activation: with GELU the vector units are busy 91 % of the time, in the gradients 72 to 82 %.
// Measured: fp32 4 x 85,995 x 48, one group, GELU (66 MB): 15.3 us (4.3 TB/s) and 25.6 us (5.2 TB/s read
// and written); gradients of fp32 4 x 21,499 x 96, four groups, GELU (33 MB a tensor): 19.4 and 22.4 us;
// of bf16 60 x 801 x 384, 32 groups, SiLU (37 MB a tensor): 19.2 and 23.7 us.
constexpr int kThreads = 256;
constexpr int kVec = 4;                  // elements of a vector: with 8 of 16 bits a channel's constants leave four waves a SIMD
constexpr int kBatch = 2;                // super-rows a thread has in flight
constexpr int kHeld = 64;                // rows summed in float before they join the sums in double
// Pairs that every apply block adds by itself: at 256 to 1,024 a slice the small kernel costs 2 to 4.5 us
// and its launch, and saves the apply kernel 0 to 1 us.
constexpr int kDirect = 2048;
constexpr int kParamChannels = 8;        // of a block that adds dweight and dbias: 32 lanes a channel

struct Geometry {
    long long B, T;
    int C, G, width;                     // groups of `width` channels, the last of what is left
    int V, R, slots, ncol;               // slots = C R = ncol V
    int cols, tiles, rws;                // columns of a block, column tiles, super-rows a block takes at once
    int chunks;
    long long srows, chunk_srows;        // super-rows of a slice, of a chunk
};

Geometry geometry(const stx_tensor* a, int n_groups) {
    Geometry g{};
    g.C = (int)a->ne[0];
    g.T = a->ne[1] * a->ne[2];
    g.B = a->ne[3];
    g.G = n_groups;
    g.width = (g.C + n_groups - 1) / n_groups;
    g.V = kVec;
    g.R = g.V / std::gcd(g.C, g.V);
    g.slots = g.C * g.R;
    g.ncol = g.slots / g.V;
    // Column tiles of up to kThreads: the fewest that keep nine tenths of the threads at work.
    double best = 0;
    for (int tiles = (g.ncol + kThreads - 1) / kThreads, n = 0; n < 16 && tiles <= g.ncol; tiles++, n++) {
        const int cols = (g.ncol + tiles - 1) / tiles;
        const double use = (double)g.ncol / ((double)cols * ((g.ncol + cols - 1) / cols)) * (cols * (kThreads / cols)) / kThreads;
        if (use > best + 0.02) {
            best = use;
            g.cols = cols;
        }
        if (use >= 0.9) break;
    }
    g.tiles = (g.ncol + g.cols - 1) / g.cols;
    g.rws = kThreads / g.cols;
    g.srows = (g.T + g.R - 1) / g.R;
    // Chunks: four blocks a CU, all resident at once and none more than the others (840 blocks took as
    // long as 1,020 that do a fifth more between them), each of at least four super-rows a thread.
    const long long most = std::max(1LL, std::min(1024 / std::max(1LL, g.B * g.tiles), g.srows / (4 * g.rws)));
    g.chunk_srows = std::max(1LL, (g.srows + most - 1) / most);
    g.chunks = (int)std::max(1LL, (g.srows + g.chunk_srows - 1) / g.chunk_srows);
    return g;
}

struct NormArgs {
    Geometry g;
    FastDiv chunks, tiles;
    const void* x;
    const void* dy;
    void* out;
    const float *w, *b;
    const double2* stats_in;             // [B][G] mean, 1 / sqrt(var + eps)
    double2* stats_out;
    double2* part;                       // [B][rows][G], rows = chunks x tiles
    double2* folded;                     // [B][G]
    double* shift;                       // [B][G], forward: what the sums are taken from
    double2* slot;                       // backward: [B][chunks][slots]
    long long rows;                      // of `part`, or 1 where they are folded (0: no elements)
    unsigned base;                       // blocks of the launches before this one
    unsigned first;                      // backward: apply blocks before this one add dweight and dbias
    float *dw, *db;
    double eps;
    int act;
};

template <class T, int V>
__device__ __forceinline__ Pack<T, V> load_vec(const T* p, long long left) {
    Pack<T, V> v;
    if (left >= V) {
        __builtin_memcpy(&v, p, sizeof v);
    } else {
#pragma unroll
        for (int e = 0; e < V; e++) v.v[e] = e < left ? p[e] : T(0.f);
    }
    return v;
}
template <class T, int V>
__device__ __forceinline__ void store_vec(T* p, long long left, const float (&f)[V]) {
    if (left >= V) {
        T v[V];
#pragma unroll
        for (int e = 0; e < V; e++) v[e] = from_f32<T>(f[e]);
        __builtin_memcpy(p, v, sizeof v);
    } else {
#pragma unroll
        for (int e = 0; e < V; e++)
            if (e < left) p[e] = from_f32<T>(f[e]);
    }
}

// Where a thread is: its slice, column and super-rows.
struct Place {
    long long slice, begin, end, full, chunk;            // super-rows before `full` are whole
    int col, row, tile;
    bool on;
};
__device__ __forceinline__ Place place(const NormArgs& a, unsigned bid) {
    Place p;
    const unsigned bc = a.tiles.div(bid);
    p.tile = (int)(bid - bc * a.tiles.d);
    const unsigned b = a.chunks.div(bc);
    p.slice = b;
    p.chunk = bc - b * a.chunks.d;
    p.row = (int)threadIdx.x / a.g.cols;
    p.col = p.tile * a.g.cols + (int)threadIdx.x % a.g.cols;
    p.begin = p.chunk * a.g.chunk_srows;
    p.end = min(p.begin + a.g.chunk_srows, a.g.srows);
    p.full = a.g.T % a.g.R ? a.g.srows - 1 : a.g.srows;
    p.on = p.row < a.g.rws && p.col < a.g.ncol;
    return p;
}

// use(r, whole, load(r, whole)) over a thread's super-rows, kBatch of them at a time, the next batch's
// loads issued before the last one's are used. whole: every vector exists in full.
template <class L, class F>
__device__ __forceinline__ void for_rows(const Place& p, int rws, L&& load, F&& use) {
    constexpr std::integral_constant<int, kBatch> batch{};
    constexpr std::integral_constant<int, 1> one{};
    long long r = p.begin + p.row;
    const long long end = min(p.end, p.full), ahead = (kBatch - 1) * rws, step = kBatch * rws;
    if (r + ahead < end) {
        auto now = load(r, batch, std::true_type{});
        for (; r + step + ahead < end; r += step) {
            const auto next = load(r + step, batch, std::true_type{});
            use(r, batch, std::true_type{}, now);
            now = next;
        }
        use(r, batch, std::true_type{}, now);
        r += step;
    }
    for (; r < end; r += rws) use(r, one, std::true_type{}, load(r, one, std::true_type{}));
    if (r < p.end) use(r, one, std::false_type{}, load(r, one, std::false_type{}));
}

// N vectors of x, and of dy in the backward pass.
template <class T, int V, int N, bool BACK>
struct Rows {
    Pack<T, V> x[N], dy[BACK ? N : 1];
};

// Sum of red[rows][width] over the rows, into red[0][]. All threads; the order depends on the shape alone.
__device__ __forceinline__ void fold_rows(double2* red, int rows, int width) {
    while (rows > 1) {
        const int half = (rows + 1) / 2;
        __syncthreads();
        for (int i = (int)threadIdx.x; i < (rows - half) * width; i += kThreads) {
            const double2 v = red[half * width + i];
            red[i].x += v.x;
            red[i].y += v.y;
        }
        rows = half;
    }
    __syncthreads();
}

// Per-channel constants, all of the centred t = x - mh, where mean = mh + a rest that joins the
// additive constants (a float mean alone would cost |mean| 2^-24 / std; a product x r - mean r, which
// would save the subtraction, costs as much):
//   xhat = t r - d,  z = xhat w + b = t A + B,  dx = r (w dz - S1/n - xhat S2/n) = t r q + (dz A + p).
// (r q as one constant would hold r^2, which leaves fp32 where the data's deviations pass 10^19.)
struct Chan {
    float mh, r, d, A, B, p, q;
    __device__ __forceinline__ void set(const NormArgs& a, double mean, double rstd, int c) {
        const double w = a.w ? (double)a.w[c] : 1.0, b = a.b ? (double)a.b[c] : 0.0;
        mh = (float)mean;
        const double rest = (mean - (double)mh) * rstd;
        r = (float)rstd;
        d = (float)rest;
        A = (float)(rstd * w);
        B = (float)(b - rest * w);
    }
    __device__ __forceinline__ void set_back(double mean, double rstd, double s1, double s2) {   // S1 / n, S2 / n
        p = (float)(((mean - (double)mh) * rstd * s2 - s1) * rstd);
        q = (float)(-rstd * s2);
    }
};

// f(e, c, g) for the channels c and groups g of a column's elements.
template <int V, class F>
__device__ __forceinline__ void for_channels(const Geometry& g, int col, F&& f) {
    int c = (int)((unsigned)(col * V) % (unsigned)g.C), group = (int)((unsigned)c / (unsigned)g.width), next = (group + 1) * g.width;
#pragma unroll
    for (int e = 0; e < V; e++) {
        f(e, c, group);
        c++;
        if (c == next) {
            group++;
            next += g.width;
        }
        if (c == g.C) {
            c = 0;
            group = 0;
            next = g.width;
        }
    }
}

template <class T>
__device__ __forceinline__ double group_shift(const T* x, int first) {
    const float v = to_f32(x[first]);
    return fabsf(v) <= 0x1.fffffep127f ? (double)v : 0.0;            // not of an infinity or NaN: those spoil the sums by themselves
}

template <class T, bool BACK, int ACT>
__global__ __launch_bounds__(kThreads) void gn_cl_sums_kernel(NormArgs a) {
    constexpr int V = kVec;
    __shared__ double2 red[kThreads * V];
    const Place p = place(a, a.base + blockIdx.x);
    const int width = a.g.cols * V, first = p.tile * width, here = min(width, a.g.slots - first);
    double2* mine = red + p.row * width + (int)threadIdx.x % a.g.cols * V;
    if (p.row < a.g.rws) {
#pragma unroll
        for (int e = 0; e < V; e++) mine[e] = make_double2(0.0, 0.0);
    }
    if (p.on) {
        const long long n = a.g.T * a.g.C;
        const T* x = static_cast<const T*>(a.x) + p.slice * n;
        const T* dy = static_cast<const T*>(a.dy) + p.slice * n;
        Chan k[BACK ? V : 1];
        double shift[BACK ? 1 : V];
        for_channels<V>(a.g, p.col, [&](int e, int c, int g) {
            if constexpr (BACK) {
                const double2 st = a.stats_in[p.slice * a.g.G + g];
                k[e].set(a, st.x, st.y, c);
            } else {
                shift[e] = group_shift(x, g * a.g.width);
            }
        });
        std::conditional_t<BACK, float, double> s1[V] = {}, s2[V] = {};
        int held = 0;
        auto flush = [&] {
#pragma unroll
            for (int e = 0; e < V; e++) {
                double t1 = (double)s1[e], t2 = (double)s2[e];
                if constexpr (BACK) t2 = fma(t2, (double)k[e].r, -t1 * (double)k[e].d);   // from dz t to dz xhat
                mine[e] = make_double2(mine[e].x + t1, mine[e].y + t2);
                s1[e] = s2[e] = 0;
            }
            held = 0;
        };
        auto load = [&](long long r, auto batch, auto whole) {
            Rows<T, V, batch(), BACK> f;
#pragma unroll
            for (int i = 0; i < batch(); i++) {
                const long long at = (r + i * a.g.rws) * a.g.slots + (long long)p.col * V, left = whole() ? V : n - at;
                f.x[i] = load_vec<T, V>(x + at, left);
                if constexpr (BACK) f.dy[i] = load_vec<T, V>(dy + at, left);
            }
            return f;
        };
        for_rows(p, a.g.rws, load, [&](long long r, auto batch, auto whole, const auto& f) {
            constexpr int N = batch();
            const long long left = whole() ? V : n - r * a.g.slots - (long long)p.col * V;
#pragma unroll
            for (int i = 0; i < N; i++) {
#pragma unroll
                for (int e = 0; e < V; e++) {
                    if (!whole() && e >= left) continue;
                    const float xe = to_f32(f.x[i].v[e]);
                    if constexpr (BACK) {
                        const float t = xe - k[e].mh;
                        float d;
                        (void)act_f32<ACT, T>(fmaf(t, k[e].A, k[e].B), d);
                        const float dz = to_f32(f.dy[i].v[e]) * d;
                        s1[e] += dz;
                        s2[e] = fmaf(dz, t, s2[e]);
                    } else {
                        const double t = (double)xe - shift[e];
                        s1[e] += t;
                        s2[e] = fma(t, t, s2[e]);
                    }
                }
            }
            if (BACK && (held += N) >= kHeld) flush();
        });
        flush();
    }
    fold_rows(red, a.g.rws, width);
    if constexpr (BACK) {
        double2* slot = a.slot + (p.slice * a.g.chunks + p.chunk) * a.g.slots + first;
        for (int i = (int)threadIdx.x; i < here; i += kThreads) {
            const double2 v = red[i];
            slot[i] = v;
            const double w = a.w ? (double)a.w[(unsigned)(first + i) % (unsigned)a.g.C] : 1.0;
            red[i] = make_double2(v.x * w, v.y * w);
        }
        __syncthreads();
    }
    // A group's slots: one run in each of the super-row's R rows. Wide groups by a wave each, narrow
    // ones by a thread.
    double2* part = a.part + ((p.slice * a.g.chunks + p.chunk) * a.g.tiles + p.tile) * a.g.G;
    const bool wide = a.g.width >= 64;
    const int lanes = wide ? 64 : 1, lane = wide ? (int)threadIdx.x % 64 : 0;
    for (int g = (int)threadIdx.x / lanes; g < a.g.G; g += kThreads / lanes) {
        double2 s = make_double2(0.0, 0.0);
        for (int r = 0; r < a.g.R; r++) {
            const int row = r * a.g.C - first, lo = max(0, row + g * a.g.width), hi = min(here, row + min((g + 1) * a.g.width, a.g.C));
            for (int i = lo + lane; i < hi; i += lanes) {
                s.x += red[i].x;
                s.y += red[i].y;
            }
        }
        if (wide) {
            s.x = lane_sum<64>(s.x);
            s.y = lane_sum<64>(s.y);
        }
        if (lane != 0) continue;
        part[g] = s;
        if (!BACK && p.chunk == 0 && p.tile == 0) a.shift[p.slice * a.g.G + g] = group_shift(static_cast<const T*>(a.x) + p.slice * a.g.T * a.g.C, g * a.g.width);
    }
}

// The pairs of one group of one slice.
__global__ __launch_bounds__(kThreads) void gn_cl_fold_kernel(NormArgs a, long long rows) {
    __shared__ double2 red[kThreads];
    const unsigned bid = a.base + blockIdx.x;
    const long long b = bid / (unsigned)a.g.G, g = bid % (unsigned)a.g.G;
    double2 s = make_double2(0.0, 0.0);
#pragma unroll 4
    for (long long r = threadIdx.x; r < rows; r += kThreads) {
        const double2 v = a.part[(b * rows + r) * a.g.G + g];
        s.x += v.x;
        s.y += v.y;
    }
    red[threadIdx.x] = s;
    fold_rows(red, kThreads, 1);
    if (threadIdx.x == 0) a.folded[bid] = red[0];
}

__device__ __forceinline__ double2 moments(const NormArgs& a, double2 s, double n, long long at) {
    if (n == 0.0) return make_double2(0.0, 1.0 / sqrt(a.eps));
    const double mean = s.x / n, var = s.y / n - mean * mean;
    return make_double2(a.shift[at] + mean, 1.0 / sqrt((var < 0.0 ? 0.0 : var) + a.eps));   // NaN stays NaN
}

// dbias and dweight of kParamChannels channels: the slots' sums over slices, chunks and R.
__device__ void add_params(const NormArgs& a, double2* red, unsigned block) {
    const int c = (int)block * kParamChannels + (int)threadIdx.x % kParamChannels, lane = (int)threadIdx.x / kParamChannels;
    const long long rows = a.g.srows ? a.g.B * a.g.chunks * a.g.R : 0;
    double2 s = make_double2(0.0, 0.0);
    if (c < a.g.C) {
#pragma unroll 8
        for (long long r = lane; r < rows; r += kThreads / kParamChannels) {
            const double2 v = a.slot[r * a.g.C + c];
            s.x += v.x;
            s.y += v.y;
        }
    }
    red[threadIdx.x] = s;
    fold_rows(red, kThreads / kParamChannels, kParamChannels);
    if (lane || c >= a.g.C) return;
    if (a.db) a.db[c] = (float)red[threadIdx.x].x;
    if (a.dw) a.dw[c] = (float)red[threadIdx.x].y;
}

template <class T, bool BACK, int ACT>
__global__ __launch_bounds__(kThreads) void gn_cl_apply_kernel(NormArgs a) {
    constexpr int V = kVec;
    extern __shared__ double2 groups[];                  // [max(G, kThreads)]
    const unsigned bid = a.base + blockIdx.x;
    if (BACK && bid < a.first) return add_params(a, groups, bid);
    const Place p = place(a, bid - a.first);
    {
        const int G = a.g.G, parts = max(1, kThreads / G);
        const double2* from = a.part + p.slice * a.rows * G;
        for (int g0 = 0; g0 < G; g0 += kThreads) {       // one pass unless there are more groups than threads
            const int g = g0 + (int)threadIdx.x % min(G, kThreads), part = (int)threadIdx.x / min(G, kThreads);
            double2 s = make_double2(0.0, 0.0);
            if (g < G && part < parts) {
#pragma unroll 4
                for (long long r = part; r < a.rows; r += parts) {
                    const double2 v = from[r * G + g];
                    s.x += v.x;
                    s.y += v.y;
                }
                groups[g0 + (int)threadIdx.x] = s;
            }
        }
        fold_rows(groups, parts, G);
        for (int g = (int)threadIdx.x; g < G; g += kThreads) {
            const double n = (double)a.g.T * (min((g + 1) * a.g.width, a.g.C) - g * a.g.width);
            const double2 s = groups[g];
            groups[g] = BACK ? make_double2(s.x / n, s.y / n) : moments(a, s, n, p.slice * G + g);
            if (!BACK && a.stats_out && p.chunk == 0 && p.tile == 0) a.stats_out[p.slice * G + g] = groups[g];
        }
    }
    __syncthreads();
    if (!p.on) return;
    const long long n = a.g.T * a.g.C;
    const T* x = static_cast<const T*>(a.x) + p.slice * n;
    const T* dy = static_cast<const T*>(a.dy) + p.slice * n;
    T* out = static_cast<T*>(a.out) + p.slice * n;
    Chan k[V];
    for_channels<V>(a.g, p.col, [&](int e, int c, int g) {
        if constexpr (BACK) {
            const double2 st = a.stats_in[p.slice * a.g.G + g];
            k[e].set(a, st.x, st.y, c);
            k[e].set_back(st.x, st.y, groups[g].x, groups[g].y);
        } else {
            k[e].set(a, groups[g].x, groups[g].y, c);
        }
    });
    auto load = [&](long long r, auto batch, auto whole) {
        Rows<T, V, batch(), BACK> f;
#pragma unroll
        for (int i = 0; i < batch(); i++) {
            const long long at = (r + i * a.g.rws) * a.g.slots + (long long)p.col * V, left = whole() ? V : n - at;
            f.x[i] = load_vec<T, V>(x + at, left);
            if constexpr (BACK) f.dy[i] = load_vec<T, V>(dy + at, left);
        }
        return f;
    };
    for_rows(p, a.g.rws, load, [&](long long r, auto batch, auto whole, const auto& f) {
        constexpr int N = batch();
#pragma unroll
        for (int i = 0; i < N; i++) {
            const long long at = (r + i * a.g.rws) * a.g.slots + (long long)p.col * V, left = whole() ? V : n - at;
            float y[V];
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float t = to_f32(f.x[i].v[e]) - k[e].mh, z = fmaf(t, k[e].A, k[e].B);
                if constexpr (BACK) {
                    float d;
                    (void)act_f32<ACT, T>(z, d);
                    y[e] = fmaf(t * k[e].r, k[e].q, fmaf(to_f32(f.dy[i].v[e]) * d, k[e].A, k[e].p));
                } else {
                    y[e] = act_f32<ACT, T>(z);
                }
            }
            store_vec<T, V>(out + at, left, y);
        }
    });
}

long long pair_rows(const Geometry& g) { return g.srows ? (long long)g.chunks * g.tiles : 0; }
bool folds(const Geometry& g) { return pair_rows(g) > 1 && (g.G > kThreads || pair_rows(g) * g.G > kDirect); }
struct Spaces {
    size_t folded, shift, slot, total;   // `part` is at 0; the forward call needs no slot
};
Spaces spaces(const Geometry& g) {
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    Spaces s{};
    s.folded = up((size_t)g.B * pair_rows(g) * g.G * sizeof(double2));
    s.shift = s.folded + up(folds(g) ? (size_t)g.B * g.G * sizeof(double2) : 0);
    s.slot = s.shift + up((size_t)g.B * g.G * sizeof(double));
    s.total = s.slot + (size_t)g.B * g.chunks * g.slots * sizeof(double2);
    return s;
}

constexpr int kMaxGroups = 4096;         // of the apply kernel's LDS: 64 KB

Geometry check_norm(const stx_tensor* a, stx_type type, int n_groups) {
    const int size = type_size(type);
    check_typed(a, size, "group_norm_cl: a");
    STX_REQUIRE(contiguous_typed(a, size), "group_norm_cl: a must be contiguous");
    const long long C = a->ne[0];
    STX_REQUIRE(n_groups > 0 && C > 0, "group_norm_cl: no groups or no channels");
    STX_REQUIRE(C < (1LL << 24), "group_norm_cl: too many channels");
    STX_REQUIRE((n_groups - 1LL) * ((C + n_groups - 1) / n_groups) < C, "group_norm_cl: %lld channels leave a group of %d empty", C,
                n_groups);
    if (n_groups > kMaxGroups) fail(STX_STATUS_UNSUPPORTED, "group_norm_cl: more than %d groups", kMaxGroups);
    const Geometry g = geometry(a, n_groups);
    STX_REQUIRE(g.B < (1LL << 31) && g.B * g.chunks * g.tiles < (1LL << 30) && g.B * g.G < (1LL << 31), "group_norm_cl: too many slices");
    return g;
}

template <bool BACK>
void run_norm(NormArgs& a, stx_type type, void* ws, hipStream_t stream) {
    const Geometry& g = a.g;
    const Spaces at = spaces(g);
    a.chunks = FastDiv((unsigned)g.chunks);
    a.tiles = FastDiv((unsigned)g.tiles);
    a.part = static_cast<double2*>(ws);
    a.folded = reinterpret_cast<double2*>(static_cast<char*>(ws) + at.folded);
    a.shift = reinterpret_cast<double*>(static_cast<char*>(ws) + at.shift);
    a.slot = reinterpret_cast<double2*>(static_cast<char*>(ws) + at.slot);
    a.rows = pair_rows(g);
    a.first = BACK && (a.dw || a.db) ? (unsigned)((g.C + kParamChannels - 1) / kParamChannels) : 0;
    const unsigned blocks = (unsigned)(g.B * g.chunks * g.tiles);
    with_type(type, [&](auto t) {
        using T = decltype(t);
        if (g.srows && g.B) {
            launch_all(blocks, [&](dim3 grid, unsigned first) {
                a.base = first;
                if constexpr (BACK) with_act(a.act, [&](auto act) { hipLaunchKernelGGL((gn_cl_sums_kernel<T, true, act()>), grid, dim3(kThreads), 0, stream, a); });
                else hipLaunchKernelGGL((gn_cl_sums_kernel<T, false, STX_ACT_NONE>), grid, dim3(kThreads), 0, stream, a);
                launch_check("gn_cl_sums_kernel");
            });
        }
        const bool apply = !BACK || a.out;
        if (folds(g) && g.B && apply) {
            launch_all(g.B * g.G, [&](dim3 grid, unsigned first) {
                a.base = first;
                hipLaunchKernelGGL(gn_cl_fold_kernel, grid, dim3(kThreads), 0, stream, a, a.rows);
                launch_check("gn_cl_fold_kernel");
            });
            a.part = a.folded;
            a.rows = 1;
        }
        launch_all(a.first + (apply ? blocks : 0), [&](dim3 grid, unsigned first) {
            a.base = first;
            with_act(a.act, [&](auto act) { hipLaunchKernelGGL((gn_cl_apply_kernel<T, BACK, act()>), grid, dim3(kThreads), sizeof(double2) * std::max(g.G, kThreads), stream, a); });
            launch_check("gn_cl_apply_kernel");
        });
    });
}

}  // namespace
}  // namespace stx

using namespace stx;

namespace {
size_t query(const stx_tensor* a, stx_type type, int n_groups, size_t Spaces::*size) {
    size_t bytes = 0;
    (void)guard([&] {
        STX_REQUIRE(a != nullptr, "group_norm_cl: a is NULL");
        stx_tensor t = *a;
        t.data = reinterpret_cast<void*>((uintptr_t)256);          // a query may have no data yet
        bytes = spaces(check_norm(&t, type, n_groups)).*size;
    });
    return bytes;
}
}  // namespace

extern "C" {

STX_API size_t stx_group_norm_cl_workspace_size(const stx_tensor* a, stx_type type, int n_groups) {
    return query(a, type, n_groups, &Spaces::total);
}

STX_API size_t stx_group_norm_cl_forward_workspace_size(const stx_tensor* a, stx_type type, int n_groups) {
    return query(a, type, n_groups, &Spaces::slot);
}

STX_API stx_status stx_group_norm_cl(const stx_tensor* a, stx_type type, int n_groups, double eps, const float* weight,
                                     const float* bias, stx_act act, const stx_tensor* dst, double* stats,
                                     void* workspace, size_t workspace_bytes_, stx_stream stream) {
    return guard([&] {
        NormArgs k{};
        k.g = check_norm(a, type, n_groups);
        check_act(act);
        const int size = type_size(type);
        check_typed(dst, size, "group_norm_cl: dst");
        check_same_shape(a, dst, "group_norm_cl");
        STX_REQUIRE(contiguous_typed(dst, size), "group_norm_cl: dst must be contiguous");
        STX_REQUIRE(dst->data == a->data || !overlap(span_of(a, size), span_of(dst, size)), "group_norm_cl: dst overlaps a in part");
        STX_REQUIRE(eps >= 0.0, "group_norm_cl: negative eps");
        const size_t need = spaces(k.g).slot, floats = (size_t)k.g.C * sizeof(float);
        check_workspace(workspace, workspace_bytes_, need, "group_norm_cl");
        const Operand w("weight", weight, floats), b("bias", bias, floats);
        check_apart("group_norm_cl", {{"dst", dst, size}, {"stats", stats, (size_t)k.g.B * k.g.G * sizeof(double2)}, {"the workspace", workspace, need}}, {w, b});
        check_apart("group_norm_cl", {{"stats", stats, (size_t)k.g.B * k.g.G * sizeof(double2)}, {"the workspace", workspace, need}}, {{"a", a, size}});
        k.x = a->data;
        k.dy = a->data;                  // not read
        k.out = dst->data;
        k.w = weight;
        k.b = bias;
        k.stats_out = reinterpret_cast<double2*>(stats);
        k.eps = eps;
        k.act = act;
        run_norm<false>(k, type, workspace, as_stream(stream));
    });
}

STX_API stx_status stx_group_norm_cl_back(const stx_tensor* dy, const stx_tensor* a, stx_type type, const double* stats,
                                          int n_groups, const float* weight, const float* bias, stx_act act,
                                          const stx_tensor* dx, float* dweight, float* dbias, void* workspace,
                                          size_t workspace_bytes_, stx_stream stream) {
    return guard([&] {
        NormArgs k{};
        k.g = check_norm(a, type, n_groups);
        check_act(act);
        const int size = type_size(type);
        check_typed(dy, size, "group_norm_cl_back: dy");
        check_same_shape(a, dy, "group_norm_cl_back");
        STX_REQUIRE(contiguous_typed(dy, size), "group_norm_cl_back: dy must be contiguous");
        if (dx) {
            check_typed(dx, size, "group_norm_cl_back: dx");
            check_same_shape(a, dx, "group_norm_cl_back");
            STX_REQUIRE(contiguous_typed(dx, size), "group_norm_cl_back: dx must be contiguous");
            STX_REQUIRE(!overlap(span_of(a, size), span_of(dx, size)) || dx->data == a->data, "group_norm_cl_back: dx overlaps a in part");
            STX_REQUIRE(dx->data == dy->data || !overlap(span_of(dy, size), span_of(dx, size)), "group_norm_cl_back: dx overlaps dy in part");
        }
        STX_REQUIRE(stats != nullptr || k.g.B == 0, "group_norm_cl_back: stats is NULL");
        const size_t need = spaces(k.g).total, floats = (size_t)k.g.C * sizeof(float);
        check_workspace(workspace, workspace_bytes_, need, "group_norm_cl_back");
        const Operand dw("dweight", dweight, floats), db("dbias", dbias, floats), ws("the workspace", workspace, need);
        const Operand s("stats", stats, (size_t)k.g.B * k.g.G * sizeof(double2)), w("weight", weight, floats), b("bias", bias, floats);
        check_apart("group_norm_cl_back", {{"dx", dx, size}, dw, db, ws}, {s, w, b});
        check_apart("group_norm_cl_back", {dw, db, ws}, {{"dy", dy, size}, {"a", a, size}});
        if (!dx && !dweight && !dbias) return;
        k.x = a->data;
        k.dy = dy->data;
        k.out = dx && k.g.srows ? dx->data : nullptr;
        k.w = weight;
        k.b = bias;
        k.stats_in = reinterpret_cast<const double2*>(stats);
        k.dw = dweight;
        k.db = dbias;
        k.act = act;
        run_norm<true>(k, type, workspace, as_stream(stream));
    });
}

}  // extern "C"

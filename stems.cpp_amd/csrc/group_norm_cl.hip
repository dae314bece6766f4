// group_norm_cl.hip — GroupNorm with an activation over channels-last tensors, forward and
// backward (stx_group_norm_cl, stx_group_norm_cl_back).
#include <algorithm>
#include <cmath>
#include <numeric>

#include "typed.hpp"

namespace stx {
namespace {

// One slice (ne3 index) is [T][C], dense. Threads move 16-byte vectors of V elements; so that a
// thread meets the same channels in every vector it takes whatever C is, the slice is walked in
// super-rows of R = V / gcd(C, V) rows, which hold a whole number of vectors: vector j of a
// super-row covers channels (j V + e) mod C. Accesses may be unaligned (odd C, odd slices); only
// the slice's last vector can be partial.
//
// A block has a tile of `cols` vector columns x `rws` super-rows at a time, and one chunk of the
// slice's super-rows. Three steps, forward and backward alike:
//   sums:  per (slice, chunk, slot = position in the super-row) two sums in double
//          (x, x^2 or dz, dz xhat); in double because E[x^2] - mean^2 cancels otherwise;
//   fold:  over chunks and the R slots of a channel, to [slice][C] pairs;
//   apply: each block adds the channels of the groups it needs from those pairs, then streams its
//          elements, one fused multiply-add and the activation each.
constexpr int kThreads = 256;

struct Geometry {
    long long B, T;
    int C, G, width;                     // groups of `width` channels, the last of what is left
    int V, R, slots, ncol;               // slots = C R = ncol V
    int cols, tiles, rws;                // columns of a block, column tiles, super-rows a block takes at once
    int chunks;
    long long srows, chunk_srows;        // super-rows of a slice, of a chunk
};

Geometry geometry(const stx_tensor* a, int size, int n_groups) {
    Geometry g{};
    g.C = (int)a->ne[0];
    g.T = a->ne[1] * a->ne[2];
    g.B = a->ne[3];
    g.G = n_groups;
    g.width = (g.C + n_groups - 1) / n_groups;
    g.V = 16 / size;
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
    // Chunks: enough blocks for eight a CU, each of at least 16 super-rows and 8 passes of its threads.
    const long long most = std::max(1LL, std::min(2048 / std::max(1LL, g.B * g.tiles), g.srows / std::max(16, 8 * g.rws)));
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
    double2* part;                       // [B][chunks][slots]
    double2* chan;                       // [B][C]
    float *dw, *db;
    double eps;
    int act;
};

template <class T, int V>
__device__ __forceinline__ void load_vec(const T* p, long long left, float (&f)[V]) {
    if (left >= V) {
        T v[V];
        __builtin_memcpy(v, p, sizeof v);
#pragma unroll
        for (int e = 0; e < V; e++) f[e] = to_f32(v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < V; e++) f[e] = e < left ? to_f32(p[e]) : 0.f;
    }
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
    long long slice, begin, end, chunk;
    int col, row;
    bool on;
};
__device__ __forceinline__ Place place(const NormArgs& a) {
    Place p;
    const unsigned bid = blockIdx.x;
    const unsigned bc = a.tiles.div(bid), tile = bid - bc * a.tiles.d;
    const unsigned b = a.chunks.div(bc);
    p.slice = b;
    p.chunk = bc - b * a.chunks.d;
    const int c = (int)threadIdx.x % a.g.cols;
    p.row = (int)threadIdx.x / a.g.cols;
    p.col = (int)tile * a.g.cols + c;
    p.begin = p.chunk * a.g.chunk_srows;
    p.end = min(p.begin + a.g.chunk_srows, a.g.srows);
    p.on = p.row < a.g.rws && p.col < a.g.ncol;
    return p;
}

// Per-channel constants of a normalisation: xhat = (x - mh) r - d, with mean = mh + the rest in d
// (a float mean alone would cost |mean| 2^-24 / std).
struct Chan {
    float mh, r, d, w, b;
};
__device__ __forceinline__ Chan chan_of(const NormArgs& a, double mean, double rstd, int c) {
    Chan k;
    k.mh = (float)mean;
    k.r = (float)rstd;
    k.d = (float)((mean - (double)k.mh) * rstd);
    k.w = a.w ? a.w[c] : 1.f;
    k.b = a.b ? a.b[c] : 0.f;
    return k;
}

template <class T, bool BACK, int ACT>
__global__ __launch_bounds__(kThreads) void gn_cl_sums_kernel(NormArgs a) {
    constexpr int V = 16 / sizeof(T);
    __shared__ double2 red[kThreads * V];
    const Place p = place(a);
    double s1[V] = {}, s2[V] = {};
    if (p.on) {
        const long long n = a.g.T * a.g.C;
        const T* x = static_cast<const T*>(a.x) + p.slice * n;
        const T* dy = static_cast<const T*>(a.dy) + p.slice * n;
        Chan k[V];
        if constexpr (BACK) {
#pragma unroll
            for (int e = 0; e < V; e++) {
                const int c = (p.col * V + e) % a.g.C;
                const double2 st = a.stats_in[p.slice * a.g.G + c / a.g.width];
                k[e] = chan_of(a, st.x, st.y, c);
            }
        }
        for (long long r = p.begin + p.row; r < p.end; r += a.g.rws) {
            const long long at = r * a.g.slots + (long long)p.col * V;
            float f[V];
            load_vec<T, V>(x + at, n - at, f);
            if constexpr (BACK) {
                float g[V];
                load_vec<T, V>(dy + at, n - at, g);
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const float xh = fmaf(f[e] - k[e].mh, k[e].r, -k[e].d);
                    float d;
                    (void)act_f32<ACT>(fmaf(xh, k[e].w, k[e].b), d);
                    const double dz = (double)(g[e] * d);        // past the end g is 0
                    s1[e] += at + e < n ? dz : 0.0;
                    s2[e] = at + e < n ? fma(dz, (double)xh, s2[e]) : s2[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const double d = (double)f[e];
                    s1[e] += d;
                    s2[e] = fma(d, d, s2[e]);
                }
            }
        }
    }
    const int width = a.g.cols * V;
#pragma unroll
    for (int e = 0; e < V; e++)
        if (p.row < a.g.rws) red[p.row * width + ((int)threadIdx.x % a.g.cols) * V + e] = make_double2(s1[e], s2[e]);
    __syncthreads();
    const int first = (p.col - (int)threadIdx.x % a.g.cols) * V;
    for (int i = (int)threadIdx.x; i < width && first + i < a.g.slots; i += kThreads) {
        double2 s = red[i];
        for (int r = 1; r < a.g.rws; r++) {
            s.x += red[r * width + i].x;
            s.y += red[r * width + i].y;
        }
        a.part[(p.slice * a.g.chunks + p.chunk) * a.g.slots + first + i] = s;
    }
}

// [B][chunks][R][C] -> [B][C]: 32 channels x 8 parts a block, in a fixed order.
__global__ __launch_bounds__(256) void gn_cl_fold_kernel(NormArgs a, FastDiv ctiles) {
    __shared__ double2 red[8][33];
    const unsigned b = ctiles.div(blockIdx.x);
    const int c = (int)(blockIdx.x - b * ctiles.d) * 32 + (int)threadIdx.x % 32, lane = (int)threadIdx.x / 32;
    double2 s = make_double2(0.0, 0.0);
    if (c < a.g.C) {
        const double2* p = a.part + (long long)b * a.g.chunks * a.g.slots + c;
        const int rows = a.g.srows ? a.g.chunks * a.g.R : 0;
        for (int i = lane; i < rows; i += 8) {
            const double2 v = p[(long long)i * a.g.C];
            s.x += v.x;
            s.y += v.y;
        }
    }
    red[lane][threadIdx.x % 32] = s;
    __syncthreads();
    if (lane == 0 && c < a.g.C) {
        for (int i = 1; i < 8; i++) {
            s.x += red[i][threadIdx.x].x;
            s.y += red[i][threadIdx.x].y;
        }
        a.chan[(long long)b * a.g.C + c] = s;
    }
}

// Group values a block's columns need: a wave adds the channels of a group (weighted in the
// backward pass, where the channel's xhat = dxhat / w).
template <bool BACK>
__device__ double2 group_total(const NormArgs& a, long long slice, int group) {
    const int lo = group * a.g.width, hi = min(lo + a.g.width, a.g.C);
    double2 s = make_double2(0.0, 0.0);
    for (int c = lo + (int)threadIdx.x % 64; c < hi; c += 64) {
        const double2 v = a.chan[slice * a.g.C + c];
        const double w = BACK && a.w ? (double)a.w[c] : 1.0;
        s.x = fma(v.x, w, s.x);
        s.y = fma(v.y, w, s.y);
    }
    s.x = lane_sum<64>(s.x);
    s.y = lane_sum<64>(s.y);
    return s;
}

__device__ __forceinline__ double2 moments(const NormArgs& a, double2 s, double n) {
    if (n == 0.0) return make_double2(0.0, 1.0 / sqrt(a.eps));
    const double mean = s.x / n;
    return make_double2(mean, 1.0 / sqrt(fmax(0.0, s.y / n - mean * mean) + a.eps));
}

template <class T, bool BACK, int ACT>
__global__ __launch_bounds__(kThreads) void gn_cl_apply_kernel(NormArgs a) {
    constexpr int V = 16 / sizeof(T);
    extern __shared__ double2 groups[];                  // [G]
    const Place p = place(a);
    // Every group of the slice (a column tile of odd C meets channels of several places).
    for (int g = (int)threadIdx.x / 64; g < a.g.G; g += kThreads / 64) {
        const double n = (double)a.g.T * (min((g + 1) * a.g.width, a.g.C) - g * a.g.width);
        const double2 s = group_total<BACK>(a, p.slice, g);
        if (threadIdx.x % 64 == 0) {
            groups[g] = BACK ? make_double2(s.x / n, s.y / n) : moments(a, s, n);
            if (!BACK && a.stats_out && p.chunk == 0 && p.col == (int)threadIdx.x % a.g.cols) a.stats_out[p.slice * a.g.G + g] = groups[g];
        }
    }
    __syncthreads();
    if (!p.on) return;
    const long long n = a.g.T * a.g.C;
    const T* x = static_cast<const T*>(a.x) + p.slice * n;
    const T* dy = static_cast<const T*>(a.dy) + p.slice * n;
    T* out = static_cast<T*>(a.out) + p.slice * n;
    Chan k[V];
    float k1[V], k2[V];
#pragma unroll
    for (int e = 0; e < V; e++) {
        const int c = (p.col * V + e) % a.g.C, g = c / a.g.width;
        if constexpr (BACK) {
            const double2 st = a.stats_in[p.slice * a.g.G + g];
            k[e] = chan_of(a, st.x, st.y, c);
            k1[e] = (float)(groups[g].x * st.y);
            k2[e] = (float)(groups[g].y * st.y);
        } else {
            k[e] = chan_of(a, groups[g].x, groups[g].y, c);
        }
    }
    for (long long r = p.begin + p.row; r < p.end; r += a.g.rws) {
        const long long at = r * a.g.slots + (long long)p.col * V;
        float f[V], y[V];
        load_vec<T, V>(x + at, n - at, f);
        if constexpr (BACK) {
            float g[V];
            load_vec<T, V>(dy + at, n - at, g);
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float xh = fmaf(f[e] - k[e].mh, k[e].r, -k[e].d);
                float d;
                (void)act_f32<ACT>(fmaf(xh, k[e].w, k[e].b), d);
                y[e] = fmaf(-xh, k2[e], fmaf(g[e] * d, k[e].r * k[e].w, -k1[e]));
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float xh = fmaf(f[e] - k[e].mh, k[e].r, -k[e].d);
                y[e] = act_f32<ACT>(fmaf(xh, k[e].w, k[e].b));
            }
        }
        if (at < n) store_vec<T, V>(out + at, n - at, y);
    }
}

// dbias and dweight: the channels' sums over the slices.
__global__ __launch_bounds__(256) void gn_cl_params_kernel(NormArgs a) {
    const int c = (int)(blockIdx.x * 256 + threadIdx.x);
    if (c >= a.g.C) return;
    double s1 = 0.0, s2 = 0.0;
    for (long long b = 0; b < a.g.B; b++) {
        const double2 v = a.chan[b * a.g.C + c];
        s1 += v.x;
        s2 += v.y;
    }
    if (a.db) a.db[c] = (float)s1;
    if (a.dw) a.dw[c] = (float)s2;
}

size_t chan_bytes(const Geometry& g) { return ((size_t)g.B * g.C * sizeof(double2) + 255) / 256 * 256; }
size_t workspace_bytes(const Geometry& g) { return chan_bytes(g) + (size_t)g.B * g.chunks * g.slots * sizeof(double2); }

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
    const Geometry g = geometry(a, size, n_groups);
    STX_REQUIRE(g.B * g.chunks * g.tiles < (1LL << 31) && g.B * ((C + 31) / 32) < (1LL << 31), "group_norm_cl: too many slices");
    return g;
}

template <bool BACK>
void run_norm(NormArgs& a, stx_type type, void* ws, hipStream_t stream) {
    const Geometry& g = a.g;
    a.chunks = FastDiv((unsigned)g.chunks);
    a.tiles = FastDiv((unsigned)g.tiles);
    a.chan = static_cast<double2*>(ws);
    a.part = reinterpret_cast<double2*>(static_cast<char*>(ws) + chan_bytes(g));
    const dim3 grid((unsigned)(g.B * g.chunks * g.tiles)), block(kThreads);
    const unsigned ctiles = (unsigned)((g.C + 31) / 32);
    with_type(type, [&](auto t) {
        using T = decltype(t);
        if (g.B == 0) return;
        if (g.srows) {
            if constexpr (BACK) with_act(a.act, [&](auto act) { hipLaunchKernelGGL((gn_cl_sums_kernel<T, true, act()>), grid, block, 0, stream, a); });
            else hipLaunchKernelGGL((gn_cl_sums_kernel<T, false, STX_ACT_NONE>), grid, block, 0, stream, a);
            launch_check("gn_cl_sums_kernel");
        }
        hipLaunchKernelGGL(gn_cl_fold_kernel, dim3((unsigned)g.B * ctiles), dim3(256), 0, stream, a, FastDiv(ctiles));
        launch_check("gn_cl_fold_kernel");
        if (BACK && !a.out) return;
        with_act(a.act, [&](auto act) { hipLaunchKernelGGL((gn_cl_apply_kernel<T, BACK, act()>), grid, block, sizeof(double2) * g.G, stream, a); });
        launch_check("gn_cl_apply_kernel");
    });
    if (BACK && (a.dw || a.db)) {
        hipLaunchKernelGGL(gn_cl_params_kernel, dim3((g.C + 255) / 256), dim3(256), 0, stream, a);
        launch_check("gn_cl_params_kernel");
    }
}

}  // namespace
}  // namespace stx

using namespace stx;

extern "C" {

STX_API size_t stx_group_norm_cl_workspace_size(const stx_tensor* a, stx_type type, int n_groups) {
    size_t bytes = 0;
    (void)guard([&] {
        STX_REQUIRE(a != nullptr, "group_norm_cl: a is NULL");
        stx_tensor t = *a;
        t.data = reinterpret_cast<void*>((uintptr_t)256);          // a query may have no data yet
        bytes = workspace_bytes(check_norm(&t, type, n_groups));
    });
    return bytes;
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
        check_workspace(workspace, workspace_bytes_, workspace_bytes(k.g), "group_norm_cl");
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
        check_workspace(workspace, workspace_bytes_, workspace_bytes(k.g), "group_norm_cl_back");
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

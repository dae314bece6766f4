// soft_max_rel.hip — the softmax of scores with a learned relative position bias by buckets, forward and
// backward (stx_soft_max_rel, stx_soft_max_rel_back).
#include <algorithm>
#include <cmath>

#include "rope_angles.hpp"

namespace stx {
namespace {

// Row i of head h: y_j = exp(z_j) / sum exp(z), z_j = scale x_j + table[bucket(j - at)][h], at = i + start, over the
// keys j < limit: the sequence's length and, causal, at + 1. Both masks end a row, so what is behind them is never
// read and zeros are written there. Gradient: g_j = y_j (dy_j - S), S = sum y dy; dx = scale g, and the table's is the
// sum of g over rows and keys of a bucket.
//
// One pass over memory, a row in the registers of some lanes of a wave, of a wave or of a block (rows of more
// than 2^14 16-bit or 2^13 32-bit scores are read twice), vectors of 16 bytes at any alignment. The bias
// costs no bytes: buckets change only where |j - at| is below the last edge `reach`, so a block keeps the head's
// biases by distance in LDS, and vectors beyond take a constant.
constexpr int kRelThreads = 256;
constexpr int kRelBuckets = 256;         // of a table
constexpr int kRelDistance = 2048;       // 2 kRelDistance + 1 distances in LDS
constexpr int kRelRows = 64;             // of a block, at most

struct RelArgs {
    const char *x, *dy;                  // backward: x is y
    char* out;
    long long x1, x2, x3, y1, y2, y3, o1, o2, o3;    // byte strides of x, dy and out
    const float* table;                  // [n_buckets][heads]
    double* part;                        // backward: sums of g, [block][n_buckets], or NULL
    const int *lengths, *starts;
    int n, queries;                      // keys, queries
    FastDiv heads, chunks;               // slice -> (i3, i2); block -> (slice, chunk of rows)
    unsigned base;                       // blocks of the launches before this one
    int rows, log_lanes;                 // rows of a block; lanes of a row of one wave
    int near, side, n_buckets;           // distances with a bucket each; buckets of a side; all
    int edge_count, reach;
    bool both, causal;
    float scale;
    int edges[kRelBuckets / 2];          // first distances of the buckets from `near` on; reach is the last
};

// Bucket of key position less query position.
__device__ __forceinline__ int bucket_of(const RelArgs& a, const int* edges, int rel) {
    const int d = a.both ? abs(rel) : max(-rel, 0);
    int k = d;
    if (d >= a.near) {
        int lo = 0, hi = a.edge_count;                               // edges[lo] <= d < edges[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (edges[mid] <= d) lo = mid;
            else hi = mid;
        }
        k = a.near + lo;
    }
    return k + (a.both && rel > 0 ? a.side : 0);
}

// What a block works on: rows [i0, i0 + rows) of slice (i2, i3).
struct RelBlock {
    int h, b, i0, rows, length;
    long long start;
    __device__ __forceinline__ explicit RelBlock(const RelArgs& a) {
        const unsigned block = a.base + blockIdx.x, slice = a.chunks.div(block);
        b = (int)a.heads.div(slice);
        h = (int)(slice - b * a.heads.d);
        i0 = (int)(block - slice * a.chunks.d) * a.rows;
        rows = min(a.rows, a.queries - i0);
        length = a.lengths ? min(max(a.lengths[b], 0), a.n) : a.n;
        start = a.starts ? a.starts[b] : 0;
    }
    __device__ __forceinline__ long long at(int r) const { return i0 + r + start; }
    __device__ __forceinline__ int limit(const RelArgs& a, int r) const {
        return a.causal ? (int)min((long long)length, max(0LL, at(r) + 1)) : length;
    }
};

template <class T>
constexpr int kVec = 16 / sizeof(T);

// V elements at p of which `left` exist; what is missing is 0.
template <class T>
__device__ __forceinline__ Pack<T, kVec<T>> load_row(const T* p, int left) {
    constexpr int V = kVec<T>;
    Pack<T, V> v;
    if (left >= V) {
        __builtin_memcpy(&v, p, sizeof v);
    } else {
#pragma unroll
        for (int e = 0; e < V; e++) {
            const T x = p[e < left ? e : 0];                         // left >= 1
            v.v[e] = e < left ? x : T(0.f);
        }
    }
    return v;
}
template <class T>
__device__ __forceinline__ void store_row(T* p, const Pack<T, kVec<T>>& v, int left) {
    if (left >= kVec<T>) {
        __builtin_memcpy(p, &v, sizeof v);
    } else {
#pragma unroll
        for (int e = 0; e < kVec<T>; e++)
            if (e < left) p[e] = v.v[e];
    }
}

// Values of a row's lanes combined, in every lane: of 2^log_lanes lanes of a wave, or (WAVES 4) of the block.
template <int WAVES, class V, class F>
__device__ __forceinline__ V over_waves(V v, V* red, F&& add) {
    if constexpr (WAVES == 1) return v;
    __syncthreads();                                                 // red is free
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = v;
    __syncthreads();
    V s = red[0];
#pragma unroll
    for (int w = 1; w < WAVES; w++) s = add(s, red[w]);
    return s;
}
template <int CTRL>
__device__ __forceinline__ float lane_of(float v) { return dpp_f32<CTRL>(v); }
__device__ __forceinline__ float max_over(float v, int lanes) {
    if (lanes >= 2) v = fmaxf(v, lane_of<0xB1>(v));
    if (lanes >= 4) v = fmaxf(v, lane_of<0x4E>(v));
    if (lanes >= 8) v = fmaxf(v, lane_of<0x141>(v));
    if (lanes >= 16) v = fmaxf(v, lane_of<0x140>(v));
    if (lanes >= 32) v = fmaxf(v, __shfl_xor(v, 16, 64));
    if (lanes >= 64) v = fmaxf(v, __shfl_xor(v, 32, 64));
    return v;
}
__device__ __forceinline__ float sum_over(float v, int lanes) {
    if (lanes >= 2) v += lane_of<0xB1>(v);
    if (lanes >= 4) v += lane_of<0x4E>(v);
    if (lanes >= 8) v += lane_of<0x141>(v);
    if (lanes >= 16) v += lane_of<0x140>(v);
    if (lanes >= 32) v += __shfl_xor(v, 16, 64);
    if (lanes >= 64) v += __shfl_xor(v, 32, 64);
    return v;
}

constexpr float kLog2e = 1.44269504088896340736f;

// Scores in units of log2, so that the exponential is the hardware's 2^y. K vectors a lane; 0: rows of any length.
template <class T, int WAVES, int K>
__global__ __launch_bounds__(kRelThreads) void soft_max_rel_kernel(RelArgs a) {
    constexpr int V = kVec<T>;
    extern __shared__ float near[];      // biases of distances -reach .. reach
    __shared__ int edges[kRelBuckets / 2];
    __shared__ float red[4];
    const RelBlock blk(a);
    for (int e = threadIdx.x; e < a.edge_count; e += kRelThreads) edges[e] = a.edges[e];
    __syncthreads();
    const int span = 2 * a.reach + 1;
    for (int e = threadIdx.x; e < span; e += kRelThreads)
        near[e] = a.table[(long long)bucket_of(a, edges, e - a.reach) * a.heads.d + blk.h] * kLog2e;
    __syncthreads();
    const float left = near[0], right = near[span - 1], scale = a.scale * kLog2e;
    const int lanes = WAVES == 1 ? 1 << a.log_lanes : kRelThreads, lane = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes;
    const char* xs = a.x + blk.h * a.x2 + blk.b * a.x3;
    char* os = a.out + blk.h * a.o2 + blk.b * a.o3;

    // The scores of vector c with their biases; -inf where there is no key.
    auto scores = [&](const Pack<T, V>& x, int c, long long at, int limit, float (&z)[V]) {
        const int j0 = c * V, rel = (int)min((long long)a.reach, max((long long)(-a.reach - V), j0 - at));
        if (rel >= a.reach || rel + V - 1 <= -a.reach) {
            const float bias = rel >= a.reach ? right : left;
#pragma unroll
            for (int e = 0; e < V; e++) z[e] = fmaf(to_f32(x.v[e]), scale, bias);
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) z[e] = fmaf(to_f32(x.v[e]), scale, near[min(max(rel + e, -a.reach), a.reach) + a.reach]);
        }
        if (j0 + V > limit) {
#pragma unroll
            for (int e = 0; e < V; e++) z[e] = j0 + e < limit ? z[e] : -__builtin_inff();
        }
    };
    const int vectors = (a.n + V - 1) / V;
    for (int r0 = 0; r0 < blk.rows; r0 += kRelThreads / lanes) {
        const int r = min(r0 + group, blk.rows - 1);
        const bool valid = r0 + group < blk.rows;
        const long long at = blk.at(r);
        const int limit = blk.limit(a, r);
        const T* x = reinterpret_cast<const T*>(xs + (long long)(blk.i0 + r) * a.x1);
        T* out = reinterpret_cast<T*>(os + (long long)(blk.i0 + r) * a.o1);
        if constexpr (K > 0) {
            Pack<T, V> raw[K];
            float z[K][V], m = -__builtin_inff(), s = 0.f;
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int c = lane + k * lanes;
                if (c * V < limit) raw[k] = load_row<T>(x + c * V, a.n - c * V);
            }
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int c = lane + k * lanes;
                if (c * V < limit) scores(raw[k], c, at, limit, z[k]);
                else
#pragma unroll
                    for (int e = 0; e < V; e++) z[k][e] = -__builtin_inff();
#pragma unroll
                for (int e = 0; e < V; e++) m = fmaxf(m, z[k][e]);
            }
            m = over_waves<WAVES>(max_over(m, min(lanes, 64)), red, [](float p, float q) { return fmaxf(p, q); });
            m = m == -__builtin_inff() ? 0.f : m;                    // a row of nothing: zeros
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int e = 0; e < V; e++) s += z[k][e] = __builtin_amdgcn_exp2f(z[k][e] - m);
            s = over_waves<WAVES>(sum_over(s, min(lanes, 64)), red, [](float p, float q) { return p + q; });
            const float inv = s == 0.f ? 0.f : 1.f / s;
            if (!valid) continue;
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int c = lane + k * lanes;
                if (c >= vectors) continue;
                Pack<T, V> y;
#pragma unroll
                for (int e = 0; e < V; e++) y.v[e] = from_f32<T>(z[k][e] * inv);
                store_row<T>(out + c * V, y, a.n - c * V);
            }
        } else {
            float m = -__builtin_inff(), s = 0.f, z[V];
            for (int c = lane; c * V < limit; c += lanes) {
                scores(load_row<T>(x + c * V, a.n - c * V), c, at, limit, z);
                float top = m;
#pragma unroll
                for (int e = 0; e < V; e++) top = fmaxf(top, z[e]);
                const float base = top == -__builtin_inff() ? 0.f : top;
                s *= __builtin_amdgcn_exp2f(m - base);
#pragma unroll
                for (int e = 0; e < V; e++) s += __builtin_amdgcn_exp2f(z[e] - base);
                m = top;
            }
            float top = over_waves<WAVES>(max_over(m, 64), red, [](float p, float q) { return fmaxf(p, q); });
            top = top == -__builtin_inff() ? 0.f : top;
            s = over_waves<WAVES>(sum_over(s * __builtin_amdgcn_exp2f(m - top), 64), red, [](float p, float q) { return p + q; });
            const float inv = s == 0.f ? 0.f : 1.f / s;
            for (int c = lane; c < vectors; c += lanes) {
                Pack<T, V> y{};
                if (c * V < limit) {
                    scores(load_row<T>(x + c * V, a.n - c * V), c, at, limit, z);
#pragma unroll
                    for (int e = 0; e < V; e++) y.v[e] = from_f32<T>(__builtin_amdgcn_exp2f(z[e] - top) * inv);
                }
                store_row<T>(out + c * V, y, a.n - c * V);
            }
        }
    }
}

// S, g and their sums are formed in double: a row's g add up to S (1 - sum y), nearly 0, and so does a bucket's
// share where most of the keys are in it. Keys beyond `reach` on either side are added up by the lanes that
// hold them. The rest, a band along the diagonal, is read again from the caches once the block's rows have
// their S: a thread takes four neighbouring distances and goes down the rows, so that every sum has one owner
// and one order (atomics in LDS would not, and have 16 lanes to a bank).
template <class T, int WAVES, int K>
__global__ __launch_bounds__(kRelThreads) void soft_max_rel_back_kernel(RelArgs a) {
    constexpr int V = kVec<T>, D = 4;
    extern __shared__ double band[];     // sums of distances -(reach - 1) .. reach - 1
    __shared__ double dots[kRelRows], far[2][4], red[4];
    const RelBlock blk(a);
    const int lanes = WAVES == 1 ? 1 << a.log_lanes : kRelThreads, lane = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes;
    const char *xs = a.x + blk.h * a.x2 + blk.b * a.x3, *ds = a.dy + blk.h * a.y2 + blk.b * a.y3;
    char* os = a.out ? a.out + blk.h * a.o2 + blk.b * a.o3 : nullptr;
    const int vectors = (a.n + V - 1) / V;
    double below = 0.0, above = 0.0;
    auto dot = [&](const Pack<T, V>& y, const Pack<T, V>& dy, int left, double s) {
#pragma unroll
        for (int e = 0; e < V; e++) s = e < left ? fma((double)to_f32(y.v[e]), (double)to_f32(dy.v[e]), s) : s;
        return s;
    };
    // dx of vector c, and its shares of the far sums.
    auto finish = [&](Pack<T, V> y, const Pack<T, V>& dy, int c, long long at, int limit, double s, T* out) {
        const int j0 = c * V, rel = (int)min((long long)a.reach, max((long long)(-a.reach - V), j0 - at)), left = limit - j0;
        double g[V];
#pragma unroll
        for (int e = 0; e < V; e++) {
            g[e] = e < left ? (double)to_f32(y.v[e]) * ((double)to_f32(dy.v[e]) - s) : 0.0;
            y.v[e] = from_f32<T>((float)(a.scale * g[e]));
        }
        if (rel <= -a.reach) {
#pragma unroll
            for (int e = 0; e < V; e++) below += rel + e <= -a.reach ? g[e] : 0.0;
        }
        if (rel + V > a.reach) {
#pragma unroll
            for (int e = 0; e < V; e++) above += rel + e >= a.reach ? g[e] : 0.0;
        }
        if (out) store_row<T>(out + j0, y, a.n - j0);
    };
    for (int r0 = 0; r0 < blk.rows; r0 += kRelThreads / lanes) {
        const int r = min(r0 + group, blk.rows - 1);
        const bool valid = r0 + group < blk.rows;
        const long long at = blk.at(r), row = blk.i0 + r;
        const int limit = blk.limit(a, r);
        const T *y = reinterpret_cast<const T*>(xs + row * a.x1), *dy = reinterpret_cast<const T*>(ds + row * a.y1);
        T* out = os ? reinterpret_cast<T*>(os + row * a.o1) : nullptr;
        double s = 0.0;
        Pack<T, V> py[K > 0 ? K : 1], pd[K > 0 ? K : 1];
        if constexpr (K > 0) {
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int c = lane + k * lanes;
                py[k] = pd[k] = Pack<T, V>{};
                if (c * V >= limit) continue;
                py[k] = load_row<T>(y + c * V, a.n - c * V);
                pd[k] = load_row<T>(dy + c * V, a.n - c * V);
            }
#pragma unroll
            for (int k = 0; k < K; k++) s = dot(py[k], pd[k], limit - (lane + k * lanes) * V, s);
        } else {
            for (int c = lane; c * V < limit; c += lanes) s = dot(load_row<T>(y + c * V, a.n - c * V), load_row<T>(dy + c * V, a.n - c * V), limit - c * V, s);
        }
        s = over_waves<WAVES>(lane_sum_dyn(s, min(lanes, 64)), red, [](double p, double q) { return p + q; });
        if (!valid) continue;
        if (lane == 0) dots[r] = s;
        if constexpr (K > 0) {
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int c = lane + k * lanes;
                if (c < vectors) finish(py[k], pd[k], c, at, limit, s, out);
            }
        } else {
            for (int c = lane; c < vectors; c += lanes) {
                const bool some = c * V < limit;
                Pack<T, V> p{}, d{};
                if (some) p = load_row<T>(y + c * V, a.n - c * V), d = load_row<T>(dy + c * V, a.n - c * V);
                finish(p, d, c, at, limit, s, out);
            }
        }
    }
    if (!a.part) return;
    below = lane_sum<64>(below);
    above = lane_sum<64>(above);
    if (threadIdx.x % 64 == 0) far[0][threadIdx.x / 64] = below, far[1][threadIdx.x / 64] = above;
    __syncthreads();
    const int width = 2 * a.reach - 1;
    for (int s0 = threadIdx.x * D; s0 < width; s0 += kRelThreads * D) {
        double acc[D] = {};
#pragma unroll 4
        for (int r = 0; r < blk.rows; r++) {
            const long long j = blk.at(r) + s0 - (a.reach - 1);
            const int limit = blk.limit(a, r), count = min(D, width - s0);
            if (j + count <= 0 || j >= limit) continue;
            const long long row = blk.i0 + r;
            const T *y = reinterpret_cast<const T*>(xs + row * a.x1), *dy = reinterpret_cast<const T*>(ds + row * a.y1);
            Pack<T, D> p, d;
            const bool whole = j >= 0 && j + D <= limit;
            if (whole) {
                __builtin_memcpy(&p, y + j, sizeof p);
                __builtin_memcpy(&d, dy + j, sizeof d);
            } else {
#pragma unroll
                for (int e = 0; e < D; e++) {
                    const bool in = j + e >= 0 && j + e < limit;
                    p.v[e] = in ? y[j + e] : T(0.f);
                    d.v[e] = in ? dy[j + e] : T(0.f);
                }
            }
#pragma unroll
            for (int e = 0; e < D; e++) {
                const double g = (double)to_f32(p.v[e]) * ((double)to_f32(d.v[e]) - dots[r]);
                acc[e] += whole || (j + e >= 0 && j + e < limit) ? g : 0.0;
            }
        }
#pragma unroll
        for (int e = 0; e < D; e++)
            if (s0 + e < width) band[s0 + e] = acc[e];
    }
    __syncthreads();
    // A wave takes a bucket: distances [first, end) before the query (after it from `side` on).
    double* part = a.part + (long long)(a.base + blockIdx.x) * a.n_buckets;
    const int wave_lane = threadIdx.x % 64, mid = a.reach - 1;
    for (int k = threadIdx.x / 64; k < a.n_buckets; k += kRelThreads / 64) {
        const bool after = a.both && k >= a.side;
        const int i = after ? k - a.side : k;
        auto first_of = [&](int i) { return i < a.near ? i : i - a.near < a.edge_count ? a.edges[i - a.near] : a.reach; };
        const int first = after ? max(1, first_of(i)) : first_of(i), end = min(first_of(i + 1), a.reach);
        double s = 0.0;
        for (int d = first + wave_lane; d < end; d += 64) s += band[after ? mid + d : mid - d];
        if (!a.both && k == 0)
            for (int d = 1 + wave_lane; d < a.reach; d += 64) s += band[mid + d];
        s = lane_sum<64>(s);
        if (i == a.side - 1) s += after ? (far[1][0] + far[1][1]) + (far[1][2] + far[1][3]) : (far[0][0] + far[0][1]) + (far[0][2] + far[0][3]);
        if (!a.both && k == 0) s += (far[1][0] + far[1][1]) + (far[1][2] + far[1][3]);
        if (wave_lane == 0) part[k] = s;
    }
}

// The table's gradient: sums over a head's blocks in order; 32 buckets x 32 lanes a block.
__global__ __launch_bounds__(1024) void rel_fold_kernel(const double* part, long long batch, int heads, int chunks, int n_buckets, float* dtable) {
    __shared__ double red[32][33];
    const int k = blockIdx.x * 32 + threadIdx.x % 32, h = blockIdx.y, lane = threadIdx.x / 32;
    double s = 0.0;
    if (k < n_buckets) {
        for (long long b = 0; b < batch; b++)
#pragma unroll 4
            for (int c = lane; c < chunks; c += 32) s += part[((b * heads + h) * chunks + c) * n_buckets + k];
    }
    red[lane][threadIdx.x % 32] = s;
    __syncthreads();
    if (lane || k >= n_buckets) return;
    for (int i = 1; i < 32; i++) s += red[i][threadIdx.x];
    dtable[(long long)k * heads + h] = (float)s;
}

// --------------------------------------------------------------------------------- host
// n^m compared with p^(m - k) q^k, in whole numbers.
bool power_reaches(long long n, int m, long long p, long long q, int k) {
    struct Big {
        std::vector<unsigned> d{1};
        void mul(unsigned f) {
            unsigned long long carry = 0;
            for (unsigned& x : d) {
                carry += (unsigned long long)x * f;
                x = (unsigned)carry;
                carry >>= 32;
            }
            if (carry) d.push_back((unsigned)carry);
        }
    } a, b;
    for (int i = 0; i < m; i++) {
        a.mul((unsigned)n);
        b.mul((unsigned)(i < k ? q : p));
    }
    if (a.d.size() != b.d.size()) return a.d.size() > b.d.size();
    for (size_t i = a.d.size(); i-- > 0;)
        if (a.d[i] != b.d[i]) return a.d[i] > b.d[i];
    return true;
}

void set_buckets(RelArgs& a, const stx_rel_params* p, const char* op) {
    STX_REQUIRE(p != nullptr && p->size >= sizeof(stx_rel_params), "%s: params are NULL or their size is too small", op);
    a.both = p->bidirectional != 0;
    a.causal = p->causal != 0;
    STX_REQUIRE(p->n_buckets >= (a.both ? 4 : 2) && (!a.both || p->n_buckets % 2 == 0), "%s: %d buckets", op, p->n_buckets);
    a.n_buckets = p->n_buckets;
    a.side = a.both ? p->n_buckets / 2 : p->n_buckets;
    a.near = a.side / 2;
    STX_REQUIRE(p->max_distance > a.near, "%s: max_distance %d is not above the %d distances with a bucket each", op, p->max_distance, a.near);
    if (p->n_buckets > kRelBuckets || p->max_distance > kRelDistance)
        fail(STX_STATUS_UNSUPPORTED, "%s: %d buckets up to distance %d (%d and %d at most)", op, p->n_buckets, p->max_distance, kRelBuckets, kRelDistance);
    a.edge_count = a.side - a.near;
    a.edges[0] = a.near;
    // Edges are found in double, and in whole numbers where that is too close to one to tell.
    for (int k = 1; k < a.edge_count; k++) {
        const double v = a.near * std::pow((double)p->max_distance / a.near, (double)k / a.edge_count), r = std::round(v);
        a.edges[k] = (int)(std::fabs(v - r) > 1e-9 * v ? std::ceil(v) : power_reaches((long long)r, a.edge_count, a.near, p->max_distance, k) ? r : r + 1);
    }
    a.reach = a.edges[a.edge_count - 1];
}

// Rows of the scores: shape, and how a block goes over them.
struct RelShape {
    long long n, queries, heads, batch;
    int waves, vectors, log_lanes;       // waves of a row, vectors a lane (0: any number)
    int rows;                            // of a block
    long long chunks() const { return (queries + rows - 1) / rows; }
    long long blocks() const { return chunks() * heads * batch; }
    bool empty() const { return n == 0 || queries == 0 || heads == 0 || batch == 0; }
};
RelShape rel_shape(const stx_tensor* x, int size, bool back, const char* op) {
    RelShape s{x->ne[0], x->ne[1], x->ne[2], x->ne[3], 1, 1, 0, 1};
    if (s.empty()) return s;
    STX_REQUIRE(s.n < (1LL << 30) && s.queries < (1LL << 30), "%s: %lld keys, %lld queries", op, s.n, s.queries);
    STX_REQUIRE(s.heads < (1LL << 24) && s.batch < (1LL << 24) && s.heads * s.batch < (1LL << 31), "%s: too many heads and sequences", op);
    const long long v = (s.n + 16 / size - 1) / (16 / size);
    while (s.log_lanes < 6 && (1 << s.log_lanes) < v) s.log_lanes++;
    if (v > 64) {
        s.waves = v > 256 ? 4 : 1;
        const long long lanes = s.waves * 64;
        s.vectors = v <= 2 * lanes ? 2 : v <= 4 * lanes ? 4 : v <= 8 * lanes ? 8 : 0;
    }
    // As many rows a block as leave four blocks a CU, of which each forms the head's biases or sums once.
    const long long round = s.waves == 1 ? kRelThreads >> s.log_lanes : 1, all = s.queries * s.heads * s.batch;
    const long long rows = std::max(round, std::min<long long>(kRelRows, all / (4 * 256)));
    s.rows = (int)std::min<long long>(std::min<long long>(back ? kRelRows : 1 << 20, rows), s.queries);
    STX_REQUIRE(s.blocks() < (1LL << 31), "%s: too many rows", op);
    return s;
}

template <class F>
void with_row(const RelShape& s, F&& f) {
    using std::integral_constant;
    constexpr integral_constant<int, 1> one{};
    constexpr integral_constant<int, 4> four{};
    if (s.waves == 1) {
        if (s.vectors == 1) f(one, one);
        else if (s.vectors == 2) f(one, integral_constant<int, 2>{});
        else f(one, four);
    } else if (s.vectors == 2) f(four, integral_constant<int, 2>{});
    else if (s.vectors == 4) f(four, four);
    else if (s.vectors == 8) f(four, integral_constant<int, 8>{});
    else f(four, integral_constant<int, 0>{});
}

void set_shape(RelArgs& a, const RelShape& s, const int32_t* lengths, const int32_t* starts, float scale) {
    a.lengths = lengths;
    a.starts = starts;
    a.n = (int)s.n;
    a.queries = (int)s.queries;
    a.heads = FastDiv((unsigned)s.heads);
    a.chunks = FastDiv((unsigned)s.chunks());
    a.rows = s.rows;
    a.log_lanes = s.log_lanes;
    a.scale = scale;
}

void soft_max_rel(const stx_tensor* x, stx_type type, const float* table, const stx_rel_params* p, float scale, const int32_t* lengths,
                  const int32_t* starts, const stx_tensor* dst, stx_stream stream) {
    const char* op = "soft_max_rel";
    const int size = type_size(type);
    check_row_output(x, dst, size, op);
    RelArgs a{};
    set_buckets(a, p, op);
    STX_REQUIRE(std::isfinite(scale), "%s: scale is not finite", op);
    const RelShape s = rel_shape(x, size, false, op);
    const size_t per = (size_t)x->ne[3] * sizeof(int32_t);
    check_apart(op, {{"dst", dst, size}}, {{"table", table, (size_t)a.n_buckets * x->ne[2] * sizeof(float)}, {"lengths", lengths, per}, {"starts", starts, per}});
    if (s.empty()) return;
    STX_REQUIRE(table != nullptr, "%s: table is NULL", op);
    set_shape(a, s, lengths, starts, scale);
    a.table = table;
    a.x = static_cast<const char*>(x->data);
    a.x1 = x->nb[1], a.x2 = x->nb[2], a.x3 = x->nb[3];
    a.out = static_cast<char*>(dst->data);
    a.o1 = dst->nb[1], a.o2 = dst->nb[2], a.o3 = dst->nb[3];
    with_type(type, [&](auto t) {
        using T = decltype(t);
        with_row(s, [&](auto waves, auto k) {
            launch_all(s.blocks(), [&](dim3 grid, unsigned first) {
                a.base = first;
                hipLaunchKernelGGL((soft_max_rel_kernel<T, waves(), k()>), grid, dim3(kRelThreads), sizeof(float) * (2 * a.reach + 1), as_stream(stream), a);
                launch_check("soft_max_rel_kernel");
            });
        });
    });
}

void soft_max_rel_back(const stx_tensor* dy, const stx_tensor* y, stx_type type, const stx_rel_params* p, float scale, const int32_t* lengths,
                       const int32_t* starts, const stx_tensor* dx, float* dtable, void* ws, size_t ws_bytes, stx_stream stream) {
    const char* op = "soft_max_rel_back";
    const int size = type_size(type);
    check_typed(y, size, "soft_max_rel_back: y");
    check_typed(dy, size, "soft_max_rel_back: dy");
    check_same_shape(y, dy, "soft_max_rel_back: dy");
    if (dx) check_row_output(y, dx, size, "soft_max_rel_back: dx");
    RelArgs a{};
    set_buckets(a, p, op);
    STX_REQUIRE(std::isfinite(scale), "%s: scale is not finite", op);
    const RelShape s = rel_shape(y, size, true, op);
    const size_t need = dtable && !s.empty() ? (size_t)s.blocks() * a.n_buckets * sizeof(double) : 0, per = (size_t)y->ne[3] * sizeof(int32_t);
    const size_t table = (size_t)a.n_buckets * y->ne[2] * sizeof(float);
    check_workspace(ws, ws_bytes, need, op);
    check_apart(op, {{"dx", dx, size}, {"dtable", dtable, table}, {"the workspace", need ? ws : nullptr, need}},
                {{"dy", dy, size}, {"y", y, size}, {"lengths", lengths, per}, {"starts", starts, per}});
    STX_REQUIRE(s.heads < 65536, "%s: more than 65,535 heads", op);
    if (!dx && !dtable) return;
    a.part = dtable ? static_cast<double*>(ws) : nullptr;
    if (!s.empty()) {
        set_shape(a, s, lengths, starts, scale);
        a.x = static_cast<const char*>(y->data);
        a.x1 = y->nb[1], a.x2 = y->nb[2], a.x3 = y->nb[3];
        a.dy = static_cast<const char*>(dy->data);
        a.y1 = dy->nb[1], a.y2 = dy->nb[2], a.y3 = dy->nb[3];
        if (dx) {
            a.out = static_cast<char*>(dx->data);
            a.o1 = dx->nb[1], a.o2 = dx->nb[2], a.o3 = dx->nb[3];
        }
        with_type(type, [&](auto t) {
            using T = decltype(t);
            with_row(s, [&](auto waves, auto k) {
                launch_all(s.blocks(), [&](dim3 grid, unsigned first) {
                    a.base = first;
                    hipLaunchKernelGGL((soft_max_rel_back_kernel<T, waves(), k()>), grid, dim3(kRelThreads), sizeof(double) * (2 * a.reach - 1),
                                       as_stream(stream), a);
                    launch_check("soft_max_rel_back_kernel");
                });
            });
        });
    }
    if (!dtable || s.heads == 0) return;
    hipLaunchKernelGGL(rel_fold_kernel, dim3((a.n_buckets + 31) / 32, (unsigned)s.heads), dim3(1024), 0, as_stream(stream), a.part, s.empty() ? 0 : s.batch,
                       (int)s.heads, s.empty() ? 0 : (int)s.chunks(), a.n_buckets, dtable);
    launch_check("rel_fold_kernel");
}

}  // namespace
}  // namespace stx

using namespace stx;

extern "C" {

STX_API stx_status stx_soft_max_rel(const stx_tensor* x, stx_type type, const float* table, const stx_rel_params* params, float scale,
                                    const int32_t* lengths, const int32_t* starts, const stx_tensor* dst, stx_stream stream) {
    return guard([&] { soft_max_rel(x, type, table, params, scale, lengths, starts, dst, stream); });
}

STX_API size_t stx_soft_max_rel_back_workspace_size(const stx_tensor* y, stx_type type, int n_buckets) {
    size_t bytes = 0;
    (void)guard([&] {
        const int size = type_size(type);
        STX_REQUIRE(y != nullptr && n_buckets > 0 && n_buckets <= kRelBuckets, "soft_max_rel_back_workspace_size: y is NULL, or %d buckets", n_buckets);
        for (int i = 0; i < 4; i++) STX_REQUIRE(y->ne[i] >= 0, "soft_max_rel_back_workspace_size: negative ne[%d]", i);
        const RelShape s = rel_shape(y, size, true, "soft_max_rel_back_workspace_size");
        if (!s.empty()) bytes = (size_t)s.blocks() * n_buckets * sizeof(double);
    });
    return bytes;
}

STX_API stx_status stx_soft_max_rel_back(const stx_tensor* dy, const stx_tensor* y, stx_type type, const stx_rel_params* params, float scale,
                                         const int32_t* lengths, const int32_t* starts, const stx_tensor* dx, float* dtable, void* workspace,
                                         size_t workspace_bytes, stx_stream stream) {
    return guard([&] { soft_max_rel_back(dy, y, type, params, scale, lengths, starts, dx, dtable, workspace, workspace_bytes, stream); });
}

}  // extern "C"

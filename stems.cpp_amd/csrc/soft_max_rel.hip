// soft_max_rel.hip — the softmax of scores with a learned relative position bias by buckets, forward and
// backward (stx_soft_max_rel, stx_soft_max_rel_back).
#include <algorithm>
#include <cmath>

#include "typed.hpp"

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
// HBM bounds both, vector units 68 to 78 % busy beside it: 8 x 1,344 x 1,344 fp32 scores (116 MB) 26 us, 4.5 TB/s; gradients
// of 8 x 8,192 x 8,192 bf16 scores (3.2 GB) 718 us, 4.5 TB/s, and of 12 x 8 x 801 x 801 fp32 scores of ragged lengths 161 us,
// 3.9 TB/s (rows at no alignment). 8 clips of one query: 5.2 us.
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
    FastDiv chunks, blocks;              // item -> (sequence, chunk of rows); block -> (head, items)
    int heads, items, each;              // items of a head, and of a block
    unsigned base;                       // blocks of the launches before this one
    int rows, log_lanes;                 // rows of an item; lanes of a row of one wave
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

// A block works on items of one head, each rows [i0, i0 + rows) of a sequence.
struct RelItem {
    int b, i0, rows, length;
    long long start;
    __device__ __forceinline__ RelItem(const RelArgs& a, int item) {
        b = (int)a.chunks.div((unsigned)item);
        i0 = (int)((unsigned)item - b * a.chunks.d) * a.rows;
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

// Vector c of a row of n >= V elements starts at min(c V, n - V): the last one is moved back over the one before, so that no
// load or store is in part (branches for those took longer than the exponentials). Its elements below `lo` are the
// other's: they are left out of sums, and stored twice where both have the same bits; those from `hi` on are masked. Vectors that see no key read the last that does.
template <int V>
struct Place {
    int j0, lo, hi, from;
    __device__ __forceinline__ Place(int c, int n, int limit)
        : j0(min(c * V, n - V)), lo(min(c * V - j0, V)), hi(limit - j0), from(hi > 0 ? j0 : min(max(limit - V, 0), n - V)) {}
};
template <class T>
__device__ __forceinline__ Pack<T, kVec<T>> load_vector(const T* p) {
    Pack<T, kVec<T>> v;
    __builtin_memcpy(&v, p, sizeof v);
    return v;
}
template <class T>
__device__ __forceinline__ void store_vector(T* p, const Pack<T, kVec<T>>& v) { __builtin_memcpy(p, &v, sizeof v); }
__device__ __forceinline__ bool every(bool b) { return __builtin_amdgcn_ballot_w64(!b) == 0; }

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

// e^v, of a score less the row's largest: in that order, since the type's lowest values, which hide keys too, times log2 e are
// infinite, and a row of them alone is a row of equal scores.
__device__ __forceinline__ float natural_exp(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504088896340736f); }
constexpr float kLowest = -0x1.fffffep127f;

// A row's maximum and sum of exponentials, of a wave's lanes already, over the block's waves: an exchange of both at
// once, in one of two places by turns, so that one barrier a row is enough.
template <int WAVES>
__device__ __forceinline__ void join_waves(float& m, float& s, float2 (&red)[2][4], int turn) {
    if constexpr (WAVES > 1) {
        if (threadIdx.x % 64 == 0) red[turn][threadIdx.x / 64] = make_float2(m, s);
        __syncthreads();
        float top = red[turn][0].x;
#pragma unroll
        for (int w = 1; w < WAVES; w++) top = fmaxf(top, red[turn][w].x);
        s = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) s += red[turn][w].y * natural_exp(red[turn][w].x - top);
        m = top;
    }
}

// K vectors a lane, those of the next row on their way while one is worked on; K 0: rows of any length, read twice.
template <class T, int WAVES, int K>
__global__ __launch_bounds__(kRelThreads) void soft_max_rel_kernel(RelArgs a) {
    constexpr int V = kVec<T>;
    extern __shared__ float near[];      // biases of distances -reach .. reach
    __shared__ int edges[kRelBuckets / 2];
    __shared__ float2 red[2][4];
    const unsigned block = a.base + blockIdx.x, h = a.blocks.div(block);
    const int item0 = (int)(block - h * a.blocks.d) * a.each, item1 = min(item0 + a.each, a.items);
    for (int e = threadIdx.x; e < a.edge_count; e += kRelThreads) edges[e] = a.edges[e];
    __syncthreads();
    const int span = 2 * a.reach + 1;
    for (int e = threadIdx.x; e < span; e += kRelThreads)
        near[e] = a.table[(long long)bucket_of(a, edges, e - a.reach) * a.heads + h];
    __syncthreads();
    const float left = near[0], right = near[span - 1], scale = a.scale;
    const int lanes = WAVES == 1 ? 1 << a.log_lanes : kRelThreads, lane = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes;
    const int vectors = (a.n + V - 1) / V, rounds = kRelThreads / lanes;

    // The scores from key j0 on with their biases.
    auto scores = [&](const Pack<T, V>& x, int j0, long long at, float (&z)[V]) {
        const int rel = (int)min((long long)a.reach, max((long long)(-a.reach - V), j0 - at));
        if (every(rel >= a.reach || rel + V - 1 <= -a.reach)) {
            const float bias = rel >= a.reach ? right : left;
#pragma unroll
            for (int e = 0; e < V; e++) z[e] = fmaf(to_f32(x.v[e]), scale, bias);
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) z[e] = fmaf(to_f32(x.v[e]), scale, near[min(max(rel + e, -a.reach), a.reach) + a.reach]);
        }
    };
    // Those past `hi` are no keys.
    auto hide = [&](int hi, float (&z)[V]) {
#pragma unroll
        for (int e = 0; e < V; e++) z[e] = e < hi ? z[e] : -__builtin_inff();
    };
    int turn = 0;
    for (int item = item0; item < item1; item++) {
        const RelItem it(a, item);
        const char* xs = a.x + h * a.x2 + it.b * a.x3 + it.i0 * a.x1;
        char* os = a.out + h * a.o2 + it.b * a.o3 + it.i0 * a.o1;
        Pack<T, V> raw[K > 0 ? K : 1], next[K > 0 ? K : 1];
        auto load = [&](int r, Pack<T, V>* to) {
            const int limit = it.limit(a, r);
            const T* x = reinterpret_cast<const T*>(xs + r * a.x1);
#pragma unroll
            for (int k = 0; k < K; k++) to[k] = load_vector(x + Place<V>(lane + k * lanes, a.n, limit).from);
        };
        if constexpr (K > 0) load(min(group, it.rows - 1), next);
        for (int r0 = 0; r0 < it.rows; r0 += rounds) {
            const int r = min(r0 + group, it.rows - 1);
            const bool valid = r0 + group < it.rows;
            const long long at = it.at(r);
            const int limit = K > 0 || valid ? it.limit(a, r) : 0;       // K 0 in place: a row is its lanes' alone
            T* out = reinterpret_cast<T*>(os + r * a.o1);
            float m = -__builtin_inff(), s = 0.f;
            turn ^= 1;
            if constexpr (K > 0) {
                float z[K][V];
#pragma unroll
                for (int k = 0; k < K; k++) raw[k] = next[k];
                if (r0 + rounds < it.rows) load(min(r0 + rounds + group, it.rows - 1), next);
#pragma unroll
                for (int k = 0; k < K; k++) {
                    const Place<V> at_k(lane + k * lanes, a.n, limit);
                    scores(raw[k], at_k.j0, at, z[k]);
                    if (!every(at_k.hi >= V)) hide(at_k.hi, z[k]);
#pragma unroll
                    for (int e = 0; e < V; e++) m = fmaxf(m, z[k][e]);
                }
                m = max_over(m, min(lanes, 64));
                m = m == -__builtin_inff() ? kLowest : m;            // a row of nothing: zeros
                const float mine = m;
#pragma unroll
                for (int k = 0; k < K; k++) {
                    const int lo = Place<V>(lane + k * lanes, a.n, limit).lo;
#pragma unroll
                    for (int e = 0; e < V; e++) z[k][e] = natural_exp(z[k][e] - mine);
                    if (every(lo == 0)) {
#pragma unroll
                        for (int e = 0; e < V; e++) s += z[k][e];
                    } else {
#pragma unroll
                        for (int e = 0; e < V; e++) s += e < lo ? 0.f : z[k][e];
                    }
                }
                s = sum_over(s, min(lanes, 64));
                join_waves<WAVES>(m, s, red, turn);
                const float inv = s == 0.f ? 0.f : (WAVES > 1 ? natural_exp(mine - m) : 1.f) / s;
                if (!valid) continue;
#pragma unroll
                for (int k = 0; k < K; k++) {
                    const int c = lane + k * lanes;
                    if (c >= vectors) continue;
                    Pack<T, V> y;
#pragma unroll
                    for (int e = 0; e < V; e++) y.v[e] = from_f32<T>(z[k][e] * inv);
                    const Place<V> at_k(c, a.n, limit);
                    if (WAVES == 1 || at_k.lo == 0) {
                        store_vector(out + at_k.j0, y);
                    } else {                                         // another wave, with a maximum of its own, stores the others
#pragma unroll
                        for (int e = 0; e < V; e++)
                            if (e >= at_k.lo) out[at_k.j0 + e] = y.v[e];
                    }
                }
            } else {
                const T* x = reinterpret_cast<const T*>(xs + r * a.x1);
                float z[V];
                for (int c = lane; c * V < limit; c += lanes) {
                    scores(load_row<T>(x + c * V, a.n - c * V), c * V, at, z);
                    hide(limit - c * V, z);
                    float top = m;
#pragma unroll
                    for (int e = 0; e < V; e++) top = fmaxf(top, z[e]);
                    const float base = top == -__builtin_inff() ? 0.f : top;
                    s *= natural_exp(m - base);
#pragma unroll
                    for (int e = 0; e < V; e++) s += natural_exp(z[e] - base);
                    m = top;
                }
                float top = max_over(m, min(lanes, 64));
                top = top == -__builtin_inff() ? kLowest : top;
                s = sum_over(s * natural_exp(m - top), min(lanes, 64));
                join_waves<WAVES>(top, s, red, turn);
                const float inv = s == 0.f ? 0.f : 1.f / s;
                if (!valid) continue;
                for (int c = lane; c < vectors; c += lanes) {
                    Pack<T, V> y{};
                    if (c * V < limit) {
                        scores(load_row<T>(x + c * V, a.n - c * V), c * V, at, z);
                        hide(limit - c * V, z);
#pragma unroll
                        for (int e = 0; e < V; e++) y.v[e] = from_f32<T>(natural_exp(z[e] - top) * inv);
                    }
                    store_row<T>(out + c * V, y, a.n - c * V);
                }
            }
        }
    }
}

// S, g and their sums are formed in double: a row's g add up to S (1 - sum y), nearly 0, and so does a bucket's share
// where most of the keys are in it (in float where 16-bit data allow it: 794 us instead of 797). Keys beyond `reach` on
// either side are added up by the lanes that hold them. The rest, a band along the diagonal, is read again from the
// caches once an item's rows have their S: a thread takes four neighbouring distances and goes down the rows, every
// G-th where the band leaves threads over, so that every sum has one owner and one order (atomics in LDS would not, and
// have 16 lanes to a bank). Sums are kept over the block's items: a head's.
template <class T>
__device__ __forceinline__ double term(T y, T dy, double s) { return (double)to_f32(y) * ((double)to_f32(dy) - s); }

template <class T, int WAVES, int K>
__global__ __launch_bounds__(kRelThreads) void soft_max_rel_back_kernel(RelArgs a) {
    constexpr int V = kVec<T>, D = 4;
    extern __shared__ double band[];     // sums of distances -(reach - 1) .. reach - 1, G of each
    __shared__ double dots[kRelRows], far[2][4], red[2][4];
    const unsigned block = a.base + blockIdx.x, h = a.blocks.div(block);
    const int item0 = (int)(block - h * a.blocks.d) * a.each, item1 = min(item0 + a.each, a.items);
    const int lanes = WAVES == 1 ? 1 << a.log_lanes : kRelThreads, lane = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes;
    const int vectors = (a.n + V - 1) / V, rounds = kRelThreads / lanes;
    const int width = 2 * a.reach - 1, slots = (width + D - 1) / D, G = max(1, kRelThreads / slots);
    if (a.part)
        for (int e = threadIdx.x; e < G * slots * D; e += kRelThreads) band[e] = 0.0;
    double below = 0.0, above = 0.0;
    // Elements [lo, hi) count.
    auto dot = [&](const Pack<T, V>& y, const Pack<T, V>& dy, int lo, int hi, double s) {
        if (every(lo == 0 && hi >= V)) {
#pragma unroll
            for (int e = 0; e < V; e++) s = fma((double)to_f32(y.v[e]), (double)to_f32(dy.v[e]), s);
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) s = e >= lo && e < hi ? fma((double)to_f32(y.v[e]), (double)to_f32(dy.v[e]), s) : s;
        }
        return s;
    };
    // dx of the vector at j0, and its shares of the far sums.
    auto finish = [&](Pack<T, V> y, const Pack<T, V>& dy, int j0, int lo, int hi, long long at, double s) {
        double g[V];
#pragma unroll
        for (int e = 0; e < V; e++) g[e] = term(y.v[e], dy.v[e], s);
        if (!every(hi >= V)) {
#pragma unroll
            for (int e = 0; e < V; e++) g[e] = e < hi ? g[e] : 0;
        }
#pragma unroll
        for (int e = 0; e < V; e++) y.v[e] = from_f32<T>((float)(a.scale * g[e]));
        if (a.part) {
            const int rel = (int)min((long long)a.reach, max((long long)(-a.reach - V), j0 - at));
            if (every(lo == 0 && (rel >= a.reach || rel + V - 1 <= -a.reach))) {
                double sum = 0.0;
#pragma unroll
                for (int e = 0; e < V; e++) sum += g[e];
                below += rel < 0 ? sum : 0;
                above += rel < 0 ? 0 : sum;
            } else if (!every(lo == 0 && rel > -a.reach && rel + V <= a.reach)) {
                double left = 0.0, right = 0.0;
#pragma unroll
                for (int e = 0; e < V; e++) {
                    left += e >= lo && rel + e <= -a.reach ? g[e] : 0;
                    right += e >= lo && rel + e >= a.reach ? g[e] : 0;
                }
                below += left;
                above += right;
            }
        }
        return y;
    };
    int turn = 0;
    for (int item = item0; item < item1; item++) {
        const RelItem it(a, item);
        const char *xs = a.x + h * a.x2 + it.b * a.x3 + it.i0 * a.x1, *ds = a.dy + h * a.y2 + it.b * a.y3 + it.i0 * a.y1;
        char* os = a.out ? a.out + h * a.o2 + it.b * a.o3 + it.i0 * a.o1 : nullptr;
        Pack<T, V> py[K > 0 ? K : 1], pd[K > 0 ? K : 1], ny[K > 0 ? K : 1], nd[K > 0 ? K : 1];
        auto load = [&](int r) {
            const int limit = it.limit(a, r);
            const T *y = reinterpret_cast<const T*>(xs + r * a.x1), *dy = reinterpret_cast<const T*>(ds + r * a.y1);
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int j = Place<V>(lane + k * lanes, a.n, limit).from;
                ny[k] = load_vector(y + j);
                nd[k] = load_vector(dy + j);
            }
        };
        if constexpr (K > 0) load(min(group, it.rows - 1));
        for (int r0 = 0; r0 < it.rows; r0 += rounds) {
            const int r = min(r0 + group, it.rows - 1);
            const bool valid = r0 + group < it.rows;
            const long long at = it.at(r);
            const int limit = it.limit(a, r);
            const T *y = reinterpret_cast<const T*>(xs + r * a.x1), *dy = reinterpret_cast<const T*>(ds + r * a.y1);
            T* out = os ? reinterpret_cast<T*>(os + r * a.o1) : nullptr;
            double s = 0.0;
            turn ^= 1;
            if constexpr (K > 0) {
#pragma unroll
                for (int k = 0; k < K; k++) py[k] = ny[k], pd[k] = nd[k];
                if (r0 + rounds < it.rows) load(min(r0 + rounds + group, it.rows - 1));
#pragma unroll
                for (int k = 0; k < K; k++) {
                    const Place<V> at_k(lane + k * lanes, a.n, limit);
                    s = dot(py[k], pd[k], at_k.lo, at_k.hi, s);
                }
            } else {
                for (int c = lane; c * V < limit; c += lanes) s = dot(load_row<T>(y + c * V, a.n - c * V), load_row<T>(dy + c * V, a.n - c * V), 0, limit - c * V, s);
            }
            s = lane_sum_dyn(s, min(lanes, 64));
            if constexpr (WAVES > 1) {
                if (threadIdx.x % 64 == 0) red[turn][threadIdx.x / 64] = s;
                __syncthreads();
                s = (red[turn][0] + red[turn][1]) + (red[turn][2] + red[turn][3]);
            }
            if (!valid) continue;
            if (lane == 0) dots[r] = s;
            if constexpr (K > 0) {
#pragma unroll
                for (int k = 0; k < K; k++) {
                    const int c = lane + k * lanes;
                    if (c >= vectors) continue;
                    const Place<V> at_k(c, a.n, limit);
                    const Pack<T, V> dx = finish(py[k], pd[k], at_k.j0, at_k.lo, at_k.hi, at, s);
                    if (out) store_vector(out + at_k.j0, dx);
                }
            } else {
                for (int c = lane; c < vectors; c += lanes) {
                    const bool some = c * V < limit;
                    Pack<T, V> p{}, d{};
                    if (some) p = load_row<T>(y + c * V, a.n - c * V), d = load_row<T>(dy + c * V, a.n - c * V);
                    p = finish(p, d, c * V, 0, limit - c * V, at, s);
                    if (out) store_row<T>(out + c * V, p, a.n - c * V);
                }
            }
        }
        if (!a.part) continue;
        __syncthreads();                                             // dots
        for (int slot = threadIdx.x; slot < G * slots; slot += kRelThreads) {
            const int g = slot / slots, s0 = (slot - g * slots) * D;
            double acc[D] = {};
#pragma unroll 4
            for (int r = g; r < it.rows; r += G) {
                const long long j = it.at(r) + s0 - (a.reach - 1);
                const int limit = it.limit(a, r);
                if (j + D <= 0 || j >= limit) continue;
                const T *y = reinterpret_cast<const T*>(xs + r * a.x1) + j, *dy = reinterpret_cast<const T*>(ds + r * a.y1) + j;
                const double s = dots[r];
                Pack<T, D> p, d;
                if (j >= 0 && j + D <= limit) {
                    __builtin_memcpy(&p, y, sizeof p);
                    __builtin_memcpy(&d, dy, sizeof d);
#pragma unroll
                    for (int e = 0; e < D; e++) acc[e] += term(p.v[e], d.v[e], s);
                } else {
#pragma unroll
                    for (int e = 0; e < D; e++)
                        if (j + e >= 0 && j + e < limit) acc[e] += term(y[e], dy[e], s);
                }
            }
#pragma unroll
            for (int e = 0; e < D; e++) band[slot * D + e] += acc[e];
        }
        __syncthreads();                                             // dots are read
    }
    if (!a.part) return;
    below = lane_sum<64>(below);
    above = lane_sum<64>(above);
    if (threadIdx.x % 64 == 0) far[0][threadIdx.x / 64] = below, far[1][threadIdx.x / 64] = above;
    __syncthreads();
    // 16 lanes take a bucket: distances [first, end) before the query (after it from `side` on).
    double* part = a.part + (long long)block * a.n_buckets;
    const int l16 = threadIdx.x % 16, mid = a.reach - 1;
    auto sum_of = [&](int from, int to, int sign) {                  // of distances sign * [from, to)
        double s = 0.0;
        for (int d = from + l16; d < to; d += 16)
            for (int g = 0; g < G; g++) s += band[g * slots * D + mid + sign * d];
        return s;
    };
    for (int k0 = 0; k0 < a.n_buckets; k0 += kRelThreads / 16) {
        const int k = min(k0 + (int)threadIdx.x / 16, a.n_buckets - 1);
        const bool after = a.both && k >= a.side;
        const int i = after ? k - a.side : k;
        auto first_of = [&](int i) { return i < a.near ? i : i - a.near < a.edge_count ? a.edges[i - a.near] : a.reach; };
        double s = sum_of(after ? max(1, first_of(i)) : first_of(i), min(first_of(i + 1), a.reach), after ? 1 : -1);
        if (!a.both && k == 0) s += sum_of(1, a.reach, 1);
        s = lane_sum<16>(s);
        if (i == a.side - 1) s += after ? (far[1][0] + far[1][1]) + (far[1][2] + far[1][3]) : (far[0][0] + far[0][1]) + (far[0][2] + far[0][3]);
        if (!a.both && k == 0) s += (far[1][0] + far[1][1]) + (far[1][2] + far[1][3]);
        if (l16 == 0 && k0 + (int)threadIdx.x / 16 < a.n_buckets) part[k] = s;
    }
}

// The table's gradient: sums over a head's blocks in order; 32 buckets x 32 lanes a block.
__global__ __launch_bounds__(1024) void rel_fold_kernel(const double* part, int heads, int blocks, int n_buckets, float* dtable) {
    __shared__ double red[32][33];
    const int k = blockIdx.x * 32 + threadIdx.x % 32, h = blockIdx.y, lane = threadIdx.x / 32;
    double s = 0.0;
    if (k < n_buckets) {
#pragma unroll 4
        for (int c = lane; c < blocks; c += 32) s += part[((long long)h * blocks + c) * n_buckets + k];
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
    int rows;                            // of an item
    long long each;                      // items of a block
    long long chunks() const { return (queries + rows - 1) / rows; }
    long long items() const { return chunks() * batch; }             // of a head
    long long head_blocks() const { return (items() + each - 1) / each; }
    long long blocks() const { return head_blocks() * heads; }
    bool empty() const { return n == 0 || queries == 0 || heads == 0 || batch == 0; }
};
RelShape rel_shape(const stx_tensor* x, int size, const char* op) {
    RelShape s{x->ne[0], x->ne[1], x->ne[2], x->ne[3], 1, 1, 0, 1, 1};
    if (s.empty()) return s;
    STX_REQUIRE(s.n < (1LL << 30) && s.queries < (1LL << 30), "%s: %lld keys, %lld queries", op, s.n, s.queries);
    STX_REQUIRE(s.heads < (1LL << 16) && s.batch < (1LL << 24), "%s: %lld heads, %lld sequences", op, s.heads, s.batch);
    const long long v = (s.n + 16 / size - 1) / (16 / size);
    if (s.n < 16 / size) s.vectors = 0;                               // a lane a row, element by element
    while (s.log_lanes < 6 && (1 << s.log_lanes) < v) s.log_lanes++;
    if (v > 64) {
        s.waves = v > 512 ? 4 : 1;
        const long long lanes = s.waves * 64;
        s.vectors = v <= 2 * lanes ? 2 : v <= 4 * lanes ? 4 : v <= 8 * lanes ? 8 : 0;
    }
    // Rows of an item and items of a block: as many as leave 16 blocks a CU (4, 8, 16: the gradients of 8 x 8,192 x 8,192
    // bf16 scores 796, 759, 719 us), of which each forms the head's biases, or its sums by bucket, once.
    constexpr long long kBlocks = 16 * 256;
    const long long round = s.waves == 1 ? kRelThreads >> s.log_lanes : 1, all = s.queries * s.heads * s.batch;
    s.rows = (int)std::min<long long>(std::min<long long>(kRelRows, std::max(round, all / kBlocks)), s.queries);
    STX_REQUIRE(s.items() < (1LL << 31), "%s: too many rows", op);
    s.each = std::max(1LL, s.items() * s.heads / kBlocks);
    STX_REQUIRE(s.blocks() < (1LL << 31), "%s: too many rows", op);
    return s;
}

template <class F>
void with_row(const RelShape& s, F&& f) {
    using std::integral_constant;
    constexpr integral_constant<int, 1> one{};
    constexpr integral_constant<int, 4> four{};
    if (s.waves == 1) {
        if (s.vectors == 0) f(one, integral_constant<int, 0>{});
        else if (s.vectors == 1) f(one, one);
        else if (s.vectors == 2) f(one, integral_constant<int, 2>{});
        else if (s.vectors == 4) f(one, four);
        else f(one, integral_constant<int, 8>{});
    } else if (s.vectors == 4) f(four, four);
    else if (s.vectors == 8) f(four, integral_constant<int, 8>{});
    else f(four, integral_constant<int, 0>{});
}

void set_shape(RelArgs& a, const RelShape& s, const int32_t* lengths, const int32_t* starts, float scale) {
    a.lengths = lengths;
    a.starts = starts;
    a.n = (int)s.n;
    a.queries = (int)s.queries;
    a.heads = (int)s.heads;
    a.chunks = FastDiv((unsigned)s.chunks());
    a.blocks = FastDiv((unsigned)s.head_blocks());
    a.items = (int)s.items();
    a.each = (int)s.each;
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
    const RelShape s = rel_shape(x, size, op);
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
    const RelShape s = rel_shape(y, size, op);
    const size_t need = dtable && !s.empty() ? (size_t)s.blocks() * a.n_buckets * sizeof(double) : 0, per = (size_t)y->ne[3] * sizeof(int32_t);
    const size_t table = (size_t)a.n_buckets * y->ne[2] * sizeof(float);
    check_workspace(ws, ws_bytes, need, op);
    check_apart(op, {{"dx", dx, size}, {"dtable", dtable, table}, {"the workspace", need ? ws : nullptr, need}},
                {{"dy", dy, size}, {"y", y, size}, {"lengths", lengths, per}, {"starts", starts, per}});
    STX_REQUIRE(s.heads < (1LL << 16), "%s: more than 65,535 heads", op);
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
                const int slots = (2 * a.reach - 1 + 3) / 4;
                launch_all(s.blocks(), [&](dim3 grid, unsigned first) {
                    a.base = first;
                    hipLaunchKernelGGL((soft_max_rel_back_kernel<T, waves(), k()>), grid, dim3(kRelThreads), sizeof(double) * std::max(kRelThreads, slots) * 4,
                                       as_stream(stream), a);
                    launch_check("soft_max_rel_back_kernel");
                });
            });
        });
    }
    if (!dtable || s.heads == 0) return;
    hipLaunchKernelGGL(rel_fold_kernel, dim3((a.n_buckets + 31) / 32, (unsigned)s.heads), dim3(1024), 0, as_stream(stream), a.part, (int)s.heads,
                       s.empty() ? 0 : (int)s.head_blocks(), a.n_buckets, dtable);
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
        const RelShape s = rel_shape(y, size, "soft_max_rel_back_workspace_size");
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

// qk_norm.hip — RMS norms of queries and keys per head with the rotation in the same pass, forward and
// backward (stx_qk_norm_rope, stx_qk_norm_rope_back).
#include <algorithm>

#include "rope_angles.hpp"

namespace stx {
namespace {

// A row x of one head (of q or k) gives y = R(pos) (w x r), r = 1 / sqrt(mean(x^2) + eps), R the rotation
// of rope.hip. Its gradient: dz = R^T dy, dw = sum over the rows of dz x r, and with g = w dz
//   dx = r (g - x r mean(g x r)).
// Both read and write every element once (the gradient reads x again instead of r), so HBM bounds them.
// A row is held by `lanes` lanes of a wave, V elements a unit and K units a lane, all of them loaded
// before the first is stored: outputs may be inputs. A lane whose pair partner lies in another unit
// (mode 2, or units of one element) loads it too, from the same lines: units stay dense for any
// n_dims, where units of a pair of halves would leave 6 of 16 lanes idle at 128 elements, 96 rotated.
// A lane's squares and products g x r (of g's size for any x) are added in float, by halves (three roundings at V 8), the lanes' in
// double; a wave that meets a row whose squares leave fp32, or products past 10^30, forms them again in double, so data of any
// size keeps its norm. (In double throughout, with a double division and root, these took more time than the memory's: the
// gradient of 2 x 16,384 tokens of 40 rows of 128 bf16 values 297 us.)
// 60 x 801 tokens of 16 rows of 64 fp32 values, slices of a projection (394 MB): 79 us, 5.0 TB/s, the rate of a large copy;
// its bf16 gradient with weights of each head (295 MB) 80 us, 3.7 TB/s, vector units 84 % busy (short rows pay the sums across
// lanes and the root as long ones do); that of 2 x 16,384 tokens above (1.0 GB) 212 us, 4.8 TB/s. One token of 16 rows: 5.0 us.
struct QkSide {
    const char *x, *dy;
    char* out;
    const float* w;
    long long x1, x2, x3, y1, y2, y3, o1, o2, o3;    // byte strides of x, dy and out
};

struct QkArgs {
    QkSide q, k;
    RopeAngles at;
    double eps, per_dim;                 // per_dim: 1 / dim
    unsigned tokens, tile;               // all tokens, and of a block
    unsigned base;                       // blocks of the launches before this one
    FastDiv q_rows, k_rows;              // rows of a token
    int dim, units, log_lanes, mode;
    int w_stride;                        // from a head's weights to the next's: dim, or 0 where heads share them
    float* part;                         // backward: sums of dz x r, [block][2 or rows][dim], or NULL
};

constexpr int kQkThreads = 256;
constexpr int kQkDim = 1024;             // of a row: 64 lanes x 16 elements

// A tensor's rows as a group of lanes goes over them, `heads` and `tokens` a step: pointers move by what is uniform over the
// launch, without a product an address (kernels that formed each row's addresses, and chose q's or k's strides by lane, ran
// 62 vector instructions an element, and as long as those took).
template <class P>
struct Walk {
    P* p;
    long long step, carry, wrap;         // a step; a head past the last one, which is the next token; a token past the last
    __device__ __forceinline__ Walk(P* base, long long s1, long long s2, long long s3, unsigned h, unsigned i2, unsigned b, unsigned heads, unsigned tokens,
                                    unsigned rows, unsigned n)
        : p(base + h * s1 + i2 * s2 + b * s3), step(heads * s1 + tokens * s2), carry(s2 - rows * s1), wrap(s3 - n * s2) {}
};
// Where a group is: its head, and its token in the sequence and in the block.
struct Spot {
    unsigned h, i2, b, tk;
    __device__ __forceinline__ Spot(const QkArgs& a, unsigned t0, unsigned tk, unsigned h) : h(h), tk(tk) {
        b = a.at.n.div(t0 + tk);
        i2 = t0 + tk - b * a.at.n.d;
    }
    template <class... W>
    __device__ __forceinline__ void next(const QkArgs& a, unsigned rows, unsigned heads, unsigned tokens, W&... w) {
        ((w.p += w.step), ...);
        h += heads, i2 += tokens, tk += tokens;
        if (h >= rows) {
            h -= rows, i2++, tk++;
            ((w.p += w.carry), ...);
        }
        if (i2 >= a.at.n.d) {
            const unsigned turns = a.at.n.div(i2);
            i2 -= turns * a.at.n.d;
            ((w.p += turns * w.wrap), ...);
        }
    }
};

// Where the partners of unit `at` start; `at` itself where they are in the unit or there are none. In mode 2 the units over a
// half's end (`torn`) have theirs in two places; kernels without TORN are for calls that have none (with it, 60 x 801 tokens of
// 16 rows of 64 elements in mode 0 took 101 us instead of 84, and their gradient 103 instead of 82).
template <int V>
__device__ __forceinline__ int partner(const QkArgs& a, int at) {
    const int half = a.at.n_dims / 2;
    if (at >= a.at.n_dims) return at;
    if (a.mode == 0) return V == 1 ? at ^ 1 : at;
    return at < half ? at + half : at - half;
}
template <int V, bool TORN>
__device__ __forceinline__ bool torn(const QkArgs& a, int at) {
    const int half = a.at.n_dims / 2;
    return TORN && V > 1 && ((at < half && at + V > half) || (at < a.at.n_dims && at + V > a.at.n_dims));
}
// Element e's partner in mode 2, or -1.
__device__ __forceinline__ int partner_of(const QkArgs& a, int e) {
    const int half = a.at.n_dims / 2;
    return e < half ? e + half : e < a.at.n_dims ? e - half : -1;
}

// The rotation of unit `at` with values f and partners p, in place.
template <int V, bool TORN>
__device__ __forceinline__ void rotate(const QkArgs& a, int at, const float2* tab, float (&f)[V], const float (&p)[V]) {
    const int half = a.at.n_dims / 2;
    if (V > 1 && a.mode == 0) {
#pragma unroll
        for (int v = 0; v + 1 < V; v += 2) {
            const int pair = (at + v) / 2;
            if (pair >= half) continue;
            const float2 r = tab[pair];
            const float x0 = f[v], x1 = f[v + 1];
            f[v] = fmaf(x0, r.x, -(x1 * r.y));
            f[v + 1] = fmaf(x0, r.y, x1 * r.x);
        }
    } else if (torn<V, TORN>(a, at)) {
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int e = at + v;
            if (e >= a.at.n_dims) continue;
            const float2 r = tab[e < half ? e : e - half];
            f[v] = e < half ? fmaf(f[v], r.x, -(p[v] * r.y)) : fmaf(p[v], r.y, f[v] * r.x);
        }
    } else if (at < a.at.n_dims) {
        const bool first = a.mode == 0 ? at % 2 == 0 : at < half;
        const int pair = a.mode == 0 ? at / 2 : first ? at : at - half;
#pragma unroll
        for (int v = 0; v < V; v++) {
            const float2 r = tab[pair + v];
            f[v] = first ? fmaf(f[v], r.x, -(p[v] * r.y)) : fmaf(p[v], r.y, f[v] * r.x);
        }
    }
}

template <class T, int V>
__device__ __forceinline__ void take(const T* p, float (&f)[V]) {
    const Pack<T, V> x = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
    for (int v = 0; v < V; v++) f[v] = to_f32(x.v[v]);
}
// The partners of unit `at` of the row at p; f stays as it is where there are none.
template <class T, int V, bool TORN>
__device__ __forceinline__ void take_partners(const QkArgs& a, const T* p, int at, float (&f)[V]) {
    const int other = partner<V>(a, at);
    if (other == at) return;
    if (torn<V, TORN>(a, at)) {
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int e = partner_of(a, at + v);
            if (e >= 0) f[v] = to_f32(p[e]);
        }
    } else {
        Pack<T, V> x;
        if constexpr (TORN) __builtin_memcpy(&x, p + other, sizeof x);   // at any alignment
        else x = *reinterpret_cast<const Pack<T, V>*>(p + other);
#pragma unroll
        for (int v = 0; v < V; v++) f[v] = to_f32(x.v[v]);
    }
}
template <class T, int V>
__device__ __forceinline__ void give(T* p, const float (&f)[V]) {
    Pack<T, V> x;
#pragma unroll
    for (int v = 0; v < V; v++) x.v[v] = from_f32<T>(f[v]);
    *reinterpret_cast<Pack<T, V>*>(p) = x;
}
template <int V>
__device__ __forceinline__ void weights(const float* w, int at, float (&f)[V]) {
    if (w) {
        __builtin_memcpy(f, w + at, sizeof f);
    } else {
#pragma unroll
        for (int v = 0; v < V; v++) f[v] = 1.f;
    }
}

// The table of a block's tokens; where they are several, from frequencies formed once, in LDS behind it (a frequency takes
// as long as the angle's cos and sin).
__device__ __forceinline__ void table(const QkArgs& a, unsigned t0, unsigned nt, float2* cs) {
    const int half = a.at.n_dims / 2;
    if (a.tile > 1) {
        double* frequency = reinterpret_cast<double*>(cs + a.tile * half);
        for (int i = threadIdx.x; i < half; i += kQkThreads) frequency[i] = rope_frequency(a.at, i);
        __syncthreads();
        rope_table<kQkThreads>(a.at, t0, nt, cs, [&](int i) { return frequency[i]; });
    } else {
        rope_table<kQkThreads>(a.at, t0, nt, cs);
    }
    __syncthreads();
}

template <int V>
__device__ __forceinline__ float by_halves(const float* f) {
    if constexpr (V == 1) return f[0];
    else return by_halves<V / 2>(f) + by_halves<V / 2>(f + V / 2);
}
// 1 / sqrt(m): the hardware's (1 ulp) and a Newton step, whose error is that of rounding m and the result; in double where m
// is not a float's.
__device__ __forceinline__ float inverse_root(double m) {
    const float f = (float)m;
    if (__builtin_amdgcn_ballot_w64(!(f > 1e-30f && f < 1e30f))) return (float)(1.0 / sqrt(m));
    const float r = __builtin_amdgcn_rsqf(f), e = fmaf(-f * r, r, 1.f);
    return fmaf(0.5f * r, e, r);
}
// Whether a lane's sum of squares may have left fp32 (a mean that eps outweighs may be too small).
__device__ __forceinline__ bool outside(const QkArgs& a, float sum) {
    return __builtin_amdgcn_ballot_w64(!(sum < 1e30f) || (sum < 1e-25f && a.eps < 1e-20));
}

// The weights of a lane's units and of their partners.
template <int V, int K, bool PARTNERS, bool TORN>
struct Weights {
    float f[K][V], p[PARTNERS ? K : 1][V];
    __device__ __forceinline__ void load(const QkArgs& a, const float* w, int lane) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int u = lane + (k << a.log_lanes), at = min(u, a.units - 1) * V;
            weights<V>(w, at, f[k]);
            if constexpr (PARTNERS) {
                if (torn<V, TORN>(a, at)) {
#pragma unroll
                    for (int v = 0; v < V; v++) {
                        const int e = partner_of(a, at + v);
                        p[k][v] = w && e >= 0 ? w[e] : 1.f;
                    }
                } else {
                    weights<V>(w, partner<V>(a, at), p[k]);
                }
            }
        }
    }
};

template <class T, int V, int K, bool TORN>
__global__ __launch_bounds__(kQkThreads) void qk_norm_rope_kernel(QkArgs a) {
    extern __shared__ float2 cs[];       // [tile][n_dims / 2], then frequencies
    const int half = a.at.n_dims / 2;
    const unsigned t0 = (a.base + blockIdx.x) * a.tile, nt = min(a.tile, a.tokens - t0);
    table(a, t0, nt, cs);
    const int lanes = 1 << a.log_lanes, lane = threadIdx.x & (lanes - 1);
    const unsigned groups = kQkThreads >> a.log_lanes, group = threadIdx.x >> a.log_lanes;
    auto rows_of = [&](const QkSide& side, FastDiv rows) {
        const unsigned heads = groups % rows.d, tokens = groups / rows.d, total = nt * rows.d;
        const unsigned tk0 = rows.div(min(group, total - 1));
        Spot s(a, t0, tk0, min(group, total - 1) - tk0 * rows.d);
        Walk<const char> x(side.x, side.x1, side.x2, side.x3, s.h, s.i2, s.b, heads, tokens, rows.d, a.at.n.d);
        Walk<char> out(side.out, side.o1, side.o2, side.o3, s.h, s.i2, s.b, heads, tokens, rows.d, a.at.n.d);
        Weights<V, K, true, TORN> w;
        if (a.w_stride == 0) w.load(a, side.w, lane);
        for (unsigned row = group; row - group < total; row += groups, s.next(a, rows.d, heads, tokens, x, out)) {
            const bool valid = row < total;                          // every lane takes part in the sums
            float f[K][V], p[K][V], squares = 0.f;
            const T* src = reinterpret_cast<const T*>(x.p);
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int u = lane + (k << a.log_lanes), at = u * V;
#pragma unroll
                for (int v = 0; v < V; v++) f[k][v] = p[k][v] = 0.f;
                if (!valid || u >= a.units) continue;
                take<T, V>(src + at, f[k]);
                take_partners<T, V, TORN>(a, src, at, p[k]);
            }
            if (a.w_stride != 0) w.load(a, side.w ? side.w + (long long)s.h * a.w_stride : nullptr, lane);
#pragma unroll
            for (int k = 0; k < K; k++) {
                float xx[V];
#pragma unroll
                for (int v = 0; v < V; v++) xx[v] = f[k][v] * f[k][v];
                squares += by_halves<V>(xx);
            }
            double sum = squares;
            if (outside(a, squares)) {
                sum = 0.0;
#pragma unroll
                for (int k = 0; k < K; k++)
#pragma unroll
                    for (int v = 0; v < V; v++) sum = fma((double)f[k][v], (double)f[k][v], sum);
            }
            const float rstd = inverse_root(fma(lane_sum_dyn(sum, lanes), a.per_dim, a.eps));
            if (!valid) continue;
            T* to = reinterpret_cast<T*>(out.p);
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int u = lane + (k << a.log_lanes), at = u * V;
                if (u >= a.units) continue;
#pragma unroll
                for (int v = 0; v < V; v++) {
                    f[k][v] = f[k][v] * rstd * w.f[k][v];
                    p[k][v] = p[k][v] * rstd * w.p[k][v];
                }
                rotate<V, TORN>(a, at, cs + s.tk * half, f[k], p[k]);
                give<T, V>(to + at, f[k]);
            }
        }
    };
    if (a.q_rows.d) rows_of(a.q, a.q_rows);
    if (a.k_rows.d) rows_of(a.k, a.k_rows);
}

// Sums over the rows of dz x r are kept by the lanes that hold the elements, over the tokens of a block, of q and then of k:
// where heads share weights, a group takes any row; where they do not (PER_HEAD), it keeps to a head, or takes its
// heads one after another. Added up in LDS in order, and over the blocks by qk_fold_kernel.
// Waves a SIMD that a row of eight elements a lane is held to (98 registers instead of 96 in fp16 leave four: 104 us
// instead of 80 for 60 x 801 tokens of 16 rows of 64).
template <int V, int K, bool PER_HEAD, bool TORN>
constexpr int kBackWaves = V * K > 8 ? 1 : V < 8 || TORN ? 4 : PER_HEAD ? 5 : 6;

template <class T, int V, int K, bool PER_HEAD, bool TORN>
__global__ __launch_bounds__(kQkThreads, (kBackWaves<V, K, PER_HEAD, TORN>)) void qk_norm_rope_back_kernel(QkArgs a) {
    extern __shared__ float2 cs[];       // [tile][n_dims / 2], frequencies, then sums [groups][units * V]
    const int half = a.at.n_dims / 2;
    const unsigned block = a.base + blockIdx.x, t0 = block * a.tile, nt = min(a.tile, a.tokens - t0);
    table(a, t0, nt, cs);
    const int lanes = 1 << a.log_lanes, lane = threadIdx.x & (lanes - 1), width = a.units * V;
    const unsigned groups = kQkThreads >> a.log_lanes, group = threadIdx.x >> a.log_lanes;
    float* red = reinterpret_cast<float*>(cs + (a.tile + 1) * half);
    // Rows from (tk, h) on, `heads` and `tokens` a step, `rounds` of them, those in the tile.
    auto rows_of = [&](const QkSide& side, unsigned rows, unsigned tk0, unsigned h0, bool some, unsigned heads, unsigned tokens, unsigned rounds, float (&acc)[K][V]) {
        Spot s(a, t0, min(tk0, nt - 1), h0);
        Walk<const char> x(side.x, side.x1, side.x2, side.x3, s.h, s.i2, s.b, heads, tokens, rows, a.at.n.d);
        Walk<const char> dy(side.dy, side.y1, side.y2, side.y3, s.h, s.i2, s.b, heads, tokens, rows, a.at.n.d);
        Walk<char> out(side.out, side.o1, side.o2, side.o3, s.h, s.i2, s.b, heads, tokens, rows, a.at.n.d);
        Weights<V, K, false, false> w;
        w.load(a, side.w ? side.w + (long long)s.h * a.w_stride : nullptr, lane);
        s.tk = tk0;
        for (unsigned round = 0; round < rounds; round++, s.next(a, rows, heads, tokens, x, dy, out)) {
            const bool valid = some && s.tk < nt;
            float f[K][V], z[K][V], p[K][V], squares = 0.f, products = 0.f;
            const T *src = reinterpret_cast<const T*>(x.p), *dsrc = reinterpret_cast<const T*>(dy.p);
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int u = lane + (k << a.log_lanes), at = u * V;
#pragma unroll
                for (int v = 0; v < V; v++) f[k][v] = z[k][v] = p[k][v] = 0.f;
                if (!valid || u >= a.units) continue;
                take<T, V>(src + at, f[k]);
                take<T, V>(dsrc + at, z[k]);
                take_partners<T, V, TORN>(a, dsrc, at, p[k]);
            }
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int u = lane + (k << a.log_lanes), at = u * V;
                if (valid && u < a.units) rotate<V, TORN>(a, at, cs + s.tk * half, z[k], p[k]);
                float xx[V];
#pragma unroll
                for (int v = 0; v < V; v++) {
                    xx[v] = f[k][v] * f[k][v];
                    p[k][v] = w.f[k][v] * z[k][v];
                }
                squares += by_halves<V>(xx);
            }
            double sum = squares;
            if (outside(a, squares)) {
                sum = 0.0;
#pragma unroll
                for (int k = 0; k < K; k++)
#pragma unroll
                    for (int v = 0; v < V; v++) sum = fma((double)f[k][v], (double)f[k][v], sum);
            }
            const float rstd = inverse_root(fma(lane_sum_dyn(sum, lanes), a.per_dim, a.eps));
#pragma unroll
            for (int k = 0; k < K; k++) {
                float gx[V];
#pragma unroll
                for (int v = 0; v < V; v++) {
                    f[k][v] *= rstd;
                    gx[v] = p[k][v] * f[k][v];
                }
                products += by_halves<V>(gx);
            }
            sum = products;
            if (__builtin_amdgcn_ballot_w64(!(fabsf(products) < 1e30f))) {
                sum = 0.0;
#pragma unroll
                for (int k = 0; k < K; k++)
#pragma unroll
                    for (int v = 0; v < V; v++) sum = fma((double)p[k][v], (double)f[k][v], sum);
            }
            const float mean = (float)(lane_sum_dyn(sum, lanes) * a.per_dim);
            if (!valid) continue;
            T* to = reinterpret_cast<T*>(out.p);
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int u = lane + (k << a.log_lanes), at = u * V;
                if (u >= a.units) continue;
#pragma unroll
                for (int v = 0; v < V; v++) {
                    acc[k][v] = fmaf(z[k][v], f[k][v], acc[k][v]);
                    f[k][v] = rstd * fmaf(-f[k][v], mean, p[k][v]);
                }
                if (side.out) give<T, V>(to + at, f[k]);
            }
        }
    };
    auto lay = [&](const float (&acc)[K][V]) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int u = lane + (k << a.log_lanes);
            if (u >= a.units) continue;
#pragma unroll
            for (int v = 0; v < V; v++) red[group * width + u * V + v] = acc[k][v];
        }
        __syncthreads();
    };
    auto side_of = [&](const QkSide& side, FastDiv by, unsigned first) {       // first: its row of the sums
        const unsigned rows = by.d;
        if constexpr (PER_HEAD) {
            const unsigned slices = groups >= rows ? groups / rows : 1, heads = groups >= rows ? rows : groups, slice = group / heads;
            for (unsigned h0 = 0; h0 < rows; h0 += heads) {
                float acc[K][V] = {};
                const unsigned h = h0 + group % heads;
                rows_of(side, rows, slice, min(h, rows - 1), slice < slices && h < rows, 0, slices, (nt + slices - 1) / slices, acc);
                if (!a.part) continue;
                lay(acc);
                const unsigned here = min(heads, rows - h0);
                for (unsigned e = threadIdx.x; e < here * a.dim; e += kQkThreads) {
                    const unsigned i = e / a.dim, d = e - i * a.dim;
                    float s = 0.f;
                    for (unsigned j = 0; j < slices; j++) s += red[(j * heads + i) * width + d];
                    a.part[((long long)block * (a.q_rows.d + a.k_rows.d) + first + h0 + i) * a.dim + d] = s;
                }
                __syncthreads();
            }
        } else {
            float acc[K][V] = {};
            const unsigned tk = by.div(group);
            rows_of(side, rows, tk, group - tk * rows, true, groups % rows, groups / rows, (nt * rows + groups - 1) / groups, acc);
            if (!a.part) return;
            lay(acc);
            for (unsigned d = threadIdx.x; d < (unsigned)a.dim; d += kQkThreads) {
                float s = 0.f;
                for (unsigned g = 0; g < groups; g++) s += red[g * width + d];
                a.part[((long long)block * 2 + (first ? 1 : 0)) * a.dim + d] = s;
            }
            __syncthreads();
        }
    };
    if (a.q_rows.d) side_of(a.q, a.q_rows, 0);
    if (a.k_rows.d) side_of(a.k, a.k_rows, a.q_rows.d);
    else if (!PER_HEAD && a.part)        // no rows: a sum of none
        for (unsigned d = threadIdx.x; d < (unsigned)a.dim; d += kQkThreads) a.part[((long long)block * 2 + 1) * a.dim + d] = 0.f;
}

// The weights' gradients: column sums of part [rows][cols], 32 columns x 32 lanes a block; the first
// q_cols of them are q's.
__global__ __launch_bounds__(1024) void qk_fold_kernel(const float* part, long long rows, unsigned cols, unsigned q_cols, float* dwq, float* dwk) {
    __shared__ double red[32][33];
    const unsigned c = blockIdx.x * 32 + threadIdx.x % 32, lane = threadIdx.x / 32;
    double s = 0.0;
    if (c < cols) {
#pragma unroll 8
        for (long long r = lane; r < rows; r += 32) s += (double)part[r * cols + c];
    }
    red[lane][threadIdx.x % 32] = s;
    __syncthreads();
    if (lane || c >= cols) return;
    for (int i = 1; i < 32; i++) s += red[i][threadIdx.x];
    float* d = c < q_cols ? dwq : dwk;
    if (d) d[c < q_cols ? c : c - q_cols] = (float)s;
}

// --------------------------------------------------------------------------------- host
// The widest access (16, then 8 bytes, then an element) that every row's start and its length allow. (Where the halves of mode 2
// had to allow it too, 15 x 775 tokens of 5 rows of 80 bf16 values, 38 of them rotated, took 129 us, now 38.)
int width_of(std::initializer_list<const stx_tensor*> all, long long dim, int size) {
    for (int bytes : {16, 8}) {
        const int w = bytes / size;
        bool ok = dim % w == 0;
        for (const stx_tensor* t : all) ok = ok && rows_aligned(t, bytes);
        if (ok) return w;
    }
    return 1;
}

struct Shape {
    long long q_rows, k_rows, tokens, dim;
    long long rows() const { return q_rows + k_rows; }
    bool empty() const { return tokens == 0 || rows() == 0; }
};

Shape shape_of(const stx_tensor* q, const stx_tensor* k, const char* op) {
    const long long n = q->ne[2], b = q->ne[3], dim = q->ne[0];
    if (k)
        STX_REQUIRE(k->ne[0] == dim && k->ne[2] == n && k->ne[3] == b, "%s: q and k differ in head size, tokens or batch", op);
    const Shape s{q->ne[1], k ? k->ne[1] : 0, n * b, dim};
    STX_REQUIRE(dim > 0, "%s: rows of no elements", op);
    STX_REQUIRE(s.q_rows > 0 || s.k_rows == 0, "%s: k without heads of q", op);
    if (dim > kQkDim) fail(STX_STATUS_UNSUPPORTED, "%s: rows of %lld elements (%d at most)", op, dim, kQkDim);
    if (s.empty()) return s;
    STX_REQUIRE(n < (1LL << 31) && b < (1LL << 31) && n * b < (1LL << 31), "%s: more than 2^31 - 1 tokens", op);
    STX_REQUIRE(s.rows() < (1LL << 24) && s.rows() * dim < (1LL << 27), "%s: too many rows a token", op);
    return s;
}

// Tokens of a block of the backward pass: 64 at most, so that its sums are a small part of its traffic, and
// four blocks a CU as long as there are tokens.
constexpr long long kQkBlocks = 4 * 256;
long long back_tile(long long tokens, int n_dims) {
    return std::max(1LL, std::min({64LL, tokens / kQkBlocks, (long long)kRopeTable / (n_dims / 2)}));
}
// Blocks of the backward pass for any rotation of rows of `dim` elements.
size_t back_part(const Shape& s, long long tile, int per_head) {
    return (size_t)((s.tokens + tile - 1) / tile) * (per_head ? s.rows() : 2) * s.dim * sizeof(float);
}

QkArgs args_of(const stx_tensor* q, const Shape& s, const RopeAngles& at, const stx_rope_params* p, const int32_t* pos, double eps, int per_head, int w) {
    QkArgs a{};
    a.at = at;
    a.at.pos = pos;
    a.at.n = FastDiv((unsigned)q->ne[2]);
    a.eps = eps;
    a.per_dim = 1.0 / (double)s.dim;
    a.tokens = (unsigned)s.tokens;
    a.q_rows.d = a.k_rows.d = 0;
    if (s.q_rows) a.q_rows = FastDiv((unsigned)s.q_rows);
    if (s.k_rows) a.k_rows = FastDiv((unsigned)s.k_rows);
    a.dim = (int)s.dim;
    a.units = (int)(s.dim / w);
    while (a.log_lanes < 6 && (1 << a.log_lanes) < a.units) a.log_lanes++;
    a.mode = p->mode;
    a.w_stride = per_head ? a.dim : 0;
    return a;
}

QkSide side(const stx_tensor* x, const stx_tensor* dy, const stx_tensor* out, const float* w) {
    QkSide s{};
    s.x = static_cast<const char*>(x->data);
    s.x1 = x->nb[1], s.x2 = x->nb[2], s.x3 = x->nb[3];
    if (dy) s.dy = static_cast<const char*>(dy->data), s.y1 = dy->nb[1], s.y2 = dy->nb[2], s.y3 = dy->nb[3];
    if (out) s.out = static_cast<char*>(out->data), s.o1 = out->nb[1], s.o2 = out->nb[2], s.o3 = out->nb[3];
    s.w = w;
    return s;
}

// Calls f(V, K, TORN) as constants: units of w elements, as many a lane as a row of them needs, and whether halves end in them.
template <class T, class F>
void with_units(int w, const QkArgs& a, F&& f) {
    constexpr int W = 16 / sizeof(T);
    auto lanes = [&](auto v) {
        constexpr int V = v();
        auto torn = [&](auto t) {
            if (a.units <= 64) f(v, std::integral_constant<int, 1>{}, t);
            else f(v, std::integral_constant<int, kQkDim / 64 / V>{}, t);
        };
        if constexpr (V > 1) {
            if (a.mode != 0 && a.at.n_dims / 2 % V != 0) return torn(std::true_type{});
        }
        torn(std::false_type{});
    };
    if (w == W) lanes(std::integral_constant<int, W>{});
    else if (w == W / 2) lanes(std::integral_constant<int, W / 2>{});
    else lanes(std::integral_constant<int, 1>{});
}

// Positions and factors of a call, as memory that its outputs leave alone.
size_t pos_bytes(const stx_tensor* q, int64_t pos_stride) {
    return q->ne[2] > 0 && q->ne[3] > 0 ? ((size_t)(q->ne[3] - 1) * pos_stride + q->ne[2]) * sizeof(int32_t) : 0;
}
size_t factor_bytes(const stx_rope_params* p) { return p->n_dims / 2 * sizeof(float); }

void check_eps(double eps, const char* op) { STX_REQUIRE(eps >= 0.0 && std::isfinite(eps), "%s: eps must be finite and not negative", op); }

size_t weight_bytes(const stx_tensor* t, int per_head) { return t ? (size_t)t->ne[0] * (per_head ? t->ne[1] : 1) * sizeof(float) : 0; }

void qk_norm_rope(const stx_tensor* q, const stx_tensor* k, stx_type type, const int32_t* pos, int64_t pos_stride, const stx_rope_params* p,
                  const float* w_q, const float* w_k, int per_head, double eps, const stx_tensor* q_dst, const stx_tensor* k_dst, stx_stream stream) {
    const char* op = "qk_norm_rope";
    const int size = type_size(type);
    check_row_output(q, q_dst, size, "qk_norm_rope: q");
    STX_REQUIRE((k == nullptr) == (k_dst == nullptr), "%s: k and k_dst go together", op);
    if (k) {
        check_row_output(k, k_dst, size, "qk_norm_rope: k");
        STX_REQUIRE(shared(q_dst, k_dst, size) != Shared::yes && shared(q_dst, k, size) != Shared::yes && shared(k_dst, q, size) != Shared::yes,
                    "%s: an output overlaps the other side's tensors", op);
    }
    const Shape s = shape_of(q, k, op);
    const RopeAngles at = rope_angles(p, s.dim, pos_stride, 1.f, op);
    check_eps(eps, op);
    for (const stx_tensor* d : {q_dst, k_dst})
        if (d)
            check_apart(op, {{"an output", d, size}}, {{"w_q", w_q, weight_bytes(q, per_head)}, {"w_k", w_k, weight_bytes(k, per_head)},
                                                       {"pos", pos, pos_bytes(q, pos_stride)}, {"freq_factors", p->freq_factors, factor_bytes(p)}});
    if (s.empty()) return;
    STX_REQUIRE(pos != nullptr, "%s: pos is NULL", op);
    const int w = width_of({q, k, q_dst, k_dst}, s.dim, size);
    QkArgs a = args_of(q, s, at, p, pos, eps, per_head, w);
    a.q = side(q, nullptr, q_dst, w_q);
    if (k) a.k = side(k, nullptr, k_dst, w_k);
    // Tokens a block: four rounds of rows, as long as two blocks a CU remain.
    const long long round = kQkThreads >> a.log_lanes;
    const long long tile = std::max(1LL, std::min({16LL, 4 * round / s.rows(), s.tokens / 512, (long long)kRopeTable / (a.at.n_dims / 2)}));
    a.tile = (unsigned)tile;
    const size_t lds = sizeof(float2) * (tile + 1) * (a.at.n_dims / 2);
    with_type(type, [&](auto t) {
        using T = decltype(t);
        with_units<T>(w, a, [&](auto v, auto n, auto torn) {
            launch_all((s.tokens + tile - 1) / tile, [&](dim3 grid, unsigned first) {
                a.base = first;
                hipLaunchKernelGGL((qk_norm_rope_kernel<T, v(), n(), torn()>), grid, dim3(kQkThreads), lds, as_stream(stream), a);
                launch_check("qk_norm_rope_kernel");
            });
        });
    });
}

void qk_norm_rope_back(const stx_tensor* dyq, const stx_tensor* dyk, const stx_tensor* q, const stx_tensor* k, stx_type type, const int32_t* pos,
                       int64_t pos_stride, const stx_rope_params* p, const float* w_q, const float* w_k, int per_head, double eps, const stx_tensor* dq,
                       const stx_tensor* dk, float* dw_q, float* dw_k, void* ws, size_t ws_bytes, stx_stream stream) {
    const char* op = "qk_norm_rope_back";
    const int size = type_size(type);
    check_typed(q, size, "qk_norm_rope_back: q");
    check_typed(dyq, size, "qk_norm_rope_back: dq_out");
    check_same_shape(q, dyq, "qk_norm_rope_back: dq_out");
    if (dq) {
        check_row_output(q, dq, size, "qk_norm_rope_back: dq");
        check_row_output(dyq, dq, size, "qk_norm_rope_back: dq");
    }
    STX_REQUIRE((k == nullptr) == (dyk == nullptr) && (k || (!dk && !dw_k)), "%s: k, dk_out and k's gradients go together", op);
    if (k) {
        check_typed(k, size, "qk_norm_rope_back: k");
        check_typed(dyk, size, "qk_norm_rope_back: dk_out");
        check_same_shape(k, dyk, "qk_norm_rope_back: dk_out");
        if (dk) {
            check_row_output(k, dk, size, "qk_norm_rope_back: dk");
            check_row_output(dyk, dk, size, "qk_norm_rope_back: dk");
        }
        auto apart = [&](const stx_tensor* a, const stx_tensor* b) {
            STX_REQUIRE(!a || !b || shared(a, b, size) != Shared::yes, "%s: an output overlaps the other side's tensors", op);
        };
        for (const stx_tensor* t : {k, dyk, dk}) apart(dq, t);
        for (const stx_tensor* t : {q, dyq}) apart(dk, t);
    }
    const Shape s = shape_of(q, k, op);
    const RopeAngles at = rope_angles(p, s.dim, pos_stride, -1.f, op);
    check_eps(eps, op);
    const bool sums = dw_q || dw_k;
    const long long tile = s.empty() ? 1 : back_tile(s.tokens, p->n_dims);
    const size_t need = sums && !s.empty() ? back_part(s, tile, per_head) : 0, wq = weight_bytes(q, per_head), wk = weight_bytes(k, per_head);
    check_workspace(ws, ws_bytes, need, op);
    check_apart(op, {{"dw_q", dw_q, wq}, {"dw_k", dw_k, wk}, {"the workspace", need ? ws : nullptr, need}},
                {{"q", q, size}, {"k", k, size}, {"dq_out", dyq, size}, {"dk_out", dyk, size}, {"dq", dq, size}, {"dk", dk, size}, {"w_q", w_q, wq}, {"w_k", w_k, wk},
                 {"pos", pos, pos_bytes(q, pos_stride)}, {"freq_factors", p->freq_factors, factor_bytes(p)}});
    for (const stx_tensor* d : {dq, dk})
        if (d)
            check_apart(op, {{"an output", d, size}}, {{"w_q", w_q, wq}, {"w_k", w_k, wk}, {"pos", pos, pos_bytes(q, pos_stride)}, {"freq_factors", p->freq_factors, factor_bytes(p)}});
    if (!dq && !dk && !sums) return;
    float* part = sums ? static_cast<float*>(ws) : nullptr;
    long long blocks = 0;
    if (!s.empty()) {
        STX_REQUIRE(pos != nullptr, "%s: pos is NULL", op);
        const int w = width_of({q, k, dyq, dyk, dq, dk}, s.dim, size);
        QkArgs a = args_of(q, s, at, p, pos, eps, per_head, w);
        a.q = side(q, dyq, dq, w_q);
        if (k) a.k = side(k, dyk, dk, w_k);
        a.tile = (unsigned)tile;
        a.part = part;
        blocks = (s.tokens + tile - 1) / tile;
        const size_t lds = sizeof(float2) * (tile + 1) * (p->n_dims / 2) + (sums ? sizeof(float) * (kQkThreads >> a.log_lanes) * a.units * w : 0);
        with_type(type, [&](auto t) {
            using T = decltype(t);
            with_units<T>(w, a, [&](auto v, auto n, auto torn) {
                launch_all(blocks, [&](dim3 grid, unsigned first) {
                    a.base = first;
                    if (per_head) hipLaunchKernelGGL((qk_norm_rope_back_kernel<T, v(), n(), true, torn()>), grid, dim3(kQkThreads), lds, as_stream(stream), a);
                    else hipLaunchKernelGGL((qk_norm_rope_back_kernel<T, v(), n(), false, torn()>), grid, dim3(kQkThreads), lds, as_stream(stream), a);
                    launch_check("qk_norm_rope_back_kernel");
                });
            });
        });
    }
    if (!sums) return;
    const unsigned cols = (unsigned)((per_head ? s.rows() : 2) * s.dim), q_cols = (unsigned)((per_head ? s.q_rows : 1) * s.dim);
    if (cols == 0) return;
    hipLaunchKernelGGL(qk_fold_kernel, dim3((cols + 31) / 32), dim3(1024), 0, as_stream(stream), part, blocks, cols, q_cols, dw_q, dw_k);
    launch_check("qk_fold_kernel");
}

}  // namespace
}  // namespace stx

using namespace stx;

extern "C" {

STX_API stx_status stx_qk_norm_rope(const stx_tensor* q, const stx_tensor* k, stx_type type, const int32_t* pos, int64_t pos_stride,
                                    const stx_rope_params* params, const float* w_q, const float* w_k, int per_head, double eps,
                                    const stx_tensor* q_dst, const stx_tensor* k_dst, stx_stream stream) {
    return guard([&] { qk_norm_rope(q, k, type, pos, pos_stride, params, w_q, w_k, per_head, eps, q_dst, k_dst, stream); });
}

STX_API size_t stx_qk_norm_rope_back_workspace_size(const stx_tensor* q, const stx_tensor* k, stx_type type, int n_dims, int per_head) {
    size_t bytes = 0;
    (void)guard([&] {
        const int size = type_size(type);
        STX_REQUIRE(q != nullptr, "qk_norm_rope_back_workspace_size: q is NULL");
        for (const stx_tensor* t : {q, k})
            for (int i = 0; t && i < 4; i++) STX_REQUIRE(t->ne[i] >= 0, "qk_norm_rope_back_workspace_size: negative ne[%d]", i);
        (void)size;
        const Shape s = shape_of(q, k, "qk_norm_rope_back_workspace_size");
        STX_REQUIRE(n_dims > 0 && n_dims % 2 == 0 && n_dims <= s.dim, "qk_norm_rope_back_workspace_size: n_dims = %d", n_dims);
        if (!s.empty()) bytes = back_part(s, back_tile(s.tokens, n_dims), per_head);
    });
    return bytes;
}

STX_API stx_status stx_qk_norm_rope_back(const stx_tensor* dq_out, const stx_tensor* dk_out, const stx_tensor* q, const stx_tensor* k,
                                         stx_type type, const int32_t* pos, int64_t pos_stride, const stx_rope_params* params,
                                         const float* w_q, const float* w_k, int per_head, double eps, const stx_tensor* dq,
                                         const stx_tensor* dk, float* dw_q, float* dw_k, void* workspace, size_t workspace_bytes,
                                         stx_stream stream) {
    return guard([&] {
        qk_norm_rope_back(dq_out, dk_out, q, k, type, pos, pos_stride, params, w_q, w_k, per_head, eps, dq, dk, dw_q, dw_k, workspace,
                          workspace_bytes, stream);
    });
}

}  // extern "C"

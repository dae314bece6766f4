// rope.hip — rotary positions over typed tensors with scaled angles, forward and backward
// (stx_rope_scaled, stx_rope_scaled_back).
#include <algorithm>

#include "rope_angles.hpp"

namespace stx {
namespace {

// Each block takes a tile of consecutive tokens (N x batch flattened, so short sequences of a
// large batch fill tiles too): it forms cos and sin of the tile's angles once, in LDS, and rotates
// all rows (heads of q, then of k) of those tokens with them. The operator reads and writes every
// element once; the angles cost half / (rows * dim) of a double-precision evaluation an element.
// With 16 rows a token or more it is bound by HBM: 60 x 801 tokens of 16 rows of 64 fp32 values, slices
// of a projection (394 MB): 73 us, 5.4 TB/s; the gradient of 2 x 16,384 tokens of 40 rows of 128 bf16 values,
// 96 of them rotated (671 MB): 131 us, 5.1 TB/s, the rate of a large copy. With fewer, by the angles:
// 200,000 tokens of 2 rows of 64 bf16 values (102 MB, 20 us at that rate): 42 us. One token of 16 rows: 2.3 us.
//
// Angles are products of a position and a frequency in double (a float angle of 10^5 radians
// would be off by 2^-8); cos and sin are reduced and evaluated in double and rounded to float
// once, with the scale m applied before the rounding. The rotation itself is two float
// operations an output: its error is that of rounding, relative to |x0| + |x1|.
struct RopeSide {
    const char* src;
    char* dst;
    long long s1, s2, s3, d1, d2, d3;    // byte strides
};

struct RopeScaledArgs {
    RopeSide q, k;
    RopeAngles at;
    unsigned tokens, tile;               // all tokens, and of a block
    unsigned base;                       // blocks of the launches before this one
    FastDiv rows, units;                 // rows of a token (q's, then k's); units of a row
    unsigned q_rows;
    int dim;
};

// What a thread moves at once. MODE 0: V elements, V/2 adjacent pairs. MODE 2: V elements of the
// first half and V of the second, or V elements past n_dims. VEC: as vectors of V; otherwise
// element by element (V = 2 in mode 0, 1 in mode 2), for rows of any length and alignment.
template <class T, int V, bool VEC>
__device__ __forceinline__ Pack<T, V> rope_load(const T* p, int valid) {
    if constexpr (VEC) return *reinterpret_cast<const Pack<T, V>*>(p);
    Pack<T, V> r;
#pragma unroll
    for (int i = 0; i < V; i++) r.v[i] = i < valid ? p[i] : T(0.f);
    return r;
}
template <class T, int V, bool VEC>
__device__ __forceinline__ void rope_store(T* p, Pack<T, V> r, int valid) {
    if constexpr (VEC) {
        *reinterpret_cast<Pack<T, V>*>(p) = r;
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < valid) p[i] = r.v[i];
    }
}

constexpr int kRopeThreads = 256;
// Units a thread of a tile, one after another. The two calls above by it: 1: 81, 134 us; 2: 72, 136; 4: 73, 132;
// 8: 77, 149. Four loaded before the first is stored: 76, 150 (the waves' registers, hence fewer waves).
constexpr int kRopeUnits = 4;
constexpr int kRopeTile = 16;

template <class T, int V, bool VEC, int MODE>
__global__ __launch_bounds__(kRopeThreads) void rope_scaled_kernel(RopeScaledArgs a) {
    extern __shared__ float2 cs[];       // [tile][n_dims / 2]
    const int half = a.at.n_dims / 2;
    const unsigned t0 = (a.base + blockIdx.x) * a.tile;
    const unsigned nt = min(a.tile, a.tokens - t0);
    rope_table<kRopeThreads>(a.at, t0, nt, cs);
    __syncthreads();
    const unsigned total = nt * a.rows.d * a.units.d;
    for (unsigned e = threadIdx.x; e < total; e += kRopeThreads) {
        const unsigned row = a.units.div(e), u = e - row * a.units.d;
        const unsigned tk = a.rows.div(row), h = row - tk * a.rows.d;
        const unsigned t = t0 + tk, i3 = a.at.n.div(t), i2 = t - i3 * a.at.n.d;
        const bool is_k = h >= a.q_rows;
        const RopeSide& side = is_k ? a.k : a.q;
        const long long i1 = is_k ? h - a.q_rows : h;
        const T* src = reinterpret_cast<const T*>(side.src + i1 * side.s1 + i2 * side.s2 + i3 * side.s3);
        T* out = reinterpret_cast<T*>(side.dst + i1 * side.d1 + i2 * side.d2 + i3 * side.d3);
        const float2* tab = cs + tk * half;
        if constexpr (MODE == 0) {
            const int at = (int)u * V;
            Pack<T, V> x = rope_load<T, V, VEC>(src + at, a.dim - at);
#pragma unroll
            for (int v = 0; v < V; v += 2) {
                const int pair = (at + v) / 2;
                if (pair >= half) continue;
                const float2 r = tab[pair];
                const float x0 = to_f32(x.v[v]), x1 = to_f32(x.v[v + 1]);
                x.v[v] = from_f32<T>(fmaf(x0, r.x, -(x1 * r.y)));
                x.v[v + 1] = from_f32<T>(fmaf(x0, r.y, x1 * r.x));
            }
            rope_store<T, V, VEC>(out + at, x, a.dim - at);
        } else {
            const int pairs = half / V, at = (int)u < pairs ? (int)u * V : a.at.n_dims + ((int)u - pairs) * V;
            Pack<T, V> x = rope_load<T, V, VEC>(src + at, V);
            if (at < half) {
                Pack<T, V> y = rope_load<T, V, VEC>(src + at + half, V);
#pragma unroll
                for (int v = 0; v < V; v++) {
                    const float2 r = tab[at + v];
                    const float x0 = to_f32(x.v[v]), x1 = to_f32(y.v[v]);
                    x.v[v] = from_f32<T>(fmaf(x0, r.x, -(x1 * r.y)));
                    y.v[v] = from_f32<T>(fmaf(x0, r.y, x1 * r.x));
                }
                rope_store<T, V, VEC>(out + at + half, y, V);
            }
            rope_store<T, V, VEC>(out + at, x, V);
        }
    }
}

RopeSide side_of(const stx_tensor* s, const stx_tensor* d) {
    if (!s) return {};
    return {static_cast<const char*>(s->data), static_cast<char*>(d->data), s->nb[1], s->nb[2], s->nb[3], d->nb[1], d->nb[2], d->nb[3]};
}

template <class T, int V, bool VEC>
void rope_launch(RopeScaledArgs a, int mode, size_t lds, hipStream_t stream) {
    launch_all((a.tokens + a.tile - 1) / a.tile, [&](dim3 grid, unsigned first) {
        const dim3 block(kRopeThreads);
        a.base = first;
        if (mode == 0) hipLaunchKernelGGL((rope_scaled_kernel<T, VEC ? V : 2, VEC, 0>), grid, block, lds, stream, a);
        else hipLaunchKernelGGL((rope_scaled_kernel<T, VEC ? V : 1, VEC, 2>), grid, block, lds, stream, a);
        launch_check("rope_scaled_kernel");
    });
}

void rope_scaled(const stx_tensor* q, const stx_tensor* k, stx_type type, const int32_t* pos, int64_t pos_stride,
                 const stx_rope_params* p, const stx_tensor* q_dst, const stx_tensor* k_dst, float sign, stx_stream stream) {
    const int size = type_size(type);
    check_row_output(q, q_dst, size, "rope_scaled: q");
    STX_REQUIRE((k == nullptr) == (k_dst == nullptr), "rope_scaled: k and k_dst go together");
    if (k) {
        check_row_output(k, k_dst, size, "rope_scaled: k");
        STX_REQUIRE(k->ne[0] == q->ne[0] && k->ne[2] == q->ne[2] && k->ne[3] == q->ne[3],
                    "rope_scaled: q and k differ in head size, tokens or batch");
        STX_REQUIRE(shared(q_dst, k_dst, size) != Shared::yes && shared(q_dst, k, size) != Shared::yes && shared(k_dst, q, size) != Shared::yes,
                    "rope_scaled: an output overlaps the other side's tensors");
    }
    const long long dim = q->ne[0];
    RopeScaledArgs a{};
    a.at = rope_angles(p, dim, pos_stride, sign, "rope_scaled");
    const long long q_rows = q->ne[1], k_rows = k ? k->ne[1] : 0, n = q->ne[2];
    if (n == 0 || q->ne[3] == 0 || q_rows + k_rows == 0) return;
    STX_REQUIRE(n < (1LL << 31) && q->ne[3] < (1LL << 31) && n * q->ne[3] < (1LL << 31), "rope_scaled: more than 2^31 - 1 tokens");
    STX_REQUIRE(q_rows + k_rows < (1LL << 24) && (q_rows + k_rows) * dim < (1LL << 27), "rope_scaled: too many rows a token");
    STX_REQUIRE(pos != nullptr, "rope_scaled: pos is NULL");
    a.q = side_of(q, q_dst);
    a.k = side_of(k, k_dst);
    a.at.pos = pos;
    a.tokens = (unsigned)(n * q->ne[3]);
    a.at.n = FastDiv((unsigned)n);
    a.rows = FastDiv((unsigned)(q_rows + k_rows));
    a.q_rows = (unsigned)q_rows;
    a.dim = (int)dim;
    // The widest access (16, then 8 bytes) that every row's start and, in mode 2, both halves allow.
    const int half = p->n_dims / 2;
    int v = 0;
    for (int bytes : {16, 8}) {
        const int w = bytes / size;
        const bool fits = p->mode == 0 ? dim % w == 0 : half % w == 0 && dim % w == 0;
        if (v == 0 && fits && rows_aligned(q, bytes) && rows_aligned(q_dst, bytes) && rows_aligned(k, bytes) && rows_aligned(k_dst, bytes)) v = w;
    }
    const int w = v ? v : p->mode == 0 ? 2 : 1;
    a.units = FastDiv((unsigned)(p->mode == 0 ? (dim + w - 1) / w : half / w + (dim - p->n_dims + w - 1) / w));
    // Tokens a block: kRopeUnits units a thread, as long as two blocks a CU remain.
    const long long items = (long long)a.rows.d * a.units.d;
    long long tile = std::max(1LL, std::min<long long>(kRopeTile, kRopeThreads * kRopeUnits / items));
    tile = std::min(tile, std::max(1LL, (long long)a.tokens / 512));
    a.tile = (unsigned)std::min<long long>(tile, kRopeTable / half);
    const size_t lds = sizeof(float2) * a.tile * half;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        constexpr int W = 16 / sizeof(T);
        if (v == W) rope_launch<T, W, true>(a, p->mode, lds, as_stream(stream));
        else if (v == W / 2) rope_launch<T, W / 2, true>(a, p->mode, lds, as_stream(stream));
        else rope_launch<T, 1, false>(a, p->mode, lds, as_stream(stream));
    });
}

}  // namespace
}  // namespace stx

using namespace stx;

extern "C" {

STX_API stx_status stx_rope_scaled(const stx_tensor* q, const stx_tensor* k, stx_type type, const int32_t* pos,
                                   int64_t pos_stride, const stx_rope_params* params, const stx_tensor* q_dst,
                                   const stx_tensor* k_dst, stx_stream stream) {
    return guard([&] { rope_scaled(q, k, type, pos, pos_stride, params, q_dst, k_dst, 1.f, stream); });
}

STX_API stx_status stx_rope_scaled_back(const stx_tensor* q, const stx_tensor* k, stx_type type, const int32_t* pos,
                                        int64_t pos_stride, const stx_rope_params* params, const stx_tensor* q_dst,
                                        const stx_tensor* k_dst, stx_stream stream) {
    return guard([&] { rope_scaled(q, k, type, pos, pos_stride, params, q_dst, k_dst, -1.f, stream); });
}

}  // extern "C"

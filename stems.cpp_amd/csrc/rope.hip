// rope.hip — rotary positions over typed tensors with scaled angles, forward and backward
// (stx_rope_scaled, stx_rope_scaled_back).
#include <algorithm>
#include <cmath>

#include "typed.hpp"

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
    const int* pos;
    const float* factors;
    long long pos_stride;
    unsigned tokens, tile;               // all tokens, and of a block
    unsigned base;                       // blocks of the launches before this one
    FastDiv n;                           // ne2: token -> (i3, i2)
    FastDiv rows, units;                 // rows of a token (q's, then k's); units of a row
    unsigned q_rows;
    int dim, n_dims;
    double log2_base, scale, ext, lo, inv_range, m;
    float sign;                          // -1: the gradient
};

// cos and sin of a finite angle |theta| < 2^40: theta - n pi/2 with pi/2 in two doubles (the fma
// makes the first product exact), then Taylor polynomials on |r| <= pi/4, cut below 2^-33.
__device__ __forceinline__ void cos_sin(double theta, double& c, double& s) {
    const double n = rint(theta * 0.63661977236758134308);
    const double r = fma(-n, 6.123233995736765886e-17, fma(-n, 1.57079632679489661923, theta));
    const double z = r * r;
    double ps = -2.50521083854417187751e-08;               // -1/11!
    ps = fma(ps, z, 2.75573192239858906526e-06);
    ps = fma(ps, z, -1.98412698412698412698e-04);
    ps = fma(ps, z, 8.33333333333333333333e-03);
    ps = fma(ps, z, -1.66666666666666666667e-01);
    const double sn = fma(ps * z, r, r);
    double pc = 2.08767569878680989792e-09;                // 1/12!
    pc = fma(pc, z, -2.75573192239858906526e-07);
    pc = fma(pc, z, 2.48015873015873015873e-05);
    pc = fma(pc, z, -1.38888888888888888889e-03);
    pc = fma(pc, z, 4.16666666666666666667e-02);
    pc = fma(pc, z, -5.00000000000000000000e-01);
    const double cn = fma(pc, z, 1.0);
    const int quad = (int)(long long)n & 3;
    c = quad & 1 ? sn : cn;
    s = quad & 1 ? cn : sn;
    if (quad == 1 || quad == 2) c = -c;
    if (quad >= 2) s = -s;
}

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
constexpr int kRopeTable = 4096;         // pairs in LDS: 32 KB
constexpr int kRopeTile = 16;

template <class T, int V, bool VEC, int MODE>
__global__ __launch_bounds__(kRopeThreads) void rope_scaled_kernel(RopeScaledArgs a) {
    extern __shared__ float2 cs[];       // [tile][n_dims / 2]
    const int half = a.n_dims / 2;
    const unsigned t0 = (a.base + blockIdx.x) * a.tile;
    const unsigned nt = min(a.tile, a.tokens - t0);
    for (unsigned e = threadIdx.x; e < nt * (unsigned)half; e += kRopeThreads) {
        const unsigned t = t0 + e / (unsigned)half;
        const int i = (int)(e % (unsigned)half);
        const unsigned i3 = a.n.div(t);
        const double p = (double)a.pos[(long long)i3 * a.pos_stride + (t - i3 * a.n.d)];
        double far = exp2(-2.0 * i / a.n_dims * a.log2_base);
        if (a.factors) far /= (double)a.factors[i];
        const double mix = a.ext * (1.0 - fmin(1.0, fmax(0.0, ((double)i - a.lo) * a.inv_range)));
        double c, s;
        cos_sin(p * (a.ext != 0.0 ? a.scale * far * (1.0 - mix) + far * mix : a.scale * far), c, s);
        cs[e] = make_float2((float)(c * a.m), a.sign * (float)(s * a.m));
    }
    __syncthreads();
    const unsigned total = nt * a.rows.d * a.units.d;
    for (unsigned e = threadIdx.x; e < total; e += kRopeThreads) {
        const unsigned row = a.units.div(e), u = e - row * a.units.d;
        const unsigned tk = a.rows.div(row), h = row - tk * a.rows.d;
        const unsigned t = t0 + tk, i3 = a.n.div(t), i2 = t - i3 * a.n.d;
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
            const int pairs = half / V, at = (int)u < pairs ? (int)u * V : a.n_dims + ((int)u - pairs) * V;
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

// Whether every row of src and dst starts at a multiple of `bytes`.
bool rows_aligned(const stx_tensor* t, int bytes) {
    if (!t) return true;
    bool ok = reinterpret_cast<uintptr_t>(t->data) % bytes == 0;
    for (int i = 1; i < 4; i++) ok = ok && (t->ne[i] <= 1 || t->nb[i] % bytes == 0);
    return ok;
}

void check_out(const stx_tensor* src, const stx_tensor* dst, int size, const char* what) {
    check_typed(src, size, what);
    check_typed(dst, size, what);
    check_same_shape(src, dst, what);
    bool same = src->data == dst->data;
    for (int i = 1; i < 4; i++) {
        STX_REQUIRE(dst->ne[i] <= 1 || dst->nb[i] > 0, "%s: output stride nb[%d] is 0", what, i);
        same = same && (dst->ne[i] <= 1 || dst->nb[i] == src->nb[i]);
    }
    STX_REQUIRE(nelem(view(dst)) == 0 || nested(dst, size), "%s: rows of the output overlap", what);
    // In place with other strides, or in part over the input, rows would be read after they were written.
    STX_REQUIRE(same || src->data != dst->data || nelem(view(src)) == 0, "%s: in place with other strides", what);
    STX_REQUIRE(same || shared(src, dst, size) != Shared::yes, "%s: the output overlaps the input in part", what);
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
    STX_REQUIRE(p != nullptr && p->size >= sizeof(stx_rope_params), "rope_scaled: params are NULL or their size is too small");
    check_out(q, q_dst, size, "rope_scaled: q");
    STX_REQUIRE((k == nullptr) == (k_dst == nullptr), "rope_scaled: k and k_dst go together");
    if (k) {
        check_out(k, k_dst, size, "rope_scaled: k");
        STX_REQUIRE(k->ne[0] == q->ne[0] && k->ne[2] == q->ne[2] && k->ne[3] == q->ne[3],
                    "rope_scaled: q and k differ in head size, tokens or batch");
        STX_REQUIRE(shared(q_dst, k_dst, size) != Shared::yes && shared(q_dst, k, size) != Shared::yes && shared(k_dst, q, size) != Shared::yes,
                    "rope_scaled: an output overlaps the other side's tensors");
    }
    const long long dim = q->ne[0];
    if (p->mode != 0 && p->mode != 2) fail(STX_STATUS_UNSUPPORTED, "rope_scaled: mode %d (only 0 and 2)", p->mode);
    STX_REQUIRE(p->n_dims > 0 && p->n_dims % 2 == 0 && p->n_dims <= dim, "rope_scaled: n_dims must be even, positive and <= ne0");
    if (p->n_dims > 2 * kRopeTable || dim > (1 << 20)) fail(STX_STATUS_UNSUPPORTED, "rope_scaled: rows of %lld with %d rotated", dim, p->n_dims);
    STX_REQUIRE(p->freq_base > 0.f && p->freq_scale > 0.f, "rope_scaled: freq_base and freq_scale must be positive");
    for (float v : {p->freq_base, p->freq_scale, p->ext_factor, p->attn_factor})
        STX_REQUIRE(std::isfinite(v), "rope_scaled: a parameter is not finite");
    STX_REQUIRE(p->ext_factor == 0.f || (std::isfinite(p->beta_fast) && std::isfinite(p->beta_slow)), "rope_scaled: beta_fast or beta_slow is not finite");
    STX_REQUIRE(pos_stride >= 0, "rope_scaled: negative pos_stride");
    RopeScaledArgs a{};
    a.log2_base = std::log2((double)p->freq_base);
    a.scale = p->freq_scale;
    a.ext = p->ext_factor;
    a.m = p->attn_factor;
    if (p->ext_factor != 0.f) {
        STX_REQUIRE(p->n_ctx_orig > 0 && p->beta_fast > 0.f && p->beta_slow > 0.f && p->freq_base != 1.f,
                    "rope_scaled: ext_factor needs n_ctx_orig, beta_fast and beta_slow above 0 and freq_base != 1");
        const double pi = 3.14159265358979323846;
        auto turns = [&](double r) { return p->n_dims * std::log(p->n_ctx_orig / (r * 2 * pi)) / (2 * std::log((double)p->freq_base)); };
        a.lo = std::fmax(0.0, std::floor(turns(p->beta_fast)));
        a.inv_range = 1.0 / std::fmax(0.001, std::fmin(p->n_dims - 1.0, std::ceil(turns(p->beta_slow))) - a.lo);
        a.m *= 1.0 + 0.1 * std::log(1.0 / (double)p->freq_scale);
    }
    const long long q_rows = q->ne[1], k_rows = k ? k->ne[1] : 0, n = q->ne[2];
    if (n == 0 || q->ne[3] == 0 || q_rows + k_rows == 0) return;
    STX_REQUIRE(n < (1LL << 31) && q->ne[3] < (1LL << 31) && n * q->ne[3] < (1LL << 31), "rope_scaled: more than 2^31 - 1 tokens");
    STX_REQUIRE(q_rows + k_rows < (1LL << 24) && (q_rows + k_rows) * dim < (1LL << 27), "rope_scaled: too many rows a token");
    STX_REQUIRE(pos != nullptr, "rope_scaled: pos is NULL");
    a.q = side_of(q, q_dst);
    a.k = side_of(k, k_dst);
    a.pos = pos;
    a.pos_stride = pos_stride;
    a.factors = p->freq_factors;
    a.tokens = (unsigned)(n * q->ne[3]);
    a.n = FastDiv((unsigned)n);
    a.rows = FastDiv((unsigned)(q_rows + k_rows));
    a.q_rows = (unsigned)q_rows;
    a.dim = (int)dim;
    a.n_dims = p->n_dims;
    a.sign = sign;
    // The widest access (16, then 8 bytes) that every row's start and, in mode 2, both halves allow.
    const int half = a.n_dims / 2;
    int v = 0;
    for (int bytes : {16, 8}) {
        const int w = bytes / size;
        const bool fits = p->mode == 0 ? dim % w == 0 : half % w == 0 && dim % w == 0;
        if (v == 0 && fits && rows_aligned(q, bytes) && rows_aligned(q_dst, bytes) && rows_aligned(k, bytes) && rows_aligned(k_dst, bytes)) v = w;
    }
    const int w = v ? v : p->mode == 0 ? 2 : 1;
    a.units = FastDiv((unsigned)(p->mode == 0 ? (dim + w - 1) / w : half / w + (dim - a.n_dims + w - 1) / w));
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

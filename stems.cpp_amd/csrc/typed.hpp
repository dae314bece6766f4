// typed.hpp — element types of the transformer-layer operators (fp32, fp16, bf16): checks of
// typed tensors on the host, conversions, vector access and activations on the device.
#pragma once

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "tensor.hpp"

namespace stx {

using f16 = _Float16;
using bf16 = __bf16;

inline int type_size(stx_type t) {
    switch (t) {
    case STX_TYPE_F32: return 4;
    case STX_TYPE_F16:
    case STX_TYPE_BF16: return 2;
    default: fail(STX_STATUS_INVALID_ARGUMENT, "unknown element type %d", (int)t);
    }
}

template <class T>
constexpr stx_type type_of = std::is_same_v<T, float> ? STX_TYPE_F32 : std::is_same_v<T, f16> ? STX_TYPE_F16 : STX_TYPE_BF16;

// Calls f(T{}) with the device type of t.
template <class F>
void with_type(stx_type t, F&& f) {
    switch (t) {
    case STX_TYPE_F32: return f(float{});
    case STX_TYPE_F16: return f(f16{});
    case STX_TYPE_BF16: return f(bf16{});
    default: fail(STX_STATUS_INVALID_ARGUMENT, "unknown element type %d", (int)t);
    }
}

inline void check_act(stx_act act) {
    STX_REQUIRE(act >= STX_ACT_NONE && act <= STX_ACT_SIGMOID, "unknown activation %d", (int)act);
}

// check_tensor (tensor.hpp) for elements of `size` bytes; the data is aligned to its elements.
inline void check_typed(const stx_tensor* t, int size, const char* what) {
    STX_REQUIRE(t != nullptr, "%s is NULL", what);
    bool none = false;
    for (int i = 0; i < 4; i++) {
        STX_REQUIRE(t->ne[i] >= 0, "%s: negative ne[%d]", what, i);
        none = none || t->ne[i] == 0;
    }
    long long n = none ? 0 : 1;
    for (int i = 0; i < 4 && !none; i++) {
        STX_REQUIRE(t->ne[i] < (1LL << 40) / n, "%s too large", what);
        n *= t->ne[i];
    }
    STX_REQUIRE(t->nb[0] == size, "%s: rows must be contiguous (nb[0] == %d, the element size)", what, size);
    for (int i = 1; i < 4; i++) STX_REQUIRE(t->nb[i] >= 0 && t->nb[i] % size == 0, "%s: bad stride nb[%d]", what, i);
    STX_REQUIRE(n == 0 || t->data != nullptr, "%s has no data", what);
    STX_REQUIRE(reinterpret_cast<uintptr_t>(t->data) % size == 0, "%s: data is not aligned to its elements", what);
}

inline bool contiguous_typed(const stx_tensor* t, int size) {
    long long expect = size;
    bool dense = true;
    for (int i = 0; i < 4; i++) {
        if (t->ne[i] == 0) return true;
        dense = dense && (t->ne[i] == 1 || t->nb[i] == expect);
        expect *= t->ne[i];
    }
    return dense;
}

// First and last byte past the end that a tensor's elements span; {0, 0} without elements.
struct Span {
    uintptr_t lo, hi;
};
inline Span span_of(const stx_tensor* t, int size) {
    uintptr_t lo = reinterpret_cast<uintptr_t>(t->data), hi = lo + size;
    for (int i = 0; i < 4; i++) {
        if (t->ne[i] == 0) return {0, 0};
        hi += (uintptr_t)((t->ne[i] - 1) * t->nb[i]);
    }
    return {lo, hi};
}
inline Span span_of(const void* p, size_t bytes) {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
    return p && bytes ? Span{lo, lo + bytes} : Span{0, 0};
}
inline bool overlap(Span a, Span b) { return a.lo < b.hi && b.lo < a.hi; }

// Whether the elements of tensors can be told apart by their strides: over the dimensions of more than
// one element the strides agree, and each is at least the extent of the dimensions below it.
enum class Shared { no, yes, unknown };
struct Nest {
    int n = 0;
    long long stride[3], na[3], nb[3];   // ascending; elements of a and of b
    bool ok = true;
    Nest(const stx_tensor* a, const stx_tensor* b, int size) {
        for (int i = 1; i < 4; i++) {
            if (a->ne[i] <= 1 && b->ne[i] <= 1) continue;
            ok = ok && (a->ne[i] <= 1 || b->ne[i] <= 1 || a->nb[i] == b->nb[i]);
            const long long s = a->ne[i] > 1 ? a->nb[i] : b->nb[i];
            int at = n++;
            for (; at > 0 && stride[at - 1] > s; at--) stride[at] = stride[at - 1], na[at] = na[at - 1], nb[at] = nb[at - 1];
            stride[at] = s, na[at] = a->ne[i], nb[at] = b->ne[i];
        }
        long long extent = std::max(a->ne[0], b->ne[0]) * size;
        for (int i = 0; i < n; i++) {
            ok = ok && stride[i] >= extent;
            extent += (std::max(na[i], nb[i]) - 1) * stride[i];
        }
    }
    // Whether rows of a and b fall together with b's data `delta` bytes behind a's; dimensions below `i`.
    bool meet(int i, long long delta, long long ra, long long rb) const {
        if (i == 0) return -rb < delta && delta < ra;
        long long la = ra, lb = rb;      // what the lower dimensions reach
        for (int k = 0; k < i - 1; k++) la += (na[k] - 1) * stride[k], lb += (nb[k] - 1) * stride[k];
        const long long s = stride[i - 1];
        auto ceil = [&](long long v) { return v >= 0 ? (v + s - 1) / s : -(-v / s); };
        // delta + d s in (-lb, la) for steps d of b's less a's: three at most, the strides being nested
        for (long long d = std::max(1 - na[i - 1], ceil(1 - lb - delta)), last = std::min(nb[i - 1] - 1, -ceil(1 - la + delta)); d <= last; d++)
            if (meet(i - 1, delta + d * s, ra, rb)) return true;
        return false;
    }
};
inline bool nested(const stx_tensor* t, int size) { return Nest(t, t, size).ok; }
inline Shared shared(const stx_tensor* a, const stx_tensor* b, int size) {
    if (!overlap(span_of(a, size), span_of(b, size))) return Shared::no;
    const Nest n(a, b, size);
    if (!n.ok) return Shared::unknown;
    const long long delta = static_cast<const char*>(b->data) - static_cast<const char*>(a->data);
    return n.meet(n.n, delta, a->ne[0] * size, b->ne[0] * size) ? Shared::yes : Shared::no;
}

// Memory of a call, as a tensor or as so many bytes, and the check that what it writes is nothing else's.
struct Operand {
    const char* what;
    Span span;
    const stx_tensor* t;
    int size;
    Operand(const char* what, const stx_tensor* t, int size) : what(what), span(t ? span_of(t, size) : Span{0, 0}), t(t), size(size) {}
    Operand(const char* what, const void* p, size_t bytes) : what(what), span(span_of(p, bytes)), t(nullptr), size(0) {}
};
inline void check_apart(const char* op, std::initializer_list<Operand> written, std::initializer_list<Operand> read) {
    auto apart = [&](const Operand& a, const Operand& b) {
        const bool same = overlap(a.span, b.span) && !(a.t && b.t && shared(a.t, b.t, a.size) == Shared::no);
        STX_REQUIRE(!same, "%s: %s overlaps %s", op, a.what, b.what);
    };
    for (auto a = written.begin(); a != written.end(); a++) {
        for (auto b = a + 1; b != written.end(); b++) apart(*a, *b);
        for (const Operand& b : read) apart(*a, b);
    }
}

// Whether every row of a tensor (NULL: of none) starts at a multiple of `bytes`.
inline bool rows_aligned(const stx_tensor* t, int bytes) {
    if (!t) return true;
    bool ok = reinterpret_cast<uintptr_t>(t->data) % bytes == 0;
    for (int i = 1; i < 4; i++) ok = ok && (t->ne[i] <= 1 || t->nb[i] % bytes == 0);
    return ok;
}

// Checks of an output of src's shape that may be src, by the strides of both.
inline void check_row_output(const stx_tensor* src, const stx_tensor* dst, int size, const char* what) {
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

inline void check_workspace(const void* ws, size_t have, size_t need, const char* what) {
    if (need == 0) return;
    STX_REQUIRE(ws != nullptr && have >= need, "%s: workspace of %zu bytes needed, %zu given", what, need, ws ? have : (size_t)0);
    STX_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 255) == 0, "%s: the workspace must be 256-byte aligned", what);
}

// Calls launch(grid, first) for blocks in turn, `first` the number of those before: a launch has at
// most 2^32 - 1 threads (here 2^31 of blocks of 256).
template <class F>
void launch_all(unsigned long long blocks, F&& launch) {
    constexpr unsigned kMost = 1u << 23;
    for (unsigned long long first = 0; first < blocks; first += kMost)
        launch(dim3((unsigned)std::min<unsigned long long>(kMost, blocks - first)), (unsigned)first);
}

// ------------------------------------------------------------------------------- device
// N elements moved as one access of N * sizeof(T) bytes.
template <class T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(f16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(bf16 x) { return (float)x; }
// Rounded to nearest even. The float is made opaque before fp16's rounding: the compiler otherwise
// takes v_fma_mixlo_f16 for some fused results and not for others, and that one rounds the
// exact sum to fp16 where the rest round the float, so vector and scalar paths would differ by a bit.
template <class T>
__device__ __forceinline__ T from_f32(float x) {
    if constexpr (std::is_same_v<T, f16>) asm("" : "+v"(x));
    return (T)x;
}

// exp(-z) on the hardware's 2^y (1 ulp), y = -z log2 e. Rounding y costs |z| / 2 ulps. FINE, for fp32
// results, adds what was rounded off (two more ulps at any z, five instructions); for 16-bit
// ones those ulps lie 2^12 below their own. The rest is held to [-1, 1] for infinite z.
template <bool FINE>
__device__ __forceinline__ float exp_neg(float z) {
    constexpr float C1 = -0x1.715476p0f, C2 = -0x1.4ae0cp-26f;       // -log2 e
    const float y = z * (FINE ? C1 : -1.44269504088896340736f), e = __builtin_amdgcn_exp2f(y);
    if constexpr (!FINE) return e;
    const float rest = __builtin_amdgcn_fmed3f(fmaf(z, C2, fmaf(z, C1, -y)), -1.f, 1.f);
    return e * fmaf(rest, 0.69314718055994530942f, 1.f);
}

// s = 1 / (1 + exp(-z)), and r = 1 - s, not by a subtraction where s is near 1.
template <bool FINE>
__device__ __forceinline__ float sigmoid_f32(float z) { return __builtin_amdgcn_rcpf(1.f + exp_neg<FINE>(z)); }
template <bool FINE>
__device__ __forceinline__ float sigmoid_f32(float z, float& r) {
    const float e = exp_neg<FINE>(z), s = __builtin_amdgcn_rcpf(1.f + e);
    r = z > 0.f ? e * s : 1.f - s;
    return s;
}

// Phi(z), the normal distribution, and zphi = z exp(-z^2/2): Phi(-|z|) = exp(-z^2/2) t P(t) / 2 with
// t = 1 / (1 + |z| / (2 sqrt2)), P the polynomial of stx_gelu_erf (gelu_phi_neg in ops.hip). Rounding the
// exponent costs z^2 / 4 ulps, and 2^y ends at 2^-126. FINE, for fp32 results, forms q = exp(-z^2/4) from an
// exponent in two parts, whose square neither loses them nor ends before fp32 does, seven
// instructions more; |z| is taken as 18 at most there, where q^2 is 0.
template <bool FINE>
__device__ __forceinline__ float normal_cdf(float z, float& zphi) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.35355339059327376220f, fabsf(z), 1.f));
    float p = -1.5161373655e-02f;
    p = fmaf(p, t, 9.183117002e-02f);
    p = fmaf(p, t, -2.2204872965e-01f);
    p = fmaf(p, t, 2.545801103e-01f);
    p = fmaf(p, t, -1.139718890e-01f);
    p = fmaf(p, t, 4.3268962765e-03f);
    p = fmaf(p, t, -3.3629499375e-02f);
    p = fmaf(p, t, -1.2177567695e-03f);
    p = fmaf(p, t, 4.1566714645e-02f);
    p = fmaf(p, t, 8.82191360e-02f);
    p = fmaf(p, t, 1.234102100e-01f);
    p = fmaf(p, t, 1.4104762675e-01f);
    p = fmaf(p, t, 1.410473883e-01f);
    float tail;
    if constexpr (FINE) {
        constexpr float C1 = -0x1.715476p-2f, C2 = -0x1.4ae0cp-28f;  // -log2 e / 4
        const float c = __builtin_amdgcn_fmed3f(z, -18.f, 18.f), h = c * c, y = h * C1;
        const float rest = fmaf(h, C2, fmaf(fmaf(c, c, -h), C1, fmaf(h, C1, -y)));
        float q = __builtin_amdgcn_exp2f(y);
        q = fmaf(q, rest * 0.69314718055994530942f, q);
        tail = q * (q * (t * p));
        zphi = c * q * q;
    } else {
        const float phi = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170368f);
        tail = phi * (t * p);
        zphi = z * phi;
    }
    return z < 0.f ? tail : 1.f - tail;
}

// act(z), and its derivative d, for results of type T.
template <int ACT, class T>
__device__ __forceinline__ float act_f32(float z) {
    constexpr bool FINE = sizeof(T) == 4;
    float zphi;
    if constexpr (ACT == STX_ACT_GELU) return z * normal_cdf<FINE>(z, zphi);
    if constexpr (ACT == STX_ACT_SILU) return z * sigmoid_f32<FINE>(z);
    if constexpr (ACT == STX_ACT_SIGMOID) return sigmoid_f32<FINE>(z);
    return z;
}
template <int ACT, class T>
__device__ __forceinline__ float act_f32(float z, float& d) {
    constexpr bool FINE = sizeof(T) == 4;
    if constexpr (ACT == STX_ACT_GELU) {
        float zphi;
        const float c = normal_cdf<FINE>(z, zphi);
        d = fmaf(zphi, 0.39894228040143267794f, c);                 // Phi + z phi / sqrt(2 pi)
        return z * c;
    } else if constexpr (ACT == STX_ACT_SILU || ACT == STX_ACT_SIGMOID) {
        float r;
        const float s = sigmoid_f32<FINE>(z, r);
        if (ACT == STX_ACT_SILU && !FINE) r = 1.f - s;               // beside 1 its digits do not count in 16 bits (4 % of a gradient's time)
        d = ACT == STX_ACT_SILU ? s * fmaf(z, r, 1.f) : s * r;
        return ACT == STX_ACT_SILU ? z * s : s;
    } else {
        d = 1.f;
        return z;
    }
}

// Calls f(std::integral_constant<int, act>{}), on the host or (act uniform over the launch) in a kernel.
template <class F>
__host__ __device__ __forceinline__ void with_act(int act, F&& f) {
    switch (act) {
    case STX_ACT_GELU: return f(std::integral_constant<int, STX_ACT_GELU>{});
    case STX_ACT_SILU: return f(std::integral_constant<int, STX_ACT_SILU>{});
    case STX_ACT_SIGMOID: return f(std::integral_constant<int, STX_ACT_SIGMOID>{});
    default: return f(std::integral_constant<int, STX_ACT_NONE>{});
    }
}

}  // namespace stx

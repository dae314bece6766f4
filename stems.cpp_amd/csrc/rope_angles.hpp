// rope_angles.hpp — the rotation of stx_rope_params: its checks on the host, its cos and sin on the
// device (rope.hip, qk_norm.hip).
#pragma once

#include <cmath>

#include "typed.hpp"

namespace stx {

constexpr int kRopeTable = 4096;         // pairs in LDS: 32 KB

struct RopeAngles {
    const int* pos;
    const float* factors;
    long long pos_stride;
    FastDiv n;                           // tokens of a sequence: token -> (i3, i2)
    int n_dims;
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

// Pair i's angle a position.
__device__ __forceinline__ double rope_frequency(const RopeAngles& a, int i) {
    double far = exp2(-2.0 * i / a.n_dims * a.log2_base);
    if (a.factors) far /= (double)a.factors[i];
    const double mix = a.ext * (1.0 - fmin(1.0, fmax(0.0, ((double)i - a.lo) * a.inv_range)));
    return a.ext != 0.0 ? a.scale * far * (1.0 - mix) + far * mix : a.scale * far;
}
// cos and sin of the pairs of `nt` tokens from t0 on, by a block of THREADS: cs[token][n_dims / 2]. frequency(i): pair i's.
template <int THREADS, class F>
__device__ __forceinline__ void rope_table(const RopeAngles& a, unsigned t0, unsigned nt, float2* cs, F&& frequency) {
    const int half = a.n_dims / 2;
    for (unsigned e = threadIdx.x; e < nt * (unsigned)half; e += THREADS) {
        const unsigned t = t0 + e / (unsigned)half;
        const int i = (int)(e % (unsigned)half);
        const unsigned i3 = a.n.div(t);
        const double p = (double)a.pos[(long long)i3 * a.pos_stride + (t - i3 * a.n.d)];
        double c, s;
        cos_sin(p * frequency(i), c, s);
        cs[e] = make_float2((float)(c * a.m), a.sign * (float)(s * a.m));
    }
}
template <int THREADS>
__device__ __forceinline__ void rope_table(const RopeAngles& a, unsigned t0, unsigned nt, float2* cs) {
    rope_table<THREADS>(a, t0, nt, cs, [&](int i) { return rope_frequency(a, i); });
}

// Checks of the parameters and positions for rows of `dim` elements; the rotation without pos and n.
inline RopeAngles rope_angles(const stx_rope_params* p, long long dim, int64_t pos_stride, float sign, const char* op) {
    STX_REQUIRE(p != nullptr && p->size >= sizeof(stx_rope_params), "%s: params are NULL or their size is too small", op);
    if (p->mode != 0 && p->mode != 2) fail(STX_STATUS_UNSUPPORTED, "%s: mode %d (only 0 and 2)", op, p->mode);
    STX_REQUIRE(p->n_dims > 0 && p->n_dims % 2 == 0 && p->n_dims <= dim, "%s: n_dims must be even, positive and <= ne0", op);
    if (p->n_dims > 2 * kRopeTable || dim > (1 << 20)) fail(STX_STATUS_UNSUPPORTED, "%s: rows of %lld with %d rotated", op, dim, p->n_dims);
    STX_REQUIRE(p->freq_base > 0.f && p->freq_scale > 0.f, "%s: freq_base and freq_scale must be positive", op);
    for (float v : {p->freq_base, p->freq_scale, p->ext_factor, p->attn_factor})
        STX_REQUIRE(std::isfinite(v), "%s: a parameter is not finite", op);
    STX_REQUIRE(p->ext_factor == 0.f || (std::isfinite(p->beta_fast) && std::isfinite(p->beta_slow)), "%s: beta_fast or beta_slow is not finite", op);
    STX_REQUIRE(pos_stride >= 0, "%s: negative pos_stride", op);
    RopeAngles a{};
    a.pos_stride = pos_stride;
    a.factors = p->freq_factors;
    a.n_dims = p->n_dims;
    a.sign = sign;
    a.log2_base = std::log2((double)p->freq_base);
    a.scale = p->freq_scale;
    a.ext = p->ext_factor;
    a.m = p->attn_factor;
    if (p->ext_factor != 0.f) {
        STX_REQUIRE(p->n_ctx_orig > 0 && p->beta_fast > 0.f && p->beta_slow > 0.f && p->freq_base != 1.f,
                    "%s: ext_factor needs n_ctx_orig, beta_fast and beta_slow above 0 and freq_base != 1", op);
        const double pi = 3.14159265358979323846;
        auto turns = [&](double r) { return p->n_dims * std::log(p->n_ctx_orig / (r * 2 * pi)) / (2 * std::log((double)p->freq_base)); };
        a.lo = std::fmax(0.0, std::floor(turns(p->beta_fast)));
        a.inv_range = 1.0 / std::fmax(0.001, std::fmin(p->n_dims - 1.0, std::ceil(turns(p->beta_slow))) - a.lo);
        a.m *= 1.0 + 0.1 * std::log(1.0 / (double)p->freq_scale);
    }
    return a;
}

}  // namespace stx

// diff_attention.hip — differential attention, forward (stx_diff_attention).
#include "diff_attention.hpp"

namespace stx {
namespace {

// out = softmax(s q1 k1^T) v - lambda softmax(s q2 k2^T) v for the rows of a (sequence, key head), one pass over the
// keys: each map keeps a running maximum m, the sum of exp(z - m) and the sum of exp(z - m) v, and both share the
// tiles of k and v in LDS. A wave has NQ x 16 rows. It forms S^T = K Q^T with the rows' q in registers, so that a
// lane holds scores of one row (column lane % 16): the softmax needs two exchanges between lanes a tile, and
// the exponentials are, where they stand, the operand of O^T = V^T P^T. v is read transposed from its tile.
// WK waves share rows and split a tile's keys between them (few rows: single tokens); others have rows of their own.
//
// m is raised only where an exponential passes 2^14, as a first tile's do against -inf: a sum scaled by any power is as
// good, most tiles then need neither the row's maximum nor a scaling of the sums, and the check is on
// exponentials, which the compiler knows to be canonical (maxima of the products take an instruction more each).
//
// P is rounded to 16 bits for its product (16-bit data). Rounding both maps once leaves the difference 1.54 times the error
// that rounding the result alone has (60 x 801 frames, lambda about 0.5: 2.5e-3 in bf16 where it is 1.65e-3), for the maps cancel and
// their errors do not. The first map, which weighs more, is taken in two parts, 1.06 times; 204 -> 232 us.
// fp16's P is scaled by 2^6 so that shares of 2^-20 keep all their bits.
//
// Those 60 x 801 frames of 4 heads of 64 and 128 take 215 to 230 us (551 TFLOP/s of the formula's products), 4 x 4 heads of 8,192 x 8,192
// 960 us (860): exponentials (vector units 56 % busy) and products (matrix cores 42 %), which two waves a SIMD overlap in part. Of 801 rows the
// last tile of 128 has 33, so two of its waves work for nothing, and 1,680 blocks are 3.3 rounds of the 512 that fit.
// One token of 8 sequences over caches of up to 16,384 (210 MB): 40 us, 5 TB/s, and 5 us to join the parts.
template <class T>
constexpr float kShift = std::is_same_v<T, f16> ? 6.f : 0.f;

// Keys of a tile: tiles of k and v of 32 KB together; where waves split them, KEYS a wave at least.
template <class T, int DP, int VP, int WK>
constexpr int tile_keys() {
    constexpr int fit = 32768 / ((2 * DP + VP) * (int)sizeof(T)), least = Tile<T, DP>::KEYS * WK;
    constexpr int p = fit >= 128 ? 128 : fit >= 64 ? 64 : fit >= 32 ? 32 : 16;
    return p > least ? p : least;
}

template <class T, int DP, int VP, int NQ, int WAVES, int WK, bool ALIGNED>
__global__ __launch_bounds__(64 * WAVES, WK == 1 ? 2 : 1) void diff_attention_kernel(DiffArgs a) {
    constexpr int NT = 64 * WAVES, BK = tile_keys<T, DP, VP, WK>(), KW = BK / WK, KG = Tile<T, DP>::KEYS, KS = KW < 64 / NQ ? KW : 64 / NQ;
    constexpr bool SPLIT = sizeof(T) == 2;
    constexpr int ROWS = 16 * NQ * (WAVES / WK), GD = Tile<T, DP>::GROUPS, NV = VP / 16;
    using KL = Loader<T, DP, BK, 2, NT, ALIGNED>;
    using VL = Loader<T, VP, BK, 1, NT, ALIGNED>;
    constexpr int STAGE = KL::BYTES + VL::BYTES, JOIN = WK > 1 ? WK * 2 * NV * 64 * 16 : 0, LDS = 2 * STAGE > JOIN ? 2 * STAGE : JOIN;
    static_assert(KW % KS == 0 && KS % KG == 0 && LDS <= 160 * 1024);
    __shared__ __align__(128) char lds[LDS];
    const unsigned lds0 = lds_address(lds);

    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, wk = wave % WK, s = lane % 16;
    const unsigned item = blockIdx.x, per = a.tile_div.div(item);
    int tile = (int)(item - per * a.tile_div.d);
    const int split = tile / a.tiles;
    tile -= split * a.tiles;
    if (a.causal) tile = a.tiles - 1 - tile;                          // the longest first
    const int b = (int)a.kv_div.div(per), kvh = (int)(per - b * a.kv_div.d);
    const Mask mask(a, b);
    const int r0 = tile * ROWS, last = min(r0 + ROWS, a.rows) - 1;
    const int most = mask.limit((int)a.group_div.div((unsigned)last)), least = mask.limit((int)a.group_div.div((unsigned)r0));
    int begin = 0, end = most;
    if (a.splits > 1) {
        const int share = ((most + BK - 1) / BK + a.splits - 1) / a.splits * BK;
        begin = min((long long)split * share, (long long)most);
        end = (int)min((long long)begin + share, (long long)most);
    }

    const char* kb = a.k.p + 2LL * kvh * a.k.s1 + b * a.k.s3;
    const char* vb = a.v.p + (long long)kvh * a.v.s1 + b * a.v.s3;
    KL kl;
    VL vl;
    kl.space(a.k.s2, a.k.s1);
    vl.space(a.v.s2, 0);
    auto fetch = [&](int key0, int stage) {
        if (ALIGNED && key0 + BK <= mask.length && a.dim == DP && a.vdim == VP) {
            kl.fetch_whole(lds0 + stage * STAGE, kb + key0 * a.k.s2, a.k.s2, a.k.s1);
            vl.fetch_whole(lds0 + stage * STAGE + KL::BYTES, vb + key0 * a.v.s2, a.v.s2, 0);
            return;
        }
        kl.fetch(lds0 + stage * STAGE, a.dim, [&](int map, int r) { return key0 + r < mask.length ? kb + map * a.k.s1 + (key0 + r) * a.k.s2 : nullptr; });
        vl.fetch(lds0 + stage * STAGE + KL::BYTES, a.vdim, [&](int, int r) { return key0 + r < mask.length ? vb + (key0 + r) * a.v.s2 : nullptr; });
    };
    if (begin < end) fetch(begin, 0);

    u32x4 qf[2][NQ][GD];
    int limit[NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const int r = min(r0 + (wave / WK * NQ + n) * 16 + s, a.rows - 1);
        const RowAt row(a, kvh, r);
        limit[n] = mask.limit(row.query);
#pragma unroll
        for (int m = 0; m < 2; m++) load_fragments<T, DP>(qf[m][n], row.at(a.q, b, 2, m), a.dim, lane);
    }
    f32x4 acc[2][NQ][NV] = {};
    float top[2][NQ], sum[2][NQ];        // m less the shift, of the row; this lane's share of the sum
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int n = 0; n < NQ; n++) top[m][n] = -__builtin_inff(), sum[m][n] = 0.f;
    const float c = a.scale * kLog2e;

    int stage = 0;
    for (int key0 = begin; key0 < end; key0 += BK) {
        kl.settle(lds + stage * STAGE);
        vl.settle(lds + stage * STAGE + KL::BYTES);
        arrived<ALIGNED>();
        if (key0 + BK < end) fetch(key0 + BK, stage ^ 1);
        const char *ks = lds + stage * STAGE, *vs = ks + KL::BYTES;
        const bool whole = key0 + BK <= least && key0 + BK <= end;
#pragma unroll 1
        for (int k0 = 0; k0 < KW; k0 += KS) {
            const int at = wk * KW + k0;
            f32x4 z[2][NQ][KS / 16];
#pragma unroll
            for (int m = 0; m < 2; m++) {
#pragma unroll
                for (int t = 0; t < KS / 16; t++) {
#pragma unroll
                    for (int n = 0; n < NQ; n++) z[m][n][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int g = 0; g < GD; g++) {
                        const u32x4 kf = Tile<T, DP>::plain(ks + m * BK * Tile<T, DP>::BYTES, at + t * 16, g, lane);
#pragma unroll
                        for (int n = 0; n < NQ; n++) z[m][n][t] = mma(kf, qf[m][n][g], z[m][n][t], T{});
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (!whole) {
                asm volatile("");
#pragma unroll
                for (int n = 0; n < NQ; n++) {
                    const int left = min(limit[n], end) - (key0 + at + lane / 16 * 4);
#pragma unroll
                    for (int m = 0; m < 2; m++)
#pragma unroll
                        for (int t = 0; t < KS / 16; t++)
#pragma unroll
                            for (int e = 0; e < 4; e++) z[m][n][t][e] = t * 16 + e < left ? z[m][n][t][e] : -__builtin_inff();
                }
            }
            u32x4 p[2][NQ][KS / KG];
            u32x4 low[SPLIT ? NQ : 1][KS / KG];
#pragma unroll
            for (int m = 0; m < 2; m++) {
#pragma unroll
                for (int n = 0; n < NQ; n++) {
                    f32x4 e[KS / 16];
                    float high = 0.f;
                    auto raise = [&](float base) {
#pragma unroll
                        for (int t = 0; t < KS / 16; t++)
#pragma unroll
                            for (int i = 0; i < 4; i++) e[t][i] = __builtin_amdgcn_exp2f(fmaf(z[m][n][t][i], c, -base));
                    };
                    raise(top[m][n]);
#pragma unroll
                    for (int t = 0; t < KS / 16; t++) high = fmaxf(fmaxf(fmaxf(high, e[t][0]), e[t][1]), fmaxf(e[t][2], e[t][3]));
                    if (__builtin_amdgcn_ballot_w64(!(high <= 0x1p14f && top[m][n] > -__builtin_inff()))) {   // -inf: no key yet
                        float most = -__builtin_inff();
#pragma unroll
                        for (int t = 0; t < KS / 16; t++)
#pragma unroll
                            for (int i = 0; i < 4; i++) most = fmaxf(most, z[m][n][t][i]);
                        const float up = fmaxf(top[m][n], column_max(most) * c - kShift<T>), base = up == -__builtin_inff() ? 0.f : up;
                        const float f = __builtin_amdgcn_exp2f(top[m][n] - base);
                        top[m][n] = up;
                        sum[m][n] *= f;
#pragma unroll
                        for (int i = 0; i < NV; i++) acc[m][n][i] *= f;
                        raise(base);
                    }
#pragma unroll
                    for (int t = 0; t < KS / 16; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) sum[m][n] += e[t][i];
#pragma unroll
                    for (int g = 0; g < KS / KG; g++) {
                        p[m][n][g] = chunk_of<T>(&e[g * KG / 16]);
                        if (SPLIT && m == 0) low[n][g] = rest_of<T>(&e[g * KG / 16], p[m][n][g]);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int g = 0; g < KS / KG; g++)
#pragma unroll
                for (int i = 0; i < NV; i++) {
                    const u32x4 vf = Tile<T, VP>::columns(vs, at + g * KG, i, lane);
#pragma unroll
                    for (int m = 0; m < 2; m++)
#pragma unroll
                        for (int n = 0; n < NQ; n++) acc[m][n][i] = mma(vf, p[m][n][g], acc[m][n][i], T{});
                    if constexpr (SPLIT) {
#pragma unroll
                        for (int n = 0; n < NQ; n++) acc[0][n][i] = mma(vf, low[n][g], acc[0][n][i], T{});
                    }
                }
        }
        stage ^= 1;
    }
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            sum[m][n] = column_sum(sum[m][n]);
        }

    if constexpr (WK > 1) {              // the waves' sums, at the largest of their maxima
        static_assert(NQ == 1);
        __shared__ float stat[WK][2][2][16];
        __syncthreads();                                             // the tiles are read
        if (lane < 16) {
#pragma unroll
            for (int m = 0; m < 2; m++) stat[wk][m][0][s] = top[m][0], stat[wk][m][1][s] = sum[m][0];
        }
        f32x4* join = reinterpret_cast<f32x4*>(lds);                 // [WK][2][NV][64]
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int i = 0; i < NV; i++) join[((wk * 2 + m) * NV + i) * 64 + lane] = acc[m][0][i];
        __syncthreads();
#pragma unroll
        for (int m = 0; m < 2; m++) {
            float up = -__builtin_inff(), f[WK];
#pragma unroll
            for (int w = 0; w < WK; w++) up = fmaxf(up, stat[w][m][0][s]);
            const float base = up == -__builtin_inff() ? 0.f : up;
            top[m][0] = up, sum[m][0] = 0.f;
#pragma unroll
            for (int w = 0; w < WK; w++) {
                f[w] = __builtin_amdgcn_exp2f(stat[w][m][0][s] - base);
                sum[m][0] = fmaf(stat[w][m][1][s], f[w], sum[m][0]);
            }
#pragma unroll
            for (int i = 0; i < NV; i++) {                           // wave wk finishes columns wk, wk + WK, ...
                if (i % WK != wk) continue;
                f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < WK; w++) v += join[((w * 2 + m) * NV + i) * 64 + lane] * f[w];
                acc[m][0][i] = v;
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const int r = r0 + (wave / WK * NQ + n) * 16 + s;
        if (r >= a.rows) continue;
        const RowAt row(a, kvh, r);
        if (a.splits > 1) {
            const long long at = ((long long)split * gridDim.x / a.tile_div.d + per) * a.rows + r;
            if (wk == 0 && lane < 16) {
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    a.part_stat[at * 4 + m * 2] = top[m][n];
                    a.part_stat[at * 4 + m * 2 + 1] = sum[m][n];
                }
            }
#pragma unroll
            for (int i = 0; i < NV; i++) {
                if (WK > 1 && i % WK != wk) continue;
#pragma unroll
                for (int m = 0; m < 2; m++) *reinterpret_cast<f32x4*>(a.part + (at * 2 + m) * VP + i * 16 + lane / 16 * 4) = acc[m][n][i];
            }
            continue;
        }
        float inv[2];
#pragma unroll
        for (int m = 0; m < 2; m++) {
            inv[m] = sum[m][n] == 0.f ? 0.f : 1.f / sum[m][n];
            if (a.lse && wk == 0 && lane < 16) a.lse[row.stat(a, b, m)] = sum[m][n] == 0.f ? -__builtin_inff() : (top[m][n] + __builtin_amdgcn_logf(sum[m][n])) * 0.69314718055994530942f;
        }
        const float lam = a.lam[row.head];
        char* out = const_cast<char*>(row.at(a.out, b, 1, 0));
        char* second = a.second.p ? const_cast<char*>(row.at(a.second, b, 1, 0)) : nullptr;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            if (WK > 1 && i % WK != wk) continue;
            const int at = i * 16 + lane / 16 * 4;
            float o[4], o2[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                o2[e] = acc[1][n][i][e] * inv[1];
                o[e] = fmaf(-lam, o2[e], acc[0][n][i][e] * inv[0]);
            }
            store4<T>(out + at * sizeof(T), a.vdim - at, o);
            if (second) store4<T>(second + at * sizeof(T), a.vdim - at, o2);
        }
    }
}

// Rows whose keys were split: a wave a row. A lane has a part (64 at most), its share of the row then goes to all.
template <class T>
__global__ __launch_bounds__(64) void diff_join_kernel(DiffArgs a, int vp, long long all) {
    __shared__ float share[2][64];
    const long long index = blockIdx.x;                              // of (sequence, key head), row
    const int lane = threadIdx.x;
    const unsigned per = (unsigned)(index / a.rows);
    const int r = (int)(index - (long long)per * a.rows), b = (int)a.kv_div.div(per), kvh = (int)(per - b * a.kv_div.d);
    const RowAt row(a, kvh, r);
    const float lam = a.lam[row.head];
#pragma unroll
    for (int m = 0; m < 2; m++) {
        const float* stat = a.part_stat + ((long long)min(lane, a.splits - 1) * all + index) * 4 + m * 2;
        const float top = lane < a.splits ? stat[0] : -__builtin_inff(), sum = lane < a.splits ? stat[1] : 0.f;
        const float up = lane_max<64>(top), base = up == -__builtin_inff() ? 0.f : up, f = __builtin_amdgcn_exp2f(top - base);
        const float total = (float)lane_sum<64>((double)(sum * f));
        share[m][lane] = total == 0.f ? 0.f : f / total;
        if (a.lse && lane == 0) a.lse[row.stat(a, b, m)] = total == 0.f ? -__builtin_inff() : (up + __builtin_amdgcn_logf(total)) * 0.69314718055994530942f;
    }
    __syncthreads();
    T* out = reinterpret_cast<T*>(const_cast<char*>(row.at(a.out, b, 1, 0)));
    T* second = a.second.p ? reinterpret_cast<T*>(const_cast<char*>(row.at(a.second, b, 1, 0))) : nullptr;
    for (int d = lane; d < a.vdim; d += 64) {
        float o[2] = {};
#pragma unroll 8
        for (int i = 0; i < a.splits; i++)
#pragma unroll
            for (int m = 0; m < 2; m++) o[m] = fmaf(a.part[((i * all + index) * 2 + m) * vp + d], share[m][i], o[m]);
        out[d] = from_f32<T>(fmaf(-lam, o[1], o[0]));
        if (second) second[d] = from_f32<T>(o[1]);
    }
}

// --------------------------------------------------------------------------------- host
// How a call goes over its rows: `few` where a block's waves split the keys of 16 rows, otherwise 64 or 128
// rows a block; keys in parts where the blocks would leave CUs idle.
constexpr int kCus = 256;
struct ForwardPlan {
    bool few;
    int nq, rows, vp, splits;
    long long tiles, blocks;
    size_t part, stat, total;
};
size_t pad256(size_t n) { return (n + 255) / 256 * 256; }
ForwardPlan forward_plan(const DiffShape& s, int size) {
    ForwardPlan p{};
    const long long rows = s.M * (s.H / s.Hk), pairs = s.B * s.Hk;
    const bool small = s.D <= 64 && s.V <= 128;
    p.few = rows <= 16;
    p.nq = !p.few && small && size == 2 && rows > 64 ? 2 : 1;
    p.rows = p.few ? 16 : 64 * p.nq;
    with_dims(s.D, s.V, [&](auto, auto v) { p.vp = v(); });
    p.tiles = (rows + p.rows - 1) / p.rows;
    p.blocks = p.tiles * pairs;
    const long long keys = p.few ? 256 : 128;                         // of a part, at least
    p.splits = (int)std::max(1LL, std::min({2LL * kCus / p.blocks, (s.N + keys - 1) / keys, 64LL}));
    if (p.splits > 1) {
        p.part = pad256((size_t)p.splits * pairs * rows * 2 * p.vp * sizeof(float));
        p.stat = pad256((size_t)p.splits * pairs * rows * 4 * sizeof(float));
    }
    p.total = p.part + p.stat;
    return p;
}

template <class T, int DP, int VP>
void launch_forward(const DiffArgs& a, const ForwardPlan& p, bool aligned, hipStream_t stream) {
    const dim3 grid((unsigned)(p.blocks * p.splits));
    constexpr int W = DP == 128 ? 2 : 4;                              // waves that split keys: what LDS holds two stages of
    if (!aligned) {
        hipLaunchKernelGGL((diff_attention_kernel<T, DP, VP, 1, 4, 1, false>), grid, dim3(256), 0, stream, a);
    } else if (p.few) {
        hipLaunchKernelGGL((diff_attention_kernel<T, DP, VP, 1, W, W, true>), grid, dim3(64 * W), 0, stream, a);
    } else if (p.nq == 1) {
        hipLaunchKernelGGL((diff_attention_kernel<T, DP, VP, 1, 4, 1, true>), grid, dim3(256), 0, stream, a);
    } else if constexpr (sizeof(T) == 2 && DP <= 64) {
        hipLaunchKernelGGL((diff_attention_kernel<T, DP, VP, 2, 4, 1, true>), grid, dim3(256), 0, stream, a);
    }
    launch_check("diff_attention_kernel");
}

}  // namespace
}  // namespace stx

using namespace stx;

extern "C" {

STX_API size_t stx_diff_attention_workspace_size(const stx_tensor* q, const stx_tensor* k, const stx_tensor* v, stx_type type) {
    size_t bytes = 0;
    (void)guard([&] {
        const char* op = "diff_attention_workspace_size";
        const int size = type_size(type);
        for (const stx_tensor* t : {q, k, v}) {
            STX_REQUIRE(t != nullptr, "%s: a tensor is NULL", op);
            for (int i = 0; i < 4; i++) STX_REQUIRE(t->ne[i] >= 0, "%s: negative ne[%d]", op, i);
        }
        const DiffShape s = diff_shape(q, k, v, op);
        if (!s.empty()) bytes = forward_plan(s, size).total;
    });
    return bytes;
}

STX_API stx_status stx_diff_attention(const stx_tensor* q, const stx_tensor* k, const stx_tensor* v, stx_type type, const float* lambda,
                                      float scale, int causal, const int32_t* lengths, const int32_t* starts, const stx_tensor* dst,
                                      const stx_tensor* second, float* lse, void* workspace, size_t workspace_bytes, stx_stream stream) {
    return guard([&] {
        const char* op = "diff_attention";
        const int size = type_size(type);
        check_typed(q, size, "diff_attention: q");
        check_typed(k, size, "diff_attention: k");
        check_typed(v, size, "diff_attention: v");
        const DiffShape s = diff_shape(q, k, v, op);
        check_out_rows(dst, s.V, s.H, s.M, s.B, size, "diff_attention: dst");
        check_nested(dst, size, "diff_attention: dst");
        if (second) {
            check_out_rows(second, s.V, s.H, s.M, s.B, size, "diff_attention: second");
            check_nested(second, size, "diff_attention: second");
        }
        check_scale(scale, op);
        if (s.empty()) return;
        ForwardPlan p = forward_plan(s, size);
        const bool aligned = rows_in_chunks(k, size) && rows_in_chunks(v, size);
        check_workspace(workspace, workspace_bytes, p.total, op);
        const size_t per = (size_t)s.B * sizeof(int32_t);
        check_apart(op, {{"dst", dst, size}, {"second", second, size}, {"lse", lse, (size_t)s.B * s.H * 2 * s.M * sizeof(float)}, {"the workspace", p.total ? workspace : nullptr, p.total}},
                    {{"q", q, size}, {"k", k, size}, {"v", v, size}, {"lambda", lambda, s.H * sizeof(float)}, {"lengths", lengths, per}, {"starts", starts, per}});
        STX_REQUIRE(lambda != nullptr, "%s: lambda is NULL", op);
        if (!aligned) {                  // one form of any alignment: 64 rows a block
            p.rows = 64;
            p.tiles = (s.M * (s.H / s.Hk) + 63) / 64;
            p.blocks = p.tiles * s.B * s.Hk;
        }
        STX_REQUIRE(p.blocks * p.splits < (1LL << 22), "%s: too many tiles", op);
        DiffArgs a = diff_args(s, q, k, v, lambda, scale, causal, lengths, starts);
        a.out = strided(dst), a.second = strided(second);
        a.lse = lse;
        a.tiles = (int)p.tiles, a.splits = p.splits;
        a.tile_div = FastDiv((unsigned)(p.tiles * p.splits));
        a.part = static_cast<float*>(workspace);
        a.part_stat = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.part);
        with_type(type, [&](auto t) {
            using T = decltype(t);
            with_dims(s.D, s.V, [&](auto d, auto v) { launch_forward<T, d(), v()>(a, p, aligned, as_stream(stream)); });
            if (p.splits == 1) return;
            const long long all = s.B * s.Hk * a.rows;
            hipLaunchKernelGGL((diff_join_kernel<T>), dim3((unsigned)all), dim3(64), 0, as_stream(stream), a, p.vp, all);
            launch_check("diff_join_kernel");
        });
    });
}

}  // extern "C"

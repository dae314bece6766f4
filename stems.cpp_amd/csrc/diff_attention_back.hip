// diff_attention_back.hip — the gradients of differential attention (stx_diff_attention_back).
#include "diff_attention.hpp"

namespace stx {
namespace {

// With P_m = exp(z_m - lse_m), O_m = P_m v and dP = dy v^T, D_m = rowsum(dy O_m):
//   dS_1 = P_1 (dP - D_1),  dS_2 = -lambda P_2 (dP - D_2),  dq_m = s dS_m k_m,  dk_m = s dS_m^T q_m,
//   dv = (P_1 - lambda P_2)^T dy,  dlambda = -sum P_2 dP.
// Two kernels form the scores again, 14 D products where one that adds to dq from every block of keys would have 10 D, and need no
// atomics: results are the same each time. The first has rows in registers and goes over the keys (dq, dlambda,
// and D, from dy and the kept outputs, for the second); the second has keys in registers and goes over the rows of
// its key head, so that gradients of shared heads add up in the accumulators. As in the forward kernel the accumulators of
// one product are, where they stand, the operand of the next, whose other operand is read transposed from the tile.
//
// dS and P are rounded to 16 bits for their products (16-bit data). fp16's range would cut them: P is
// scaled by 2^8 (the second kernel's by less where lambda is large), and dP - D by a power of two that keeps
// 2^8 P (dP - D) max(1, |lambda|) below 2^15, from |dP - D| <= 2 V max|v| max|dy|. The maxima are those of what meets in a block,
// so that what other sequences, key heads and hidden keys hold costs no bits: in the first kernel, a row's dy and
// the values up to the last key that the block's rows see; in the second, the key head's values and the rows that see a key
// of the block. (With the call's maxima a sequence of gradients 2^16 below another's kept 7 bits. A power for each key or
// row, lowered as elements pass fp16's range, cost 13 % of the first kernel and 7 of the second.)
//
// 16,384 x 16,384 causal, 8 heads to 2, bf16: 1,030 us (801 TFLOP/s of the first kernel's products; vector units 68 %, matrix cores 39 %
// busy) and 1,725 us (637 TFLOP/s; 42 and 28 %): a wave of 16 keys reads the rows' q and dy from LDS both ways, 32 KB for 32
// matrix instructions, twice what the 32 rows of a wave of the first need; 32 keys do not fit the registers of two waves a
// SIMD (v in LDS instead: 45 of them spilled, the call 3,670 us where it is 2,650), and one wave a SIMD was no faster. 1,344 x 2,688, 4 heads, fp32: 120 and 188 us, matrix cores 71 and 65 % busy.
constexpr int kMostKeys = 64;            // keys of a block of the second kernel, and of a largest |v|
template <class T>
constexpr float kShift = std::is_same_v<T, f16> ? 8.f : 0.f;

__device__ __forceinline__ float range_scale(const DiffArgs& a, float v, float dy, float shift) {
    return __builtin_amdgcn_exp2f(fminf(fmaxf(15.f - shift - ceilf(__builtin_amdgcn_logf(2.f * a.vdim * v * dy)), -100.f), 100.f));
}
// The largest of values [from, to) at p, by `threads` threads of which this is `t`: this thread's share.
__device__ __forceinline__ float largest(const float* p, int from, int to, int t, int threads) {
    float most = 0.f;
#pragma unroll 4
    for (int i = from + t; i < to; i += threads) most = fmaxf(most, p[i]);
    return most;
}

template <class T, int DP, int VP, int NQ, bool ALIGNED>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP > 64 ? 1 : 2) void diff_dq_kernel(DiffArgs a) {
    constexpr int NT = 256, KG = Tile<T, DP>::KEYS, GD = Tile<T, DP>::GROUPS, GV = Tile<T, VP>::GROUPS, ND = DP / 16, ROWS = 64 * NQ;
    constexpr int FIT = 32768 / ((2 * DP + VP) * (int)sizeof(T)), BK = FIT >= 64 ? 64 : FIT >= 32 ? 32 : 16;
    using KL = Loader<T, DP, BK, 2, NT, ALIGNED>;
    using VL = Loader<T, VP, BK, 1, NT, ALIGNED>;
    constexpr int STAGE = KL::BYTES + VL::BYTES;
    __shared__ __align__(128) char lds[2 * STAGE];
    const unsigned lds0 = lds_address(lds);

    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, s = lane % 16;
    const unsigned per = a.tile_div.div(blockIdx.x);
    const int index = (int)(blockIdx.x - per * a.tile_div.d), part = index % a.splits;
    const int tile = a.causal ? a.tiles - 1 - index / a.splits : index / a.splits;   // the longest first
    const int b = (int)a.kv_div.div(per), kvh = (int)(per - b * a.kv_div.d);
    const Mask mask(a, b);
    const int r0 = tile * ROWS, last = min(r0 + ROWS, a.rows) - 1;
    const int most = mask.limit((int)a.group_div.div((unsigned)last)), least = mask.limit((int)a.group_div.div((unsigned)r0));
    const int each = ((most + BK - 1) / BK + a.splits - 1) / a.splits * BK;   // keys of a part
    const int begin = (int)min((long long)part * each, (long long)most), end = (int)min((long long)begin + each, (long long)most);
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

    u32x4 qf[2][NQ][GD], yf[NQ][GV];
    int limit[NQ];
    float base[2][NQ], dot[2][NQ], lam[NQ], unit[NQ];                 // lse in units of log2; D; of the row
    float share[NQ], rest[NQ];           // of lambda's gradient; what rounding left of it
    const float c = a.scale * kLog2e;
    float values = 0.f, loud = 0.f;      // fp16: largest |v| of the keys that the block sees; largest |dy| max(1, |lambda|) of the wave's rows
    if constexpr (std::is_same_v<T, f16>)
        values = lane_max<64>(largest(a.most + (long long)per * ((a.keys + kMostKeys - 1) / kMostKeys), 0, (most + kMostKeys - 1) / kMostKeys, lane, 64));
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const int r = r0 + (wave * NQ + n) * 16 + s;
        const RowAt row(a, kvh, min(r, a.rows - 1));
        limit[n] = mask.limit(row.query);
        lam[n] = a.lam[row.head];
        share[n] = rest[n] = 0.f;
#pragma unroll
        for (int m = 0; m < 2; m++) load_fragments<T, DP>(qf[m][n], row.at(a.q, b, 2, m), a.dim, lane);
        load_fragments<T, VP>(yf[n], limit[n] > 0 ? row.at(a.dy, b, 1, 0) : nullptr, a.vdim, lane);   // a row without keys holds anything
        const char *out = row.at(a.out, b, 1, 0), *second = row.at(a.second, b, 1, 0);
        float d1 = 0.f, d2 = 0.f, most = 0.f;
#pragma unroll
        for (int g = 0; g < GV; g++) {
            constexpr int E = 16 / sizeof(T);
            const int at = g * 4 + lane / 16;
            float y[E], o[E], o2[E];
            unpack<T>(yf[n][g], y);
            unpack<T>(load_chunk<T>(out + at * 16, a.vdim - at * E), o);
            unpack<T>(load_chunk<T>(second + at * 16, a.vdim - at * E), o2);
#pragma unroll
            for (int e = 0; e < E; e++) {
                d1 = fmaf(y[e], fmaf(lam[n], o2[e], o[e]), d1);
                d2 = fmaf(y[e], o2[e], d2);
                most = fmaxf(most, fabsf(y[e]));
            }
        }
        dot[0][n] = column_sum(d1), dot[1][n] = column_sum(d2);
        most = column_max(most);
#pragma unroll
        for (int m = 0; m < 2; m++) {
            const long long at = row.stat(a, b, m);
            base[m][n] = fmaf(a.lse[at], kLog2e, -kShift<T>);
            if (lane < 16 && r < a.rows && part == 0) a.dots[at] = dot[m][n];
        }
        unit[n] = 1.f;
        if constexpr (std::is_same_v<T, f16>) {
            most *= fmaxf(1.f, fabsf(lam[n]));
            unit[n] = range_scale(a, values, most, kShift<T>);
            loud = fmaxf(loud, most);
            dot[0][n] *= unit[n], dot[1][n] *= unit[n];
        }
        // The 16-bit products round low by a hundredth of an ulp in the mean, which dlambda's sum over rows and keys keeps: every
        // other query has -dy and so -dP, and a negative unit.
        if (sizeof(T) == 2 && (row.query + b) % 2) {
            unit[n] = -unit[n];
#pragma unroll
            for (int g = 0; g < GV; g++) yf[n][g] ^= 0x80008000u;
        }
    }
    if constexpr (std::is_same_v<T, f16>) {
        loud = lane_max<64>(loud);
        if (lane == 0 && part == 0) a.loud[((long long)per * a.tiles + tile) * 4 + wave] = loud;
    }
    f32x4 acc[2][NQ][ND] = {};
    constexpr int KS = KG;
    int stage = 0;
    for (int key0 = begin; key0 < end; key0 += BK) {
        kl.settle(lds + stage * STAGE);
        vl.settle(lds + stage * STAGE + KL::BYTES);
        arrived<ALIGNED>();
        if (key0 + BK < end) fetch(key0 + BK, stage ^ 1);
        const char *ks = lds + stage * STAGE, *vs = ks + KL::BYTES;
        const bool whole = key0 + BK <= least && key0 + BK <= end;
        float sum[NQ] = {};
#pragma unroll 1
        for (int k0 = 0; k0 < BK; k0 += KS) {
            f32x4 z[2][NQ][KS / 16], dp[NQ][KS / 16];
#pragma unroll
            for (int t = 0; t < KS / 16; t++) {
#pragma unroll
                for (int n = 0; n < NQ; n++) z[0][n][t] = z[1][n][t] = dp[n][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int m = 0; m < 2; m++)
#pragma unroll
                    for (int g = 0; g < GD; g++) {
                        const u32x4 kf = Tile<T, DP>::plain(ks + m * BK * Tile<T, DP>::BYTES, k0 + t * 16, g, lane);
#pragma unroll
                        for (int n = 0; n < NQ; n++) z[m][n][t] = mma(kf, qf[m][n][g], z[m][n][t], T{});
                    }
#pragma unroll
                for (int g = 0; g < GV; g++) {
                    const u32x4 vf = Tile<T, VP>::plain(vs, k0 + t * 16, g, lane);
#pragma unroll
                    for (int n = 0; n < NQ; n++) dp[n][t] = mma(vf, yf[n][g], dp[n][t], T{});
                }
            }
            if constexpr (DP > 64) __builtin_amdgcn_sched_barrier(0);
            u32x4 ds[2][NQ];
#pragma unroll
            for (int n = 0; n < NQ; n++) {
                const int left = whole ? KS : min(limit[n], end) - (key0 + k0 + lane / 16 * 4);
#pragma unroll
                for (int t = 0; t < KS / 16; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float p1 = __builtin_amdgcn_exp2f(fmaf(z[0][n][t][e], c, -base[0][n])), p2 = __builtin_amdgcn_exp2f(fmaf(z[1][n][t][e], c, -base[1][n]));
                        if (!whole) {
                            p1 = t * 16 + e < left ? p1 : 0.f;
                            p2 = t * 16 + e < left ? p2 : 0.f;
                        }
                        const float d = dp[n][t][e];
                        sum[n] = fmaf(p2, d, sum[n]);
                        z[0][n][t][e] = p1 * fmaf(d, unit[n], -dot[0][n]);
                        z[1][n][t][e] = p2 * -lam[n] * fmaf(d, unit[n], -dot[1][n]);
                    }
#pragma unroll
                for (int m = 0; m < 2; m++) ds[m][n] = chunk_of<T>(z[m][n]);
            }
            if constexpr (DP <= 64) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int i = 0; i < ND; i++) {
                    const u32x4 kf = Tile<T, DP>::columns(ks + m * BK * Tile<T, DP>::BYTES, k0, i, lane);
#pragma unroll
                    for (int n = 0; n < NQ; n++) acc[m][n][i] = mma(kf, ds[m][n], acc[m][n][i], T{});
                }
        }
#pragma unroll
        for (int n = 0; n < NQ; n++) {   // dlambda is a sum of both signs over rows and keys: a tile's share is added without loss
            const float y = sum[n] - rest[n], up = share[n] + y;
            rest[n] = (up - share[n]) - y;
            share[n] = up;
        }
        stage ^= 1;
    }
    // lambda's shares of the tile's rows, added up by head.
    __syncthreads();
    float* shares = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const int at = (wave * NQ + n) * 16 + s;
        const float sum = column_sum(share[n]) * copysignf(1.f, unit[n]);
        if (lane < 16) shares[at] = r0 + at < a.rows ? sum * __builtin_amdgcn_exp2f(-kShift<T>) : 0.f;
    }
    __syncthreads();
    for (int g = tid; g < a.group; g += NT) {
        double sum = 0.0;
        for (int at = (g + a.group - r0 % a.group) % a.group; at < ROWS; at += a.group) sum += (double)shares[at];
        a.tiles_lam[((long long)blockIdx.x) * a.group + g] = sum;
    }
    if (!a.dq.p) return;
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const int r = r0 + (wave * NQ + n) * 16 + s;
        if (r >= a.rows) continue;
        const RowAt row(a, kvh, r);
        const float f = a.scale * __builtin_amdgcn_exp2f(-kShift<T>) / fabsf(unit[n]);
        float* to = a.part ? a.part + (((long long)part * (gridDim.x / a.tile_div.d) + per) * a.rows + r) * (2 * DP) : nullptr;
#pragma unroll
        for (int m = 0; m < 2; m++) {
            char* out = const_cast<char*>(row.at(a.dq, b, 2, m));
#pragma unroll
            for (int i = 0; i < ND; i++) {
                const int at = i * 16 + lane / 16 * 4;
                const f32x4 v = acc[m][n][i] * f;
                if (to) {
                    *reinterpret_cast<f32x4*>(to + m * DP + at) = v;
                } else {
                    const float o[4] = {v[0], v[1], v[2], v[3]};
                    store4<T>(out + at * sizeof(T), a.dim - at, o);
                }
            }
        }
    }
}

// Rows of a tile (of one head), and what the kernel takes of each: both maps' lse and D, and the keys that it sees.
constexpr int kRows = 32;
struct RowStats {
    float base[2][kRows], dot[2][kRows];
    int limit[kRows];
};

template <class T, int DP, int VP, bool ALIGNED>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP > 64 ? 1 : 2) void diff_dkv_kernel(DiffArgs a) {
    constexpr int NT = 256, RG = Tile<T, DP>::KEYS, GD = Tile<T, DP>::GROUPS, GV = Tile<T, VP>::GROUPS, ND = DP / 16, NV = VP / 16, KEYS = kMostKeys;
    using QL = Loader<T, DP, kRows, 2, NT, ALIGNED>;
    using YL = Loader<T, VP, kRows, 1, NT, ALIGNED>;
    constexpr int STAGE = QL::BYTES + YL::BYTES;
    __shared__ __align__(128) char lds[2 * STAGE];
    __shared__ RowStats stats[2];
    const unsigned lds0 = lds_address(lds);

    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, s = lane % 16;
    const unsigned per = a.tile_div.div(blockIdx.x);
    const int index = (int)(blockIdx.x - per * a.tile_div.d), tile = index / a.splits, part = index - tile * a.splits;
    const int b = (int)a.kv_div.div(per), kvh = (int)(per - b * a.kv_div.d);
    const Mask mask(a, b);
    const int key0 = tile * KEYS, key_end = min(key0 + KEYS, a.keys);
    // Of each head that shares the key head, the tiles from the first query that sees a key of this one on; in parts.
    const int first = key0 >= mask.length ? a.queries : !a.causal ? 0 : (int)min((long long)a.queries, max(0LL, key0 - mask.start));
    const int tiles = (a.queries - first + kRows - 1) / kRows;
    const long long all = (long long)tiles * a.group, each = (all + a.splits - 1) / a.splits;
    const long long begin = min(part * each, all), end = min(begin + each, all);
    QL ql;
    YL yl;
    ql.space(a.q.s2, a.q.s1);
    yl.space(a.dy.s2, 0);
    float held[5];                       // a row's stats on their way
    float unit = 1.f, shift = kShift<T>;
    if constexpr (std::is_same_v<T, f16>) {
        float lam = 0.f;
        for (int g = 0; g < a.group; g++) lam = fmaxf(lam, fabsf(a.lam[kvh * a.group + g]));
        // P1 - lambda P2 is dv's operand: from |lambda| 2^6 on both maps give way, so that 2^shift |lambda| stays below 2^14.
        shift -= fminf(fmaxf(ceilf(__builtin_amdgcn_logf(lam)) - 6.f, 0.f), 100.f);
        __shared__ float red[2][4];
        const int waves = (a.rows + a.loud_rows - 1) / a.loud_rows;
        const float v = lane_max<64>(largest(a.most + (long long)per * a.tiles, 0, a.tiles, tid, NT));
        const float y = lane_max<64>(largest(a.loud + (long long)per * a.loud_count, (int)((long long)first * a.group / a.loud_rows), waves, tid, NT));
        if (lane == 0) red[0][wave] = v, red[1][wave] = y;
        __syncthreads();
        unit = range_scale(a, fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3])), fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3])), shift);
    }
    auto fetch = [&](int head, int i0, int stage) {
        const char* q = a.q.p + 2LL * head * a.q.s1 + i0 * a.q.s2 + b * a.q.s3;
        const char* y = a.dy.p + (long long)head * a.dy.s1 + i0 * a.dy.s2 + b * a.dy.s3;
        if (ALIGNED && i0 + kRows <= a.queries && a.dim == DP && a.vdim == VP) {
            ql.fetch_whole(lds0 + stage * STAGE, q, a.q.s2, a.q.s1);
            yl.fetch_whole(lds0 + stage * STAGE + QL::BYTES, y, a.dy.s2, 0);
        } else {
            ql.fetch(lds0 + stage * STAGE, a.dim, [&](int map, int r) { return i0 + r < a.queries ? q + map * a.q.s1 + r * a.q.s2 : nullptr; });
            yl.fetch(lds0 + stage * STAGE + QL::BYTES, a.vdim, [&](int, int r) { return i0 + r < a.queries ? y + r * a.dy.s2 : nullptr; });
        }
        if (tid < kRows) {
            const int i = min(i0 + tid, a.queries - 1);
            const long long at = ((long long)b * a.heads + head) * 2 * a.queries + i;
#pragma unroll
            for (int m = 0; m < 2; m++) {
                held[m] = fmaf(a.lse[at + m * a.queries], kLog2e, -shift);
                held[2 + m] = a.dots[at + m * a.queries] * unit;
            }
            held[4] = __int_as_float(i0 + tid < a.queries ? mask.limit(i) : 0);
        }
    };
    auto settle = [&](int stage) {
        ql.settle(lds + stage * STAGE);
        yl.settle(lds + stage * STAGE + QL::BYTES);
        if (tid < kRows) {
            RowStats& st = stats[stage];
            st.base[0][tid] = held[0], st.base[1][tid] = held[1], st.dot[0][tid] = held[2], st.dot[1][tid] = held[3];
            st.limit[tid] = __float_as_int(held[4]);
        }
        arrived<ALIGNED>();
    };
    // The next tile: of the same head, or the next head's first.
    int head = kvh * a.group + (tiles ? (int)(begin / tiles) : 0), i0 = first + (tiles ? (int)(begin % tiles) : 0) * kRows;
    auto step = [&](int& head, int& i0) {
        i0 += kRows;
        if (i0 >= a.queries) head++, i0 = first;
    };
    if (begin < end) fetch(head, i0, 0);

    u32x4 kf[2][GD], vf[GV];
    const int key = key0 + wave * 16 + s;
    const bool there = key < mask.length;
#pragma unroll
    for (int m = 0; m < 2; m++) load_fragments<T, DP>(kf[m], there ? a.k.p + (2LL * kvh + m) * a.k.s1 + key * a.k.s2 + b * a.k.s3 : nullptr, a.dim, lane);
    load_fragments<T, VP>(vf, there ? a.v.p + (long long)kvh * a.v.s1 + key * a.v.s2 + b * a.v.s3 : nullptr, a.vdim, lane);
    f32x4 dk[2][ND] = {}, dv[NV] = {};
    const float c = a.scale * kLog2e;
    int stage = 0;
    for (long long t = begin; t < end; t++) {
        settle(stage);
        const float lam = -a.lam[head];
        const bool whole = i0 + kRows <= a.queries && mask.limit(i0) >= key_end && key0 + KEYS <= a.keys;   // limits never fall
        step(head, i0);
        if (t + 1 < end) fetch(head, i0, stage ^ 1);
        const char *qs = lds + stage * STAGE, *ys = qs + QL::BYTES;
        const RowStats& st = stats[stage];
#pragma unroll 1
        for (int k0 = 0; k0 < kRows; k0 += RG) {
            f32x4 z[2][RG / 16], dp[RG / 16];
#pragma unroll
            for (int t = 0; t < RG / 16; t++) {
                z[0][t] = z[1][t] = dp[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int m = 0; m < 2; m++)
#pragma unroll
                    for (int g = 0; g < GD; g++) {
                        const u32x4 qf = Tile<T, DP>::plain(qs + m * kRows * Tile<T, DP>::BYTES, k0 + t * 16, g, lane);
                        z[m][t] = mma(qf, kf[m][g], z[m][t], T{});
                    }
#pragma unroll
                for (int g = 0; g < GV; g++) {
                    const u32x4 yf = Tile<T, VP>::plain(ys, k0 + t * 16, g, lane);
                    dp[t] = mma(yf, vf[g], dp[t], T{});
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            f32x4 pm[RG / 16];
#pragma unroll
            for (int t = 0; t < RG / 16; t++) {
                const int at = k0 + t * 16 + lane / 16 * 4;
                const f32x4 base1 = *reinterpret_cast<const f32x4*>(&st.base[0][at]), base2 = *reinterpret_cast<const f32x4*>(&st.base[1][at]);
                const f32x4 dot1 = *reinterpret_cast<const f32x4*>(&st.dot[0][at]), dot2 = *reinterpret_cast<const f32x4*>(&st.dot[1][at]);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float p1 = __builtin_amdgcn_exp2f(fmaf(z[0][t][e], c, -base1[e])), p2 = lam * __builtin_amdgcn_exp2f(fmaf(z[1][t][e], c, -base2[e]));
                    if (!whole) {
                        const bool in = key < st.limit[at + e];
                        p1 = in ? p1 : 0.f;
                        p2 = in ? p2 : 0.f;
                    }
                    pm[t][e] = p1 + p2;
                    z[0][t][e] = p1 * fmaf(dp[t][e], unit, -dot1[e]);
                    z[1][t][e] = p2 * fmaf(dp[t][e], unit, -dot2[e]);
                }
            }
            const u32x4 mix = chunk_of<T>(pm), ds[2] = {chunk_of<T>(z[0]), chunk_of<T>(z[1])};
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const u32x4 yf = Tile<T, VP>::columns(ys, k0, i, lane);
                dv[i] = mma(yf, mix, dv[i], T{});
            }
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int i = 0; i < ND; i++) {
                    const u32x4 qf = Tile<T, DP>::columns(qs + m * kRows * Tile<T, DP>::BYTES, k0, i, lane);
                    dk[m][i] = mma(qf, ds[m], dk[m][i], T{});
                }
        }
        stage ^= 1;
    }
    const float fv = __builtin_amdgcn_exp2f(-shift), fk = a.scale * fv / unit;
    if (key >= a.keys) return;
    float* to = a.part ? a.part + (((long long)part * (gridDim.x / a.tile_div.d) + per) * a.keys + key) * (2 * DP + VP) : nullptr;
#pragma unroll
    for (int m = 0; m < 3; m++) {        // dk of both maps, dv
        const Strided& d = m < 2 ? a.dk : a.dv;
        char* out = const_cast<char*>(d.p) + (m < 2 ? 2LL * kvh + m : (long long)kvh) * d.s1 + key * d.s2 + b * d.s3;
        const int width = m < 2 ? a.dim : a.vdim;
        const float f = m < 2 ? fk : fv;
#pragma unroll
        for (int i = 0; i < (m < 2 ? ND : NV); i++) {
            const int at = i * 16 + lane / 16 * 4;
            const f32x4 v = (m < 2 ? dk[m < 2 ? m : 0][m < 2 ? i : 0] : dv[i]) * f;
            if (to) {
                *reinterpret_cast<f32x4*>(to + m * DP + at) = v;
            } else if (d.p) {
                const float o[4] = {v[0], v[1], v[2], v[3]};
                store4<T>(out + at * sizeof(T), width - at, o);
            }
        }
    }
}

// Sums of the parts, in order: of a row's dq, or (KEYS) of a key's dk and dv; four elements a thread.
template <class T, bool KEYS>
__global__ __launch_bounds__(256) void diff_fold_kernel(DiffArgs a, int dp, int vp, long long all) {
    const int width = KEYS ? 2 * dp + vp : 2 * dp, quads = width / 4, each = KEYS ? a.keys : a.rows;
    const long long e = blockIdx.x * 256LL + threadIdx.x, index = e / quads;   // of (sequence, key head), row or key
    if (index >= all) return;
    const int at = (int)(e - index * quads) * 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < a.splits; i++) v += *reinterpret_cast<const f32x4*>(a.part + (i * all + index) * width + at);
    const unsigned per = (unsigned)(index / each);
    const int at_row = (int)(index - (long long)per * each), b = (int)a.kv_div.div(per), kvh = (int)(per - b * a.kv_div.d);
    const int m = at < dp ? 0 : at < 2 * dp ? 1 : 2, col = at - m * dp;
    const float o[4] = {v[0], v[1], v[2], v[3]};
    if constexpr (KEYS) {
        const Strided& d = m < 2 ? a.dk : a.dv;
        char* out = const_cast<char*>(d.p) + (m < 2 ? 2LL * kvh + m : (long long)kvh) * d.s1 + at_row * d.s2 + b * d.s3;
        store4<T>(out + col * (long long)sizeof(T), (m < 2 ? a.dim : a.vdim) - col, o);
    } else {
        store4<T>(const_cast<char*>(RowAt(a, kvh, at_row).at(a.dq, b, 2, m)) + col * (long long)sizeof(T), a.dim - col, o);
    }
}

// lambda's gradient: less the sum of its head's shares, which lie [sequence][key head][tile and part][group].
__global__ __launch_bounds__(256) void diff_lambda_kernel(const double* shares, long long batch, int kv_heads, int group, int tiles, float* dlam) {
    __shared__ double red[4];
    const int kvh = blockIdx.x / group, g = blockIdx.x % group;
    double s = 0.0;
    const long long n = batch * tiles;
#pragma unroll 4
    for (long long i = threadIdx.x; i < n; i += 256) {
        const long long b = i / tiles;
        s += shares[((b * kv_heads + kvh) * tiles + (i - b * tiles)) * group + g];
    }
    s = lane_sum<64>(s);
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = s;
    __syncthreads();
    if (threadIdx.x == 0) dlam[blockIdx.x] = (float)-((red[0] + red[1]) + (red[2] + red[3]));
}

// fp16: the largest |v| of each kMostKeys keys of a (sequence, key head), a block each; keys past the length are not there.
__global__ __launch_bounds__(256) void diff_most_kernel(DiffArgs a, int tiles, float* mosts) {
    const unsigned per = blockIdx.x / tiles;
    const int key0 = (int)(blockIdx.x - per * tiles) * kMostKeys, b = (int)a.kv_div.div(per), kvh = (int)(per - b * a.kv_div.d);
    const Mask mask(a, b);
    const int chunks = (a.vdim + 7) / 8, rows = min(kMostKeys, mask.length - key0);
    float most = 0.f;
#pragma unroll 4
    for (int e = threadIdx.x; e < rows * chunks; e += 256) {
        const int r = e / chunks, c = e - r * chunks;
        float f[8];
        unpack<f16>(load_chunk<f16>(a.v.p + (long long)kvh * a.v.s1 + (key0 + r) * a.v.s2 + b * a.v.s3 + c * 16, a.vdim - c * 8), f);
#pragma unroll
        for (int i = 0; i < 8; i++) most = fmaxf(most, fabsf(f[i]));
    }
    __shared__ float red[4];
    most = lane_max<64>(most);
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = most;
    __syncthreads();
    if (threadIdx.x == 0) mosts[blockIdx.x] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// --------------------------------------------------------------------------------- host
constexpr int kCus = 256;
size_t pad256(size_t n) { return (n + 255) / 256 * 256; }
struct BackPlan {
    int nq, dp, vp, q_splits, k_splits;
    long long q_tiles, k_tiles;
    size_t dots, tiles_lam, most, loud, part, total;
};
BackPlan back_plan(const DiffShape& s, int size, bool causal) {
    BackPlan p{};
    const long long group = s.H / s.Hk, rows = s.M * group, pairs = s.B * s.Hk;
    const bool small = s.D <= 64 && s.V <= 128 && size == 2;
    with_dims(s.D, s.V, [&](auto d, auto v) { p.dp = d(), p.vp = v(); });
    p.nq = small && rows > 64 ? 2 : 1;
    p.q_tiles = (rows + 64 * p.nq - 1) / (64 * p.nq);
    p.k_tiles = (s.N + kMostKeys - 1) / kMostKeys;
    // Parts of the keys or rows: as many as give two blocks a CU, or eight where causality makes tiles differ in length,
    // of 256 keys or rows at least.
    const long long want = (causal ? 8LL : 4LL) * kCus;
    p.q_splits = (int)std::max(1LL, std::min({2LL * kCus / std::max(1LL, p.q_tiles * pairs), s.N / 256, 64LL}));
    p.k_splits = (int)std::max(1LL, std::min({want / std::max(1LL, p.k_tiles * pairs), rows / 256, 64LL}));
    auto take = [&](size_t bytes) {
        const size_t at = p.total;
        p.total += pad256(bytes);
        return at;
    };
    p.dots = take((size_t)s.B * s.H * 2 * s.M * sizeof(float));
    p.tiles_lam = take((size_t)((rows + 63) / 64) * p.q_splits * s.B * s.H * sizeof(double));   // of the smallest tiles
    p.most = take((size_t)p.k_tiles * pairs * sizeof(float));
    p.loud = take((size_t)((rows + 63) / 64) * 4 * pairs * sizeof(float));                      // of the smallest tiles
    const size_t q_part = p.q_splits > 1 ? (size_t)p.q_splits * pairs * rows * 2 * p.dp : 0;
    const size_t k_part = p.k_splits > 1 ? (size_t)p.k_splits * pairs * s.N * (2 * p.dp + p.vp) : 0;
    p.part = take(std::max(q_part, k_part) * sizeof(float));         // one after the other
    return p;
}

template <class T, int DP, int VP>
void launch_dq(const DiffArgs& a, const BackPlan& p, bool aligned, unsigned blocks, hipStream_t stream) {
    if (!aligned) hipLaunchKernelGGL((diff_dq_kernel<T, DP, VP, 1, false>), dim3(blocks), dim3(256), 0, stream, a);
    else if (p.nq == 1) hipLaunchKernelGGL((diff_dq_kernel<T, DP, VP, 1, true>), dim3(blocks), dim3(256), 0, stream, a);
    else if constexpr (sizeof(T) == 2 && DP <= 64) hipLaunchKernelGGL((diff_dq_kernel<T, DP, VP, 2, true>), dim3(blocks), dim3(256), 0, stream, a);
    launch_check("diff_dq_kernel");
}
template <class T, int DP, int VP>
void launch_dkv(const DiffArgs& a, bool aligned, unsigned blocks, hipStream_t stream) {
    if (aligned) hipLaunchKernelGGL((diff_dkv_kernel<T, DP, VP, true>), dim3(blocks), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((diff_dkv_kernel<T, DP, VP, false>), dim3(blocks), dim3(256), 0, stream, a);
    launch_check("diff_dkv_kernel");
}

void check_like(const stx_tensor* t, const stx_tensor* like, int size, const char* what) {
    check_out_rows(t, like->ne[0], like->ne[1], like->ne[2], like->ne[3], size, what);
    check_nested(t, size, what);
}

}  // namespace
}  // namespace stx

using namespace stx;

extern "C" {

STX_API size_t stx_diff_attention_back_workspace_size(const stx_tensor* q, const stx_tensor* k, const stx_tensor* v, stx_type type) {
    size_t bytes = 0;
    (void)guard([&] {
        const char* op = "diff_attention_back_workspace_size";
        const int size = type_size(type);
        for (const stx_tensor* t : {q, k, v}) {
            STX_REQUIRE(t != nullptr, "%s: a tensor is NULL", op);
            for (int i = 0; i < 4; i++) STX_REQUIRE(t->ne[i] >= 0, "%s: negative ne[%d]", op, i);
        }
        const DiffShape s = diff_shape(q, k, v, op);
        if (s.B > 0 && s.H > 0) bytes = std::max(back_plan(s, size, false).total, back_plan(s, size, true).total);
    });
    return bytes;
}

STX_API stx_status stx_diff_attention_back(const stx_tensor* dy, const stx_tensor* q, const stx_tensor* k, const stx_tensor* v,
                                           stx_type type, const float* lambda, float scale, int causal, const int32_t* lengths,
                                           const int32_t* starts, const stx_tensor* out, const stx_tensor* second, const float* lse,
                                           const stx_tensor* dq, const stx_tensor* dk, const stx_tensor* dv, float* dlambda,
                                           void* workspace, size_t workspace_bytes, stx_stream stream) {
    return guard([&] {
        const char* op = "diff_attention_back";
        const int size = type_size(type);
        check_typed(q, size, "diff_attention_back: q");
        check_typed(k, size, "diff_attention_back: k");
        check_typed(v, size, "diff_attention_back: v");
        const DiffShape s = diff_shape(q, k, v, op);
        check_out_rows(dy, s.V, s.H, s.M, s.B, size, "diff_attention_back: dy");
        check_out_rows(out, s.V, s.H, s.M, s.B, size, "diff_attention_back: out");
        check_out_rows(second, s.V, s.H, s.M, s.B, size, "diff_attention_back: second");
        if (dq) check_like(dq, q, size, "diff_attention_back: dq");
        STX_REQUIRE((dk == nullptr) == (dv == nullptr), "%s: dk and dv go together", op);
        if (dk) {
            check_like(dk, k, size, "diff_attention_back: dk");
            check_like(dv, v, size, "diff_attention_back: dv");
        }
        check_scale(scale, op);
        if (s.B == 0 || s.H == 0) {
            if (dlambda && s.H > 0) {
                hipLaunchKernelGGL(diff_lambda_kernel, dim3(s.H), dim3(256), 0, as_stream(stream), nullptr, 0, 1, s.H, 1, dlambda);
                launch_check("diff_lambda_kernel");
            }
            return;
        }
        BackPlan p = back_plan(s, size, causal != 0);
        check_workspace(workspace, workspace_bytes, p.total, op);
        const size_t per = (size_t)s.B * sizeof(int32_t), kept = (size_t)s.B * s.H * 2 * s.M * sizeof(float), heads = s.H * sizeof(float);
        check_apart(op, {{"dq", dq, size}, {"dk", dk, size}, {"dv", dv, size}, {"dlambda", dlambda, heads}, {"the workspace", workspace, p.total}},
                    {{"dy", dy, size}, {"q", q, size}, {"k", k, size}, {"v", v, size}, {"lambda", lambda, heads}, {"lengths", lengths, per},
                     {"starts", starts, per}, {"out", out, size}, {"second", second, size}, {"lse", lse, kept}});
        STX_REQUIRE(lambda != nullptr && (s.M == 0 || lse != nullptr), "%s: lambda or lse is NULL", op);
        if (!dq && !dk && !dlambda) return;
        DiffArgs a = diff_args(s, q, k, v, lambda, scale, causal, lengths, starts);
        a.out = strided(out), a.second = strided(second), a.dy = strided(dy);
        a.dq = strided(dq), a.dk = strided(dk), a.dv = strided(dv);
        a.lse = const_cast<float*>(lse);
        char* ws = static_cast<char*>(workspace);
        a.dots = reinterpret_cast<float*>(ws + p.dots);
        a.tiles_lam = reinterpret_cast<double*>(ws + p.tiles_lam);
        float* most = reinterpret_cast<float*>(ws + p.most);
        a.most = most;
        a.loud = reinterpret_cast<float*>(ws + p.loud);
        const hipStream_t st = as_stream(stream);
        const long long pairs = s.B * s.Hk;
        const bool keys_aligned = rows_in_chunks(k, size) && rows_in_chunks(v, size), rows_aligned = rows_in_chunks(q, size) && rows_in_chunks(dy, size);
        if (!keys_aligned && p.nq > 1) p.nq = 1, p.q_tiles = (a.rows + 63) / 64;
        a.loud_rows = 16 * p.nq, a.loud_count = 4 * (int)p.q_tiles;
        STX_REQUIRE(p.q_tiles * p.q_splits * pairs < (1LL << 22) && p.k_tiles * p.k_splits * pairs < (1LL << 22), "%s: too many tiles", op);
        auto fold_blocks = [&](long long quads) { return dim3((unsigned)((quads + 255) / 256)); };   // split calls have few tiles
        with_type(type, [&](auto t) {
            using T = decltype(t);
            with_dims(s.D, s.V, [&](auto d, auto vd) {
                if constexpr (std::is_same_v<T, f16>) {
                    if (s.N > 0) {
                        hipLaunchKernelGGL(diff_most_kernel, dim3((unsigned)(p.k_tiles * pairs)), dim3(256), 0, st, a, (int)p.k_tiles, most);
                        launch_check("diff_most_kernel");
                    }
                }
                float* part = reinterpret_cast<float*>(ws + p.part);
                if (s.M > 0) {
                    a.tiles = (int)p.q_tiles, a.splits = p.q_splits;
                    a.tile_div = FastDiv((unsigned)(p.q_tiles * p.q_splits));
                    a.part = p.q_splits > 1 ? part : nullptr;
                    launch_dq<T, d(), vd()>(a, p, keys_aligned, (unsigned)(p.q_tiles * p.q_splits * pairs), st);
                    if (dq && a.part) {
                        hipLaunchKernelGGL((diff_fold_kernel<T, false>), fold_blocks(pairs * a.rows * (p.dp / 2)), dim3(256), 0, st, a, p.dp, p.vp, pairs * a.rows);
                        launch_check("diff_fold_kernel");
                    }
                }
                if (dk && s.N > 0) {
                    a.tiles = (int)p.k_tiles, a.splits = p.k_splits;
                    a.tile_div = FastDiv((unsigned)(p.k_tiles * p.k_splits));
                    a.part = p.k_splits > 1 ? part : nullptr;
                    launch_dkv<T, d(), vd()>(a, rows_aligned, (unsigned)(p.k_tiles * p.k_splits * pairs), st);
                    if (a.part) {
                        hipLaunchKernelGGL((diff_fold_kernel<T, true>), fold_blocks(pairs * s.N * ((2 * p.dp + p.vp) / 4)), dim3(256), 0, st, a, p.dp, p.vp, pairs * s.N);
                        launch_check("diff_fold_kernel");
                    }
                }
            });
        });
        if (dlambda) {
            hipLaunchKernelGGL(diff_lambda_kernel, dim3(s.H), dim3(256), 0, st, a.tiles_lam, s.M > 0 ? s.B : 0, s.Hk, a.group, (int)std::max(1LL, p.q_tiles * p.q_splits), dlambda);
            launch_check("diff_lambda_kernel");
        }
    });
}

}  // extern "C"

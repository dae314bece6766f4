// gated_ff.hip — the gated feed-forward block act(x Wg^T + bg) * (x Wv^T + bv), forward and
// backward (stx_gated_ff, stx_gated_ff_back).
#include <algorithm>

#include "typed.hpp"

namespace stx {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// acc += A B^T over one 16-byte chunk a lane: A and B have 16 rows, lane l holds the chunk of row
// l % 16 at reduction position l / 16. acc[r] is element (A row (l / 16) * 4 + r, B row l % 16).
// The order of the reduction positions is free as long as A's and B's agree, so the fp32
// instruction (one value a lane) takes element e of every lane's chunk in step e.
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 acc, float) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; e++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], acc, 0, 0, 0);
    return acc;
}
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 acc, f16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 acc, bf16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
}

// The products of the block, all of the form out[m][j] = sum_r P[j][r] Q[m][r] with r contiguous:
//   FORWARD  P = rows of Wg and Wv, 16 by 16 in turn (a lane then holds gate and value of the same
//            outputs), Q = x; the epilogue forms act(g) v.
//   GRAD     the same products again; the epilogue takes dh and writes dg = dh v act'(g) and
//            dv = dh act(g), and per wave the sums of its columns for the biases' gradients.
//   DX       P = the transposed weights, Q = dg, then dv: both reductions into one accumulator.
//   DW       P = x^T, Q = dg^T or dv^T (grid z), a part of the tokens (split), fp32 partial sums.
enum Mode { FORWARD, GRAD, DX, DW };

struct FfArgs {
    const char* p[2];
    const char* q[2];
    long long ps[2], qs[2];              // row strides in bytes
    int J, M;                            // rows of one P, rows of Q
    long long R;                         // reduction length
    long long split;                     // DW: reduction length of a part
    int jtiles, mtiles;
    const float* b[2];
    int act;
    const char* dh;
    long long dhs;
    char* out[2];
    long long os;                        // output row stride in bytes
    int jpad;                            // GRAD: columns written, zeros from J on
    float* db;                           // GRAD: [wave rows][2][J]
};

__device__ const u32x4 zero_chunk = {0, 0, 0, 0};

// 16 bytes at p of which the first `left` elements exist; the rest are zeros.
template <class T>
__device__ __forceinline__ u32x4 load_chunk(const char* p, long long left) {
    constexpr int E = 16 / sizeof(T);
    u32x4 v = {0, 0, 0, 0};
    if (left >= E) {
        __builtin_memcpy(&v, p, 16);
    } else if (left > 0) {
        T e[E];
#pragma unroll
        for (int i = 0; i < E; i++) e[i] = i < left ? reinterpret_cast<const T*>(p)[i] : T(0.f);
        __builtin_memcpy(&v, e, 16);
    }
    return v;
}

__device__ __forceinline__ void load_to_lds(const void* src, void* lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                     (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

template <class T>
__device__ __forceinline__ void load4(const char* p, int left, float (&f)[4]) {
    if (left >= 4) {
        T v[4];
        __builtin_memcpy(v, p, sizeof v);
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = to_f32(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = i < left ? to_f32(reinterpret_cast<const T*>(p)[i]) : 0.f;
    }
}
template <class T>
__device__ __forceinline__ void store4(char* p, int left, const float (&f)[4]) {
    if (left >= 4) {
        T v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = from_f32<T>(f[i]);
        __builtin_memcpy(p, v, sizeof v);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < left) reinterpret_cast<T*>(p)[i] = from_f32<T>(f[i]);
    }
}

// Sum over the 16 lanes of a row, in every lane.
__device__ __forceinline__ float row_sum(float v) {
    v += dpp_f32<0xB1>(v);
    v += dpp_f32<0x4E>(v);
    v += dpp_f32<0x141>(v);
    v += dpp_f32<0x140>(v);
    return v;
}

// Tiles of TJ x TM outputs, WAVES_J x WAVES_M waves. A stage of LDS holds 128 bytes of every row
// (8 chunks); chunk c of row r lies at position c ^ (r % 8), so the 16 rows that a fragment reads
// spread over all banks. Two stages: the next is filled (ALIGNED: straight from memory to LDS;
// otherwise through registers, any alignment and length) while the waves multiply the other.
template <class T, int MODE, int TJ, int TM, int WAVES_J, int WAVES_M, bool ALIGNED>
__global__ __launch_bounds__(64 * WAVES_J* WAVES_M) void ff_kernel(FfArgs a) {
    constexpr int NT = 64 * WAVES_J * WAVES_M, E = 16 / sizeof(T);
    constexpr int NJ = TJ / WAVES_J / 16, NM = TM / WAVES_M / 16;   // 16 x 16 tiles of a wave
    constexpr int PL = TJ * 8 / NT, QL = TM * 8 / NT;                // chunks a thread fetches for a stage
    constexpr bool GATED = MODE == FORWARD || MODE == GRAD;
    __shared__ __align__(128) char lds[2][(TJ + TM) * 128];

    // Tiles in groups of 8 along m, m fastest: the tiles that an XCD works on share rows of both.
    int id = xcd_block();
    if (id >= a.jtiles * a.mtiles) return;
    const int per = 8 * a.jtiles, group = id / per, in = id - group * per;
    const int gm = min(8, a.mtiles - group * 8);
    const int m0 = (group * 8 + in % gm) * TM, jt = in / gm;
    const int j0 = GATED ? jt * (TJ / 2) : jt * TJ;

    long long r0 = 0, r1 = a.R;
    int which = 0;
    if constexpr (MODE == DW) {
        which = blockIdx.y;
        r0 = blockIdx.z * a.split;
        r1 = min(r0 + a.split, a.R);
    }
    constexpr int SEGMENTS = MODE == DX ? 2 : 1;

    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const int wj = wave / WAVES_M, wm = wave % WAVES_M;
    const char *pp[PL], *qq[QL];
    const int chunk = (tid % 8) ^ (tid / 8 % 8);                     // rows of a thread differ by multiples of NT / 8
    auto aim = [&](int seg) {
#pragma unroll
        for (int i = 0; i < PL; i++) {
            const int row = (i * NT + tid) / 8;
            const int s = GATED ? row / 16 % 2 : seg;
            const int j = min(GATED ? j0 + row / 32 * 16 + row % 16 : j0 + row, a.J - 1);
            pp[i] = a.p[s] + j * a.ps[s] + (r0 + chunk * E) * (long long)sizeof(T);
        }
#pragma unroll
        for (int i = 0; i < QL; i++) {
            const int s = MODE == DW ? which : seg;
            qq[i] = a.q[s] + min(m0 + (i * NT + tid) / 8, a.M - 1) * a.qs[s] + (r0 + chunk * E) * (long long)sizeof(T);
        }
    };
    const int steps = (int)((r1 - r0 + 8 * E - 1) / (8 * E));
    u32x4 hold[ALIGNED ? 1 : PL + QL];
    auto fetch = [&](int step, int stage) {
        const long long at = (long long)step * 128, left = r1 - r0 - (long long)step * 8 * E - chunk * E;
#pragma unroll
        for (int i = 0; i < PL + QL; i++) {
            const char* src = (i < PL ? pp[i < PL ? i : 0] : qq[i < PL ? 0 : i - PL]) + at;
            if constexpr (ALIGNED) load_to_lds(left > 0 ? (const void*)src : (const void*)&zero_chunk, &lds[stage][(i * NT + wave * 64) * 16]);
            else hold[i] = load_chunk<T>(src, left);
        }
    };
    auto settle = [&](int stage) {
        if constexpr (!ALIGNED) {
#pragma unroll
            for (int i = 0; i < PL + QL; i++) *reinterpret_cast<u32x4*>(&lds[stage][(i * NT + tid) * 16]) = hold[i];
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        __syncthreads();
    };

    f32x4 acc[NJ][NM];
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
        for (int m = 0; m < NM; m++) acc[j][m] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int frag = (lane % 16) * 128 + ((lane / 16) ^ (lane % 8)) * 16;
    const int pbase = wj * NJ * 16 * 128, qbase = (TJ + wm * NM * 16) * 128;
#pragma unroll 1
    for (int seg = 0; seg < SEGMENTS; seg++) {
        aim(seg);
        fetch(0, 0);
        settle(0);
#pragma unroll 1
        for (int s = 0; s < steps; s++) {
            const int stage = s & 1;
            if (s + 1 < steps) fetch(s + 1, stage ^ 1);
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                u32x4 fp[NJ], fq[NM];
#pragma unroll
                for (int j = 0; j < NJ; j++) fp[j] = *reinterpret_cast<const u32x4*>(&lds[stage][pbase + j * 2048 + (frag ^ (kk * 64))]);
#pragma unroll
                for (int m = 0; m < NM; m++) fq[m] = *reinterpret_cast<const u32x4*>(&lds[stage][qbase + m * 2048 + (frag ^ (kk * 64))]);
#pragma unroll
                for (int j = 0; j < NJ; j++)
#pragma unroll
                    for (int m = 0; m < NM; m++) acc[j][m] = mma(fp[j], fq[m], acc[j][m], T{});
            }
            if (s + 1 < steps) settle(stage ^ 1);
        }
        if (seg + 1 < SEGMENTS) __syncthreads();
    }

    const int mrow = m0 + wm * NM * 16 + lane % 16;
    if constexpr (GATED) with_act(a.act, [&](auto act) {
#pragma unroll
        for (int j = 0; j < NJ; j += 2) {
            const int n = j0 + (wj * NJ + j) * 8 + lane / 16 * 4, left = a.J - n;
            float bg[4], bv[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                bg[r] = a.b[0] && r < left ? a.b[0][n + r] : 0.f;
                bv[r] = a.b[1] && r < left ? a.b[1][n + r] : 0.f;
            }
            float sg[4] = {}, sv[4] = {};
#pragma unroll
            for (int m = 0; m < NM; m++) {
                const int row = mrow + m * 16;
                if constexpr (MODE == FORWARD) {
                    float h[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) h[r] = act_f32<act()>(acc[j][m][r] + bg[r]) * (acc[j + 1][m][r] + bv[r]);
                    if (row < a.M) store4<T>(a.out[0] + row * a.os + n * (long long)sizeof(T), left, h);
                } else {
                    float dh[4], dg[4], dv[4];
                    load4<T>(a.dh + row * a.dhs + n * (long long)sizeof(T), row < a.M ? left : 0, dh);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        float d;
                        const float g = act_f32<act()>(acc[j][m][r] + bg[r], d), v = acc[j + 1][m][r] + bv[r];
                        const bool in = row < a.M && r < left;
                        dg[r] = in ? dh[r] * v * d : 0.f;
                        dv[r] = in ? dh[r] * g : 0.f;
                        sg[r] += dg[r];
                        sv[r] += dv[r];
                    }
                    if (row < a.M && a.out[0]) {
                        store4<T>(a.out[0] + row * a.os + n * (long long)sizeof(T), a.jpad - n, dg);
                        store4<T>(a.out[1] + row * a.os + n * (long long)sizeof(T), a.jpad - n, dv);
                    }
                }
            }
            if constexpr (MODE == GRAD) {
                if (a.db) {
                    float* part = a.db + ((long long)(m0 / TM) * WAVES_M + wm) * 2 * a.J;
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float g = row_sum(sg[r]), v = row_sum(sv[r]);
                        if (lane % 16 == 0 && r < left) {
                            part[n + r] = g;
                            part[a.J + n + r] = v;
                        }
                    }
                }
            }
        }
    });
    else {
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int c = j0 + (wj * NJ + j) * 16 + lane / 16 * 4;
#pragma unroll
            for (int m = 0; m < NM; m++) {
                const int row = mrow + m * 16;
                const float f[4] = {acc[j][m][0], acc[j][m][1], acc[j][m][2], acc[j][m][3]};
                if (row >= a.M) continue;
                if constexpr (MODE == DX) store4<T>(a.out[0] + row * a.os + c * (long long)sizeof(T), a.J - c, f);
                else store4<float>(a.out[0] + (((long long)blockIdx.z * 2 + which) * a.M + row) * a.os + c * 4LL, a.J - c, f);
            }
        }
    }
}

// Few tokens (at most 64): the weights' bytes are the floor, each read by one block, straight into
// the matrix instructions' registers. A block has 16 outputs; its 8 waves take the 64-byte
// steps of the rows in turn and add their accumulators in LDS.
template <class T, int NM>
__global__ __launch_bounds__(512) void ff_few_kernel(FfArgs a) {
    constexpr int E = 16 / sizeof(T), WAVES = 8;
    __shared__ f32x4 part[WAVES][2 * NM][64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int j0 = blockIdx.x * 16, j = min(j0 + lane % 16, a.J - 1);
    const char* p[2] = {a.p[0] + j * a.ps[0], a.p[1] + j * a.ps[1]};
    const char* q[NM];
#pragma unroll
    for (int m = 0; m < NM; m++) q[m] = a.q[0] + min(m * 16 + lane % 16, a.M - 1) * a.qs[0];
    f32x4 acc[2][NM] = {};
    const int steps = (int)((a.R + 4 * E - 1) / (4 * E));
    auto take = [&](int s, auto whole) {
        const long long r = (long long)s * 4 * E + lane / 16 * E, at = r * (long long)sizeof(T), left = whole() ? E : a.R - r;
        const u32x4 g = load_chunk<T>(p[0] + at, left), v = load_chunk<T>(p[1] + at, left);
#pragma unroll
        for (int m = 0; m < NM; m++) {
            const u32x4 x = load_chunk<T>(q[m] + at, left);
            acc[0][m] = mma(g, x, acc[0][m], T{});
            acc[1][m] = mma(v, x, acc[1][m], T{});
        }
    };
    const int full = (int)(a.R / (4 * E));
    int s = wave;
    for (; s + 3 * WAVES < full; s += 4 * WAVES) {
#pragma unroll
        for (int u = 0; u < 4; u++) take(s + u * WAVES, std::true_type{});
    }
    for (; s < steps; s += WAVES) take(s, std::false_type{});
#pragma unroll
    for (int m = 0; m < NM; m++) {
        part[wave][2 * m][lane] = acc[0][m];
        part[wave][2 * m + 1][lane] = acc[1][m];
    }
    __syncthreads();
    const int m = wave, n = j0 + lane / 16 * 4, row = m * 16 + lane % 16;
    if (m >= NM || row >= a.M) return;
    f32x4 g = part[0][2 * m][lane], v = part[0][2 * m + 1][lane];
#pragma unroll
    for (int w = 1; w < WAVES; w++) {
        g += part[w][2 * m][lane];
        v += part[w][2 * m + 1][lane];
    }
    float h[4];
    with_act(a.act, [&](auto act) {
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const bool in = n + r < a.J;
        h[r] = act_f32<act()>(g[r] + (a.b[0] && in ? a.b[0][n + r] : 0.f)) * (v[r] + (a.b[1] && in ? a.b[1][n + r] : 0.f));
    }
    });
    store4<T>(a.out[0] + row * a.os + n * (long long)sizeof(T), a.J - n, h);
}

// src [rows][cols] -> dst [cols][ld], zeros from `rows` to the next multiple of 64.
template <class T>
__global__ __launch_bounds__(256) void ff_transpose_kernel(const char* src, long long ss, int rows, int cols, T* dst, long long ld) {
    __shared__ T tile[64][66];
    const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64, x = threadIdx.x % 64, y = threadIdx.x / 64;
    for (int i = y; i < 64; i += 4)
        tile[i][x] = r0 + i < rows && c0 + x < cols ? reinterpret_cast<const T*>(src + (r0 + i) * ss)[c0 + x] : T(0.f);
    __syncthreads();
    for (int i = y; i < 64; i += 4)
        if (c0 + i < cols) dst[(long long)(c0 + i) * ld + r0 + x] = tile[x][i];
}

// Weight gradients: the parts of the tokens added in order.
template <class T>
__global__ __launch_bounds__(256) void ff_dw_fold_kernel(const float* part, int splits, int N, int K, char* dg, char* dv, long long sg, long long sv) {
    const long long i = blockIdx.x * 256LL + threadIdx.x, n = (long long)N * K;
    if (i >= 2 * n) return;
    float s = 0.f;
    for (int k = 0; k < splits; k++) s += part[k * 2 * n + i];
    const long long e = i < n ? i : i - n, row = e / K, col = e - row * K;
    reinterpret_cast<T*>(i < n ? dg + row * sg : dv + row * sv)[col] = from_f32<T>(s);
}

// Bias gradients: the waves' column sums, 32 columns x 8 lanes a block.
__global__ __launch_bounds__(256) void ff_db_fold_kernel(const float* part, long long rows, int N, float* dg, float* dv) {
    __shared__ double red[8][33];
    const int c = blockIdx.x * 32 + threadIdx.x % 32, lane = threadIdx.x / 32;
    double s = 0.0;
    if (c < 2 * N)
        for (long long r = lane; r < rows; r += 8) s += (double)part[r * 2 * N + c];
    red[lane][threadIdx.x % 32] = s;
    __syncthreads();
    if (lane || c >= 2 * N) return;
    for (int i = 1; i < 8; i++) s += red[i][threadIdx.x];
    float* d = c < N ? dg : dv;
    if (d) d[c < N ? c : c - N] = (float)s;
}

// --------------------------------------------------------------------------------- host
long long pad64(long long n) { return (n + 63) / 64 * 64; }
size_t pad256(size_t n) { return (n + 255) / 256 * 256; }

// A tensor [ne0, rows] over up to three evenly spaced dimensions.
struct Rows {
    char* data;
    long long n, stride;
};
Rows rows_of(const stx_tensor* t, int size, const char* what) {
    check_typed(t, size, what);
    Rows r{static_cast<char*>(t->data), t->ne[1] * t->ne[2] * t->ne[3], 0};
    bool first = true;
    long long expect = 0;
    for (int i = 1; i < 4 && r.n > 0; i++) {
        if (t->ne[i] == 1) continue;
        if (first) r.stride = t->nb[i];
        STX_REQUIRE(first || t->nb[i] == expect, "%s: rows are not evenly spaced", what);
        first = false;
        expect = t->nb[i] * t->ne[i];
    }
    if (first) r.stride = t->ne[0] * size;
    return r;
}

bool aligned_rows(const void* p, long long stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 16 == 0; }

template <class T, int MODE, int TJ, int TM, int WJ, int WM, bool AL>
void launch_tiles(FfArgs a, dim3 yz, hipStream_t stream) {
    const int width = MODE == FORWARD || MODE == GRAD ? TJ / 2 : TJ;
    a.jtiles = (a.J + width - 1) / width;
    a.mtiles = (int)(((long long)a.M + TM - 1) / TM);
    const long long tiles = (long long)a.jtiles * a.mtiles;
    if (tiles >= (1LL << 30)) fail(STX_STATUS_UNSUPPORTED, "gated_ff: too many tiles");
    hipLaunchKernelGGL((ff_kernel<T, MODE, TJ, TM, WJ, WM, AL>), dim3(xcd_grid(tiles), yz.y, yz.z), dim3(64 * WJ * WM), 0, stream, a);
    launch_check("ff_kernel");
}

constexpr int kSmall = 128;              // tile edge; its waves' rows of bias sums are 64 tokens
constexpr int kFew = 64;
constexpr long long kMaxWidth = 1 << 20, kMaxTokens = 1 << 30;   // of K and N; of the tokens (row indexes of tiles fit 32 bits)

template <class T, int MODE>
void launch_ff(const FfArgs& a, bool aligned, dim3 yz, hipStream_t stream) {
    if (aligned) launch_tiles<T, MODE, kSmall, kSmall, 2, 2, true>(a, yz, stream);
    else launch_tiles<T, MODE, kSmall, kSmall, 2, 2, false>(a, yz, stream);
}

struct Block {
    Rows x, wg, wv;
    long long M;
    int K, N;
};
Block check_block(const stx_tensor* x, const stx_tensor* wg, const stx_tensor* wv, int size) {
    Block b{};
    b.x = rows_of(x, size, "gated_ff: x");
    b.wg = rows_of(wg, size, "gated_ff: w_gate");
    b.wv = rows_of(wv, size, "gated_ff: w_value");
    STX_REQUIRE(x->ne[0] > 0 && x->ne[0] <= kMaxWidth, "gated_ff: K = %lld", (long long)x->ne[0]);
    STX_REQUIRE(wg->ne[0] == x->ne[0] && wv->ne[0] == x->ne[0], "gated_ff: the weights' rows differ from x's");
    for (const stx_tensor* w : {wg, wv})
        STX_REQUIRE(w->ne[1] > 0 && w->ne[1] <= kMaxWidth && w->ne[2] == 1 && w->ne[3] == 1, "gated_ff: weights must be [K, N]");
    STX_REQUIRE(wg->ne[1] == wv->ne[1], "gated_ff: w_gate and w_value differ in N");
    STX_REQUIRE(b.x.n <= kMaxTokens, "gated_ff: more than 2^30 tokens");
    b.M = b.x.n;
    b.K = (int)x->ne[0];
    b.N = (int)wg->ne[1];
    return b;
}

void check_tokens(const stx_tensor* t, const stx_tensor* x, long long width, const char* what) {
    STX_REQUIRE(t->ne[0] == width, "gated_ff: %s has rows of %lld, not %lld", what, (long long)t->ne[0], width);
    for (int i = 1; i < 4; i++) STX_REQUIRE(t->ne[i] == x->ne[i], "gated_ff: %s and x differ in ne[%d]", what, i);
}
void check_output(const stx_tensor* t, const Rows& r, int size, const char* what) {
    STX_REQUIRE(r.n <= 1 || r.stride >= t->ne[0] * size, "gated_ff: rows of %s overlap", what);
}

FfArgs products(const Block& b, const float* bg, const float* bv, stx_act act) {
    FfArgs k{};
    k.p[0] = b.wg.data;
    k.p[1] = b.wv.data;
    k.ps[0] = b.wg.stride;
    k.ps[1] = b.wv.stride;
    k.q[0] = b.x.data;
    k.qs[0] = b.x.stride;
    k.J = b.N;
    k.M = (int)b.M;
    k.R = b.K;
    k.b[0] = bg;
    k.b[1] = bv;
    k.act = act;
    return k;
}
bool products_aligned(const Block& b, int size) {
    return b.K % (16 / size) == 0 && aligned_rows(b.x.data, b.x.stride) && aligned_rows(b.wg.data, b.wg.stride) && aligned_rows(b.wv.data, b.wv.stride);
}

// Workspace of the backward pass. The split of the token reduction of the weights' gradients is
// chosen so that its tiles come to about two a CU of the MI355X's 256.
struct BackPlan {
    long long Mp, Np;
    int splits;
    long long split, db_rows;
    size_t dg, dgt, xt, wt, dw, db, total;
};
BackPlan back_plan(long long M, long long K, long long N, int size) {
    BackPlan p{};
    p.Mp = pad64(M);
    p.Np = pad64(N);
    const long long tiles = 2 * ((K + kSmall - 1) / kSmall) * ((N + kSmall - 1) / kSmall);
    const long long most = std::max(1LL, std::min(p.Mp / 512, 512 / tiles));
    p.split = pad64((p.Mp + most - 1) / most);
    p.splits = p.split ? (int)std::max(1LL, (p.Mp + p.split - 1) / p.split) : 1;
    p.db_rows = (M + kSmall - 1) / kSmall * 2;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += pad256(bytes);
        return here;
    };
    p.dg = take(2 * (size_t)(M * p.Np) * size);
    p.dgt = take(2 * (size_t)(N * p.Mp) * size);
    p.xt = take((size_t)(K * p.Mp) * size);
    p.wt = take(2 * (size_t)(K * p.Np) * size);
    p.dw = take((size_t)p.splits * 2 * N * K * sizeof(float));
    p.db = take((size_t)p.db_rows * 2 * N * sizeof(float));
    p.total = at;
    return p;
}

template <class T>
void transpose(const char* src, long long stride, long long rows, int cols, T* dst, long long ld, hipStream_t stream) {
    hipLaunchKernelGGL(ff_transpose_kernel<T>, dim3((unsigned)(pad64(rows) / 64), (cols + 63) / 64), dim3(256), 0, stream, src, stride, (int)rows, cols, dst, ld);
    launch_check("ff_transpose_kernel");
}

template <class T>
void run_back(const Block& b, const Rows& dh, const float* bg, const float* bv, stx_act act, const Rows* dx, const Rows* dwg, const Rows* dwv,
              float* dbg, float* dbv, char* ws, hipStream_t stream) {
    const BackPlan p = back_plan(b.M, b.K, b.N, sizeof(T));
    T* dg = reinterpret_cast<T*>(ws + p.dg);
    T* dv = dg + b.M * p.Np;
    T* dgt = reinterpret_cast<T*>(ws + p.dgt);
    T* dvt = dgt + b.N * p.Mp;
    T* xt = reinterpret_cast<T*>(ws + p.xt);
    T* wgt = reinterpret_cast<T*>(ws + p.wt);
    T* wvt = wgt + b.K * p.Np;
    float* dw = reinterpret_cast<float*>(ws + p.dw);
    float* db = reinterpret_cast<float*>(ws + p.db);
    if (b.M > 0) {
        FfArgs k = products(b, bg, bv, act);
        k.dh = dh.data;
        k.dhs = dh.stride;
        k.out[0] = dx || dwg ? reinterpret_cast<char*>(dg) : nullptr;
        k.out[1] = reinterpret_cast<char*>(dv);
        k.os = p.Np * (long long)sizeof(T);
        k.jpad = (int)p.Np;
        k.db = dbg || dbv ? db : nullptr;
        launch_ff<T, GRAD>(k, products_aligned(b, sizeof(T)), dim3(1), stream);
    }
    if (dbg || dbv) {
        hipLaunchKernelGGL(ff_db_fold_kernel, dim3((2 * b.N + 31) / 32), dim3(256), 0, stream, db, b.M > 0 ? p.db_rows : 0, b.N, dbg, dbv);
        launch_check("ff_db_fold_kernel");
    }
    if (dx && b.M > 0) {
        transpose<T>(b.wg.data, b.wg.stride, b.N, b.K, wgt, p.Np, stream);
        transpose<T>(b.wv.data, b.wv.stride, b.N, b.K, wvt, p.Np, stream);
        FfArgs k{};
        k.p[0] = reinterpret_cast<char*>(wgt);
        k.p[1] = reinterpret_cast<char*>(wvt);
        k.q[0] = reinterpret_cast<char*>(dg);
        k.q[1] = reinterpret_cast<char*>(dv);
        k.ps[0] = k.ps[1] = k.qs[0] = k.qs[1] = p.Np * (long long)sizeof(T);
        k.J = b.K;
        k.M = (int)b.M;
        k.R = p.Np;
        k.out[0] = dx->data;
        k.os = dx->stride;
        launch_ff<T, DX>(k, true, dim3(1), stream);
    }
    if (dwg) {
        int splits = 0;
        if (b.M > 0) {
            splits = p.splits;
            transpose<T>(b.x.data, b.x.stride, b.M, b.K, xt, p.Mp, stream);
            transpose<T>(reinterpret_cast<char*>(dg), p.Np * (long long)sizeof(T), b.M, b.N, dgt, p.Mp, stream);
            transpose<T>(reinterpret_cast<char*>(dv), p.Np * (long long)sizeof(T), b.M, b.N, dvt, p.Mp, stream);
            FfArgs k{};
            k.p[0] = reinterpret_cast<char*>(xt);
            k.q[0] = reinterpret_cast<char*>(dgt);
            k.q[1] = reinterpret_cast<char*>(dvt);
            k.ps[0] = k.qs[0] = k.qs[1] = p.Mp * (long long)sizeof(T);
            k.J = b.K;
            k.M = b.N;
            k.R = p.Mp;
            k.split = p.split;
            k.out[0] = reinterpret_cast<char*>(dw);
            k.os = b.K * 4LL;
            launch_ff<T, DW>(k, true, dim3(1, 2, splits), stream);
        }
        const long long n = 2LL * b.N * b.K;
        hipLaunchKernelGGL(ff_dw_fold_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, dw, splits, b.N, b.K, dwg->data, dwv->data, dwg->stride, dwv->stride);
        launch_check("ff_dw_fold_kernel");
    }
}

}  // namespace
}  // namespace stx

using namespace stx;

extern "C" {

STX_API stx_status stx_gated_ff(const stx_tensor* x, const stx_tensor* w_gate, const stx_tensor* w_value, stx_type type,
                                const float* b_gate, const float* b_value, stx_act act, const stx_tensor* dst,
                                stx_stream stream) {
    return guard([&] {
        const int size = type_size(type);
        const Block b = check_block(x, w_gate, w_value, size);
        check_act(act);
        const Rows d = rows_of(dst, size, "gated_ff: dst");
        check_tokens(dst, x, b.N, "dst");
        check_output(dst, d, size, "dst");
        for (const stx_tensor* t : {x, w_gate, w_value})
            STX_REQUIRE(!overlap(span_of(t, size), span_of(dst, size)), "gated_ff: dst overlaps an input");
        if (b.M == 0) return;
        FfArgs k = products(b, b_gate, b_value, act);
        k.out[0] = d.data;
        k.os = d.stride;
        with_type(type, [&](auto t) {
            using T = decltype(t);
            if (b.M > kFew) return launch_ff<T, FORWARD>(k, products_aligned(b, size), dim3(1), as_stream(stream));
            const dim3 grid((b.N + 15) / 16), block(512);
            if (b.M <= 16) hipLaunchKernelGGL((ff_few_kernel<T, 1>), grid, block, 0, as_stream(stream), k);
            else if (b.M <= 32) hipLaunchKernelGGL((ff_few_kernel<T, 2>), grid, block, 0, as_stream(stream), k);
            else hipLaunchKernelGGL((ff_few_kernel<T, 4>), grid, block, 0, as_stream(stream), k);
            launch_check("ff_few_kernel");
        });
    });
}

STX_API size_t stx_gated_ff_back_workspace_size(int64_t n_tokens, int64_t n_in, int64_t n_hidden, stx_type type) {
    size_t bytes = 0;
    (void)guard([&] {
        const int size = type_size(type);
        STX_REQUIRE(n_tokens >= 0 && n_tokens <= kMaxTokens && n_in > 0 && n_in <= kMaxWidth && n_hidden > 0 && n_hidden <= kMaxWidth,
                    "gated_ff_back_workspace_size: %lld tokens, K = %lld, N = %lld", (long long)n_tokens, (long long)n_in, (long long)n_hidden);
        bytes = back_plan(n_tokens, n_in, n_hidden, size).total;
    });
    return bytes;
}

STX_API stx_status stx_gated_ff_back(const stx_tensor* dh, const stx_tensor* x, const stx_tensor* w_gate,
                                     const stx_tensor* w_value, stx_type type, const float* b_gate, const float* b_value,
                                     stx_act act, const stx_tensor* dx, const stx_tensor* dw_gate,
                                     const stx_tensor* dw_value, float* db_gate, float* db_value, void* workspace,
                                     size_t workspace_bytes, stx_stream stream) {
    return guard([&] {
        const int size = type_size(type);
        const Block b = check_block(x, w_gate, w_value, size);
        check_act(act);
        const Rows h = rows_of(dh, size, "gated_ff_back: dh");
        check_tokens(dh, x, b.N, "dh");
        STX_REQUIRE((dw_gate == nullptr) == (dw_value == nullptr), "gated_ff_back: dw_gate and dw_value go together");
        Rows rx{}, rg{}, rv{};
        if (dx) {
            rx = rows_of(dx, size, "gated_ff_back: dx");
            check_tokens(dx, x, b.K, "dx");
            check_output(dx, rx, size, "dx");
        }
        if (dw_gate) {
            rg = rows_of(dw_gate, size, "gated_ff_back: dw_gate");
            rv = rows_of(dw_value, size, "gated_ff_back: dw_value");
            for (const stx_tensor* t : {dw_gate, dw_value}) check_same_shape(w_gate, t, "gated_ff_back: weight gradients");
            check_output(dw_gate, rg, size, "dw_gate");
            check_output(dw_value, rv, size, "dw_value");
            STX_REQUIRE(!overlap(span_of(dw_gate, size), span_of(dw_value, size)), "gated_ff_back: dw_gate overlaps dw_value");
        }
        for (const stx_tensor* o : {dx, dw_gate, dw_value})
            for (const stx_tensor* i : {dh, x, w_gate, w_value})
                STX_REQUIRE(!o || !overlap(span_of(o, size), span_of(i, size)), "gated_ff_back: an output overlaps an input");
        check_workspace(workspace, workspace_bytes, back_plan(b.M, b.K, b.N, size).total, "gated_ff_back");
        if (!dx && !dw_gate && !db_gate && !db_value) return;
        with_type(type, [&](auto t) {
            run_back<decltype(t)>(b, h, b_gate, b_value, act, dx ? &rx : nullptr, dw_gate ? &rg : nullptr, dw_value ? &rv : nullptr, db_gate,
                                  db_value, static_cast<char*>(workspace), as_stream(stream));
        });
    });
}

}  // extern "C"

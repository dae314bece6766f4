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

// fp32 values as sums of three bf16 ones (Henry, Tang and Heinecke, "Leveraging the bfloat16 artificial
// intelligence datatype for higher-precision computations", 2019): x = h + m + l with h = bf16(x), m =
// bf16(x - h), l = x - h - m, all exact. Rounded to nearest, |m| <= 2^-8 |x| and |l| <= 2^-17 |x| have either
// sign, and a product of two such sums without its three smallest terms (2 |m l| + |l l|: below 2^-24 of it)
// is six bf16 products without bias: 2.7 times the rate of the fp32 matrix instruction, at its
// accuracy. (Parts cut off instead drop up to 2^-21, always towards zero.) Values beyond the largest
// bf16 are rare enough for a form of their own (EDGE): h stays finite where x is, and an infinity is
// +-1 + 0 +- inf, so that in the six products it meets the other's h alone and gives what it gives there.
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
template <bool EDGE>
struct Split {
    static constexpr float most = 0x1.fep127f;
    u32x2 part[3];                       // four values' h, m, l as bf16
    static __device__ __forceinline__ float largest(u32x4 bits, float v) {
        const f32x4 x = __builtin_bit_cast(f32x4, bits);
        return fmaxf(fmaxf(fmaxf(fmaxf(v, fabsf(x[0])), fabsf(x[1])), fabsf(x[2])), fabsf(x[3]));   // NaN is passed over
    }
    __device__ __forceinline__ explicit Split(u32x4 bits) {
        f32x4 x = __builtin_bit_cast(f32x4, bits);
        float beyond[4] = {};
        if constexpr (EDGE) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const bool inf = fabsf(x[i]) == __builtin_inff();
                beyond[i] = inf ? x[i] : 0.f;
                x[i] = inf ? copysignf(1.f, x[i]) : x[i];
            }
        }
#pragma unroll
        for (int k = 0; k < 3; k++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                f32x2 v = {x[2 * i], x[2 * i + 1]};
                if (EDGE && k == 0) v = f32x2{__builtin_amdgcn_fmed3f(v[0], -most, most), __builtin_amdgcn_fmed3f(v[1], -most, most)};
                if (EDGE && k == 2) v += f32x2{beyond[2 * i], beyond[2 * i + 1]};
                const unsigned pair = __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
                part[k][i] = pair;
                x[2 * i] -= __uint_as_float(pair << 16);
                x[2 * i + 1] -= __uint_as_float(pair & 0xffff0000u);
            }
    }
};
// x as a high and a low bf16 part; the high one is finite, so that a finite x stays so and an infinity,
// in the low part, meets no zero of another high part.
__device__ __forceinline__ void halves(float x, bf16& hi, bf16& lo) {
    hi = (bf16)__builtin_amdgcn_fmed3f(x, -0x1.fep127f, 0x1.fep127f);
    lo = (bf16)(x - (float)hi);
}
__device__ __forceinline__ f32x4 mma(const u32x4 (&a)[1], const u32x4 (&b)[2], f32x4 acc) {   // smallest terms first
    acc = mma(a[0], b[1], acc, bf16{});
    return mma(a[0], b[0], acc, bf16{});
}
__device__ __forceinline__ f32x4 mma(const u32x4 (&a)[2], const u32x4 (&b)[2], f32x4 acc) {
    acc = mma(a[1], b[0], acc, bf16{});
    acc = mma(a[0], b[1], acc, bf16{});
    return mma(a[0], b[0], acc, bf16{});
}
__device__ __forceinline__ f32x4 mma(const u32x4 (&a)[3], const u32x4 (&b)[3], f32x4 acc) {
    acc = mma(a[2], b[0], acc, bf16{});
    acc = mma(a[0], b[2], acc, bf16{});
    acc = mma(a[1], b[1], acc, bf16{});
    acc = mma(a[1], b[0], acc, bf16{});
    acc = mma(a[0], b[1], acc, bf16{});
    return mma(a[0], b[0], acc, bf16{});
}

// The products of the block, all of the form out[m][j] = sum_r P(j, r) Q(m, r):
//   FORWARD  P = rows of Wg and Wv, 16 by 16 in turn (a lane then holds gate and value of the same
//            outputs), Q = x; the epilogue forms act(g) v.
//   GRAD     the same products again; the epilogue takes dh and writes dg = dh v act'(g) and
//            dv = dh act(g), and per wave the sums of its columns for the biases' gradients.
//   DX       P = the weights, Q = dg, then dv: both reductions (over the N outputs) into one
//            accumulator.
//   DW       P = x, Q = dg or dv, reduced over the tokens.
// GRAD leaves dg and dv in fp32, of 16-bit data as two bf16 parts, high and low: 16 bits at any
// exponent. Rounded to the data's type instead they would add an error as large as that of the
// results' own rounding (bf16, 48,060 tokens, K 384, N 1,536: 2.3e-3 where it is 1.65e-3), and fp16's would end
// at 65,504 and 2^-24, where a sum that they enter need not. DX and DW multiply both parts, by
// bf16's P as it is and by fp16's in two bf16 parts (without the product of the two low ones, below
// 2^-17 of the whole). An infinity in P may give NaN there: infinity times a low part of 0.
// In FORWARD and GRAD r is the fastest dimension of both operands, in DX of Q only and in DW of
// neither; an operand whose r is not its fastest dimension is "strided" below.
enum Mode { FORWARD, GRAD, DX, DW };

// Tiles of TJ x TM outputs, WJ x WM waves. A step of the reduction is 64 values
// of every row in FORWARD and GRAD of 16-bit data, in two stages of LDS (five stages of 32, which keep
// twice as much in flight, took 5 to 10 % longer: twice the barriers), and 32 elsewhere, where an
// operand has two or three parts.
constexpr bool splits(Mode mode, stx_type type) { return type == STX_TYPE_F32 || (type == STX_TYPE_F16 && (mode == DX || mode == DW)); }   // P, on its way to LDS
constexpr int step_of(Mode mode, int size) { return size == 2 && (mode == FORWARD || mode == GRAD) ? 64 : 32; }
// Blocks of a tile (0 Large, 1 Medium, 2 Small) that a CU holds: what LDS has room for, and the registers are held to.
constexpr int slots_of(int tile, Mode mode, stx_type type) {
    return tile == 0 ? 1 : tile == 1 && !(type == STX_TYPE_BF16 && (mode == DX || mode == DW)) ? 2 : 3;
}
template <int TJ_, int TM_, int WJ_, int WM_>
struct Tile {
    static constexpr int TJ = TJ_, TM = TM_, WJ = WJ_, WM = WM_, NT = 64 * WJ * WM;
    template <class T, int MODE>
    static constexpr int slots = slots_of(TJ == 256 ? 0 : TM == 128 ? 1 : 2, (Mode)MODE, type_of<T>);
};
using Large = Tile<256, 256, 2, 4>;
using Medium = Tile<128, 128, 2, 2>;
using Small = Tile<128, 64, 2, 2>;

struct FfArgs {
    const char* p[2];
    const char* q[2];
    long long ps[2], qs[2];              // row strides in bytes
    int J, M;                            // extents of P's and Q's other dimension
    long long RP, RQ;                    // reduction lengths: past RP (of a strided P or Q past its own) zeros are taken
    int steps, chunk;                    // steps of one reduction; of a part of it (DX, DW)
    int jtiles, tiles, items;            // column tiles, output tiles, tiles x parts (x 2 in DW)
    const float* b[2];
    int act;
    const char* dh;
    long long dhs;
    char* out[2];
    long long os[2];                     // output row strides in bytes
    int jpad;                            // columns written: J, in GRAD padded with zeros
    int qpad;                            // DW: columns that a row of Q has
    long long plane;                     // of 16-bit data: bytes from dg's and dv's high parts to their low ones
    float* part;                         // GRAD: column sums [wave rows][2][J]; DX, DW: [parts][M][J] or NULL
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
        T e[E];                                          // clamped, not skipped: a load each, no branches
#pragma unroll
        for (int i = 0; i < E; i++) {
            const T x = reinterpret_cast<const T*>(p)[i < left ? i : 0];
            e[i] = i < left ? x : T(0.f);
        }
        __builtin_memcpy(&v, e, 16);
    }
    return v;
}
// 16 bytes a lane from memory to LDS at lds + lane * 16 (lds uniform over the wave): at base + off,
// base uniform; or at p. Written out because the compiler takes every such load for one that a
// transposing LDS read might depend on, and waits for all of them before it; the waits are
// settle()'s. No register is written. s_nop: a wait state between m0 and its use, five between a
// vector instruction that may have written the base (a lane read, a reloaded spill) and its use.
__device__ __forceinline__ unsigned lds_address(const void* p) {
    return (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(unsigned long long)(__attribute__((address_space(3))) const void*)p);
}
// m0 is named as overwritten, so that no use of the compiler's own is placed across; it warns that it
// never allocates that register.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(const char* base, unsigned off, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void load_to_lds(const void* p, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}
#pragma clang diagnostic pop

template <class T>
__device__ __forceinline__ void load4(const char* p, int left, float (&f)[4]) {
    if (left >= 4) {
        T v[4];
        __builtin_memcpy(v, p, sizeof v);
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = to_f32(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = 0.f;
        if (left > 0) {
#pragma unroll
            for (int i = 0; i < 4; i++) f[i] = to_f32(reinterpret_cast<const T*>(p)[i < left ? i : 0]);
        }
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

// An operand's tile of X rows (or columns) of 16-bit values in a stage of LDS. Plain: [X][PER] chunks
// of 8 values, chunk c of row x at c ^ bend(x), so that eight rows which a fragment reads together
// lie in different banks. Strided: rows of the reduction, [8 PER][X / 8] chunks, chunk c of row r at
// c ^ turn(r), so that the 4 rows of 32 bytes which the transposing read takes do. A 16-bit
// operand is fetched in this form (PER 8: a step of 64; 4: of 32), dg and dv in two planes of it; an
// fp32 one is split on its way into three planes, fp16's P of DX and DW into two.
template <int PER>
__device__ __forceinline__ int bend(int x) {
    return PER == 8 ? x % 8 : x / 2 % 4;
}
template <int X>
__device__ __forceinline__ int turn(int r) {
    return 2 * (r % 4 + r / 8 % 2 * 4) % (X / 8);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));

// Fragments of 16-row tiles from `first` on, for lane l: the chunk of row l % 16 at position l / 16 of
// group kk (see mma).
template <int X, int N, int PER, bool STRIDED>
struct Fragments {
    int at[STRIDED ? N : 1];
    __device__ __forceinline__ Fragments(int lane, int first) {
        const int s = lane % 16, q = lane / 16;
        if constexpr (!STRIDED) {
            at[0] = (first * 16 + s) * PER * 16 + (q ^ bend<PER>(s)) * 16;
        } else {                                         // lane s reads row s / 4, columns 4 (s % 4) .. + 3
            const int row = q * 8 + s / 4;
#pragma unroll
            for (int i = 0; i < N; i++) at[i] = row * X * 2 + (((first + i) * 2 + s % 4 / 2) ^ turn<X>(row)) * 16 + s % 2 * 8;
        }
    }
    __device__ __forceinline__ u32x4 read(const char* lds, int kk, int i) const {
        u32x4 f;
        if constexpr (!STRIDED) {
            f = *reinterpret_cast<const u32x4*>(lds + i * 256 * PER + (at[0] ^ (kk * 64)));
        } else {
            s16x4 h[2];
#pragma unroll
            for (int e = 0; e < 2; e++)
                h[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds + at[i] + (kk * 32 + e * 4) * X * 2));
            __builtin_memcpy(&f, h, 16);
        }
        return f;
    }
};

// The 16-byte chunks of an operand's tile that a thread fetches in a step of R values: [X][R / E],
// strided [R][X / E].
template <class T, int X, int NT, bool STRIDED, int R>
struct Source {
    static constexpr int E = 16 / sizeof(T), N = X * R / E / NT, PER = STRIDED ? X / E : R / E;   // chunks a thread; chunks a row
    static_assert(X * R / E % NT == 0);
    static __device__ __forceinline__ int row(int i) { return (i * NT + (int)threadIdx.x) / PER; }
    static __device__ __forceinline__ int chunk(int i) {
        const int c = (i * NT + (int)threadIdx.x) % PER;
        if constexpr (sizeof(T) == 4) return c;
        else return c ^ (STRIDED ? turn<X>(row(i)) : bend<R / 8>(row(i)));
    }
    // fp32: where the four values of chunk i lie in a plane.
    static __device__ __forceinline__ int spot(int i) {
        const int r = row(i), c = chunk(i);
        return (STRIDED ? r * X * 2 + ((c / 2) ^ turn<X>(r)) * 16 : r * 64 + ((c / 2) ^ bend<4>(r)) * 16) + c % 2 * 8;
    }
};

// Persistent blocks: each takes tiles of its XCD's share in turn, and the steps of all its tiles
// form one stream: while the waves multiply one stage of LDS, the other is filled with the next
// step, the next tile's first included: straight from memory to LDS for aligned 16-bit operands
// (ALIGNED), otherwise through registers, for any alignment and length. fp32 operands are split
// between the registers and LDS, once a block (by every wave from its fragments, splitting took
// longer than the products), and have one stage of three planes: two would leave room for one
// block a CU. fp16's P of DX and DW is split there too.
template <class T, int MODE, class C, bool ALIGNED>
__global__ __launch_bounds__(C::NT, (C::template slots<T, MODE> * C::NT / 256)) void ff_kernel(FfArgs a) {
    constexpr int NT = C::NT, E = 16 / sizeof(T), TJ = C::TJ, TM = C::TM;
    constexpr int NJ = TJ / C::WJ / 16, NM = TM / C::WM / 16;       // 16 x 16 tiles of a wave
    constexpr bool GATED = MODE == FORWARD || MODE == GRAD, PS = !GATED, QS = MODE == DW;
    constexpr int WIDTH = GATED ? TJ / 2 : TJ;                       // output columns of a tile
    constexpr bool SPLIT = sizeof(T) == 4, HALVE = !GATED && std::is_same_v<T, f16>;
    constexpr int R = step_of((Mode)MODE, sizeof(T)), PER = R / 8, STAGES = SPLIT ? 1 : 2;
    constexpr int PP = SPLIT ? 3 : HALVE ? 2 : 1, QP = SPLIT ? 3 : GATED ? 1 : 2;              // planes
    constexpr int QIN = SPLIT ? 1 : QP;                              // of Q in memory
    constexpr int PPLANE = TJ * PER * 16, QPLANE = TM * PER * 16, QAT = PPLANE * PP, STAGE = QAT + QPLANE * QP;
    static_assert(!((SPLIT || HALVE) && ALIGNED));
    using PSource = Source<T, TJ, NT, PS, R>;
    using QSource = Source<T, TM, NT, QS, R>;
    __shared__ __align__(128) char lds[STAGES][STAGE];

    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const int wj = wave / C::WM, wm = wave % C::WM;

    // Item `id`: part z of a tile. Tiles in groups of 8 along m, m fastest: the tiles that an XCD
    // works on at a time share rows of both operands.
    struct Item {
        int m0, j0, z, begin, end;       // end: steps [begin, end) of the reduction (DX: of both)
    };
    const int mtiles = a.tiles / a.jtiles;
    auto item_of = [&](int id) {
        Item t;
        t.z = id / a.tiles;
        id -= t.z * a.tiles;
        const int per = 8 * a.jtiles, group = id / per, in = id - group * per, gm = min(8, mtiles - group * 8);
        t.m0 = (group * 8 + in % gm) * TM;
        t.j0 = in / gm * WIDTH;
        t.begin = 0;
        t.end = a.steps;
        if constexpr (!GATED) {
            t.begin = (MODE == DW ? t.z / 2 : t.z) * a.chunk;
            t.end = min(t.begin + a.chunk, MODE == DX ? 2 * a.steps : a.steps);
        }
        return t;
    };
    const int per = (a.items + kXcds - 1) / kXcds, last = min(((int)blockIdx.x % kXcds + 1) * per, a.items);
    int id = (int)blockIdx.x % kXcds * per + (int)blockIdx.x / kXcds;
    const int stride = (int)gridDim.x / kXcds;
    if (id >= last) return;

    // A step's chunks lie at a base (of the tile and step, in scalar registers) plus a lane's own
    // offset of less than 2^31 (ALIGNED: row strides below 2^23), which changes with the tile only
    // where rows are clamped. With unaligned operands the offset is 64-bit.
    using Off = std::conditional_t<ALIGNED, unsigned, long long>;
    Off poff[PSource::N], qoff[QSource::N];
    const int pside = GATED ? __builtin_amdgcn_readfirstlane(tid / PSource::PER / 16 % 2) : 0;   // the matrix of a wave's rows
    auto aim = [&](const Item& t, int seg, int qs) {
#pragma unroll
        for (int i = 0; i < PSource::N; i++) {
            const int row = PSource::row(i), at = PSource::chunk(i) * E;
            if constexpr (PS) poff[i] = (Off)(row * a.ps[seg] + (ALIGNED ? min(at, a.J - E - t.j0) : at) * (long long)sizeof(T));
            else poff[i] = (Off)(min(row / 32 * 16 + row % 16, a.J - 1 - t.j0) * a.ps[pside] + at * (long long)sizeof(T));
        }
#pragma unroll
        for (int i = 0; i < QSource::N; i++) {
            const int row = QSource::row(i), at = QSource::chunk(i) * E;
            if constexpr (QS) qoff[i] = (Off)(row * a.qs[qs] + min(at, a.qpad - E - t.m0) * (long long)sizeof(T));
            else qoff[i] = (Off)(min(row, a.M - 1 - t.m0) * a.qs[qs] + at * (long long)sizeof(T));
        }
    };
    constexpr int HELD = PSource::N + QSource::N * QIN;
    u32x4 hold[ALIGNED ? 1 : HELD];
    auto fetch = [&](const Item& t, int step, int stage) {
        const int seg = MODE == DX && step >= a.steps ? 1 : 0, qs = MODE == DW ? t.z % 2 : seg;
        if (step == t.begin || (MODE == DX && step == a.steps)) aim(t, seg, qs);
        const long long r = (long long)(step - seg * a.steps) * R;
        const char* pb = PS ? a.p[seg] + r * a.ps[seg] + t.j0 * (long long)sizeof(T) : a.p[pside] + t.j0 * a.ps[pside] + r * (long long)sizeof(T);
        const char* qb = QS ? a.q[qs] + r * a.qs[qs] + t.m0 * (long long)sizeof(T) : a.q[qs] + t.m0 * a.qs[qs] + r * (long long)sizeof(T);
        if constexpr (ALIGNED) {
            const unsigned pl = lds_address(lds[stage] + wave * 1024), ql = pl + QAT;
            if (r + R <= a.RP && r + R <= a.RQ) {
#pragma unroll
                for (int i = 0; i < PSource::N; i++) load_to_lds(pb, poff[i], pl + i * NT * 16);
#pragma unroll
                for (int k = 0; k < QIN; k++)
#pragma unroll
                    for (int i = 0; i < QSource::N; i++) load_to_lds(qb + k * a.plane, qoff[i], ql + k * QPLANE + i * NT * 16);
            } else {                                     // the reduction's end: zeros for what is past it
#pragma unroll
                for (int i = 0; i < PSource::N; i++)
                    load_to_lds(r + (PS ? PSource::row(i) : PSource::chunk(i) * E) < a.RP ? (const void*)(pb + poff[i]) : (const void*)&zero_chunk, pl + i * NT * 16);
#pragma unroll
                for (int k = 0; k < QIN; k++)
#pragma unroll
                    for (int i = 0; i < QSource::N; i++)
                        load_to_lds(r + (QS ? QSource::row(i) : QSource::chunk(i) * E) < a.RQ ? (const void*)(qb + k * a.plane + qoff[i]) : (const void*)&zero_chunk,
                                    ql + k * QPLANE + i * NT * 16);
            }
        } else if (r + R <= a.RP && r + R <= a.RQ && (!PS || t.j0 + TJ <= a.J)) {
#pragma unroll
            for (int i = 0; i < PSource::N; i++) __builtin_memcpy(&hold[i], pb + poff[i], 16);
#pragma unroll
            for (int i = 0; i < QSource::N * QIN; i++) __builtin_memcpy(&hold[PSource::N + i], qb + i / QSource::N * a.plane + qoff[i % QSource::N], 16);
        } else {
#pragma unroll
            for (int i = 0; i < PSource::N; i++)
                hold[i] = load_chunk<T>(pb + poff[i], !PS ? a.RP - r - PSource::chunk(i) * E : r + PSource::row(i) < a.RP ? a.J - t.j0 - PSource::chunk(i) * E : 0);
#pragma unroll
            for (int k = 0; k < QIN; k++)
#pragma unroll
                for (int i = 0; i < QSource::N; i++)
                    hold[PSource::N + k * QSource::N + i] =
                        load_chunk<T>(qb + k * a.plane + qoff[i], !QS ? a.RQ - r - QSource::chunk(i) * E : r + QSource::row(i) < a.RQ ? E : 0);
        }
    };
    // The stream of fetches, one step ahead of the products.
    Item ft = item_of(id);
    int fid = id, fstep = ft.begin, fstage = 0;
    bool more = true;
    auto fetch_next = [&] {
        fetch(ft, fstep, fstage);
        if constexpr (STAGES == 2) fstage ^= 1;
        if (++fstep == ft.end) {
            fid += stride;
            more = fid < last;
            if (more) {
                ft = item_of(fid);
                fstep = ft.begin;
            }
        }
    };
    // Waits for the step in `stage`.
    auto settle = [&](int stage) {
        if constexpr (ALIGNED) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        } else if constexpr (SPLIT) {
            __syncthreads();                             // the one stage is read
            auto split = [&](auto edge) {
#pragma unroll
                for (int i = 0; i < PSource::N + QSource::N; i++) {
                    const Split<edge()> v(hold[i]);
                    char* to = lds[0] + (i < PSource::N ? PSource::spot(i) : QAT + QSource::spot(i - PSource::N));
#pragma unroll
                    for (int k = 0; k < 3; k++) *reinterpret_cast<u32x2*>(to + k * (i < PSource::N ? PPLANE : QPLANE)) = v.part[k];
                }
            };
            float v = 0.f;
#pragma unroll
            for (int i = 0; i < PSource::N + QSource::N; i++) v = Split<false>::largest(hold[i], v);
            if (__builtin_amdgcn_ballot_w64(v > Split<false>::most)) split(std::true_type{});
            else split(std::false_type{});
        } else {
#pragma unroll
            for (int i = 0; i < HELD; i++) {
                char* to = lds[stage] + (i < PSource::N ? i * NT * 16 : QAT + (i - PSource::N) * NT * 16) + tid * 16;   // planes of Q follow one another
                if (HALVE && i < PSource::N) {
                    f16 x[8];
                    bf16 part[2][8];
                    __builtin_memcpy(x, &hold[i], 16);
#pragma unroll
                    for (int e = 0; e < 8; e++) halves(to_f32(x[e]), part[0][e], part[1][e]);
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        u32x4 v;
                        __builtin_memcpy(&v, part[k], 16);
                        *reinterpret_cast<u32x4*>(to + k * PPLANE) = v;
                    }
                } else {
                    *reinterpret_cast<u32x4*>(to) = hold[i];
                }
            }
        }
        __syncthreads();
    };

    const Fragments<TJ, NJ, PER, PS> pf(lane, wj * NJ);
    const Fragments<TM, NM, PER, QS> qf(lane, wm * NM);
    f32x4 acc[NJ][NM];

    // A wave's outputs leave 16 rows at a time. 16-bit results go through the wave's share of the
    // stage that was multiplied last, as 16-byte pieces of rows of COLS columns: stored from the
    // accumulators' own layout they would be runs of 32 bytes (the forward product of 48,060 tokens,
    // K 384, N 1536 then spends 41 us of 167 on its stores).
    constexpr int COLS = GATED ? NJ * 8 : NJ * 16, CR = COLS / 8, AREA = 16 * COLS * 2, SHARE = STAGE / (NT / 64), PIECES = 16 * CR / 64;
    constexpr int AREAS = MODE == GRAD ? 4 : 1, TURNS = AREA * AREAS * 2 <= SHARE ? 2 : 1;   // areas of 16 rows; groups in turn
    static_assert(AREA * AREAS <= SHARE && PIECES >= 1 && 16 * CR % 64 == 0, "staging");
    auto spot = [&](unsigned row, unsigned col) { return row * COLS * 2 + (col / 8 + row) % CR * 16 + col % 8 * 2; };
    auto pack = [&](char* p, const float (&f)[4]) {
        T v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = from_f32<T>(f[i]);
        __builtin_memcpy(__builtin_assume_aligned(p, 8), v, sizeof v);
    };
    auto pack_halves = [&](char* p, const float (&f)[4]) {
        bf16 hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; i++) halves(f[i], hi[i], lo[i]);
        __builtin_memcpy(__builtin_assume_aligned(p, 8), hi, sizeof hi);
        __builtin_memcpy(__builtin_assume_aligned(p + AREA, 8), lo, sizeof lo);
    };
    // The lane's number as a new value: addresses formed from it are not kept from one group of rows
    // for the next, there being no registers for them beside the accumulators.
    auto fresh = [&] {
        unsigned l = lane;
        asm volatile("" : "+v"(l));
        return l;
    };
    auto flush = [&](unsigned lane, const char* area, char* out, long long os, int row0, int col0) {
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const int row = (int)((i * 64 + lane) / CR), c = (int)((i * 64 + lane) % CR * 8), left = a.jpad - col0 - c;
            const char* from = area + spot(row, c);
            char* to = out + (row0 + row) * os + (col0 + c) * (long long)sizeof(T);
            if (row0 + row >= a.M) continue;
            if (left >= 8) {
                const u32x4 v = *reinterpret_cast<const u32x4*>(from);
                __builtin_memcpy(to, &v, 16);
            } else {
#pragma unroll 1
                for (int e = 0; e < left; e++) reinterpret_cast<T*>(to)[e] = reinterpret_cast<const T*>(from)[e];
            }
        }
    };
    constexpr bool WIDE = sizeof(T) == 2, TAKES = MODE == GRAD && WIDE;
    u32x4 dhv[TAKES ? NM : 1][TAKES ? PIECES : 1];       // the wave's part of dh
    auto take = [&](unsigned lane, const Item& t, int m) {
        if constexpr (TAKES) {
#pragma unroll
            for (int i = 0; i < PIECES; i++) {
                const int row = t.m0 + (wm * NM + m) * 16 + (int)((i * 64 + lane) / CR), col = t.j0 + wj * NJ * 8 + (int)((i * 64 + lane) % CR * 8);
                dhv[m][i] = load_chunk<T>(a.dh + row * a.dhs + col * (long long)sizeof(T), row < a.M ? a.J - col : 0);
            }
        }
    };

    auto gated = [&](const Item& t, char* share, auto act, auto whole) {
        const int nw = t.j0 + wj * NJ * 8;               // the wave's first column
        float sg[MODE == GRAD ? NJ / 2 : 1][4] = {}, sv[MODE == GRAD ? NJ / 2 : 1][4] = {};
#pragma unroll
        for (int m = 0; m < NM; m++) {
            const unsigned lane = fresh();
            const int row0 = t.m0 + (wm * NM + m) * 16, row = row0 + (int)(lane % 16);
            char* area = share + m % TURNS * AREAS * AREA;
            if constexpr (TAKES) {
#pragma unroll
                for (int i = 0; i < PIECES; i++) *reinterpret_cast<u32x4*>(area + spot((i * 64 + lane) / CR, (i * 64 + lane) % CR * 8)) = dhv[m][i];
            }
#pragma unroll
            for (int j = 0; j < NJ; j += 2) {
                const int col = j * 8 + (int)(lane / 16 * 4), n = nw + col;
                char* here = area + spot(lane % 16, col);
                if constexpr (MODE == FORWARD) {
                    float h[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) h[r] = act_f32<act(), T>(acc[j][m][r]) * acc[j + 1][m][r];
                    if constexpr (WIDE) pack(here, h);
                    else if (row < a.M) store4<T>(a.out[0] + row * a.os[0] + n * (long long)sizeof(T), a.J - n, h);
                } else {
                    float dh[4], dg[4], dv[4];
                    if constexpr (WIDE) load4<T>(static_cast<const char*>(__builtin_assume_aligned(here, 8)), 4, dh);
                    else load4<T>(a.dh + row * a.dhs + n * (long long)sizeof(T), row < a.M ? a.J - n : 0, dh);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        float d;
                        const float g = act_f32<act(), T>(acc[j][m][r], d);
                        const bool in = whole() || (row < a.M && n + r < a.J);   // what lies past the edges may be anything, NaN too
                        dg[r] = in ? dh[r] * acc[j + 1][m][r] * d : 0.f;
                        dv[r] = in ? dh[r] * g : 0.f;
                        sg[j / 2][r] += dg[r];
                        sv[j / 2][r] += dv[r];
                    }
                    if constexpr (WIDE) {
                        pack_halves(here, dg);
                        pack_halves(here + 2 * AREA, dv);
                    } else if (row < a.M && a.out[0]) {
                        store4<T>(a.out[0] + row * a.os[0] + n * (long long)sizeof(T), a.jpad - n, dg);
                        store4<T>(a.out[1] + row * a.os[1] + n * (long long)sizeof(T), a.jpad - n, dv);
                    }
                    __builtin_amdgcn_sched_barrier(0);   // one at a time: there are no registers for more
                }
            }
            if constexpr (WIDE) {
                if (MODE == FORWARD || a.out[0]) {
                    flush(lane, area, a.out[0], a.os[0], row0, nw);
                    if constexpr (MODE == GRAD) {
                        flush(lane, area + AREA, a.out[0] + a.plane, a.os[0], row0, nw);
                        flush(lane, area + 2 * AREA, a.out[1], a.os[1], row0, nw);
                        flush(lane, area + 3 * AREA, a.out[1] + a.plane, a.os[1], row0, nw);
                    }
                }
            }
        }
        if constexpr (MODE == GRAD) {
            if (!a.part) return;
            float* part = a.part + ((long long)(t.m0 / TM) * C::WM + wm) * 2 * a.J;
#pragma unroll
            for (int j = 0; j < NJ / 2; j++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int n = nw + j * 16 + lane / 16 * 4 + r;
                    const float g = row_sum(sg[j][r]), v = row_sum(sv[j][r]);
                    if (lane % 16 == 0 && n < a.J) {
                        part[n] = g;
                        part[a.J + n] = v;
                    }
                }
        }
    };
    auto plain = [&](const Item& t, char* share) {
        const int jw = t.j0 + wj * NJ * 16, which = MODE == DW ? t.z % 2 : 0;
        float* part = a.part ? a.part + (long long)t.z * a.M * a.J : nullptr;
#pragma unroll
        for (int m = 0; m < NM; m++) {
            const unsigned lane = fresh();
            const int row0 = t.m0 + (wm * NM + m) * 16, row = row0 + (int)(lane % 16);
            char* area = share + m % TURNS * AREA;
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const float f[4] = {acc[j][m][0], acc[j][m][1], acc[j][m][2], acc[j][m][3]};
                const int c = j * 16 + (int)(lane / 16 * 4), col = jw + c;
                if (part) {
                    if (row < a.M) store4<float>(reinterpret_cast<char*>(part + (long long)row * a.J + col), a.J - col, f);
                } else if constexpr (WIDE) {
                    pack(area + spot(lane % 16, c), f);
                } else if (row < a.M) {
                    store4<T>(a.out[which] + row * a.os[which] + col * (long long)sizeof(T), a.J - col, f);
                }
            }
            if constexpr (WIDE)
                if (!part) flush(lane, area, a.out[which], a.os[which], row0, jw);
        }
    };
    // A tile starts from its biases, or from zeros.
    auto start = [&](const Item& t) {
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            float b[4] = {};
            if constexpr (GATED) {
                const int n = t.j0 + (wj * NJ + j) / 2 * 16 + lane / 16 * 4;
                if (a.b[j % 2]) {
#pragma unroll
                    for (int r = 0; r < 4; r++) b[r] = a.b[j % 2][min(n + r, a.J - 1)];
                }
            }
#pragma unroll
            for (int m = 0; m < NM; m++) acc[j][m] = f32x4{b[0], b[1], b[2], b[3]};
        }
    };

    fetch_next();
    int stage = 0;
    while (true) {
        const Item t = item_of(id);
        start(t);
        char* share = nullptr;
#pragma unroll 1
        for (int s = t.begin; s < t.end; s++) {
            settle(stage);                               // every wave is done with the stage before it, too
            if (more) fetch_next();
            if constexpr (TAKES) {
                if (s + 1 == t.end) {
#pragma unroll
                    for (int m = 0; m < NM; m++) take(lane, t, m);
                }
            }
            const char *pl = lds[stage], *ql = pl + QAT;
            if constexpr (QP > 1) {
                static_assert(PER == 4);
                u32x4 fq[NM][QP];
#pragma unroll
                for (int m = 0; m < NM; m++)
#pragma unroll
                    for (int k = 0; k < QP; k++) fq[m][k] = qf.read(ql + k * QPLANE, 0, m);
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    u32x4 fp[PP];
#pragma unroll
                    for (int k = 0; k < PP; k++) fp[k] = pf.read(pl + k * PPLANE, 0, j);
#pragma unroll
                    for (int m = 0; m < NM; m++) acc[j][m] = mma(fp, fq[m], acc[j][m]);
                }
            } else {
#pragma unroll
                for (int kk = 0; kk < PER / 4; kk++) {
                    u32x4 fp[NJ], fq[NM];
#pragma unroll
                    for (int j = 0; j < NJ; j++) fp[j] = pf.read(pl, kk, j);
#pragma unroll
                    for (int m = 0; m < NM; m++) fq[m] = qf.read(ql, kk, m);
#pragma unroll
                    for (int j = 0; j < NJ; j++)
#pragma unroll
                        for (int m = 0; m < NM; m++) acc[j][m] = mma(fp[j], fq[m], acc[j][m], T{});
                }
            }
            share = lds[stage];
            if constexpr (STAGES == 2) stage ^= 1;
        }
        __syncthreads();                                 // the last stage is read; its shares are free until the next step settles
        share += wave * SHARE;
        if constexpr (MODE == FORWARD) {
            with_act(a.act, [&](auto act) { gated(t, share, act, std::true_type{}); });
        } else if constexpr (MODE == GRAD) {
            if (t.m0 + TM <= a.M && t.j0 + WIDTH <= a.J) with_act(a.act, [&](auto act) { gated(t, share, act, std::true_type{}); });
            else with_act(a.act, [&](auto act) { gated(t, share, act, std::false_type{}); });
        }
        else plain(t, share);
        id += stride;
        if (id >= last) return;
    }
}

// Few tokens (at most 64): the weights' bytes are the floor, each read by one block, straight into
// the matrix instructions' registers. A block has 16 outputs; its 8 waves take the 64-byte
// steps of the rows in turn and add their accumulators in LDS. bf16, K 2,048, N 8,192: one token 13 us (67 MB
// at 5.2 TB/s), 16 tokens 14 us, 32 18, 64 26 us, where the tiles take 27 to 29; fp32 28, 39 and 68 us
// against 85 (K 384, N 1,536: bf16 4.5 to 5.7 us against 7; fp32 5.4 to 9.1 against 18).
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
    const int steps = (int)((a.RP + 4 * E - 1) / (4 * E));
    auto take = [&](int s, auto whole) {
        const long long r = (long long)s * 4 * E + lane / 16 * E, at = r * (long long)sizeof(T), left = whole() ? E : a.RP - r;
        const u32x4 g = load_chunk<T>(p[0] + at, left), v = load_chunk<T>(p[1] + at, left);
#pragma unroll
        for (int m = 0; m < NM; m++) {
            const u32x4 x = load_chunk<T>(q[m] + at, left);
            acc[0][m] = mma(g, x, acc[0][m], T{});
            acc[1][m] = mma(v, x, acc[1][m], T{});
        }
    };
    const int full = (int)(a.RP / (4 * E));
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
        h[r] = act_f32<act(), T>(g[r] + (a.b[0] && in ? a.b[0][n + r] : 0.f)) * (v[r] + (a.b[1] && in ? a.b[1][n + r] : 0.f));
    }
    });
    store4<T>(a.out[0] + row * a.os[0] + n * (long long)sizeof(T), a.J - n, h);
}

// Sums of the parts of a split reduction, in order: part [splits][W][rows][cols] to out[w][rows][cols].
template <class T, int V>
__global__ __launch_bounds__(256) void ff_fold_kernel(const float* part, int splits, long long rows, int cols, int w, char* o0, char* o1, long long s0, long long s1,
                                                     unsigned base) {
    const long long n = rows * cols, i = ((base + blockIdx.x) * 256LL + threadIdx.x) * V;
    if (i >= w * n) return;
    float s[V] = {};
#pragma unroll 4
    for (int k = 0; k < splits; k++) {
        float f[V];
        __builtin_memcpy(f, part + k * w * n + i, sizeof f);
#pragma unroll
        for (int e = 0; e < V; e++) s[e] += f[e];
    }
    const long long e = i < n ? i : i - n, row = e / cols, col = e - row * cols;
    T v[V];
#pragma unroll
    for (int k = 0; k < V; k++) v[k] = from_f32<T>(s[k]);
    __builtin_memcpy((i < n ? o0 + row * s0 : o1 + row * s1) + col * (long long)sizeof(T), v, sizeof v);
}

// Bias gradients: the waves' column sums, 32 columns x 32 lanes a block.
__global__ __launch_bounds__(1024) void ff_db_fold_kernel(const float* part, long long rows, int N, float* dg, float* dv) {
    __shared__ double red[32][33];
    const int c = blockIdx.x * 32 + threadIdx.x % 32, lane = threadIdx.x / 32;
    double s = 0.0;
    if (c < 2 * N) {
#pragma unroll 8
        for (long long r = lane; r < rows; r += 32) s += (double)part[r * 2 * N + c];
    }
    red[lane][threadIdx.x % 32] = s;
    __syncthreads();
    if (lane || c >= 2 * N) return;
    for (int i = 1; i < 32; i++) s += red[i][threadIdx.x];
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

bool aligned_rows(const void* p, long long stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 16 == 0 && stride < (1 << 23); }

constexpr int kFew = 64;
constexpr long long kMaxWidth = 1 << 20, kMaxTokens = 1 << 30;   // of K and N; of the tokens (row indexes of tiles fit 32 bits)
constexpr int kCus = 256;                                         // of an MI355X: plans are made without a device at hand

// How a product is run: its tile and the number of parts of its reduction, by the least estimated time.
// A step of a tile takes time in proportion to its area, the larger tiles' at a better rate (the
// measured ones of a long reduction); a part ends in an epilogue and a fold. Measured, bf16, 48,060 tokens,
// K 384, N 1,536: FORWARD Large 143, Medium 156, Small 182 us (113 GFLOP: 790 TFLOP/s); GRAD Medium 299; DX
// Large 350, Medium 281 (328 with two blocks a CU), Small 305; DW Medium in 10 parts 227, in 7 on two blocks a CU
// 249. fp32, 1,344 tokens, K 512, N 2,048: DX Small 44 (split, with 6 of the fold) where
// Medium takes 48 and an unsplit one 157; DW 43 (and 6), 47 and 59.
struct Plan {
    int tile, splits, part;              // 0 Large, 1 Medium, 2 Small; parts, steps of a part
};
long long steps_of(Mode mode, long long r, int size) { return std::max(1LL, (r + step_of(mode, size) - 1) / step_of(mode, size)); }
Plan plan_of(Mode mode, long long J, long long M, long long steps, stx_type type) {
    struct Kind {
        int tj, tm;
        double rate[2];                  // relative rate, 16-bit and fp32
    };
    static constexpr Kind kinds[] = {{256, 256, {1.0, 1.0}}, {128, 128, {0.86, 0.96}}, {128, 64, {0.62, 0.85}}};
    static constexpr double alone[3][3] = {{1, 1, 1}, {0.6, 1, 1}, {0.4, 0.75, 1}};   // of 1, 2, 3 blocks on a CU that holds 1, 2, 3
    const bool gated = mode == FORWARD || mode == GRAD;
    const int size = type_size(type);
    const int w = mode == DW ? 2 : 1;
    Plan best{};
    double least = 0;
    // Large has no registers for GRAD's epilogue (460 us where Medium took 250), nor for operands that are split.
    for (int k = mode == GRAD || splits(mode, type) ? 1 : 0; k < 3; k++) {
        const Kind& c = kinds[k];
        const int slots = slots_of(k, mode, type);
        const long long tiles = (J * (gated ? 2 : 1) + c.tj - 1) / c.tj * ((M + c.tm - 1) / c.tm) * w;
        const double area = c.tj * (double)c.tm / 65536, step = area / c.rate[size == 4] * (size == 4 ? 5.5 : 0.95);   // us on a whole CU
        for (int s = 1; s <= (gated ? 1 : 32) && (s == 1 || steps / s >= 4); s++) {
            const long long part = (steps + s - 1) / s, items = tiles * ((steps + part - 1) / part), rest = items % (kCus * slots);
            const long long k_rest = (rest + kCus - 1) / kCus;
            const double busy = (double)(items / (kCus * slots)) * slots + (rest ? k_rest / alone[slots - 1][k_rest - 1] : 0.0);
            double us = busy * (part * step + 4.0 * area) + 2.0;
            if (s > 1) us += 4.0 + 8.0 * s * J * M * w / 4e6;
            if (least == 0 || us < least) {
                least = us;
                best = {k, (int)((steps + part - 1) / part), (int)part};
            }
        }
    }
    return best;
}

template <class T, int MODE, class C, bool AL>
void launch_tiles(FfArgs a, int parts, hipStream_t stream) {
    const int width = MODE == FORWARD || MODE == GRAD ? C::TJ / 2 : C::TJ;
    a.jtiles = (a.J + width - 1) / width;
    const long long tiles = (long long)a.jtiles * (((long long)a.M + C::TM - 1) / C::TM);
    if (tiles * parts >= (1LL << 30)) fail(STX_STATUS_UNSUPPORTED, "gated_ff: too many tiles");
    a.tiles = (int)tiles;
    a.items = (int)(tiles * parts);
    const long long blocks = std::min<long long>(a.items, (long long)device_cus() * C::template slots<T, MODE>);
    hipLaunchKernelGGL((ff_kernel<T, MODE, C, AL>), dim3(xcd_grid(blocks)), dim3(C::NT), 0, stream, a);
    launch_check("ff_kernel");
}

// What goes through registers has no Large tile.
template <class T, int MODE>
void launch_ff(const FfArgs& a, bool aligned, int tile, int parts, hipStream_t stream) {
    if constexpr (splits((Mode)MODE, type_of<T>)) return tile == 2 ? launch_tiles<T, MODE, Small, false>(a, parts, stream) : launch_tiles<T, MODE, Medium, false>(a, parts, stream);
    else if (!aligned) tile == 2 ? launch_tiles<T, MODE, Small, false>(a, parts, stream) : launch_tiles<T, MODE, Medium, false>(a, parts, stream);
    else if (MODE != GRAD && tile == 0) launch_tiles<T, MODE == GRAD ? FORWARD : MODE, Large, true>(a, parts, stream);
    else if (tile == 1) launch_tiles<T, MODE, Medium, true>(a, parts, stream);
    else launch_tiles<T, MODE, Small, true>(a, parts, stream);
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

FfArgs products(const Block& b, const float* bg, const float* bv, stx_act act, int size) {
    FfArgs k{};
    k.p[0] = b.wg.data;
    k.p[1] = b.wv.data;
    k.ps[0] = b.wg.stride;
    k.ps[1] = b.wv.stride;
    k.q[0] = b.x.data;
    k.qs[0] = b.x.stride;
    k.J = b.N;
    k.M = (int)b.M;
    k.RP = k.RQ = b.K;
    k.steps = (int)steps_of(FORWARD, b.K, size);
    k.jpad = b.N;
    k.b[0] = bg;
    k.b[1] = bv;
    k.act = act;
    return k;
}
bool products_aligned(const Block& b, int size) {
    return b.K % (16 / size) == 0 && aligned_rows(b.x.data, b.x.stride) && aligned_rows(b.wg.data, b.wg.stride) && aligned_rows(b.wv.data, b.wv.stride);
}

// Workspace of the backward pass: dg and dv with rows of a multiple of 64 elements (of 16-bit data the
// high parts and the low ones of each), the parts of split reductions, the biases' column sums (for the smallest tile's waves).
struct BackPlan {
    long long Np;
    Plan grad, dx, dw;
    size_t dg, part, db, total;
};
// Rows of column sums that GRAD writes with a tile: one a wave along the tokens, of whole tiles.
template <class C>
long long sum_rows(long long M) { return (M + C::TM - 1) / C::TM * C::WM; }
BackPlan back_plan(long long M, long long K, long long N, stx_type type) {
    BackPlan p{};
    const int size = type_size(type);
    p.Np = pad64(N);
    p.grad = plan_of(GRAD, N, M, steps_of(GRAD, K, size), type);
    p.dx = plan_of(DX, K, M, 2 * steps_of(DX, N, size), type);
    p.dw = plan_of(DW, K, N, steps_of(DW, M, size), type);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += pad256(bytes);
        return here;
    };
    p.dg = take(2 * (size_t)(M * p.Np) * sizeof(float));
    // One after another, in the same place: the products run in one stream.
    const size_t dx = p.dx.splits > 1 ? (size_t)p.dx.splits * M * K : 0, dw = p.dw.splits > 1 ? (size_t)p.dw.splits * 2 * N * K : 0;
    p.part = take(std::max(dx, dw) * sizeof(float));
    p.db = take((size_t)std::max(sum_rows<Medium>(M), sum_rows<Small>(M)) * 2 * N * sizeof(float));
    p.total = at;
    return p;
}

template <class T>
void fold(const float* part, int splits, long long rows, int cols, int w, char* o0, char* o1, long long s0, long long s1, hipStream_t stream) {
    const long long n = rows * cols * w;
    auto launch = [&](auto v) {
        constexpr int V = v();
        launch_all((n / V + 255) / 256, [&](dim3 grid, unsigned first) {
            hipLaunchKernelGGL((ff_fold_kernel<T, V>), grid, dim3(256), 0, stream, part, splits, rows, cols, w, o0, o1, s0, s1, first);
            launch_check("ff_fold_kernel");
        });
    };
    STX_REQUIRE(n / 256 < (1LL << 31), "gated_ff_back: gradients too large");
    if (cols % 4 == 0) launch(std::integral_constant<int, 4>{});
    else launch(std::integral_constant<int, 1>{});
}

template <class T>
void run_back(const Block& b, const Rows& dh, const float* bg, const float* bv, stx_act act, const Rows* dx, const Rows* dwg, const Rows* dwv,
              float* dbg, float* dbv, char* ws, hipStream_t stream) {
    constexpr int size = sizeof(T);
    const BackPlan p = back_plan(b.M, b.K, b.N, type_of<T>);
    char* dg = ws + p.dg;
    char* dv = dg + b.M * p.Np * (long long)sizeof(float);
    const long long plane = b.M * p.Np * 2;
    float* part = reinterpret_cast<float*>(ws + p.part);
    float* db = reinterpret_cast<float*>(ws + p.db);
    const bool aligned = products_aligned(b, size);
    if (b.M > 0) {
        FfArgs k = products(b, bg, bv, act, size);
        k.dh = dh.data;
        k.dhs = dh.stride;
        k.out[0] = dx || dwg ? dg : nullptr;
        k.out[1] = dv;
        k.os[0] = k.os[1] = p.Np * size;
        k.jpad = (int)p.Np;
        k.plane = plane;
        k.part = dbg || dbv ? db : nullptr;
        launch_ff<T, GRAD>(k, aligned, p.grad.tile, 1, stream);
    }
    if (dbg || dbv) {
        const long long rows = b.M == 0 ? 0 : p.grad.tile == 2 ? sum_rows<Small>(b.M) : sum_rows<Medium>(b.M);
        hipLaunchKernelGGL(ff_db_fold_kernel, dim3((2 * b.N + 31) / 32), dim3(1024), 0, stream, db, rows, b.N, dbg, dbv);
        launch_check("ff_db_fold_kernel");
    }
    if (dx && b.M > 0) {
        FfArgs k{};
        k.p[0] = b.wg.data;
        k.p[1] = b.wv.data;
        k.ps[0] = b.wg.stride;
        k.ps[1] = b.wv.stride;
        k.q[0] = dg;
        k.q[1] = dv;
        k.qs[0] = k.qs[1] = p.Np * size;
        k.J = k.jpad = b.K;
        k.M = (int)b.M;
        k.RP = b.N;
        k.RQ = p.Np;
        k.steps = (int)steps_of(DX, b.N, size);
        k.plane = plane;
        k.chunk = p.dx.part;
        k.out[0] = dx->data;
        k.os[0] = dx->stride;
        k.part = p.dx.splits > 1 ? part : nullptr;
        launch_ff<T, DX>(k, aligned, p.dx.tile, p.dx.splits, stream);
        if (k.part) fold<T>(part, p.dx.splits, b.M, b.K, 1, dx->data, dx->data, dx->stride, dx->stride, stream);
    }
    if (dwg && b.M > 0) {
        FfArgs k{};
        k.p[0] = b.x.data;
        k.ps[0] = b.x.stride;
        k.q[0] = dg;
        k.q[1] = dv;
        k.qs[0] = k.qs[1] = p.Np * size;
        k.J = k.jpad = b.K;
        k.M = b.N;
        k.qpad = (int)p.Np;
        k.RP = k.RQ = b.M;
        k.steps = (int)steps_of(DW, b.M, size);
        k.plane = plane;
        k.chunk = p.dw.part;
        k.out[0] = dwg->data;
        k.out[1] = dwv->data;
        k.os[0] = dwg->stride;
        k.os[1] = dwv->stride;
        k.part = p.dw.splits > 1 ? part : nullptr;
        launch_ff<T, DW>(k, aligned, p.dw.tile, 2 * p.dw.splits, stream);
    }
    if (dwg && (p.dw.splits > 1 || b.M == 0))                        // without tokens: sums of no parts
        fold<T>(part, b.M > 0 ? p.dw.splits : 0, b.N, b.K, 2, dwg->data, dwv->data, dwg->stride, dwv->stride, stream);
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
        const size_t floats = (size_t)b.N * sizeof(float);
        check_apart("gated_ff", {{"dst", dst, size}},
                    {{"x", x, size}, {"w_gate", w_gate, size}, {"w_value", w_value, size}, {"b_gate", b_gate, floats}, {"b_value", b_value, floats}});
        if (b.M == 0) return;
        FfArgs k = products(b, b_gate, b_value, act, size);
        k.out[0] = d.data;
        k.os[0] = d.stride;
        with_type(type, [&](auto t) {
            using T = decltype(t);
            if (b.M > kFew)
                return launch_ff<T, FORWARD>(k, products_aligned(b, size), plan_of(FORWARD, b.N, b.M, k.steps, type).tile, 1, as_stream(stream));
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
        (void)type_size(type);
        STX_REQUIRE(n_tokens >= 0 && n_tokens <= kMaxTokens && n_in > 0 && n_in <= kMaxWidth && n_hidden > 0 && n_hidden <= kMaxWidth,
                    "gated_ff_back_workspace_size: %lld tokens, K = %lld, N = %lld", (long long)n_tokens, (long long)n_in, (long long)n_hidden);
        bytes = back_plan(n_tokens, n_in, n_hidden, type).total;
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
        }
        const size_t need = back_plan(b.M, b.K, b.N, type).total, floats = (size_t)b.N * sizeof(float);
        check_workspace(workspace, workspace_bytes, need, "gated_ff_back");
        check_apart("gated_ff_back",
                    {{"dx", dx, size}, {"dw_gate", dw_gate, size}, {"dw_value", dw_value, size}, {"db_gate", db_gate, floats}, {"db_value", db_value, floats},
                     {"the workspace", workspace, need}},
                    {{"dh", dh, size}, {"x", x, size}, {"w_gate", w_gate, size}, {"w_value", w_value, size}, {"b_gate", b_gate, floats}, {"b_value", b_value, floats}});
        if (!dx && !dw_gate && !db_gate && !db_value) return;
        with_type(type, [&](auto t) {
            run_back<decltype(t)>(b, h, b_gate, b_value, act, dx ? &rx : nullptr, dw_gate ? &rg : nullptr, dw_value ? &rv : nullptr, db_gate,
                                  db_value, static_cast<char*>(workspace), as_stream(stream));
        });
    });
}

}  // extern "C"

// diff_attention.hpp — differential attention: arguments, tiles in LDS and fragments shared by its forward
// and backward kernels (diff_attention.hip, diff_attention_back.hip), and its checks.
#pragma once

#include <algorithm>
#include <cmath>

#include "mfma.hpp"

namespace stx {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kDiffDim = 128, kDiffValue = 256;          // largest rows of q and k, and of v

// Queries that share a key head are the rows of one problem: row r of (sequence b, key head) is query
// r / group of head (key head) * group + r % group. Their limits (keys seen) never fall.
struct Strided {
    const char* p;
    long long s1, s2, s3;                // byte strides: heads, tokens, sequences
};
struct DiffArgs {
    Strided q, k, v, out, second, dy, dq, dk, dv;    // dy: the gradient of out
    const float* lam;                    // [heads]
    float* lse;                          // [sequence][head][map][query]
    float* dots;                         // backward: dy . o of each map, laid out as lse
    double* tiles_lam;                   // backward: a block's shares of lambda's gradient, [block][group]
    const float* most;                   // fp16's backward: largest |v| of a tile of keys, [sequence][key head][tile],
    float* loud;                         // and largest |dy| max(1, |lambda|) of a wave's rows, [sequence][key head][loud_count]
    int loud_rows, loud_count;
    float* part;                         // split keys (forward) or rows (keys' gradients)
    float* part_stat;
    const int *lengths, *starts;
    int queries, keys, rows;             // rows: queries * group
    int dim, vdim;
    int kv_heads, group, heads;
    FastDiv group_div, kv_div, tile_div; // row -> query; (sequence, key head); block -> (that, tile)
    int tiles, splits;                   // tiles of rows or keys; parts of the other axis
    bool causal;
    float scale;
};

// A sequence's masks.
struct Mask {
    int length;                          // keys that a query sees are below it
    long long start;
    bool causal;
    __device__ __forceinline__ Mask(const DiffArgs& a, int b) : causal(a.causal) {
        length = a.lengths ? min(max(a.lengths[b], 0), a.keys) : a.keys;
        start = a.starts ? a.starts[b] : 0;
        if (causal) length = (int)min((long long)length, max(0LL, start + a.queries));
    }
    __device__ __forceinline__ int limit(int query) const { return causal ? (int)min((long long)length, max(0LL, query + start + 1)) : length; }
};

// A tile in LDS: rows of W elements in 16-byte chunks, chunk c of row r at c ^ turn(r). Fragments read 16
// rows of a chunk at once (plain), or 16-bit columns by the transposing read, 8 rows of 32 bytes at once,
// or 32-bit columns, 4 rows (4 apart) of 64 bytes: each meets every bank once.
template <class T, int W>
struct Tile {
    static constexpr int BYTES = W * sizeof(T), CHUNKS = BYTES / 16, E = 16 / sizeof(T), GROUPS = CHUNKS / 4;   // groups: of 4 chunks, one product each
    static constexpr int KEYS = sizeof(T) == 2 ? 32 : 16;                          // rows of a transposed fragment
    static __device__ __forceinline__ int turn(int r) {
        constexpr int R = BYTES >= 256 ? 1 : 256 / BYTES;
        if constexpr (sizeof(T) == 2) return (2 * (r / R % (8 / R)) + r / 8 % 2) % CHUNKS;
        else return r / R % (CHUNKS < 16 ? CHUNKS : 16);
    }
    static __device__ __forceinline__ u32x4 plain(const char* lds, int row0, int group, int lane) {
        const int r = row0 + lane % 16;
        return *reinterpret_cast<const u32x4*>(lds + r * BYTES + ((group * 4 + lane / 16) ^ turn(r)) * 16);
    }
    // Column lane % 16 of columns 16 i ..: rows row0 + 4 (lane / 16) + 0 .. 3, of 16-bit data those 16 further too.
    static __device__ __forceinline__ u32x4 columns(const char* lds, int row0, int i, int lane) {
        const int s = lane % 16, q = lane / 16;
        u32x4 f;
        if constexpr (sizeof(T) == 2) {
            s16x4 h[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int r = row0 + e * 16 + 4 * q + s / 4;
                const char* at = lds + r * BYTES + ((2 * i + s % 4 / 2) ^ turn(r)) * 16 + s % 2 * 8;
                h[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
            }
            __builtin_memcpy(&f, h, 16);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int r = row0 + 4 * q + e;
                f[e] = *reinterpret_cast<const unsigned*>(lds + r * BYTES + ((4 * i + s / 4) ^ turn(r)) * 16 + s % 4 * 4);
            }
        }
        return f;
    }
};

// The chunks that a thread brings of MAPS tiles of ROWS rows, straight to LDS (ALIGNED; `lds` is an address there) or
// through registers.
template <class T, int W, int ROWS, int MAPS, int NT, bool ALIGNED>
struct Loader {
    using L = Tile<T, W>;
    static constexpr int N = MAPS * ROWS * L::CHUNKS / NT, BYTES = MAPS * ROWS * L::BYTES;
    static_assert(MAPS * ROWS * L::CHUNKS % NT == 0);
    static constexpr int STEP = NT / L::CHUNKS, PERIOD = STEP % 16 == 0 ? 1 : 16 / STEP;   // rows from a chunk to the thread's next; chunks until turn() repeats
    static_assert(NT % L::CHUNKS == 0);
    u32x4 hold[ALIGNED ? 1 : N];
    unsigned off[ALIGNED ? PERIOD : 1];  // of the thread's first chunks in a tile of evenly spaced rows
    static __device__ __forceinline__ unsigned wave_start() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64 * 1024); }
    __device__ __forceinline__ void space(long long stride, long long map) {
        if constexpr (ALIGNED) {
#pragma unroll
            for (int i = 0; i < PERIOD; i++) {
                const int r = i * STEP + (int)threadIdx.x / L::CHUNKS;
                off[i] = (unsigned)(r / ROWS * map + r % ROWS * stride) + (((int)threadIdx.x % L::CHUNKS) ^ L::turn(r)) * 16;
            }
        }
    }
    // The whole tile that starts at p, rows `stride` apart, maps `map` apart: a scalar base and one offset a load (with
    // rows one by one, the addresses took a sixth of the forward kernel's instructions). Rows have W elements.
    __device__ __forceinline__ void fetch_whole(unsigned lds, const char* p, long long stride, long long map) {
        if constexpr (ALIGNED) {
            const unsigned to = lds + wave_start();
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int r = i / PERIOD * PERIOD * STEP;
                load_to_lds(p + r / ROWS * map + r % ROWS * stride, off[i % PERIOD], to + i * NT * 16);
            }
        }
    }
    // row(map, r): a row's start, or NULL for one of zeros. `width` elements exist.
    // (Tiles in a sequence's end, and rows that LDS pads.)
    template <class F>
    __device__ __forceinline__ void fetch(unsigned lds, int width, F&& row) {
        const int tid = threadIdx.x;
        const unsigned to = lds + wave_start();
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int e = i * NT + tid, r = e / L::CHUNKS, c = (e % L::CHUNKS) ^ L::turn(r % ROWS);
            const char* p = row(r / ROWS, r % ROWS);
            if constexpr (ALIGNED) load_to_lds(p && c * L::E < width ? (const void*)(p + c * 16) : (const void*)&zero_chunk, to + i * NT * 16);
            else hold[i] = load_chunk<T>(p ? p + c * 16 : nullptr, p ? width - c * L::E : 0);
        }
    }
    __device__ __forceinline__ void settle(char* lds) {
        if constexpr (!ALIGNED) {
#pragma unroll
            for (int i = 0; i < N; i++) *reinterpret_cast<u32x4*>(lds + (i * NT + (int)threadIdx.x) * 16) = hold[i];
        }
    }
};
template <bool ALIGNED>
__device__ __forceinline__ void arrived() {
    if constexpr (ALIGNED) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// Over the four lanes (16 apart) that hold a column of an accumulator.
__device__ __forceinline__ float column_sum(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ float column_max(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Accumulators of KEYS rows (two tiles of 16 for 16-bit data, one for fp32) as a chunk of the next product.
template <class T>
__device__ __forceinline__ u32x4 chunk_of(const f32x4* acc) {
    u32x4 f;
    if constexpr (sizeof(T) == 4) {
        f = __builtin_bit_cast(u32x4, acc[0]);
    } else {
        typedef T Pair __attribute__((ext_vector_type(2)));           // converted together, to nearest even
        typedef float Floats __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int e = 0; e < 4; e++) f[e] = __builtin_bit_cast(unsigned, __builtin_convertvector((Floats{acc[e / 2][e % 2 * 2], acc[e / 2][e % 2 * 2 + 1]}), Pair));
    }
    return f;
}

template <class T>
__device__ __forceinline__ void unpack(u32x4 f, float (&v)[16 / sizeof(T)]) {
    T t[16 / sizeof(T)];
    __builtin_memcpy(t, &f, 16);
#pragma unroll
    for (int e = 0; e < 16 / (int)sizeof(T); e++) v[e] = to_f32(t[e]);
}
// What rounding to chunk f (16-bit data) left of them, rounded.
template <class T>
__device__ __forceinline__ u32x4 rest_of(const f32x4* acc, u32x4 f) {
    float v[16 / sizeof(T)];
    unpack<T>(f, v);
    f32x4 r[2];
#pragma unroll
    for (int e = 0; e < 16 / (int)sizeof(T); e++) r[e / 4][e % 4] = acc[e / 4][e % 4] - v[e];
    return chunk_of<T>(r);
}

// A row's chunks as a fragment in registers: lane l's row, chunk (l / 16) + 4 group.
template <class T, int W>
__device__ __forceinline__ void load_fragments(u32x4* f, const char* p, int width, int lane) {
#pragma unroll
    for (int g = 0; g < Tile<T, W>::GROUPS; g++) {
        const int c = g * 4 + lane / 16;
        f[g] = load_chunk<T>(p + c * 16, p ? width - c * Tile<T, W>::E : 0);
    }
}

// Row r of (sequence b, key head kvh).
struct RowAt {
    int query, head;
    __device__ __forceinline__ RowAt(const DiffArgs& a, int kvh, int r) {
        query = (int)a.group_div.div((unsigned)r);
        head = kvh * a.group + (r - query * a.group);
    }
    __device__ __forceinline__ const char* at(const Strided& t, int b, int per_head, int map) const {
        return t.p + (long long)(head * per_head + map) * t.s1 + query * t.s2 + b * t.s3;
    }
    __device__ __forceinline__ long long stat(const DiffArgs& a, int b, int map) const {
        return (((long long)b * a.heads + head) * 2 + map) * a.queries + query;
    }
};

// --------------------------------------------------------------------------------- host
struct DiffShape {
    long long B, M, N;
    int H, Hk, D, V;
    bool empty() const { return B == 0 || M == 0 || H == 0; }
};

// q [D, 2 H, M, B], k [D, 2 Hk, N, B], v [V, Hk, N, B].
inline DiffShape diff_shape(const stx_tensor* q, const stx_tensor* k, const stx_tensor* v, const char* op) {
    STX_REQUIRE(q->ne[1] % 2 == 0 && k->ne[1] % 2 == 0, "%s: q and k have two heads for each of the output's", op);
    const long long H = q->ne[1] / 2, Hk = k->ne[1] / 2;
    STX_REQUIRE(k->ne[0] == q->ne[0] && k->ne[3] == q->ne[3], "%s: q and k differ in head size or batch", op);
    STX_REQUIRE(v->ne[1] == Hk && v->ne[2] == k->ne[2] && v->ne[3] == k->ne[3], "%s: v's heads, keys or batch differ from k's", op);
    STX_REQUIRE(q->ne[0] > 0 && v->ne[0] > 0, "%s: rows of no elements", op);
    if (q->ne[0] > kDiffDim || v->ne[0] > kDiffValue)
        fail(STX_STATUS_UNSUPPORTED, "%s: heads of %lld and %lld elements (%d and %d at most)", op, (long long)q->ne[0], (long long)v->ne[0], kDiffDim, kDiffValue);
    STX_REQUIRE(Hk > 0 ? H > 0 && H % Hk == 0 : H == 0, "%s: %lld heads do not share %lld key heads evenly", op, H, Hk);
    STX_REQUIRE(q->ne[2] < (1LL << 28) && k->ne[2] < (1LL << 28) && q->ne[3] < (1LL << 20) && H < (1 << 16), "%s: more than 2^28 queries or keys, 2^20 sequences or 2^16 heads", op);
    STX_REQUIRE(Hk == 0 || q->ne[2] * (H / Hk) < (1LL << 30), "%s: more than 2^30 queries to a key head", op);
    return {q->ne[3], q->ne[2], k->ne[2], (int)H, (int)Hk, (int)q->ne[0], (int)v->ne[0]};
}

inline void check_out_rows(const stx_tensor* t, long long ne0, long long ne1, long long ne2, long long ne3, int size, const char* what) {
    check_typed(t, size, what);
    const long long want[4] = {ne0, ne1, ne2, ne3};
    for (int i = 0; i < 4; i++) STX_REQUIRE(t->ne[i] == want[i], "%s has ne[%d] = %lld, not %lld", what, i, (long long)t->ne[i], want[i]);
}
inline void check_nested(const stx_tensor* t, int size, const char* what) {
    STX_REQUIRE(nelem(view(t)) == 0 || nested(t, size), "%s: rows of the output overlap", what);
}

inline Strided strided(const stx_tensor* t) {
    return t ? Strided{static_cast<const char*>(t->data), t->nb[1], t->nb[2], t->nb[3]} : Strided{};
}
inline bool rows_in_chunks(const stx_tensor* t, int size) {
    bool ok = reinterpret_cast<uintptr_t>(t->data) % 16 == 0 && t->ne[0] * size % 16 == 0;
    for (int i = 1; i < 4; i++) ok = ok && (t->ne[i] <= 1 || t->nb[i] % 16 == 0);
    return ok && (t->ne[1] <= 1 || t->nb[1] < (1 << 23)) && (t->ne[2] <= 1 || t->nb[2] < (1 << 23));   // offsets in a tile fit 31 bits
}

inline DiffArgs diff_args(const DiffShape& s, const stx_tensor* q, const stx_tensor* k, const stx_tensor* v, const float* lam, float scale, int causal,
                          const int32_t* lengths, const int32_t* starts) {
    DiffArgs a{};
    a.q = strided(q), a.k = strided(k), a.v = strided(v);
    a.lam = lam;
    a.lengths = lengths, a.starts = starts;
    a.queries = (int)s.M, a.keys = (int)s.N;
    a.group = s.H / s.Hk;
    a.rows = (int)(s.M * a.group);
    a.dim = s.D, a.vdim = s.V;
    a.kv_heads = s.Hk, a.heads = s.H;
    a.group_div = FastDiv((unsigned)a.group);
    a.kv_div = FastDiv((unsigned)s.Hk);
    a.causal = causal != 0;
    a.scale = scale;
    return a;
}
inline void check_scale(float scale, const char* op) { STX_REQUIRE(std::isfinite(scale) && scale > 0.f, "%s: scale must be finite and positive", op); }

// Calls f(DP, VP): the smallest sizes of rows in LDS that hold D and V.
template <class F>
void with_dims(int D, int V, F&& f) {
    using std::integral_constant;
    if (D <= 32 && V <= 64) f(integral_constant<int, 32>{}, integral_constant<int, 64>{});
    else if (D <= 64 && V <= 64) f(integral_constant<int, 64>{}, integral_constant<int, 64>{});
    else if (D <= 64 && V <= 128) f(integral_constant<int, 64>{}, integral_constant<int, 128>{});
    else if (V <= 128) f(integral_constant<int, 128>{}, integral_constant<int, 128>{});
    else f(integral_constant<int, 128>{}, integral_constant<int, 256>{});
}

}  // namespace
}  // namespace stx

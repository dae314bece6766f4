// mfma.hpp — the matrix instructions over 16-byte chunks and the loads that feed them (gated_ff.hip,
// diff_attention*.hip).
#pragma once

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

typedef short s16x4 __attribute__((ext_vector_type(4)));

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

}  // namespace
}  // namespace stx

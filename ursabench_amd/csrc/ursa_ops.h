// ursa_ops.h — what the K15 - K17 launches (ursa_linear.hip, ursa_norm.hip) share: 16-byte pieces of fp32 / bf16 / fp16 rows
// at any alignment, and the 8-bit form of an activation (K17).
#ifndef URSA_OPS_H
#define URSA_OPS_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ursa_hip.h"

namespace ursa {

typedef __bf16 bf16;
typedef _Float16 f16;

template <typename T> struct Piece { static constexpr int kN = 16 / (int)sizeof(T); };    // elements of a 16-byte piece

// N elements of a row from `p`, of which the first `valid` exist (the rest read as 0). Rows of an odd length start at any multiple
// of the element size: the hardware takes 16-byte accesses at such addresses, so a whole piece is one load there too.
template <typename T, int N>
__device__ __forceinline__ void load_piece(const T* __restrict__ p, int64_t valid, float (&v)[N]) {
    if (valid >= N) {
        T t[N];
        __builtin_memcpy(t, p, sizeof t);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)t[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < valid ? (float)p[i] : 0.f;
    }
}

template <typename T, int N>
__device__ __forceinline__ void store_piece(T* __restrict__ p, int64_t valid, const float (&v)[N]) {
    if (valid >= N) {
        T t[N];
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = (T)v[i];
        __builtin_memcpy(p, t, sizeof t);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < valid) p[i] = (T)v[i];
    }
}

// ---- K17: 32 features of a row share the power of two 2^e; a value is q 2^e, |q| <= 127 -------------------------------------
constexpr int kBlock8 = 32;
constexpr int kNonFinite8 = 127;        // the exponent byte of a block with an infinity or a NaN in it: it reads as NaN

__device__ __forceinline__ float pow2_bits(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }   // -126 <= e <= 127

// the exponent byte of a block from the largest |v| in it, as its bits (integers compare like the magnitudes, NaN above all).
// Largest magnitude m 2^k, 1/2 <= m < 1: e = k - 7, so the largest |q| is in [64, 128] and saturates at 127: off by at most half a
// step below 127.5 and by less than one step above. Least e: -126 (2^-126 is normal); fp16 -24, its smallest step, so that q 2^e
// always is an fp16 number. (The largest is 121; 127 2^e is finite in every type that reached it.)
template <typename T>
__device__ __forceinline__ int exponent8(uint32_t top) {
    if (top >= 0x7f800000u) return kNonFinite8;
    const int e = (int)(top >> 23) - 126 - 7, least = sizeof(T) == 2 && __is_same(T, f16) ? -24 : -126;
    return e < least ? least : e;
}

__device__ __forceinline__ int quantise8(float v, int e) {
    if (e == kNonFinite8) return 0;
    return (int)fminf(fmaxf(rintf(v * pow2_bits(-e)), -127.f), 127.f);      // the product is exact: a power of two
}

__device__ __forceinline__ float value8(int q, int e) {
    return e == kNonFinite8 ? __builtin_nanf("") : (float)q * pow2_bits(e);
}

__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

inline int launch_status() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? URSA_OK : (int)e;
}

inline int64_t element_size(int32_t dtype) { return dtype == URSA_F32 ? 4 : 2; }

}  // namespace ursa

#endif

// lm_device.hpp -- device helpers of the language-model operators: element
// types, e4m3 codes, the two-factor roots, and the search for a block's or a
// token's sequence in an array of offsets.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mfft_internal.hpp"

namespace mfft {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <class E>
__device__ __forceinline__ float to_float(E v) {
    return (float)v;
}
template <class E>
__device__ __forceinline__ E from_float(float v) {
    return (E)v;  // to nearest, ties to even
}

// x w as complex values.  Which product is rounded first is written out, as the
// compiler otherwise chooses for each place: a query turned by the append would
// differ from one turned alone, and the append turns keys once for their page's
// scale and, where it cannot hold them, again for their codes, where one unit
// more in the last place would be past the largest code.
__device__ __forceinline__ float2 rotate_pair(float2 x, float2 w) {
    return make_float2(__builtin_fmaf(x.x, w.x, -(x.y * w.y)), __builtin_fmaf(x.y, w.x, x.x * w.y));
}

// The root of position p, pair j.  p < 0 or past the table: NaN, so that a
// position the plan does not hold shows in the output.
__device__ __forceinline__ float2 rotary_root(const RotaryTables& t, int64_t p, int j) {
    if (p < 0 || p >= t.max_positions) return make_float2(__builtin_nanf(""), __builtin_nanf(""));
    const float2 a = t.lo[(p & ((1 << kRotaryLoLog2) - 1)) * t.pairs + j];
    const float2 b = t.hi[(p >> kRotaryLoLog2) * t.pairs + j];
    return rotate_pair(a, b);
}

// Channels of pair e of a head: the rotated pairs first, then the rest two
// by two.
__device__ __forceinline__ void pair_channels(int layout, int pairs, int e, int& d0, int& d1) {
    if (e >= pairs || layout == MFFT_ROTARY_INTERLEAVED) {
        d0 = 2 * e;
        d1 = 2 * e + 1;
    } else {
        d0 = e;
        d1 = e + pairs;
    }
}

// Offsets as the kernels use them: within [0, tokens], NULL = one token each
// (`per` of them).
__device__ __forceinline__ int64_t seq_offset(const int32_t* offsets, int64_t per, int64_t tokens, int b) {
    const int64_t o = offsets ? (int64_t)offsets[b] : b * per;
    return o < 0 ? 0 : o > tokens ? tokens : o;
}

// The last sequence whose offset is at most t (binary search; offsets rise).
__device__ __forceinline__ int token_sequence(const int32_t* offsets, int64_t per, int64_t tokens, int sequences,
                                              int64_t t) {
    if (!offsets) return (int)(t / per);
    int lo = 0, hi = sequences - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (seq_offset(offsets, per, tokens, mid) <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// ---- e4m3 codes -------------------------------------------------------------
constexpr uint8_t kNaNCode = 0x7f;

// the e4m3 code of x, |x| <= 448, to nearest, ties to even; NaN for what is
// larger (only infinities and NaN are, a page's scale covers the rest)
__device__ __forceinline__ uint8_t to_code(float x) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false);
    return __builtin_fabsf(x) <= 448.0f ? (uint8_t)(w & 0xff) : kNaNCode;
}
__device__ __forceinline__ float from_code(uint8_t c) { return __builtin_amdgcn_cvt_f32_fp8((int)c, 0); }

// The least power of two 2^e with amax <= 448 * 2^e (448 = 1.75 * 2^8),
// e in [-126, 120], from amax's bits: amax finite and >= 0.
__device__ __forceinline__ float code_scale(float amax) {
    const uint32_t u = __float_as_uint(amax);
    int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffff) > 0x600000 ? 1 : 0);
    e = e < -126 ? -126 : e;
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// |x| where it is finite, else 0: what counts for a page's scale
__device__ __forceinline__ float finite_abs(float x) {
    const float a = __builtin_fabsf(x);
    return a <= 3.402823466e38f ? a : 0.0f;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) v = __builtin_fmaxf(v, __shfl_xor(v, s));
    return v;
}

}  // namespace mfft

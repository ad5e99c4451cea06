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

// A channel of rotate_pair in the element type.  In float16 the last fma and the
// conversion are one instruction, which rounds once; conversions of two
// neighbours at a time are not, and round twice, so each is kept by itself.
template <class E>
__device__ __forceinline__ E rounded_channel(float v) {
    E r = (E)v;
    if constexpr (__is_same(E, _Float16)) asm("" : "+v"(r));
    return r;
}

// A position as the tables are indexed: kNoPosition if the plan does not hold it.
constexpr uint32_t kNoPosition = 0xffffffff;
__device__ __forceinline__ uint32_t held_position(const RotaryTables& t, int64_t p) {
    return (uint64_t)p < (uint64_t)t.max_positions ? (uint32_t)p : kNoPosition;
}

// The root of a held position, pair j; NaN of one that is not, so that it shows
// in the output.  Loaded whatever the position is: a branch around a load ends
// in a wait for it, and a thread needs roots of several positions at once.  (32
// bits hold both tables' indexes: 2^24 positions, 256 pairs.)
__device__ __forceinline__ float2 held_root(const RotaryTables& t, uint32_t p, int j) {
    const uint32_t q = p == kNoPosition ? 0 : p, pairs = (uint32_t)t.pairs;
    const float2 a = t.lo[(q & ((1u << kRotaryLoLog2) - 1)) * pairs + (uint32_t)j];
    const float2 b = t.hi[(q >> kRotaryLoLog2) * pairs + (uint32_t)j];
    const float2 z = rotate_pair(a, b);
    return p == kNoPosition ? make_float2(__builtin_nanf(""), __builtin_nanf("")) : z;
}
// The same of one position for all of a thread's pairs: one branch for them.
__device__ __forceinline__ float2 rotary_root(const RotaryTables& t, int64_t p, int j) {
    if (p < 0 || p >= t.max_positions) return make_float2(__builtin_nanf(""), __builtin_nanf(""));
    const float2 a = t.lo[(p & ((1 << kRotaryLoLog2) - 1)) * t.pairs + j];
    const float2 b = t.hi[(p >> kRotaryLoLog2) * t.pairs + j];
    return rotate_pair(a, b);
}

__device__ __forceinline__ int64_t position(const void* p, int32_t wide, int64_t at) {
    return wide ? ((const int64_t*)p)[at] : ((const int32_t*)p)[at];
}
__device__ __forceinline__ int operator/(int x, Divisor d) { return (int)((uint64_t)(uint32_t)x * d.m >> d.shift); }

// The roots of C pairs of one token, from pair j on (C a power of two, j a
// multiple of it), each by its axis of the positions that stand from p[place]
// on.  (Positions are chosen by bits, not from an array, which would be one in LDS.)
template <int C>
struct AxisRoots {
    static_assert(MFFT_MAX_AXES == 4);
    const RotaryTables& t;
    uint64_t axis;  // a byte a pair
    uint32_t at0, to1, at2, to3;
    int j;
    __device__ __forceinline__ AxisRoots(const RotaryTables& t_, const void* p, int32_t wide, int64_t place,
                                         int64_t axis_stride, int j_) : t(t_), j(j_) {
        if constexpr (C == 8) axis = *(const uint64_t*)(t.axis + j);
        else if constexpr (C == 4) axis = *(const uint32_t*)(t.axis + j);
        else axis = t.axis[j];
        // (of axes there are not, the first's again: no branches)
        const int64_t s1 = t.axes > 1 ? place + axis_stride : place, s2 = t.axes > 2 ? place + 2 * axis_stride : place,
                      s3 = t.axes > 3 ? place + 3 * axis_stride : place;
        int64_t p0, p1, p2, p3;
        auto load = [&](auto* from) {
            p0 = from[place];
            p1 = from[s1];
            p2 = from[s2];
            p3 = from[s3];
        };
        if (wide) load((const int64_t*)p);
        else load((const int32_t*)p);
        at0 = held_position(t, p0);
        to1 = at0 ^ held_position(t, p1);
        at2 = held_position(t, p2);
        to3 = at2 ^ held_position(t, p3);
    }
    __device__ __forceinline__ float2 operator()(int x) const {
        const uint32_t a = (uint32_t)(axis >> (8 * x)), odd = 0u - (a & 1), high = 0u - (a >> 1 & 1);
        const uint32_t lo = at0 ^ (to1 & odd), hi = at2 ^ (to3 & odd);
        return held_root(t, lo ^ ((lo ^ hi) & high), j + x);
    }
};

// The roots of a workgroup's tokens, in LDS: a thread that takes C pairs of a
// head (a chunk) would load them in C pieces of eight bytes, every lane from
// lines of its own, and with few heads for each that is most of what the caches
// deliver.  Here neighbouring lanes load neighbouring pairs, once for all
// chunks and heads.  Root x of chunk c of token n is half x % 2 of
// ws[(x / 2) * 256 + n * stride + c]: a chunk's own pieces, as adjacent threads
// read them, are adjacent.  All 256 threads call it; tokens * stride <= 256,
// and stride chunks hold at least all pairs.  at(n, axis): a token's held position.
template <int C, class At>
__device__ __forceinline__ void stage_roots(const RotaryTables& t, float4* ws, int tokens, int stride, Divisor by_pairs,
                                            bool inverse, At&& at) {
    const int n = tokens * t.pairs;
    if (n <= 0) return;
    uint32_t p[C];
#pragma unroll
    for (int k = 0; k < C; ++k) {
        const int r = min((int)threadIdx.x + 256 * k, n - 1), tok = r / by_pairs;
        p[k] = at(tok, (int)t.axis[r - tok * t.pairs]);
    }
    float2 w[C];
#pragma unroll
    for (int k = 0; k < C; ++k) {
        const int r = min((int)threadIdx.x + 256 * k, n - 1), tok = r / by_pairs;
        w[k] = held_root(t, p[k], r - tok * t.pairs);
        if (inverse) w[k].y = -w[k].y;
    }
#pragma unroll
    for (int k = 0; k < C; ++k) {
        const int r = (int)threadIdx.x + 256 * k;
        if (r < n) {
            const int tok = r / by_pairs, j = r - tok * t.pairs;
            ((float2*)ws)[2 * (j % C / 2 * 256 + tok * stride + j / C) + j % 2] = w[k];
        }
    }
}
// a chunk's, of slot n * stride + c
template <int C>
__device__ __forceinline__ void staged_roots(const float4* ws, int slot, float2 (&w)[C]) {
#pragma unroll
    for (int x = 0; x < C; x += 2) {
        const float4 v = ws[x / 2 * 256 + slot];
        w[x] = make_float2(v.x, v.y);
        w[x + 1] = make_float2(v.z, v.w);
    }
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

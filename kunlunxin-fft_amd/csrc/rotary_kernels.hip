// rotary_kernels.hip -- rotary positions: pairs of a head's channels, as
// complex values, times m exp(i p theta_j) for the token's position p
// (MFFT_INVERSE: the conjugate roots, which is the gradient).  A pair (a, b)
// becomes (a c - b s, b c + a s); channels past the pairs are copied.
// Bound: one read and one write of the tensor.  bf16, 8192 tokens of 32 heads
// of 128 channels, 134 MB: 29 us, 4.6 TB/s (a pair a thread: 73 us); float32,
// 100003 tokens of 8 heads of 96, 614 MB: 111 us, 5.5 TB/s (209 us).
#include <algorithm>
#include <type_traits>

#include "lm_device.hpp"

namespace mfft {
namespace {

// One thread per (token, head, pair), any strides, alignment and sizes.  (Which
// axis turns a pair is one more load before its position's, so plans of one are
// a kernel of their own: 8856 tokens of 56 heads of 96 in float16 84 us, not 90.)
template <class E, bool AXES>
__global__ __launch_bounds__(256) void rotary_pair_kernel(RotaryTables t, mfft_rotary_args a, int64_t axis_stride,
                                                          uint32_t half_dim, uint32_t total) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= total) return;
    const uint32_t e = i % half_dim, th = i / half_dim;
    const uint32_t h = th % (uint32_t)a.heads, bt = th / (uint32_t)a.heads;
    const uint32_t n = bt % (uint32_t)a.tokens, b = bt / (uint32_t)a.tokens;
    const int64_t po = b * a.position_strides[0] + n * a.position_strides[1];
    int d0, d1;
    pair_channels(t.layout, t.pairs, (int)e, d0, d1);
    const E* x = (const E*)a.in + b * a.in_strides[0] + n * a.in_strides[1] + h * a.in_strides[2];
    E* y = (E*)a.out + b * a.out_strides[0] + n * a.out_strides[1] + h * a.out_strides[2];
    E va = x[d0], vb = x[d1];
    if ((int)e < t.pairs) {
        float2 w = rotary_root(t, position(a.positions, a.positions_64, AXES ? po + t.axis[e] * axis_stride : po), (int)e);
        if (a.direction == MFFT_INVERSE) w.y = -w.y;
        const float2 z = rotate_pair({to_float(va), to_float(vb)}, w);
        va = rounded_channel<E>(z.x);
        vb = rounded_channel<E>(z.y);
    }
    y[d0] = va;
    y[d1] = vb;
}

// Sixteen bytes at a time: a chunk is V = 16 bytes' worth of pairs (V / 2 where
// pairs lie side by side), which two loads (one) of a head take; a thread holds
// its chunk's roots and applies them to `heads` heads of one token, so that a
// token's roots are loaded and multiplied once for them.  Channels past the
// pairs are chunks of 2 V (V) copied.
template <class E, bool HALF>
__global__ __launch_bounds__(256) void rotary_chunk_kernel(RotaryTables t, mfft_rotary_args a, uint32_t chunks,
                                                           uint32_t total, int heads) {
    constexpr int V = 16 / sizeof(E), C = HALF ? V : V / 2;  // elements of a load, pairs of a chunk
    struct alignas(16) Vec {
        E e[V];
    };
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= total) return;
    const uint32_t c = i % chunks, bt = i / chunks;
    const uint32_t n = bt % (uint32_t)a.tokens, b = bt / (uint32_t)a.tokens;
    const bool turned = (int)c * C < t.pairs;
    // first channels of the chunk's two (one) loads
    const int d0 = !HALF || !turned ? (int)c * (HALF ? 2 * V : V) : (int)c * C;
    const int d1 = turned ? d0 + t.pairs : d0 + V;
    float2 w[C];
    if (turned) {
        const int64_t po = b * a.position_strides[0] + n * a.position_strides[1];
        const int64_t p = position(a.positions, a.positions_64, po);
#pragma unroll
        for (int x = 0; x < C; ++x) {
            w[x] = rotary_root(t, p, (int)c * C + x);
            if (a.direction == MFFT_INVERSE) w[x].y = -w[x].y;
        }
    }
    const int h0 = blockIdx.y * heads, h1 = h0 + heads < a.heads ? h0 + heads : a.heads;
    const E* x = (const E*)a.in + b * a.in_strides[0] + n * a.in_strides[1] + h0 * a.in_strides[2];
    E* y = (E*)a.out + b * a.out_strides[0] + n * a.out_strides[1] + h0 * a.out_strides[2];
    auto turn = [&](Vec& u, Vec& v) {
        if (!turned) return;
#pragma unroll
        for (int k = 0; k < C; ++k) {
            E& ea = HALF ? u.e[k] : u.e[2 * k];
            E& eb = HALF ? v.e[k] : u.e[2 * k + 1];
            const float2 z = rotate_pair({to_float(ea), to_float(eb)}, w[k]);
            ea = rounded_channel<E>(z.x);
            eb = rounded_channel<E>(z.y);
        }
    };
    int h = h0;
    // four heads' loads before their stores (in and out may be one tensor, so
    // the compiler keeps the order written)
    for (; h + 4 <= h1; h += 4) {
        Vec u[4], v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            u[k] = *(const Vec*)(x + k * a.in_strides[2] + d0);
            if constexpr (HALF) v[k] = *(const Vec*)(x + k * a.in_strides[2] + d1);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            turn(u[k], v[k]);
            *(Vec*)(y + k * a.out_strides[2] + d0) = u[k];
            if constexpr (HALF) *(Vec*)(y + k * a.out_strides[2] + d1) = v[k];
        }
        x += 4 * a.in_strides[2];
        y += 4 * a.out_strides[2];
    }
    for (; h < h1; ++h, x += a.in_strides[2], y += a.out_strides[2]) {
        Vec u = *(const Vec*)(x + d0), v;
        if constexpr (HALF) v = *(const Vec*)(x + d1);
        turn(u, v);
        *(Vec*)(y + d0) = u;
        if constexpr (HALF) *(Vec*)(y + d1) = v;
    }
}

// The same of positions with several axes, where a chunk's roots lie in rows of
// their own: the workgroup makes its tokens' roots together.  Roots loaded by
// each thread as above: 1024 tokens of 40 heads of 128 21 us, so 9.3 (plain
// positions 7.5, and 9.3 made together, as they take one more round of loads);
// 50001 of 16 heads of 64 in float32 97 and 85 us (4.8 TB/s).  V is 16 bytes of
// elements, or 4 (8 where neighbours are pairs or E is float) where pairs,
// strides or addresses keep no more: 2142 tokens of 49 heads of 128 of which 20
// channels are turned, 14.9 us, neighbouring pairs 12.4 (a pair a thread: 30.7).
template <class E, bool HALF, int V>
__global__ __launch_bounds__(256) void rotary_axes_kernel(RotaryTables t, mfft_rotary_args a, int64_t axis_stride,
                                                           int chunks, int tokens, Divisor by_pairs, int heads) {
    constexpr int C = HALF ? V : V / 2;  // V: elements of a load; pairs of a chunk
    typedef uint32_t Words __attribute__((ext_vector_type(V * sizeof(E) / 4)));
    typedef typename std::conditional<V * sizeof(E) == 4, uint32_t, Words>::type Held;
    union Vec {
        E e[V];
        Held w;
    };
    __shared__ float4 ws[C / 2 * 256];
    // tokens of all batches, one after the other: this workgroup's first, how many
    // it has, and this thread's (a thread past the last takes the last again, and
    // stores nothing)
    const uint32_t first = blockIdx.x * (uint32_t)tokens, all = (uint32_t)(a.batch * a.tokens);
    const int count = (int)min((uint32_t)tokens, all - first);
    const int mine = (int)threadIdx.x / chunks, c = (int)threadIdx.x - mine * chunks, tok = min(mine, count - 1);
    auto place = [&](int tok, int64_t& b, int64_t& n) {
        n = first + (uint32_t)tok;
        b = 0;
        if (a.batch > 1) {
            b = (uint32_t)n / (uint32_t)a.tokens;
            n -= b * a.tokens;
        }
    };
    int64_t b, n;
    place(tok, b, n);
    const bool turned = c * C < t.pairs;
    // first channels of the chunk's two (one) loads
    const int d0 = !HALF || !turned ? c * (HALF ? 2 * V : V) : c * C;
    const int d1 = turned ? d0 + t.pairs : d0 + V;
    const int h0 = blockIdx.y * heads, h1 = h0 + heads < a.heads ? h0 + heads : a.heads;
    const E* x = (const E*)a.in + b * a.in_strides[0] + n * a.in_strides[1] + h0 * a.in_strides[2];
    E* y = (E*)a.out + b * a.out_strides[0] + n * a.out_strides[1] + h0 * a.out_strides[2];
    // four heads' loads before their stores (in and out may be one tensor, so the
    // compiler keeps the order written), the first four's before the roots, which
    // are two loads one after the other
    Vec u[4], v[4];
    auto load = [&] {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            u[k] = *(const Vec*)(x + k * a.in_strides[2] + d0);
            if constexpr (HALF) v[k] = *(const Vec*)(x + k * a.in_strides[2] + d1);
        }
    };
    int h = h0;
    if (h + 4 <= h1) load();
    stage_roots<C>(t, ws, count, chunks, by_pairs, a.direction == MFFT_INVERSE, [&](int tok, int axis) {
        int64_t b, n;
        place(tok, b, n);
        return held_position(t, position(a.positions, a.positions_64,
                                         b * a.position_strides[0] + n * a.position_strides[1] + axis * axis_stride));
    });
    __syncthreads();
    if (mine >= count) return;
    float2 w[C];
    if (turned) staged_roots<C>(ws, mine * chunks + c, w);
    // (here they are first used: the compiler otherwise converts them, and so waits
    // for them, before it asks for positions and roots)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        asm volatile("" : "+v"(u[k].w));
        if constexpr (HALF) asm volatile("" : "+v"(v[k].w));
    }
    auto turn = [&](Vec& u, Vec& v) {
        if (!turned) return;
#pragma unroll
        for (int k = 0; k < C; ++k) {
            E& ea = HALF ? u.e[k] : u.e[2 * k];
            E& eb = HALF ? v.e[k] : u.e[2 * k + 1];
            const float2 z = rotate_pair({to_float(ea), to_float(eb)}, w[k]);
            ea = rounded_channel<E>(z.x);
            eb = rounded_channel<E>(z.y);
        }
    };
    for (; h + 4 <= h1; h += 4) {
        if (h > h0) load();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            turn(u[k], v[k]);
            *(Vec*)(y + k * a.out_strides[2] + d0) = u[k];
            if constexpr (HALF) *(Vec*)(y + k * a.out_strides[2] + d1) = v[k];
        }
        x += 4 * a.in_strides[2];
        y += 4 * a.out_strides[2];
    }
    for (; h < h1; ++h, x += a.in_strides[2], y += a.out_strides[2]) {
        Vec u = *(const Vec*)(x + d0), v;
        if constexpr (HALF) v = *(const Vec*)(x + d1);
        turn(u, v);
        *(Vec*)(y + d0) = u;
        if constexpr (HALF) *(Vec*)(y + d1) = v;
    }
}

// Whether chunks hold whole loads of v elements, each of them aligned.
bool chunked(const RotaryTables& t, const mfft_rotary_args& a, int v) {
    const bool half = t.layout == MFFT_ROTARY_HALF;
    if (t.pairs % (half ? v : v / 2) || a.head_dim % (half ? 2 * v : v)) return false;
    if (t.axes > 1 && a.head_dim / (half ? 2 * v : v) > 256) return false;  // a workgroup has whole tokens
    if (((uintptr_t)a.in | (uintptr_t)a.out) & (v * (a.dtype == MFFT_F32 ? 4 : 2) - 1)) return false;
    for (int i = 0; i < 3; ++i)
        if (a.in_strides[i] % v || a.out_strides[i] % v) return false;
    return true;
}

// Heads a thread takes: all of them once tokens and chunks alone fill the chip
// (2^17 threads: two waves a SIMD), one while they do not.
int heads_a_thread(int64_t threads, int heads) {
    const int64_t slabs = (((int64_t)1 << 17) + threads - 1) / threads;
    const int least = heads / 65535 + 1;  // of a grid's second size
    return slabs >= heads ? least : std::max((int)((heads + slabs - 1) / slabs), least);
}

template <class E, bool HALF, int V>
void launch_axes(const RotaryTables& t, const mfft_rotary_args& a, int64_t axis_stride, hipStream_t s) {
    const int chunks = a.head_dim / (HALF ? 2 * V : V), tokens = 256 / chunks;
    const int64_t all = a.batch * a.tokens;
    const int heads = heads_a_thread(all * chunks, a.heads);
    const dim3 grid((uint32_t)((all + tokens - 1) / tokens), (uint32_t)((a.heads + heads - 1) / heads));
    rotary_axes_kernel<E, HALF, V><<<grid, 256, 0, s>>>(t, a, axis_stride, chunks, tokens, divisor(t.pairs), heads);
}

template <class E>
void launch_type(const RotaryTables& t, const mfft_rotary_args& a, int64_t axis_stride, hipStream_t s) {
    constexpr int V = 16 / sizeof(E);
    const bool half = t.layout == MFFT_ROTARY_HALF;
    if (t.axes > 1) {
        if (half && chunked(t, a, V)) return launch_axes<E, true, V>(t, a, axis_stride, s);
        if (half && chunked(t, a, 2)) return launch_axes<E, true, 2>(t, a, axis_stride, s);
        if (!half && chunked(t, a, V)) return launch_axes<E, false, V>(t, a, axis_stride, s);
        if constexpr (V > 4)
            if (!half && chunked(t, a, 4)) return launch_axes<E, false, 4>(t, a, axis_stride, s);
    } else if (chunked(t, a, V)) {
        const uint32_t chunks = (uint32_t)(a.head_dim / (half ? 2 * V : V));
        const uint32_t total = (uint32_t)(a.batch * a.tokens) * chunks;
        const int heads = heads_a_thread(total, a.heads);
        const uint32_t slabs = (uint32_t)((a.heads + heads - 1) / heads);
        const dim3 grid((uint32_t)(((uint64_t)total + 255) / 256), slabs);
        if (half) rotary_chunk_kernel<E, true><<<grid, 256, 0, s>>>(t, a, chunks, total, heads);
        else rotary_chunk_kernel<E, false><<<grid, 256, 0, s>>>(t, a, chunks, total, heads);
        return;
    }
    const uint32_t pairs = (uint32_t)a.head_dim / 2;
    const uint32_t total = (uint32_t)(a.batch * a.tokens * a.heads) * pairs;
    const uint32_t grid = (uint32_t)(((uint64_t)total + 255) / 256);
    if (t.axes > 1) rotary_pair_kernel<E, true><<<grid, 256, 0, s>>>(t, a, axis_stride, pairs, total);
    else rotary_pair_kernel<E, false><<<grid, 256, 0, s>>>(t, a, axis_stride, pairs, total);
}

}  // namespace

bool rotary_launch_fits(const RotaryTables&, const mfft_rotary_args& a) {
    const int64_t half = a.head_dim / 2;
    return a.batch <= (kMaxLaunchItems - 256) / a.heads / half / a.tokens;
}

hipError_t launch_rotary(const RotaryTables& t, const mfft_rotary_args& a, int64_t axis_stride, hipStream_t stream) {
    if (a.dtype == MFFT_F32) launch_type<float>(t, a, axis_stride, stream);
    else if (a.dtype == MFFT_F16) launch_type<_Float16>(t, a, axis_stride, stream);
    else launch_type<__bf16>(t, a, axis_stride, stream);
    mark(stream);
    return hipGetLastError();
}

}  // namespace mfft

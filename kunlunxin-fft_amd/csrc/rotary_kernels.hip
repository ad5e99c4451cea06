// rotary_kernels.hip -- rotary positions: pairs of a head's channels, as
// complex values, times m exp(i p theta_j) for the token's position p
// (MFFT_INVERSE: the conjugate roots, which is the gradient).  A pair (a, b)
// becomes (a c - b s, b c + a s); channels past the pairs are copied.
// Bound: one read and one write of the tensor.  bf16, 8192 tokens of 32 heads
// of 128 channels, 134 MB: 29 us, 4.6 TB/s (a pair a thread: 73 us); float32,
// 100003 tokens of 8 heads of 96, 614 MB: 111 us, 5.5 TB/s (209 us).
#include <algorithm>

#include "lm_device.hpp"

namespace mfft {
namespace {

// One thread per (token, head, pair), any strides, alignment and sizes.
template <class E>
__global__ __launch_bounds__(256) void rotary_pair_kernel(RotaryTables t, mfft_rotary_args a, uint32_t half_dim,
                                                          uint32_t total) {
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
        const int64_t p = a.positions_64 ? ((const int64_t*)a.positions)[po] : ((const int32_t*)a.positions)[po];
        float2 w = rotary_root(t, p, (int)e);
        if (a.direction == MFFT_INVERSE) w.y = -w.y;
        const float2 z = rotate_pair({to_float(va), to_float(vb)}, w);
        va = from_float<E>(z.x);
        vb = from_float<E>(z.y);
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
        const int64_t p = a.positions_64 ? ((const int64_t*)a.positions)[po] : ((const int32_t*)a.positions)[po];
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
            ea = from_float<E>(z.x);
            eb = from_float<E>(z.y);
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

// Whether every load and store of rotary_chunk_kernel is 16-byte aligned.
bool chunked(const RotaryTables& t, const mfft_rotary_args& a) {
    const int v = a.dtype == MFFT_F32 ? 4 : 8;
    const bool half = t.layout == MFFT_ROTARY_HALF;
    if (t.pairs % (half ? v : v / 2) || a.head_dim % (half ? 2 * v : v)) return false;
    if (((uintptr_t)a.in | (uintptr_t)a.out) & 15) return false;
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

template <class E>
void launch_type(const RotaryTables& t, const mfft_rotary_args& a, hipStream_t s) {
    if (chunked(t, a)) {
        const bool half = t.layout == MFFT_ROTARY_HALF;
        const uint32_t chunks = (uint32_t)(a.head_dim * sizeof(E) / (half ? 32 : 16));
        const uint32_t total = (uint32_t)(a.batch * a.tokens) * chunks;
        const int heads = heads_a_thread(total, a.heads);
        const dim3 grid((uint32_t)(((uint64_t)total + 255) / 256), (uint32_t)((a.heads + heads - 1) / heads));
        if (half) rotary_chunk_kernel<E, true><<<grid, 256, 0, s>>>(t, a, chunks, total, heads);
        else rotary_chunk_kernel<E, false><<<grid, 256, 0, s>>>(t, a, chunks, total, heads);
        return;
    }
    const uint32_t half = (uint32_t)a.head_dim / 2;
    const uint32_t total = (uint32_t)(a.batch * a.tokens * a.heads) * half;
    rotary_pair_kernel<E><<<(uint32_t)(((uint64_t)total + 255) / 256), 256, 0, s>>>(t, a, half, total);
}

}  // namespace

bool rotary_launch_fits(const RotaryTables&, const mfft_rotary_args& a) {
    const int64_t half = a.head_dim / 2;
    return a.batch <= (kMaxLaunchItems - 256) / a.heads / half / a.tokens;
}

hipError_t launch_rotary(const RotaryTables& t, const mfft_rotary_args& a, hipStream_t stream) {
    if (a.dtype == MFFT_F32) launch_type<float>(t, a, stream);
    else if (a.dtype == MFFT_F16) launch_type<_Float16>(t, a, stream);
    else launch_type<__bf16>(t, a, stream);
    mark(stream);
    return hipGetLastError();
}

}  // namespace mfft

// rotary_kernels.hip -- rotary positions: pairs of a head's channels, as
// complex values, times m exp(i p theta_j) for the token's position p
// (MFFT_INVERSE: the conjugate roots, which is the gradient).  A pair (a, b)
// becomes (a c - b s, b c + a s); channels past the pairs are copied.
// Bound: one read and one write of the tensor.
#include "lm_device.hpp"

namespace mfft {
namespace {

// One thread per (token, head, pair), any strides and sizes.
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
        const float fa = to_float(va), fb = to_float(vb);
        va = from_float<E>(fa * w.x - fb * w.y);
        vb = from_float<E>(fb * w.x + fa * w.y);
    }
    y[d0] = va;
    y[d1] = vb;
}

}  // namespace

bool rotary_launch_fits(const RotaryTables&, const mfft_rotary_args& a) {
    const int64_t half = a.head_dim / 2;
    return a.batch <= (kMaxLaunchItems - 256) / a.heads / half / a.tokens;
}

hipError_t launch_rotary(const RotaryTables& t, const mfft_rotary_args& a, hipStream_t stream) {
    const uint32_t half = (uint32_t)a.head_dim / 2;
    const uint32_t total = (uint32_t)(a.batch * a.tokens * a.heads) * half;
    const uint32_t grid = (uint32_t)(((uint64_t)total + 255) / 256);
    if (a.dtype == MFFT_F32)
        rotary_pair_kernel<float><<<grid, 256, 0, stream>>>(t, a, half, total);
    else if (a.dtype == MFFT_F16)
        rotary_pair_kernel<_Float16><<<grid, 256, 0, stream>>>(t, a, half, total);
    else
        rotary_pair_kernel<__bf16><<<grid, 256, 0, stream>>>(t, a, half, total);
    mark(stream);
    return hipGetLastError();
}

}  // namespace mfft

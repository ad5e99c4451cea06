// read_kernels.hip -- cached tokens read back: code * scale, rounded to the
// output's type (exact in float32 and bfloat16, as are codes whose scale is in
// float16's range).
#include "lm_device.hpp"

namespace mfft {
namespace {

// One thread per token, key head and channel.
template <class E>
__global__ __launch_bounds__(256) void read_kernel(mfft_cache c, mfft_read_args a, uint32_t total) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= total) return;
    const int D = c.head_dim, P = c.page_size;
    const int d = (int)(i % (uint32_t)D);
    const uint32_t nh = i / (uint32_t)D;
    const int h = (int)(nh % (uint32_t)c.kv_heads);
    const int64_t n = nh / (uint32_t)c.kv_heads, per = a.offsets ? 1 : a.tokens / a.sequences;
    E* k = (E*)a.k + n * a.k_strides[0] + h * a.k_strides[1] + d;
    E* v = (E*)a.v + n * a.v_strides[0] + h * a.v_strides[1] + d;
    const int b = token_sequence(a.offsets, per, a.tokens, a.sequences, n);
    const int64_t first = seq_offset(a.offsets, per, a.tokens, b);
    if (n < first || n >= seq_offset(a.offsets, per, a.tokens, b + 1)) {  // no sequence's
        *k = *v = (E)0.0f;
        return;
    }
    const int64_t at = a.starts[b] + (n - first), entry = at / P;
    const int slot = (int)(at % P);
    const int32_t page = at < 0 || entry >= a.table_width ? -1 : a.page_table[b * a.table_stride + entry];
    if (page < 0 || page >= c.pages) {
        *k = *v = (E)__builtin_nanf("");
        return;
    }
    const int64_t ph = (int64_t)page * c.kv_heads + h;
    *k = from_float<E>(from_code(((const uint8_t*)c.k)[(ph * P + slot) * D + d]) * c.k_scale[ph]);
    *v = from_float<E>(from_code(((const uint8_t*)c.v)[(ph * P + (slot & ~15)) * D + 16 * d + (slot & 15)]) * c.v_scale[ph]);
}

template <class E>
void launch_type(const mfft_cache& c, const mfft_read_args& a, hipStream_t s) {
    const uint32_t total = (uint32_t)(a.tokens * c.kv_heads * c.head_dim);
    read_kernel<E><<<(uint32_t)(((uint64_t)total + 255) / 256), 256, 0, s>>>(c, a, total);
}

}  // namespace

bool read_launch_fits(const mfft_cache& c, const mfft_read_args& a) {
    return a.tokens <= (kMaxLaunchItems - 256) / c.kv_heads / c.head_dim;
}

hipError_t launch_read(const mfft_cache& c, const mfft_read_args& a, hipStream_t stream) {
    if (a.dtype == MFFT_F32) launch_type<float>(c, a, stream);
    else if (a.dtype == MFFT_F16) launch_type<_Float16>(c, a, stream);
    else launch_type<__bf16>(c, a, stream);
    mark(stream);
    return hipGetLastError();
}

}  // namespace mfft

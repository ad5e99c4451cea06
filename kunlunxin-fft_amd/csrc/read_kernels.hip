// read_kernels.hip -- cached tokens read back: code * scale, rounded once to the
// output's type.  Exact in float32 and bfloat16, but for codes of 256 and more
// under a scale of 2^120, which are infinite, and, in bfloat16, for scales below
// 2^-124, under which the least codes fall between its least steps.
//
// A thread takes sixteen tokens whose slots go together (a unit of a page's
// values) and eight channels of one head, of the keys or of the values: sixteen
// loads of eight bytes, or eight of sixteen bytes that its registers turn from
// channels to tokens, and a store of 16 bytes (32 in float32) a token.
// Neighbouring threads take the channels, then the heads: a token's outputs of
// one head are whole lines.
//
// Bound: codes read and outputs written once.  bf16, 131072 tokens of 8 heads of
// 128, 805 MB: 143 us, 5.6 TB/s (a value a thread: 786); with the values turned
// in LDS, so that a wave's loads are adjacent, 142.  The same in float32, 1342 MB:
// 416 us, 3.2 TB/s, where a thread's 32 bytes of a token are two stores and each
// store of a wave leaves every other 16 bytes out.
#include "lm_device.hpp"

namespace mfft {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kChannels = 8;

// Units of sixteen slots that a call's tokens can touch: sequence b owns those
// from offsets[b] / 16 + 2 b on (n / 16 rounded down, plus two).
__host__ __device__ inline int64_t read_units(const mfft_read_args& a) {
    return a.offsets ? a.tokens / 16 + 2 * (int64_t)a.sequences : a.sequences * (a.tokens / a.sequences / 16 + 2);
}

// eight values of one token
template <bool PAST, class E>
__device__ __forceinline__ void store(E* y, const float (&f)[kChannels]) {
    constexpr int V = 16 / sizeof(E);
    union {
        E e[V];
        u32x4 w;
    } u;
#pragma unroll
    for (int i = 0; i < kChannels; i += V) {
#pragma unroll
        for (int x = 0; x < V; ++x) u.e[x] = from_float<E>(f[i + x]);
        if constexpr (PAST) __builtin_nontemporal_store(u.w, (u32x4*)(y + i));
        else *(u32x4*)(y + i) = u.w;
    }
}

// PAST: outputs larger than the L2s go past them (143 us instead of 155, and of
// 216 MB 61 instead of 71); smaller ones stay there for who reads them next.
constexpr int64_t kL2Bytes = 32 << 20;
template <class E, bool PAST>
__global__ __launch_bounds__(256) void read_kernel(mfft_cache c, mfft_read_args a, uint32_t total, uint32_t blocks) {
    const bool values = blockIdx.y;
    E* const out = (E*)(values ? a.v : a.k);
    const int64_t s_token = values ? a.v_strides[0] : a.k_strides[0], s_head = values ? a.v_strides[1] : a.k_strides[1];
    const uint32_t chunks = (uint32_t)c.head_dim / kChannels, heads = (uint32_t)c.kv_heads;
    const float nothing[kChannels] = {};
    if (blockIdx.x >= blocks) {  // rows of no sequence
        const int64_t lo = seq_offset(a.offsets, 1, a.tokens, 0), hi = seq_offset(a.offsets, 1, a.tokens, a.sequences);
        const int64_t pieces = (lo + a.tokens - hi) * heads * chunks;
        for (int64_t i = (blockIdx.x - blocks) * 256 + threadIdx.x; i < pieces; i += (gridDim.x - blocks) * 256) {
            const int64_t nh = i / chunks, n = nh / heads;
            store<PAST>(out + (n < lo ? n : n + hi - lo) * s_token + nh % heads * s_head + i % chunks * kChannels, nothing);
        }
        return;
    }
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= total) return;
    const uint32_t ch = i % chunks, uh = i / chunks, h = uh % heads;
    const int64_t slot = uh / heads;

    // the sequence that owns this unit, and which tokens of the unit are the call's
    const int64_t per = a.offsets ? 1 : a.tokens / a.sequences;
    int b;
    int64_t first;
    if (a.offsets) {
        int lo = 0, hi = a.sequences - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (seq_offset(a.offsets, 1, a.tokens, mid) / 16 + 2 * (int64_t)mid <= slot) lo = mid;
            else hi = mid - 1;
        }
        b = lo;
        first = seq_offset(a.offsets, 1, a.tokens, b) / 16 + 2 * (int64_t)b;
    } else {
        b = (int)((uint32_t)slot / (uint32_t)(per / 16 + 2));
        first = b * (per / 16 + 2);
    }
    const int64_t row0 = seq_offset(a.offsets, per, a.tokens, b), n = seq_offset(a.offsets, per, a.tokens, b + 1) - row0;
    const int64_t start = a.starts[b], unit = (start >> 4) + (slot - first);
    // row of the unit's first token, if it were one, and the tokens that are
    const int64_t row = row0 + 16 * unit - start;
    const int t0 = (int)(start > 16 * unit ? start - 16 * unit : 0);
    const int t1 = (int)(start + n < 16 * unit + 16 ? start + n - 16 * unit : 16);
    if (t0 >= t1) return;
    E* y = out + row * s_token + h * s_head + ch * kChannels;

    const int units = c.page_size / 16, D = c.head_dim;
    const int64_t entry = unit / units;
    const int32_t page = unit < 0 || entry >= a.table_width ? -1 : a.page_table[b * a.table_stride + entry];
    if (page < 0 || page >= c.pages) {
        float f[kChannels];
#pragma unroll
        for (int x = 0; x < kChannels; ++x) f[x] = __builtin_nanf("");
        for (int t = t0; t < t1; ++t) store<PAST>(y + t * s_token, f);
        return;
    }
    const int64_t ph = (int64_t)page * c.kv_heads + h;
    const int64_t at = (ph * units + (unit - entry * units)) * 16 * D;
    auto tokens = [&](auto&& each) {
        if (t1 - t0 == 16) {
#pragma unroll
            for (int t = 0; t < 16; t += 2) each(t, true, true);
        } else {
#pragma unroll
            for (int t = 0; t < 16; t += 2) each(t, t >= t0 && t < t1, t + 1 >= t0 && t + 1 < t1);
        }
    };
    if (values) {
        const float scale = c.v_scale[ph];
        const uint8_t* v = (const uint8_t*)c.v + at + ch * kChannels * 16;
        u32x4 w[kChannels];
#pragma unroll
        for (int x = 0; x < kChannels; ++x) w[x] = *(const u32x4*)(v + 16 * x);
        tokens([&](int t, bool one, bool two) {
            float f[2][kChannels];
#pragma unroll
            for (int x = 0; x < kChannels; ++x) {
                const uint32_t word = w[x][t / 4];
                const f32x2 p = t % 4 ? __builtin_amdgcn_cvt_pk_f32_fp8((int)word, true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)word, false);
                f[0][x] = p[0] * scale;
                f[1][x] = p[1] * scale;
            }
            if (one) store<PAST>(y + t * s_token, f[0]);
            if (two) store<PAST>(y + (t + 1) * s_token, f[1]);
        });
    } else {
        const float scale = c.k_scale[ph];
        const uint8_t* k = (const uint8_t*)c.k + at + ch * kChannels;
        u32x2 w[16];
#pragma unroll
        for (int t = 0; t < 16; ++t) w[t] = *(const u32x2*)(k + t * D);
        tokens([&](int t, bool one, bool two) {
            float f[2][kChannels];
#pragma unroll
            for (int z = 0; z < 2; ++z)
#pragma unroll
                for (int x = 0; x < kChannels; x += 4) {
                    const f32x2 p = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[t + z][x / 4], false);
                    const f32x2 q = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[t + z][x / 4], true);
                    f[z][x] = p[0] * scale;
                    f[z][x + 1] = p[1] * scale;
                    f[z][x + 2] = q[0] * scale;
                    f[z][x + 3] = q[1] * scale;
                }
            if (one) store<PAST>(y + t * s_token, f[0]);
            if (two) store<PAST>(y + (t + 1) * s_token, f[1]);
        });
    }
}

// workgroups that only clear rows of no sequence
constexpr int kClear = 32;

template <class E>
void launch_type(const mfft_cache& c, const mfft_read_args& a, hipStream_t s) {
    const uint32_t total = (uint32_t)(read_units(a) * c.kv_heads * (c.head_dim / kChannels));
    const uint32_t blocks = (uint32_t)(((uint64_t)total + 255) / 256);
    const dim3 grid(blocks + (a.offsets ? kClear : 0), 2);
    if (2 * a.tokens * c.kv_heads * c.head_dim * (int64_t)sizeof(E) > kL2Bytes) read_kernel<E, true><<<grid, 256, 0, s>>>(c, a, total, blocks);
    else read_kernel<E, false><<<grid, 256, 0, s>>>(c, a, total, blocks);
}

}  // namespace

bool read_launch_fits(const mfft_cache& c, const mfft_read_args& a) {
    return read_units(a) <= (kMaxLaunchItems / 2 - 256 * (kClear + 1)) / c.kv_heads / (c.head_dim / kChannels);
}

hipError_t launch_read(const mfft_cache& c, const mfft_read_args& a, hipStream_t stream) {
    if (a.dtype == MFFT_F32) launch_type<float>(c, a, stream);
    else if (a.dtype == MFFT_F16) launch_type<_Float16>(c, a, stream);
    else launch_type<__bf16>(c, a, stream);
    mark(stream);
    return hipGetLastError();
}

}  // namespace mfft

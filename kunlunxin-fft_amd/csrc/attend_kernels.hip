// attend_kernels.hip -- attention over the paged 8-bit cache.
//
// One pass over the keys a row of queries sees, with a running maximum m and
// sum l of exponentials: for each 64 keys s = scale * K q, m' = max(m, s),
// p = 2^(s - m'), l = l 2^(m - m') + sum p, O = O 2^(m - m') + V p, and
// out = O / l at the end (s in units of log 2).
//
// Both products run on the matrix cores with queries as columns: S^T = K Q^T
// and O^T = V^T P^T, sixteen rows of queries (the query heads of one key head,
// and the tokens of one sequence) by 64 keys at a time, v_mfma 16x16x32.
// A lane l = 16 g + j holds, of D = A B, column j of rows 4 g .. 4 g + 3, and
// of A (B) the contraction indices 8 g .. 8 g + 7 of row (column) j.  Which key
// is which row of S^T is free, and it is chosen so that nothing moves between
// lanes: row i of the t-th of the four products is key 16 (i / 4) + 4 t + i % 4,
// so lane (j, g) gets the scores of keys 16 g .. 16 g + 15 of query row j, and
// those sixteen weights, in order, are its contraction indices of P^T.  V's
// codes of sixteen tokens of a channel are adjacent in the cache, so one
// 16-byte load a lane is the matching part of V^T.  m, l and the rescaling of
// O stay in column j: only the maximum crosses lanes (g), twice per 64 keys.
//
// Codes become the queries' type exactly (e4m3 fits both); V's power-of-two
// scale goes in with the conversion, K's into the 32-bit score.
#include "lm_device.hpp"
#include "mfft_device.hpp"

namespace mfft {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLowest = -1e30f;  // start of the running maximum: no score seen

// ---- the two query types ----------------------------------------------------
template <class E>
struct Mat;
template <>
struct Mat<__bf16> {
    typedef bf16x8 x8;
    typedef bf16x2 x2;
    static __device__ __forceinline__ f32x4 mfma(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    template <bool HI>
    static __device__ __forceinline__ x2 decode(uint32_t w, float scale) {
        return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI);
    }
};
template <>
struct Mat<_Float16> {
    typedef f16x8 x8;
    typedef f16x2 x2;
    static __device__ __forceinline__ f32x4 mfma(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    template <bool HI>
    static __device__ __forceinline__ x2 decode(uint32_t w, float scale) {
        return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI);
    }
};

// eight codes times a power-of-two scale
template <class E>
__device__ __forceinline__ typename Mat<E>::x8 decode8(uint32_t w0, uint32_t w1, float scale) {
    union {
        typename Mat<E>::x2 h[4];
        typename Mat<E>::x8 v;
    } u;
    u.h[0] = Mat<E>::template decode<false>(w0, scale);
    u.h[1] = Mat<E>::template decode<true>(w0, scale);
    u.h[2] = Mat<E>::template decode<false>(w1, scale);
    u.h[3] = Mat<E>::template decode<true>(w1, scale);
    return u.v;
}

// The head's channels as contraction indices: pairs of products cover 64
// channels (lane group g the sixteen from 16 g on, so that a load is 16
// bytes), and the last 32 of head_dim 96 one product (eight from 8 g on).
template <int D>
struct Dims {
    static constexpr int J = D / 64;         // 64-channel parts
    static constexpr bool REM = D % 64 != 0; // and one of 32
    static constexpr int KK = D / 32;        // products of 32 channels
    static constexpr int N = D / 16;         // 16-channel tiles of the output
};

// bytes [from, to) of a 16-byte unit kept, the others 0
__device__ __forceinline__ u32x4 keep_bytes(u32x4 w, int from, int to) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        int lo = from - 4 * i, hi = to - 4 * i;
        lo = lo < 0 ? 0 : lo > 4 ? 4 : lo;
        hi = hi < 0 ? 0 : hi > 4 ? 4 : hi;
        const uint64_t m = hi > lo ? (((uint64_t)1 << (8 * hi)) - 1) & ~(((uint64_t)1 << (8 * lo)) - 1) : 0;
        r[i] = w[i] & (uint32_t)m;
    }
    return r;
}

// 0x01 in each byte that is a NaN code
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return (((w & 0x7f7f7f7f) + 0x01010101) >> 7) & 0x01010101; }

// One workgroup: sixteen rows of one sequence and key head, its four waves on
// every fourth group of 64 keys; the waves' (m, l, O) are joined in LDS.
template <class E, int D>
__global__ __launch_bounds__(256) void attend_kernel(mfft_cache c, mfft_attend_args a, int group) {
    using M = Mat<E>;
    typedef typename M::x8 x8;
    using S = Dims<D>;
    const int H = c.kv_heads, P = c.page_size;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j = lane & 15, g = lane >> 4;
    const int kg = j >> 2, kr = j & 3;  // K rows of lane j: keys 16 kg + 4 t + kr

    // the sequence that owns this block of rows
    const int64_t slot = blockIdx.x / H;
    const int h = (int)(blockIdx.x % H);
    const int64_t per = a.offsets ? 1 : a.tokens / a.sequences;
    auto first_slot = [&](int b) { return seq_offset(a.offsets, per, a.tokens, b) * group / 16 + b; };
    int lo = 0, hi = a.sequences - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first_slot(mid) <= slot) lo = mid;
        else hi = mid - 1;
    }
    const int b = lo;
    const int64_t row0 = seq_offset(a.offsets, per, a.tokens, b);
    const int64_t n = seq_offset(a.offsets, per, a.tokens, b + 1) - row0;
    const int64_t block = (slot - first_slot(b)) * 16;
    if (block >= n * group) return;

    int64_t len = a.lengths[b];
    len = len < 0 ? 0 : len;
    const bool poison = len > (int64_t)a.table_width * P;
    if (poison) len = (int64_t)a.table_width * P;

    // this lane's query row (rows past the last repeat it and are not stored)
    int64_t r = block + j;
    const bool stored = r < n * group;
    if (!stored) r = n * group - 1;
    const int64_t tok = r / group;
    const int qh = h * group + (int)(r % group);
    const E* q = (const E*)a.q + (row0 + tok) * a.q_strides[0] + qh * a.q_strides[1];
    const int64_t pos = len - n + tok;
    int top = (int)(a.causal && pos + 1 < len ? pos + 1 : len);  // keys [low, top) are seen
    int low = (int)(a.window && pos + 1 > a.window ? pos + 1 - a.window : 0);
    if (top < low) top = low;

    // over all rows: the keys any row sees, and those all of them do
    int all_lo = low, all_hi = top, any_lo = low, any_hi = top;
#pragma unroll
    for (int s = 1; s < 16; s <<= 1) {
        all_lo = max(all_lo, __shfl_xor(all_lo, s));
        all_hi = min(all_hi, __shfl_xor(all_hi, s));
        any_lo = min(any_lo, __shfl_xor(any_lo, s));
        any_hi = max(any_hi, __shfl_xor(any_hi, s));
    }
    all_lo = __builtin_amdgcn_readfirstlane(all_lo);
    all_hi = __builtin_amdgcn_readfirstlane(all_hi);
    any_lo = __builtin_amdgcn_readfirstlane(any_lo);
    any_hi = __builtin_amdgcn_readfirstlane(any_hi);

    x8 qv[S::KK];
    static_for<0, S::J>([&](auto jj) {
        qv[2 * jj.value] = *(const x8*)(q + 64 * jj.value + 16 * g);
        qv[2 * jj.value + 1] = *(const x8*)(q + 64 * jj.value + 16 * g + 8);
    });
    if constexpr (S::REM) qv[S::KK - 1] = *(const x8*)(q + 64 * S::J + 8 * g);

    f32x4 o[S::N];
    static_for<0, S::N>([&](auto i) { o[i.value] = f32x4{0, 0, 0, 0}; });
    float m = kLowest, l = 0.0f;
    const float unit = a.scale * 1.44269504088896340736f;  // scores in units of log 2

    const int32_t* table = a.page_table + b * a.table_stride;
    const int64_t page_bytes = (int64_t)P * D;
    for (int64_t key0 = (any_lo / 64 + wave) * 64; key0 < any_hi; key0 += 256) {
        // K rows of this lane (page of 16 kg) and its scores' and V's keys (page of 16 g)
        const int64_t kk = key0 + 16 * kg, kv = key0 + 16 * g;
        int64_t kp = kk < len ? table[kk / P] : 0, vp = kv < len ? table[kv / P] : 0;
        const bool bad = vp < 0 || vp >= c.pages;
        kp = kp < 0 || kp >= c.pages ? 0 : kp;
        vp = bad ? 0 : vp;
        const uint8_t* kb = (const uint8_t*)c.k + (kp * H + h) * page_bytes + (int64_t)(kk % P + kr) * D;
        const uint8_t* vb = (const uint8_t*)c.v + (vp * H + h) * page_bytes + (int64_t)(kv % P) * D + 16 * j;
        const float cs = bad ? __builtin_nanf("") : unit * c.k_scale[vp * H + h];
        // past the end the page is a stand-in, whose scale must not count either
        const float vs = kv < len ? c.v_scale[vp * H + h] : 1.0f;

        f32x4 s[4];
        static_for<0, 4>([&](auto t) {
            const uint8_t* kt = kb + 4 * t.value * D;
            f32x4 acc = {0, 0, 0, 0};
            static_for<0, S::J>([&](auto jj) {
                const u32x4 w = *(const u32x4*)(kt + 64 * jj.value + 16 * g);
                acc = M::mfma(decode8<E>(w[0], w[1], 1.0f), qv[2 * jj.value], acc);
                acc = M::mfma(decode8<E>(w[2], w[3], 1.0f), qv[2 * jj.value + 1], acc);
            });
            if constexpr (S::REM) {
                const u32x2 w = *(const u32x2*)(kt + 64 * S::J + 8 * g);
                acc = M::mfma(decode8<E>(w[0], w[1], 1.0f), qv[S::KK - 1], acc);
            }
            s[t.value] = acc;
        });
        const bool edge = key0 < all_lo || key0 + 64 > all_hi;
        static_for<0, 16>([&](auto i) {
            float v = s[i.value / 4][i.value % 4] * cs;
            if (edge) {
                const int64_t key = kv + i.value;
                v = key >= low && key < top ? v : -__builtin_inff();
            }
            s[i.value / 4][i.value % 4] = v;
        });
        float mx = m;
        static_for<0, 16>([&](auto i) { mx = __builtin_fmaxf(mx, s[i.value / 4][i.value % 4]); });
        mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16));
        mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32));
        const float shrink = __builtin_amdgcn_exp2f(m - mx);
        m = mx;
        l *= shrink;
        static_for<0, S::N>([&](auto i) { o[i.value] *= shrink; });
        union {
            E e[16];
            x8 v[2];
        } p;
        static_for<0, 16>([&](auto i) {
            const float w = __builtin_amdgcn_exp2f(s[i.value / 4][i.value % 4] - m);
            l += w;
            p.e[i.value] = (E)w;
        });
        static_for<0, S::N>([&](auto i) {
            u32x4 w = *(const u32x4*)(vb + i.value * 256);
            if (edge) {
                // keys that no row sees may hold anything: their codes count as 0
                w = keep_bytes(w, (int)(any_lo - kv), (int)(any_hi - kv));
                uint32_t bad_codes = 0;
                u32x4 nan;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    nan[x] = nan_bytes(w[x]);
                    bad_codes |= nan[x];
                }
                if (__any(bad_codes != 0)) {
                    // a NaN value counts only for the rows that see its key: it
                    // leaves the product (0 * NaN is NaN), and is counted apart
                    x8 seen[2], is_nan[2];
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        seen[x / 8][x % 8] = (E)(kv + x >= low && kv + x < top ? 1.0f : 0.0f);
                        is_nan[x / 8][x % 8] = (E)(float)(nan[x / 4] >> (8 * (x % 4)) & 1);
                    }
                    f32x4 count = {0, 0, 0, 0};
                    count = M::mfma(is_nan[0], seen[0], count);
                    count = M::mfma(is_nan[1], seen[1], count);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        o[i.value][x] = count[x] > 0.0f ? __builtin_nanf("") : o[i.value][x];
                        w[x] &= ~(nan[x] * 0xffu);
                    }
                }
            }
            o[i.value] = M::mfma(decode8<E>(w[0], w[1], vs), p.v[0], o[i.value]);
            o[i.value] = M::mfma(decode8<E>(w[2], w[3], vs), p.v[1], o[i.value]);
        });
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // join the four waves: each writes its m, l and O, wave 0 adds them up
    __shared__ float sm[4][16], sl[4][16];
    __shared__ f32x4 so[3][S::N][64];
    if (lane < 16) {
        sm[wave][j] = m;
        sl[wave][j] = l;
    }
    if (wave > 0) static_for<0, S::N>([&](auto i) { so[wave - 1][i.value][lane] = o[i.value]; });
    __syncthreads();
    if (wave > 0) return;
    float mt = m;
    for (int w = 1; w < 4; ++w) mt = __builtin_fmaxf(mt, sm[w][j]);
    const float f0 = __builtin_amdgcn_exp2f(m - mt);
    l *= f0;
    static_for<0, S::N>([&](auto i) { o[i.value] *= f0; });
    for (int w = 1; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f(sm[w][j] - mt);
        l += sl[w][j] * f;
        static_for<0, S::N>([&](auto i) { o[i.value] += so[w - 1][i.value][lane] * f; });
    }
    if (!stored) return;
    float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (poison) inv = __builtin_nanf("");
    E* y = (E*)a.out + (row0 + tok) * a.out_strides[0] + qh * a.out_strides[1];
    static_for<0, S::N>([&](auto i) {
        union {
            E e[4];
            u32x2 w;
        } u;
#pragma unroll
        for (int x = 0; x < 4; ++x) u.e[x] = (E)(o[i.value][x] * inv);
        *(u32x2*)(y + 16 * i.value + 4 * g) = u.w;
    });
    if (a.lse && g == 0)
        a.lse[(row0 + tok) * a.q_heads + qh] =
            poison ? __builtin_nanf("") : l == 0.0f ? -__builtin_inff() : mt * 0.69314718055994530942f + __logf(l);
}

template <class E>
void launch_dim(const mfft_cache& c, const mfft_attend_args& a, int group, uint32_t grid, hipStream_t s) {
    switch (c.head_dim) {
        case 64: attend_kernel<E, 64><<<grid, 256, 0, s>>>(c, a, group); break;
        case 96: attend_kernel<E, 96><<<grid, 256, 0, s>>>(c, a, group); break;
        case 128: attend_kernel<E, 128><<<grid, 256, 0, s>>>(c, a, group); break;
        case 256: attend_kernel<E, 256><<<grid, 256, 0, s>>>(c, a, group); break;
    }
}

}  // namespace

bool attend_supported(int head_dim) { return head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 256; }

int64_t attend_workspace(const mfft_cache&, const mfft_attend_args&) { return 0; }

hipError_t launch_attend(const mfft_cache& c, const mfft_attend_args& a, hipStream_t stream) {
    const int group = a.q_heads / c.kv_heads;
    const int64_t blocks = (a.tokens * group / 16 + a.sequences) * c.kv_heads;
    if (!launch_fits(blocks, 256)) return hipErrorInvalidConfiguration;
    if (a.dtype == MFFT_F16)
        launch_dim<_Float16>(c, a, group, (uint32_t)blocks, stream);
    else
        launch_dim<__bf16>(c, a, group, (uint32_t)blocks, stream);
    mark(stream);
    return hipGetLastError();
}

}  // namespace mfft

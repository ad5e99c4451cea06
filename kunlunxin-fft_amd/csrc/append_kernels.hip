// append_kernels.hip -- new keys and values written to a paged 8-bit cache,
// keys (and the step's queries) rotated on the way.
//
// Page and head share one power-of-two scale, the least 2^e with every
// magnitude at most 448 * 2^e.  The scale only grows while a page fills, and
// then the codes it holds are multiplied by 2^(e_old - e_new): with three
// fraction bits at every size that is a change of the code's exponent, exact
// until a value falls below the smallest normal code, so a code is rounded
// once however often its page grows.  (A scale of 8-bit integers would round
// all of a page's codes again at every growth.)
//
// One workgroup takes one page and key head: all of this call's tokens in that
// page, found from the offsets alone, so that no two workgroups share a scale
// and no atomics are needed.  Sequence b owns the workgroups from
// offsets[b] / P + 2 b on, which are at least as many as the pages its tokens
// can touch (n / P rounded down, plus two).
#include "lm_device.hpp"

namespace mfft {
namespace {

struct AppendGrid {
    int64_t slots;       // page slots (workgroups = slots * kv_heads)
    int64_t kv_blocks;
    int64_t q_blocks;    // workgroups that rotate queries, after the others
};

__host__ __device__ inline AppendGrid append_grid(const mfft_cache& c, const mfft_append_args& a) {
    AppendGrid g;
    g.slots = a.offsets ? a.tokens / c.page_size + 2 * (int64_t)a.sequences : a.sequences;
    g.kv_blocks = g.slots * c.kv_heads;
    g.q_blocks = a.q ? (a.tokens * a.q_heads * (c.head_dim / 2) + 255) / 256 : 0;
    return g;
}

template <class E>
__device__ void rotate_query(const RotaryTables& t, const mfft_cache& c, const mfft_append_args& a, int64_t i) {
    const int half = c.head_dim / 2;
    const int e = (int)(i % half);
    const int64_t th = i / half;
    const int h = (int)(th % a.q_heads);
    const int64_t n = th / a.q_heads;
    if (n >= a.tokens) return;
    const int b = token_sequence(a.offsets, 1, a.tokens, a.sequences, n);
    const int64_t p = a.starts[b] + (n - seq_offset(a.offsets, 1, a.tokens, b));
    int d0, d1;
    pair_channels(t.layout, t.pairs, e, d0, d1);
    const E* x = (const E*)a.q + n * a.q_strides[0] + h * a.q_strides[1];
    E* y = (E*)a.q_out + n * a.q_out_strides[0] + h * a.q_out_strides[1];
    E va = x[d0], vb = x[d1];
    if (e < t.pairs) {
        const float2 w = rotary_root(t, p, e);
        const float fa = to_float(va), fb = to_float(vb);
        va = from_float<E>(fa * w.x - fb * w.y);
        vb = from_float<E>(fb * w.x + fa * w.y);
    }
    y[d0] = va;
    y[d1] = vb;
}

template <class E>
__global__ __launch_bounds__(256) void append_kernel(RotaryTables t, mfft_cache c, mfft_append_args a) {
    const AppendGrid grid = append_grid(c, a);
    if ((int64_t)blockIdx.x >= grid.kv_blocks) {
        rotate_query<E>(t, c, a, ((int64_t)blockIdx.x - grid.kv_blocks) * 256 + threadIdx.x);
        return;
    }
    const int64_t slot = blockIdx.x / c.kv_heads;
    const int h = (int)(blockIdx.x % c.kv_heads);
    const int P = c.page_size, D = c.head_dim, half = D / 2;

    // the sequence that owns this slot, its page and the tokens in it
    int b = (int)slot;
    int64_t first = slot;
    if (a.offsets) {
        int lo = 0, hi = a.sequences - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (seq_offset(a.offsets, 1, a.tokens, mid) / P + 2 * (int64_t)mid <= slot) lo = mid;
            else hi = mid - 1;
        }
        b = lo;
        first = seq_offset(a.offsets, 1, a.tokens, b) / P + 2 * (int64_t)b;
    }
    const int64_t row0 = seq_offset(a.offsets, 1, a.tokens, b);
    const int64_t n = seq_offset(a.offsets, 1, a.tokens, b + 1) - row0;
    const int64_t start = a.starts[b];
    if (start < 0 || n <= 0) return;
    const int64_t pg = start / P + (slot - first);
    const int64_t p0 = pg * P > start ? pg * P : start;
    const int64_t p1 = (pg + 1) * P < start + n ? (pg + 1) * P : start + n;
    if (p0 >= p1 || pg >= a.table_width) return;
    const int64_t page = a.page_table[b * a.table_stride + pg];
    if (page < 0 || page >= c.pages) return;
    const int o = (int)(p0 - pg * P);   // first slot written
    const int m = (int)(p1 - p0);       // tokens written
    const int64_t row = row0 + (p0 - start);

    const E* k = (const E*)a.k + row * a.k_strides[0] + h * a.k_strides[1];
    const E* v = (const E*)a.v + row * a.v_strides[0] + h * a.v_strides[1];
    uint8_t* kc = (uint8_t*)c.k + (page * c.kv_heads + h) * (int64_t)P * D;
    uint8_t* vc = (uint8_t*)c.v + (page * c.kv_heads + h) * (int64_t)P * D;

    auto rotated = [&](int i, int e, int& d0, int& d1) {
        pair_channels(t.layout, t.pairs, e, d0, d1);
        const float fa = to_float(k[i * a.k_strides[0] + d0]), fb = to_float(k[i * a.k_strides[0] + d1]);
        if (e >= t.pairs) return make_float2(fa, fb);
        const float2 w = rotary_root(t, p0 + i, e);
        return make_float2(fa * w.x - fb * w.y, fb * w.x + fa * w.y);
    };

    float mk = 0.0f, mv = 0.0f;
    for (int i = threadIdx.x; i < m * half; i += 256) {
        const int tok = i / half, e = i % half;
        int d0, d1;
        const float2 r = rotated(tok, e, d0, d1);
        mk = __builtin_fmaxf(mk, __builtin_fmaxf(finite_abs(r.x), finite_abs(r.y)));
        mv = __builtin_fmaxf(mv, __builtin_fmaxf(finite_abs(to_float(v[tok * a.v_strides[0] + 2 * e])),
                                                 finite_abs(to_float(v[tok * a.v_strides[0] + 2 * e + 1]))));
    }
    __shared__ float peak[2][4];
    mk = wave_max(mk);
    mv = wave_max(mv);
    if ((threadIdx.x & 63) == 0) {
        peak[0][threadIdx.x >> 6] = mk;
        peak[1][threadIdx.x >> 6] = mv;
    }
    float* ks = c.k_scale + page * c.kv_heads + h;
    float* vs = c.v_scale + page * c.kv_heads + h;
    const float k_old = o ? *ks : 0.0f, v_old = o ? *vs : 0.0f;
    __syncthreads();
    mk = __builtin_fmaxf(__builtin_fmaxf(peak[0][0], peak[0][1]), __builtin_fmaxf(peak[0][2], peak[0][3]));
    mv = __builtin_fmaxf(__builtin_fmaxf(peak[1][0], peak[1][1]), __builtin_fmaxf(peak[1][2], peak[1][3]));
    const float k_new = __builtin_fmaxf(code_scale(mk), k_old), v_new = __builtin_fmaxf(code_scale(mv), v_old);
    if (threadIdx.x == 0) {
        *ks = k_new;
        *vs = v_new;
    }
    // the page grew: its codes, before this call's are written
    if (o && (k_new > k_old || v_new > v_old)) {
        const float fk = k_old / k_new, fv = v_old / v_new;
        for (int i = threadIdx.x; i < P * D; i += 256) {
            kc[i] = to_code(from_code(kc[i]) * fk);
            vc[i] = to_code(from_code(vc[i]) * fv);
        }
        __syncthreads();
    }
    const float k_inv = 1.0f / k_new, v_inv = 1.0f / v_new;
    for (int i = threadIdx.x; i < m * half; i += 256) {
        const int tok = i / half, e = i % half;
        int d0, d1;
        const float2 r = rotated(tok, e, d0, d1);
        uint8_t* kr = kc + (int64_t)(o + tok) * D;
        kr[d0] = to_code(r.x * k_inv);
        kr[d1] = to_code(r.y * k_inv);
        const int s = o + tok;
        uint8_t* vr = vc + ((s >> 4) * D + 2 * e) * 16 + (s & 15);
        vr[0] = to_code(to_float(v[tok * a.v_strides[0] + 2 * e]) * v_inv);
        vr[16] = to_code(to_float(v[tok * a.v_strides[0] + 2 * e + 1]) * v_inv);
    }
}

}  // namespace

bool append_launch_fits(const RotaryTables&, const mfft_cache& c, const mfft_append_args& a) {
    const AppendGrid g = append_grid(c, a);
    return launch_fits(g.kv_blocks + g.q_blocks, 256);
}

hipError_t launch_append(const RotaryTables& t, const mfft_cache& c, const mfft_append_args& a, hipStream_t stream) {
    const AppendGrid g = append_grid(c, a);
    const uint32_t grid = (uint32_t)(g.kv_blocks + g.q_blocks);
    if (a.dtype == MFFT_F32)
        append_kernel<float><<<grid, 256, 0, stream>>>(t, c, a);
    else if (a.dtype == MFFT_F16)
        append_kernel<_Float16><<<grid, 256, 0, stream>>>(t, c, a);
    else
        append_kernel<__bf16><<<grid, 256, 0, stream>>>(t, c, a);
    mark(stream);
    return hipGetLastError();
}

}  // namespace mfft

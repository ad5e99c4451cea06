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
//
// Bound: the tokens read and the codes and rotated queries written once.  bf16,
// 32768 tokens of 8 key and 32 query heads of 128, 738 MB: 200 us, 3.7 TB/s;
// 256 sequences of one token, 6 MB: 9.6 us, where one sequence takes 4.8 with
// the same chain of loads: 64 of a workgroup's 256 threads have a pair of a key
// of 128 channels, and a page that grows is rescaled whole, filled or not.
#include "lm_device.hpp"

namespace mfft {
namespace {

struct AppendGrid {
    int64_t slots;       // page slots (workgroups = slots * kv_heads)
    int64_t kv_blocks;
    int64_t q_slabs;     // pieces the query heads come in
    int64_t q_blocks;    // workgroups that rotate queries, after the others
    int q_heads;         // heads of a piece
};

// Query heads a thread takes: sixteen, or as few as it takes to have 2^18
// threads (four waves on each of 1024 SIMDs).
constexpr int kQueryHeads = 16;

__host__ __device__ inline AppendGrid append_grid(const mfft_cache& c, const mfft_append_args& a, int v) {
    AppendGrid g;
    g.slots = a.offsets ? a.tokens / c.page_size + 2 * (int64_t)a.sequences : a.sequences;
    g.kv_blocks = g.slots * c.kv_heads;
    // v pairs (2 v channels) of a token and piece of the heads a thread
    const int64_t chunks = a.tokens * (c.head_dim / (2 * v));
    g.q_heads = 1;
    while (v > 1 && g.q_heads < kQueryHeads && g.q_heads < a.q_heads && chunks * a.q_heads > ((int64_t)1 << 18) * g.q_heads) g.q_heads *= 2;
    g.q_slabs = a.q ? (a.q_heads + g.q_heads - 1) / g.q_heads : 0;
    g.q_blocks = (chunks * g.q_slabs + 255) / 256;
    return g;
}

// Queries: thread i takes V pairs of a token and `grid.q_heads` of its heads.
template <class E, int V>
__device__ void rotate_query(const RotaryTables& t, const mfft_cache& c, const mfft_append_args& a, const AppendGrid& grid, int64_t at) {
    struct alignas(V * sizeof(E)) Vec {
        E e[V];
    };
    const int chunks = c.head_dim / (2 * V);
    const uint32_t i = (uint32_t)at;  // fewer than 2^32
    const int ch = (int)(i % chunks);
    const uint32_t ts = i / chunks;
    const int64_t n = ts / (uint32_t)grid.q_slabs;
    if (n >= a.tokens) return;
    const int h0 = (int)(ts % (uint32_t)grid.q_slabs) * grid.q_heads, h1 = min(h0 + grid.q_heads, a.q_heads);
    const int b = token_sequence(a.offsets, 1, a.tokens, a.sequences, n);
    const int64_t p = a.starts[b] + (n - seq_offset(a.offsets, 1, a.tokens, b));
    const bool turned = ch * V < t.pairs, half = t.layout == MFFT_ROTARY_HALF;
    const int d0 = turned && half ? ch * V : ch * 2 * V, d1 = turned && half ? d0 + t.pairs : d0 + V;
    float2 w[V];
    if (turned)
#pragma unroll
        for (int x = 0; x < V; ++x) w[x] = rotary_root(t, p, ch * V + x);
    const E* x = (const E*)a.q + n * a.q_strides[0] + h0 * a.q_strides[1];
    E* y = (E*)a.q_out + n * a.q_out_strides[0] + h0 * a.q_out_strides[1];
    auto turn = [&](Vec& u, Vec& v) {
        if (!turned) return;
        E f[2 * V];
#pragma unroll
        for (int z = 0; z < V; ++z) {
            f[z] = u.e[z];
            f[V + z] = v.e[z];
        }
#pragma unroll
        for (int z = 0; z < V; ++z) {
            const float fa = to_float(half ? f[z] : f[2 * z]), fb = to_float(half ? f[V + z] : f[2 * z + 1]);
            const float2 to = rotate_pair({fa, fb}, w[z]);
            const E ra = from_float<E>(to.x), rb = from_float<E>(to.y);
            if (half) {
                u.e[z] = ra;
                v.e[z] = rb;
            } else {
                (2 * z < V ? u.e[2 * z % V] : v.e[2 * z % V]) = ra;
                (2 * z + 1 < V ? u.e[(2 * z + 1) % V] : v.e[(2 * z + 1) % V]) = rb;
            }
        }
    };
    int h = h0;
    for (; h + 4 <= h1; h += 4) {  // four heads' loads before their stores
        Vec u[4], v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            u[k] = *(const Vec*)(x + k * a.q_strides[1] + d0);
            v[k] = *(const Vec*)(x + k * a.q_strides[1] + d1);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            turn(u[k], v[k]);
            *(Vec*)(y + k * a.q_out_strides[1] + d0) = u[k];
            *(Vec*)(y + k * a.q_out_strides[1] + d1) = v[k];
        }
        x += 4 * a.q_strides[1];
        y += 4 * a.q_out_strides[1];
    }
    for (; h < h1; ++h, x += a.q_strides[1], y += a.q_out_strides[1]) {
        Vec u = *(const Vec*)(x + d0), v = *(const Vec*)(x + d1);
        turn(u, v);
        *(Vec*)(y + d0) = u;
        *(Vec*)(y + d1) = v;
    }
}

// four codes times a factor
__device__ __forceinline__ uint32_t scale_codes(uint32_t w, float f) {
    uint32_t r = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) r |= (uint32_t)to_code(from_code((uint8_t)(w >> (8 * x))) * f) << (8 * x);
    return r;
}
// four values as to_code does each
__device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    uint32_t r = (uint32_t)w;
    r = __builtin_fabsf(a) <= 448.0f ? r : (r & 0xffffff00u) | kNaNCode;
    r = __builtin_fabsf(b) <= 448.0f ? r : (r & 0xffff00ffu) | (uint32_t)kNaNCode << 8;
    r = __builtin_fabsf(c) <= 448.0f ? r : (r & 0xff00ffffu) | (uint32_t)kNaNCode << 16;
    r = __builtin_fabsf(d) <= 448.0f ? r : (r & 0x00ffffffu) | (uint32_t)kNaNCode << 24;
    return r;
}

template <class E, bool WIDE>
__global__ __launch_bounds__(256) void append_kernel(RotaryTables t, mfft_cache c, mfft_append_args a) {
    constexpr int W = WIDE ? 16 / (int)sizeof(E) : 1;
    const AppendGrid grid = append_grid(c, a, W);
    if ((int64_t)blockIdx.x >= grid.kv_blocks) {
        rotate_query<E, W>(t, c, a, grid, ((int64_t)blockIdx.x - grid.kv_blocks) * 256 + threadIdx.x);
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

    __shared__ float peak[2][4];
    float* ks = c.k_scale + page * c.kv_heads + h;
    float* vs = c.v_scale + page * c.kv_heads + h;
    float k_new, v_new;
    // once each thread has its part of the largest magnitudes: the page's new
    // scales, and its codes made to fit them
    auto settle = [&](float mk, float mv) {
        const float k_old = o ? *ks : 0.0f, v_old = o ? *vs : 0.0f;
        mk = wave_max(mk);
        mv = wave_max(mv);
        if ((threadIdx.x & 63) == 0) {
            peak[0][threadIdx.x >> 6] = mk;
            peak[1][threadIdx.x >> 6] = mv;
        }
        __syncthreads();
        mk = __builtin_fmaxf(__builtin_fmaxf(peak[0][0], peak[0][1]), __builtin_fmaxf(peak[0][2], peak[0][3]));
        mv = __builtin_fmaxf(__builtin_fmaxf(peak[1][0], peak[1][1]), __builtin_fmaxf(peak[1][2], peak[1][3]));
        k_new = __builtin_fmaxf(code_scale(mk), k_old);
        v_new = __builtin_fmaxf(code_scale(mv), v_old);
        if (threadIdx.x == 0) {
            *ks = k_new;
            *vs = v_new;
        }
        if (o && (k_new > k_old || v_new > v_old)) {
            const float fk = k_old / k_new, fv = v_old / v_new;
            for (int i = threadIdx.x; i < P * D / 4; i += 256) {
                ((uint32_t*)kc)[i] = scale_codes(((uint32_t*)kc)[i], fk);
                ((uint32_t*)vc)[i] = scale_codes(((uint32_t*)vc)[i], fv);
            }
            __syncthreads();
        }
    };

    if constexpr (WIDE) {
        constexpr int V = 16 / sizeof(E);
        struct alignas(16) Vec {
            E e[V];
        };
        // K: a thread takes 2 V channels of one token (V pairs, or V and V more
        // past them) at a time, D / 2 V threads a token; kept in registers where
        // a page has at most four rounds of them
        const int half_chunks = D / (2 * V), rounds = (m * half_chunks + 255) / 256;
        constexpr int KEEP = 4;
        float held[KEEP][2 * V];
        auto channels = [&](int ch, int& d0, int& d1) {
            const bool turned = ch * V < t.pairs;
            if (turned && t.layout == MFFT_ROTARY_HALF) {
                d0 = ch * V;
                d1 = d0 + t.pairs;
            } else {
                d0 = ch * 2 * V;
                d1 = d0 + V;
            }
            return turned;
        };
        auto key = [&](int i, float (&f)[2 * V]) {
            const int tok = i / half_chunks, ch = i % half_chunks;
            int d0, d1;
            const bool turned = channels(ch, d0, d1);
            const Vec u = *(const Vec*)(k + tok * a.k_strides[0] + d0), w = *(const Vec*)(k + tok * a.k_strides[0] + d1);
#pragma unroll
            for (int x = 0; x < V; ++x) {
                f[x] = to_float(u.e[x]);
                f[V + x] = to_float(w.e[x]);
            }
            if (!turned) return;
            const bool half = t.layout == MFFT_ROTARY_HALF;
#pragma unroll
            for (int x = 0; x < V; ++x) {
                const float2 r = rotary_root(t, p0 + tok, ch * V + x);
                // pairs (x, V + x), or (2 x, 2 x + 1)
                const float fa = half ? f[x] : f[2 * x], fb = half ? f[V + x] : f[2 * x + 1];
                const float2 y = rotate_pair({fa, fb}, r);
                if (half) {
                    f[x] = y.x;
                    f[V + x] = y.y;
                } else {
                    f[2 * x] = y.x;
                    f[2 * x + 1] = y.y;
                }
            }
        };
        float mk = 0.0f, mv = 0.0f;
#pragma unroll
        for (int r = 0; r < KEEP; ++r) {
            const int i = threadIdx.x + 256 * r;
            if (i < m * half_chunks) {
                key(i, held[r]);
#pragma unroll
                for (int x = 0; x < 2 * V; ++x) mk = __builtin_fmaxf(mk, finite_abs(held[r][x]));
            }
        }
        for (int i = threadIdx.x + 256 * KEEP; i < m * half_chunks; i += 256) {
            float f[2 * V];
            key(i, f);
#pragma unroll
            for (int x = 0; x < 2 * V; ++x) mk = __builtin_fmaxf(mk, finite_abs(f[x]));
        }
        // V: first for its magnitudes, then (from cache) four channels of a
        // unit of sixteen slots a thread, whose codes are adjacent
        const int row_chunks = D / V;
        for (int i = threadIdx.x; i < m * row_chunks; i += 256) {
            const Vec u = *(const Vec*)(v + i / row_chunks * a.v_strides[0] + i % row_chunks * V);
#pragma unroll
            for (int x = 0; x < V; ++x) mv = __builtin_fmaxf(mv, finite_abs(to_float(u.e[x])));
        }
        settle(mk, mv);
        const float k_inv = 1.0f / k_new, v_inv = 1.0f / v_new;
        auto write_key = [&](int i, const float (&f)[2 * V]) {
            const int tok = i / half_chunks, ch = i % half_chunks;
            int d0, d1;
            (void)channels(ch, d0, d1);
            uint8_t* kr = kc + (int64_t)(o + tok) * D;
#pragma unroll
            for (int x = 0; x < V; x += 4) {
                *(uint32_t*)(kr + d0 + x) = to_codes(f[x] * k_inv, f[x + 1] * k_inv, f[x + 2] * k_inv, f[x + 3] * k_inv);
                *(uint32_t*)(kr + d1 + x) = to_codes(f[V + x] * k_inv, f[V + x + 1] * k_inv, f[V + x + 2] * k_inv, f[V + x + 3] * k_inv);
            }
        };
#pragma unroll
        for (int r = 0; r < KEEP; ++r) {
            const int i = threadIdx.x + 256 * r;
            if (r < rounds && i < m * half_chunks) write_key(i, held[r]);
        }
        for (int i = threadIdx.x + 256 * KEEP; i < m * half_chunks; i += 256) {
            float f[2 * V];
            key(i, f);
            write_key(i, f);
        }
        struct alignas(4 * sizeof(E)) Quad {
            E e[4];
        };
        const int quads = D / 4, u0 = o >> 4, u1 = (o + m - 1) >> 4;
        for (int i = threadIdx.x; i < (u1 - u0 + 1) * quads; i += 256) {
            const int u = u0 + i / quads, d = i % quads * 4;
            const int s0 = max(16 * u - o, 0), s1 = min(16 * u + 16 - o, m);  // tokens of this call in the unit
            uint8_t* vu = vc + ((int64_t)u * D + d) * 16;
            if (s1 - s0 == 16) {
                uint32_t w[4][4];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    Quad q[4];
#pragma unroll
                    for (int z = 0; z < 4; ++z) q[z] = *(const Quad*)(v + (s0 + 4 * y + z) * a.v_strides[0] + d);
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        w[x][y] = to_codes(to_float(q[0].e[x]) * v_inv, to_float(q[1].e[x]) * v_inv, to_float(q[2].e[x]) * v_inv,
                                           to_float(q[3].e[x]) * v_inv);
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) *(uint4*)(vu + 16 * x) = make_uint4(w[x][0], w[x][1], w[x][2], w[x][3]);
            } else {
                for (int s = s0; s < s1; ++s) {
                    const Quad q = *(const Quad*)(v + s * a.v_strides[0] + d);
#pragma unroll
                    for (int x = 0; x < 4; ++x) vu[16 * x + ((o + s) & 15)] = to_code(to_float(q.e[x]) * v_inv);
                }
            }
        }
        return;
    }

    auto rotated = [&](int i, int e, int& d0, int& d1) {
        pair_channels(t.layout, t.pairs, e, d0, d1);
        const float fa = to_float(k[i * a.k_strides[0] + d0]), fb = to_float(k[i * a.k_strides[0] + d1]);
        if (e >= t.pairs) return make_float2(fa, fb);
        return rotate_pair({fa, fb}, rotary_root(t, p0 + i, e));
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
    settle(mk, mv);
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

// Whether append_kernel takes 16 bytes of k and v, and of q and q_out, at a time:
// chunks of V pairs, everything 16-byte aligned, and tokens enough that threads
// are not what is short.  32768 tokens of 8 key and 32 query heads: 201 us so,
// 541 us a pair a thread; one token each of 256 sequences, where a page's
// sixteen chunks would each wait for eight pairs' roots: 15.2 and 8.5 us.
bool wide(const RotaryTables& t, const mfft_append_args& a) {
    const int v = a.dtype == MFFT_F32 ? 4 : 8;
    if (!a.offsets || t.pairs % v) return false;
    const void* p[] = {a.k, a.v, a.q, a.q_out};
    const int64_t* s[] = {a.k_strides, a.v_strides, a.q_strides, a.q_out_strides};
    for (int i = 0; i < (a.q ? 4 : 2); ++i)
        if (((uintptr_t)p[i] & 15) || s[i][0] % v || s[i][1] % v) return false;
    return true;
}

template <class E>
void launch_type(const RotaryTables& t, const mfft_cache& c, const mfft_append_args& a, hipStream_t s) {
    if (wide(t, a)) {
        const AppendGrid g = append_grid(c, a, a.dtype == MFFT_F32 ? 4 : 8);
        append_kernel<E, true><<<(uint32_t)(g.kv_blocks + g.q_blocks), 256, 0, s>>>(t, c, a);
    } else {
        const AppendGrid g = append_grid(c, a, 1);
        append_kernel<E, false><<<(uint32_t)(g.kv_blocks + g.q_blocks), 256, 0, s>>>(t, c, a);
    }
}

}  // namespace

bool append_launch_fits(const RotaryTables&, const mfft_cache& c, const mfft_append_args& a) {
    const AppendGrid g = append_grid(c, a, 1);
    return launch_fits(g.kv_blocks + g.q_blocks, 256);
}

hipError_t launch_append(const RotaryTables& t, const mfft_cache& c, const mfft_append_args& a, hipStream_t stream) {
    if (a.dtype == MFFT_F32) launch_type<float>(t, c, a, stream);
    else if (a.dtype == MFFT_F16) launch_type<_Float16>(t, c, a, stream);
    else launch_type<__bf16>(t, c, a, stream);
    mark(stream);
    return hipGetLastError();
}

}  // namespace mfft

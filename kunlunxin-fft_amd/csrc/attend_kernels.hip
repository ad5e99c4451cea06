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

// a mask of bytes [from, to) of a 16-byte unit
__device__ __forceinline__ u32x4 keep_bytes(int from, int to) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        int lo = from - 4 * i, hi = to - 4 * i;
        lo = lo < 0 ? 0 : lo > 4 ? 4 : lo;
        hi = hi < 0 ? 0 : hi > 4 ? 4 : hi;
        r[i] = hi > lo ? (uint32_t)((((uint64_t)1 << (8 * hi)) - 1) & ~(((uint64_t)1 << (8 * lo)) - 1)) : 0;
    }
    return r;
}

// 0x01 in each byte that is a NaN code
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return (((w & 0x7f7f7f7f) + 0x01010101) >> 7) & 0x01010101; }

// the log of a row's sum of exponentials, from its maximum in units of log 2
__device__ __forceinline__ float log_sum(float m, float l, bool poison) {
    if (poison) return __builtin_nanf("");
    return l == 0.0f ? -__builtin_inff() : m * 0.69314718055994530942f + __logf(l);
}

// ---- which part of the work a workgroup takes ---------------------------------
// An item is (sequence, block of query rows, key head); its work is the groups
// of 64 keys its sequence has.  All items' groups, one item after the other,
// form one list, and each of `grid` workgroups takes an equal share of it, so
// that the chip is filled evenly whatever the lengths are: a share is some
// whole items and at most two cut ones, at its ends.  The list follows from the
// lengths, which only the device knows; every workgroup works its place out for
// itself with one pass of a wave over the sequences.  Cut items leave their
// (m, l, O) in the workspace and join_kernel adds them up.
struct AttendShape {
    int group;        // query heads a key head
    int rows;         // rows of a block
    int units;        // page_size / 16
    uint64_t magic;   // floor(2^32 / units) + 1: x / units = x * magic >> 32, exact for x < 2^26
    int grid;         // shares; 0: one workgroup an item, none cut
    int least;        // fewest groups of 64 keys in a share
    int live;         // rows of a block that can be in use
    int64_t per;      // queries of each sequence without offsets
};

// the item that starts in share i and is cut at its end: its parts are in
// slots 2 i + 1, 2 (i + 1), 2 (i + 2), ... of the workspace
struct Cut {
    int parts;  // 0: none
    int b, block, h;
};

struct Sequence {
    int64_t row0, n;  // its queries
    int len;          // its keys, within the table
    bool poison;      // it has more than the table's
    int low, tiles;   // first key that any query sees (a multiple of 64), groups of 64 keys from there
    int blocks;       // of rows
};

__device__ __forceinline__ Sequence sequence(const mfft_cache& c, const mfft_attend_args& a, const AttendShape& sh, int b) {
    Sequence q;
    q.row0 = seq_offset(a.offsets, sh.per, a.tokens, b);
    q.n = seq_offset(a.offsets, sh.per, a.tokens, b + 1) - q.row0;
    if (q.n < 0) q.n = 0;
    const int most = a.table_width * c.page_size;
    const int len = a.lengths[b];
    q.poison = len > most;
    q.len = len < 0 ? 0 : q.poison ? most : len;
    q.low = 0;
    if (a.window) {
        const int64_t lo = q.len - q.n + 1 - a.window;
        q.low = lo > 0 ? (int)(lo & ~(int64_t)63) : 0;
    }
    q.tiles = (q.len - q.low + 63) >> 6;
    if (q.tiles < 1) q.tiles = 1;  // rows that see nothing are still written
    q.blocks = (int)((q.n * sh.group + sh.rows - 1) / sh.rows);
    return q;
}

// a value that is the same in all lanes, as a scalar
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    const uint32_t lo = (uint32_t)uniform((int)v), hi = (uint32_t)uniform((int)(v >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// v, in a form that keeps what is computed from it where it is written: the
// compiler otherwise computes every address an item's end needs before the
// loop over items, and holds them in registers through the loop over keys
__device__ __forceinline__ int here(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

__device__ __forceinline__ int64_t wave_scan(int64_t v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const int64_t o = __shfl_up(v, s);
        if (lane >= s) v += o;
    }
    return v;
}

// The sequence in whose work (groups of keys, or items where `by_item`) place
// `at` lies, and what comes before it; -1 past the end.
__device__ __forceinline__ int locate(const mfft_cache& c, const mfft_attend_args& a, const AttendShape& sh, bool by_item,
                                      int64_t at, int64_t& before) {
    const int lane = threadIdx.x & 63;
    before = 0;
    for (int i = 0; i < a.sequences; i += 64) {
        int64_t w = 0;
        if (i + lane < a.sequences) {
            const Sequence q = sequence(c, a, sh, i + lane);
            w = (int64_t)q.blocks * c.kv_heads * (by_item ? 1 : q.tiles);
        }
        const int64_t upto = wave_scan(w);
        const uint64_t hit = __ballot(before + upto > at);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            before += uniform(__shfl(upto - w, l));
            return uniform(i + l);
        }
        before += uniform(__shfl(upto, 63));
    }
    return -1;
}

__device__ __forceinline__ int64_t all_work(const mfft_cache& c, const mfft_attend_args& a, const AttendShape& sh) {
    int64_t none;
    (void)locate(c, a, sh, false, INT64_MAX, none);
    return none;
}

// ---- one item, some of its keys --------------------------------------------------
// KEYS: the workgroup's four waves share 16 R rows and take every fourth group
// of 64 keys, each straight from memory into registers, one group ahead; their
// (m, l, O) are joined in LDS.  For few rows: nothing but the cache's bytes
// counts, and a wave's loads wait for no other wave.
// not KEYS: each wave has 16 R rows of its own and all take every group, which
// goes through LDS once for the four.  For many rows.
template <class E, int D, int R, bool KEYS>
struct Attend {
    using M = Mat<E>;
    typedef typename M::x8 x8;
    using S = Dims<D>;
    static constexpr int ROWS = KEYS ? 16 * R : 64 * R;  // of a block
    static constexpr int STEP = KEYS ? 256 : 64;         // keys between a wave's groups

    // LDS of the two forms.  Keys: rows of D codes 16 bytes apart and 64 more
    // after each sixteen, so that the sixteen rows a load takes at once
    // (16 kg + kr) lie in different banks.  Values: as in memory.
    static constexpr int KROW = D + 16, KLDS = 64 * KROW + 4 * 64, VLDS = 64 * D;
    union Shared {
        struct {
            float m[2][R][16], l[2][R][16];
            f32x4 o[2][R][S::N][64];
        } join;
        struct {
            uint8_t k[2][KLDS], v[2][VLDS];
            int nan;
        } tile;
    };
    typedef typename std::conditional<KEYS, decltype(Shared::join), decltype(Shared::tile)>::type Lds;

    const mfft_cache& c;
    const mfft_attend_args& a;
    const AttendShape& sh;
    Lds& lds;
    int lane, wave, j, g, kg, kr;

    // of the item
    Sequence seq;
    const int32_t* table;
    int h;
    int64_t all, block;
    x8 qv[R][S::KK];
    int low[R], top[R];                // keys [low, top) that each of this lane's rows sees
    int all_lo, all_hi, any_lo, any_hi;  // and all, and any, of the wave's rows
    f32x4 o[R][S::N];
    float m[R], l[R];

    // of the group at hand
    u32x4 kw[4][S::J > 0 ? S::J : 1];
    u32x2 kx[4];
    u32x4 vw[S::N];
    float cs, vs;

    __device__ __forceinline__ Attend(const mfft_cache& c_, const mfft_attend_args& a_, const AttendShape& sh_, Lds& lds_)
        : c(c_), a(a_), sh(sh_), lds(lds_) {
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        j = lane & 15;
        g = lane >> 4;
        kg = j >> 2;  // K rows of lane j: keys 16 kg + 4 t + kr
        kr = j & 3;
    }

    __device__ __forceinline__ int64_t row_of(int r, int j) const { return block + (KEYS ? 0 : 16 * R * wave) + 16 * r + j; }

    __device__ __forceinline__ void begin(int b, int block_, int h_) {
        h = h_;
        table = a.page_table + b * a.table_stride;
        all = seq.n * sh.group;
        block = (int64_t)block_ * ROWS;
        all_lo = 0;
        all_hi = seq.len;
        any_lo = seq.len;
        any_hi = 0;
        nan_left = false;
        const int j = here(this->j), g = here(this->g);
        static_for<0, R>([&](auto r) {
            int64_t row = row_of(r.value, j);
            row = row < all ? row : all - 1;  // rows past the last repeat it and are not stored
            const int64_t tok = row / sh.group;
            const int qh = h * sh.group + (int)(row % sh.group);
            const E* q = (const E*)a.q + (seq.row0 + tok) * a.q_strides[0] + qh * a.q_strides[1];
            static_for<0, S::J>([&](auto jj) {
                qv[r.value][2 * jj.value] = *(const x8*)(q + 64 * jj.value + 16 * g);
                qv[r.value][2 * jj.value + 1] = *(const x8*)(q + 64 * jj.value + 16 * g + 8);
            });
            if constexpr (S::REM) qv[r.value][S::KK - 1] = *(const x8*)(q + 64 * S::J + 8 * g);
            const int64_t pos = seq.len - seq.n + tok;
            int hi = a.causal && pos + 1 < seq.len ? (int)(pos + 1) : seq.len;
            int lo = a.window && pos + 1 > a.window ? (int)(pos + 1 - a.window) : 0;
            if (hi < lo) hi = lo;
            low[r.value] = lo;
            top[r.value] = hi;
            all_lo = max(all_lo, lo);
            all_hi = min(all_hi, hi);
            any_lo = min(any_lo, lo);
            any_hi = max(any_hi, hi);
            static_for<0, S::N>([&](auto i) { o[r.value][i.value] = f32x4{0, 0, 0, 0}; });
            m[r.value] = kLowest;
            l[r.value] = 0.0f;
        });
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
    }

    // Table entry of the sixteen keys `u` of the sequence, and where in the page
    // they are.  Past the sequence's end the entry is its last page's (the
    // table's first if it has none), so that loads need no branch: a branch
    // around a load ends in a wait for all loads before it.
    __device__ __forceinline__ int page_entry(uint32_t u) const {
        const uint32_t most = seq.len > 0 ? (uint32_t)(seq.len - 1) >> 4 : 0;
        return table[(uint32_t)(min(u, most) * sh.magic >> 32)];
    }
    __device__ __forceinline__ uint32_t unit_in_page(uint32_t u) const { return u - (uint32_t)(u * sh.magic >> 32) * sh.units; }
    __device__ __forceinline__ int64_t page_of(int entry) const { return (uint32_t)entry < (uint32_t)c.pages ? entry : 0; }
    // first byte of sixteen tokens' codes (keys: their first row; values: their unit)
    __device__ __forceinline__ int64_t unit_at(int entry, uint32_t u) const {
        return ((page_of(entry) * c.kv_heads + h) * sh.units + unit_in_page(u)) * (16 * D);
    }
    // the scales of this lane's sixteen keys, as loaded, and as they count:
    // scores in units of log 2, NaN for a page number that is none; past the
    // end of the sequence neither may count, whatever they are
    float ks_raw, vs_raw;
    bool bad_page;
    __device__ __forceinline__ void load_scales(int entry) {
        const int64_t at = page_of(entry) * c.kv_heads + h;
        ks_raw = c.k_scale[at];
        vs_raw = c.v_scale[at];
        bad_page = (uint32_t)entry >= (uint32_t)c.pages;
    }
    __device__ __forceinline__ void take_scales(int key0) {
        const bool in = key0 + 16 * g < seq.len;
        cs = bad_page ? __builtin_nanf("") : a.scale * 1.44269504088896340736f * ks_raw;
        vs = in ? vs_raw : 1.0f;
    }

    // S = K Q of the group at hand, kw(t, jj) and kx(t) its codes
    template <class K, class X>
    __device__ __forceinline__ void scores(f32x4 (&s)[R][4], K&& k16, X&& k8) {
        static_for<0, 4>([&](auto t) {
            static_for<0, R>([&](auto r) { s[r.value][t.value] = f32x4{0, 0, 0, 0}; });
            static_for<0, S::J>([&](auto jj) {
                const u32x4 w = k16(t, jj);
                const x8 k0 = decode8<E>(w[0], w[1], 1.0f), k1 = decode8<E>(w[2], w[3], 1.0f);
                static_for<0, R>([&](auto r) {
                    s[r.value][t.value] = M::mfma(k0, qv[r.value][2 * jj.value], s[r.value][t.value]);
                    s[r.value][t.value] = M::mfma(k1, qv[r.value][2 * jj.value + 1], s[r.value][t.value]);
                });
            });
            if constexpr (S::REM) {
                const u32x2 w = k8(t);
                const x8 k0 = decode8<E>(w[0], w[1], 1.0f);
                static_for<0, R>([&](auto r) { s[r.value][t.value] = M::mfma(k0, qv[r.value][S::KK - 1], s[r.value][t.value]); });
            }
            if constexpr (R > 1 && t.value % 2 == 1) __builtin_amdgcn_sched_barrier(0);
        });
    }

    // P from S, m and l moved on, O rescaled where m grew
    __device__ __forceinline__ void weights(f32x4 (&s)[R][4], x8 (&p)[R][2], bool at_edge, int kv) {
        static_for<0, R>([&](auto r) {
            float unit = cs;
            if (at_edge) {
                // bit i: key kv + i is seen; as masks of whole words, which
                // take no condition registers
                const int lo = min(max(low[r.value] - kv, 0), 16), hi = min(max(top[r.value] - kv, 0), 16);
                const int seen = (int)((1u << hi) - (1u << lo));
                static_for<0, 16>([&](auto i) {
                    const uint32_t bit = (uint32_t)((seen << (31 - i.value)) >> 31);
                    const uint32_t v = __float_as_uint(s[r.value][i.value / 4][i.value % 4] * cs);
                    s[r.value][i.value / 4][i.value % 4] = __uint_as_float((v & bit) | (0xff800000u & ~bit));
                });
                unit = 1.0f;
            }
            float mx = s[r.value][0][0];
            static_for<1, 16>([&](auto i) { mx = __builtin_fmaxf(mx, s[r.value][i.value / 4][i.value % 4]); });
            mx = __builtin_fmaxf(m[r.value], mx * unit);
            mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16));
            mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32));
            if (__any(mx > m[r.value])) {
                const float shrink = __builtin_amdgcn_exp2f(m[r.value] - mx);
                m[r.value] = mx;
                l[r.value] *= shrink;
                static_for<0, S::N>([&](auto i) { o[r.value][i.value] *= shrink; });
            }
            static_for<0, 16>([&](auto i) {
                const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r.value][i.value / 4][i.value % 4], unit, -m[r.value]));
                l[r.value] += w;
                p[r.value][i.value / 8][i.value % 8] = (E)w;
            });
        });
    }

    // O += V P, v(i) the codes of channels 16 i .. 16 i + 15
    template <class V>
    __device__ __forceinline__ void values(x8 (&p)[R][2], V&& v) {
        static_for<0, S::N>([&](auto i) {
            const u32x4 w = v(i);
            const x8 v0 = decode8<E>(w[0], w[1], vs), v1 = decode8<E>(w[2], w[3], vs);
            static_for<0, R>([&](auto r) {
                o[r.value][i.value] = M::mfma(v0, p[r.value][0], o[r.value][i.value]);
                o[r.value][i.value] = M::mfma(v1, p[r.value][1], o[r.value][i.value]);
            });
            if constexpr (R > 1 && i.value % 2 == 1) __builtin_amdgcn_sched_barrier(0);
        });
    }

    // Values of a group where not every row sees every key.  Keys that no row
    // sees may hold anything: their codes count as 0 (`keep` masks the others).
    // A NaN of the others counts only for the rows that see its key, while 0 * NaN
    // is NaN: its code becomes 0 here, and mark_nans() finds the rows that see
    // it once the item is done.
    bool nan_left;
    int block_lo, block_hi, block_all_lo, block_all_hi;
    __device__ __forceinline__ u32x4 clean(u32x4 w, u32x4 keep) {
        uint32_t bad = 0;
        static_for<0, 4>([&](auto x) {
            const uint32_t v = w[x.value] & keep[x.value], n = nan_bytes(v);
            bad |= n;
            w[x.value] = v & ~(n * 0xffu);
        });
        nan_left |= bad != 0;
        return w;
    }
    // (a group in LDS is cleaned for all four waves' rows at once)
    __device__ __forceinline__ bool edge(int key0) const {
        return KEYS ? key0 < all_lo || key0 + 64 > all_hi : key0 < block_all_lo || key0 + 64 > block_all_hi;
    }

    // (rare, and so key by key from memory, after the loop it would slow down)
    __device__ __forceinline__ void mark_nans(int from, int end) {
        if (!__any(nan_left)) return;
        const int g = here(this->g);
#pragma unroll 1
        for (int key = from; key < end; ++key) {
            const int key0 = key & ~63;
            if (!edge(key0) || (KEYS && ((key0 - from) / 64) % 4 != wave)) continue;
            const uint32_t u = (uint32_t)key >> 4;
            const uint8_t* vb = (const uint8_t*)c.v + unit_at(page_entry(u), u) + 64 * g + (key & 15);
            static_for<0, S::N>([&](auto i) {
                static_for<0, 4>([&](auto x) {
                    if ((vb[16 * (16 * i.value + x.value)] & 0x7f) == kNaNCode) {
                        static_for<0, R>([&](auto r) {
                            if (key >= low[r.value] && key < top[r.value]) o[r.value][i.value][x.value] = __builtin_nanf("");
                        });
                    }
                });
            });
        }
    }

    // ---- the waves share the rows
    __device__ __forceinline__ void load_keys(int key0, int entry) {
        const uint8_t* kb = (const uint8_t*)c.k + unit_at(entry, (uint32_t)(key0 >> 4) + kg) + kr * D;
        static_for<0, 4>([&](auto t) {
            static_for<0, S::J>([&](auto jj) { kw[t.value][jj.value] = *(const u32x4*)(kb + 4 * t.value * D + 64 * jj.value + 16 * g); });
            if constexpr (S::REM) kx[t.value] = *(const u32x2*)(kb + 4 * t.value * D + 64 * S::J + 8 * g);
        });
    }
    __device__ __forceinline__ void load_values(int key0, int entry) {
        const uint8_t* vb = (const uint8_t*)c.v + unit_at(entry, (uint32_t)(key0 >> 4) + g) + 16 * j;
        static_for<0, S::N>([&](auto i) { vw[i.value] = *(const u32x4*)(vb + i.value * 256); });
    }

    __device__ __forceinline__ void run_keys(int from, int end) {
        from = max(from, any_lo & ~63);
        end = min(end, any_hi);
        int key0 = from + 64 * wave;
        // Loads come back in order, so each is issued before those that need
        // not wait for it: table entries two groups ahead, then scales and K
        // of the next, and V once this group's is used up.
        int k1 = 0, v1 = 0, k2 = 0, v2 = 0;
        auto entries = [&](int k0, int& k, int& v) {
            k = page_entry((uint32_t)(k0 >> 4) + kg);
            v = page_entry((uint32_t)(k0 >> 4) + g);
        };
        if (key0 < end) {
            entries(key0, k1, v1);
            entries(key0 + STEP, k2, v2);
            load_scales(v1);
            load_keys(key0, k1);
            load_values(key0, v1);
        }
        for (; key0 < end; key0 += STEP) {
            f32x4 s[R][4];
            x8 p[R][2];
            take_scales(key0);
            scores(s, [&](auto t, auto jj) { return kw[t.value][jj.value]; }, [&](auto t) { return kx[t.value]; });
            const bool more = key0 + STEP < end;
            k1 = k2;
            v1 = v2;
            if (more) {
                entries(key0 + 2 * STEP, k2, v2);
                load_scales(v1);
                load_keys(key0 + STEP, k1);
            }
            const int kv = key0 + 16 * g;
            weights(s, p, edge(key0), kv);
            if (edge(key0)) {
                const u32x4 keep = keep_bytes(any_lo - kv, any_hi - kv);
                static_for<0, S::N>([&](auto i) { vw[i.value] = clean(vw[i.value], keep); });
            }
            values(p, [&](auto i) { return vw[i.value]; });
            if (more) load_values(key0 + STEP, v1);
        }
        mark_nans(from, end);
        static_for<0, R>([&](auto r) {
            l[r.value] += __shfl_xor(l[r.value], 16);
            l[r.value] += __shfl_xor(l[r.value], 32);
        });
        // join the waves, two and two; the result is wave 0's
        const int lane = here(this->lane), j = lane & 15, g = lane >> 4;
        static_for<0, 2>([&](auto round) {
            constexpr int from_w = round.value == 0 ? 2 : 1;
            __syncthreads();
            if (wave >= from_w && wave < 2 * from_w) {
                static_for<0, R>([&](auto r) {
                    if (g == 0) {
                        lds.m[wave - from_w][r.value][j] = m[r.value];
                        lds.l[wave - from_w][r.value][j] = l[r.value];
                    }
                    static_for<0, S::N>([&](auto i) { lds.o[wave - from_w][r.value][i.value][lane] = o[r.value][i.value]; });
                });
            }
            __syncthreads();
            if (wave < from_w) {
                static_for<0, R>([&](auto r) {
                    const float mo = lds.m[wave][r.value][j], mt = __builtin_fmaxf(m[r.value], mo);
                    const float f = __builtin_amdgcn_exp2f(m[r.value] - mt), fo = __builtin_amdgcn_exp2f(mo - mt);
                    m[r.value] = mt;
                    l[r.value] = l[r.value] * f + lds.l[wave][r.value][j] * fo;
                    static_for<0, S::N>([&](auto i) {
                        o[r.value][i.value] = o[r.value][i.value] * f + lds.o[wave][r.value][i.value][lane] * fo;
                    });
                });
            }
        });
    }

    // ---- each wave has rows of its own
    // Wave w fetches keys 16 w .. 16 w + 15 of a group: D / 64 loads of 16 bytes
    // a lane for K and as many for V.
    static constexpr int L = (D + 63) / 64;
    u32x4 fk[L], fv[L];
    __device__ __forceinline__ void fetch(int key0, int entry) {
        const int64_t at = unit_at(entry, (uint32_t)(key0 >> 4) + wave);
        static_for<0, L>([&](auto x) {
            const int i = lane + 64 * x.value;
            if (D % 64 == 0 || i < D) {
                fk[x.value] = *(const u32x4*)((const uint8_t*)c.k + at + 16 * i);
                fv[x.value] = *(const u32x4*)((const uint8_t*)c.v + at + 16 * i);
            }
        });
    }
    __device__ __forceinline__ void stash(int buf, int key0) {
        if (edge(key0)) {
            const int kv = key0 + 16 * wave;
            const u32x4 keep = keep_bytes(block_lo - kv, block_hi - kv);
            static_for<0, L>([&](auto x) { fv[x.value] = clean(fv[x.value], keep); });
            if (nan_left) lds.nan = 1;
        }
        static_for<0, L>([&](auto x) {
            const int i = lane + 64 * x.value;
            if (D % 64 == 0 || i < D) {
                const int row = i / (D / 16), at = i % (D / 16);
                *(u32x4*)(lds.k[buf] + (16 * wave + row) * KROW + 64 * wave + 16 * at) = fk[x.value];
                *(u32x4*)(lds.v[buf] + (wave * D + i) * 16) = fv[x.value];
            }
        });
    }

    __device__ __forceinline__ void run_rows(int from, int end) {
        // of the workgroup's rows: both ends of what a row sees rise with it
        {
            const int64_t p0 = seq.len - seq.n + block / sh.group;
            const int64_t p1 = seq.len - seq.n + (min(block + ROWS, all) - 1) / sh.group;
            auto lower = [&](int64_t p) { return a.window && p + 1 > a.window ? (int)(p + 1 - a.window) : 0; };
            auto upper = [&](int64_t p) { return !a.causal || p + 1 > seq.len ? seq.len : p < 0 ? 0 : (int)(p + 1); };
            block_lo = lower(p0);
            block_hi = upper(p1);
            block_all_lo = lower(p1);
            block_all_hi = upper(p0);
        }
        from = max(from, block_lo & ~63);
        end = min(end, block_hi);
        __syncthreads();  // a share's last item may still be read
        if (threadIdx.x == 0) lds.nan = 0;
        __syncthreads();
        int e1 = 0, v1 = 0;  // table entries of the next group, fetched and of this lane's keys
        if (from < end) {
            e1 = page_entry((uint32_t)(from >> 4) + wave);
            v1 = page_entry((uint32_t)(from >> 4) + g);
            load_scales(v1);
            fetch(from, e1);
            e1 = page_entry((uint32_t)((from + 64) >> 4) + wave);
            v1 = page_entry((uint32_t)((from + 64) >> 4) + g);
            stash(0, from);
        }
        int buf = 0;
        for (int key0 = from; key0 < end; key0 += 64) {
            __syncthreads();
            const bool more = key0 + 64 < end;
            take_scales(key0);
            if (more) {
                load_scales(v1);
                const int e0 = e1;
                e1 = page_entry((uint32_t)((key0 + 128) >> 4) + wave);
                v1 = page_entry((uint32_t)((key0 + 128) >> 4) + g);
                fetch(key0 + 64, e0);
            }
            if (key0 + 64 > any_lo && key0 < any_hi) {
                f32x4 s[R][4];
                x8 p[R][2];
                const uint8_t* kb = lds.k[buf] + (16 * kg + kr) * KROW + 64 * kg;
                scores(s, [&](auto t, auto jj) { return *(const u32x4*)(kb + 4 * t.value * KROW + 64 * jj.value + 16 * g); },
                       [&](auto t) { return *(const u32x2*)(kb + 4 * t.value * KROW + 64 * S::J + 8 * g); });
                weights(s, p, key0 < all_lo || key0 + 64 > all_hi, key0 + 16 * g);
                const uint8_t* vb = lds.v[buf] + (g * D + j) * 16;
                values(p, [&](auto i) { return *(const u32x4*)(vb + 256 * i.value); });
            }
            buf ^= 1;
            if (more) stash(buf, key0 + 64);
        }
        __syncthreads();
        nan_left = lds.nan != 0;
        mark_nans(from, end);
        static_for<0, R>([&](auto r) {
            l[r.value] += __shfl_xor(l[r.value], 16);
            l[r.value] += __shfl_xor(l[r.value], 32);
        });
    }

    __device__ __forceinline__ void run(int from, int end) {
        if constexpr (KEYS) run_keys(from, end);
        else run_rows(from, end);
    }

    // ---- out of the registers
    __device__ __forceinline__ void store() const {
        if (KEYS && wave > 0) return;
        const int j = here(this->j), g = here(this->g);
        static_for<0, R>([&](auto r) {
            const int64_t row = row_of(r.value, j);
            if (row >= all) return;
            const int64_t tok = seq.row0 + row / sh.group;
            const int qh = h * sh.group + (int)(row % sh.group);
            float inv = l[r.value] == 0.0f ? 0.0f : 1.0f / l[r.value];
            if (seq.poison) inv = __builtin_nanf("");
            E* y = (E*)a.out + tok * a.out_strides[0] + qh * a.out_strides[1];
            static_for<0, S::N>([&](auto i) {
                union {
                    E e[4];
                    u32x2 w;
                } u;
#pragma unroll
                for (int x = 0; x < 4; ++x) u.e[x] = (E)(o[r.value][i.value][x] * inv);
                *(u32x2*)(y + 16 * i.value + 4 * g) = u.w;
            });
            if (a.lse && g == 0) a.lse[tok * a.q_heads + qh] = log_sum(m[r.value], l[r.value], seq.poison);
        });
    }
    __device__ __forceinline__ void store_part(int slot, float* part_o, float2* part_ml) const {
        if (KEYS && wave > 0) return;
        const int j = here(this->j), g = here(this->g);
        static_for<0, R>([&](auto r) {
            const int64_t row = row_of(r.value, j);
            if (row >= all) return;
            const int64_t at = (int64_t)slot * ROWS + (row - block);
            static_for<0, S::N>([&](auto i) { *(f32x4*)(part_o + at * D + 16 * i.value + 4 * g) = o[r.value][i.value]; });
            if (g == 0) part_ml[at] = make_float2(m[r.value], l[r.value]);
        });
    }
};

template <class E, int D, int R, bool KEYS>
__global__ __launch_bounds__(256, KEYS && D * R >= 256 ? 1 : 2) void attend_kernel(mfft_cache c, mfft_attend_args a, AttendShape sh,
                                                                        float* part_o, float2* part_ml, Cut* cuts) {
    using A = Attend<E, D, R, KEYS>;
    __shared__ __align__(16) typename A::Lds lds;
    A w(c, a, sh, lds);
    // groups [at, stop) of the list; with one workgroup an item, of that item
    int64_t before, at = 0, stop, share = INT64_MAX;
    int b, item, tile = 0;
    if (sh.grid == 0) {
        b = locate(c, a, sh, true, blockIdx.x, before);
        if (b < 0) return;
        w.seq = sequence(c, a, sh, b);
        item = (int)((int64_t)blockIdx.x - before);
        stop = w.seq.tiles;
    } else {
        const int64_t total = all_work(c, a, sh);
        const int64_t even = (total + sh.grid - 1) / sh.grid;
        share = even > sh.least ? even : sh.least;
        at = blockIdx.x * share;
        stop = at + share < total ? at + share : total;
        if (at >= stop) {
            if (threadIdx.x == 0) cuts[blockIdx.x].parts = 0;
            return;
        }
        b = locate(c, a, sh, false, at, before);
        w.seq = sequence(c, a, sh, b);
        item = uniform((int)((at - before) / w.seq.tiles));
        tile = uniform((int)((at - before) - (int64_t)item * w.seq.tiles));
    }
    Cut cut{0, 0, 0, 0};
    while (true) {
        const int upto = stop - at < w.seq.tiles - tile ? tile + (int)(stop - at) : w.seq.tiles;
        const int block = item / c.kv_heads, h = item % c.kv_heads;
        w.begin(b, block, h);
        w.run(w.seq.low + 64 * tile, w.seq.low + 64 * upto);
        if (tile == 0 && upto == w.seq.tiles) {
            w.store();
        } else {
            w.store_part(2 * (int)blockIdx.x + (tile == 0 ? 1 : 0), part_o, part_ml);
            if (tile == 0) cut = {(int)((at + w.seq.tiles - 1) / share) - (int)blockIdx.x + 1, b, block, h};
        }
        at += upto - tile;
        if (at >= stop) break;
        tile = 0;
        if (++item == w.seq.blocks * c.kv_heads) {
            item = 0;
            do {  // there is one: work is left
                w.seq = sequence(c, a, sh, ++b);
            } while (w.seq.blocks == 0);
        }
    }
    if (sh.grid && threadIdx.x == 0) cuts[blockIdx.x] = cut;
}

// A cut item's row: one workgroup, its waves every fourth part, each lane
// D / 64 channels.
template <class E, int D>
__global__ __launch_bounds__(256) void join_kernel(mfft_cache c, mfft_attend_args a, AttendShape sh, const float* part_o,
                                                   const float2* part_ml, const Cut* cuts) {
    constexpr int C = (D + 63) / 64;
    const int share = blockIdx.x / sh.live, row_in = blockIdx.x % sh.live;
    const Cut cut = cuts[share];
    if (cut.parts == 0) return;
    const Sequence seq = sequence(c, a, sh, cut.b);
    const int64_t row = (int64_t)cut.block * sh.rows + row_in;
    if (row >= seq.n * sh.group) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    auto slot = [&](int p) { return (int64_t)(2 * (share + p) + (p == 0 ? 1 : 0)) * sh.rows + row_in; };

    float m = kLowest;
    for (int p = lane; p < cut.parts; p += 64) m = __builtin_fmaxf(m, part_ml[slot(p)].x);
    m = wave_max(m);
    float l = 0.0f, o[C] = {};
#pragma unroll 4
    for (int p = wave; p < cut.parts; p += 4) {
        const int64_t s = slot(p);
        const float2 ml = part_ml[s];
        const float f = __builtin_amdgcn_exp2f(ml.x - m);
        l += ml.y * f;
#pragma unroll
        for (int x = 0; x < C; ++x)
            if (D % 64 == 0 || lane + 64 * x < D) o[x] += part_o[s * D + lane + 64 * x] * f;
    }
    __shared__ float sl[4], so[4][64 * C];
    if (lane == 0) sl[wave] = l;
#pragma unroll
    for (int x = 0; x < C; ++x) so[wave][lane + 64 * x] = o[x];
    __syncthreads();
    l = sl[0] + sl[1] + sl[2] + sl[3];
    float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (seq.poison) inv = __builtin_nanf("");
    const int64_t tok = seq.row0 + row / sh.group;
    const int qh = cut.h * sh.group + (int)(row % sh.group);
    E* y = (E*)a.out + tok * a.out_strides[0] + qh * a.out_strides[1];
    if (threadIdx.x < D)
        y[threadIdx.x] = (E)((so[0][threadIdx.x] + so[1][threadIdx.x] + so[2][threadIdx.x] + so[3][threadIdx.x]) * inv);
    if (a.lse && threadIdx.x == 0) a.lse[tok * a.q_heads + qh] = log_sum(m, l, seq.poison);
}

// ---- the launch ---------------------------------------------------------------
constexpr int kShares = 512;    // two workgroups on each of 256 CUs
constexpr int kLeastTiles = 4;  // one group of 64 keys a wave

struct AttendLaunch {
    AttendShape sh;
    int r;            // row tiles of a wave
    bool keys;
    int64_t grid, o_bytes, ml_bytes, cut_bytes;
};

AttendLaunch attend_launch(const mfft_cache& c, const mfft_attend_args& a) {
    AttendLaunch w{};
    w.sh.group = a.q_heads / c.kv_heads;
    w.sh.units = c.page_size / 16;
    w.sh.magic = ((uint64_t)1 << 32) / w.sh.units + 1;
    w.sh.per = a.offsets ? 1 : a.tokens / a.sequences;
    w.sh.least = kLeastTiles;
    // rows of a sequence and key head, on average where there are offsets
    const int64_t rows = (a.tokens * w.sh.group + a.sequences - 1) / a.sequences;
    w.keys = rows <= 32;
    w.r = w.keys ? (rows <= 16 ? 1 : 2) : (rows <= 64 || c.head_dim > 128 ? 1 : 2);
    w.sh.rows = w.keys ? 16 * w.r : 64 * w.r;
    w.sh.live = !a.offsets && rows < w.sh.rows ? (int)rows : w.sh.rows;
    const int64_t items = (a.tokens * w.sh.group / w.sh.rows + a.sequences) * c.kv_heads;  // at most
    const bool whole = a.max_length && a.max_length <= kLeastTiles * 64;
    w.sh.grid = whole ? 0 : kShares;
    w.grid = whole ? items : kShares;
    if (!whole) {
        w.o_bytes = (int64_t)2 * kShares * w.sh.rows * c.head_dim * 4;
        w.ml_bytes = (int64_t)2 * kShares * w.sh.rows * 8;
        w.cut_bytes = kShares * sizeof(Cut);
    }
    return w;
}

template <class E, int D>
void launch_dim(const mfft_cache& c, const mfft_attend_args& a, const AttendLaunch& w, hipStream_t s) {
    float* po = (float*)a.workspace;
    float2* ml = (float2*)((char*)a.workspace + w.o_bytes);
    Cut* cuts = (Cut*)((char*)ml + w.ml_bytes);
    const uint32_t grid = (uint32_t)w.grid;
    if (w.keys && w.r == 1) attend_kernel<E, D, 1, true><<<grid, 256, 0, s>>>(c, a, w.sh, po, ml, cuts);
    else if (w.keys) attend_kernel<E, D, 2, true><<<grid, 256, 0, s>>>(c, a, w.sh, po, ml, cuts);
    else if (w.r == 1) attend_kernel<E, D, 1, false><<<grid, 256, 0, s>>>(c, a, w.sh, po, ml, cuts);
    else if constexpr (D <= 128) attend_kernel<E, D, 2, false><<<grid, 256, 0, s>>>(c, a, w.sh, po, ml, cuts);
    mark(s);
    if (w.sh.grid) {
        join_kernel<E, D><<<kShares * w.sh.live, 256, 0, s>>>(c, a, w.sh, po, ml, cuts);
        mark(s);
    }
}

template <class E>
void launch_type(const mfft_cache& c, const mfft_attend_args& a, const AttendLaunch& w, hipStream_t s) {
    switch (c.head_dim) {
        case 64: launch_dim<E, 64>(c, a, w, s); break;
        case 96: launch_dim<E, 96>(c, a, w, s); break;
        case 128: launch_dim<E, 128>(c, a, w, s); break;
        case 256: launch_dim<E, 256>(c, a, w, s); break;
    }
}

}  // namespace

bool attend_supported(int head_dim) { return head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 256; }

int64_t attend_workspace(const mfft_cache& c, const mfft_attend_args& a) {
    const AttendLaunch w = attend_launch(c, a);
    return w.o_bytes + w.ml_bytes + w.cut_bytes;
}

bool attend_launch_fits(const mfft_cache& c, const mfft_attend_args& a) { return launch_fits(attend_launch(c, a).grid, 256); }

hipError_t launch_attend(const mfft_cache& c, const mfft_attend_args& a, hipStream_t stream) {
    const AttendLaunch w = attend_launch(c, a);
    if (a.dtype == MFFT_F16)
        launch_type<_Float16>(c, a, w, stream);
    else
        launch_type<__bf16>(c, a, w, stream);
    return hipGetLastError();
}

}  // namespace mfft

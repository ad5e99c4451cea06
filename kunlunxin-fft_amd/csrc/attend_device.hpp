// attend_device.hpp -- attention over the paged 8-bit cache: the kernels,
// templates of the part of the keys that a launch is about (attend.hpp).
//
// One pass over the keys a row of queries sees, with a running maximum m and
// sum l of exponentials: for each 64 keys s = scale * K q, m' = max(m, s),
// p = 2^(s - m'), l = l 2^(m - m') + sum p, O = O 2^(m - m') + V p, and
// out = O / l at the end (s in units of log 2; in float16 m is kept 14 lower,
// see Mat).
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
// Codes become the queries' type exactly (e4m3 fits both).  K's power-of-two
// scale goes into the 32-bit score.  V's goes in with the conversion to
// bfloat16, which holds every product; float16 does not, and there it goes into
// the weights, as the exponent it is, and is taken out of l again: 2^(s + e) V
// with 2^e the scale, m the maximum of s + e, l = sum 2^-e p.  The weights are
// rounded to the queries' type for the second product, as the matrix
// instructions need; maxima, sums and O are 32-bit.
//
// Bound: for few rows the codes' bytes (one token over 2^18 tokens of 8 heads
// of 128, 537 MB: 99 us, 5.4 TB/s), for many the products and, not overlapped
// with them, the softmax (2048 tokens of 32 heads over 32768: 1.18 ms, 910
// TFLOP/s; the products alone 732 us).
//
// A window's sinks are a second run of keys of the same pass: an item's list
// is the sinks' groups and then its own rows' windows, and nothing between is
// fetched.  One token of 64 sequences of up to 16384, window 4096 and 16 sinks,
// 4 key heads of 128, 207 MB: 44 us, 4.7 TB/s; 2048 tokens of 32 heads, window
// 4096 and 128 sinks: 178 us, 800 TFLOP/s.
//
// Keys that sequences share are a pass of their own in which all their rows are
// rows of one item, so that a code is fetched and decoded once for up to 128 of
// them instead of once a sequence; it leaves m, l and O, unscaled, from which
// each sequence's pass goes on: softmax is the same in any order of its keys.
// 64 sequences of one token, 32768 shared keys and 1 to 1000 of their own, 32
// query and 8 key heads of 128: 89 us (without, 2.1 million keys are read
// instead of 65 thousand); in a trace the launch over the shared keys, whose
// products are 25 us by the rate of a large matrix product, takes 62, the one over
// the own keys, 66 MB, 31, and the join, which finds nothing cut, 5.
#pragma once

#include <algorithm>

#include "attend.hpp"
#include "lm_device.hpp"
#include "mfft_device.hpp"

namespace mfft {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLowest = -3.402823466e38f;  // start of the running maximum: no score seen

// Up to here (in units of log 2) a score less its row's maximum is one fma of
// the unscaled score, whose maximum alone is rounded: weights are off by half a
// unit of the maximum's last place, 2^-13.5 of themselves at most (and not all
// alike: where keys are masked the product is rounded).  That is below what
// float16 rounds them by, and it grows with the scores until the largest weight
// is no number; past it the products are rounded before the difference, as the
// maximum is.
constexpr float kFusedScores = 4096.0f;

// a b, rounded whatever is done with it
__device__ __forceinline__ float product(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}

// ---- the two query types ----------------------------------------------------
// `offset`: what a row's weights are relative to, 2^(s - offset), from its
// largest score x.  l and O are relative to the same and out = O / l, so any
// offset gives the same row; m below is the offset.  In float16, whose least
// step is 2^-24, the largest weight is 2^14 instead of 1, so that those 2^-25
// to 2^-38 of it, which l counts, are not lost from O; the offset is the largest
// score less 14, and moves on once a score is past it by kMost, 15.  (A power of
// two, so that the type's rounding leaves a weight without others alone: a row
// that sees one key gives its value.)
// `large_offset`: the same past kFusedScores, where s + e below would be rounded
// and with it what one page's weights are to another's: from the scores alone,
// by 7 less, or as much less as still can be told from x.  Weights of any values
// that float16 holds (2^e to 2^8) stay in the type; values past 114688 overflow
// beside such scores, and those of pages below 2^-22 (2^-15 past 2^24) vanish.
// `shift`: the exponent of a V scale that goes into the weights.  Below 2^-40
// it is taken for that: such values are less than 2^-31, nothing in float16
// either way, and their 2^-e (a page of zeros has 2^126) stays within 32 bits.
template <class E>
struct Mat;
template <>
struct Mat<__bf16> {
    typedef bf16x8 x8;
    typedef bf16x2 x2;
    static __device__ __forceinline__ f32x4 mfma(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    template <bool HI>
    static __device__ __forceinline__ x2 decode(uint32_t w, float scale) {
        return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI);
    }
    static __device__ __forceinline__ float offset(float x) { return x; }
    static constexpr float kMost = 0.0f;
    static constexpr bool kShifts = false;
};
template <>
struct Mat<_Float16> {
    typedef f16x8 x8;
    typedef f16x2 x2;
    static __device__ __forceinline__ f32x4 mfma(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    template <bool HI>
    static __device__ __forceinline__ x2 decode(uint32_t w, float scale) {
        return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI);
    }
    static __device__ __forceinline__ float offset(float x) { return x - 14.0f; }
    static __device__ __forceinline__ float large_offset(float x) {
        const float y = x - 7.0f;
        return x - y <= 7.0f ? y : x;
    }
    static constexpr float kMost = 15.0f;
    static constexpr bool kShifts = true;
    static __device__ __forceinline__ int shift(float scale) { return max((int)(__float_as_uint(scale) >> 23) - 127, -40); }
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

// A row's offset m, from its largest score (plus e) x and, once `large`, from its
// largest score alone, which `score` finds.
template <class M, class S>
__device__ __forceinline__ float moved_on(float m, float x, bool& large, S&& score) {
    float to = M::offset(x);
    large |= __any(__builtin_fabsf(x) > kFusedScores && x > kLowest);
    if constexpr (M::kShifts) {
        if (large) {
            const float y = score();
            if (__builtin_fabsf(y) > kFusedScores) to = M::large_offset(y);
        }
    }
    return __builtin_fmaxf(m, to);
}

// Whether a row that goes on from offset m may have scores past kFusedScores:
// its largest lies at most kMost above m (float16's is the larger), and m is
// rounded.
__device__ __forceinline__ bool carried_large(float m) {
    return __any(m > kLowest && __builtin_fabsf(m) > kFusedScores - (Mat<_Float16>::kMost + 1.0f));
}

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

// the larger of v in lanes l and l ^ 32 (l ^ 16): the swaps exchange the upper
// half (odd rows of sixteen) of one register with the lower (even) of another
__device__ __forceinline__ float max_across_32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_across_16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
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
// form one list, and each of `grid` workgroups takes an equal share of it,
// whatever the lengths are: a share is some whole items and at most two cut
// ones, at its ends.  (An item is charged all its sequence's groups from the
// window of the first query on, also those that only later or earlier blocks of
// rows see, which it leaves out.  Shares of a prompt piece over many cached
// keys are so within a few percent of equal; those of a prompt of which nothing
// is cached are not: 8192 tokens of 32 heads 1.04 ms, 530 TFLOP/s, where 2048
// over 32768 reach 910; nor those of a long piece in a short window: 2048
// tokens in one of 512, 43 us.)  The list follows from the
// lengths, which only the device knows; every workgroup works its place out for
// itself with one pass of a wave over the sequences.  Cut items leave their
// (m, l, O) in the workspace and join_kernel adds them up.
struct Sequence {
    int row0, n;      // its queries
    int len;          // its keys, within the table
    bool poison;      // it has more than the table's
    int low, tiles;   // first key that any query sees (a multiple of 64), groups of 64 keys in the list
    int blocks;       // of rows
    int prefix, shared_by;  // kRest: keys that are not its own, and the group whose they are
    int first, last;  // kPrefix: its sequences
};

// Keys that group g of sequences shares: whole pages.
__device__ __forceinline__ int prefix_keys(const mfft_cache& c, const mfft_attend_args& a, const PartShape& sh, int g) {
    return min(max(sh.prefix_pages[g], 0), a.table_width) * c.page_size;
}
__device__ __forceinline__ int group_start(const mfft_attend_args& a, const PartShape& sh, int g) {
    const int b = sh.prefix_groups ? sh.prefix_groups[g] : g * a.sequences;
    return min(max(b, 0), a.sequences);
}

// kPrefix: group b as the kernels take a sequence: its rows are all its
// sequences' rows, its keys the shared ones.
template <Part PART>
__device__ __forceinline__ Sequence sequence(const mfft_cache& c, const mfft_attend_args& a, const ShapeOf<PART>& sh, int b) {
    Sequence q{};
    if constexpr (PART == kPrefix) {
        q.first = group_start(a, sh, b);
        q.last = group_start(a, sh, b + 1);
        q.len = prefix_keys(c, a, sh, b);
        q.row0 = (int)seq_offset(a.offsets, sh.per, a.tokens, q.first);
        if (q.last > q.first && q.len > 0) q.n = max((int)seq_offset(a.offsets, sh.per, a.tokens, q.last) - q.row0, 0);
        q.tiles = max((q.len + 63) >> 6, 1);
        q.blocks = (q.n * sh.group + (1 << sh.prefix.log_rows) - 1) >> sh.prefix.log_rows;
        return q;
    }
    q.row0 = (int)seq_offset(a.offsets, sh.per, a.tokens, b);
    q.n = (int)seq_offset(a.offsets, sh.per, a.tokens, b + 1) - q.row0;
    if (q.n < 0) q.n = 0;
    const int most = a.table_width * c.page_size;
    const int len = a.lengths[b];
    q.poison = len > most;
    q.len = len < 0 ? 0 : q.poison ? most : len;
    q.low = 0;
    if (a.window) {
        const int lo = q.len - q.n + 1 - (int)a.window;
        q.low = lo > 0 ? lo & ~63 : 0;
    }
    if constexpr (PART == kRest) {
        // the last group that starts at or before b
        int g = 0, hi = sh.groups - 1;
        while (g < hi) {
            const int mid = (g + hi + 1) >> 1;
            if (group_start(a, sh, mid) <= b) g = mid;
            else hi = mid - 1;
        }
        if (group_start(a, sh, g) <= b && b < group_start(a, sh, g + 1)) q.prefix = prefix_keys(c, a, sh, g);
        q.shared_by = g;
        q.low = min(q.prefix, q.len) & ~63;
    }
    q.tiles = (q.len - q.low + 63) >> 6;
    if constexpr (PART == kSinks) {
        // of a block: its own rows' windows and the sinks, not all the sequence's
        const int tokens = min(sh.block_tokens, q.n);
        if (a.causal) q.tiles = min(q.tiles, ((int)a.window + tokens + 62 + 63) >> 6);
        q.tiles = min(q.tiles + ((sh.sinks + 63) >> 6), (q.len + 63) >> 6);
    }
    if (q.tiles < 1) q.tiles = 1;  // rows that see nothing are still written
    q.blocks = (q.n * sh.group + sh.rows - 1) >> sh.log_rows;
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

// v is loaded by here.  A loop that uses v, loaded before it, otherwise waits in
// every round for all loads, those for its next round among them: the waits are
// placed for the first round.
template <class V>
__device__ __forceinline__ void loaded(V& v) {
    asm volatile("" : "+v"(v));
}

// floor(x / d) of 0 <= x < 2^52, d > 0, the same in all lanes: a double's
// quotient is off by one at most
__device__ __forceinline__ int64_t quotient(int64_t x, int d) {
    int64_t q = (int64_t)((double)x / (double)d);
    if (q * d > x) --q;
    if ((q + 1) * d <= x) ++q;
    return uniform(q);
}

// sum over the wave up to and including this lane, without LDS: within sixteen
// lanes by row shifts, then the rows before by broadcasts of their last lane
__device__ __forceinline__ int64_t wave_scan(int64_t v) {
    auto step = [&](auto ctrl, auto rows) {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
        v += (int64_t)((uint64_t)hi << 32 | lo);
    };
    step(ic<0x111>{}, ic<0xf>{});  // row_shr 1, 2, 4, 8
    step(ic<0x112>{}, ic<0xf>{});
    step(ic<0x114>{}, ic<0xf>{});
    step(ic<0x118>{}, ic<0xf>{});
    step(ic<0x142>{}, ic<0xa>{});  // row_bcast 15 into rows 1 and 3, 31 into 2 and 3
    step(ic<0x143>{}, ic<0xc>{});
    return v;
}
__device__ __forceinline__ int64_t from_lane(int64_t v, int l) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)v, l), hi = (uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l);
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// The list of all work: groups of keys (or items, where `by_item`), sequence
// after sequence, 64 sequences at a time.
template <Part PART>
struct WorkList {
    const mfft_cache& c;
    const mfft_attend_args& a;
    const ShapeOf<PART>& sh;
    bool by_item;
    int64_t w, upto;  // of the 64 sequences at hand: this lane's, and with those before
    int most = 0;     // kRest: this lane's longest item
    int items = 0;    // and its items of the 64 sequences at hand

    __device__ __forceinline__ int count() const {
        if constexpr (PART == kPrefix) return sh.groups;
        return a.sequences;
    }
    __device__ __forceinline__ void take(int i) {
        const int b = i + (int)(threadIdx.x & 63);
        w = 0;
        if (b < count()) {
            const Sequence q = sequence<PART>(c, a, sh, b);
            w = (int64_t)q.blocks * c.kv_heads * (by_item ? 1 : q.tiles);
            if constexpr (PART == kRest) {
                if (q.blocks > 0) most = max(most, q.tiles);
                items = q.blocks * c.kv_heads;
            }
        }
        upto = wave_scan(w);
    }
    __device__ __forceinline__ int64_t total() {
        int64_t t = 0;
        for (int i = 0; i < count(); i += 64) {
            take(i);
            t += from_lane(upto, 63);
        }
        return t;
    }
    // the sequence in whose work place `at` lies, and what comes before it;
    // -1 past the end.  `taken`: the first 64 sequences are at hand.
    __device__ __forceinline__ int find(int64_t at, int64_t& before, bool taken) {
        before = 0;
        for (int i = 0; i < count(); i += 64) {
            if (!taken) take(i);
            taken = false;
            const uint64_t hit = __ballot(before + upto > at);
            if (hit) {
                const int l = __builtin_ctzll(hit);
                before += from_lane(upto, l) - from_lane(w, l);
                return uniform(i + l);
            }
            before += from_lane(upto, 63);
        }
        return -1;
    }
};

// ---- one item, some of its keys --------------------------------------------------
// What every form of the kernel needs of its item: pages and bounds.
template <int D, Part PART>
struct Item {
    const mfft_cache& c;
    const mfft_attend_args& a;
    const ShapeOf<PART>& sh;
    Sequence seq;
    const int32_t* table;
    int h;
    int all, block;  // rows of the sequence and key head, first row of the block
    int block_lo, block_hi, block_all_lo, block_all_hi;  // keys that any, and that all, rows of the block see
    bool all_see, some_blind;  // kPrefix: every row but blind ones sees all keys; there are blind ones

    __device__ __forceinline__ Item(const mfft_cache& c_, const mfft_attend_args& a_, const ShapeOf<PART>& sh_) : c(c_), a(a_), sh(sh_) {}

    // the keys [lower, upper) that query `tok` of the sequence sees (kSinks: and
    // those of sink_keys)
    __device__ __forceinline__ int lower(int tok) const {
        if constexpr (PART == kPrefix) return 0;
        if constexpr (PART == kRest) return seq.prefix;
        return a.window ? max(seq.len - seq.n + tok + 1 - (int)a.window, 0) : 0;
    }
    __device__ __forceinline__ int upper(int tok) const {
        if constexpr (PART == kPrefix) {  // of its own sequence, as far as they are shared; 0: see `blind`
            int lo = seq.first, hi = seq.last - 1;
            if (!a.offsets) lo = (seq.row0 + tok) / sh.by_per;
            else
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (seq_offset(a.offsets, 1, a.tokens, mid) <= seq.row0 + tok) lo = mid;
                    else hi = mid - 1;
                }
            return min(seen_by(lo, seq.row0 + tok), seq.len);
        }
        return a.causal ? max(min(seq.len - seq.n + tok + 1, seq.len), 0) : seq.len;
    }
    // kPrefix: the keys that row `row` of the call, of sequence b, sees: up to here
    __device__ __forceinline__ int seen_by(int b, int row) const {
        const int len = min(max(a.lengths[b], 0), a.table_width * c.page_size);
        if (!a.causal) return len;
        return max(min(len - (int)seq_offset(a.offsets, sh.per, a.tokens, b + 1) + row + 1, len), 0);
    }
    // kRest: items of kPrefix that come before the group's
    __device__ __forceinline__ int prefix_items() const {
        int64_t blocks = 0;
        for (int g = (int)(threadIdx.x & 63); g < seq.shared_by; g += 64) blocks += sequence<kPrefix>(c, a, sh, g).blocks;
        return seq.shared_by ? (int)(from_lane(wave_scan(blocks), 63) * c.kv_heads) : 0;
    }
    // Where the shared keys' m, l and O of a row (token tok of the sequence, query
    // head qh) are: in `parts` rows of the prefix's workspace, the first and those
    // after it `step` apart; 0: one row of `carry`.
    struct Carried {
        int parts;
        int64_t first, second, step;
        __device__ __forceinline__ int64_t at(int p) const { return p == 0 ? first : second + (p - 1) * step; }
    };
    __device__ __forceinline__ Carried carried(int items, int tok, int qh) const {
        const int64_t row = (int64_t)(seq.row0 + tok) * a.q_heads + qh;
        if (sh.prefix.grid == 0) return {0, row, 0, 0};
        const int start = (int)seq_offset(a.offsets, sh.per, a.tokens, group_start(a, sh, seq.shared_by));
        const int end = (int)seq_offset(a.offsets, sh.per, a.tokens, group_start(a, sh, seq.shared_by + 1));
        const int r = (seq.row0 + tok - start) * sh.group + qh - h * sh.group, rows = 1 << sh.prefix.log_rows;
        const int64_t number = items + (int64_t)(r >> sh.prefix.log_rows) * c.kv_heads + h;
        // (offsets that do not rise, or groups that overlap: any row there is)
        if (seq.row0 + tok < start || seq.row0 + tok >= end || number >= sh.prefix.items) return {0, row, 0, 0};
        const Cut cut = sh.prefix.cuts[number];
        if (cut.parts == 0) return {0, row, 0, 0};
        const int64_t slot = 2 * (int64_t)cut.h;  // cut.h: its share
        return {cut.parts, (slot + 1) * rows + (r & (rows - 1)), (slot + 2) * rows + (r & (rows - 1)), 2 * (int64_t)rows};
    }
    // kSinks: of rows that see [.., top) the keys [0, sink_keys(top)) too
    __device__ __forceinline__ int sink_keys(int top) const {
        if constexpr (PART == kSinks) return min(sh.sinks, top);
        return 0;
    }
    // (not a comparison with 0 elsewhere: that a key's number is not negative the
    // compiler does not know)
    __device__ __forceinline__ bool in_sinks(int key, int top) const { return PART == kSinks && key < sink_keys(top); }

    // The keys of groups [tile, upto) of the item's list that rows of the block
    // see, as one run [from, end) of places.  The place of a key is its number;
    // kSinks: the sinks' groups come first and the block's windows follow, from
    // `split` on, their numbers less `gap`.
    int split, gap;
    __device__ __forceinline__ int key_at(int place) const { return PART != kSinks || place < split ? place : place + gap; }
    __device__ __forceinline__ void span(int tile, int upto, int& from, int& end) {
        if constexpr (PART != kSinks) {
            from = max(seq.low + 64 * tile, block_lo & ~63);
            end = min(seq.low + 64 * upto, block_hi);
            return;
        }
        split = min((sink_keys(block_hi) + 63) & ~63, block_lo & ~63);
        gap = (block_lo & ~63) - split;
        from = 64 * tile;
        end = min(64 * upto, block_hi - gap);
    }

    __device__ __forceinline__ void take(int b, int block_, int h_, int rows) {
        h = h_;
        all = seq.n * sh.group;
        block = block_ * rows;
        nan_left = false;
        if constexpr (PART == kPrefix) {
            // The shared pages stand in all its sequences' rows of the table; taken
            // are those of the first that is long enough (an empty one may name
            // none), or else of the longest.
            int from = -1, long_one = 0, long_len = -1;
            all_see = true;
            some_blind = false;
            for (int s0 = seq.first; s0 < seq.last; s0 += 64) {
                const int s = min(s0 + (int)(threadIdx.x & 63), seq.last - 1);
                const int row = (int)seq_offset(a.offsets, sh.per, a.tokens, s);
                const int len = min(max(a.lengths[s], 0), a.table_width * c.page_size);
                const bool rows = (int)seq_offset(a.offsets, sh.per, a.tokens, s + 1) > row;
                const uint64_t fits = __ballot(len >= seq.len);
                if (from < 0 && fits) from = min(s0 + (int)__builtin_ctzll(fits), seq.last - 1);
                some_blind |= __any(len == 0 && rows);
                all_see &= !__any(len > 0 && rows && seen_by(s, row) < seq.len);
                if (from < 0 && len > long_len) {
                    long_len = len;
                    long_one = s;
                }
            }
            block_lo = block_all_lo = 0;
            block_hi = block_all_hi = seq.len;
            if (from < 0) {
#pragma unroll
                for (int s = 1; s < 64; s <<= 1) {
                    const int len = __shfl_xor(long_len, s), one = __shfl_xor(long_one, s);
                    if (len > long_len || (len == long_len && one < long_one)) {
                        long_len = len;
                        long_one = one;
                    }
                }
                from = uniform(long_one);
                block_hi = uniform(long_len);
            }
            table = a.page_table + from * a.table_stride;
            // rows that see not all: what all rows of a block see is not looked for
            if (!all_see) block_all_hi = 0;
            return;
        }
        table = a.page_table + b * a.table_stride;
        // both ends of what a row sees rise with it
        const int t0 = block / sh.by_group, t1 = (min(block + rows, all) - 1) / sh.by_group;
        block_lo = lower(t0);
        block_hi = upper(t1);
        block_all_lo = lower(t1);
        block_all_hi = upper(t0);
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
    // Values of a group where not every row sees every key.  Keys that no row
    // sees may hold anything: their codes count as 0 (`keep` masks the others).
    // A NaN of the others counts only for the rows that see its key, while 0 * NaN
    // is NaN: its code becomes 0 here, and mark_nans() finds the rows that see
    // it once the item is done.
    bool nan_left;
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

    __device__ __forceinline__ bool block_edge(int key0) const { return key0 < block_all_lo || key0 + 64 > block_all_hi; }
};

// KEYS: the workgroup's four waves share 16 R rows and take every fourth group
// of 64 keys, each straight from memory into registers, one group ahead; their
// (m, l, O) are joined in LDS.  For few rows: nothing but the cache's bytes
// counts, and a wave's loads wait for no other wave (32 sequences of 4000, 32
// rows of 128: 59 us so, 78 us through LDS).
// not KEYS: each wave has 16 R rows of its own and all take every group, which
// goes through LDS once for the four.  For many rows.
template <class E, int D, int R, bool KEYS, Part PART>
struct Attend : Item<D, PART> {
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

    using I = Item<D, PART>;
    using I::a, I::c, I::sh, I::seq, I::h, I::all, I::block, I::nan_left;
    Lds& lds;
    int lane, wave, j, g, kg, kr;

    // of the item
    x8 qv[R][S::KK];
    int low[R], top[R];                // keys [low, top) that each of this lane's rows sees
    int all_lo, all_hi, any_lo, any_hi;  // and all, and any, of the wave's rows
    f32x4 o[R][S::N];
    float m[R], l[R];
    bool large;                        // some row's maximum has been past kFusedScores
    // kPrefix: rows that see none of the keys (of an empty place in a batch, say)
    // go through the loop as if they saw all, so that a group's other rows need no
    // masks, and are cleared at its end
    bool blind[R];

    // of the group at hand
    u32x4 kw[4][S::J > 0 ? S::J : 1];
    u32x2 kx[4];
    u32x4 vw[S::N];
    float cs, vs;
    int ve = 0;

    __device__ __forceinline__ Attend(const mfft_cache& c_, const mfft_attend_args& a_, const ShapeOf<PART>& sh_, Lds& lds_)
        : I(c_, a_, sh_), lds(lds_) {
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        j = lane & 15;
        g = lane >> 4;
        kg = j >> 2;  // K rows of lane j: keys 16 kg + 4 t + kr
        kr = j & 3;
    }

    __device__ __forceinline__ int row_of(int r, int j) const { return block + (KEYS ? 0 : 16 * R * wave) + 16 * r + j; }

    __device__ __forceinline__ void begin(int b, int block_, int h_) {
        this->take(b, block_, h_, ROWS);
        all_lo = 0;
        all_hi = seq.len;
        any_lo = seq.len;
        any_hi = 0;
        large = false;
        const int j = here(this->j), g = here(this->g);
        static_for<0, R>([&](auto r) {
            const int row = min(row_of(r.value, j), all - 1);  // rows past the last repeat it and are not stored
            const int tok = row / sh.by_group;
            const int qh = h * sh.group + row - tok * sh.group;
            const E* q = (const E*)a.q + (seq.row0 + tok) * a.q_strides[0] + qh * a.q_strides[1];
            static_for<0, S::J>([&](auto jj) {
                qv[r.value][2 * jj.value] = *(const x8*)(q + 64 * jj.value + 16 * g);
                qv[r.value][2 * jj.value + 1] = *(const x8*)(q + 64 * jj.value + 16 * g + 8);
            });
            if constexpr (S::REM) qv[r.value][S::KK - 1] = *(const x8*)(q + 64 * S::J + 8 * g);
            const int lo = this->lower(tok);
            int hi = this->block_hi;
            if constexpr (PART == kPrefix) {
                blind[r.value] = false;
                if (!this->all_see || this->some_blind) {
                    hi = this->upper(tok);
                    blind[r.value] = hi == 0;
                    if (hi == 0) hi = this->block_hi;
                }
            } else {
                hi = max(this->upper(tok), lo);
            }
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
        static_for<0, R>([&](auto r) { static_for<0, S::KK>([&](auto i) { loaded(qv[r.value][i.value]); }); });
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

    __device__ __forceinline__ void clear_blind() {
        static_for<0, R>([&](auto r) {
            if (blind[r.value]) {
                m[r.value] = kLowest;
                l[r.value] = 0.0f;
                static_for<0, S::N>([&](auto i) { o[r.value][i.value] = f32x4{0, 0, 0, 0}; });
            }
        });
    }
    // kRest: the shared keys' m, l and O, for the part of the item that has its
    // first key.  KEYS: the waves take every fourth part, as of the keys.
    __device__ __forceinline__ void carry_in() {
        constexpr int STRIDE = KEYS ? 4 : 1, U = 4;
        const int items = this->prefix_items();
        const int j = here(this->j), g = here(this->g);
        static_for<0, R>([&](auto r) {
            const int row = row_of(r.value, j);
            if (row < all) {
                const int tok = row / sh.by_group;
                const auto from = this->carried(items, tok, h * sh.group + row - tok * sh.group);
                const float* po = from.parts ? sh.prefix.part_o : sh.carry_o;
                const float2* pml = from.parts ? sh.prefix.part_ml : sh.carry_ml;
                const int parts = max(from.parts, 1);
                for (int p0 = KEYS ? wave : 0; p0 < parts; p0 += U * STRIDE) {
                    float2 ml[U];
                    f32x4 w[U][S::N];
                    static_for<0, U>([&](auto u) {  // (past the last: the last again, weighed 0)
                        const int64_t at = from.at(min(p0 + u.value * STRIDE, parts - 1));
                        ml[u.value] = pml[at];
                        static_for<0, S::N>([&](auto i) { w[u.value][i.value] = *(const f32x4*)(po + at * D + 16 * i.value + 4 * g); });
                    });
                    float to = m[r.value];
                    static_for<0, U>([&](auto u) { to = __builtin_fmaxf(to, ml[u.value].x); });
                    const float shrink = __builtin_amdgcn_exp2f(m[r.value] - to);
                    m[r.value] = to;
                    l[r.value] *= shrink;
                    static_for<0, S::N>([&](auto i) { o[r.value][i.value] *= shrink; });
                    static_for<0, U>([&](auto u) {
                        const float f = p0 + u.value * STRIDE < parts ? __builtin_amdgcn_exp2f(ml[u.value].x - to) : 0.0f;
                        if (g == 0) l[r.value] += ml[u.value].y * f;  // (a lane's part of the sum)
                        static_for<0, S::N>([&](auto i) { o[r.value][i.value] += w[u.value][i.value] * f; });
                    });
                }
            }
            large |= carried_large(m[r.value]);
        });
    }

    // the scales of this lane's sixteen keys, as loaded, and as they count:
    // scores in units of log 2, NaN for a page number that is none.  Those of
    // keys that no row sees may be anything (pages before the window that the
    // caller has given to others, the stand-in past the end) and must not
    // count: scores are masked one by one, and values' codes are 0 there.
    float ks_raw, vs_raw;
    bool bad_page;
    __device__ __forceinline__ void load_scales(int entry) {
        const int64_t at = this->page_of(entry) * c.kv_heads + h;
        ks_raw = c.k_scale[at];
        vs_raw = c.v_scale[at];
        bad_page = (uint32_t)entry >= (uint32_t)c.pages;
    }
    __device__ __forceinline__ void take_scales(int key0) {
        const int kv = key0 + 16 * g;
        vs = (kv + 16 > any_lo && kv < any_hi) || this->in_sinks(kv, any_hi) ? vs_raw : 1.0f;
        bool bad = bad_page;
        if constexpr (M::kShifts) {
            ve = M::shift(vs);
            bad |= !(vs < __builtin_inff());
            vs = 1.0f;
        }
        cs = bad ? __builtin_nanf("") : a.scale * 1.44269504088896340736f * ks_raw;
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
        });
    }

    // P from S, m and l moved on, O rescaled where m grew
    __device__ __forceinline__ void weights(f32x4 (&s)[R][4], x8 (&p)[R][2], bool at_edge, int kv) {
        const float unit = at_edge ? 1.0f : cs;
        static_for<0, R>([&](auto r) {
            if (at_edge) {
                // bit i: key kv + i is seen; as masks of whole words, which
                // take no condition registers
                const int lo = min(max(low[r.value] - kv, 0), 16), hi = min(max(top[r.value] - kv, 0), 16);
                int seen = (int)((1u << hi) - (1u << lo));
                if constexpr (PART == kSinks) seen |= (int)((1u << min(max(this->sink_keys(top[r.value]) - kv, 0), 16)) - 1);
                static_for<0, 16>([&](auto i) {
                    const uint32_t bit = (uint32_t)((seen << (31 - i.value)) >> 31);
                    const uint32_t v = __float_as_uint(s[r.value][i.value / 4][i.value % 4] * cs);
                    s[r.value][i.value / 4][i.value % 4] = __uint_as_float((v & bit) | (0xff800000u & ~bit));
                });
            }
            float mx = s[r.value][0][0];
            static_for<1, 16>([&](auto i) { mx = __builtin_fmaxf(mx, s[r.value][i.value / 4][i.value % 4]); });
            const float x = max_across_32(max_across_16(__builtin_fmaf(mx, unit, (float)ve)));
            if ((M::kShifts && large) || __any(x > m[r.value] + M::kMost)) {
                const float to = moved_on<M>(m[r.value], x, large, [&] { return max_across_32(max_across_16(product(mx, unit))); });
                const float shrink = __builtin_amdgcn_exp2f(m[r.value] - to);
                m[r.value] = to;
                l[r.value] *= shrink;
                static_for<0, S::N>([&](auto i) { o[r.value][i.value] *= shrink; });
            }
        });
        float from[R], by = unit;
        static_for<0, R>([&](auto r) { from[r.value] = (float)ve - m[r.value]; });
        if (large) {
            static_for<0, R>([&](auto r) {
                static_for<0, 16>([&](auto i) {
                    s[r.value][i.value / 4][i.value % 4] = product(s[r.value][i.value / 4][i.value % 4], unit) - m[r.value];
                });
                from[r.value] = (float)ve;
            });
            by = 1.0f;
        }
        static_for<0, R>([&](auto r) {
            float sum = M::kShifts ? 0.0f : l[r.value];
            static_for<0, 16>([&](auto i) {
                const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r.value][i.value / 4][i.value % 4], by, from[r.value]));
                sum += w;
                p[r.value][i.value / 8][i.value % 8] = (E)w;
            });
            l[r.value] = M::kShifts ? l[r.value] + __builtin_ldexpf(sum, -ve) : sum;
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
        });
    }

    // (a group in LDS is cleaned for all four waves' rows at once)
    __device__ __forceinline__ bool edge(int key0) const {
        return KEYS ? key0 < all_lo || key0 + 64 > all_hi : this->block_edge(key0);
    }

    // (rare, and so key by key from memory, after the loop it would slow down)
    __device__ __forceinline__ void mark_nans(int from, int end) {
        if (!__any(nan_left)) return;
        const int g = here(this->g);
#pragma unroll 1
        for (int place = from; place < end; ++place) {
            const int key = this->key_at(place), key0 = key & ~63;
            if (!edge(key0) || (KEYS && (((place & ~63) - from) / 64) % 4 != wave)) continue;
            const uint32_t u = (uint32_t)key >> 4;
            const uint8_t* vb = (const uint8_t*)c.v + this->unit_at(this->page_entry(u), u) + 64 * g + (key & 15);
            static_for<0, S::N>([&](auto i) {
                static_for<0, 4>([&](auto x) {
                    if ((vb[16 * (16 * i.value + x.value)] & 0x7f) == kNaNCode) {
                        static_for<0, R>([&](auto r) {
                            if ((key >= low[r.value] && key < top[r.value]) || this->in_sinks(key, top[r.value]))
                                o[r.value][i.value][x.value] = __builtin_nanf("");
                        });
                    }
                });
            });
        }
    }

    // ---- the waves share the rows
    __device__ __forceinline__ void load_keys(int key0, int entry) {
        const uint8_t* kb = (const uint8_t*)c.k + this->unit_at(entry, (uint32_t)(key0 >> 4) + kg) + kr * D;
        static_for<0, 4>([&](auto t) {
            static_for<0, S::J>([&](auto jj) { kw[t.value][jj.value] = *(const u32x4*)(kb + 4 * t.value * D + 64 * jj.value + 16 * g); });
            if constexpr (S::REM) kx[t.value] = *(const u32x2*)(kb + 4 * t.value * D + 64 * S::J + 8 * g);
        });
    }
    __device__ __forceinline__ void load_values(int key0, int entry) {
        const uint8_t* vb = (const uint8_t*)c.v + this->unit_at(entry, (uint32_t)(key0 >> 4) + g) + 16 * j;
        static_for<0, S::N>([&](auto i) { vw[i.value] = *(const u32x4*)(vb + i.value * 256); });
    }

    __device__ __forceinline__ void run_keys(int from, int end) {
        int place = from + 64 * wave;
        // Loads come back in order, so each is issued before those that need
        // not wait for it: table entries two groups ahead, then scales and K
        // of the next, and V once this group's is used up.
        int k1 = 0, v1 = 0, k2 = 0, v2 = 0;
        auto entries = [&](int place, int& k, int& v) {
            const int k0 = this->key_at(place);
            k = this->page_entry((uint32_t)(k0 >> 4) + kg);
            v = this->page_entry((uint32_t)(k0 >> 4) + g);
        };
        if (place < end) {
            entries(place, k1, v1);
            entries(place + STEP, k2, v2);
            load_scales(v1);
            load_keys(this->key_at(place), k1);
            load_values(this->key_at(place), v1);
        }
        for (; place < end; place += STEP) {
            const int key0 = this->key_at(place);
            f32x4 s[R][4];
            x8 p[R][2];
            take_scales(key0);
            scores(s, [&](auto t, auto jj) { return kw[t.value][jj.value]; }, [&](auto t) { return kx[t.value]; });
            const bool more = place + STEP < end;
            k1 = k2;
            v1 = v2;
            if (more) {
                entries(place + 2 * STEP, k2, v2);
                load_scales(v1);
                load_keys(this->key_at(place + STEP), k1);
            }
            const int kv = key0 + 16 * g;
            weights(s, p, edge(key0), kv);
            if (edge(key0)) {
                u32x4 keep = keep_bytes(any_lo - kv, any_hi - kv);
                if constexpr (PART == kSinks) keep |= keep_bytes(-kv, this->sink_keys(any_hi) - kv);
                static_for<0, S::N>([&](auto i) { vw[i.value] = this->clean(vw[i.value], keep); });
            }
            values(p, [&](auto i) { return vw[i.value]; });
            if (more) load_values(this->key_at(place + STEP), v1);
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
        const int64_t at = this->unit_at(entry, (uint32_t)(key0 >> 4) + wave);
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
            u32x4 keep = keep_bytes(this->block_lo - kv, this->block_hi - kv);
            if constexpr (PART == kSinks) keep |= keep_bytes(-kv, this->sink_keys(this->block_hi) - kv);
            static_for<0, L>([&](auto x) {
                // (what a lane has not fetched may look like a NaN, and then all of the
                // block's keys were looked through for it)
                if (D % 64 == 0 || lane + 64 * x.value < D) fv[x.value] = this->clean(fv[x.value], keep);
            });
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
        __syncthreads();  // a share's last item may still be read
        if (threadIdx.x == 0) lds.nan = 0;
        __syncthreads();
        int e1 = 0, v1 = 0;  // table entries of the next group, fetched and of this lane's keys
        auto entries = [&](int place) {
            const int k0 = this->key_at(place);
            e1 = this->page_entry((uint32_t)(k0 >> 4) + wave);
            v1 = this->page_entry((uint32_t)(k0 >> 4) + g);
        };
        if (from < end) {
            entries(from);
            load_scales(v1);
            fetch(this->key_at(from), e1);
            entries(from + 64);
            stash(0, this->key_at(from));
        }
        int buf = 0;
        for (int place = from; place < end; place += 64) {
            const int key0 = this->key_at(place);
            __syncthreads();
            const bool more = place + 64 < end;
            take_scales(key0);
            if (more) {
                load_scales(v1);
                const int e0 = e1;
                entries(place + 128);
                fetch(this->key_at(place + 64), e0);
            }
            if ((key0 + 64 > any_lo && key0 < any_hi) || this->in_sinks(key0, any_hi)) {
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
            if (more) stash(buf, this->key_at(place + 64));
        }
        __syncthreads();
        nan_left = lds.nan != 0;
        mark_nans(from, end);
        static_for<0, R>([&](auto r) {
            l[r.value] += __shfl_xor(l[r.value], 16);
            l[r.value] += __shfl_xor(l[r.value], 32);
        });
    }

    __device__ __forceinline__ void run(int tile, int upto) {
        int from, end;
        if constexpr (KEYS && PART == kAll) {
            // the waves share the block's rows: what any of them sees is at hand
            from = max(seq.low + 64 * tile, any_lo & ~63);
            end = min(seq.low + 64 * upto, any_hi);
        } else {
            this->span(tile, upto, from, end);
        }
        if constexpr (KEYS) run_keys(from, end);
        else run_rows(from, end);
        if constexpr (PART == kPrefix) clear_blind();
    }

    // ---- out of the registers
    __device__ __forceinline__ void store() const {
        if (KEYS && wave > 0) return;
        const int j = here(this->j), g = here(this->g);
        static_for<0, R>([&](auto r) {
            const int row = row_of(r.value, j);
            if (row >= all) return;
            const int place = row / sh.by_group;
            const int64_t tok = seq.row0 + place;
            const int qh = h * sh.group + row - place * sh.group;
            if constexpr (PART == kPrefix) {
                const int64_t at = tok * a.q_heads + qh;
                static_for<0, S::N>([&](auto i) { *(f32x4*)(sh.carry_o + at * D + 16 * i.value + 4 * g) = o[r.value][i.value]; });
                if (g == 0) sh.carry_ml[at] = make_float2(m[r.value], l[r.value]);
                return;
            }
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
            const int row = row_of(r.value, j);
            if (row >= all) return;
            const int64_t at = (int64_t)slot * ROWS + (row - block);
            static_for<0, S::N>([&](auto i) { *(f32x4*)(part_o + at * D + 16 * i.value + 4 * g) = o[r.value][i.value]; });
            if (g == 0) part_ml[at] = make_float2(m[r.value], l[r.value]);
        });
    }
};

// Many rows: a wave has 32 of its own, as columns of v_mfma 32x32x16, and the
// four waves of a workgroup take every group of 64 keys together.  Each wave
// fetches sixteen keys of it, decodes them and leaves them in LDS as the
// queries' type, so that a code is decoded once for 128 rows.
// A lane l = 32 e + n holds, of D = A B, column n of rows 8 x + 4 e .. + 3, and
// of A (B) contraction indices 8 e .. 8 e + 7; row 8 x + 4 e + y of the t-th of
// the two products S^T = K Q^T is key 32 t + 16 e + 4 x + y, so that again the
// sixteen scores of a lane are sixteen keys in order, and its weights are its
// contraction indices of P^T.
template <class E, int D, Part PART>
struct Tall : Item<D, PART> {
    using I = Item<D, PART>;
    using I::a, I::c, I::sh, I::seq, I::h, I::all, I::block, I::nan_left;
    using M = Mat<E>;
    typedef typename M::x8 x8;
    static constexpr int ROWS = 128;
    // keys: rows 16 bytes apart and 128 more after each sixteen, so that the
    // sixteen rows a load takes at once (keys 0 .. 7 and 16 .. 23, or 8 .. 15
    // and 24 .. 31) lie in different banks; values: eight tokens of a channel
    // (16 bytes), then the next channel
    static constexpr int KROW = 2 * D + 16, KLDS = 64 * KROW + 4 * 128, VLDS = 64 * 2 * D;
    struct Lds {
        uint8_t k[2][KLDS], v[2][VLDS];
        int nan;
    };
    Lds& lds;
    int lane, wave, n, e;

    x8 qv[D / 16];
    int low, top, all_lo, all_hi, any_lo, any_hi;
    f32x16 o[D / 32];
    float m, l;
    bool large;  // some row's maximum has been past kFusedScores
    bool blind;  // see Attend

    __device__ __forceinline__ Tall(const mfft_cache& c_, const mfft_attend_args& a_, const ShapeOf<PART>& sh_, Lds& lds_)
        : I(c_, a_, sh_), lds(lds_) {
        lane = threadIdx.x & 63;
        wave = uniform((int)(threadIdx.x >> 6));
        n = lane & 31;
        e = lane >> 5;
    }

    __device__ __forceinline__ void begin(int b, int block_, int h_) {
        this->take(b, block_, h_, ROWS);
        const int n = here(this->n), e = here(this->e);
        const int row = min(block + 32 * wave + n, all - 1);
        const int tok = row / sh.by_group;
        const int qh = h * sh.group + row - tok * sh.group;
        const E* q = (const E*)a.q + (seq.row0 + tok) * a.q_strides[0] + qh * a.q_strides[1] + 8 * e;
        static_for<0, D / 16>([&](auto i) { qv[i.value] = *(const x8*)(q + 16 * i.value); });
        low = this->lower(tok);
        if constexpr (PART == kPrefix) {
            top = this->block_hi;
            blind = false;
            if (!this->all_see || this->some_blind) {
                top = this->upper(tok);
                blind = top == 0;
                if (blind) top = this->block_hi;
            }
        } else {
            top = max(this->upper(tok), low);
        }
        all_lo = any_lo = low;
        all_hi = any_hi = top;
        if (PART != kPrefix || !this->all_see) {
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                all_lo = max(all_lo, __shfl_xor(all_lo, s));
                all_hi = min(all_hi, __shfl_xor(all_hi, s));
                any_lo = min(any_lo, __shfl_xor(any_lo, s));
                any_hi = max(any_hi, __shfl_xor(any_hi, s));
            }
        }
        all_lo = uniform(all_lo);
        all_hi = uniform(all_hi);
        any_lo = uniform(any_lo);
        any_hi = uniform(any_hi);
        static_for<0, D / 32>([&](auto i) { static_for<0, 16>([&](auto x) { o[i.value][x.value] = 0.0f; }); });
        m = kLowest;
        l = 0.0f;
        large = false;
        static_for<0, D / 16>([&](auto i) { loaded(qv[i.value]); });
    }
    __device__ __forceinline__ void carry_in() {
        const int items = this->prefix_items();
        const int n = here(this->n), e = here(this->e);
        const int row = block + 32 * wave + n;
        if (row < all) {
            const int tok = row / sh.by_group;
            const auto from = this->carried(items, tok, h * sh.group + row - tok * sh.group);
            const float* po = from.parts ? sh.prefix.part_o : sh.carry_o;
            const float2* pml = from.parts ? sh.prefix.part_ml : sh.carry_ml;
            const int parts = max(from.parts, 1);
            for (int p = 0; p < parts; ++p) {
                const int64_t at = from.at(p);
                const float2 ml = pml[at];
                f32x4 w[D / 8];
                static_for<0, D / 32>([&](auto i) {
                    static_for<0, 4>([&](auto x) { w[4 * i.value + x.value] = *(const f32x4*)(po + at * D + 32 * i.value + 8 * x.value + 4 * e); });
                });
                const float to = __builtin_fmaxf(m, ml.x), f = __builtin_amdgcn_exp2f(ml.x - to), shrink = __builtin_amdgcn_exp2f(m - to);
                m = to;
                l = l * shrink + (e == 0 ? ml.y * f : 0.0f);  // (a lane's part of the sum)
                static_for<0, D / 32>([&](auto i) {
                    static_for<0, 16>([&](auto x) {
                        o[i.value][x.value] = o[i.value][x.value] * shrink + w[4 * i.value + x.value / 4][x.value % 4] * f;
                    });
                });
            }
        }
        large |= carried_large(m);
    }

    static constexpr int L = (D + 63) / 64;
    u32x4 fk[L], fv[L];
    float fvs;  // value scale of the sixteen keys this wave fetches
    __device__ __forceinline__ void fetch(int key0, int entry) {
        const uint32_t u = (uint32_t)(key0 >> 4) + wave;
        const int64_t at = this->unit_at(entry, u);
        static_for<0, L>([&](auto x) {
            const int i = lane + 64 * x.value;
            if (D % 64 == 0 || i < D) {
                fk[x.value] = *(const u32x4*)((const uint8_t*)c.k + at + 16 * i);
                fv[x.value] = *(const u32x4*)((const uint8_t*)c.v + at + 16 * i);
            }
        });
        fvs = c.v_scale[this->page_of(entry) * c.kv_heads + h];
    }
    // whether some row of the block sees some of sixteen keys
    __device__ __forceinline__ bool block_sees(int kv) const {
        return (kv + 16 > this->block_lo && kv < this->block_hi) || this->in_sinks(kv, this->block_hi);
    }
    __device__ __forceinline__ void stash(int buf, int key0) {
        const int kv = key0 + 16 * wave;
        if (this->block_edge(key0)) {
            u32x4 keep = keep_bytes(this->block_lo - kv, this->block_hi - kv);
            if constexpr (PART == kSinks) keep |= keep_bytes(-kv, this->sink_keys(this->block_hi) - kv);
            static_for<0, L>([&](auto x) {
                if (D % 64 == 0 || lane + 64 * x.value < D) fv[x.value] = this->clean(fv[x.value], keep);  // see Attend
            });
            if (nan_left) lds.nan = 1;
        }
        // keys that no row sees may have any scale, see Attend
        float vs = block_sees(kv) ? fvs : 1.0f;
        if constexpr (M::kShifts) vs = 1.0f;  // it is weights()' there
        static_for<0, L>([&](auto x) {
            const int i = lane + 64 * x.value;
            if (D % 64 == 0 || i < D) {
                const int row = i / (D / 16), at = i % (D / 16);
                uint8_t* k = lds.k[buf] + (16 * wave + row) * KROW + 128 * wave + 32 * at;
                *(x8*)k = decode8<E>(fk[x.value][0], fk[x.value][1], 1.0f);
                *(x8*)(k + 16) = decode8<E>(fk[x.value][2], fk[x.value][3], 1.0f);
                uint8_t* v = lds.v[buf] + (wave * D + i) * 16;
                *(x8*)v = decode8<E>(fv[x.value][0], fv[x.value][1], vs);
                *(x8*)(v + 4 * D * 16) = decode8<E>(fv[x.value][2], fv[x.value][3], vs);
            }
        });
    }

    // scales of the keys of this lane's scores, as Attend's load_scales
    float ks_raw[2], cs[2], vs_raw[2];
    int ve[2] = {0, 0};
    bool bad_page[2];
    __device__ __forceinline__ void load_scales(const int (&entry)[2]) {
        static_for<0, 2>([&](auto t) {
            const int64_t at = this->page_of(entry[t.value]) * c.kv_heads + h;
            ks_raw[t.value] = c.k_scale[at];
            if constexpr (M::kShifts) vs_raw[t.value] = c.v_scale[at];
            bad_page[t.value] = (uint32_t)entry[t.value] >= (uint32_t)c.pages;
        });
    }

    __device__ __forceinline__ void weights(f32x16 (&s)[2], x8 (&p)[4], bool at_edge, int key0) {
        float unit[2] = {cs[0], cs[1]};
        if (at_edge) {
            static_for<0, 2>([&](auto t) {
                const int kv = key0 + 32 * t.value + 16 * e;
                const int lo = min(max(low - kv, 0), 16), hi = min(max(top - kv, 0), 16);
                int seen = (int)((1u << hi) - (1u << lo));
                if constexpr (PART == kSinks) seen |= (int)((1u << min(max(this->sink_keys(top) - kv, 0), 16)) - 1);
                static_for<0, 16>([&](auto i) {
                    const uint32_t bit = (uint32_t)((seen << (31 - i.value)) >> 31);
                    const uint32_t v = __float_as_uint(s[t.value][i.value] * cs[t.value]);
                    s[t.value][i.value] = __uint_as_float((v & bit) | (0xff800000u & ~bit));
                });
                unit[t.value] = 1.0f;
            });
        }
        float mx[2];
        static_for<0, 2>([&](auto t) {
            mx[t.value] = s[t.value][0];
            static_for<1, 16>([&](auto i) { mx[t.value] = __builtin_fmaxf(mx[t.value], s[t.value][i.value]); });
        });
        const float x = max_across_32(__builtin_fmaxf(__builtin_fmaf(mx[0], unit[0], (float)ve[0]), __builtin_fmaf(mx[1], unit[1], (float)ve[1])));
        if ((M::kShifts && large) || __any(x > m + M::kMost)) {
            const float to = moved_on<M>(m, x, large, [&] {
                return max_across_32(__builtin_fmaxf(product(mx[0], unit[0]), product(mx[1], unit[1])));
            });
            const float shrink = __builtin_amdgcn_exp2f(m - to);
            m = to;
            l *= shrink;
            static_for<0, D / 32>([&](auto i) { o[i.value] *= shrink; });
        }
        float from[2] = {(float)ve[0] - m, (float)ve[1] - m};
        if (large) {
            static_for<0, 2>([&](auto t) {
                static_for<0, 16>([&](auto i) { s[t.value][i.value] = product(s[t.value][i.value], unit[t.value]) - m; });
                unit[t.value] = 1.0f;
                from[t.value] = (float)ve[t.value];
            });
        }
        static_for<0, 2>([&](auto t) {
            float sum = M::kShifts ? 0.0f : l;
            static_for<0, 16>([&](auto i) {
                const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t.value][i.value], unit[t.value], from[t.value]));
                sum += w;
                p[2 * t.value + i.value / 8][i.value % 8] = (E)w;
            });
            l = M::kShifts ? l + __builtin_ldexpf(sum, -ve[t.value]) : sum;
        });
    }

    // N products, each with an operand from LDS: kAhead loads are under way while as
    // many products are made.  Left alone the compiler puts each load right before
    // its product, which then waits for it: 2048 tokens of 32 heads over 32768 took
    // 1241 us instead of 1179, the case of sinks above 189 instead of 178.  Eight
    // ahead need more registers than two workgroups a CU have.  Head dim 64, with
    // eight products where 128 has sixteen, is left to the compiler: 2048 tokens of
    // 32 heads over 16384 406 us, 416 so, in float16 402 and 427.
    static constexpr int kAhead = 4;
    template <int N, class At, class Use>
    static __device__ __forceinline__ void products(At at, Use use) {
        static_assert(N % kAhead == 0);
        if constexpr (D <= 64) {
            static_for<0, N>([&](auto x) { use(x, *(const x8*)at(x)); });
            return;
        }
        x8 f[2][kAhead];
        static_for<0, kAhead>([&](auto x) { f[0][x.value] = *(const x8*)at(x); });
        static_for<0, N / kAhead>([&](auto b) {
            if constexpr (b.value + 1 < N / kAhead)
                static_for<0, kAhead>([&](auto x) {
                    f[(b.value + 1) % 2][x.value] = *(const x8*)at(std::integral_constant<int, (b.value + 1) * kAhead + x.value>{});
                });
            __builtin_amdgcn_sched_barrier(0);
            static_for<0, kAhead>([&](auto x) { use(std::integral_constant<int, b.value * kAhead + x.value>{}, f[b.value % 2][x.value]); });
            __builtin_amdgcn_sched_barrier(0);
        });
    }

    __device__ __forceinline__ void run(int tile, int upto) {
        int from, end;
        this->span(tile, upto, from, end);
        __syncthreads();  // a share's last item may still be read
        if (threadIdx.x == 0) lds.nan = 0;
        __syncthreads();
        int e1 = 0, k1[2] = {0, 0};  // table entries of the next group, fetched and of this lane's keys
        auto entries = [&](int place) {
            const int key0 = this->key_at(place);
            e1 = this->page_entry((uint32_t)(key0 >> 4) + wave);
            k1[0] = this->page_entry((uint32_t)(key0 >> 4) + e);
            k1[1] = this->page_entry((uint32_t)(key0 >> 4) + 2 + e);
        };
        if (from < end) {
            entries(from);
            load_scales(k1);
            fetch(this->key_at(from), e1);
            entries(from + 64);
            stash(0, this->key_at(from));
        }
        // of K: row n of a product, see above
        const int key_row = 16 * ((n >> 2) & 1) + 4 * (n >> 3) + (n & 3);
        const int k_at = key_row * KROW + 128 * ((n >> 2) & 1) + 16 * e, v_at = (e * D + n) * 16;
        int buf = 0;
        for (int place = from; place < end; place += 64) {
            const int key0 = this->key_at(place);
            __syncthreads();
            const bool more = place + 64 < end;
            static_for<0, 2>([&](auto t) {
                bool bad = bad_page[t.value];
                if constexpr (M::kShifts) {
                    const int kv = key0 + 32 * t.value + 16 * e;
                    const float vs = block_sees(kv) ? vs_raw[t.value] : 1.0f;
                    ve[t.value] = M::shift(vs);
                    bad |= !(vs < __builtin_inff());
                }
                cs[t.value] = bad ? __builtin_nanf("") : a.scale * 1.44269504088896340736f * ks_raw[t.value];
            });
            if (more) {
                load_scales(k1);
                const int e0 = e1;
                entries(place + 128);
                fetch(this->key_at(place + 64), e0);
            }
            if ((key0 + 64 > any_lo && key0 < any_hi) || this->in_sinks(key0, any_hi)) {
                f32x16 s[2];
                x8 p[4];
                const uint8_t* kb = lds.k[buf] + k_at;
                static_for<0, 2>([&](auto t) {
                    static_for<0, 16>([&](auto x) { s[t.value][x.value] = 0.0f; });
                });
                products<2 * D / 16>(
                    [&](auto x) { return kb + (x.value % 2) * (32 * KROW + 256) + 32 * (x.value / 2); },
                    [&](auto x, x8 k) { s[x.value % 2] = M::mfma(k, qv[x.value / 2], s[x.value % 2]); });
                weights(s, p, key0 < all_lo || key0 + 64 > all_hi, key0);
                const uint8_t* vb = lds.v[buf] + v_at;
                // product x of a block of channels: keys 32 (x / 2) + 16 e + 8 (x % 2) and on
                products<4 * D / 32>(
                    [&](auto z) {
                        constexpr int i = z.value % (D / 32), x = z.value / (D / 32);
                        return vb + (((x % 2) * 4 + 2 * (x / 2)) * D + 32 * i) * 16;
                    },
                    [&](auto z, x8 v) {
                        constexpr int i = z.value % (D / 32), x = z.value / (D / 32);
                        o[i] = M::mfma(v, p[x], o[i]);
                    });
            }
            buf ^= 1;
            if (more) stash(buf, this->key_at(place + 64));
        }
        __syncthreads();
        nan_left = lds.nan != 0;
        mark_nans(from, end);
        l += __shfl_xor(l, 32);
        if constexpr (PART == kPrefix) {
            if (blind) {
                m = kLowest;
                l = 0.0f;
                static_for<0, D / 32>([&](auto i) { static_for<0, 16>([&](auto x) { o[i.value][x.value] = 0.0f; }); });
            }
        }
    }

    __device__ __forceinline__ void mark_nans(int from, int end) {
        if (!__any(nan_left)) return;
        const int e = here(this->e);
#pragma unroll 1
        for (int place = from; place < end; ++place) {
            const int key = this->key_at(place);
            if (!this->block_edge(key & ~63)) continue;
            const uint32_t u = (uint32_t)key >> 4;
            const uint8_t* vb = (const uint8_t*)c.v + this->unit_at(this->page_entry(u), u) + 64 * e + (key & 15);
            const bool seen = (key >= low && key < top) || this->in_sinks(key, top);
            static_for<0, D / 32>([&](auto i) {
                static_for<0, 16>([&](auto x) {
                    if ((vb[16 * (32 * i.value + 8 * (x.value / 4) + x.value % 4)] & 0x7f) == kNaNCode && seen)
                        o[i.value][x.value] = __builtin_nanf("");
                });
            });
        }
    }

    __device__ __forceinline__ void store() const {
        const int n = here(this->n), e = here(this->e);
        const int row = block + 32 * wave + n;
        if (row >= all) return;
        const int place = row / sh.by_group;
        const int64_t tok = seq.row0 + place;
        const int qh = h * sh.group + row - place * sh.group;
        if constexpr (PART == kPrefix) {
            const int64_t at = tok * a.q_heads + qh;
            static_for<0, D / 32>([&](auto i) {
                static_for<0, 4>([&](auto x) {
                    f32x4 w;
                    static_for<0, 4>([&](auto z) { w[z.value] = o[i.value][4 * x.value + z.value]; });
                    *(f32x4*)(sh.carry_o + at * D + 32 * i.value + 8 * x.value + 4 * e) = w;
                });
            });
            if (e == 0) sh.carry_ml[at] = make_float2(m, l);
            return;
        }
        float inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (seq.poison) inv = __builtin_nanf("");
        E* y = (E*)a.out + tok * a.out_strides[0] + qh * a.out_strides[1] + 4 * e;
        static_for<0, D / 32>([&](auto i) {
            static_for<0, 4>([&](auto x) {
                union {
                    E e[4];
                    u32x2 w;
                } u;
                static_for<0, 4>([&](auto z) { u.e[z.value] = (E)(o[i.value][4 * x.value + z.value] * inv); });
                *(u32x2*)(y + 32 * i.value + 8 * x.value) = u.w;
            });
        });
        if (a.lse && e == 0) a.lse[tok * a.q_heads + qh] = log_sum(m, l, seq.poison);
    }
    __device__ __forceinline__ void store_part(int slot, float* part_o, float2* part_ml) const {
        const int n = here(this->n), e = here(this->e);
        if (block + 32 * wave + n >= all) return;
        const int64_t at = (int64_t)slot * ROWS + 32 * wave + n;
        static_for<0, D / 32>([&](auto i) {
            static_for<0, 4>([&](auto x) {
                f32x4 w;
                static_for<0, 4>([&](auto z) { w[z.value] = o[i.value][4 * x.value + z.value]; });
                *(f32x4*)(part_o + at * D + 32 * i.value + 8 * x.value + 4 * e) = w;
            });
        });
        if (e == 0) part_ml[at] = make_float2(m, l);
    }
};

template <class E, int D, Form F, Part PART>
struct FormOf {
    typedef Attend<E, D, F == kKeys4 ? 4 : F == kKeys2 ? 2 : 1, F != kRows, PART> type;
};
template <class E, int D, Part PART>
struct FormOf<E, D, kTall, PART> {
    typedef Tall<E, D, PART> type;
};

// Rows of no sequence, before the first offset and past the last (padding): they
// see no key.  Workgroup i of n takes every n-th 256 pieces.
template <class E, int D>
__device__ __forceinline__ void clear_rest(const mfft_attend_args& a, int64_t i, int64_t n) {
    if (!a.offsets) return;
    const int64_t lo = seq_offset(a.offsets, 1, a.tokens, 0), hi = seq_offset(a.offsets, 1, a.tokens, a.sequences);
    const int64_t pieces = (lo + a.tokens - hi) * a.q_heads * (D / 4);
    for (i = i * 256 + threadIdx.x; i < pieces; i += n * 256) {
        const int64_t row = i / (D / 4);
        const int at = (int)(i % (D / 4)), h = (int)(row % a.q_heads);
        int64_t tok = row / a.q_heads;
        if (tok >= lo) tok += hi - lo;
        *(u32x2*)((E*)a.out + tok * a.out_strides[0] + h * a.out_strides[1] + 4 * at) = u32x2{0, 0};
        if (a.lse && at == 0) a.lse[tok * a.q_heads + h] = -__builtin_inff();
    }
}

template <class E, int D, Form F, Part PART>
__global__ __launch_bounds__(256, attend_per_cu(D, F)) void attend_kernel(mfft_cache c, mfft_attend_args a, ShapeOf<PART> sh,
                                                                          float* part_o, float2* part_ml, Cut* cuts) {
    using A = typename FormOf<E, D, F, PART>::type;
    __shared__ __align__(16) typename A::Lds lds;
    A w(c, a, sh, lds);
    // groups [at, stop) of the list; with one workgroup an item, of that item
    int64_t before, at = 0, stop, share = INT64_MAX;
    int b, item, tile = 0;
    WorkList<PART> list{c, a, sh, sh.grid == 0, 0, 0};
    int64_t total = 0;
    bool whole = sh.grid == 0;
    if (!whole) {
        total = list.total();
        if constexpr (PART == kRest) {
            // how long items are only the device knows (attend_launch has workgroups
            // enough for one an item)
            int most = list.most;
#pragma unroll
            for (int s = 1; s < 64; s <<= 1) most = max(most, __shfl_xor(most, s));
            const int64_t even = quotient(total + sh.grid - 1, sh.grid);
            whole = uniform(most) <= max(sh.whole_tiles, 4 * (int)even + sh.whole_more);
            if (whole && (int)blockIdx.x < sh.grid && threadIdx.x == 0) cuts[blockIdx.x].parts = 0;
            list.by_item = whole;
            if (whole) {
                list.w = list.items;
                list.upto = wave_scan(list.w);
            }
            if (!whole && (int)blockIdx.x >= sh.grid) return;
        }
    }
    if (whole) {
        b = list.find(blockIdx.x, before, PART == kRest && sh.grid && list.count() <= 64);
        if (b < 0) {
            if constexpr (PART != kPrefix) {
                if (sh.grid == 0) clear_rest<E, D>(a, blockIdx.x - before, gridDim.x - before);
            }
            return;
        }
        w.seq = sequence<PART>(c, a, sh, b);
        item = (int)((int64_t)blockIdx.x - before);
        stop = w.seq.tiles;
    } else {
        const int64_t even = quotient(total + sh.grid - 1, sh.grid);
        share = even > sh.least ? even : sh.least;
        at = blockIdx.x * share;
        stop = at + share < total ? at + share : total;
        if (at >= stop) {
            if (PART != kPrefix && threadIdx.x == 0) cuts[blockIdx.x].parts = 0;
            return;
        }
        b = list.find(at, before, list.count() <= 64);
        w.seq = sequence<PART>(c, a, sh, b);
        const int64_t i = quotient(at - before, w.seq.tiles);
        item = (int)i;
        tile = (int)(at - before - i * w.seq.tiles);
    }
    // kPrefix: which of all items this is, whose cut is cuts[] of that
    int64_t number = 0;
    if constexpr (PART == kPrefix) {
        number = item;
        if (sh.grid && b > 0) {
            int64_t blocks = 0;
            for (int g = (int)(threadIdx.x & 63); g < b; g += 64) blocks += sequence<PART>(c, a, sh, g).blocks;
            number += from_lane(wave_scan(blocks), 63) * c.kv_heads;
        }
    }
    Cut cut{0, 0, 0, 0};
    while (true) {
        const int upto = stop - at < w.seq.tiles - tile ? tile + (int)(stop - at) : w.seq.tiles;
        const int block = item / sh.by_heads, h = item - block * c.kv_heads;
        w.begin(b, block, h);
        if constexpr (PART == kRest) {
            if (tile == 0 && w.seq.prefix > 0) w.carry_in();
        }
        w.run(tile, upto);
        if (tile == 0 && upto == w.seq.tiles) {
            w.store();
            if constexpr (PART == kPrefix) {
                if (sh.grid && threadIdx.x == 0 && number < sh.prefix.items) cuts[number].parts = 0;
            }
        } else {
            w.store_part(2 * (int)blockIdx.x + (tile == 0 ? 1 : 0), part_o, part_ml);
            if (tile == 0) {  // its last group lies `past` groups past this share's end
                const int past = (int)(at + w.seq.tiles - 1 - stop);
                cut = {share > past ? 2 : past / (int)share + 2, b, block, PART == kPrefix ? (int)blockIdx.x : h};
                if constexpr (PART == kPrefix) {
                    if (threadIdx.x == 0 && number < sh.prefix.items) cuts[number] = cut;
                }
            }
        }
        at += upto - tile;
        if (at >= stop) break;
        tile = 0;
        ++number;
        if (++item == w.seq.blocks * c.kv_heads) {
            item = 0;
            do {  // there is one: work is left
                w.seq = sequence<PART>(c, a, sh, ++b);
            } while (w.seq.blocks == 0);
        }
    }
    if (PART != kPrefix && !whole && threadIdx.x == 0) cuts[blockIdx.x] = cut;
}

// Cut items, `sh.join_rows` rows a workgroup: of few parts, a wave a row; of
// many, all four waves every fourth part of one row after the other.  Each lane
// takes D / 64 channels.
template <class E, int D, Part PART>
__global__ __launch_bounds__(256) void join_kernel(mfft_cache c, mfft_attend_args a, ShapeOf<PART> sh, const float* part_o,
                                                   const float2* part_ml, const Cut* cuts) {
    constexpr int C = (D + 63) / 64;
    const int groups = (sh.live + sh.join_rows - 1) / sh.join_rows;
    const int share = blockIdx.x / groups;
    if (share >= sh.grid) {
        clear_rest<E, D>(a, blockIdx.x - sh.grid * groups, gridDim.x - sh.grid * groups);
        return;
    }
    const Cut cut = cuts[share];
    if (cut.parts == 0) return;
    const Sequence seq = sequence<PART>(c, a, sh, cut.b);
    const int block = cut.block * sh.rows, all = seq.n * sh.group;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool wide = cut.parts > 8;
    const int first = (int)(blockIdx.x % groups) * sh.join_rows;
    const int end = min(min(first + sh.join_rows, sh.live), all - block);
    __shared__ float sl[4], so[4][64 * C];

    for (int row = first + (wide ? 0 : wave); row < end; row += wide ? 1 : 4) {
        auto slot = [&](int p) { return (int64_t)(2 * (share + p) + (p == 0 ? 1 : 0)) * sh.rows + row; };
        float m = kLowest;
        for (int p = lane; p < cut.parts; p += 64) m = __builtin_fmaxf(m, part_ml[slot(p)].x);
        m = wave_max(m);
        float l = 0.0f, o[C] = {};
#pragma unroll 8
        for (int p = wide ? wave : 0; p < cut.parts; p += wide ? 4 : 1) {
            const int64_t s = slot(p);
            const float2 ml = part_ml[s];
            const float f = __builtin_amdgcn_exp2f(ml.x - m);
            l += ml.y * f;
#pragma unroll
            for (int x = 0; x < C; ++x)
                if (D % 64 == 0 || lane + 64 * x < D) o[x] += part_o[s * D + lane + 64 * x] * f;
        }
        if (wide) {
            __syncthreads();
            if (lane == 0) sl[wave] = l;
#pragma unroll
            for (int x = 0; x < C; ++x) so[wave][lane + 64 * x] = o[x];
            __syncthreads();
            if (wave > 0) continue;
            l = sl[0] + sl[1] + sl[2] + sl[3];
#pragma unroll
            for (int x = 0; x < C; ++x) o[x] = so[0][lane + 64 * x] + so[1][lane + 64 * x] + so[2][lane + 64 * x] + so[3][lane + 64 * x];
        }
        float inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (seq.poison) inv = __builtin_nanf("");
        const int place = (block + row) / sh.by_group;
        const int64_t tok = seq.row0 + place;
        const int qh = cut.h * sh.group + block + row - place * sh.group;
        E* y = (E*)a.out + tok * a.out_strides[0] + qh * a.out_strides[1];
#pragma unroll
        for (int x = 0; x < C; ++x)
            if (D % 64 == 0 || lane + 64 * x < D) y[lane + 64 * x] = (E)(o[x] * inv);
        if (a.lse && lane == 0) a.lse[tok * a.q_heads + qh] = log_sum(m, l, seq.poison);
    }
}

// ---- the launch ---------------------------------------------------------------
template <class E, int D, Part PART>
void launch_dim(const mfft_cache& c, const mfft_attend_args& a, const AttendLaunch& w, hipStream_t s) {
    float* po = (float*)a.workspace;
    float2* ml = (float2*)((char*)a.workspace + w.o_bytes);
    Cut* cuts = (Cut*)((char*)ml + w.ml_bytes);
    const uint32_t grid = (uint32_t)w.grid;
    if (w.form == kKeys1) attend_kernel<E, D, kKeys1, PART><<<grid, 256, 0, s>>>(c, a, w.sh, po, ml, cuts);
    else if (w.form == kRows) attend_kernel<E, D, kRows, PART><<<grid, 256, 0, s>>>(c, a, w.sh, po, ml, cuts);
    else if constexpr (D <= 128) {
        if (w.form == kKeys2) attend_kernel<E, D, kKeys2, PART><<<grid, 256, 0, s>>>(c, a, w.sh, po, ml, cuts);
        else if (w.form == kTall) attend_kernel<E, D, kTall, PART><<<grid, 256, 0, s>>>(c, a, w.sh, po, ml, cuts);
        else if constexpr (D <= 96) attend_kernel<E, D, kKeys4, PART><<<grid, 256, 0, s>>>(c, a, w.sh, po, ml, cuts);
    }
    mark(s);
    if constexpr (PART != kPrefix) {
        if (w.sh.grid) {
            join_kernel<E, D, PART><<<(uint32_t)w.join_grid, 256, 0, s>>>(c, a, w.sh, po, ml, cuts);
            mark(s);
        }
    }
}

template <class E, Part PART>
void launch_type(const mfft_cache& c, const mfft_attend_args& a, const AttendLaunch& w, hipStream_t s) {
    switch (c.head_dim) {
        case 64: launch_dim<E, 64, PART>(c, a, w, s); break;
        case 96: launch_dim<E, 96, PART>(c, a, w, s); break;
        case 128: launch_dim<E, 128, PART>(c, a, w, s); break;
        case 256: launch_dim<E, 256, PART>(c, a, w, s); break;
    }
}

}  // namespace

template <Part PART>
void launch_part(const mfft_cache& c, const mfft_attend_args& a, const AttendLaunch& w, hipStream_t s) {
    if (a.dtype == MFFT_F16)
        launch_type<_Float16, PART>(c, a, w, s);
    else
        launch_type<__bf16, PART>(c, a, w, s);
}

}  // namespace mfft

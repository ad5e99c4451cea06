// attend_kernels.hip -- attention over the paged 8-bit cache: which launches a
// call makes, and their shapes.  The kernels are in attend_device.hpp, compiled
// for each part of the keys in a file of its own.
#include <algorithm>
#include <cmath>

#include "attend.hpp"
#include "mfft_device.hpp"

namespace mfft {
namespace {

// Sinks without a window change nothing, and a window ends the sharing: what it
// leaves visible of a prefix differs from row to row.
bool with_sinks(const mfft_attend_args& a, const mfft_attend_options& o) { return a.window && o.sinks; }
bool with_prefix(const mfft_attend_args& a, const mfft_attend_options& o) { return !a.window && o.prefix_pages; }

AttendLaunch attend_launch(const mfft_cache& c, const mfft_attend_args& a, const mfft_attend_options& o, Part part) {
    AttendLaunch w{};
    const int sequences = part == kPrefix ? o.groups : a.sequences;
    w.sh.group = a.q_heads / c.kv_heads;
    w.sh.units = c.page_size / 16;
    w.sh.magic = ((uint64_t)1 << 32) / w.sh.units + 1;
    w.sh.per = a.offsets ? 1 : a.tokens / a.sequences;
    w.sh.sinks = (int)o.sinks;
    w.sh.groups = o.groups;
    w.sh.prefix_pages = o.prefix_pages;
    w.sh.prefix_groups = o.prefix_groups;
    // rows of a sequence and key head, on average where there are offsets
    const int64_t rows = (a.tokens * w.sh.group + sequences - 1) / sequences;
    const int D = c.head_dim;
    // 32 sequences of 4096, 8 key heads (4 of dim 256), in us of every form
    // at 16 / 24 / 32 / 48 / 64 / 96 / 128 rows:
    //   dim 64   kKeys1 33 35 36 71 59 82 86, kKeys2 39 40 39 46 46 76 79, kKeys4 55 54 53 53 55 97 97,
    //            kRows 68 67 66 66 66 97 96, kTall 90 89 87 88 87 88 90
    //   dim 96   kKeys1 43 40 41 100 71 103 117, kKeys2 48 49 49 52 52 107 95, kKeys4 59 60 60 61 63 110 110,
    //            kRows 77 78 78 78 79 113 113, kTall 114 116 116 117 117 120 124
    //   dim 128  kKeys1 55 56 57 133 99 137 168, kKeys2 51 51 52 93 94 133 156, kKeys4 75 76 77 78 80 140 143,
    //            kRows 86 88 86 90 91 138 138, kTall 117 119 117 121 121 125 130
    //   dim 256  kKeys1 57 91 92 130 165 242 194, kRows 89 91 91 93 96 143 143
    // and thousands of rows need kTall, which decodes a code once for 128.  What
    // is taken is not the least everywhere: at 48 and 64 rows kKeys2 would be
    // at dims to 96, and kKeys4, which is not built for it, at 128.
    w.form = rows <= 16 ? kKeys1 : rows <= 32 && D <= 128 ? kKeys2 : rows <= 64 && D <= 96 ? kKeys4 : rows <= 64 || D > 128 ? kRows : kTall;
    w.sh.rows = w.form == kKeys1 ? 16 : w.form == kKeys2 ? 32 : w.form == kTall ? 128 : 64;
    // a cut costs its rows' partial sums, written and read again: about a
    // quarter as many groups of keys as it has rows
    w.sh.least = w.sh.rows / 4 > kLeastTiles ? w.sh.rows / 4 : kLeastTiles;
    w.sh.log_rows = ilog2(w.sh.rows);
    w.sh.by_per = divisor((uint32_t)w.sh.per);
    w.sh.by_group = divisor(w.sh.group);
    w.sh.by_heads = divisor(c.kv_heads);
    w.sh.live = !a.offsets && part != kPrefix && rows < w.sh.rows ? (int)rows : w.sh.rows;
    const int64_t items = (a.tokens * w.sh.group / w.sh.rows + sequences) * c.kv_heads;  // at most
    const int64_t at_once = kCUs * attend_per_cu(D, w.form);
    const int64_t table = (int64_t)a.table_width * c.page_size;
    int64_t longest = a.max_length && a.max_length < table ? a.max_length : table;
    w.sh.block_tokens = (w.sh.rows - 1) / w.sh.group + 2;
    if (part == kSinks && a.causal)
        longest = std::min(longest, ((o.sinks + 63) & ~(int64_t)63) + a.window + std::min<int64_t>(w.sh.block_tokens, a.tokens) + 126);
    const int64_t each_items = std::max<int64_t>(sequences, a.tokens * w.sh.group / w.sh.rows) * c.kv_heads;
    const int64_t each = std::max<int64_t>(1, each_items / at_once);
    bool whole = longest <= 64 * kWholeTiles * each;
    if (part == kSinks && a.causal) {
        const int64_t tiles = (longest + 63) / 64, even = each_items * tiles / at_once;
        whole = tiles <= std::max<int64_t>(kAloneTiles, 4 * even + kMoreTiles);
    }
    if (part == kPrefix) {
        // Its cuts cost no launch, so that items are cut as soon as workgroups are
        // left (134 sequences of 8 heads of 256 in 7 groups of 701 shared tokens 53 us
        // instead of 63).  But each sequence's launch reads all parts of its group's
        // item: of T groups of keys about 2 sqrt(T) (shares of four groups at least,
        // of half and of the whole root, in us: 4 sequences in 2 groups of 26241
        // tokens 45, 37 and 39, 24 of 65536 together 76, 63 and 83, 8 tokens of 3
        // heads of 256 over 57908 483, 204 and 187; 8 sequences of 32768 together 40,
        // 40 and 47).
        if (each_items < at_once) whole = longest <= 64 * kLeastTiles;
        const double root = std::sqrt((double)longest / 64.0);
        w.sh.least = std::max(kLeastTiles, (int)(root / 2));
    }
    w.idle = a.offsets && part != kPrefix ? kIdle : 0;
    w.grid = items + w.idle;
    w.sh.prefix.log_rows = w.sh.log_rows;
    w.sh.prefix.items = items;
    if (!whole) {
        // as many shares as workgroups run at once
        w.sh.grid = (int)at_once;
        w.sh.prefix.grid = w.sh.grid;
        w.grid = w.sh.grid;
        if (part == kRest) {
            w.sh.whole_tiles = kAloneTiles;
            w.sh.whole_more = kMoreTiles;
            w.grid = std::max<int64_t>(w.grid, items);
        }
        // few sequences and heads: their items are cut into many parts
        w.sh.join_rows = w.sh.live <= 16 && w.sh.grid >= 8 * (int64_t)sequences * c.kv_heads ? 1 : w.sh.live > 16 ? 8 : 4;
        w.o_bytes = (int64_t)2 * w.sh.grid * w.sh.rows * D * 4;
        w.ml_bytes = (int64_t)2 * w.sh.grid * w.sh.rows * 8;
        // (more items than `items` there are only of groups that overlap, which are none)
        w.cut_bytes = (part == kPrefix ? items : w.sh.grid) * (int64_t)sizeof(Cut);
        if (part != kPrefix) w.join_grid = (int64_t)w.sh.grid * ((w.sh.live + w.sh.join_rows - 1) / w.sh.join_rows) + w.idle;
    }
    return w;
}

int64_t part_bytes(const AttendLaunch& w) { return (w.o_bytes + w.ml_bytes + w.cut_bytes + 255) & ~(int64_t)255; }

}  // namespace

bool attend_supported(int head_dim) { return head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 256; }

// kPrefix's, kRest's, then what the former leaves for each row.
int64_t attend_workspace(const mfft_cache& c, const mfft_attend_args& a, const mfft_attend_options& o) {
    if (with_prefix(a, o))
        return part_bytes(attend_launch(c, a, o, kPrefix)) + part_bytes(attend_launch(c, a, o, kRest)) +
               a.tokens * a.q_heads * (4 * c.head_dim + 8);
    const AttendLaunch w = attend_launch(c, a, o, with_sinks(a, o) ? kSinks : kAll);
    return w.o_bytes + w.ml_bytes + w.cut_bytes;
}

bool attend_launch_fits(const mfft_cache& c, const mfft_attend_args& a, const mfft_attend_options& o) {
    auto fits = [&](Part part) {
        const AttendLaunch w = attend_launch(c, a, o, part);
        return launch_fits(std::max(w.grid, w.join_grid), 256);
    };
    return with_prefix(a, o) ? fits(kPrefix) && fits(kRest) : fits(with_sinks(a, o) ? kSinks : kAll);
}

hipError_t launch_attend(const mfft_cache& c, const mfft_attend_args& a, const mfft_attend_options& o, hipStream_t stream) {
    if (with_prefix(a, o)) {
        AttendLaunch p = attend_launch(c, a, o, kPrefix), r = attend_launch(c, a, o, kRest);
        char* const ws = (char*)a.workspace;
        p.sh.carry_o = r.sh.carry_o = (float*)(ws + part_bytes(p) + part_bytes(r));
        p.sh.carry_ml = r.sh.carry_ml = (float2*)(r.sh.carry_o + a.tokens * a.q_heads * c.head_dim);
        r.sh.prefix = p.sh.prefix;
        r.sh.prefix.part_o = (const float*)ws;
        r.sh.prefix.part_ml = (const float2*)(ws + p.o_bytes);
        r.sh.prefix.cuts = (const Cut*)(ws + p.o_bytes + p.ml_bytes);
        launch_part<kPrefix>(c, a, p, stream);
        mfft_attend_args rest = a;
        rest.workspace = ws + part_bytes(p);
        launch_part<kRest>(c, rest, r, stream);
    } else if (with_sinks(a, o)) {
        launch_part<kSinks>(c, a, attend_launch(c, a, o, kSinks), stream);
    } else {
        launch_part<kAll>(c, a, attend_launch(c, a, o, kAll), stream);
    }
    return hipGetLastError();
}

}  // namespace mfft

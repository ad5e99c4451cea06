// attend.hpp -- what the launches of attention over the paged cache and its
// kernels share: which keys a launch is about, its shape, and what it leaves
// for the next.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "mfft_internal.hpp"

namespace mfft {

// The keys that a launch is about.
//   kAll:    what its sequences' queries see, one run of keys for each query
//   kSinks:  the same in a window, and the sequence's first `sinks` keys
//   kPrefix: the keys that groups of sequences share, for all rows of a group;
//            each row's m, l and O (unscaled) are left in `carry`, or, of items
//            that were cut, in the parts' workspace
//   kRest:   each sequence's keys after those, going on from there
enum Part { kAll, kSinks, kPrefix, kRest };

// the item that starts in share i and is cut at its end: its parts are in
// slots 2 i + 1, 2 (i + 1), 2 (i + 2), ... of the workspace
// (kPrefix: not in the order of shares but of items, `h` the share)
struct Cut {
    int parts;  // 0: none
    int b, block, h;
};

struct AttendShape {
    int group;        // query heads a key head
    Divisor by_group, by_heads;
    int rows, log_rows;  // rows of a block, a power of two
    int units;        // page_size / 16
    uint64_t magic;   // floor(2^32 / units) + 1: x / units = x * magic >> 32, exact for x < 2^26
    int grid;         // shares; 0: one workgroup an item, none cut
    int least;        // fewest groups of 64 keys in a share
    int live;         // rows of a block that can be in use
    int join_rows;    // rows of a workgroup of the join
    int64_t per;      // queries of each sequence without offsets
};
// What the other parts' kernels need too.  kAll's are not given it: arguments
// that they do not use, between and before those that they do, are more and
// smaller loads of arguments, each waited for, wherever an item begins (117
// sequences of 4 keys of 4 heads of 256 20.6 us instead of 19.7).
struct PartShape : AttendShape {
    Divisor by_per;
    int whole_tiles, whole_more;  // kRest: see kAloneTiles
    int block_tokens; // kSinks: tokens of a sequence whose rows a block can have
    // kSinks
    int sinks;        // keys that stay visible
    // kPrefix, kRest
    int groups;                   // of sequences
    const int32_t* prefix_pages;  // [groups]
    const int32_t* prefix_groups; // [groups + 1], NULL: one group of all sequences
    float* carry_o;               // [tokens][q_heads][head_dim]
    float2* carry_ml;             // [tokens][q_heads]
    struct {                      // of kPrefix
        int log_rows, grid;
        int64_t items;            // that `cuts`, in the order of items, has room for
        const Cut* cuts;          // kRest: and its parts
        const float* part_o;
        const float2* part_ml;
    } prefix;
};
template <Part PART>
using ShapeOf = typename std::conditional<PART == kAll, AttendShape, PartShape>::type;

constexpr int kCUs = 256;
constexpr int kLeastTiles = 4;  // one group of 64 keys a wave
// Up to here, times the items there are for each workgroup at once, an item is
// never cut: the second launch costs more than it saves, and many items balance
// by themselves.  One token a sequence of 32 query and 8 key heads of 128,
// lengths to the one given (several sequences: mixed), in us, whole and cut:
// 1 sequence of 1000 10.7 and 15.1, 2000 16.2 and 12.1, 4000 24.8 and 16.2;
// 8 of 2000 16.2 and 17.0, 4000 26.1 and 19.8, 8000 45 and 34; 256 of 1000 55
// and 111.  64 of 2000 and 4000, past the bound, would be faster whole: 30 and
// 54, 55 and 68; of 8000 it is the same, 121.
constexpr int kWholeTiles = 16;
// Windows with sinks and the rests behind shared prefixes are about as long as
// each other, and there an item is left whole up to kAloneTiles or, if that is
// more, up to four equal shares and kMoreTiles: the other workgroups have no
// more to do.  The same heads, in us, whole and cut: a window of 1024 of one
// sequence 14.3 and 18.7, 2000 18.7 and 18.8, 3000 23.0 and 18.2; of 8 sequences
// 1024 15.3 and 20.5, 2000 20.7 and 22.9, 4000 29 and 22; of 64 1024 30 and 33,
// 4000 97 and 101; 300 tokens of one prompt in a window of 512 35 and 103.  Rests
// behind 8192 shared tokens: 32 of 1000 44 and 82, 64 of 4000 99 and 158, 8 of
// 6000 49 and 46.
constexpr int kAloneTiles = 36, kMoreTiles = 8;

// The forms and the workgroups that a CU holds at once, by their registers and
// LDS: O and Q are D R / 4 + D R / 8 registers a lane, and kKeys holds K and V
// of the next group too.
enum Form { kKeys1, kKeys2, kKeys4, kRows, kTall };
constexpr int attend_per_cu(int d, Form f) {
    return f == kKeys1 ? (d >= 256 ? 1 : 2) : f == kKeys2 ? (d >= 128 ? 1 : 2) : f == kKeys4 ? 1 : 2;
}

// Rows of no sequence are written by workgroups that have nothing else to do,
// kIdle more than there may be work for: after the work of all workgroups,
// 0.7 us were added to the shortest call.
constexpr int kIdle = 32;

struct AttendLaunch {
    PartShape sh;
    Form form;
    int64_t grid, join_grid, o_bytes, ml_bytes, cut_bytes;
    int idle;  // workgroups more than work, see clear_rest: of the join where there is one
};

// One part's launches (attend_<part>_kernels.hip); workspace: args->workspace.
template <Part PART>
void launch_part(const mfft_cache& c, const mfft_attend_args& a, const AttendLaunch& w, hipStream_t s);

}  // namespace mfft

// paged_internal.h -- the paged cache: geometry, what its kernels are given, launchers.
#pragma once
#include "../../include/mechta_paged.h"
#include "mkv_internal.h"
#include "paged_book.h"

namespace mkv {
namespace paged {

// The batch as it lies on the device, in 4-byte words from `base`: counts of each list, then the lists.
struct Lists {
    size_t items[KINDS], joins, words;  // word offsets of the lists; words of the whole
};
constexpr size_t COUNTS = 8;  // words in front of a list: items of each kind, joins; of the runs: how many, the longest
static_assert(KINDS < COUNTS, "counts");

struct Geometry {
    int layers, q_heads, kv_heads, head_dim, fmt, pages, page, most_pages;  // most_pages: of a sequence
    size_t page_elems() const { return (size_t)kv_heads * page * head_dim; }
    size_t plane_elems() const { return page_elems() * pages; }
};

struct Rows {  // a caller's rows: element (token, head, d) at token * tok + head * head + d
    const void* p;
    int64_t tok, head;
};

using RopeArgs = mpg_turns;

struct Segment {
    unsigned dst, src, words, pad;
};

hipError_t launch_apply(int* dev, const unsigned* stage, int segments, hipStream_t s);
hipError_t launch_copies(const Geometry& g, char* pool, const Pair* pairs, int n, hipStream_t s);
constexpr int MOST_GRID = 1 << 20;  // work-groups of a launch, which takes less than 2^32 threads; all loop over their lists

// grid: work-groups, or 0: by the runs (most of them) and the tokens of the longest
hipError_t launch_append(const Geometry& g, char* pool, int layer, const int* table, const Run* runs, const int* nruns,
                         int grid, int most, int longest, int rows, const Rows& k, const Rows& v, const Rows& q, void* q_out,
                         const RopeArgs* rope, hipStream_t s);
hipError_t launch_read(const Geometry& g, const char* pool, int layer, int which, const int* table, int p0, int p1, void* dst,
                       hipStream_t s);
hipError_t launch_rotate(const RopeArgs& r, int fmt, int rows, int heads, int dim, const Rows& x, const int* pos,
                         const Rows& out, hipStream_t s);

struct AttendArgs {
    const char* pool;
    int layer, window, rows;
    const int* table;
    Rows q, gate;
    const float* sinks;
    void* out;
    float scale;
    float *pm, *pl, *pacc;  // split partials: reference maximum, sum, accumulator rows
    const std::vector<Join>* joins;  // the plan's, for the launch's shape
    bool captured;                   // a captured launch serves any plan
};
// grid[kind] work-groups for each kind of item (0: not launched), joins likewise; lists and counts on the device.
hipError_t launch_attend(const Geometry& g, const AttendArgs& a, const int* batch, const Lists& l, const int* grid,
                         int join_grid, hipStream_t s);

}  // namespace paged
}  // namespace mkv

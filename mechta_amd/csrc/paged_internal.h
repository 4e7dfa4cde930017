// paged_internal.h -- the paged cache: geometry, what its kernels are given, launchers.
#pragma once
#include "../../include/mechta_paged.h"
#include "mkv_internal.h"
#include "paged_book.h"

namespace mkv {
namespace paged {

// The batch as it lies on the device, in 4-byte words from `base`: counts of each list, then the lists.
struct Lists {
    size_t items[KINDS], joins, segs, words;  // word offsets of the lists; words of the whole
};
constexpr size_t COUNTS = 8;  // words in front of a list: items of each kind, joins; of the runs: how many, the longest
static_assert(KINDS < COUNTS && WEIGH_LISTS <= COUNTS, "counts");

struct Geometry {
    int layers, q_heads, kv_heads, head_dim, fmt, pages, page, most_pages;  // most_pages: of a sequence
    const int* shift = nullptr;  // device: positions evicted from each sequence, where any may be
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
    const Place* order;              // the tokens of shared tiles
    const std::vector<Join>* joins;  // the plan's, for the launch's shape
    bool captured;                   // a captured launch serves any plan
    bool shared;                     // joins may have splits of shared keys
};
// grid[kind] work-groups for each kind of item (0: not launched), joins likewise; lists and counts on the device.
hipError_t launch_attend(const Geometry& g, const AttendArgs& a, const int* batch, const Lists& l, const int* grid,
                         int join_grid, hipStream_t s);

// Accumulated attention weights: of (layer, sequence, kv head), `stride` floats.
struct WeightsAt {
    float* p;
    int layers, seqs, kv_heads;
    size_t stride;
    __host__ __device__ size_t at(int layer, int seq, int head) const {
        return (((size_t)layer * seqs + seq) * kv_heads + head) * stride;
    }
};
struct Change {  // positions [a, a + count) of a sequence; a copy's source is `other`
    int seq, a, count, other;
};
hipError_t launch_clear(const WeightsAt& w, const Change* c, int n, hipStream_t s);
hipError_t launch_weights_copy(const WeightsAt& w, const Change* c, int n, hipStream_t s);

struct WeighLists {  // word offsets in a batch's lists, behind COUNTS of their lengths
    size_t at[WEIGH_LISTS], words;
};
struct WeighArgs {
    const char* pool;
    int layer, window, rows;
    const int* table;
    Rows q;
    const float* sinks;
    float scale, decay;
    float* stats;  // pairs
    float* work;
};
// grid: work-groups for each list, 0: not launched
hipError_t launch_weigh(const Geometry& g, const WeightsAt& w, const WeighArgs& a, const int* batch, const WeighLists& l,
                        const int* grid, hipStream_t s);

struct Eviction {  // `keep` of a sequence's `len` positions; their indexes at `off` of each layer and head's
    int seq, len, keep, off;
};
struct NewPage {  // page `nth` of a sequence (entry of the evictions) is `page` now
    int entry, nth, page;
};
// Which positions stay: to picks[(layer * kv_heads + head) * stride + off ..], in order, and their weights likewise to `kept`; `entries`
// has the list for the others.
hipError_t launch_pick(const Geometry& g, const WeightsAt& w, const Eviction* e, int n, int first, int recent, Eviction* entries,
                       int* picks, float* kept, size_t stride, hipStream_t s);
hipError_t launch_gather(const Geometry& g, char* pool, const int* table, const Eviction* entries, const int* picks, size_t stride,
                         const NewPage* pages, int n, hipStream_t s);
// The weights that stay to their places; longest: the most positions that stay of a sequence.
hipError_t launch_pack(const WeightsAt& w, const Eviction* entries, int n, int longest, const float* kept, size_t stride, hipStream_t s);

}  // namespace paged
}  // namespace mkv

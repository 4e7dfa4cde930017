// paged_book.h -- the paged cache's host side that needs no device: which pages belong to whom, and how a batch's
// attention is cut into work.
#pragma once
#include <cstddef>
#include <cstdint>
#include <functional>
#include <vector>

namespace mkv {
int fail(int code, const char* fmt, ...);  // notes the message of a refused call, returns its code

namespace paged {

constexpr int KEYS = 32;            // positions of a tile: the least page, a V block
constexpr int PART_ROWS = 65536;    // split partials' query rows a handle holds

struct Pair {
    int src, dst;
};

// What set_len gave up: the sequence's length and its pages from `from` on; copied: page `from` was replaced by a copy.
struct Cut {
    int len, from;
    bool copied;
    std::vector<int> pages;
};

// Which pages belong to whom. Pure host state. Each call checks everything first; a refused one changes nothing. What the
// device is then told can fail: undo_* put the book back to what it was before the call right before, and never fail.
struct Book {
    int pages = 0, page = 0, seqs = 0, ctx = 0, free = 0;
    std::vector<int> owners;              // per page
    std::vector<uint64_t> open;           // free pages, one bit each
    size_t low = 0;                       // no word of `open` below this one has a bit
    std::vector<std::vector<int>> table;  // per sequence
    std::vector<int> len;
    std::vector<int> fresh;               // per sequence: entries of its table from here on are not on the device yet
    void init(int pages, int page, int seqs, int ctx);
    int reserve(const char* who, int n, const int* seq, const int* count);
    int fork(const char* who, int n, const int* src, const int* dst, const int* len, bool own, std::vector<Pair>& copies);
    // before: called when all is checked, before anything changes; where it fails, so does the call
    int release(const char* who, int n, const int* seq, const std::function<int()>& before = nullptr);
    int set_len(const char* who, int seq, int len, std::vector<Pair>& copies, Cut* cut = nullptr);
    int compact(std::vector<Pair>& copies);
    void undo_reserve(int n, const int* seq, const int* count);
    void undo_fork(int n, const int* dst) { clear(n, dst); }
    void undo_set_len(int seq, const Cut& cut);
    void undo_compact(const std::vector<Pair>& copies);
    int need(int len) const { return (len + page - 1) / page; }

   private:
    int take();
    void drop(int p);
    void clear(int n, const int* seq);
    void reopen();
    void stale(int seq, int from) {
        if (fresh[seq] > from) fresh[seq] = from;
    }
    int distinct(const char* who, int n, const int* seq) const;
};

// Work of one work-group of an attention kernel: a tile of query rows of one kv head (row = token * group + head in the
// group, counted over the sequence's new tokens) against keys [k0, k1).
struct Item {
    int seq, head;
    int tok0;        // the sequence's first token in the batch
    int row0, rows;  // first row of the tile; rows of the sequence (tokens * group)
    int pos0;        // position of the sequence's first new token
    int k0, k1;      // k0 a multiple of KEYS
    int part;        // first row of the split partials it writes, -1: it writes the output
    int split, pad[2];
};
// Join of a tile's splits: split s of row r at part + s * count + r. wide: a work-group for every 64 dims of a row.
struct Join {
    int head, tok0, row0, count, part, splits, wide, pad;
};
// A run of at most KEYS new tokens inside one KEYS-aligned run of positions.
struct Run {
    int seq, tok, pos, count;
};
enum { FEW, SOME, HALF, MANY, KINDS };  // Item lists by the rows of a tile: 16, 32, 128, 256
constexpr int TILE_ROWS[KINDS] = {16, 32, 128, 256};
constexpr int SPLITS_MOST = 1024;  // splits of a tile at most; work-groups that splits add to a plan at most
// Splits that a tile of so many rows can have at most, behind `part` rows of partials and `more` work items of splits.
int splits_room(int rows, int kv_heads, int part, int more);
struct Plan {
    std::vector<Item> items[KINDS];
    std::vector<Join> joins;
};
struct Shape {  // what a plan depends on besides the batch
    int q_heads, kv_heads, head_dim;
};
struct Member {
    int seq, count, len;
};
void plan_window(const Shape& g, const std::vector<Member>& batch, int window, Plan& out);
// Entries a plan of `tokens` tokens of `seqs` sequences can have at most.
size_t most_items(const Shape& g, int tokens, int seqs);
size_t most_joins(const Shape& g, int tokens, int seqs);

}  // namespace paged
}  // namespace mkv

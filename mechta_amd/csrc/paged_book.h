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
    int shift = 0, floor = 0;
};
// What evict took from a sequence.
struct Evicted {
    int seq, len, shift, floor;
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
    std::vector<int> shift;               // per sequence: positions evicted; position i of what is left, from `floor` - 1 on, was
    std::vector<int> floor;               //   i + shift once (below that, each layer and head has kept others)
    std::vector<char> moved;              // per sequence: its shift is not on the device yet
    void init(int pages, int page, int seqs, int ctx);
    int reserve(const char* who, int n, const int* seq, const int* count);
    int fork(const char* who, int n, const int* src, const int* dst, const int* len, bool own, std::vector<Pair>& copies);
    // before: called when all is checked, before anything changes; where it fails, so does the call
    int release(const char* who, int n, const int* seq, const std::function<int()>& before = nullptr);
    int set_len(const char* who, int seq, int len, std::vector<Pair>& copies, Cut* cut = nullptr);
    int compact(std::vector<Pair>& copies);
    // Cuts each sequence of more than keep[i] positions to keep[i], on new pages in place of its own.
    int can_evict(const char* who, int n, const int* seq, const int* keep) const;
    int evict(const char* who, int n, const int* seq, const int* keep, std::vector<Evicted>& cut);
    void undo_evict(std::vector<Evicted>& cut);
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
    void own_again(int page);
    void stale(int seq, int from) {
        if (fresh[seq] > from) fresh[seq] = from;
    }
    void move(int seq, int by, int from) {
        moved[seq] |= shift[seq] != by;
        shift[seq] = by;
        floor[seq] = from;
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
    int split;
    int top;         // 0, or the tile is of keys that several sequences have (seq is one of them): its tokens are entries tok0 ..
                     // of the batch's order, all behind the keys, the furthest at position top - 1; pos0: the end of the keys, k1 or
                     // behind it
    int pad;
};
// Join of a tile's splits: split s of row r at part + s * count + r, and those of the shared tiles that its rows are in, Seg
// `segs` of them. wide: a work-group for every 64 dims of a row, or (ROW_WIDE) for a row.
struct Join {
    int head, tok0, row0, count, part, splits, wide, segs;
};
// Splits of shared keys: split s of a join's row r at part + s * stride + r. Join n's are entries LEVELS n ..
struct Seg {
    int part, stride, splits, pad;
};
constexpr int ROW_WIDE = 2;
constexpr int LEVELS = 3;  // shared ranges that a sequence's tokens are in at most
// An entry of a batch's order: a token and its position.
struct Place {
    int tok, pos;
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
    std::vector<Seg> segs;  // none: no join has any
};
struct Shape {  // what a plan depends on besides the batch
    int q_heads, kv_heads, head_dim;
};
struct Member {
    int seq, count, len;
};
void plan_window(const Shape& g, const std::vector<Member>& batch, int window, Plan& out);

// What sequences of a batch have in common. Pages come to be shared by forks alone, so two sequences that have a page have
// all pages before it: the page lists make a tree.
struct Range {  // positions [k0, k1), on the same pages for the sequences members[first .. first + count)
    int k0, k1, first, count, parent;
};
struct Share {
    std::vector<Range> ranges;   // parents before children
    std::vector<int> members;    // places in the batch, in an order in which those of every range lie together
    std::vector<int> from;       // per place in the batch: the first position that is attended for it alone
    std::vector<int> range;      // per place in the batch: the innermost range it is in, -1: none
    std::vector<Place> order;    // the tokens of `members`, one sequence behind the other
    std::vector<int> at;         // per place in the batch: its first token's entry in `order`
};
void share(const Book& b, const Shape& g, const std::vector<Member>& batch, Share& out);
// plan_window with the keys that several sequences have taken once for all of them; plan_window's plan where the split
// partials of that find no room.
void plan_shared(const Shape& g, const std::vector<Member>& batch, const Share& s, int window, Plan& out);
// Entries a plan of `tokens` tokens of `seqs` sequences can have at most.
size_t most_items(const Shape& g, int tokens, int seqs);
size_t most_joins(const Shape& g, int tokens, int seqs);

// ---- accumulated attention weights ----
// Per window, the work of weighing a batch: what each position is given by the sequences' counted tokens (rows = counted
// tokens x group). First the statistics of the rows, for few rows with their scores, then the sums over them.
struct Score {  // rows row0 .. of one kv head against keys [k0, k1): the reference and the sum of each to stats[stat ..]
    int seq, head, tok0, rows, row0, pos0;  // tok0, pos0: the first counted token and its position
    int k0, k1, stat;
    int keep;        // few rows: where the scores go in the work space, 16 keys behind 16 keys, [row][key]
    int whole;       // there is no other piece: many rows: what goes to stats is final; few: the sums are taken at once
    int pad;
};
struct Merge {  // rows r0 .. r1 of several pieces: the final statistics to the first piece's place
    int head, tok0, rows, r0, r1, stat, pieces, pad;
};
struct Sum {  // keys [k0, k1) from rows [r0, r1)
    int seq, head, tok0, rows, pos0, k0, k1;
    int r0, r1;
    int stat, pieces;  // few rows: statistics of piece p of row r at stats[stat + p * rows + r]; many: the final ones at stats[stat + r]
    int scores, s0;    // few rows: kept scores, the first of key s0
    int part;          // where the sums go in the work space, -1: to the position's weight
    int pad[2];
};
struct Fade {  // weights of keys [k0, k1), faded, plus `sums` partial sums, of key k0 + i at part + s * stride + i
    int seq, head, k0, k1, part, sums, stride, pad;
};
constexpr int MERGE_WAYS = 8;  // work-groups of a merge: 16 rows each
// few: up to 16 rows, some: up to 32, many: tiles of 128
enum { SCORE_FEW, SCORE_SOME, SCORE_MANY, MERGES, SUM_FEW, SUM_MANY, FADES, WEIGH_LISTS };
struct WeighPlan {
    std::vector<Score> scores[SCORE_MANY + 1];
    std::vector<Merge> merges;
    std::vector<Sum> sums[2];
    std::vector<Fade> fades;
};
struct WeighRoom {
    long long stats, work;  // pairs, floats
};
constexpr int SCORE_ROWS = 128, SUM_KEYS = 256;  // of a tile: rows of SCORE_MANY, keys of SUM_MANY
constexpr int WEIGH_MOST = 4096;                 // entries of a list at most, besides one for each tile of SCORE_ROWS or sequence, and head
constexpr int CUS = 256;
constexpr int SUM_PLACES = 6 * CUS - 64;         // work-groups that take many rows' sums, about
constexpr int WEIGH_PARTS = (SUM_PLACES + WEIGH_MOST) * SUM_KEYS;  // floats of the room: those sums' parts, which always find room
// Whether a batch of up to `tokens` tokens of up to `seqs` sequences of up to `ctx` positions can have entries in a list.
bool may_weigh(const Shape& g, int tokens, int seqs, int ctx, int window, int last, const WeighRoom& room, int list);
size_t weigh_entries(const Shape& g, int tokens, int seqs);
void plan_weigh(const Shape& g, const std::vector<Member>& batch, int window, int last, const WeighRoom& room, WeighPlan& out);

}  // namespace paged
}  // namespace mkv

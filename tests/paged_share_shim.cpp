// C functions over what a batch's sequences have in common, for tests/test_paged_share.py (compiled there with the sources'
// own paged_book.cpp, undefined-behaviour checks on).
#include <cstdarg>
#include <cstdio>

#include "../mechta_amd/csrc/paged_book.h"

using namespace mkv::paged;

static char message[512];
namespace mkv {
int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(message, sizeof message, fmt, ap);
    va_end(ap);
    return code;
}
}  // namespace mkv

static Share common;
static Plan plan;
static std::vector<Member> batch;

extern "C" {
const char* shim_message() { return message; }
Book* shim_new(int pages, int page, int seqs, int ctx) {
    Book* b = new Book;
    b->init(pages, page, seqs, ctx);
    return b;
}
void shim_delete(Book* b) { delete b; }
int shim_reserve(Book* b, int n, const int* seq, const int* count) { return b->reserve("reserve", n, seq, count); }
int shim_fork(Book* b, int n, const int* src, const int* dst, const int* len) {
    std::vector<Pair> copies;
    return b->fork("fork", n, src, dst, len, false, copies);
}
int shim_set_len(Book* b, int seq, int len) {
    std::vector<Pair> copies;
    return b->set_len("set_len", seq, len, copies);
}
int shim_len(Book* b, int seq) { return b->len[seq]; }
int shim_table(Book* b, int seq, int* out) {
    for (size_t i = 0; i < b->table[seq].size(); i++) out[i] = b->table[seq][i];
    return (int)b->table[seq].size();
}
// ranges that the batch's sequences have in common
int shim_share(Book* b, int q_heads, int kv_heads, int head_dim, int n, const int* seq, const int* count) {
    batch.clear();
    for (int i = 0; i < n; i++) batch.push_back({seq[i], count[i], b->len[seq[i]]});
    share(*b, Shape{q_heads, kv_heads, head_dim}, batch, common);
    return (int)common.ranges.size();
}
void shim_plan(int q_heads, int kv_heads, int head_dim, int window, int* sizes) {
    plan_shared(Shape{q_heads, kv_heads, head_dim}, batch, common, window, plan);
    for (int k = 0; k < KINDS; k++) sizes[k] = (int)plan.items[k].size();
    sizes[KINDS] = (int)plan.joins.size();
    sizes[KINDS + 1] = (int)plan.segs.size();
    sizes[KINDS + 2] = (int)common.order.size();
}
// whether plan_shared's plan is plan_window's
int shim_plain(int q_heads, int kv_heads, int head_dim, int window) {
    Plan p;
    plan_window(Shape{q_heads, kv_heads, head_dim}, batch, window, p);
    bool same = p.joins.size() == plan.joins.size();
    for (int k = 0; k < KINDS; k++) same &= p.items[k].size() == plan.items[k].size();
    for (int k = 0; k < KINDS && same; k++)
        for (size_t i = 0; i < p.items[k].size(); i++) {
            const Item &x = p.items[k][i], &y = plan.items[k][i];
            same &= x.seq == y.seq && x.head == y.head && x.tok0 == y.tok0 && x.row0 == y.row0 && x.k0 == y.k0 && x.k1 == y.k1 && x.part == y.part && !y.top;
        }
    return same;
}
void shim_items(int kind, int* out) {  // 12 ints each
    for (size_t i = 0; i < plan.items[kind].size(); i++) *(Item*)(out + 12 * i) = plan.items[kind][i];
}
void shim_joins(int* out) {  // 8 ints each
    for (size_t i = 0; i < plan.joins.size(); i++) *(Join*)(out + 8 * i) = plan.joins[i];
}
void shim_segs(int* out) {  // 4 ints each
    for (size_t i = 0; i < plan.segs.size(); i++) *(Seg*)(out + 4 * i) = plan.segs[i];
}
void shim_order(int* out) {
    for (size_t i = 0; i < common.order.size(); i++) out[2 * i] = common.order[i].tok, out[2 * i + 1] = common.order[i].pos;
}
int shim_levels() { return LEVELS; }
int shim_splits_most() { return SPLITS_MOST; }
int shim_part_rows() { return PART_ROWS; }
size_t shim_most_items(int q_heads, int kv_heads, int head_dim, int tokens, int seqs) {
    return most_items(Shape{q_heads, kv_heads, head_dim}, tokens, seqs);
}
size_t shim_most_joins(int q_heads, int kv_heads, int head_dim, int tokens, int seqs) {
    return most_joins(Shape{q_heads, kv_heads, head_dim}, tokens, seqs);
}
}

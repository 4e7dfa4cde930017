// C functions over the paged cache's host side, for tests/test_paged_book.py (compiled there with the sources' own
// paged_book.cpp, address and undefined-behaviour checks on).
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

static std::vector<Pair> copies;
static Plan plan;

extern "C" {
const char* shim_message() { return message; }
Book* shim_new(int pages, int page, int seqs, int ctx) {
    Book* b = new Book;
    b->init(pages, page, seqs, ctx);
    return b;
}
void shim_delete(Book* b) { delete b; }
int shim_reserve(Book* b, int n, const int* seq, const int* count) { return b->reserve("reserve", n, seq, count); }
int shim_fork(Book* b, int n, const int* src, const int* dst, const int* len, int own) {
    copies.clear();
    return b->fork("fork", n, src, dst, len, own, copies);
}
int shim_free(Book* b, int n, const int* seq) { return b->release("free", n, seq); }
int shim_set_len(Book* b, int seq, int len) {
    copies.clear();
    return b->set_len("set_len", seq, len, copies);
}
int shim_compact(Book* b) {
    copies.clear();
    return b->compact(copies);
}
int shim_copies(int* out) {  // pairs of the last call
    for (size_t i = 0; i < copies.size(); i++) out[2 * i] = copies[i].src, out[2 * i + 1] = copies[i].dst;
    return (int)copies.size();
}
int shim_len(Book* b, int seq) { return b->len[seq]; }
int shim_fresh(Book* b, int seq) { return b->fresh[seq]; }
void shim_sent(Book* b) {  // as if the tables had gone to the device
    for (int s = 0; s < b->seqs; s++) b->fresh[s] = (int)b->table[s].size();
}
int shim_free_pages(Book* b) { return b->free; }
int shim_owners(Book* b, int page) { return b->owners[page]; }
int shim_table(Book* b, int seq, int* out) {
    for (size_t i = 0; i < b->table[seq].size(); i++) out[i] = b->table[seq][i];
    return (int)b->table[seq].size();
}
// members: seq, count, len each
void shim_plan(int q_heads, int kv_heads, int head_dim, int n, const int* members, int window, int* sizes) {
    std::vector<Member> batch;
    for (int i = 0; i < n; i++) batch.push_back({members[3 * i], members[3 * i + 1], members[3 * i + 2]});
    plan_window(Shape{q_heads, kv_heads, head_dim}, batch, window, plan);
    for (int k = 0; k < KINDS; k++) sizes[k] = (int)plan.items[k].size();
    sizes[KINDS] = (int)plan.joins.size();
}
void shim_items(int kind, int* out) {  // 12 ints each
    for (size_t i = 0; i < plan.items[kind].size(); i++) *(Item*)(out + 12 * i) = plan.items[kind][i];
}
void shim_joins(int* out) {  // 8 ints each
    for (size_t i = 0; i < plan.joins.size(); i++) *(Join*)(out + 8 * i) = plan.joins[i];
}
size_t shim_most_items(int q_heads, int kv_heads, int head_dim, int tokens, int seqs) {
    return most_items(Shape{q_heads, kv_heads, head_dim}, tokens, seqs);
}
size_t shim_most_joins(int q_heads, int kv_heads, int head_dim, int tokens, int seqs) {
    return most_joins(Shape{q_heads, kv_heads, head_dim}, tokens, seqs);
}
int shim_part_rows() { return PART_ROWS; }
}

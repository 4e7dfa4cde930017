// C functions over the work of weighing a batch, for tests/test_paged_weights.py (compiled there with the sources' own
// paged_book.cpp, undefined-behaviour checks on).
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

static WeighPlan plan;

extern "C" {
const char* shim_message() { return message; }
// members: seq, count, len each; sizes of the lists
void shim_weigh(int q_heads, int kv_heads, int head_dim, int n, const int* members, int window, int last, long long stats,
                long long work, int* sizes) {
    std::vector<Member> batch;
    for (int i = 0; i < n; i++) batch.push_back({members[3 * i], members[3 * i + 1], members[3 * i + 2]});
    plan_weigh(Shape{q_heads, kv_heads, head_dim}, batch, window, last, WeighRoom{stats, work}, plan);
    for (int k = 0; k <= SCORE_MANY; k++) sizes[k] = (int)plan.scores[k].size();
    sizes[MERGES] = (int)plan.merges.size();
    for (int k = 0; k < 2; k++) sizes[SUM_FEW + k] = (int)plan.sums[k].size();
    sizes[FADES] = (int)plan.fades.size();
}
void shim_scores(int list, int* out) {  // 12 ints each
    for (size_t i = 0; i < plan.scores[list].size(); i++) *(Score*)(out + 12 * i) = plan.scores[list][i];
}
void shim_sums(int list, int* out) {  // 16 ints each
    for (size_t i = 0; i < plan.sums[list].size(); i++) *(Sum*)(out + 16 * i) = plan.sums[list][i];
}
void shim_merges(int* out) {  // 8 ints each
    for (size_t i = 0; i < plan.merges.size(); i++) *(Merge*)(out + 8 * i) = plan.merges[i];
}
void shim_fades(int* out) {  // 8 ints each
    for (size_t i = 0; i < plan.fades.size(); i++) *(Fade*)(out + 8 * i) = plan.fades[i];
}
int shim_may(int q_heads, int kv_heads, int tokens, int seqs, int ctx, int window, int last, long long work, int list) {
    return may_weigh(Shape{q_heads, kv_heads, 64}, tokens, seqs, ctx, window, last, WeighRoom{0, work}, list);
}
int shim_parts() { return WEIGH_PARTS; }
size_t shim_entries(int q_heads, int kv_heads, int tokens, int seqs) { return weigh_entries(Shape{q_heads, kv_heads, 64}, tokens, seqs); }

Book* shim_new(int pages, int page, int seqs, int ctx) {
    Book* b = new Book;
    b->init(pages, page, seqs, ctx);
    return b;
}
void shim_delete(Book* b) { delete b; }
int shim_reserve(Book* b, int n, const int* seq, const int* count) { return b->reserve("reserve", n, seq, count); }
static std::vector<Pair> copies;
int shim_fork(Book* b, int n, const int* src, const int* dst, const int* len, int own) {
    copies.clear();
    return b->fork("fork", n, src, dst, len, own, copies);
}
int shim_free(Book* b, int n, const int* seq) { return b->release("free", n, seq); }
static Cut cut;
int shim_set_len(Book* b, int seq, int len) {
    copies.clear();
    return b->set_len("set_len", seq, len, copies, &cut);
}
void shim_undo_set_len(Book* b, int seq) { b->undo_set_len(seq, cut); }
int shim_compact(Book* b) {
    copies.clear();
    return b->compact(copies);
}
static std::vector<Evicted> evicted;
int shim_evict(Book* b, int n, const int* seq, const int* keep) {
    evicted.clear();
    return b->evict("evict", n, seq, keep, evicted);
}
void shim_undo_evict(Book* b) { b->undo_evict(evicted); }
// length, shift, floor, whether the shift goes up, pages that are not on the device
void shim_state(Book* b, int seq, int* out) {
    out[0] = b->len[seq], out[1] = b->shift[seq], out[2] = b->floor[seq], out[3] = b->moved[seq], out[4] = b->fresh[seq];
}
void shim_sent(Book* b) {
    for (int s = 0; s < b->seqs; s++) b->fresh[s] = (int)b->table[s].size(), b->moved[s] = 0;
}
int shim_free_pages(Book* b) { return b->free; }
int shim_owners(Book* b, int page) { return b->owners[page]; }
int shim_table(Book* b, int seq, int* out) {
    for (size_t i = 0; i < b->table[seq].size(); i++) out[i] = b->table[seq][i];
    return (int)b->table[seq].size();
}
}

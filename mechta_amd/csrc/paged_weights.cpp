// paged_weights.cpp -- what the positions of a paged cache are looked at: attention weights accumulated position by position,
// and eviction by them (include/mechta_paged.h).
#include <climits>
#include <cmath>

#include <algorithm>

#include "paged_handle.h"

using mkv::fail;
using mkv::hip_fail;
using namespace mkv::paged;

namespace {

// Work-groups of each kernel of a captured weighing, of whatever batch it finds. (1 token at 300 positions of 2 x 256, 64 at 3,000 and 4
// of one sequence at 65,536 of 4 x 128, in a graph: 15.3 / 58.5 / 50.0 us; with 8,192 for the merges 16.6 / 60.1 / 51.6, with 512 of
// each kind 15.2 / 60.8 / 65.8. Of a handle that counts a token of each sequence, whose graphs have two kernels: 7.4 / 50.6.)
constexpr int GRAPH_WEIGH = 1024, GRAPH_MERGES = 512;
constexpr long long WORK_MOST = 1ll << 28;  // floats: kept scores
constexpr long long STATS_MORE = 1ll << 18;  // statistics of rows in more than one piece

struct Kept : Weights {
    mpg_store* h;
    int last;
    WeightsAt at;
    WeighRoom room;
    WeighLists lists_at;
    size_t batch_at = 0;         // word offset in dev
    float* stats = nullptr;      // pairs
    float* work = nullptr;
    int* picks = nullptr;        // [layer][kv head][positions of the pool]: of an eviction, the positions that stay
    float* heavy = nullptr;      // and their weights
    Eviction* entries = nullptr;  // [seqs]
    std::vector<WeighPlan> plans, next;  // per window
    std::vector<int> counts;     // COUNTS a window, of `next`

    ~Kept() override {
        for (void* p : {(void*)at.p, (void*)stats, (void*)work, (void*)picks, (void*)heavy, (void*)entries})
            if (p) (void)hipFree(p);
    }
    int changes(bool copy, int n, const int* seq, const int* from, const int* count, const int* other, const char* who) {
        std::vector<Change> c;
        for (int i = 0; i < n; i++)
            if (count[i] > 0) c.push_back({seq[i], from ? from[i] : 0, count[i], other ? other[i] : 0});
        if (c.empty()) return MKV_OK;
        const hipError_t e = copy ? launch_weights_copy(at, c.data(), (int)c.size(), h->stream)
                                  : launch_clear(at, c.data(), (int)c.size(), h->stream);
        return e == hipSuccess ? MKV_OK : hip_fail(e, who);
    }
    int clear(int n, const int* seq, const int* from, const int* count, const char* who) override {
        return changes(false, n, seq, from, count, nullptr, who);
    }
    int copy(int n, const int* src, const int* dst, const int* len, const char* who) override {
        return changes(true, n, dst, nullptr, len, src, who);
    }
    void lay_out(const std::vector<Member>& batch) override {
        for (size_t w = 0; w < h->kinds.size(); w++) plan_weigh(h->shape, batch, h->kinds[w], last, room, next[w]);
    }
    void lists(bool none, const std::function<void(size_t, const void*, size_t)>& put) override {
        counts.assign(h->kinds.size() * COUNTS, 0);
        for (size_t w = 0; w < h->kinds.size(); w++) {
            const size_t base = batch_at + w * lists_at.words;
            int* const c = counts.data() + w * COUNTS;
            const WeighPlan& p = next[w];
            if (!none) {
                for (int k = 0; k <= SCORE_MANY; k++) c[k] = (int)p.scores[k].size();
                c[MERGES] = (int)p.merges.size();
                for (int k = 0; k < 2; k++) c[SUM_FEW + k] = (int)p.sums[k].size();
                c[FADES] = (int)p.fades.size();
            }
            put(base, c, COUNTS);
            if (none) continue;
            for (int k = 0; k <= SCORE_MANY; k++) put(base + lists_at.at[k], p.scores[k].data(), p.scores[k].size() * (sizeof(Score) / 4));
            put(base + lists_at.at[MERGES], p.merges.data(), p.merges.size() * (sizeof(Merge) / 4));
            for (int k = 0; k < 2; k++) put(base + lists_at.at[SUM_FEW + k], p.sums[k].data(), p.sums[k].size() * (sizeof(Sum) / 4));
            put(base + lists_at.at[FADES], p.fades.data(), p.fades.size() * (sizeof(Fade) / 4));
        }
    }
    void stands() override { plans.swap(next); }
};

Kept* kept(const mpg_store* h) { return static_cast<Kept*>(h->weights.get()); }

struct WeightSizes {
    size_t stride, weights, stats, work, picks, words;  // floats, floats, pairs, floats, ints, words of the lists and shifts
    WeighLists l;
};
WeightSizes weight_sizes(const mpg_config& c, int last) {
    WeightSizes s;
    s.stride = ((size_t)c.ctx + 31) / 32 * 32;
    s.weights = (size_t)c.layers * c.seqs * c.kv_heads * s.stride;
    const long long counted = last ? std::min((long long)c.tokens, (long long)std::min(c.seqs, c.tokens) * last) : c.tokens;
    s.stats = counted * c.q_heads + STATS_MORE;  // (and a tile of rows behind: the last is read whole)
    // Scores of a token of each sequence, however many of them share their pages, and of up to 32 rows of every position of the pool,
    // as far as that is not too much; what finds no room is scored twice.
    s.work = (size_t)(std::min<double>(WORK_MOST, std::max(32. * c.pages * c.page * c.kv_heads,
                                                           (double)s.stride * std::min(c.seqs, c.tokens) * c.q_heads)) + WEIGH_PARTS);
    s.picks = (size_t)c.layers * c.kv_heads * c.pages * c.page;
    const Shape g{c.q_heads, c.kv_heads, c.head_dim};
    const size_t entries = weigh_entries(g, c.tokens, c.seqs);
    size_t at = COUNTS;
    for (int k = 0; k < WEIGH_LISTS; k++) {
        s.l.at[k] = at;
        at += entries * (k <= SCORE_MANY ? sizeof(Score) : k == MERGES ? sizeof(Merge) : k < FADES ? sizeof(Sum) : sizeof(Fade)) / 4;
    }
    s.l.words = at;
    s.words = s.l.words * MPG_WINDOWS_MAX + c.seqs;
    return s;
}
double bytes_of(const WeightSizes& s, const mpg_config& c) {
    return 4. * s.weights + 8. * (s.stats + KEYS) + 4. * s.work + 8. * s.picks + 4. * s.words + sizeof(Eviction) * (double)c.seqs;
}

int check_last(const char* who, int last) {
    return last < 0 ? fail(MKV_E_ARG, "%s: the last %d tokens", who, last) : MKV_OK;
}
// What is refused before anything is allocated.
int check_sizes(const char* who, const WeightSizes& s, const mpg_config& c) {
    const double all = bytes_of(s, c);
    if (all > 1ll << 48) return fail(MKV_E_NOMEM, "%s: %g bytes", who, all);
    const size_t words = handle_words(c) + s.words;
    return words < WORDS_MOST ? (int)MKV_OK : fail(MKV_E_NOMEM, "%s: lists of %zu words", who, words);
}

}  // namespace

extern "C" {

size_t mpg_weights_bytes(const mpg_config* c, int last) {
    if (!mpg_bytes(c) || check_last("mpg_weights_bytes", last)) return 0;
    const WeightSizes s = weight_sizes(*c, last);
    return check_sizes("mpg_weights_bytes", s, *c) ? 0 : (size_t)bytes_of(s, *c);
}

static int keep_weights(mpg_t* h, int last) {
    if (int rc = check_last("mpg_keep_weights", last)) return rc;
    if (h->weights) return fail(MKV_E_ARG, "mpg_keep_weights: the handle keeps them already");
    if (h->used) return fail(MKV_E_ARG, "mpg_keep_weights: sequences have had positions already");
    const mpg_config& c = h->c;
    const WeightSizes s = weight_sizes(c, last);
    if (int rc = check_sizes("mpg_keep_weights", s, c)) return rc;
    std::unique_ptr<Kept> k(new Kept);
    k->h = h;
    k->last = last;
    k->at = WeightsAt{nullptr, c.layers, c.seqs, c.kv_heads, s.stride};
    k->room = WeighRoom{(long long)s.stats, (long long)s.work};
    k->lists_at = s.l;
    k->plans.resize(h->kinds.size());
    k->next.resize(h->kinds.size());
    // the lists and shifts go where the handle's uploads go: behind what is there
    const size_t words = h->words + s.words;
    int* dev = nullptr;
    hipError_t e = hipMalloc((void**)&dev, words * 4);
    if (e == hipSuccess) e = hipMalloc((void**)&k->at.p, s.weights * 4);
    if (e == hipSuccess) e = hipMalloc((void**)&k->stats, (s.stats + KEYS) * 8);
    if (e == hipSuccess) e = hipMalloc((void**)&k->work, s.work * 4);
    if (e == hipSuccess) e = hipMalloc((void**)&k->picks, s.picks * 4);
    if (e == hipSuccess) e = hipMalloc((void**)&k->heavy, s.picks * 4);
    if (e == hipSuccess) e = hipMalloc((void**)&k->entries, sizeof(Eviction) * c.seqs);
    if (e == hipSuccess) e = hipMemsetAsync(dev, 0, words * 4, h->stream);
    if (e == hipSuccess) e = hipMemsetAsync(k->at.p, 0, s.weights * 4, h->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(h->stream);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        if (dev) (void)hipFree(dev);
        return fail(MKV_E_NOMEM, "mpg_keep_weights: %.0f bytes: %s", bytes_of(s, c), hipGetErrorString(e));
    }
    (void)hipFree(h->dev);
    h->dev = dev;
    k->batch_at = h->words;
    h->shift_at = h->words + s.l.words * MPG_WINDOWS_MAX;
    h->words = words;
    h->g.shift = dev + h->shift_at;
    h->weights = std::move(k);
    return MKV_OK;
}
int mpg_keep_weights(mpg_t* h, int last) {
    MPG_HOST_CALL(h, "mpg_keep_weights");
    return guarded("mpg_keep_weights", [&] { return keep_weights(h, last); });
}

int mpg_weights(const mpg_t* h, int layer, float** base, int64_t* seq_stride, int64_t* head_stride) {
    if (int rc = check_layer(h, layer, "mpg_weights")) return rc;
    if (!h->weights) return fail(MKV_E_ARG, "mpg_weights: the handle keeps none (mpg_keep_weights)");
    if (!base || !seq_stride || !head_stride) return fail(MKV_E_ARG, "mpg_weights: NULL argument");
    const WeightsAt& at = kept(h)->at;
    *base = at.p + at.at(layer, 0, 0);
    *head_stride = (int64_t)at.stride;
    *seq_stride = (int64_t)at.stride * at.kv_heads;
    return MKV_OK;
}

int mpg_weigh(mpg_t* h, int layer, int rows, const void* q, int64_t q_tok, int64_t q_head, float scale, const float* sinks,
              float decay) {
    if (int rc = check_layer(h, layer, "mpg_weigh")) return rc;
    if (!h->weights) return fail(MKV_E_ARG, "mpg_weigh: the handle keeps no weights (mpg_keep_weights)");
    if (int rc = check_batch(h, rows, "mpg_weigh")) return rc;
    if (!rows) return MKV_OK;
    if (int rc = check_rows("mpg_weigh", "q", q, rows, q_tok, h->c.q_heads, q_head)) return rc;
    if (!(scale > 0) || !std::isfinite(scale)) return fail(MKV_E_ARG, "mpg_weigh: scale %g", scale);
    if (!(decay >= 0) || !std::isfinite(decay)) return fail(MKV_E_ARG, "mpg_weigh: decay %g", decay);
    if ((uintptr_t)sinks % 4) return fail(MKV_E_ARG, "mpg_weigh: misaligned sinks");
    OnDevice on(h->device);
    const int cap = capturing(h, "mpg_weigh");
    if (cap < 0) return cap;
    const int w = h->windows[layer];
    Kept* const k = kept(h);
    const WeighPlan& p = k->plans[w];
    WeighArgs a;
    a.pool = h->pool;
    a.layer = layer;
    a.window = h->kinds[w];
    a.rows = std::min(rows, h->c.tokens);  // (a batch has no more; rows x group stays a number of 32 bits)
    a.table = h->dev;
    a.q = Rows{q, q_tok, q_head};
    a.sinks = sinks;
    a.scale = scale;
    a.decay = decay;
    a.stats = k->stats;
    a.work = k->work;
    int grid[WEIGH_LISTS];
    auto size = [&](int list) {
        return list <= SCORE_MANY ? p.scores[list].size()
               : list == MERGES   ? p.merges.size() * MERGE_WAYS
               : list < FADES     ? p.sums[list - SUM_FEW].size()
                                  : p.fades.size();
    };
    // a captured call has the kernels that some batch of the handle needs
    for (int l = 0; l < WEIGH_LISTS; l++)
        grid[l] = cap ? !may_weigh(h->shape, h->c.tokens, h->c.seqs, h->c.ctx, a.window, k->last, k->room, l) ? 0
                        : l == MERGES ? GRAPH_MERGES : GRAPH_WEIGH
                      : (int)std::min<size_t>(size(l), MOST_GRID);
    if (!cap && decay == 1) {  // what is not given anything stays as it is
        bool sums = false;
        for (const Fade& f : p.fades) sums |= f.sums > 0;
        if (!sums) grid[FADES] = 0;
    }
    const hipError_t e = launch_weigh(h->g, k->at, a, h->dev + k->batch_at + w * k->lists_at.words, k->lists_at, grid, h->stream);
    return e == hipSuccess ? MKV_OK : hip_fail(e, "mpg_weigh");
}

static int evict(mpg_t* h, int n, const int* seq, const int* keep, int first, int recent) {
    const char* const who = "mpg_evict";
    if (!h->weights) return fail(MKV_E_ARG, "%s: the handle keeps no weights (mpg_keep_weights)", who);
    if (first < 0 || recent < 0) return fail(MKV_E_ARG, "%s: %d first and %d last positions", who, first, recent);
    for (int w : h->kinds)
        if (recent < w) return fail(MKV_E_ARG, "%s: the last %d positions, a layer sees %d", who, recent, w);
    for (int i = 0; i < n && keep; i++)
        if (keep[i] < 1 || (long long)first + recent > keep[i])
            return fail(MKV_E_ARG, "%s: %d positions kept, %d first and %d last ones among them", who, keep[i], first, recent);
    if (int rc = h->book.can_evict(who, n, seq, keep)) return rc;
    // the device finds the rows that stay by the pages that the sequences have now
    if (const int rc = end_batch(h, who)) return rc;
    if (const int rc = upload_tables(h, who)) return rc;
    std::vector<Evicted> cut;
    if (int rc = h->book.evict(who, n, seq, keep, cut)) return rc;
    Kept* const k = kept(h);
    auto send = [&] {
        if (cut.empty()) return (int)MKV_OK;
        std::vector<Eviction> e;
        std::vector<NewPage> pages;
        int off = 0, longest = 0;
        for (const Evicted& c : cut) {
            const int m = h->book.len[c.seq];
            longest = std::max(longest, m);
            const std::vector<int>& t = h->book.table[c.seq];
            for (int p = 0; p < (int)t.size(); p++) pages.push_back({(int)e.size(), p, t[p]});
            e.push_back({c.seq, c.len, m, off});
            off += m;
        }
        const size_t stride = (size_t)h->c.pages * h->c.page;
        hipError_t err = launch_pick(h->g, k->at, e.data(), (int)e.size(), first, recent, k->entries, k->picks, k->heavy, stride, h->stream);
        if (err == hipSuccess)
            err = launch_gather(h->g, h->pool, h->dev, k->entries, k->picks, stride, pages.data(), (int)pages.size(), h->stream);
        if (err != hipSuccess) return hip_fail(err, who);
        // The weights move last, in one launch: whatever fails before it leaves them as they were. (The new tables go up when the
        // device next needs them.)
        err = launch_pack(k->at, k->entries, (int)e.size(), longest, k->heavy, stride, h->stream);
        return err == hipSuccess ? (int)MKV_OK : hip_fail(err, who);
    };
    int rc;
    try {
        rc = send();
    } catch (...) {
        h->book.undo_evict(cut);
        throw;
    }
    if (rc) h->book.undo_evict(cut);
    return rc;
}
int mpg_evict(mpg_t* h, int n, const int* seq, const int* keep, int first, int recent) {
    MPG_HOST_CALL(h, "mpg_evict");
    return guarded("mpg_evict", [&] { return evict(h, n, seq, keep, first, recent); });
}

int mpg_position(const mpg_t* h, int seq, int* position) {
    if (!h) return fail(MKV_E_ARG, "mpg_position: NULL handle");
    if (seq < 0 || seq >= h->c.seqs) return fail(MKV_E_ARG, "mpg_position: sequence %d outside [0, %d)", seq, h->c.seqs);
    if (!position) return fail(MKV_E_ARG, "mpg_position: NULL argument");
    *position = h->book.len[seq] + h->book.shift[seq];
    return MKV_OK;
}

}  // extern "C"

// paged_store.cpp -- the paged cache's handle and its C ABI (include/mechta_paged.h).
//
// The host knows every length and page, so it refuses what cannot be done before anything is enqueued and cuts a batch
// into work with its lengths in hand. What the kernels need of that (new entries of the page tables, the batch's runs of
// new tokens, the lists of work per window) goes to the device once per batch: the host writes it into pinned memory, one
// kernel puts it in place. The kernels of the layers read it there, so captured calls follow the batch.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <exception>
#include <memory>
#include <vector>

#include "mkv_store.h"
#include "paged_internal.h"

using mkv::fail;
using mkv::hip_fail;
using namespace mkv::paged;

namespace {
constexpr int RING = 4;           // staged uploads in flight
// Work-groups of a captured kernel, of whatever batch it finds (all loop over their lists): not many more than run at once,
// since those that find nothing are in the way too. 1 token at 100 positions, 4 at 20,000, 64 at 3,000 of 4 x 128: attention
// 10.3 / 21.1 / 65.8 us; with 512 of each kind and 16,384 for the joins 13.1 / 28.8 / 68.6.
constexpr int GRAPH_GRID = 1024, GRAPH_CHUNKS = 256, GRAPH_ROWS = 1024;
constexpr unsigned SEG = 256;     // words of an upload's segment at most: a thread of one work-group each
}  // namespace

struct mpg_store {
    mpg_config c;
    Geometry g;
    Shape shape;
    Book book;
    std::vector<int> windows;       // per layer
    std::vector<int> kinds;         // the different windows
    bool has_rope = false;
    RopeArgs rope;
    int device = 0;
    hipStream_t stream = nullptr;
    char* pool = nullptr;           // [layer][K|V][page]
    int* dev = nullptr;             // page tables, runs, one batch of lists per window
    size_t runs_at = 0, batch_at = 0, words = 0;  // word offsets in dev; its size
    Lists lists;
    float* part = nullptr;          // split partials
    unsigned* stage[RING] = {};     // pinned
    hipEvent_t done[RING] = {};
    size_t stage_words[RING] = {};
    int turn = 0;
    int tokens = -1;                // of the batch; -1: none stands
    int nruns = 0, longest = 0;     // its runs, and the tokens of the longest
    bool listed = false;            // the lists on the device are a batch's: replays would do it
    std::vector<Plan> plans, next;  // per window, of the batch and of the one that is being laid out
};

namespace {

struct OnDevice {  // makes a handle's device current, and the caller's again
    int was = -1;
    explicit OnDevice(int device) {
        int now = 0;
        if (hipGetDevice(&now) == hipSuccess && now != device && hipSetDevice(device) == hipSuccess) was = now;
    }
    ~OnDevice() {
        if (was >= 0) (void)hipSetDevice(was);
    }
};

int check_config(const char* who, const mpg_config* c) {
    if (!c) return fail(MKV_E_ARG, "%s: NULL argument", who);
    if (c->layers < 1 || c->layers > 4096) return fail(MKV_E_ARG, "%s: %d layers", who, c->layers);
    if (c->kv_heads < 1 || c->kv_heads > 1024 || c->q_heads < c->kv_heads || c->q_heads > 4096 || c->q_heads % c->kv_heads)
        return fail(MKV_E_ARG, "%s: %d query heads on %d kv heads", who, c->q_heads, c->kv_heads);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(MKV_E_ARG, "%s: head_dim %d (64, 128 or 256)", who, c->head_dim);
    if (c->fmt != MKV_F16 && c->fmt != MPG_BF16) return fail(MKV_E_ARG, "%s: format %d (f16 or bf16)", who, c->fmt);
    if (c->page != 32 && c->page != 64 && c->page != 128 && c->page != 256)
        return fail(MKV_E_ARG, "%s: pages of %d positions (32, 64, 128 or 256)", who, c->page);
    if (c->pages < 1 || c->pages > 1 << 27) return fail(MKV_E_ARG, "%s: %d pages", who, c->pages);
    if (c->seqs < 1 || c->seqs > 65536) return fail(MKV_E_ARG, "%s: %d sequences", who, c->seqs);
    if (c->ctx < 1 || c->ctx > MPG_CTX_MAX) return fail(MKV_E_CTX, "%s: context %d outside [1, %d]", who, c->ctx, MPG_CTX_MAX);
    if (c->tokens < 1 || c->tokens > MPG_TOKENS_MAX)
        return fail(MKV_E_ARG, "%s: batches of %d tokens outside [1, %d]", who, c->tokens, MPG_TOKENS_MAX);
    const size_t table = (size_t)c->seqs * ((c->ctx + c->page - 1) / c->page);
    if (table > 1u << 30) return fail(MKV_E_ARG, "%s: page tables of %zu entries", who, table);
    const double pool = 4. * c->layers * c->pages * c->kv_heads * c->page * c->head_dim;
    if (pool > 1ll << 48) return fail(MKV_E_NOMEM, "%s: a pool of %g bytes", who, pool);
    return MKV_OK;
}

struct Sizes {
    size_t pool, table, lists, words, part;
    Lists l;
};
Sizes sizes(const mpg_config& c, int kinds) {
    Sizes s;
    const Shape g{c.q_heads, c.kv_heads, c.head_dim};
    s.pool = (size_t)c.layers * 2 * c.pages * c.kv_heads * c.page * c.head_dim * 2;
    s.table = (size_t)c.seqs * ((c.ctx + c.page - 1) / c.page);
    const size_t items = most_items(g, c.tokens, c.seqs);
    size_t at = COUNTS;
    for (int k = 0; k < KINDS; k++) {
        s.l.items[k] = at;
        at += items * (sizeof(Item) / 4);
    }
    s.l.joins = at;
    at += most_joins(g, c.tokens, c.seqs) * (sizeof(Join) / 4);
    s.l.words = (at + 3) / 4 * 4;
    s.table = (s.table + 3) / 4 * 4;
    s.words = s.table + COUNTS + (size_t)c.tokens * (sizeof(Run) / 4) + s.l.words * kinds;
    s.part = (size_t)PART_ROWS * (2 + c.head_dim);
    return s;
}

int check_rope(const char* who, const mpg_rope* r) {
    if (!r) return fail(MKV_E_ARG, "%s: NULL argument", who);
    if (r->dim < 2 || r->dim > MPG_ROPE_DIM_MAX || r->dim % 2)
        return fail(MKV_E_ARG, "%s: rotated dim %d (even, 2 to %d)", who, r->dim, MPG_ROPE_DIM_MAX);
    if (r->layout != MPG_HALF && r->layout != MPG_INTERLEAVED) return fail(MKV_E_ARG, "%s: layout %d", who, r->layout);
    if (!(r->base > 1) || !std::isfinite(r->base)) return fail(MKV_E_ARG, "%s: base %g", who, r->base);
    if (r->scaling < MPG_PLAIN || r->scaling > MPG_BANDS) return fail(MKV_E_ARG, "%s: scaling %d", who, r->scaling);
    if (r->scaling != MPG_PLAIN && !(r->factor > 0 && std::isfinite(r->factor)))
        return fail(MKV_E_ARG, "%s: factor %g", who, r->factor);
    if (r->scaling == MPG_NTK && r->dim < 4) return fail(MKV_E_ARG, "%s: NTK scaling of %d elements", who, r->dim);
    if ((r->scaling == MPG_YARN || r->scaling == MPG_BANDS) && r->original < 1)
        return fail(MKV_E_ARG, "%s: original context %d", who, r->original);
    if (r->scaling == MPG_YARN && !(r->beta_fast > 0 && r->beta_slow > 0 && std::isfinite(r->beta_fast) && std::isfinite(r->beta_slow)))
        return fail(MKV_E_ARG, "%s: beta %g, %g", who, r->beta_fast, r->beta_slow);
    if (r->scaling == MPG_BANDS && !(r->high > r->low && std::isfinite(r->high) && std::isfinite(r->low)))
        return fail(MKV_E_ARG, "%s: bands %g, %g", who, r->low, r->high);
    if (!(r->amplitude >= 0) || !std::isfinite(r->amplitude)) return fail(MKV_E_ARG, "%s: amplitude %g", who, r->amplitude);
    return MKV_OK;
}

void freqs(const mpg_rope& r, double* th, double* amp) {
    const double two_pi = 2 * M_PI, base = r.scaling == MPG_NTK ? r.base * std::pow(r.factor, r.dim / (r.dim - 2.0)) : r.base;
    double lo = 0, hi = 0;
    if (r.scaling == MPG_YARN) {
        auto edge = [&](double turns) { return r.dim * std::log(r.original / (turns * two_pi)) / (2 * std::log(r.base)); };
        lo = std::max(std::floor(edge(r.beta_fast)), 0.0);
        hi = std::min(std::ceil(edge(r.beta_slow)), r.dim - 1.0);
    }
    for (int i = 0; i < r.dim / 2; i++) {
        double t = std::pow(base, -2.0 * i / r.dim);
        if (r.scaling == MPG_LINEAR) t /= r.factor;
        if (r.scaling == MPG_YARN) {
            const double m = std::min(1.0, std::max(0.0, (i - lo) / std::max(hi - lo, 0.001)));
            t = m * t / r.factor + (1 - m) * t;
        }
        if (r.scaling == MPG_BANDS) {
            const double m = std::min(1.0, std::max(0.0, (r.original * t / two_pi - r.low) / (r.high - r.low)));
            t = (1 - m) * t / r.factor + m * t;
        }
        th[i] = t;
    }
    *amp = r.amplitude > 0 ? r.amplitude : r.scaling == MPG_YARN && r.factor > 1 ? 0.1 * std::log(r.factor) + 1 : 1;
}

RopeArgs rope_args(const mpg_rope& r) {
    RopeArgs a;
    double amp;
    freqs(r, a.turns, &amp);
    for (int i = 0; i < r.dim / 2; i++) a.turns[i] /= 2 * M_PI;
    for (int i = r.dim / 2; i < MPG_ROPE_DIM_MAX / 2; i++) a.turns[i] = 0;
    a.amplitude = (float)amp;
    a.dim = r.dim;
    a.layout = r.layout;
    return a;
}

int check_layer(const mpg_store* h, int layer, const char* who) {
    if (!h) return fail(MKV_E_ARG, "%s: NULL handle", who);
    if (layer < 0 || layer >= h->c.layers) return fail(MKV_E_LAYER, "%s: layer %d outside [0, %d)", who, layer, h->c.layers);
    return MKV_OK;
}

// 0: not capturing, 1: capturing, < 0: an error that has been noted
int capturing(const mpg_store* h, const char* who) {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    const hipError_t e = hipStreamIsCapturing(h->stream, &st);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        return hip_fail(e, who);
    }
    return st == hipStreamCaptureStatusNone ? 0 : 1;
}

template <typename F>
int guarded(const char* who, F f) {  // no exception crosses the C boundary
    try {
        return f();
    } catch (const std::exception&) {
        return fail(MKV_E_NOMEM, "%s: host allocation", who);
    }
}

// A call that changes the host's book: with the handle's device current, refused while the stream captures.
#define MPG_HOST_CALL(h, who)                                                                                \
    if (!(h)) return fail(MKV_E_ARG, "%s: NULL handle", who);                                                \
    OnDevice on((h)->device);                                                                                \
    if (const int cap = capturing(h, who))                                                                   \
        return cap < 0 ? cap : fail(MKV_E_ARG, "%s: the stream is capturing; page calls run outside a graph", who)

int copy_pages(mpg_store* h, const std::vector<Pair>& copies, const char* who) {
    if (copies.empty()) return MKV_OK;
    const hipError_t e = launch_copies(h->g, h->pool, copies.data(), (int)copies.size(), h->stream);
    return e == hipSuccess ? MKV_OK : hip_fail(e, who);
}

// The new entries of the page tables to the device, and with `runs` the lists of a batch: its runs and plans, or (plans NULL)
// none. A call that fails has sent nothing.
int upload(mpg_store* h, const std::vector<Run>* runs, const std::vector<Plan>* plans, const char* who) {
    std::vector<Segment> segs;
    size_t at = 0;  // words of payload so far
    auto add = [&](size_t dst, size_t words) {
        for (size_t o = 0; o < words; o += SEG)
            segs.push_back({(unsigned)(dst + o), (unsigned)(at + o), (unsigned)std::min((size_t)SEG, words - o), 0});
        at += words;
    };
    struct Piece {
        const void* p;
        size_t words;
    };
    std::vector<Piece> pieces;
    auto put = [&](size_t dst, const void* p, size_t words) {
        if (!words) return;
        add(dst, words);
        pieces.push_back({p, words});
    };
    Book& b = h->book;
    for (int s = 0; s < b.seqs; s++) {
        const int n = (int)b.table[s].size();
        if (b.fresh[s] < n) put((size_t)s * h->g.most_pages + b.fresh[s], b.table[s].data() + b.fresh[s], n - b.fresh[s]);
    }
    int run_count[COUNTS] = {};
    std::vector<std::vector<int>> counts;
    if (runs) {
        run_count[0] = (int)runs->size();
        for (const Run& r : *runs) run_count[1] = std::max(run_count[1], r.count);
        put(h->runs_at, run_count, COUNTS);
        put(h->runs_at + COUNTS, runs->data(), runs->size() * (sizeof(Run) / 4));
        counts.assign(h->kinds.size(), std::vector<int>(COUNTS, 0));
        for (size_t w = 0; w < h->kinds.size(); w++) {
            const size_t base = h->batch_at + w * h->lists.words;
            if (!plans) {
                put(base, counts[w].data(), COUNTS);
                continue;
            }
            const Plan& p = (*plans)[w];
            for (int k = 0; k < KINDS; k++) counts[w][k] = (int)p.items[k].size();
            counts[w][KINDS] = (int)p.joins.size();
            put(base, counts[w].data(), COUNTS);
            for (int k = 0; k < KINDS; k++)
                put(base + h->lists.items[k], p.items[k].data(), p.items[k].size() * (sizeof(Item) / 4));
            put(base + h->lists.joins, p.joins.data(), p.joins.size() * (sizeof(Join) / 4));
        }
    }
    if (segs.empty()) return MKV_OK;
    const size_t head = segs.size() * (sizeof(Segment) / 4), all = head + at;
    const int slot = h->turn;
    hipError_t e = hipEventSynchronize(h->done[slot]);  // its upload of RING calls ago has been read
    if (e == hipSuccess && all > h->stage_words[slot]) {
        if (h->stage[slot]) (void)hipHostFree(h->stage[slot]);
        h->stage[slot] = nullptr;
        h->stage_words[slot] = 0;
        const size_t cap = std::max(all + all / 2, (size_t)16384);
        e = hipHostMalloc((void**)&h->stage[slot], cap * 4, hipHostMallocDefault);
        if (e == hipSuccess) h->stage_words[slot] = cap;
    }
    if (e != hipSuccess) {
        (void)hipGetLastError();
        return hip_fail(e, who);
    }
    unsigned* to = h->stage[slot];
    for (Segment& s : segs) s.src += (unsigned)head;
    memcpy(to, segs.data(), head * 4);
    to += head;
    for (const Piece& p : pieces) {
        memcpy(to, p.p, p.words * 4);
        to += p.words;
    }
    e = launch_apply(h->dev, h->stage[slot], (int)segs.size(), h->stream);
    if (e != hipSuccess) return hip_fail(e, who);
    if (hipEventRecord(h->done[slot], h->stream) != hipSuccess) {
        // on its way all the same, but nothing will tell when the buffer has been read: it is neither written nor freed again
        (void)hipGetLastError();
        h->stage[slot] = nullptr;
        h->stage_words[slot] = 0;
    }
    h->turn = (slot + 1) % RING;
    for (int s = 0; s < b.seqs; s++) b.fresh[s] = (int)b.table[s].size();
    return MKV_OK;
}

// What replays of captured calls do once pages have changed hands and no batch stands: nothing. The batch stands until the
// empty lists are on their way.
int end_batch(mpg_store* h, const char* who) {
    if (!h->listed) return MKV_OK;
    const std::vector<Run> none;
    if (const int rc = upload(h, &none, nullptr, who)) return rc;
    h->listed = false;
    h->tokens = -1;
    return MKV_OK;
}

// What the device has to do for a call that has changed the book: the batch ends, pages are copied. Where it cannot be told,
// the book is put back.
template <typename U>
int settle(mpg_store* h, const std::vector<Pair>& copies, const char* who, U undo) {
    int rc;
    try {
        rc = end_batch(h, who);
        if (!rc) rc = copy_pages(h, copies, who);
    } catch (...) {
        undo();
        throw;
    }
    if (rc) undo();
    return rc;
}

int check_batch(const mpg_store* h, int rows, const char* who) {
    if (h->tokens < 0) return fail(MKV_E_ARG, "%s: no batch stands (mpg_begin)", who);
    if (rows < h->tokens) return fail(MKV_E_SIZE, "%s: %d rows, the batch has %d tokens", who, rows, h->tokens);
    return MKV_OK;
}

int check_rows(const char* who, const char* what, const void* p, int rows, int64_t tok, int heads, int64_t head) {
    if (!p) return fail(MKV_E_ARG, "%s: NULL %s", who, what);
    if ((uintptr_t)p % 16 || (rows > 1 && tok % 8) || (heads > 1 && head % 8))
        return fail(MKV_E_ARG, "%s: %s must be 16-byte aligned, its strides multiples of 8 elements", who, what);
    return MKV_OK;
}

}  // namespace

extern "C" {

int mpg_rope_freqs(const mpg_rope* r, double* th, double* amplitude) {
    if (int rc = check_rope("mpg_rope_freqs", r)) return rc;
    if (!th || !amplitude) return fail(MKV_E_ARG, "mpg_rope_freqs: NULL argument");
    freqs(*r, th, amplitude);
    return MKV_OK;
}

int mpg_rope_turns(const mpg_rope* r, mpg_turns* turns) {
    if (int rc = check_rope("mpg_rope_turns", r)) return rc;
    if (!turns) return fail(MKV_E_ARG, "mpg_rope_turns: NULL argument");
    *turns = rope_args(*r);
    return MKV_OK;
}

int mpg_rotate(const mpg_turns* r, int fmt, int rows, int heads, int dim, const void* x, int64_t x_row, int64_t x_head,
               const int* pos, void* out, int64_t o_row, int64_t o_head, void* stream) {
    if (!r) return fail(MKV_E_ARG, "mpg_rotate: NULL argument");
    if (r->dim < 2 || r->dim > MPG_ROPE_DIM_MAX || r->dim % 2 || (r->layout != MPG_HALF && r->layout != MPG_INTERLEAVED))
        return fail(MKV_E_ARG, "mpg_rotate: rotated dim %d, layout %d", r->dim, r->layout);
    if (fmt != MKV_F16 && fmt != MKV_F32 && fmt != MPG_BF16) return fail(MKV_E_ARG, "mpg_rotate: format %d", fmt);
    if (rows < 0 || heads < 0 || heads > 65536) return fail(MKV_E_ARG, "mpg_rotate: %d rows x %d heads", rows, heads);
    if (dim < r->dim || dim > 4096) return fail(MKV_E_ARG, "mpg_rotate: heads of %d elements, %d of them rotated", dim, r->dim);
    if (!rows || !heads) return MKV_OK;
    if (!x || !pos || !out) return fail(MKV_E_ARG, "mpg_rotate: NULL argument");
    if (x == out && (x_row != o_row || x_head != o_head))
        return fail(MKV_E_ARG, "mpg_rotate: in place needs the same strides");
    const int64_t row = std::llabs(o_row), head = std::llabs(o_head);
    if ((rows > 1 && row < dim) || (heads > 1 && head < dim) || (rows > 1 && heads > 1 && row == head))
        return fail(MKV_E_ARG, "mpg_rotate: rows or heads of out lie on each other (strides %lld, %lld)", (long long)o_row, (long long)o_head);
    const size_t bytes = fmt == MKV_F32 ? 4 : 2;
    if ((uintptr_t)x % bytes || (uintptr_t)out % bytes || (uintptr_t)pos % 4)
        return fail(MKV_E_ARG, "mpg_rotate: misaligned pointer");
    const hipError_t e = launch_rotate(*r, fmt, rows, heads, dim, Rows{x, x_row, x_head}, pos,
                                       Rows{out, o_row, o_head}, (hipStream_t)stream);
    return e == hipSuccess ? MKV_OK : hip_fail(e, "mpg_rotate");
}

size_t mpg_bytes(const mpg_config* c) {
    if (check_config("mpg_bytes", c)) return 0;
    const Sizes s = sizes(*c, MPG_WINDOWS_MAX);
    return s.pool + (s.words + s.part) * 4;
}

static int create(mpg_t** out, const mpg_config* c, const int* windows, const mpg_rope* rope, void* stream) {
    if (!out) return fail(MKV_E_ARG, "mpg_create: NULL argument");
    *out = nullptr;
    if (int rc = check_config("mpg_create", c)) return rc;
    if (rope) {
        if (int rc = check_rope("mpg_create", rope)) return rc;
        if (rope->dim > c->head_dim)
            return fail(MKV_E_ARG, "mpg_create: %d rotated elements of heads of %d", rope->dim, c->head_dim);
    }
    std::vector<int> per_layer(c->layers, 0), kinds;
    for (int l = 0; l < c->layers; l++) {
        const int w = windows ? windows[l] : 0;
        if (w < 0) return fail(MKV_E_ARG, "mpg_create: window %d of layer %d", w, l);
        auto it = std::find(kinds.begin(), kinds.end(), w);
        per_layer[l] = (int)(it - kinds.begin());
        if (it == kinds.end()) kinds.push_back(w);
    }
    if (kinds.size() > MPG_WINDOWS_MAX)
        return fail(MKV_E_ARG, "mpg_create: %zu different windows, at most %d", kinds.size(), MPG_WINDOWS_MAX);
    std::unique_ptr<mpg_store> owner(new mpg_store);
    mpg_store* const h = owner.get();
    const Sizes s = sizes(*c, MPG_WINDOWS_MAX);
    h->c = *c;
    h->g = Geometry{c->layers, c->q_heads, c->kv_heads, c->head_dim, c->fmt, c->pages, c->page, (c->ctx + c->page - 1) / c->page};
    h->shape = Shape{c->q_heads, c->kv_heads, c->head_dim};
    h->windows = per_layer;
    h->kinds = kinds;
    h->plans.resize(kinds.size());
    h->next.resize(kinds.size());
    h->has_rope = rope != nullptr;
    if (rope) h->rope = rope_args(*rope);
    h->stream = (hipStream_t)stream;
    h->lists = s.l;
    h->runs_at = s.table;
    h->batch_at = s.table + COUNTS + (size_t)c->tokens * (sizeof(Run) / 4);
    h->words = s.words;
    h->book.init(c->pages, c->page, c->seqs, c->ctx);
    if (const int cap = capturing(h, "mpg_create"))
        return cap < 0 ? cap : fail(MKV_E_ARG, "mpg_create: the stream is capturing");
    hipError_t e = s.words < 1ull << 32 ? hipGetDevice(&h->device) : hipErrorOutOfMemory;
    if (e == hipSuccess) e = hipMalloc((void**)&h->pool, s.pool);
    if (e == hipSuccess) e = hipMalloc((void**)&h->dev, s.words * 4);
    if (e == hipSuccess) e = hipMalloc((void**)&h->part, s.part * 4);
    if (e == hipSuccess) e = hipMemsetAsync(h->pool, 0, s.pool, h->stream);
    if (e == hipSuccess) e = hipMemsetAsync(h->dev, 0, s.words * 4, h->stream);
    for (int i = 0; i < RING && e == hipSuccess; i++) e = hipEventCreateWithFlags(&h->done[i], hipEventDisableTiming);
    if (e == hipSuccess) e = hipStreamSynchronize(h->stream);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        const size_t all = s.pool + (s.words + s.part) * 4;
        for (hipEvent_t ev : h->done)
            if (ev) (void)hipEventDestroy(ev);
        if (h->pool) (void)hipFree(h->pool);
        if (h->dev) (void)hipFree(h->dev);
        if (h->part) (void)hipFree(h->part);
        return fail(MKV_E_NOMEM, "mpg_create: %zu bytes: %s", all, hipGetErrorString(e));
    }
    *out = owner.release();
    return MKV_OK;
}

int mpg_create(mpg_t** out, const mpg_config* c, const int* windows, const mpg_rope* rope, void* stream) {
    return guarded("mpg_create", [&] { return create(out, c, windows, rope, stream); });
}

int mpg_destroy(mpg_t* h) {
    if (!h) return MKV_OK;
    OnDevice on(h->device);
    const hipError_t e = hipStreamSynchronize(h->stream);
    for (int i = 0; i < RING; i++) {
        if (h->done[i]) (void)hipEventDestroy(h->done[i]);
        if (h->stage[i]) (void)hipHostFree(h->stage[i]);
    }
    (void)hipFree(h->pool);
    (void)hipFree(h->dev);
    (void)hipFree(h->part);
    delete h;
    return e == hipSuccess ? MKV_OK : hip_fail(e, "mpg_destroy");
}

int mpg_set_stream(mpg_t* h, void* stream) {
    if (!h) return fail(MKV_E_ARG, "mpg_set_stream: NULL handle");
    h->stream = (hipStream_t)stream;
    return MKV_OK;
}

int mpg_sync(mpg_t* h) {
    if (!h) return fail(MKV_E_ARG, "mpg_sync: NULL handle");
    OnDevice on(h->device);
    const hipError_t e = hipStreamSynchronize(h->stream);
    return e == hipSuccess ? MKV_OK : hip_fail(e, "mpg_sync");
}

static int check_seq(const mpg_t* h, int seq, const char* who) {
    if (!h) return fail(MKV_E_ARG, "%s: NULL handle", who);
    if (seq < 0 || seq >= h->c.seqs) return fail(MKV_E_ARG, "%s: sequence %d outside [0, %d)", who, seq, h->c.seqs);
    return MKV_OK;
}

int mpg_len(const mpg_t* h, int seq, int* len) {
    if (int rc = check_seq(h, seq, "mpg_len")) return rc;
    if (len) *len = h->book.len[seq];
    return MKV_OK;
}

int mpg_table(const mpg_t* h, int seq, int* pages, int cap) {
    if (int rc = check_seq(h, seq, "mpg_table")) return rc;
    const std::vector<int>& t = h->book.table[seq];
    if (cap > 0 && !pages) return fail(MKV_E_ARG, "mpg_table: NULL argument");
    for (int i = 0; i < (int)t.size() && i < cap; i++) pages[i] = t[i];
    return (int)t.size();
}

int mpg_free_pages(const mpg_t* h, int* n) {
    if (!h || !n) return fail(MKV_E_ARG, "mpg_free_pages: NULL argument");
    *n = h->book.free;
    return MKV_OK;
}

int mpg_pages(const mpg_t* h, int layer, int which, void** base) {
    if (int rc = check_layer(h, layer, "mpg_pages")) return rc;
    if (which != MKV_K && which != MKV_V) return fail(MKV_E_ARG, "mpg_pages: which = %d", which);
    if (!base) return fail(MKV_E_ARG, "mpg_pages: NULL argument");
    *base = h->pool + ((size_t)layer * 2 + which) * h->g.plane_elems() * 2;
    return MKV_OK;
}

int mpg_reserve(mpg_t* h, int n, const int* seq, const int* count) {
    MPG_HOST_CALL(h, "mpg_reserve");
    return guarded("mpg_reserve", [&] {
        if (int rc = h->book.reserve("mpg_reserve", n, seq, count)) return rc;
        return settle(h, {}, "mpg_reserve", [&] { h->book.undo_reserve(n, seq, count); });
    });
}

// The batch of sequences that have been lengthened already: its runs, its plans, and both on their way to the device. Where
// that fails the batch before stands.
static int lay_out(mpg_t* h, int n, const int* seq, const int* count) {
    std::vector<Member> batch;
    std::vector<Run> runs;
    int tok = 0, longest = 0;
    for (int i = 0; i < n; i++) {
        const int len = h->book.len[seq[i]];
        batch.push_back({seq[i], count[i], len});
        for (int p = len - count[i]; p < len;) {
            const int m = std::min(len, (p / KEYS + 1) * KEYS) - p;
            runs.push_back({seq[i], tok, p, m});
            p += m;
            tok += m;
            longest = std::max(longest, m);
        }
    }
    for (size_t w = 0; w < h->kinds.size(); w++) plan_window(h->shape, batch, h->kinds[w], h->next[w]);
    if (int rc = upload(h, &runs, &h->next, "mpg_begin")) return rc;
    h->listed = true;
    h->plans.swap(h->next);
    h->tokens = tok;
    h->nruns = (int)runs.size();
    h->longest = longest;
    return MKV_OK;
}

static int begin(mpg_t* h, int n, const int* seq, const int* count, int* tokens) {
    long long sum = 0;
    for (int i = 0; i < n && seq && count; i++) sum += std::max(count[i], 0);
    if (sum > h->c.tokens)
        return fail(MKV_E_ARG, "mpg_begin: %lld tokens, the handle's batches have at most %d", sum, h->c.tokens);
    if (int rc = h->book.reserve("mpg_begin", n, seq, count)) return rc;
    try {
        const int rc = lay_out(h, n, seq, count);
        if (rc) h->book.undo_reserve(n, seq, count);
        else if (tokens) *tokens = h->tokens;
        return rc;
    } catch (...) {
        h->book.undo_reserve(n, seq, count);
        throw;
    }
}

int mpg_begin(mpg_t* h, int n, const int* seq, const int* count, int* tokens) {
    MPG_HOST_CALL(h, "mpg_begin");
    return guarded("mpg_begin", [&] { return begin(h, n, seq, count, tokens); });
}
int mpg_set_len(mpg_t* h, int seq, int len) {
    MPG_HOST_CALL(h, "mpg_set_len");
    return guarded("mpg_set_len", [&] {
        std::vector<Pair> copies;
        Cut cut;
        if (int rc = h->book.set_len("mpg_set_len", seq, len, copies, &cut)) return rc;
        return settle(h, copies, "mpg_set_len", [&] { h->book.undo_set_len(seq, cut); });
    });
}

static int fork_pages(mpg_t* h, int n, const int* src, const int* dst, const int* len, bool own, const char* who) {
    MPG_HOST_CALL(h, who);
    return guarded(who, [&] {
        std::vector<Pair> copies;
        if (int rc = h->book.fork(who, n, src, dst, len, own, copies)) return rc;
        return settle(h, copies, who, [&] { h->book.undo_fork(n, dst); });
    });
}

int mpg_fork(mpg_t* h, int n, const int* src, const int* dst, const int* len) {
    return fork_pages(h, n, src, dst, len, false, "mpg_fork");
}
int mpg_copy(mpg_t* h, int n, const int* src, const int* dst) {
    return fork_pages(h, n, src, dst, nullptr, true, "mpg_copy");
}

int mpg_free(mpg_t* h, int n, const int* seq) {
    MPG_HOST_CALL(h, "mpg_free");
    return guarded("mpg_free", [&] {
        return h->book.release("mpg_free", n, seq, [&] { return end_batch(h, "mpg_free"); });
    });
}

int mpg_compact(mpg_t* h, int* moved) {
    MPG_HOST_CALL(h, "mpg_compact");
    return guarded("mpg_compact", [&] {
        std::vector<Pair> copies;
        const int n = h->book.compact(copies);
        if (int rc = settle(h, copies, "mpg_compact", [&] { h->book.undo_compact(copies); })) return rc;
        if (moved) *moved = n;
        return MKV_OK;
    });
}

int mpg_append(mpg_t* h, int layer, int rows, const void* k, int64_t k_tok, int64_t k_head, const void* v, int64_t v_tok,
               int64_t v_head, const void* q, int64_t q_tok, int64_t q_head, void* q_out, int rotate) {
    if (int rc = check_layer(h, layer, "mpg_append")) return rc;
    if (int rc = check_batch(h, rows, "mpg_append")) return rc;
    if (!rows) return MKV_OK;
    if (int rc = check_rows("mpg_append", "k", k, rows, k_tok, h->c.kv_heads, k_head)) return rc;
    if (int rc = check_rows("mpg_append", "v", v, rows, v_tok, h->c.kv_heads, v_head)) return rc;
    if (rotate && !h->has_rope) return fail(MKV_E_ARG, "mpg_append: the handle has no rotary positions");
    if (q) {
        if (!rotate) return fail(MKV_E_ARG, "mpg_append: q without rotation");
        if (int rc = check_rows("mpg_append", "q", q, rows, q_tok, h->c.q_heads, q_head)) return rc;
        if (int rc = check_rows("mpg_append", "q_out", q_out, 1, 0, 1, 0)) return rc;
        if (q == q_out && ((h->c.q_heads > 1 && q_head != h->c.head_dim) ||
                           (rows > 1 && q_tok != (int64_t)h->c.q_heads * h->c.head_dim)))
            return fail(MKV_E_ARG, "mpg_append: in place needs q in one piece");
    }
    OnDevice on(h->device);
    const int cap = capturing(h, "mpg_append");
    if (cap < 0) return cap;
    if (!cap && !h->nruns) return MKV_OK;
    const hipError_t e = launch_append(h->g, h->pool, layer, h->dev, (const Run*)(h->dev + h->runs_at + COUNTS),
                                       h->dev + h->runs_at, cap ? GRAPH_ROWS : 0, h->nruns, h->longest, rows,
                                       Rows{k, k_tok, k_head}, Rows{v, v_tok, v_head}, Rows{q, q_tok, q_head}, q_out,
                                       rotate ? &h->rope : nullptr, h->stream);
    return e == hipSuccess ? MKV_OK : hip_fail(e, "mpg_append");
}

int mpg_attend(mpg_t* h, int layer, int rows, const void* q, int64_t q_tok, int64_t q_head, float scale, const float* sinks,
               const void* gate, int64_t g_tok, int64_t g_head, void* out) {
    if (int rc = check_layer(h, layer, "mpg_attend")) return rc;
    if (int rc = check_batch(h, rows, "mpg_attend")) return rc;
    if (!rows) return MKV_OK;
    if (int rc = check_rows("mpg_attend", "q", q, rows, q_tok, h->c.q_heads, q_head)) return rc;
    if (int rc = check_rows("mpg_attend", "out", out, 1, 0, 1, 0)) return rc;
    if (gate)
        if (int rc = check_rows("mpg_attend", "gate", gate, rows, g_tok, h->c.q_heads, g_head)) return rc;
    if (out == q || out == gate) return fail(MKV_E_ARG, "mpg_attend: out takes the place of an input");
    if (!(scale > 0) || !std::isfinite(scale)) return fail(MKV_E_ARG, "mpg_attend: scale %g", scale);
    if ((uintptr_t)sinks % 4) return fail(MKV_E_ARG, "mpg_attend: misaligned sinks");
    OnDevice on(h->device);
    const int cap = capturing(h, "mpg_attend");
    if (cap < 0) return cap;
    const int w = h->windows[layer];
    const Plan& p = h->plans[w];
    AttendArgs a;
    a.pool = h->pool;
    a.layer = layer;
    a.rows = rows;
    a.window = h->kinds[w];
    a.table = h->dev;
    a.q = Rows{q, q_tok, q_head};
    a.gate = Rows{gate, g_tok, g_head};
    a.sinks = sinks;
    a.out = out;
    a.scale = scale;
    a.pm = h->part;
    a.pl = h->part + PART_ROWS;
    a.pacc = h->part + 2 * (size_t)PART_ROWS;
    a.joins = &p.joins;
    a.captured = cap != 0;
    int grid[KINDS];
    for (int k = 0; k < KINDS; k++)
        grid[k] = cap ? (k < HALF ? GRAPH_GRID : GRAPH_CHUNKS) : (int)std::min<size_t>(p.items[k].size(), MOST_GRID);
    const hipError_t e = launch_attend(h->g, a, h->dev + h->batch_at + w * h->lists.words, h->lists, grid,
                                       cap ? GRAPH_ROWS : (int)std::min<size_t>(p.joins.size(), MOST_GRID), h->stream);
    return e == hipSuccess ? MKV_OK : hip_fail(e, "mpg_attend");
}

int mpg_read_rows(mpg_t* h, int layer, int which, int seq, int p0, int p1, void* dst) {
    if (int rc = check_layer(h, layer, "mpg_read_rows")) return rc;
    if (int rc = check_seq(h, seq, "mpg_read_rows")) return rc;
    if (which != MKV_K && which != MKV_V) return fail(MKV_E_ARG, "mpg_read_rows: which = %d", which);
    if (p0 < 0 || p1 < p0 || p1 > h->book.len[seq])
        return fail(MKV_E_POS, "mpg_read_rows: positions [%d, %d) of %d", p0, p1, h->book.len[seq]);
    if (p0 == p1) return MKV_OK;
    if (!dst || (uintptr_t)dst % 16) return fail(MKV_E_ARG, "mpg_read_rows: the buffer must be 16-byte aligned");
    OnDevice on(h->device);
    const int cap = capturing(h, "mpg_read_rows");
    if (cap < 0) return cap;
    const Book& b = h->book;
    if (cap && b.fresh[seq] < (int)b.table[seq].size())
        return fail(MKV_E_ARG, "mpg_read_rows: the device does not have the sequence's pages yet; read once before capturing");
    if (!cap)
        if (int rc = guarded("mpg_read_rows", [&] { return upload(h, nullptr, nullptr, "mpg_read_rows"); })) return rc;
    const hipError_t e = launch_read(h->g, h->pool, layer, which, h->dev + (size_t)seq * h->g.most_pages, p0, p1, dst, h->stream);
    return e == hipSuccess ? MKV_OK : hip_fail(e, "mpg_read_rows");
}

}  // extern "C"

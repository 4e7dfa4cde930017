// paged_handle.h -- the paged cache's handle, and what the calls on it have in common.
#pragma once
#include <hip/hip_runtime.h>

#include <exception>
#include <functional>
#include <memory>
#include <vector>

#include "mkv_store.h"
#include "paged_internal.h"

namespace mkv {
namespace paged {
constexpr int RING = 4;           // staged uploads in flight

// What a handle that keeps attention weights has to do when its sequences change (paged_weights.cpp).
struct Weights {
    virtual ~Weights() = default;
    // Positions [from, from + count) of the sequences are new: they weigh nothing. (What lies behind a sequence's length may
    // be anything, so it does not matter if the call that is about to lengthen it fails.)
    virtual int clear(int n, const int* seq, const int* from, const int* count, const char* who) = 0;
    // The first len[i] positions of dst[i], which is empty, weigh what those of src[i] do.
    virtual int copy(int n, const int* src, const int* dst, const int* len, const char* who) = 0;
    // The work of a batch, its lists for the device (none: no batch), and that it stands.
    virtual void lay_out(const std::vector<Member>& batch) = 0;
    virtual void lists(bool none, const std::function<void(size_t, const void*, size_t)>& put) = 0;
    virtual void stands() = 0;
};

// Work-groups of a captured kernel, of whatever batch it finds (all loop over their lists): not many more than run at once,
// since those that find nothing are in the way too. 1 token at 100 positions, 4 at 20,000, 64 at 3,000 of 4 x 128: attention
// 10.3 / 21.1 / 65.8 us; with 512 of each kind and 16,384 for the joins 13.1 / 28.8 / 68.6.
constexpr int GRAPH_GRID = 1024, GRAPH_CHUNKS = 256, GRAPH_ROWS = 1024;
}  // namespace paged
}  // namespace mkv

struct mpg_store {
    mpg_config c;
    mkv::paged::Geometry g;
    mkv::paged::Shape shape;
    mkv::paged::Book book;
    std::vector<int> windows;       // per layer
    std::vector<int> kinds;         // the different windows
    bool has_rope = false;
    mkv::paged::RopeArgs rope;
    int device = 0;
    hipStream_t stream = nullptr;
    char* pool = nullptr;           // [layer][K|V][page]
    int* dev = nullptr;             // page tables, runs, one batch of lists per window, the order of a shared batch
    size_t runs_at = 0, batch_at = 0, order_at = 0, words = 0;  // word offsets in dev; its size
    mkv::paged::Lists lists;
    float* part = nullptr;          // split partials
    unsigned* stage[mkv::paged::RING] = {};     // pinned
    hipEvent_t done[mkv::paged::RING] = {};
    size_t stage_words[mkv::paged::RING] = {};
    int turn = 0;
    int tokens = -1;                // of the batch; -1: none stands
    int nruns = 0, longest = 0;     // its runs, and the tokens of the longest
    bool listed = false;            // the lists on the device are a batch's: replays would do it
    std::vector<mkv::paged::Plan> plans, next;  // per window, of the batch and of the one that is being laid out
    bool used = false;              // sequences have had positions: captured calls may hold the handle's addresses
    size_t shift_at = 0;            // word offset in dev of the sequences' evicted positions; 0: nothing is ever evicted
    std::unique_ptr<mkv::paged::Weights> weights;  // none: the handle keeps no weights
};

namespace mkv {
namespace paged {

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

inline int check_layer(const mpg_store* h, int layer, const char* who) {
    if (!h) return fail(MKV_E_ARG, "%s: NULL handle", who);
    if (layer < 0 || layer >= h->c.layers) return fail(MKV_E_LAYER, "%s: layer %d outside [0, %d)", who, layer, h->c.layers);
    return MKV_OK;
}

inline int check_batch(const mpg_store* h, int rows, const char* who) {
    if (h->tokens < 0) return fail(MKV_E_ARG, "%s: no batch stands (mpg_begin)", who);
    if (rows < h->tokens) return fail(MKV_E_SIZE, "%s: %d rows, the batch has %d tokens", who, rows, h->tokens);
    return MKV_OK;
}

inline int check_rows(const char* who, const char* what, const void* p, int rows, int64_t tok, int heads, int64_t head) {
    if (!p) return fail(MKV_E_ARG, "%s: NULL %s", who, what);
    if ((uintptr_t)p % 16 || (rows > 1 && tok % 8) || (heads > 1 && head % 8))
        return fail(MKV_E_ARG, "%s: %s must be 16-byte aligned, its strides multiples of 8 elements", who, what);
    return MKV_OK;
}

// 0: not capturing, 1: capturing, < 0: an error that has been noted
inline int capturing(const mpg_store* h, const char* who) {
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

// paged_store.cpp: words of a handle's tables and lists on the device, which with those of its weights are fewer than WORDS_MOST
// (an upload's offsets are numbers of 32 bits).
constexpr size_t WORDS_MOST = 1ull << 32;
size_t handle_words(const mpg_config& c);
// The batch that stands ends; what the device does not know of the page tables and shifts goes up.
int end_batch(mpg_store* h, const char* who);
int upload_tables(mpg_store* h, const char* who);

}  // namespace paged
}  // namespace mkv

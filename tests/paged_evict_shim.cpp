// The paged cache's handle with weights, and eviction, on a device made of host memory (paged_store_shim.cpp has the calls of it that
// can be told to fail), for tests/test_paged_evict.py.
#include "paged_store_shim.cpp"
#include "../mechta_amd/csrc/paged_weights.cpp"

static int weighed = 0;
namespace mkv {
namespace paged {
hipError_t launch_clear(const WeightsAt& w, const Change* c, int n, hipStream_t) {
    for (int i = 0; i < n; i++) {
        if (const hipError_t e = step(hipErrorLaunchFailure)) return e;
        for (int l = 0; l < w.layers; l++)
            for (int h = 0; h < w.kv_heads; h++) memset(w.p + w.at(l, c[i].seq, h) + c[i].a, 0, c[i].count * 4);
    }
    return hipSuccess;
}
hipError_t launch_weights_copy(const WeightsAt& w, const Change* c, int n, hipStream_t) {
    for (int i = 0; i < n; i++) {
        if (const hipError_t e = step(hipErrorLaunchFailure)) return e;
        for (int l = 0; l < w.layers; l++)
            for (int h = 0; h < w.kv_heads; h++) memcpy(w.p + w.at(l, c[i].seq, h) + c[i].a, w.p + w.at(l, c[i].other, h) + c[i].a, c[i].count * 4);
    }
    return hipSuccess;
}
hipError_t launch_weigh(const Geometry&, const WeightsAt&, const WeighArgs&, const int*, const WeighLists&, const int*, hipStream_t) {
    weighed++;
    return hipSuccess;
}
// every second of the positions between, whatever they weigh
hipError_t launch_pick(const Geometry& g, const WeightsAt& w, const Eviction* e, int n, int first, int recent, Eviction* entries, int* picks,
                       float* heavy, size_t stride, hipStream_t) {
    for (int i = 0; i < n; i++) {
        if (const hipError_t err = step(hipErrorLaunchFailure)) return err;
        entries[i] = e[i];
        for (int u = 0; u < g.layers * g.kv_heads; u++)
            for (int k = 0, m = 0; k < e[i].keep; k++) {
                const int mid = e[i].keep - first - recent, free = e[i].len - first - recent - mid;
                const int p = picks[u * stride + e[i].off + k] = k < first ? k : k < first + mid ? first + std::min(free, ++m) + k - first : e[i].len - e[i].keep + k;
                heavy[u * stride + e[i].off + k] = w.p[w.at(u / w.kv_heads, e[i].seq, u % w.kv_heads) + p];
            }
    }
    return hipSuccess;
}
// a position's mark stands for its rows, in every plane
hipError_t launch_gather(const Geometry& g, char* pool, const int* table, const Eviction* entries, const int* picks, size_t, const NewPage* pages,
                         int n, hipStream_t) {
    for (int i = 0; i < n; i++) {
        if (const hipError_t err = step(hipErrorLaunchFailure)) return err;
        const Eviction e = entries[pages[i].entry];
        for (int at = 0; at < g.page && pages[i].nth * g.page + at < e.keep; at++) {
            const int p = picks[e.off + pages[i].nth * g.page + at], from = table[(size_t)e.seq * g.most_pages + p / g.page];
            for (int l = 0; l < 2 * g.layers; l++) {
                char* const plane = pool + l * g.plane_elems() * 2;
                *(int*)(plane + pages[i].page * g.page_elems() * 2 + at * 4) = *(int*)(plane + from * g.page_elems() * 2 + p % g.page * 4);
            }
        }
    }
    return hipSuccess;
}
hipError_t launch_pack(const WeightsAt& w, const Eviction* entries, int n, int longest, const float* heavy, size_t stride, hipStream_t) {
    if (const hipError_t err = step(hipErrorLaunchFailure)) return err;
    for (int i = 0; i < n; i++)
        for (int u = 0; u < w.layers * w.kv_heads; u++) {
            float* const p = w.p + w.at(u / w.kv_heads, entries[i].seq, u % w.kv_heads);
            for (int k = 0; k < std::min(longest, entries[i].keep); k++) p[k] = heavy[u * stride + entries[i].off + k];
        }
    return hipSuccess;
}
}  // namespace paged
}  // namespace mkv

extern "C" {
int shim_weighed() { return weighed; }
int shim_shift(const mpg_t* h, int seq) { return h->dev[h->shift_at + seq]; }
int shim_moved(const mpg_t* h, int seq) { return h->book.moved[seq]; }
// entries of all lists of weighing on the device, of a window
int shim_weigh_work(const mpg_t* h, int window) {
    const Kept* const k = kept(h);
    int n = 0;
    for (int l = 0; l < WEIGH_LISTS; l++) n += h->dev[k->batch_at + window * k->lists_at.words + l];
    return n;
}
}

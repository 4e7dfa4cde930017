// The paged cache's handle on a device made of host memory, for tests/test_paged_store.py: the HIP calls and launches that
// paged_store.cpp makes, each of which can be told to fail, and what a replay of captured calls would find "on the device".
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <new>

#include "../mechta_amd/csrc/paged_store.cpp"

static long left = -1;  // fallible steps that still succeed; -1: all of them
static long steps = 0;  // taken since the last shim_fail_after
static bool fails() {
    steps++;
    return left >= 0 && left-- == 0;
}
static hipError_t step(hipError_t bad) { return fails() ? bad : hipSuccess; }

void* operator new(size_t n) {
    if (fails()) throw std::bad_alloc();
    if (void* p = malloc(n ? n : 1)) return p;
    throw std::bad_alloc();
}
void operator delete(void* p) noexcept { free(p); }
void operator delete(void* p, size_t) noexcept { free(p); }

static char message[512];
static int record_fails = 0, capturing_now = 0, copied = 0, appended = 0, attended = 0;
namespace mkv {
int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(message, sizeof message, fmt, ap);
    va_end(ap);
    return code;
}
int hip_fail(hipError_t, const char* what) { return fail(MKV_E_HIP, "%s: device", what); }

namespace paged {
hipError_t launch_apply(int* dev, const unsigned* stage, int segments, hipStream_t) {
    if (const hipError_t e = step(hipErrorLaunchFailure)) return e;
    for (int i = 0; i < segments; i++) {
        const Segment s = ((const Segment*)stage)[i];
        memcpy(dev + s.dst, stage + s.src, s.words * 4);
    }
    return hipSuccess;
}
hipError_t launch_copies(const Geometry& g, char* pool, const Pair* pairs, int n, hipStream_t) {
    const size_t page = g.page_elems() * 2, plane = g.plane_elems() * 2;
    for (int i = 0; i < n; i++) {
        if (i % 2 == 0)  // two pairs a launch
            if (const hipError_t e = step(hipErrorLaunchFailure)) return e;
        for (int p = 0; p < 2 * g.layers; p++) memcpy(pool + p * plane + pairs[i].dst * page, pool + p * plane + pairs[i].src * page, page);
        copied++;
    }
    return hipSuccess;
}
hipError_t launch_append(const Geometry&, char*, int, const int*, const Run*, const int*, int, int, int, int, const Rows&,
                         const Rows&, const Rows&, void*, const RopeArgs*, hipStream_t) {
    appended++;
    return hipSuccess;
}
hipError_t launch_read(const Geometry&, const char*, int, int, const int*, int, int, void*, hipStream_t) { return hipSuccess; }
hipError_t launch_rotate(const RopeArgs&, int, int, int, int, const Rows&, const int*, const Rows&, hipStream_t) { return hipSuccess; }
hipError_t launch_attend(const Geometry&, const AttendArgs&, const int*, const Lists&, const int*, int, hipStream_t) {
    attended++;
    return hipSuccess;
}
}  // namespace paged
}  // namespace mkv

extern "C" {
hipError_t hipMalloc(void** p, size_t n) { return (*p = calloc(n, 1)) ? hipSuccess : hipErrorOutOfMemory; }
hipError_t hipFree(void* p) {
    free(p);
    return hipSuccess;
}
hipError_t hipHostMalloc(void** p, size_t n, unsigned) {
    *p = nullptr;
    if (const hipError_t e = step(hipErrorOutOfMemory)) return e;
    *p = calloc(n, 1);
    return hipSuccess;
}
hipError_t hipHostFree(void* p) {
    free(p);
    return hipSuccess;
}
hipError_t hipMemsetAsync(void* p, int x, size_t n, hipStream_t) {
    memset(p, x, n);
    return hipSuccess;
}
hipError_t hipGetDevice(int* d) {
    *d = 0;
    return hipSuccess;
}
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "device"; }
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) {
    *e = (hipEvent_t)malloc(1);
    return hipSuccess;
}
hipError_t hipEventDestroy(hipEvent_t e) {
    free(e);
    return hipSuccess;
}
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return record_fails ? hipErrorUnknown : step(hipErrorUnknown); }
hipError_t hipEventSynchronize(hipEvent_t) { return step(hipErrorUnknown); }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* st) {
    *st = capturing_now ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
    return hipSuccess;
}

const char* shim_message() { return message; }
void shim_fail_after(long n) {  // the fallible step after the next n fails; -1: none
    left = n;
    steps = 0;
}
long shim_steps() { return steps; }
void shim_fail_records(int on) { record_fails = on; }
int shim_splits_room(int rows, int kv_heads, int part, int more) { return splits_room(rows, kv_heads, part, more); }
int shim_splits_most() { return SPLITS_MOST; }
int shim_copied() { return copied; }
int shim_launches() { return appended + attended; }
int shim_owners(const mpg_t* h, int page) { return h->book.owners[page]; }
int shim_fresh(const mpg_t* h, int seq) { return h->book.fresh[seq]; }
int shim_tokens(const mpg_t* h) { return h->tokens; }
// What a replay finds: runs (seq, token, position, count each) and the lengths of every list of every window behind them.
int shim_runs(const mpg_t* h, int* out) {
    const int n = h->dev[h->runs_at];
    memcpy(out, h->dev + h->runs_at + COUNTS, n * sizeof(Run));
    return n;
}
int shim_work(const mpg_t* h, int window) {  // items and joins
    int n = 0;
    for (int k = 0; k <= KINDS; k++) n += h->dev[h->batch_at + window * h->lists.words + k];
    return n;
}
int shim_device_table(const mpg_t* h, int seq, int at) { return h->dev[(size_t)seq * h->g.most_pages + at]; }
void shim_mark(mpg_t* h, int page, int at, int mark) {  // position `at` of a page: a mark in every plane
    for (int p = 0; p < 2 * h->c.layers; p++)
        *(int*)(h->pool + p * h->g.plane_elems() * 2 + page * h->g.page_elems() * 2 + at * 4) = mark + p;
}
int shim_marked(const mpg_t* h, int page, int at, int mark) {
    for (int p = 0; p < 2 * h->c.layers; p++)
        if (*(int*)(h->pool + p * h->g.plane_elems() * 2 + page * h->g.page_elems() * 2 + at * 4) != mark + p) return 0;
    return 1;
}
}

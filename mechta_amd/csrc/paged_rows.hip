// paged_rows.hip -- what moves rows of the paged cache: uploads of its tables, page copies, the append with rotary
// positions, rotary positions alone, rows out of the pages. All bound by memory or, small, by their launch.
#include <algorithm>

#include "paged_device.h"

namespace mkv {
namespace paged {
namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// ---- uploads: segments of words out of pinned host memory into place, a work-group each, a word a thread: two trips over
// the bus and no more (the lists of 64 sequences: 4.4 us; in segments of 512, 1,024 and 2,048 words 5.7, 8.3 and 13.2) ----
__global__ void __launch_bounds__(256) apply_kernel(int* __restrict__ dev, const unsigned* __restrict__ stage) {
    const Segment s = ((const Segment*)stage)[blockIdx.x];
    if (threadIdx.x < s.words) dev[s.dst + threadIdx.x] = (int)stage[s.src + threadIdx.x];
}

// ---- page copies: every plane (layer, K|V) of a list of pages. Sources and destinations of a launch are different
// pages. A work-group moves 4 KB of one plane's page (the least page of the least shape), 16 bytes a thread, past the L2:
// 256 pages of 1.3 MB in 105 us, 6.4 TB/s (with 2, 4, 8 units in flight a thread 112, 116 and 119, through the L2 122).
constexpr int PAIRS = 256;  // of a launch, in its arguments
struct PairList {
    Pair p[PAIRS];
};
__global__ void __launch_bounds__(256) copy_kernel(char* __restrict__ pool, PairList list, unsigned per_page,
                                                   size_t page_bytes, size_t plane_bytes) {
    const unsigned at = blockIdx.x % per_page, pair = blockIdx.x / per_page;
    char* const p = pool + blockIdx.y * plane_bytes + (size_t)at * 4096 + threadIdx.x * 16;
    const u32x4 x = __builtin_nontemporal_load((const u32x4*)(p + list.p[pair].src * page_bytes));
    __builtin_nontemporal_store(x, (u32x4*)(p + list.p[pair].dst * page_bytes));
}

// ---- rotary positions ----
// cos and sin of a position's pairs: the angle in whole turns in 64 bits, its fraction alone goes on in 32.
__device__ inline float2 turn(const RopeArgs& r, int pos, int pair) {
    const double t = (double)pos * r.turns[pair];
    const float f = 2.f * (float)(t - rint(t));
    float s, c;
    sincospif(f, &s, &c);
    return make_float2(c * r.amplitude, s * r.amplitude);
}
__device__ inline void rotate_pair(float& a, float& b, float2 cs) {
    const float x = a * cs.x - b * cs.y;
    b = b * cs.x + a * cs.y;
    a = x;
}

// One unit of a row's rotation: 8 elements of either side of their pairs (half layout), 8 elements (interleaved), 8
// elements that are copied; without 8-element alignment a pair or an element. Whoever reads an element writes it, so a
// row may be rotated in place. cs(i): the row's pair i. to(d): where element d (and, for units of 8, those behind it) goes.
template <typename T, bool WIDE>
__device__ inline int row_units(int dim, int rot, int layout) {
    if (!WIDE) return rot / 2 + dim - rot;
    return layout == MPG_HALF ? rot / 16 + (dim - rot) / 8 : dim / 8;
}
template <bool STREAM, typename T>
__device__ inline void put8(T* p, Vec8<T> x) {
    if constexpr (STREAM) __builtin_nontemporal_store(x, (Vec8<T>*)p);
    else store8(p, x);
}
template <typename T, bool WIDE, bool STREAM = false, typename Pairs, typename To>
__device__ inline void rotate_unit(const T* __restrict__ x, int u, int rot, int layout, Pairs cs, To to) {
    if constexpr (!WIDE) {
        if (u >= rot / 2) {
            *to(rot / 2 + u) = x[rot / 2 + u];
            return;
        }
        const int i = layout == MPG_HALF ? u : 2 * u, j = layout == MPG_HALF ? u + rot / 2 : 2 * u + 1;
        float a = (float)x[i], b = (float)x[j];
        rotate_pair(a, b, cs(u));
        *to(i) = (T)a;
        *to(j) = (T)b;
    } else if (layout == MPG_HALF && u < rot / 16) {
        Vec8<T> a = load8(x + 8 * u), b = load8(x + rot / 2 + 8 * u);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float p = (float)a[e], q = (float)b[e];
            rotate_pair(p, q, cs(8 * u + e));
            a[e] = (T)p;
            b[e] = (T)q;
        }
        put8<STREAM>(to(8 * u), a);
        put8<STREAM>(to(rot / 2 + 8 * u), b);
    } else {
        const int d = layout == MPG_HALF ? rot / 2 + 8 * u : 8 * u;
        Vec8<T> a = load8(x + d);
        if (d < rot) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                float p = (float)a[e], q = (float)a[e + 1];
                rotate_pair(p, q, cs((d + e) / 2));
                a[e] = (T)p;
                a[e + 1] = (T)q;
            }
        }
        put8<STREAM>(to(d), a);
    }
}

// A thread's places in a grid of rows x heads x units, `by` apart, without a division each.
struct Walk {
    int row, head, unit, rows_by, heads_by, units_by, heads, units;
    __device__ Walk(int at, int by, int heads_, int units_) : heads(heads_), units(units_) {
        split(at, row, head, unit);
        split(by, rows_by, heads_by, units_by);
    }
    __device__ void split(int x, int& r, int& h, int& u) const {
        u = x % units;
        x /= units;
        h = x % heads;
        r = x / heads;
    }
    __device__ void next() {
        unit += units_by;
        head += heads_by;
        row += rows_by;
        if (unit >= units) {
            unit -= units;
            head++;
        }
        if (head >= heads) {
            head -= heads;
            row++;
        }
    }
};

constexpr int ROT_ROWS = 2;  // rows of a work-group: their angles are shared by the heads
// n rows of `heads` heads from x (row and head strides) to out, cs: their pairs
template <typename T, bool WIDE, bool STREAM = false>
__device__ inline void rotate_rows(const RopeArgs& r, int n, int heads, int dim, const T* x, int64_t x_row, int64_t x_head,
                                   T* out, int64_t o_row, int64_t o_head, const float2* cs, int at, int by) {
    const int half = r.dim / 2;
    for (Walk w(at, by, heads, row_units<T, WIDE>(dim, r.dim, r.layout)); w.row < n; w.next()) {
        T* const o = out + w.row * o_row + w.head * o_head;
        const float2* const pairs = cs + w.row * half;
        rotate_unit<T, WIDE, STREAM>(x + w.row * x_row + w.head * x_head, w.unit, r.dim, r.layout,
                                     [&](int i) { return pairs[i]; }, [&](int d) { return o + d; });
    }
}

// Work-group = ROT_ROWS rows; where those are few, blockIdx.y shares out their heads. STREAM: outputs that the L2s cannot
// hold anyway are stored past them (8,192 rows of 32 heads of 128 in bf16, 134 MB moved: 28.8 -> 21.8 us).
template <typename T, bool WIDE, bool STREAM>
__global__ void __launch_bounds__(256) rotate_kernel(RopeArgs r, int rows, int heads, int dim, const T* x, int64_t x_row,
                                                     int64_t x_head, const int* __restrict__ pos, T* out, int64_t o_row,
                                                     int64_t o_head) {
    extern __shared__ float2 cs[];  // [ROT_ROWS][r.dim / 2]
    const int row0 = blockIdx.x * ROT_ROWS, n = min(ROT_ROWS, rows - row0), half = r.dim / 2;
    for (Walk w(threadIdx.x, 256, 1, half); w.row < n; w.next()) cs[w.row * half + w.unit] = turn(r, pos[row0 + w.row], w.unit);
    __syncthreads();
    rotate_rows<T, WIDE, STREAM>(r, n, heads, dim, x + row0 * x_row, x_row, x_head, out + row0 * o_row, o_row, o_head, cs,
                         threadIdx.x + 256 * blockIdx.y, 256 * gridDim.y);
}

// ---- append ----
// A run is new tokens inside one 32-position block of a page. The first work-groups take a run's K and V of a head each,
// those behind them the query heads of 2 tokens each; neighbours have neighbouring rows. K rows go into the pages as they
// are rotated, neighbouring lanes on neighbouring positions. A V block that is all new is turned in registers (8 positions
// of 8 dims a thread) and written in 16-byte pieces, others element by element. Bound by memory: 4,096 + 2,500 + 1,031 +
// 565 tokens of 32 + 2 x 4 heads of 128 move 168 MB in 32.6 us, 5.2 TB/s (query heads of 4 tokens a work-group 35.4, of 1 and
// 8 36.9; K and V of all heads in one work-group behind the query heads 44).
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) append_kernel(const Run* __restrict__ runs, const int* __restrict__ nruns,
                                                     const int* __restrict__ table, int most_pages, int page, int dim,
                                                     int kv_heads, int q_heads, T* __restrict__ kpool, T* __restrict__ vpool,
                                                     int rows, const T* __restrict__ k, int64_t k_tok, int64_t k_head,
                                                     const T* __restrict__ v, int64_t v_tok, int64_t v_head, const T* q,
                                                     int64_t q_tok, int64_t q_head, T* q_out, RopeArgs r,
                                                     const int* __restrict__ shift) {
    extern __shared__ float2 cs[];  // [ROT_ROWS][r.dim / 2]
    const int half = r.dim / 2, tid = threadIdx.x, count = *uniform(nruns);
    const int q_parts = q ? (uniform(nruns)[1] + ROT_ROWS - 1) / ROT_ROWS : 0;  // by the longest run
    const int kv_items = count * kv_heads, items = kv_items + count * q_parts;
    for (int i = blockIdx.x; i < items; i += gridDim.x) {
        const bool is_q = i >= kv_items;
        const int x = is_q ? i - kv_items : i, per = is_q ? q_parts : kv_heads, of = x % per;
        const Uniform<int> ri = uniform((const int*)(runs + x / per));
        Run run{ri[0], ri[1], ri[2], ri[3]};
        run.count = min(run.count, rows - run.tok);
        const int pos = run.pos + (shift ? uniform(shift)[run.seq] : 0);  // what eviction has taken lies in front
        if (is_q) {
            const int t0 = of * ROT_ROWS, n = min(ROT_ROWS, run.count - t0);
            if (n <= 0) continue;
            __syncthreads();  // the angles before have been read
            for (Walk w(tid, 256, 1, half); w.row < n; w.next())
                cs[w.row * half + w.unit] = turn(r, pos + t0 + w.row, w.unit);
            __syncthreads();
            const int64_t tok = run.tok + t0;
            rotate_rows<T, WIDE>(r, n, q_heads, dim, q + tok * q_tok, q_tok, q_head, q_out + tok * q_heads * dim,
                                 (int64_t)q_heads * dim, dim, cs, tid, 256);
            continue;
        }
        if (run.count <= 0) continue;
        const size_t p = uniform(table)[(size_t)run.seq * most_pages + run.pos / page];
        const int in = run.pos % page, at = in % KEYS, chunks = dim / 8, head = of;
        const size_t base = (p * kv_heads + head) * page * dim + (size_t)(in / KEYS) * KEYS * dim;  // of the 32-position block
        const T* const ks = k + run.tok * k_tok + head * k_head;
        // units of all rows, row by row; neighbours in the pages are of neighbouring rows
        for (Walk w(tid, 256, row_units<T, WIDE>(dim, r.dim, r.layout), run.count); w.row < 1; w.next()) {
            const int t = w.unit, b = at + t;
            T* const o = kpool + base + b / 16 * 16 * dim + b % 16 * 8;
            rotate_unit<T, WIDE>(ks + t * k_tok, w.head, r.dim, r.layout, [&](int i) { return turn(r, pos + t, i); },
                                 [&](int d) { return o + d / 8 * 128 + d % 8; });
        }
        const T* const vs = v + run.tok * v_tok + head * v_head;
        T* const vb = vpool + base;
        if (run.count == KEYS) {
            for (int j = tid; j < dim / 2; j += 256) {  // (group of 8 positions, 8 dims)
                const int g = j / chunks, d = j % chunks * 8;
                Vec8<T> x[8];
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = load8(vs + (16 * (e / 4) + 4 * g + e % 4) * v_tok + d);
#pragma unroll
                for (int c = 0; c < 8; c++)
                    store8(vb + (g * dim + d + c) * 8,
                           Vec8<T>{x[0][c], x[1][c], x[2][c], x[3][c], x[4][c], x[5][c], x[6][c], x[7][c]});
            }
        } else {
            for (Walk w(tid, 256, 1, chunks); w.row < run.count; w.next()) {
                const int d = w.unit * 8, b = at + w.row;
                const Vec8<T> x = load8(vs + w.row * v_tok + d);
                T* const o = vb + (b % 16 / 4 * dim + d) * 8 + b / 16 * 4 + b % 4;
#pragma unroll
                for (int c = 0; c < 8; c++) o[c * 8] = x[c];
            }
        }
    }
}

// ---- rows out of the pages: 8 elements a thread ----
template <typename T>
__global__ void __launch_bounds__(256) read_kernel(const T* __restrict__ pool, const int* __restrict__ table, int page,
                                                   int kv_heads, int dim, int is_v, int p0, int p1, T* __restrict__ dst) {
    const size_t per = (size_t)kv_heads * dim / 8, i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= per * (p1 - p0)) return;
    const int pos = p0 + (int)(i / per), head = (int)(i % per) / (dim / 8), d = (int)(i % (dim / 8)) * 8, in = pos % page;
    const T* const b = pool + ((size_t)table[pos / page] * kv_heads + head) * page * dim;
    Vec8<T> x;
    if (!is_v) {
        x = load8(b + (size_t)(in / 16) * 16 * dim + d * 16 + in % 16 * 8);
    } else {
        const T* const s = b + (size_t)(in / KEYS) * KEYS * dim + (in % 16 / 4 * dim + d) * 8 + in % KEYS / 16 * 4 + in % 4;
#pragma unroll
        for (int c = 0; c < 8; c++) x[c] = s[c * 8];
    }
    store8(dst + i * 8, x);
}

template <typename T>
hipError_t append_as(const Geometry& g, char* pool, int layer, const int* table, const Run* runs, const int* nruns, int grid,
                     int most, int longest, int rows, const Rows& k, const Rows& v, const Rows& q, void* q_out,
                     const RopeArgs* rope, hipStream_t s) {
    RopeArgs none{};
    none.layout = MPG_HALF;
    const RopeArgs& r = rope ? *rope : none;
    T* const kp = (T*)pool + (size_t)layer * 2 * g.plane_elems();
    const size_t lds = (size_t)ROT_ROWS * (r.dim / 2) * sizeof(float2);
    const auto kernel = r.dim % 16 ? append_kernel<T, false> : append_kernel<T, true>;
    const size_t items = (size_t)most * (g.kv_heads + (q.p ? (longest + ROT_ROWS - 1) / ROT_ROWS : 0));
    if (!grid) grid = (int)std::min<size_t>(items, MOST_GRID);
    kernel<<<dim3(grid), dim3(256), lds, s>>>(
        runs, nruns, table, g.most_pages, g.page, g.head_dim, g.kv_heads, g.q_heads, kp, kp + g.plane_elems(), rows,
        (const T*)k.p, k.tok, k.head, (const T*)v.p, v.tok, v.head, (const T*)q.p, q.tok, q.head, (T*)q_out, r, g.shift);
    return hipGetLastError();
}

template <typename T>
hipError_t rotate_as(const RopeArgs& r, int rows, int heads, int dim, const Rows& x, const int* pos, const Rows& out,
                     hipStream_t s) {
    const bool wide = r.dim % 16 == 0 && dim % 8 == 0 && x.tok % 8 == 0 && x.head % 8 == 0 && out.tok % 8 == 0 &&
                      out.head % 8 == 0 && (uintptr_t)x.p % 16 == 0 && (uintptr_t)out.p % 16 == 0;
    const size_t lds = (size_t)ROT_ROWS * (r.dim / 2) * sizeof(float2);
    constexpr size_t L2 = 32 << 20;  // of the eight dies together
    const bool stream = (size_t)rows * heads * dim * sizeof(T) > L2;
    const auto kernel = !wide    ? rotate_kernel<T, false, false>
                        : stream ? rotate_kernel<T, true, true>
                                 : rotate_kernel<T, true, false>;
    const int groups = (rows + ROT_ROWS - 1) / ROT_ROWS, n = rows < ROT_ROWS ? rows : ROT_ROWS;
    // few rows of many heads: heads shared out, a unit or two a thread
    const int y = groups >= 256 ? 1 : std::max(1, std::min(256 / groups, n * heads * (dim / 16) / 512));
    kernel<<<dim3(groups, y), dim3(256), lds, s>>>(r, rows, heads, dim, (const T*)x.p, x.tok, x.head,
                                                                         pos, (T*)out.p, out.tok, out.head);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_apply(int* dev, const unsigned* stage, int segments, hipStream_t s) {
    apply_kernel<<<dim3(segments), dim3(256), 0, s>>>(dev, stage);
    return hipGetLastError();
}

hipError_t launch_copies(const Geometry& g, char* pool, const Pair* pairs, int n, hipStream_t s) {
    const size_t page = g.page_elems() * 2;
    const unsigned per_page = (unsigned)(page / 4096);
    for (int i = 0; i < n; i += PAIRS) {
        PairList list;
        const int m = std::min(PAIRS, n - i);
        std::copy(pairs + i, pairs + i + m, list.p);
        std::fill(list.p + m, list.p + PAIRS, Pair{0, 0});
        copy_kernel<<<dim3(m * per_page, 2 * g.layers), dim3(256), 0, s>>>(pool, list, per_page, page, g.plane_elems() * 2);
        if (const hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
}

hipError_t launch_append(const Geometry& g, char* pool, int layer, const int* table, const Run* runs, const int* nruns,
                         int grid, int most, int longest, int rows, const Rows& k, const Rows& v, const Rows& q, void* q_out,
                         const RopeArgs* rope, hipStream_t s) {
    const auto as = g.fmt == MKV_F16 ? append_as<_Float16> : append_as<__bf16>;
    return as(g, pool, layer, table, runs, nruns, grid, most, longest, rows, k, v, q, q_out, rope, s);
}

// A launch takes less than 2^32 threads: what needs more goes in several.
hipError_t launch_read(const Geometry& g, const char* pool, int layer, int which, const int* table, int p0, int p1, void* dst,
                       hipStream_t s) {
    const size_t per = (size_t)g.kv_heads * g.head_dim / 8;  // threads of a position
    const char* const base = pool + ((size_t)layer * 2 + which) * g.plane_elems() * 2;
    const int most = (int)std::min<size_t>((1ull << 31) / per, MPG_CTX_MAX);
    for (int p = p0; p < p1; p += most) {
        const int e = std::min(p + most, p1);
        // both types are 16 bits that are only moved
        read_kernel<_Float16><<<dim3((unsigned)((per * (e - p) + 255) / 256)), dim3(256), 0, s>>>(
            (const _Float16*)base, table, g.page, g.kv_heads, g.head_dim, which == MKV_V, p, e,
            (_Float16*)dst + (size_t)(p - p0) * per * 8);
        if (const hipError_t err = hipGetLastError()) return err;
    }
    return hipSuccess;
}

hipError_t launch_rotate(const RopeArgs& r, int fmt, int rows, int heads, int dim, const Rows& x, const int* pos,
                         const Rows& out, hipStream_t s) {
    constexpr int MOST = ROT_ROWS << 23;  // 2^31 threads
    const int bytes = fmt == MKV_F32 ? 4 : 2;
    for (int64_t i = 0; i < rows; i += MOST) {
        const int n = (int)std::min<int64_t>(MOST, rows - i);
        const Rows xi{(const char*)x.p + i * x.tok * bytes, x.tok, x.head};
        const Rows oi{(const char*)out.p + i * out.tok * bytes, out.tok, out.head};
        const hipError_t e = fmt == MKV_F16   ? rotate_as<_Float16>(r, n, heads, dim, xi, pos + i, oi, s)
                             : fmt == MKV_F32 ? rotate_as<float>(r, n, heads, dim, xi, pos + i, oi, s)
                                              : rotate_as<__bf16>(r, n, heads, dim, xi, pos + i, oi, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace paged
}  // namespace mkv

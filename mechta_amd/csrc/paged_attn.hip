// paged_attn.hip -- attention of a batch's new tokens over their sequences' pages.
//
// Row r of a sequence's query rows is (token r / group, query head head * group + r % group): the query heads of a kv head
// and the tokens of a chunk share the keys they read. A work-group takes a tile of rows and a range of keys (Item); where
// a tile's keys are split, join_kernel puts the splits together.
#include "paged_device.h"

namespace mkv {
namespace paged {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr float NEG_INF = -__builtin_huge_valf();

__device__ inline f32x4 mfma16(Vec8<_Float16> a, Vec8<_Float16> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ inline f32x4 mfma16(Vec8<__bf16> a, Vec8<__bf16> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The weights 2^(s - ref) of a row are rounded to the cache's type for the matrix units (half a step: 2^-11 of a weight
// in f16, 2^-8 in bf16; the sum takes them unrounded). ref is the largest score of the first tile, and moves up, with the
// sums rescaled, only where a score exceeds it by more than LAZY. f16 has no room below 2^-14: its weights are taken
// 2^LIFT times as large, so that a score 24 below the largest still keeps all its bits, and stay below
// 2^(LIFT + LAZY) = 2^15.
template <typename T>
struct Weights;
template <>
struct Weights<_Float16> {
    static constexpr float LIFT = 10.f, LAZY = 5.f;
    static constexpr unsigned INF2 = 0x7C007C00u;
};
template <>
struct Weights<__bf16> {
    static constexpr float LIFT = 0.f, LAZY = 8.f;
    static constexpr unsigned INF2 = 0x7F807F80u;
};

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

struct Args {
    const int* table;
    int most_pages, page, page_shift;
    int q_heads, kv_heads, group, window, rows;
    const void *kpool, *vpool;  // the layer's pages
    const void* q;
    int64_t q_tok, q_head;
    const void* gate;
    int64_t g_tok, g_head;
    const float* sinks;
    void* out;
    float scale2;  // scale * log2 e
    float *pm, *pl, *pacc;
};

// Four dims of a finished row: acc / l with the sink in the sum, gated, rounded once.
template <typename T, int D>
__device__ inline void finish(const Args& a, int tok, int head, int d, f32x4 acc, float m, float l) {
    if (a.sinks) {  // m is the reference of acc and l, in log2 units
        const float s = a.sinks[head] * LOG2E, top = fmaxf(m, s);
        const float f = m == NEG_INF ? 0.f : exp2_fast(m - top);
        acc *= f;
        l = l * f + exp2_fast(s - top);
    }
    acc *= 1.f / l;
    if (a.gate) {
        const Vec4<T> g = *(const Vec4<T>*)((const T*)a.gate + tok * a.g_tok + head * a.g_head + d);
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] *= 1.f / (1.f + exp2_fast(-LOG2E * (float)g[i]));
    }
    Vec4<T> o;
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = (T)acc[i];
    *(Vec4<T>*)((T*)a.out + ((size_t)tok * a.q_heads + head) * D + d) = o;
}

// Whether any of a wave's V operands holds an infinity or NaN.
template <typename T, int N>
__device__ inline bool odd_values(const Vec8<T> (&v)[N]) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 top = {0, 0};
#pragma unroll
    for (int i = 0; i < N; i++) {
        const u32x4 x = __builtin_bit_cast(u32x4, v[i]);
#pragma unroll
        for (int j = 0; j < 4; j++) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, x[j] & 0x7FFF7FFFu));
    }
    constexpr unsigned short inf = Weights<T>::INF2 & 0xFFFF;
    return __any(top.x >= inf || top.y >= inf);
}

// P.V where a tile's V holds infinities or NaN that some row does not see (0 x NaN would reach it): the finite part as
// ever, and per row how many +inf, -inf and NaN of each dim it sees, counted by the matrix units (a tile has 32
// positions: at most 32 of each), which then decide the sum.
template <typename T, int NRT>
__device__ inline void odd_product(Vec8<T> v, const Vec8<T> (&p)[NRT], const Vec8<T> (&seen)[NRT],
                                                     f32x4 (&o)[NRT]) {
    Vec8<T> fine, odd;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float x = (float)v[e];
        const bool nan = x != x, inf = __builtin_isinf(x);
        fine[e] = nan || inf ? (T)0.f : v[e];
        odd[e] = (T)(nan ? 16384.f : inf ? (x > 0 ? 1.f : 128.f) : 0.f);
    }
#pragma unroll
    for (int t = 0; t < NRT; t++) {
        o[t] = mfma16(fine, p[t], o[t]);
        const f32x4 c = mfma16(odd, seen[t], f32x4{});
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int n = (int)c[i];
            if (n & 127) o[t][i] += -NEG_INF;
            if (n >> 7 & 127) o[t][i] += NEG_INF;
            if (n >> 14) o[t][i] = __builtin_nanf("");
        }
    }
}

// ---- few rows: NRT x 16 query rows against keys streamed once ----
// 4 waves, each with every fourth 32-position block of the range, its K and V straight from memory into matrix operands
// (16x16x32; the pages' layout is the operands'). Per block and wave:
//   S^T[32 keys][rows] = K . Q^T        lane (r, g): row r, keys 4g + i and 16 + 4g + i
//   softmax of the rows in registers    (the four lane groups of a row hold 8 keys each)
//   O^T[D][rows] += V^T . P^T           P^T straight from the scores' registers; lane (r, g): row r, dims 4g + i of each 16
// The next block's K is on its way while the softmax runs, its V while the next scores are computed. The waves' states
// meet in LDS at the end.
template <typename T, int D, int NRT>
__global__ void __launch_bounds__(256, NRT* D <= 256 ? 2 : 1) few_rows(Args a, const Item* __restrict__ items,
                                                                       const int* __restrict__ nitems) {
    constexpr int NS = D / 32, NV = D / 16;
    __shared__ __attribute__((aligned(16))) float so[4][16][D + 4];
    __shared__ float sm[4][16], sl[4][16];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int count = *nitems;
    for (int n = blockIdx.x; n < count; n += gridDim.x) {
        const Item it = items[n];
        const T* const kp = (const T*)a.kpool + (size_t)it.head * a.page * D;
        const T* const vp = (const T*)a.vpool + (size_t)it.head * a.page * D;
        const size_t page_elems = (size_t)a.kv_heads * a.page * D;
        const int* const table = a.table + (size_t)it.seq * a.most_pages;
        const int last_row = min(it.row0 + 16 * NRT, it.rows) - 1;
        // blocks with every key in [all_lo, all_hi] are seen by all rows whole
        const int all_hi = it.pos0 + it.row0 / a.group;
        const int all_lo = a.window ? it.pos0 + last_row / a.group - a.window + 1 : 0;

        Vec8<T> q[NRT][NS];
        int lo[NRT], hi[NRT];  // keys the lane's row sees
#pragma unroll
        for (int t = 0; t < NRT; t++) {
            const int row = it.row0 + 16 * t + r, tok = row / a.group, head = it.head * a.group + row % a.group;
            const bool is = row <= last_row && it.tok0 + tok < a.rows;
            hi[t] = is ? it.pos0 + tok : -1;
            lo[t] = a.window ? it.pos0 + tok - a.window + 1 : 0;
            const T* const src = (const T*)a.q + (int64_t)(it.tok0 + tok) * a.q_tok + head * a.q_head + 8 * g;
#pragma unroll
            for (int s = 0; s < NS; s++) q[t][s] = is ? load8(src + 32 * s) : Vec8<T>{};
        }
        f32x4 o[NRT][NV];
        float m[NRT], l[NRT];  // the reference of the row's weights (log2 units), the lane's share of their sum
#pragma unroll
        for (int t = 0; t < NRT; t++) {
            m[t] = NEG_INF;
            l[t] = 0.f;
#pragma unroll
            for (int i = 0; i < NV; i++) o[t][i] = f32x4{};
        }
        const int blocks = (it.k1 - it.k0 + KEYS - 1) / KEYS;
        auto key_of = [&](int j) { return it.k0 + KEYS * j; };
        auto page_of = [&](int j) { return table[key_of(min(j, blocks - 1)) >> a.page_shift]; };
        auto offset = [&](int j, int page) {  // of block j, its page known
            return page * page_elems + (size_t)(key_of(j) & (a.page - 1)) * D;
        };
        Vec8<T> kf[2][NS], vf[NV];
        auto load_k = [&](size_t off) {
#pragma unroll
            for (int s = 0; s < NS; s++)
#pragma unroll
                for (int b = 0; b < 2; b++) kf[b][s] = load8(kp + off + b * 16 * D + (4 * s + g) * 128 + r * 8);
        };
        auto load_v = [&](size_t off) {
#pragma unroll
            for (int i = 0; i < NV; i++) vf[i] = load8(vp + off + (g * D + 16 * i + r) * 8);
        };
        if (w < blocks) {
            size_t off = offset(w, page_of(w));
            load_k(off);
            load_v(off);
            int page = page_of(w + 4);
            for (int j = w; j < blocks; j += 4) {
                const int jn = j + 4 < blocks ? j + 4 : j;
                const size_t next = j + 4 < blocks ? offset(jn, page) : off;
                page = page_of(j + 8);
                f32x4 s[NRT][2];
#pragma unroll
                for (int t = 0; t < NRT; t++) s[t][0] = s[t][1] = f32x4{};
#pragma unroll
                for (int i = 0; i < NS; i++)
#pragma unroll
                    for (int t = 0; t < NRT; t++)
#pragma unroll
                        for (int b = 0; b < 2; b++) s[t][b] = mfma16(kf[b][i], q[t][i], s[t][b]);
                load_k(next);
                const int k0 = key_of(j);
                const bool edge = k0 + KEYS - 1 > all_hi || k0 < all_lo;
                Vec8<T> p[NRT];
#pragma unroll
                for (int t = 0; t < NRT; t++) {
                    if (edge) {
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const int key = k0 + e / 4 * 16 + 4 * g + e % 4;
                            if (key > hi[t] || key < lo[t]) s[t][e / 4][e % 4] = NEG_INF;
                        }
                    }
                    float top = fmaxf(fmaxf(fmaxf(s[t][0][0], s[t][0][1]), fmaxf(s[t][0][2], s[t][0][3])),
                                      fmaxf(fmaxf(s[t][1][0], s[t][1][1]), fmaxf(s[t][1][2], s[t][1][3])));
                    top = fmaxf(top, __shfl_xor(top, 16));
                    top = fmaxf(top, __shfl_xor(top, 32)) * a.scale2 - Weights<T>::LIFT;
                    const bool move = m[t] != NEG_INF && top > m[t] + Weights<T>::LAZY;
                    if (__any(move)) {
                        const float f = move ? exp2_fast(m[t] - top) : 1.f;
                        l[t] *= f;
#pragma unroll
                        for (int i = 0; i < NV; i++) o[t][i] *= f;
                    }
                    if (move || m[t] == NEG_INF) m[t] = top;
                    const float ref = m[t] == NEG_INF ? 0.f : m[t];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float x = exp2_fast(__builtin_fmaf(s[t][e / 4][e % 4], a.scale2, -ref));
                        l[t] += x;
                        p[t][e] = (T)x;
                    }
                }
                if (edge && odd_values(vf)) {
                    Vec8<T> seen[NRT];
#pragma unroll
                    for (int t = 0; t < NRT; t++)
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const int key = k0 + e / 4 * 16 + 4 * g + e % 4;
                            seen[t][e] = (T)(key > hi[t] || key < lo[t] ? 0.f : 1.f);
                        }
#pragma unroll
                    for (int i = 0; i < NV; i++) {
                        f32x4 x[NRT];
#pragma unroll
                        for (int t = 0; t < NRT; t++) x[t] = o[t][i];
                        odd_product<T, NRT>(vf[i], p, seen, x);
#pragma unroll
                        for (int t = 0; t < NRT; t++) o[t][i] = x[t];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < NV; i++)
#pragma unroll
                        for (int t = 0; t < NRT; t++) o[t][i] = mfma16(vf[i], p[t], o[t][i]);
                }
                load_v(next);
                off = next;
            }
        }
        // the four waves' states of 16 rows at a time
#pragma unroll
        for (int t = 0; t < NRT; t++) {
            float sum = l[t] + __shfl_xor(l[t], 16);
            sum += __shfl_xor(sum, 32);
            __syncthreads();  // the states before have been read
            if (g == 0) {
                sm[w][r] = m[t];
                sl[w][r] = sum;
            }
#pragma unroll
            for (int i = 0; i < NV; i++) *(f32x4*)&so[w][r][16 * i + 4 * g] = o[t][i];
            __syncthreads();
            const int rr = threadIdx.x >> 4, row = it.row0 + 16 * t + rr, tok = it.tok0 + row / a.group;
            if (row > last_row || tok >= a.rows) continue;
            const float top = fmaxf(fmaxf(sm[0][rr], sm[1][rr]), fmaxf(sm[2][rr], sm[3][rr]));
            float f[4], total = 0.f;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                f[x] = sm[x][rr] == NEG_INF ? 0.f : exp2_fast(sm[x][rr] - top);
                total += f[x] * sl[x][rr];
            }
#pragma unroll
            for (int c = 0; c < D / 64; c++) {
                const int d = ((int)(threadIdx.x & 15) + 16 * c) * 4;
                f32x4 acc = f32x4{};
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const f32x4 y = *(const f32x4*)&so[x][rr][d];
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[i] += f[x] == 0.f ? 0.f : f[x] * y[i];
                }
                if (it.part < 0) {
                    finish<T, D>(a, tok, it.head * a.group + row % a.group, d, acc, top, total);
                } else {
                    const size_t at = it.part + 16 * t + rr;
                    *(f32x4*)(a.pacc + at * D + d) = acc;
                    if (d == 0) {
                        a.pm[at] = top;
                        a.pl[at] = total;
                    }
                }
            }
        }
    }
}

// ---- splits of a tile's rows put together: D / 4 lanes a row, four dims each ----
template <typename T, int D>
__global__ void __launch_bounds__(256) join_kernel(Args a, const Join* __restrict__ joins, const int* __restrict__ njoins) {
    constexpr int LANES = D / 4, ROWS = 256 / LANES;
    const int count = *njoins;
    for (int n = blockIdx.x; n < count; n += gridDim.x) {
        const Join j = joins[n];
        for (int r = blockIdx.y * ROWS + threadIdx.x / LANES; r < j.count; r += gridDim.y * ROWS) {
            const int row = j.row0 + r, tok = j.tok0 + row / a.group, d = threadIdx.x % LANES * 4;
            if (tok >= a.rows) continue;
            const size_t first = j.part + r;
            float top = NEG_INF;
            for (int s = 0; s < j.splits; s++) top = fmaxf(top, a.pm[first + (size_t)s * j.count]);
            f32x4 acc = f32x4{};
            float total = 0.f;
            for (int s = 0; s < j.splits; s++) {
                const size_t at = first + (size_t)s * j.count;
                const float m = a.pm[at], f = m == NEG_INF ? 0.f : exp2_fast(m - top);
                const f32x4 x = *(const f32x4*)(a.pacc + at * D + d);
#pragma unroll
                for (int i = 0; i < 4; i++) acc[i] += f == 0.f ? 0.f : f * x[i];
                total += f * a.pl[at];
            }
            finish<T, D>(a, tok, j.head * a.group + row % a.group, d, acc, top, total);
        }
    }
}

template <typename T, int D>
hipError_t attend_as(const Geometry& g, const AttendArgs& x, const int* batch, const Lists& l, const int* grid, int join_grid,
                     hipStream_t s) {
    Args a;
    a.table = x.table;
    a.most_pages = g.most_pages;
    a.page = g.page;
    a.page_shift = __builtin_ctz(g.page);
    a.q_heads = g.q_heads;
    a.kv_heads = g.kv_heads;
    a.group = g.q_heads / g.kv_heads;
    a.window = x.window;
    a.rows = x.rows;
    a.kpool = x.pool + (size_t)x.layer * 2 * g.plane_elems() * 2;
    a.vpool = x.pool + ((size_t)x.layer * 2 + 1) * g.plane_elems() * 2;
    a.q = x.q.p;
    a.q_tok = x.q.tok;
    a.q_head = x.q.head;
    a.gate = x.gate.p;
    a.g_tok = x.gate.tok;
    a.g_head = x.gate.head;
    a.sinks = x.sinks;
    a.out = x.out;
    a.scale2 = x.scale * LOG2E;
    a.pm = x.pm;
    a.pl = x.pl;
    a.pacc = x.pacc;
    hipError_t e = hipSuccess;
    if (grid[FEW]) {
        few_rows<T, D, 1><<<dim3(grid[FEW]), dim3(256), 0, s>>>(a, (const Item*)(batch + l.items[FEW]), batch + FEW);
        e = hipGetLastError();
    }
    if (grid[SOME] && e == hipSuccess) {
        few_rows<T, D, 2><<<dim3(grid[SOME]), dim3(256), 0, s>>>(a, (const Item*)(batch + l.items[SOME]), batch + SOME);
        e = hipGetLastError();
    }
    if (join_grid && e == hipSuccess) {
        constexpr int rows = 256 / (D / 4);
        join_kernel<T, D><<<dim3(join_grid, 32 / rows), dim3(256), 0, s>>>(a, (const Join*)(batch + l.joins), batch + KINDS);
        e = hipGetLastError();
    }
    return e;
}

template <typename T>
hipError_t attend_dim(const Geometry& g, const AttendArgs& x, const int* batch, const Lists& l, const int* grid, int join_grid,
                      hipStream_t s) {
    return g.head_dim == 64    ? attend_as<T, 64>(g, x, batch, l, grid, join_grid, s)
           : g.head_dim == 128 ? attend_as<T, 128>(g, x, batch, l, grid, join_grid, s)
                               : attend_as<T, 256>(g, x, batch, l, grid, join_grid, s);
}

}  // namespace

hipError_t launch_attend(const Geometry& g, const AttendArgs& a, const int* batch, const Lists& l, const int* grid,
                         int join_grid, hipStream_t s) {
    return g.fmt == MKV_F16 ? attend_dim<_Float16>(g, a, batch, l, grid, join_grid, s)
                            : attend_dim<__bf16>(g, a, batch, l, grid, join_grid, s);
}

}  // namespace paged
}  // namespace mkv

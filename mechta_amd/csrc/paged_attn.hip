// paged_attn.hip -- attention of a batch's new tokens over their sequences' pages.
//
// Row r of a sequence's query rows is (token r / group, query head head * group + r % group): the query heads of a kv head
// and the tokens of a chunk share the keys they read. A work-group takes a tile of rows and a range of keys (Item); where
// a tile's keys are split, join_kernel puts the splits together.
#include <algorithm>
#include <type_traits>

#include "mkv_device.h"
#include "paged_device.h"

namespace mkv {
namespace paged {
namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
// lambdas that hold a kernel's registers by reference: one that is not inlined puts them into memory
#define INLINE __attribute__((always_inline))

__device__ inline f32x4 mfma16(Vec8<_Float16> a, Vec8<_Float16> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ inline f32x4 mfma16(Vec8<__bf16> a, Vec8<__bf16> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ inline f32x16 mfma32(Vec8<_Float16> a, Vec8<_Float16> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ inline f32x16 mfma32(Vec8<__bf16> a, Vec8<__bf16> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// The weights 2^(s - ref) of a row are rounded to the cache's type for the matrix units (half a step: 2^-11 of a weight
// in f16, 2^-8 in bf16); their sum, in f32, is of the rounded ones, so that a row's weights still add up to one. ref is the largest score of the first tile, and moves up, with the
// sums rescaled, only where a score exceeds it by more than LAZY. f16 has no room below 2^-14: its weights are taken
// 2^LIFT times as large, so that a score 24 below the largest still keeps all its bits, and stay below
// 2^(LIFT + LAZY) = 2^15.
template <typename T>
struct Weights;
template <>
struct Weights<_Float16> {
    static constexpr float LIFT = 10.f, LAZY = 5.f;
    static constexpr unsigned short INF = 0x7C00;
};
template <>
struct Weights<__bf16> {
    static constexpr float LIFT = 0.f, LAZY = 8.f;
    static constexpr unsigned short INF = 0x7F80;
};

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
    const Place* order;  // tokens of tiles that several sequences share
};

__device__ inline Item load_item(const Item* p) {
    const Uniform<int> x = uniform((const int*)p);
    return Item{x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7], x[8], 0, x[10], 0};
}
// Token and position of a tile's row (last_row: the tile's last; rows behind it are nobody's).
__device__ inline Place place_of(const Args& a, const Item& it, int row, int last_row) {
    if (it.top) return a.order[it.tok0 + min(row, last_row) / a.group];
    return Place{it.tok0 + row / a.group, it.pos0 + row / a.group};
}
// The position of the furthest of rows up to `row`.
__device__ inline int furthest(const Args& a, const Item& it, int row) {
    return it.top ? it.top - 1 : it.pos0 + row / a.group;
}

// The factor of a finished row's sums: 1 / l, with the sink (m: the reference of acc and l, in log2 units).
__device__ inline float row_factor(const Args& a, int head, float m, float l) {
    if (!a.sinks) return __builtin_amdgcn_rcpf(l);  // 2^-23: far below the output's rounding
    const float s = a.sinks[head] * LOG2E, top = fmaxf(m, s), f = m == NEG_INF ? 0.f : fast_exp2(m - top);
    return f * __builtin_amdgcn_rcpf(l * f + fast_exp2(s - top));
}
// N dims of a finished row: gated, rounded once.
template <typename T, int D, int N>
__device__ inline void store_out(const Args& a, int tok, int head, int d, const float (&x)[N]) {
    typedef T vec __attribute__((ext_vector_type(N)));
    vec o;
    if (a.gate) {
        const vec g = *(const vec*)((const T*)a.gate + tok * a.g_tok + head * a.g_head + d);
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = (T)(x[i] * __builtin_amdgcn_rcpf(1.f + fast_exp2(-LOG2E * (float)g[i])));
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = (T)x[i];
    }
    *(vec*)((T*)a.out + ((size_t)tok * a.q_heads + head) * D + d) = o;
}

// The maximum, or sum, over lanes l and l ^ 16, in every lane: two registers that both hold x exchange their odd and even
// rows of 16 lanes.
__device__ inline float max_xor16(float x) {
    float y;
    asm volatile("v_mov_b32 %0, %1" : "=v"(y) : "v"(x));
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return vmax(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float add_xor16(float x) {
    float y;
    asm volatile("v_mov_b32 %0, %1" : "=v"(y) : "v"(x));
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ inline float add_pair(_Float16 a, _Float16 b, float c) {
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(pair{a, b}, pair{(_Float16)1.f, (_Float16)1.f}, c, false);
}
__device__ inline float add_pair(__bf16 a, __bf16 b, float c) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(pair{a, b}, pair{(__bf16)1.f, (__bf16)1.f}, c, false);
}

// Infinities and NaN of V in positions that some of a wave's rows do not see: 0 x NaN would reach those rows through the
// products. Only tiles that cross a row's bounds can hold such (edge tiles); there the operands are looked through, and
// what is not finite is taken as zero. The rows that see it get it after the loop, by plain additions, value by value
// (add_odd): slow, and rare.
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
    return __any(top.x >= Weights<T>::INF || top.y >= Weights<T>::INF);
}
template <typename T>
__device__ inline Vec8<T> finite(Vec8<T> v) {
    typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
    u16x8 x = __builtin_bit_cast(u16x8, v);
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = (x[e] & 0x7FFF) >= Weights<T>::INF ? 0 : x[e];
    return __builtin_bit_cast(Vec8<T>, x);
}
// v: element 0 of dim 0 of a 32-position block of V; position x of it, dims d .. d + 3, added to o where not finite
template <typename T, int D>
__device__ inline f32x4 add_odd(const T* v, int x, int d, bool seen, f32x4 o) {
    const unsigned short* const p = (const unsigned short*)v + (size_t)((x % 16 / 4) * D + d) * 8 + x / 16 * 4 + x % 4;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (seen && (p[8 * i] & 0x7FFF) >= Weights<T>::INF) o[i] += (float)__builtin_bit_cast(T, p[8 * i]);
    __builtin_amdgcn_sched_barrier(0);  // a few registers at a time
    return o;
}

// ---- few rows: NRT x 16 query rows against keys streamed once ----
// 4 waves, each with every fourth 32-position block of the range, its K and V straight from memory into matrix operands
// (16x16x32; the pages' layout is the operands'). Per block and wave:
//   S^T[32 keys][rows] = K . Q^T        lane (r, g): row r, keys 4g + i and 16 + 4g + i
//   softmax of the rows in registers    (the four lane groups of a row hold 8 keys each)
//   O^T[D][rows] += V^T . P^T           P^T straight from the scores' registers; lane (r, g): row r, dims 4g + i of each 16
// The next block's K is on its way while the softmax runs, its V while the next scores are computed. The waves' states
// meet in LDS at the end. Bound by memory: 64 sequences at 500 .. 8,001 positions of 4 x 128 (359 MB) 61 us, 5.9 TB/s; 4
// tokens at 65,540 of 2 x 256 (134 MB) 29 us, 4.6 TB/s: five blocks a wave, the first one's latency and the meeting of the
// states stay uncovered. 1 token at 17 positions 5.3 us: a launch and four reads one behind the other.
template <typename T, int D, int NRT>
__global__ void __launch_bounds__(256, NRT* D <= 256 ? 2 : 1) few_rows(Args a, const Item* __restrict__ items,
                                                                       const int* __restrict__ nitems) {
    constexpr int NS = D / 32, NV = D / 16;
    // Q in registers, or where they are scarce (two waves a SIMD, heads of 256) in LDS, rows 16 bytes apart in the banks
    constexpr bool QLDS = D == 256 && NRT == 1;
    __shared__ __attribute__((aligned(16))) T sq[QLDS ? 16 : 1][D + 8];
    __shared__ __attribute__((aligned(16))) float so[4][16][D + 4];
    __shared__ float sm[4][16], sl[4][16];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const unsigned klane = lane * 16, vlane = g * D * 16 + r * 16;  // a lane's bytes of a K operand's KB, of a V group
    const int count = *uniform(nitems);
    for (int n = blockIdx.x; n < count; n += gridDim.x) {
        const Item it = load_item(items + n);
        const size_t page_bytes = (size_t)a.kv_heads * a.page * D * 2;
        const char* const kp = (const char*)a.kpool + (size_t)it.head * a.page * D * 2;
        const char* const vp = (const char*)a.vpool + (size_t)it.head * a.page * D * 2;
        const Uniform<int> table = uniform(a.table) + (size_t)it.seq * a.most_pages;
        const int last_row = min(it.row0 + 16 * NRT, it.rows) - 1;
        // blocks with every key in [all_lo, all_hi] are seen by all rows whole
        const int all_hi = it.pos0 + it.row0 / a.group;
        const int all_lo = a.window ? furthest(a, it, last_row) - a.window + 1 : 0;
        const int blocks = (it.k1 - it.k0 + KEYS - 1) / KEYS;
        auto key_of = [&](int j) { return it.k0 + KEYS * j; };
        auto page_of = [&](int j) { return table[key_of(min(j, blocks - 1)) >> a.page_shift]; };
        auto offset = [&](int j, int page) {  // of block j in K and V, its page known
            return page * page_bytes + (size_t)(key_of(j) & (a.page - 1)) * D * 2;
        };
        Vec8<T> kf[2][NS], vf[NV];
        // read once: non-temporal. A uniform base and a lane's 32-bit offset: no 64-bit address per lane and load.
        auto load_k = [&](size_t off) INLINE {
#pragma unroll
            for (int s = 0; s < NS; s++)
#pragma unroll
                for (int b = 0; b < 2; b++)
                    kf[b][s] = __builtin_nontemporal_load((const Vec8<T>*)(kp + off + b * 16 * D * 2 + s * 1024 + klane));
        };
        auto load_v = [&](size_t off) INLINE {
#pragma unroll
            for (int i = 0; i < NV; i++) vf[i] = __builtin_nontemporal_load((const Vec8<T>*)(vp + off + i * 256 + vlane));
        };
        size_t off = 0;
        int page = 0;
        if (w < blocks) {  // the first block is on its way while Q is prepared
            off = offset(w, page_of(w));
            load_k(off);
            load_v(off);
            page = page_of(w + 4);
        }
        Vec8<T> q[NRT][QLDS ? 1 : NS];
        int lo[NRT], hi[NRT];  // keys the lane's row sees
#pragma unroll
        for (int t = 0; t < NRT; t++) {
            const int row = it.row0 + 16 * t + r, head = it.head * a.group + row % a.group;
            const Place at = place_of(a, it, row, last_row);
            const bool is = row <= last_row && at.tok < a.rows;
            hi[t] = is ? at.pos : -1;
            lo[t] = a.window ? at.pos - a.window + 1 : 0;
            const T* const src = (const T*)a.q + (int64_t)at.tok * a.q_tok + head * a.q_head + 8 * g;
            if constexpr (QLDS) {
                // each wave brings a quarter of the rows' dims
#pragma unroll
                for (int s = 0; s < NS / 4; s++) {
                    const int d = 32 * (w * (NS / 4) + s);
                    *(Vec8<T>*)&sq[r][d + 8 * g] = is ? load8(src + d) : Vec8<T>{};
                }
            } else {
#pragma unroll
                for (int s = 0; s < NS; s++) q[t][s] = is ? load8(src + 32 * s) : Vec8<T>{};
            }
        }
        if constexpr (QLDS) lds_barrier();
        f32x4 o[NRT][NV];
        float m[NRT], l[NRT];  // the reference of the row's weights (log2 units), the lane's share of their sum
#pragma unroll
        for (int t = 0; t < NRT; t++) {
            m[t] = NEG_INF;
            l[t] = 0.f;
#pragma unroll
            for (int i = 0; i < NV; i++) o[t][i] = f32x4{};
        }
        bool odd = false;
        for (int j = w; j < blocks; j += 4) {
            const size_t next = j + 4 < blocks ? offset(j + 4, page) : off;
            page = page_of(j + 8);
            f32x4 s[NRT][2];
#pragma unroll
            for (int t = 0; t < NRT; t++) s[t][0] = s[t][1] = f32x4{};
#pragma unroll
            for (int i = 0; i < NS; i++)
#pragma unroll
                for (int t = 0; t < NRT; t++) {
                    const Vec8<T> x = QLDS ? *(const Vec8<T>*)&sq[r][32 * i + 8 * g] : q[t][QLDS ? 0 : i];
#pragma unroll
                    for (int b = 0; b < 2; b++) s[t][b] = mfma16(kf[b][i], x, s[t][b]);
                }
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
                float top = fmaxf(s[t][0][0], s[t][1][0]);  // the compiler's: it waits for both products
                top = vmax3(vmax3(vmax3(top, s[t][0][1], s[t][0][2]), s[t][0][3], s[t][1][1]), s[t][1][2], s[t][1][3]);
                top = max_xor32(max_xor16(top)) * a.scale2 - Weights<T>::LIFT;
                const bool move = m[t] != NEG_INF && top > m[t] + Weights<T>::LAZY;
                if (__any(move)) {
                    const float f = move ? fast_exp2(m[t] - top) : 1.f;
                    l[t] *= f;
#pragma unroll
                    for (int i = 0; i < NV; i++) o[t][i] *= f;
                }
                if (move || m[t] == NEG_INF) m[t] = top;
                const float ref = m[t] == NEG_INF ? 0.f : m[t];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    p[t][e] = (T)fast_exp2(__builtin_fmaf(s[t][e / 4][e % 4], a.scale2, -ref));
                    if (e % 2) l[t] = add_pair(p[t][e - 1], p[t][e], l[t]);
                }
            }
            if (edge && odd_values(vf)) {
                odd = true;
#pragma unroll
                for (int i = 0; i < NV; i++) vf[i] = finite(vf[i]);
            }
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int t = 0; t < NRT; t++) o[t][i] = mfma16(vf[i], p[t], o[t][i]);
            load_v(next);
            off = next;
        }
        if (odd) {
            for (int j = w; j < blocks; j += 4) {
                const int k0 = key_of(j);
                if (k0 + KEYS - 1 <= all_hi && k0 >= all_lo) continue;
                const T* const v = (const T*)(vp + offset(j, page_of(j)));
                for (int x = 0; x < KEYS; x++) {
#pragma unroll
                    for (int t = 0; t < NRT; t++) {
                        const bool seen = k0 + x <= hi[t] && k0 + x >= lo[t];
                        if (!__any(seen)) continue;
#pragma unroll
                        for (int i = 0; i < NV; i++) o[t][i] = add_odd<T, D>(v, x, 16 * i + 4 * g, seen, o[t][i]);
                    }
                }
            }
        }
        // the four waves' states of 16 rows at a time: 16 threads a row, 8 dims each and again (a wave that saw nothing of a
        // row has zeros)
#pragma unroll
        for (int t = 0; t < NRT; t++) {
            const float sum = add_xor32(add_xor16(l[t]));
            lds_barrier();  // the states before have been read
            if (g == 0) {
                sm[w][r] = m[t];
                sl[w][r] = sum;
            }
#pragma unroll
            for (int i = 0; i < NV; i++) *(f32x4*)&so[w][r][16 * i + 4 * g] = o[t][i];
            lds_barrier();
            const int rr = threadIdx.x >> 4, row = it.row0 + 16 * t + rr, tok = it.tok0 + row / a.group;
            if (row > last_row || (it.part < 0 && tok >= a.rows)) continue;
            const int head = it.head * a.group + row % a.group;
            const float top = fmaxf(fmaxf(sm[0][rr], sm[1][rr]), fmaxf(sm[2][rr], sm[3][rr]));
            float f[4], total = 0.f;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                f[x] = sm[x][rr] == NEG_INF ? 0.f : fast_exp2(sm[x][rr] - top);
                total += f[x] * sl[x][rr];
            }
            const float factor = it.part < 0 ? row_factor(a, head, top, total) : 1.f;
#pragma unroll
            for (int c = 0; c < (D + 127) / 128; c++) {
                const int d = ((int)(threadIdx.x & 15) + 16 * c) * 8;
                if (d >= D) continue;
                f32x4 acc[2] = {f32x4{}, f32x4{}};
#pragma unroll
                for (int x = 0; x < 4; x++)
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        const f32x4 z = *(const f32x4*)&so[x][rr][d + 4 * y];
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[y][i] += f[x] * z[i];
                    }
                acc[0] *= factor;
                acc[1] *= factor;
                if (it.part < 0) {
                    const float x[8] = {acc[0][0], acc[0][1], acc[0][2], acc[0][3], acc[1][0], acc[1][1], acc[1][2], acc[1][3]};
                    store_out<T, D, 8>(a, tok, head, d, x);
                } else {
                    float* const to = a.pacc + (size_t)(it.part + 16 * t + rr) * D + d;
                    *(f32x4*)to = acc[0];
                    *(f32x4*)(to + 4) = acc[1];
                }
            }
            if (it.part >= 0 && (threadIdx.x & 15) == 0) {
                a.pm[it.part + 16 * t + rr] = top;
                a.pl[it.part + 16 * t + rr] = total;
            }
        }
    }
}

// ---- chunks: tiles of 256 or 128 query rows against keys shared in LDS ----
// 8 waves, two to a SIMD (w and w + 4). KS = 1: each has 32 rows of the work-group's 256 and takes every key. KS = 2: waves
// 0-3 have the 32-row parts of 128 rows and waves 4-7 the same rows; a step has keys for either, and the states meet in LDS
// at the end. Per step of KT keys a wave does
//   matrix phase   O^T[D][32 rows] += V^T . P^T of the step before, S^T[KT keys][32 rows] = K . Q^T of this one
//                  (32x32x16; K rows are read in such an order that register i = 8 s + e of lane half h holds key
//                  16 (e / 4) + 4 (2 s + h) + e % 4 of its 32, element e of V's group 2 s + h: the scores become the B
//                  operand of the next product where they are, and a lane's values of O all belong to its row)
//   softmax phase  of its row (two lanes a row), in registers
// Waves 4-7 run one phase behind waves 0-3, so of a SIMD's two waves one feeds the matrix unit while the other computes
// weights. K and V come by direct loads into rings of SL steps each; barriers hand over what has landed and free what has
// been read. Bound by the matrix units, which are busy 56% of the cycles, at the 1.7 to 1.9 GHz that the card's power allows
// then: a prompt of 4,096 tokens, 32 heads of 128 on 4, 128 us, 1.07 PFLOP/s (a library's product of 16,384^3 1.3); 512 tokens
// at 9,512 positions, 16 heads of 256 on 2, 83 us and 10 for the join. By count, 64 keys at heads of 128 are 1,024 cycles of
// products and about 950 of softmax for each of a SIMD's two waves; a phase takes some 1,600.
template <int D, int KS>
struct Chunk {
    static constexpr int NW = 8, RW = NW / KS;                   // waves, waves over the rows
    static constexpr int KT = D <= 128 && KS == 1 ? 64 : KEYS;   // keys of a step for a wave
    static constexpr int SUB = KT / KEYS;                        // 32-key tiles of it
    static constexpr int TILE = KEYS * D * 2;                    // bytes of a tile's K, or V
    static constexpr int STEP = KS * SUB * TILE;                 // of a step's
    static constexpr int SL = D == 256 && KS == 2 ? 2 : 4;
    static constexpr int PIECES = SUB * TILE / 1024 / RW;        // 1 KB pieces of K, and of V, a wave copies a step
    static constexpr int LDS = SL * 2 * STEP;
    static_assert(PIECES >= 1 && TILE / 1024 % PIECES == 0 && LDS <= 150 * 1024, "rings");
};

template <typename T, int D, int KS>
__global__ void __launch_bounds__(512) chunk_rows(Args a, const Item* __restrict__ items, const int* __restrict__ nitems) {
    using C = Chunk<D, KS>;
    constexpr int NS = D / 16, NB = D / 32, SUB = C::SUB, SL = C::SL;
    __shared__ __attribute__((aligned(1024))) unsigned char ring[C::LDS];
    __shared__ float sm[C::NW][32], sl[C::NW][32];
    __shared__ int odd;
    unsigned char* const kring = ring;
    unsigned char* const vring = ring + SL * C::STEP;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, h = lane >> 5;
    const int wr = w % C::RW, kg = w / C::RW;
    const bool late = w >= 4;  // the SIMD's second wave
    const int count = *uniform(nitems);
    const unsigned lds_k = (unsigned)(uintptr_t)(lds_void*)ring, lds_v = lds_k + SL * C::STEP, voff = lane * 16;
    // the K row a lane feeds: m = r goes to key 16 (m / 8 % 2) + 8 (m / 16) + m % 8. Tiles lie in LDS as in the pages: every 16
    // lanes that are served at once have 256 bytes of their own (conflicts in 0.4% of the cycles).
    const int kaddr = kg * SUB * C::TILE + (r >> 3 & 1) * 16 * D * 2 + ((r >> 4) * 8 + (r & 7)) * 16 + h * 256;
    const int vaddr = kg * SUB * C::TILE + h * D * 16 + r * 16;
    for (int n = blockIdx.x; n < count; n += gridDim.x) {
        const Item it = load_item(items + n);
        const size_t page_bytes = (size_t)a.kv_heads * a.page * D * 2;
        const char* const kp = (const char*)a.kpool + (size_t)it.head * a.page * D * 2;
        const char* const vp = (const char*)a.vpool + (size_t)it.head * a.page * D * 2;
        const Uniform<int> table = uniform(a.table) + (size_t)it.seq * a.most_pages;
        const int tiles = (it.k1 - it.k0 + KEYS - 1) / KEYS, steps = (tiles + KS * SUB - 1) / (KS * SUB);
        // step j of key group x: tiles (j * KS + x) * SUB .. + SUB - 1; behind the last tile the last again, whose keys then
        // lie behind every row's bound (k1 at most)
        auto tile_of = [&](int j, int t) { return (j * KS + kg) * SUB + t; };
        // A wave's pieces of a step lie in one tile. Where that is in the pages is looked up a step ahead: the look-up's
        // latency stood in front of every copy otherwise.
        constexpr int PER = C::TILE / 1024;
        const int own = wr * C::PIECES / PER, at0 = wr * C::PIECES % PER;
        auto key_of = [&](int j) { return it.k0 + KEYS * min(tile_of(min(j, steps - 1), own), tiles - 1); };
        auto page_of = [&](int j) { return table[key_of(j) >> a.page_shift]; };
        auto offset = [&](int j, int page) { return page * page_bytes + (size_t)(key_of(j) & (a.page - 1)) * D * 2 + at0 * 1024; };
        auto issue_k = [&](int j, size_t off) {
            const unsigned to = lds_k + j % SL * C::STEP + (kg * SUB + own) * C::TILE + at0 * 1024;
#pragma unroll
            for (int p = 0; p < C::PIECES; p++) dma16s(kp + off + p * 1024, voff, to + p * 1024);
        };
        auto issue_v = [&](int j, size_t off) {
            const unsigned to = lds_v + j % SL * C::STEP + (kg * SUB + own) * C::TILE + at0 * 1024;
#pragma unroll
            for (int p = 0; p < C::PIECES; p++) dma16s(vp + off + p * 1024, voff, to + p * 1024);
        };
        // ONE: a barrier a step; with rings of two steps two, and copies a step further ahead. Copies go out in the softmax
        // phase, which is the shorter one (in the matrix phase they took 430 of its 1,700 cycles): K of step i + SL - 1 + LEAD
        // and V of the step before it in that of step i, into the places of K of step i - 1 + LEAD and of the V before it.
        // Those have been read by then: ONE, before the barrier in front of waves 0-3's step i, behind waves 4-7's matrix
        // phase i - 1; else by the wave's own key group, before the barrier in front.
        constexpr bool ONE = SL >= 3;
        constexpr int LEAD = ONE ? 0 : 1;
        __syncthreads();  // the rings and the flag of the item before have been read
        if (threadIdx.x == 0) odd = 0;
#pragma unroll
        for (int j = 0; j < SL - 1 + LEAD; j++) {
            const size_t off = offset(j, page_of(j));
            issue_k(j, off);
            if (j < SL - 2 + LEAD) issue_v(j, off);
        }
        // of the next copies: V of the one, K of the other
        size_t v_next = offset(SL - 2 + LEAD, page_of(SL - 2 + LEAD)), k_next = offset(SL - 1 + LEAD, page_of(SL - 1 + LEAD));

        const int row = it.row0 + 32 * wr + r, last_row = min(it.row0 + 32 * C::RW, it.rows) - 1;
        const int head = it.head * a.group + row % a.group;
        const Place at = place_of(a, it, row, last_row);
        const bool is = row <= last_row && at.tok < a.rows;
        const int hi = is ? min(at.pos, it.k1 - 1) : -1, lo = a.window ? at.pos - a.window + 1 : 0;
        // keys in [tile_lo, tile_hi] are seen by all rows of the work-group, in [all_lo, all_hi] by all of the wave's
        const int tile_hi = min(it.pos0 + it.row0 / a.group, it.k1 - 1);
        const int tile_lo = a.window ? furthest(a, it, last_row) - a.window + 1 : 0;
        const int all_hi = min(it.pos0 + (it.row0 + 32 * wr) / a.group, it.k1 - 1);
        const int all_lo = a.window ? furthest(a, it, min(it.row0 + 32 * wr + 31, last_row)) - a.window + 1 : 0;
        // infinities and NaN of V in a tile that crosses some row's bounds: each wave looks through the pieces it has copied
        // and puts zeros there before the others read them (add_odd brings them in after the loop)
        auto mend = [&](int j) INLINE {
#pragma unroll
            for (int p = 0; p < C::PIECES; p++) {
                const int at = wr * C::PIECES + p, k0 = it.k0 + KEYS * tile_of(j, own);
                if (k0 + KEYS - 1 <= tile_hi && k0 >= tile_lo) break;
                Vec8<T>* const x = (Vec8<T>*)(vring + j % SL * C::STEP + kg * SUB * C::TILE + at * 1024 + lane * 16);
                const Vec8<T> v[1] = {*x};
                if (odd_values(v)) {
                    *x = finite(v[0]);
                    odd = 1;
                }
            }
        };
        Vec8<T> q[NS];
        const T* const src = (const T*)a.q + (int64_t)at.tok * a.q_tok + head * a.q_head + 8 * h;
#pragma unroll
        for (int s = 0; s < NS; s++) q[s] = is ? load8(src + 16 * s) : Vec8<T>{};
        f32x16 o[NB], s[SUB];
        Vec8<T> p[2 * SUB];
#pragma unroll
        for (int i = 0; i < NB; i++) o[i] = f32x16{};
        float m = NEG_INF, l = 0.f;

        // What a wave has copied of step i's K and of the V of the step before has landed, mended. Behind it may be on their
        // way: what it issued after those, `behind` steps' K and V.
        auto landed = [&](int i, auto behind) INLINE {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * C::PIECES * decltype(behind)::value) : "memory");
            if (i > 0) mend(i - 1);
        };
        auto k_of = [&](int i, int x) {  // operand x of step i: tile x / NS, dims 16 (x % NS) ..
            return *(const Vec8<T>*)(kring + i % SL * C::STEP + kaddr + x / NS * C::TILE + x % NS * 512);
        };
        auto v_of = [&](int i, int x) {  // dim block x % NB, tile x / NB / 2, groups 2 (x / NB % 2) + h
            const int at = x / NB / 2 * C::TILE + x / NB % 2 * 2 * D * 16 + x % NB * 512;
            return *(const Vec8<T>*)(vring + i % SL * C::STEP + vaddr + at);
        };
        constexpr int AHEAD = D == 256 ? 3 : 4, NK = NS * SUB, NVO = 2 * NB * SUB;  // operands on their way ahead; of a step
        auto products = [&](int i, auto with_v, auto with_k) INLINE {  // P.V of step i - 1, scores of step i
            constexpr bool PV = decltype(with_v)::value, QK = decltype(with_k)::value;
            constexpr int ALL = (PV ? NVO : 0) + (QK ? NK : 0), V0 = PV ? NVO : 0;
            Vec8<T> x[AHEAD];
            auto get = [&](int y) { return y < V0 ? v_of(i - 1, y) : k_of(i, y - V0); };
#pragma unroll
            for (int y = 0; y < AHEAD; y++) x[y] = get(y);
            if constexpr (QK) {
#pragma unroll
                for (int t = 0; t < SUB; t++) s[t] = f32x16{};
            }
#pragma unroll
            for (int y = 0; y < ALL; y++) {
                const Vec8<T> z = x[y % AHEAD];
                if (y + AHEAD < ALL) x[y % AHEAD] = get(y + AHEAD);
                if (y < V0) o[y % NB] = mfma32(z, p[y / NB], o[y % NB]);
                else s[(y - V0) / NS] = mfma32(z, q[(y - V0) % NS], s[(y - V0) / NS]);
            }
            __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
            for (int y = 0; y < ALL - AHEAD; y++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
        };
        auto softmax = [&](int j) INLINE {
            float top = NEG_INF;
#pragma unroll
            for (int t = 0; t < SUB; t++) {
                const int k0 = it.k0 + KEYS * tile_of(j, t);
                if (k0 + KEYS - 1 > all_hi || k0 < all_lo) {
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int key = k0 + i % 8 / 4 * 16 + 4 * (i / 8 * 2 + h) + i % 4;
                        if (key > hi || key < lo) s[t][i] = NEG_INF;
                    }
                }
                top = fmaxf(top, fmaxf(s[t][0], s[t][1]));  // the compiler's: it waits for the products
#pragma unroll
                for (int i = 2; i < 16; i += 2) top = vmax3(top, s[t][i], s[t][i + 1]);
            }
            top = max_xor32(top) * a.scale2 - Weights<T>::LIFT;
            const bool move = m != NEG_INF && top > m + Weights<T>::LAZY;
            if (__any(move)) {
                const float f = move ? fast_exp2(m - top) : 1.f;
                l *= f;
#pragma unroll
                for (int i = 0; i < NB; i++) o[i] *= f;
            }
            if (move || m == NEG_INF) m = top;
            const float ref = m == NEG_INF ? 0.f : m;
            float sum = 0.f;
#pragma unroll
            for (int t = 0; t < SUB; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    p[2 * t + i / 8][i % 8] = (T)fast_exp2(__builtin_fmaf(s[t][i], a.scale2, -ref));
                    if (i % 2) sum = add_pair(p[2 * t + i / 8][i % 8 - 1], p[2 * t + i / 8][i % 8], sum);
                }
            l += sum;
            // the weights are done here, not where they are used: the compiler moved the exponentials behind the phase's
            // barrier, into the matrix phase
#pragma unroll
            for (int t = 0; t < 2 * SUB; t++) {
                u32x4 x = __builtin_bit_cast(u32x4, p[t]);
                asm volatile("" : "+v"(x));
                p[t] = __builtin_bit_cast(Vec8<T>, x);
            }
        };
        auto phase_end = [&](bool wait, int i, auto behind) INLINE {  // wait: this wave's copies for step i are due
            __builtin_amdgcn_sched_barrier(0);
            if (wait) landed(i, behind);
            lds_barrier();
            __builtin_amdgcn_sched_barrier(0);
        };
        using std::false_type;
        using std::true_type;
        const std::integral_constant<int, SL - 2 + LEAD> behind{};
        phase_end(true, 0, behind);
        if (!ONE && late) phase_end(false, 0, behind);
        // ONE: barrier i + 1 stands behind waves 0-3's softmax phase i and waves 4-7's matrix phase i; copies for step i + 1 are
        // due in front of it. Else barriers stand behind every phase; copies are due at the end of the softmax phase.
        auto step = [&](int i, auto with_v) INLINE {
            __builtin_amdgcn_s_setprio(1);
            products(i, with_v, true_type{});
            __builtin_amdgcn_s_setprio(0);
            if (!ONE || late) phase_end(ONE, i + 1, std::integral_constant<int, ONE ? SL - 3 : 0>{});
            __builtin_amdgcn_sched_barrier(0);
            issue_v(i + SL - 2 + LEAD, v_next);
            issue_k(i + SL - 1 + LEAD, k_next);
            __builtin_amdgcn_sched_barrier(0);
            const int page = page_of(i + SL + LEAD);
            softmax(i);
            v_next = k_next;
            k_next = offset(i + SL + LEAD, page);
            if (!ONE || !late) phase_end(true, i + 1, behind);
        };
        step(0, false_type{});
        for (int i = 1; i < steps; i++) step(i, true_type{});
        products(steps, true_type{}, false_type{});
        if (!ONE && !late) phase_end(false, 0, behind);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // copies that no step needs write the rings no more behind this
        __syncthreads();
        if (odd) {
            for (int j = 0; j < tiles; j++) {
                const int k0 = it.k0 + KEYS * j;
                if (j / SUB % KS != kg || (k0 + KEYS - 1 <= tile_hi && k0 >= tile_lo)) continue;
                const T* const v = (const T*)vp + table[k0 >> a.page_shift] * (page_bytes / 2) + (size_t)(k0 & (a.page - 1)) * D;
                for (int x = 0; x < KEYS; x++) {
                    const bool seen = k0 + x <= hi && k0 + x >= lo;
                    if (!__any(seen)) continue;
#pragma unroll
                    for (int i = 0; i < 4 * NB; i++) {
                        const f32x16& z = o[i / 4];
                        f32x4 y = {z[i % 4 * 4], z[i % 4 * 4 + 1], z[i % 4 * 4 + 2], z[i % 4 * 4 + 3]};
                        y = add_odd<T, D>(v, x, 32 * (i / 4) + 8 * (i % 4) + 4 * h, seen, y);
#pragma unroll
                        for (int c = 0; c < 4; c++) o[i / 4][i % 4 * 4 + c] = y[c];
                    }
                }
            }
        }
        l += __shfl_xor(l, 32);
        // o[b][4 c + i]: dim 32 b + 8 c + 4 h + i of row r. The rows go out through the wave's part of the rings, which nobody
        // reads any more, BLOCKS x 32 dims at a time: whole runs of a row, with the gate read in such runs too.
        constexpr int OB = NB / KS, BLOCKS = D == 64 ? 1 : 2, DW = 32 * BLOCKS, ROW = DW + 4, PER_ROW = DW / 8;
        static_assert(C::NW * 32 * ROW * 4 <= C::LDS, "output rows");
        float* const rows_lds = (float*)ring + w * 32 * ROW;
        auto put = [&](auto first, float factor) INLINE {  // blocks first .. + BLOCKS - 1, times the factor of the lane's row
#pragma unroll
            for (int b = 0; b < BLOCKS; b++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    f32x4 x;
#pragma unroll
                    for (int i = 0; i < 4; i++) x[i] = o[first + b][4 * c + i] * factor;
                    *(f32x4*)(rows_lds + r * ROW + 32 * b + 8 * c + 4 * h) = x;
                }
            __builtin_amdgcn_wave_barrier();
#pragma unroll 2
            for (int i = lane; i < 32 * PER_ROW; i += 64) {
                const int x = i / PER_ROW, d = i % PER_ROW * 8, row = it.row0 + 32 * wr + x;
                const int tok = it.tok0 + row / a.group, head = it.head * a.group + row % a.group;
                if (row > last_row || (it.part < 0 && tok >= a.rows)) continue;
                const f32x4 lo = *(const f32x4*)(rows_lds + x * ROW + d), hi = *(const f32x4*)(rows_lds + x * ROW + d + 4);
                const int dim = 32 * first + d;
                if (it.part >= 0) {
                    float* const to = a.pacc + (size_t)(it.part + 32 * wr + x) * D + dim;
                    *(f32x4*)to = lo;
                    *(f32x4*)(to + 4) = hi;
                } else {
                    const float y[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                    store_out<T, D, 8>(a, tok, head, dim, y);
                }
            }
            __builtin_amdgcn_wave_barrier();
        };
        auto finish_rows = [&](auto first) INLINE {
            const float factor = it.part >= 0 ? 1.f : row_factor(a, min(head, a.q_heads - 1), m, l);
            constexpr int B = decltype(first)::value;
            put(first, factor);
            if constexpr (OB > BLOCKS) put(std::integral_constant<int, B + BLOCKS>{}, factor);
            if constexpr (OB > 2 * BLOCKS) {
                put(std::integral_constant<int, B + 2 * BLOCKS>{}, factor);
                put(std::integral_constant<int, B + 3 * BLOCKS>{}, factor);
            }
        };
        const std::integral_constant<int, 0> low{};
        const std::integral_constant<int, NB / 2> high{};
        if constexpr (KS == 1) {
            finish_rows(low);
        } else {
            // two states of each row, in waves w and w ^ RW: both taken to the larger reference, each wave finishes half of
            // the dims with its partner's half of them, which goes through the ring
            if (h == 0) {
                sm[w][r] = m;
                sl[w][r] = l;
            }
            __syncthreads();
            const float mo = sm[w ^ C::RW][r], lo2 = sl[w ^ C::RW][r], top = fmaxf(m, mo);
            const float f = m == NEG_INF ? 0.f : fast_exp2(m - top), fo = mo == NEG_INF ? 0.f : fast_exp2(mo - top);
            f32x4* const give = (f32x4*)ring + w * (NB / 2 * 256) + lane;
            const f32x4* const take = (const f32x4*)ring + (w ^ C::RW) * (NB / 2 * 256) + lane;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                o[b] *= f;
                if (b / (NB / 2) != kg) {
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        give[(b % (NB / 2) * 4 + c) * 64] = f32x4{o[b][4 * c], o[b][4 * c + 1], o[b][4 * c + 2], o[b][4 * c + 3]};
                }
            }
            __syncthreads();
#pragma unroll
            for (int b = 0; b < NB; b++)
                if (b / (NB / 2) == kg) {
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const f32x4 x = take[(b % (NB / 2) * 4 + c) * 64];
#pragma unroll
                        for (int i = 0; i < 4; i++) o[b][4 * c + i] += x[i];
                    }
                }
            m = top;
            l = l * f + lo2 * fo;
            __syncthreads();  // what was given has been taken
            if (kg == 0) finish_rows(low);
            else finish_rows(high);
        }
        if (it.part >= 0 && kg == 0 && h == 0 && is) {
            a.pm[it.part + 32 * wr + r] = m;
            a.pl[it.part + 32 * wr + r] = l;
        }
    }
}

// ---- splits of a tile's rows put together ----
// A split with no weight for a row counts all the same: it is zeros where the row sees nothing of it, and NaN or infinities
// where the row does see them, which reach it however small their weights (m = -inf beside l = NaN: the one key that the
// row sees there has a NaN score, which no maximum takes).
// D / 4 lanes hold a row, four dims each, and read its splits four at a time; a work-group takes 1024 / D rows. Wide: a
// work-group takes 64 dims of a row; 16 lanes hold them, and each 16 lanes add up every 16th split, with the
// splits' factors in LDS. (A row whole in a work-group, 32 rows of 121 splits: 7.9 us; by 64 dims 5.2.) ROW_WIDE, many splits of many
// rows: a work-group takes a row, each D / 4 lanes four splits of it at a time.
constexpr int JOIN_DIMS = 64;
//
// Rows of sequences that share keys have more splits, those of the shared tiles they are in: Seg by Seg behind their own.
struct Segs {  // of a join; one that it does not have has no splits
    Seg x[LEVELS];
    int splits = 0;
    __device__ Segs(const Seg* p, int n) {
#pragma unroll
        for (int i = 0; i < LEVELS; i++) {
            x[i] = Seg{0, 0, 0, 0};
            if (i < n) {
                const Uniform<int> u = uniform((const int*)(p + i));
                x[i] = Seg{u[0], u[1], u[2], 0};
                splits += u[2];
            }
        }
    }
    // the partial of row r of the join in split s of them
    __device__ size_t row(int s, int r) const {
        int part = x[0].part, stride = x[0].stride;
#pragma unroll
        for (int i = 1, before = x[0].splits; i < LEVELS; before += x[i++].splits)
            if (s >= before) {
                part = x[i].part - before * x[i].stride;
                stride = x[i].stride;
            }
        return (size_t)(part + s * stride + r);
    }
};
// SHARED: the join may have such.
template <typename T, int D, bool SHARED>
__device__ __forceinline__ void join_rows(const Args& a, const Join& j, const Seg* segs, int way, int ways, float (&factor)[SPLITS_MOST],
                                          f32x4 (&sa)[16][16], float (&red)[2][4]) {
    const int tid = threadIdx.x;
    auto finish = [&](int tok, int head, int d, f32x4 acc, float m, float l) INLINE {
        acc *= row_factor(a, head, m, l);
        const float x[4] = {acc[0], acc[1], acc[2], acc[3]};
        store_out<T, D, 4>(a, tok, head, d, x);
    };
    const Segs shared(segs, SHARED ? j.segs : 0);
    if (!j.wide) {
        constexpr int LANES = D / 4, GROUPS = 256 / LANES;
        const int d = tid % LANES * 4;
        for (int r = way * GROUPS + tid / LANES; r < j.count; r += ways * GROUPS) {
            const int row = j.row0 + r, tok = j.tok0 + row / a.group;
            if (tok >= a.rows) continue;
            f32x4 acc = f32x4{};
            float top = NEG_INF, total = 0.f;
            // splits s0 .. s0 + 3 of those at `part`; behind the last: the last again, not counted
            auto four = [&](int part, int stride, int splits, int s0, bool begun) INLINE {
                float m[4], l[4];
                f32x4 x[4];
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const size_t at = part + r + (size_t)min(s0 + s, splits - 1) * stride;
                    m[s] = a.pm[at];
                    l[s] = a.pl[at];
                    x[s] = *(const f32x4*)(a.pacc + at * D + d);
                }
                const float was = top;
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    if (s0 + s >= splits) {
                        m[s] = NEG_INF;
                        l[s] = 0.f;
                        x[s] = f32x4{};
                    }
                    top = fmaxf(top, m[s]);
                }
                if (begun) {
                    const float f = was == NEG_INF ? 0.f : fast_exp2(was - top);
                    acc *= f;
                    total *= f;
                }
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const float f = m[s] == NEG_INF ? 0.f : fast_exp2(m[s] - top);
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[i] += f * x[s][i];
                    total += f * l[s];
                }
            };
            four(j.part, j.count, j.splits, 0, false);
            for (int s = 4; s < j.splits; s += 4) four(j.part, j.count, j.splits, s, true);
#pragma unroll
            for (int i = 0; i < (SHARED ? LEVELS : 0); i++)
                for (int s = 0; s < shared.x[i].splits; s += 4) four(shared.x[i].part, shared.x[i].stride, shared.x[i].splits, s, true);
            finish(tok, j.head * a.group + row % a.group, d, acc, top, total);
        }
        return;
    }
    const int splits = j.splits + shared.splits;
    if (SHARED && j.wide == ROW_WIDE) {
        constexpr int LANES = D / 4, GROUPS = 256 / LANES;
        const int group = tid / LANES, lane = tid % LANES;
        for (int r = way; r < j.count; r += ways) {
            const int row = j.row0 + r, tok = j.tok0 + row / a.group;
            if (tok >= a.rows) continue;
            f32x4 acc = f32x4{};
            float top = NEG_INF, total = 0.f;
            for (int s0 = 4 * group; s0 < splits; s0 += 4 * GROUPS) {  // behind the last the last again, not counted
                float m[4], l[4];
                f32x4 x[4];
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const int at = min(s0 + s, splits - 1);
                    const size_t p = at < j.splits ? j.part + r + (size_t)at * j.count : shared.row(at - j.splits, r);
                    m[s] = a.pm[p];
                    l[s] = a.pl[p];
                    x[s] = *(const f32x4*)(a.pacc + p * D + lane * 4);
                }
                const float was = top;
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    if (s0 + s >= splits) {
                        m[s] = NEG_INF;
                        l[s] = 0.f;
                        x[s] = f32x4{};
                    }
                    top = fmaxf(top, m[s]);
                }
                const float f = was == NEG_INF ? 0.f : fast_exp2(was - top);
                acc *= f;
                total *= f;
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const float f = m[s] == NEG_INF ? 0.f : fast_exp2(m[s] - top);
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[i] += f * x[s][i];
                    total += f * l[s];
                }
            }
            __syncthreads();  // the row before has been read
            (&sa[0][0])[tid] = acc;
            if (lane == 0) {
                factor[group] = top;
                factor[16 + group] = total;
            }
            lds_barrier();
            if (group) continue;
            float all = top;
#pragma unroll
            for (int x = 1; x < GROUPS; x++) all = fmaxf(all, factor[x]);
            const float f = top == NEG_INF ? 0.f : fast_exp2(top - all);
            acc *= f;
            total *= f;
#pragma unroll
            for (int x = 1; x < GROUPS; x++) {
                const float f = factor[x] == NEG_INF ? 0.f : fast_exp2(factor[x] - all);
                const f32x4 y = (&sa[0][0])[x * LANES + lane];
#pragma unroll
                for (int i = 0; i < 4; i++) acc[i] += f * y[i];
                total += f * factor[16 + x];
            }
            finish(tok, j.head * a.group + row % a.group, lane * 4, acc, all, total);
        }
        return;
    }
    constexpr int PER_ROW = D / JOIN_DIMS;
    const int part = tid / 16, lane = tid % 16;
    for (int u = way; u < j.count * PER_ROW; u += ways) {
        const int r = u / PER_ROW, d = u % PER_ROW * JOIN_DIMS + lane * 4;
        const int row = j.row0 + r, tok = j.tok0 + row / a.group;
        if (tok >= a.rows) continue;
        const size_t first = j.part + r;
        auto partial = [&](int s) INLINE { return !SHARED || s < j.splits ? first + (size_t)s * j.count : shared.row(s - j.splits, r); };
        float top = NEG_INF;
        for (int s = tid; s < splits; s += 256) top = fmaxf(top, a.pm[partial(s)]);
        // the first splits' values are on their way meanwhile
        constexpr int EARLY = 8;
        f32x4 x[EARLY];
#pragma unroll
        for (int i = 0; i < EARLY; i++) x[i] = *(const f32x4*)(a.pacc + partial(min(part + 16 * i, splits - 1)) * D + d);
#pragma unroll
        for (int i = 1; i < 64; i *= 2) top = fmaxf(top, __shfl_xor(top, i));
        __syncthreads();  // the row before has been read
        if (tid % 64 == 0) red[0][tid / 64] = top;
        lds_barrier();
        top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
        float total = 0.f;
        for (int s = tid; s < splits; s += 256) {
            const size_t at = partial(s);
            const float m = a.pm[at], f = m == NEG_INF ? 0.f : fast_exp2(m - top);
            factor[s] = f;
            total += f * a.pl[at];
        }
#pragma unroll
        for (int i = 1; i < 64; i *= 2) total += __shfl_xor(total, i);
        if (tid % 64 == 0) red[1][tid / 64] = total;
        lds_barrier();
        total = red[1][0] + red[1][1] + red[1][2] + red[1][3];
        f32x4 acc = f32x4{};
        auto add = [&](int s, f32x4 y) INLINE {
            const float f = factor[s];
#pragma unroll
            for (int c = 0; c < 4; c++) acc[c] += f * y[c];
        };
#pragma unroll
        for (int i = 0; i < EARLY; i++)
            if (part + 16 * i < splits) add(part + 16 * i, x[i]);
#pragma unroll 4
        for (int s = part + 16 * EARLY; s < splits; s += 16) add(s, *(const f32x4*)(a.pacc + partial(s) * D + d));
        sa[part][lane] = acc;
        lds_barrier();
        if (part) continue;
        acc = sa[0][lane];
#pragma unroll
        for (int i = 1; i < 16; i++) acc += sa[i][lane];
        finish(tok, j.head * a.group + row % a.group, d, acc, top, total);
    }
}
template <typename T, int D, bool SHARED>
__global__ void __launch_bounds__(256) join_kernel(Args a, const Join* __restrict__ joins, const int* __restrict__ njoins,
                                                   const Seg* __restrict__ segs) {
    __shared__ float factor[SPLITS_MOST];
    __shared__ __attribute__((aligned(16))) f32x4 sa[16][16];
    __shared__ float red[2][4];
    const int count = *uniform(njoins);
    // work-groups of a join: as many as there are for each
    const int ways = max(1, (int)gridDim.x / max(1, count)), way = blockIdx.x % ways;
    for (int n = blockIdx.x / ways; n < count; n += gridDim.x / ways) {
        const Uniform<int> ji = uniform((const int*)(joins + n));
        const Join j{ji[0], ji[1], ji[2], ji[3], ji[4], ji[5], ji[6], ji[7]};
        if (SHARED && j.segs) join_rows<T, D, true>(a, j, segs + (size_t)n * LEVELS, way, ways, factor, sa, red);
        else join_rows<T, D, false>(a, j, nullptr, way, ways, factor, sa, red);
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
    a.order = x.order;
    hipError_t e = hipSuccess;
    if (grid[FEW]) {
        few_rows<T, D, 1><<<dim3(grid[FEW]), dim3(256), 0, s>>>(a, (const Item*)(batch + l.items[FEW]), batch + FEW);
        e = hipGetLastError();
    }
    if (grid[SOME] && e == hipSuccess) {
        few_rows<T, D, 2><<<dim3(grid[SOME]), dim3(256), 0, s>>>(a, (const Item*)(batch + l.items[SOME]), batch + SOME);
        e = hipGetLastError();
    }
    if (grid[HALF] && e == hipSuccess) {
        chunk_rows<T, D, 2><<<dim3(grid[HALF]), dim3(512), 0, s>>>(a, (const Item*)(batch + l.items[HALF]), batch + HALF);
        e = hipGetLastError();
    }
    if (grid[MANY] && e == hipSuccess) {
        chunk_rows<T, D, 1><<<dim3(grid[MANY]), dim3(512), 0, s>>>(a, (const Item*)(batch + l.items[MANY]), batch + MANY);
        e = hipGetLastError();
    }
    if (join_grid && e == hipSuccess) {
        int ways = 1;  // for a join: the most that one of them has rows for
        if (!x.captured)
            for (const Join& j : *x.joins) {
                const int groups = 1024 / D;
                ways = std::max(ways, j.wide == ROW_WIDE ? j.count : j.wide ? j.count * (D / JOIN_DIMS) : (j.count + groups - 1) / groups);
            }
        const int all = std::min(join_grid, MOST_GRID / ways) * ways;
        const auto kernel = x.shared ? join_kernel<T, D, true> : join_kernel<T, D, false>;
        kernel<<<dim3(all), dim3(256), 0, s>>>(a, (const Join*)(batch + l.joins), batch + KINDS, (const Seg*)(batch + l.segs));
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

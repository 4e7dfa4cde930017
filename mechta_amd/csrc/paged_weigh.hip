// paged_weigh.hip -- attention weights accumulated position by position, and eviction by them.
//
// What the counted tokens t of a batch give to position j of kv head g, over the query heads h of its group:
//   w_j = sum over t, h of exp(s_thj - m_th) / l_th,   l_th = sum over j of exp(s_thj - m_th) [+ exp(sink_h - m_th)]
// so it takes two readings of the scores: of every row's m and l (score_few, score_rows), then of every position's sum over
// the rows (sum_few, sum_rows). Few rows keep their scores between the two, 4 bytes a score against 2 x head_dim of K; many
// rows' scores are computed again. Everything behind the products is in f32, nothing is rounded in between, and sums are taken
// in an order that does not depend on timing.
#include <algorithm>

#include "mkv_device.h"
#include "paged_device.h"

namespace mkv {
namespace paged {
namespace {

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

struct Args {
    const int* table;
    int most_pages, page, page_shift;
    int kv_heads, group, window, rows;
    const void* kpool;  // the layer's K pages
    const void* q;
    int64_t q_tok, q_head;
    const float* sinks;
    float scale2, decay;  // scale * log2 e
    float2* stats;        // a row's reference (log2 units) and sum, piece by piece of its keys
    float* work;
    float* weights;       // of the layer
    size_t stride, seq_stride;
};

// K of a sequence: where the 32 positions from `key` on lie.
template <int D>
struct Keys {
    const char* p;
    Uniform<int> table;
    size_t page_bytes;
    int shift, mask;
    __device__ Keys(const Args& a, int seq, int head)
        : p((const char*)a.kpool + (size_t)head * a.page * D * 2), table(uniform(a.table) + (size_t)seq * a.most_pages),
          page_bytes((size_t)a.kv_heads * a.page * D * 2), shift(a.page_shift), mask(a.page - 1) {}
    __device__ const char* block(int key) const { return p + table[key >> shift] * page_bytes + (size_t)(key & mask) * D * 2; }
};

// (m, l) of the same row put together; m = -inf: nothing but what l says (NaN of a score that no maximum takes).
__device__ inline float2 merge(float2 x, float2 y) {
    const float m = fmaxf(x.x, y.x);
    const float f = x.x == NEG_INF ? 0.f : fast_exp2(x.x - m), g = y.x == NEG_INF ? 0.f : fast_exp2(y.x - m);
    return make_float2(m, x.y * f + y.y * g);
}
__device__ inline float2 shuffled(float2 x, int by) { return make_float2(__shfl_xor(x.x, by), __shfl_xor(x.y, by)); }
// What turns a row's scores into weights: exp2(score - m) * r.
__device__ inline float2 factor_of(const Args& a, float2 s, int head) {
    if (a.sinks) s = merge(s, make_float2(a.sinks[head] * LOG2E, 1.f));
    return make_float2(s.x, 1.f / s.y);
}
// The same for row `row` of a sequence's kv head; a row that the call does not have weighs nothing, exp2(score - inf) * 0.
__device__ inline float2 final_of(const Args& a, float2 s, int tok0, int head, int row) {
    return tok0 + row / a.group < a.rows ? factor_of(a, s, head * a.group + row % a.group) : make_float2(-NEG_INF, 0.f);
}
// Scores of a row (log2 units) in its (m, l).
template <int N>
__device__ inline void add_scores(float2& ml, const float (&s)[N]) {
    float top = ml.x;
#pragma unroll
    for (int i = 0; i < N; i += 2) top = vmax3(top, s[i], s[i + 1]);
    const float ref = top == NEG_INF ? 0.f : top;
    float sum = ml.x == NEG_INF ? ml.y : ml.y * fast_exp2(ml.x - ref);
#pragma unroll
    for (int i = 0; i < N; i++) sum += fast_exp2(s[i] - ref);
    ml = make_float2(top, sum);
}

__device__ inline Score load_score(const Score* p) {
    const Uniform<int> x = uniform((const int*)p);
    return Score{x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7], x[8], x[9], x[10], 0};
}
__device__ inline Sum load_sum(const Sum* p) {
    const Uniform<int> x = uniform((const int*)p);
    return Sum{x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7], x[8], x[9], x[10], x[11], x[12], x[13], {0, 0}};
}

// ---- few rows' kept scores summed up: a thread a key, a row's scores of 16 neighbours in one 64-byte run ----
__device__ inline void put_factor(const Args& a, float2 s, int head, int row, float2* f, int& odd) {
    f[row] = s = factor_of(a, s, head * a.group + row % a.group);
    if (!(s.y < -NEG_INF)) odd = 1;  // its weights are no numbers where it sees, and nothing all the same where it does not
}
// rows: of the sequence, there: of them in the call; f: their factors
__device__ inline void sum_kept(const Args& a, int seq, int head, int pos0, int k0, int k1, int rows, int there, int scores, int s0,
                                const float2* f, int odd) {
    float* const weights = a.weights + seq * a.seq_stride + head * a.stride;
    for (int key = k0 + (int)threadIdx.x; key < k1; key += 256) {
        const int i = key - s0;
        const float* const s = a.work + scores + (size_t)(i / 16) * 16 * rows + i % 16;
        const float was = a.decay == 0.f ? 0.f : a.decay * weights[key];
        float sum = 0.f;
#pragma unroll 8
        for (int r = 0; r < there; r++) sum += fast_exp2(s[r * 16] - f[r].x) * f[r].y;
        if (odd) {
            sum = 0.f;
            for (int r = 0; r < there; r++) {
                const int pos = pos0 + r / a.group;
                if (key <= pos && (!a.window || key > pos - a.window)) sum += fast_exp2(s[r * 16] - f[r].x) * f[r].y;
            }
        }
        weights[key] = was + sum;
    }
}

// ---- statistics of few rows, NRT x 16 of them, with their scores ----
// 4 waves, each with every fourth block of 32 keys, its K straight from memory into the operands of the 16x16x32 products, the
// next block's on its way meanwhile. Lane (r, g): row r, keys 4g + i and 16 + 4g + i of the block; each lane has an m and l of
// its own until the end. Where there is no other piece, the sums are taken at once. Bound by memory: 64 sequences of a token at
// 500 .. 8,001 positions of 4 x 128, 185 MB of K, 41 us; 8 of them are the 23 MB of scores that it writes (33 without, 5.5 TB/s),
// 16 keys of a row behind the other, whole lines a store, which spare the second reading of K. One token at 300 positions of
// 2 x 256, a launch: 6.0 us.
template <typename T, int D, int NRT>
__global__ void __launch_bounds__(256) score_few(Args a, const Score* __restrict__ items, const int* __restrict__ nitems) {
    constexpr int NS = D / 32;
    __shared__ float2 sml[4][16 * NRT], f[16 * NRT];
    __shared__ int odd;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int count = *uniform(nitems);
    for (int n = blockIdx.x; n < count; n += gridDim.x) {
        const Score it = load_score(items + n);
        const Keys<D> keys(a, it.seq, it.head);
        const int blocks = (it.k1 - it.k0 + KEYS - 1) / KEYS;
        Vec8<T> kf[2][NS];
        auto load_k = [&](int j) INLINE {
            const char* const p = keys.block(it.k0 + KEYS * min(j, blocks - 1));
#pragma unroll
            for (int s = 0; s < NS; s++)
#pragma unroll
                for (int b = 0; b < 2; b++)
                    kf[b][s] = __builtin_nontemporal_load((const Vec8<T>*)(p + b * 16 * D * 2 + s * 1024 + lane * 16));
        };
        if (w < blocks) load_k(w);
        Vec8<T> q[NRT][NS];
        int lo[NRT], hi[NRT];
        float2 ml[NRT];
#pragma unroll
        for (int t = 0; t < NRT; t++) {
            const int row = 16 * t + r, tok = row / a.group, head = it.head * a.group + row % a.group;
            const bool is = row < it.rows && it.tok0 + tok < a.rows;
            hi[t] = is ? it.pos0 + tok : -1;
            lo[t] = a.window ? it.pos0 + tok - a.window + 1 : 0;
            const T* const src = (const T*)a.q + (int64_t)(it.tok0 + tok) * a.q_tok + head * a.q_head + 8 * g;
#pragma unroll
            for (int s = 0; s < NS; s++) q[t][s] = is ? load8(src + 32 * s) : Vec8<T>{};
            ml[t] = make_float2(NEG_INF, 0.f);
        }
        const int all_hi = it.pos0, all_lo = a.window ? it.pos0 + (it.rows - 1) / a.group - a.window + 1 : 0;
        for (int j = w; j < blocks; j += 4) {
            f32x4 s[NRT][2];
#pragma unroll
            for (int t = 0; t < NRT; t++) s[t][0] = s[t][1] = f32x4{};
#pragma unroll
            for (int i = 0; i < NS; i++)
#pragma unroll
                for (int t = 0; t < NRT; t++)
#pragma unroll
                    for (int b = 0; b < 2; b++) s[t][b] = mfma16(kf[b][i], q[t][i], s[t][b]);
            load_k(j + 4);
            const int k0 = it.k0 + KEYS * j;
            const bool edge = k0 + KEYS - 1 > all_hi || k0 < all_lo;
            float* const to = a.work + it.keep + (size_t)j * KEYS * it.rows;
#pragma unroll
            for (int t = 0; t < NRT; t++) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    x[e] = s[t][e / 4][e % 4] * a.scale2;
                    const int key = k0 + e / 4 * 16 + 4 * g + e % 4;
                    if (edge && (key > hi[t] || key < lo[t])) x[e] = NEG_INF;
                }
                add_scores(ml[t], x);
                const int row = 16 * t + r;
                if (row < it.rows) {
                    *(f32x4*)(to + row * 16 + 4 * g) = f32x4{x[0], x[1], x[2], x[3]};
                    *(f32x4*)(to + (it.rows + row) * 16 + 4 * g) = f32x4{x[4], x[5], x[6], x[7]};
                }
            }
        }
        __syncthreads();  // the item before has been read
#pragma unroll
        for (int t = 0; t < NRT; t++) {
            ml[t] = merge(ml[t], shuffled(ml[t], 16));
            ml[t] = merge(ml[t], shuffled(ml[t], 32));
            if (g == 0) sml[w][16 * t + r] = ml[t];
        }
        if (threadIdx.x == 0) odd = 0;
        __syncthreads();
        const int row = threadIdx.x, there = min(it.rows, (a.rows - it.tok0) * a.group);
        if (row < 16 * NRT && row < it.rows) {
            const float2 all = merge(merge(sml[0][row], sml[1][row]), merge(sml[2][row], sml[3][row]));
            if (!it.whole) a.stats[it.stat + row] = all;
            else if (row < there) put_factor(a, all, it.head, row, f, odd);
        }
        if (!it.whole) continue;
        __syncthreads();  // (and the scores, from whichever wave)
        sum_kept(a, it.seq, it.head, it.pos0, it.k0, it.k1, it.rows, there, it.keep, it.k0, f, odd);
    }
}

// ---- many rows ----
// Both readings compute S^T[32 keys][32 rows] = K . Q^T (32x32x16): lane (r, h) has row r, keys 8c + 4h + i, so a row's statistics,
// and what turns its scores into weights, are its lane's. One side stays in registers, 32 rows or 32 keys a wave; the other comes
// by direct loads into a ring in LDS that the work-group's waves share, tiles of 32, one barrier a tile: what lands is
// waited for by each wave before the barrier, and what is overwritten behind it has been read before it. Bound by the vector
// units (an exponential, 8 cycles of a wave, and two to three others a score, in either reading) and the products, which run beside
// them only in part: a prompt of 4,096 of 32 heads on 4 x 128, 68.7 GFLOP a reading, 84 us for the statistics (0.82 PFLOP/s; without
// the exponentials 80, without the products 69) and 112 for the sums (0.61; 107 and 77).
constexpr int RING_TILES = 4;
// 64 lanes x 16 or 4 bytes from addresses of their own, to `lds` and behind
__device__ inline void dma16v(const void* src, unsigned lds) {
    asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(__builtin_amdgcn_readfirstlane(lds)) : "memory", "m0");
}
__device__ inline void dma4v(const void* src, unsigned lds) {
    asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(__builtin_amdgcn_readfirstlane(lds)) : "memory", "m0");
}
template <int N>
__device__ inline void landed() {  // but for the wave's last N direct loads
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Operands that have been loaded: the compiler waits for them here. (Where they are used, in the loop, its wait for them is one for every
// direct load on its way.)
template <typename T, int N>
__device__ inline void arrived(Vec8<T> (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
        u32x4 x = __builtin_bit_cast(u32x4, v[i]);
        asm volatile("" : "+v"(x));
        v[i] = __builtin_bit_cast(Vec8<T>, x);
    }
}

// Work-group: 128 rows, 32 a wave.
template <typename T, int D>
__global__ void __launch_bounds__(256) score_rows(Args a, const Score* __restrict__ items, const int* __restrict__ nitems) {
    constexpr int NS = D / 16, TILE = KEYS * D * 2, PER = D / 64;  // bytes of a tile; KB of it that a wave brings
    __shared__ __attribute__((aligned(1024))) unsigned char ring[RING_TILES * TILE];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, h = lane >> 5;
    const unsigned lds = (unsigned)(uintptr_t)(lds_void*)ring, voff = lane * 16;
    const int kaddr = (r >> 4) * 16 * D * 2 + h * 256 + (r & 15) * 16;
    const int count = *uniform(nitems);
    for (int n = blockIdx.x; n < count; n += gridDim.x) {
        const Score it = load_score(items + n);
        const Keys<D> keys(a, it.seq, it.head);
        const int first = it.row0 + 32 * w, row = first + r, last = min(first + 32, it.rows) - 1;
        const int blocks = (it.k1 - it.k0 + KEYS - 1) / KEYS;
        auto block = [&](int j) INLINE { return keys.block(it.k0 + KEYS * min(j, blocks - 1)); };
        auto issue = [&](int j, const char* p) INLINE {
            const unsigned to = lds + j % RING_TILES * TILE + w * PER * 1024;
#pragma unroll
            for (int i = 0; i < PER; i++) dma16s(p + (w * PER + i) * 1024, voff, to + i * 1024);
        };
        const char* next = nullptr;  // where the next block is, looked up a step ahead
        __syncthreads();  // the ring of the item before has been read
        if (blocks > 0) {
#pragma unroll
            for (int j = 0; j < RING_TILES - 1; j++) issue(j, block(j));
            next = block(RING_TILES - 1);
        }
        Vec8<T> q[NS];
        const int tok = row / a.group, head = it.head * a.group + row % a.group;
        const bool is = row < it.rows && it.tok0 + tok < a.rows;
        const int hi = is ? it.pos0 + tok : -1, lo = a.window ? it.pos0 + tok - a.window + 1 : 0;
        const T* const src = (const T*)a.q + (int64_t)(it.tok0 + tok) * a.q_tok + head * a.q_head + 8 * h;
#pragma unroll
        for (int s = 0; s < NS; s++) q[s] = is ? load8(src + 16 * s) : Vec8<T>{};
        arrived(q);
        float2 ml = make_float2(NEG_INF, 0.f);
        const int all_hi = it.pos0 + first / a.group, all_lo = a.window ? it.pos0 + last / a.group - a.window + 1 : 0;
        for (int j = 0; j < blocks; j++) {
            landed<(RING_TILES - 2) * PER>();
            lds_barrier();
            issue(j + RING_TILES - 1, next);
            next = block(j + RING_TILES);
            const unsigned char* const k = ring + j % RING_TILES * TILE + kaddr;
            f32x16 s = f32x16{};
#pragma unroll
            for (int i = 0; i < NS; i++) s = mfma32(*(const Vec8<T>*)(k + i * 512), q[i], s);
            if constexpr (NS <= 8) {  // all operands on their way at once, where there are registers for them
                __builtin_amdgcn_sched_group_barrier(0x100, NS, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, NS, 0);
            }
            const int k0 = it.k0 + KEYS * j;
            if (k0 + KEYS - 1 > all_hi || k0 < all_lo) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int key = k0 + i / 4 * 8 + 4 * h + i % 4;
                    if (key > hi || key < lo) s[i] = NEG_INF;
                }
            }
            float top = fmaxf(s[0], s[1]);  // the compiler's: it waits for the products
#pragma unroll
            for (int i = 2; i < 16; i += 2) top = vmax3(top, s[i], s[i + 1]);
            top = vmax(ml.x, top * a.scale2);
            const float ref = top == NEG_INF ? 0.f : top;
            float sum = ml.x == NEG_INF ? ml.y : ml.y * fast_exp2(ml.x - ref), more = 0.f;
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                sum += fast_exp2(__builtin_fmaf(s[i], a.scale2, -ref));
                more += fast_exp2(__builtin_fmaf(s[i + 1], a.scale2, -ref));
            }
            ml = make_float2(top, sum + more);
        }
        landed<0>();  // copies that no block needs write the ring no more behind this
        ml = merge(ml, shuffled(ml, 32));
        if (h || row >= it.rows) continue;
        if (it.whole) ml = final_of(a, ml, it.tok0, it.head, row);
        a.stats[it.stat + row - it.row0] = ml;
    }
}

// Several pieces of many rows' statistics: 16 lanes a row, 16 rows of an item a work-group, up to 8 pieces a lane on their way at
// once. Bound by latency: 512 rows of 125 pieces 3.9 us.
__global__ void __launch_bounds__(256) merge_kernel(Args a, const Merge* __restrict__ items, const int* __restrict__ nitems) {
    const int count = *uniform(nitems) * MERGE_WAYS, lane = threadIdx.x % 16;
    for (int n = blockIdx.x; n < count; n += gridDim.x) {
        const Uniform<int> u = uniform((const int*)(items + n / MERGE_WAYS));
        const Merge it{u[0], u[1], u[2], u[3], u[4], u[5], u[6], 0};
        const int row = it.r0 + n % MERGE_WAYS * 16 + (int)threadIdx.x / 16;
        float2 all = make_float2(NEG_INF, 0.f);
        for (int p0 = 0; p0 < it.pieces; p0 += 128) {
            float2 x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int p = p0 + 16 * i + lane;
                x[i] = row < it.r1 && p < it.pieces ? a.stats[it.stat + (size_t)p * it.rows + row] : make_float2(NEG_INF, 0.f);
            }
#pragma unroll
            for (int y = 4; y; y /= 2)
#pragma unroll
                for (int i = 0; i < y; i++) x[i] = merge(x[i], x[i + y]);
            all = merge(all, x[0]);
        }
#pragma unroll
        for (int i = 1; i < 16; i *= 2) all = merge(all, shuffled(all, i));
        if (lane == 0 && row < it.r1) a.stats[it.stat + row] = final_of(a, all, it.tok0, it.head, row);
    }
}

// ---- sums over few rows' kept scores ----
// Bound by the reading of the scores, from caches as far as they are there: 23 MB of 64 sequences 7.3 us.
__global__ void __launch_bounds__(256) sum_few(Args a, const Sum* __restrict__ items, const int* __restrict__ nitems) {
    __shared__ float2 f[32];
    __shared__ int odd;
    const int count = *uniform(nitems), tid = threadIdx.x;
    for (int n = blockIdx.x; n < count; n += gridDim.x) {
        const Sum it = load_sum(items + n);
        __syncthreads();  // the item before has been read
        if (tid == 0) odd = 0;
        __syncthreads();
        // 8 lanes a row
        const int row = tid / 8, rows = min(it.rows, (a.rows - it.tok0) * a.group);
        float2 s = make_float2(NEG_INF, 0.f);
        if (row < rows)
            for (int p = tid % 8; p < it.pieces; p += 8) s = merge(s, a.stats[it.stat + p * it.rows + row]);
#pragma unroll
        for (int i = 1; i < 8; i *= 2) s = merge(s, shuffled(s, i));
        if (tid % 8 == 0 && row < rows) put_factor(a, s, it.head, row, f, odd);
        __syncthreads();
        sum_kept(a, it.seq, it.head, it.pos0, it.k0, it.k1, it.rows, rows, it.scores, it.s0, f, odd);
    }
}

// ---- sums over many rows: 8 waves of 32 keys in registers, the rows through the ring ----
// A row tile lies in LDS as its operands are read, [8 dims][row][8], and its final statistics behind it. Sums over the rows stay by
// row and key in the lanes' registers until the end. (4 waves of 64 keys, some of whose registers go to memory: 235 us for both
// readings of the prompt above, against 188; the next tile's products among this one's exponentials by hand: 230.)
template <typename T, int D>
__global__ void __launch_bounds__(512) sum_rows(Args a, const Sum* __restrict__ items, const int* __restrict__ nitems) {
    constexpr int NS = D / 16, TILE = 32 * D * 2, SLOT = TILE + 256, PER = D == 64 ? 1 : D / 128;  // (heads of 64: two waves bring the same)
    __shared__ __attribute__((aligned(1024))) unsigned char ring[RING_TILES * SLOT];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), x = lane & 31, h = lane >> 5;
    const int piece0 = w * PER % (D / 16);
    const unsigned lds = (unsigned)(uintptr_t)(lds_void*)ring;
    const int count = *uniform(nitems);
    // rows go on 32 at a time: tokens and heads of the group
    const int tok_by = 32 / a.group, head_by = 32 % a.group;
    const int64_t by = tok_by * a.q_tok + head_by * a.q_head, wrap = a.q_tok - a.group * a.q_head;
    for (int n = blockIdx.x; n < count; n += gridDim.x) {
        const Sum it = load_sum(items + n);
        const Keys<D> keys(a, it.seq, it.head);
        float* const weights = a.weights + it.seq * a.seq_stride + it.head * a.stride;
        const int there = (int)min((long long)it.r1, (long long)(a.rows - it.tok0) * a.group);  // rows that the call has
        for (int k0 = it.k0; k0 < it.k1; k0 += SUM_KEYS) {
            const int first = k0 + 32 * w;  // the wave's keys; behind the last the last block again, not counted
            // the first rows that see any of these keys
            const int r0 = max(it.r0, (int)(min((long long)(k0 - it.pos0) * a.group, (long long)it.rows)) / KEYS * KEYS);
            const int tiles = max(0, (there - r0 + 31) / 32);
            int row = r0 + x, rem = row % a.group;  // of the next tile to come
            const T* const own = (const T*)a.q + it.head * a.group * a.q_head + piece0 * 16 + h * 8;
            const T* src = own + (int64_t)(it.tok0 + row / a.group) * a.q_tok + rem * a.q_head;
            const T* const q0 = own + (int64_t)(it.tok0 + r0 / a.group) * a.q_tok + r0 % a.group * a.q_head;
            auto issue = [&](int j) INLINE {  // (rows behind the last: the first again; tiles behind the last: its statistics)
                const T* const p = row < there ? src : q0;
                const unsigned to = lds + j % RING_TILES * SLOT;
#pragma unroll
                for (int i = 0; i < PER; i++) dma16v(p + i * 16, to + (piece0 + i) * 1024);
                dma4v((const float*)(a.stats + it.stat + r0 + 32 * min(j, tiles - 1)) + lane, to + TILE);
                row += 32;
                rem += head_by;
                src += by;
                if (rem >= a.group) {
                    rem -= a.group;
                    src += wrap;
                }
            };
            __syncthreads();  // the ring before has been read
            if (tiles > 0)
#pragma unroll
                for (int j = 0; j < RING_TILES - 1; j++) issue(j);
            Vec8<T> k[NS];
            const char* const kp = keys.block(min(first, (it.k1 - 1) / KEYS * KEYS)) + (x >> 4) * 16 * D * 2 + h * 256 + (x & 15) * 16;
#pragma unroll
            for (int s = 0; s < NS; s++) k[s] = load8((const T*)(kp + s * 512));
            arrived(k);
            f32x16 sum = f32x16{};
            for (int j = 0; j < tiles; j++) {
                landed<(RING_TILES - 2) * (PER + 1)>();
                lds_barrier();
                issue(j + RING_TILES - 1);
                const unsigned char* const slot = ring + j % RING_TILES * SLOT;
                const float2 f = ((const float2*)(slot + TILE))[x];
                f32x16 s = f32x16{};
#pragma unroll
                for (int i = 0; i < NS; i++) s = mfma32(k[i], *(const Vec8<T>*)(slot + (2 * i + h) * 512 + x * 16), s);
                const int at = r0 + 32 * j;
                const int low = it.pos0 + at / a.group, high = it.pos0 + (at + 31) / a.group;
                if (at + 32 > there || first + 31 > low || (a.window && first < high - a.window + 1)) {
                    // the lane's keys as seen from the last that its row sees, in [0, span): one comparison each
                    const int pos = at + x < there ? it.pos0 + (at + x) / a.group : -1;
                    const unsigned span = pos < 0 ? 0 : a.window ? a.window : pos + 1;
                    int back = pos - first - 4 * h;
                    asm volatile("" : "+v"(back));  // (here: the keys in registers through the loop otherwise)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float y = fast_exp2(__builtin_fmaf(s[i], a.scale2, -f.x)) * f.y;
                        if ((unsigned)(back - i / 4 * 8 - i % 4) < span) sum[i] += y;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i++) sum[i] = __builtin_fmaf(fast_exp2(__builtin_fmaf(s[i], a.scale2, -f.x)), f.y, sum[i]);
                }
            }
            landed<0>();  // copies that no tile needs write the ring no more behind this
            __syncthreads();
            float* const sums = (float*)ring;  // of the work-group's keys
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float y = reduce16(sum[i], [](float p, float q) { return p + q; });
                y += __shfl_xor(y, 16);
                if (x == 0) sums[32 * w + i / 4 * 8 + 4 * h + i % 4] = y;
            }
            __syncthreads();
            const int key = k0 + (int)threadIdx.x;
            if (threadIdx.x < SUM_KEYS && key < it.k1) {
                const float y = sums[threadIdx.x];
                if (it.part >= 0) a.work[it.part + key - it.k0] = y;
                else weights[key] = (a.decay == 0.f ? 0.f : a.decay * weights[key]) + y;
            }
        }
    }
}

// ---- weights that fade, and partial sums that join them: bound by latency, 4.7 us of the prompt's 4 x 4,096 positions ----
__global__ void __launch_bounds__(256) fade_kernel(Args a, const Fade* __restrict__ items, const int* __restrict__ nitems) {
    const int count = *uniform(nitems);
    for (int n = blockIdx.x; n < count; n += gridDim.x) {
        const Uniform<int> u = uniform((const int*)(items + n));
        const Fade it{u[0], u[1], u[2], u[3], u[4], u[5], u[6], 0};
        if (!it.sums && a.decay == 1.f) continue;
        float* const weights = a.weights + it.seq * a.seq_stride + it.head * a.stride;
        for (int key = it.k0 + threadIdx.x; key < it.k1; key += 256) {
            const float* const p = a.work + it.part + key - it.k0;
            float sum = 0.f;
#pragma unroll 8
            for (int s = 0; s < it.sums; s++) sum += p[(size_t)s * it.stride];
            weights[key] = (a.decay == 0.f ? 0.f : a.decay * weights[key]) + sum;
        }
    }
}

// ---- weights of positions that are new, or another sequence's: 20 x 65,536 copied in 4.7 us ----
constexpr int CHANGES = 128;  // of a launch, in its arguments
struct ChangeList {
    Change c[CHANGES];
};
constexpr int SPAN = 4096;  // positions of a work-group, 16 a thread
template <bool COPY>
__global__ void __launch_bounds__(256) change_kernel(WeightsAt w, ChangeList list, int n, int spans, size_t all) {
    for (size_t i = blockIdx.x; i < all; i += gridDim.x) {  // (layer and head, change, span)
        const int span = (int)(i % spans), c = (int)(i / spans % n);
        const size_t unit = i / spans / n;
        const int layer = (int)(unit / w.kv_heads), head = (int)(unit % w.kv_heads);
        const Change x = list.c[c];
        float* const p = w.p + w.at(layer, x.seq, head) + x.a;
        const float* const from = COPY ? w.p + w.at(layer, x.other, head) + x.a : nullptr;
        const int first = span * SPAN, end = min(x.count, first + SPAN);
        if (x.a % 4 == 0 && end - first == SPAN) {  // whole, 16 bytes a time
            f32x4 y[4];
#pragma unroll
            for (int j = 0; j < 4; j++) y[j] = COPY ? ((const f32x4*)(from + first))[threadIdx.x + 256 * j] : f32x4{};
#pragma unroll
            for (int j = 0; j < 4; j++) ((f32x4*)(p + first))[threadIdx.x + 256 * j] = y[j];
        } else {
#pragma unroll 4
            for (int j = first + threadIdx.x; j < end; j += 256) p[j] = COPY ? from[j] : 0.f;
        }
    }
}

// ---- eviction ----
constexpr int EVICTIONS = 128, NEW_PAGES = 480;  // of a launch, in its arguments (4 KB)
struct EvictionList {
    Eviction e[EVICTIONS];
};
// a new page: 27 bits of page and 5 of the entry's, 11 more and 17 of which page of the sequence it is (the limits of mpg_create)
struct PageList {
    unsigned p[NEW_PAGES][2];
};

typedef int i32x4 __attribute__((ext_vector_type(4)));

// Weights in an order of whole numbers, from 0x7FFFFF on; NaN weighs most, both zeros the same.
__device__ inline unsigned order_of(float x) {
    if (x != x) return ~0u;
    const unsigned u = __float_as_uint(x == 0.f ? 0.f : x);
    return u >> 31 ? ~u : u | 0x80000000u;
}

__device__ inline float weight_of(unsigned x) { return __uint_as_float(x >> 31 ? x & 0x7FFFFFFF : ~x); }
__device__ inline int before_lane(unsigned long long lanes) {  // how many of them lie below this one
    return __builtin_amdgcn_mbcnt_hi((unsigned)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)lanes, 0));
}

// The picks of one sequence, layer and head by a work-group: the least weight that stays, by digits of 11, 11 and 10 bits from the
// highest on, then the positions in order; of those with just that weight the first ones. 65,536 weights stay in registers from one
// reading to the next, four neighbours a thread and 4,096; longer sequences are read again for each. Each digit is counted in four
// places by lane: weights are of few magnitudes, and lanes that count the same wait for each other. Bound by latency, barriers and
// these counts: 20 x 65,536 43 us (counted in one place, with sums over the lanes for the kept ones' places, 62), 2,000 9.4.
constexpr int GROUP = 16, PICKED = 4096 * GROUP, COUNTED = 4;
__global__ void __launch_bounds__(1024) pick_kernel(WeightsAt w, EvictionList list, int n, int entry0, int first, int recent,
                                                    Eviction* __restrict__ entries, int* __restrict__ picks, float* __restrict__ kept,
                                                    size_t stride, int units) {
    // (at most EVICTIONS x 2^22 pairs of a sequence and a layer's head)
    __shared__ __attribute__((aligned(16))) int hist[2048 * COUNTED];
    __shared__ int waves[16];
    __shared__ int2 before_of[GROUP * 16];  // tile by tile, of each wave: heavier ones before it, ones of the least weight
    __shared__ int found[3];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int b = blockIdx.x; b < n * units; b += gridDim.x) {
        const int c = b / units, unit = b % units;
        const Eviction e = list.e[c];
        if (unit == 0 && tid == 0) entries[entry0 + c] = e;
        int* const to = picks + (size_t)unit * stride + e.off;
        float* const heavy = kept + (size_t)unit * stride + e.off;
        const float* const src = w.p + w.at(unit / w.kv_heads, e.seq, unit % w.kv_heads);
        const int lo = first, hi = e.len - recent, want = e.keep - first - recent;
        auto pick = [&](int k, int i, float x) INLINE {
            to[k] = i;
            heavy[k] = x;
        };
        for (int i = tid; i < first; i += 1024) pick(i, i, src[i]);
#pragma unroll 4
        for (int i = tid; i < recent; i += 1024) pick(e.keep - recent + i, hi + i, src[hi + i]);
        if (!want) continue;
        unsigned v[GROUP][4];
        auto bring = [&](int g0) INLINE {  // positions g0 .. g0 + PICKED - 1 (rows are whole runs of 32); 0 for what is not in [lo, hi)
#pragma unroll
            for (int t = 0; t < GROUP; t++) {
                const int i = g0 + 4096 * t + 4 * tid;
                if (g0 + 4096 * t >= hi) break;
                f32x4 x = f32x4{};
                if (i < hi) x = *(const f32x4*)(src + i);
#pragma unroll
                for (int y = 0; y < 4; y++) v[t][y] = i + y >= lo && i + y < hi ? order_of(x[y]) : 0;
            }
        };
        unsigned known = 0, mask = 0;  // the digits of the least weight that stays
        int left = want;               // of those that have them
        bring(0);
        for (int shift = 21; shift >= 0; shift = shift ? max(0, shift - 11) : -1) {  // 21, 10, 0: of 11, 11 and 10 bits
            const unsigned digit = shift ? 2047 : 1023;
            __syncthreads();
#pragma unroll
            for (int x = 0; x < 2; x++) ((i32x4*)hist)[tid + 1024 * x] = i32x4{};
            __syncthreads();
            for (int g0 = 0; g0 < hi; g0 += PICKED) {
                if (hi > PICKED) bring(g0);
#pragma unroll
                for (int t = 0; t < GROUP; t++) {
                    if (g0 + 4096 * t >= hi) break;
#pragma unroll
                    for (int y = 0; y < 4; y++)
                        if (v[t][y] && (v[t][y] & mask) == known)
                            atomicAdd(&hist[(v[t][y] >> shift & digit) * COUNTED + lane % COUNTED], 1);
                }
            }
            __syncthreads();
            // from the highest digit down: thread t has digits 2047 - 2 t and 2046 - 2 t
            auto counted = [&](int d) INLINE {
                const i32x4 x = ((const i32x4*)hist)[d];
                return x[0] + x[1] + x[2] + x[3];
            };
            const int h0 = counted(2047 - 2 * tid), h1 = counted(2046 - 2 * tid);
            int before = h0 + h1;
#pragma unroll
            for (int x = 1; x < 64; x *= 2) {
                const int y = __shfl_up(before, x);
                if (lane >= x) before += y;
            }
            if (lane == 63) waves[wave] = before;
            __syncthreads();
            before -= h0 + h1;
#pragma unroll
            for (int x = 0; x < 15; x++) {
                const int y = waves[x];
                if (x < wave) before += y;
            }
            if (before < left && before + h0 >= left) {
                found[0] = 2047 - 2 * tid;
                found[1] = left - before;
                found[2] = h0;
            } else if (before + h0 < left && before + h0 + h1 >= left) {
                found[0] = 2046 - 2 * tid;
                found[1] = left - before - h0;
                found[2] = h1;
            }
            __syncthreads();
            known |= (unsigned)__builtin_amdgcn_readfirstlane(found[0]) << shift;
            mask |= digit << shift;
            left = __builtin_amdgcn_readfirstlane(found[1]);
            if (left == __builtin_amdgcn_readfirstlane(found[2])) {  // all with these digits stay, whatever the others: those above the number below
                known--;
                left = 0;
                break;
            }
        }
        // left: how many of those with just the least weight stay (no weight's number is 0: `known` never went below)
        int2 all = make_int2(0, 0);  // before the tiles: heavier ones, ones of the least weight
        for (int g0 = 0; g0 < hi; g0 += PICKED) {
            if (hi > PICKED) bring(g0);
            if (wave == 0)
#pragma unroll
                for (int x = 0; x < GROUP / 4; x++) before_of[lane + 64 * x] = make_int2(0, 0);
            __syncthreads();
#pragma unroll
            for (int t = 0; t < GROUP; t++) {
                if (g0 + 4096 * t >= hi) break;
                int2 mine = make_int2(0, 0);
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    mine.x += __popcll(__ballot(v[t][y] > known));
                    mine.y += __popcll(__ballot(v[t][y] == known));
                }
                if (lane == 0) before_of[16 * t + wave] = mine;
            }
            __syncthreads();
            // every wave adds up all 256 itself, four a lane, and takes its own
            int2 four[4], sum = make_int2(0, 0);
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int2 y = before_of[4 * lane + x];
                four[x] = sum;
                sum = make_int2(sum.x + y.x, sum.y + y.y);
            }
            int2 upto = sum;
#pragma unroll
            for (int x = 1; x < 64; x *= 2) {
                const int y = __shfl_up(upto.x, x), z = __shfl_up(upto.y, x);
                if (lane >= x) upto = make_int2(upto.x + y, upto.y + z);
            }
            const int2 start = make_int2(all.x + upto.x - sum.x, all.y + upto.y - sum.y);
            const int x_of = wave % 4;
            const int2 own = make_int2(start.x + (x_of == 0 ? four[0].x : x_of == 1 ? four[1].x : x_of == 2 ? four[2].x : four[3].x),
                                       start.y + (x_of == 0 ? four[0].y : x_of == 1 ? four[1].y : x_of == 2 ? four[2].y : four[3].y));
            asm volatile("" : "+s"(known));  // (compared anew: the lanes' answers of all tiles do not fit in registers)
#pragma unroll
            for (int t = 0; t < GROUP; t++) {
                if (g0 + 4096 * t >= hi) break;
                const int i0 = g0 + 4096 * t + 4 * tid, from = 4 * t + wave / 4;  // the lane that has the wave's
                int m = __builtin_amdgcn_readlane(own.x, from), s = __builtin_amdgcn_readlane(own.y, from);
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    m += before_lane(__ballot(v[t][y] > known));
                    s += before_lane(__ballot(v[t][y] == known));
                }
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    if (v[t][y] > known) pick(first + m++ + min(s, left), i0 + y, weight_of(v[t][y]));
                    else if (v[t][y] == known) {
                        if (s < left) pick(first + m + s, i0 + y, weight_of(v[t][y]));
                        s++;
                    }
                }
            }
            all = make_int2(all.x + __builtin_amdgcn_readlane(upto.x, 63), all.y + __builtin_amdgcn_readlane(upto.y, 63));
            __syncthreads();
        }
    }
}

// A new page's block of 32 positions of a head and layer, K or V: 16 bytes of K a thread (8 dims of a position), 16 bytes of V
// (a dim of 8 positions, which come from 8 places), all on their way at once; `parts` work-groups share a block's dims where blocks are
// few. Positions behind the last that stays are left as they were. Bound by memory, which gives whole lines: 128 bytes are 8
// positions of 8 dims of K, or 8 dims of 8 positions of V, so that of a sequence cut to a quarter nearly all lines are read: 65,536
// to 16,384 of 10 layers of 2 x 256 280 us, 335 MB written and 1.16 GB read, 5.35 TB/s. K comes past the caches (nothing else is
// in its lines that another work-group takes; through them 0.7% slower); V through them, a line serves 4 loads of a wave (past
// them 12% slower).
template <int D>
__global__ void __launch_bounds__(256) gather_kernel(unsigned short* __restrict__ pool, const int* __restrict__ table, int most_pages,
                                                     int page, int kv_heads, int units, size_t plane,
                                                     const Eviction* __restrict__ entries, const int* __restrict__ picks,
                                                     size_t stride, int parts, PageList list) {
    constexpr int ROUNDS = D / 64;  // of 256 units of 16 bytes
    __shared__ size_t from[KEYS];
    __shared__ int in[KEYS];
    typedef Vec8<unsigned short> Unit;
    const int tid = threadIdx.x, blocks = page / KEYS;
    const unsigned n0 = list.p[blockIdx.x / blocks][0], n1 = list.p[blockIdx.x / blocks][1];
    const NewPage np{(int)(n0 >> 27 | (n1 & 0x7FF) << 5), (int)(n1 >> 11), (int)(n0 & 0x7FFFFFF)};
    const int block = blockIdx.x % blocks, part = blockIdx.z / 2;
    const bool is_v = blockIdx.z % 2;
    const Eviction e = entries[np.entry];
    const int p0 = np.nth * page + block * KEYS, count = min(KEYS, e.keep - p0);
    if (count <= 0) return;
    for (int unit = blockIdx.y; unit < units; unit += gridDim.y) {
        const int head = unit % kv_heads, layer = unit / kv_heads;
        unsigned short* const base = pool + ((size_t)layer * 2 + is_v) * plane;
        __syncthreads();  // the places before have been read
        if (tid < count) {
            const int p = picks[(size_t)unit * stride + e.off + p0 + tid];
            from[tid] = ((size_t)table[(size_t)e.seq * most_pages + p / page] * kv_heads + head) * page * D + (size_t)(p % page / KEYS) * KEYS * D;
            in[tid] = p % KEYS;
        }
        __syncthreads();
        unsigned short* const to = base + ((size_t)np.page * kv_heads + head) * page * D + (size_t)block * KEYS * D;
        if (!is_v) {
            const int x = tid % KEYS;
            if (x >= count) continue;
            const int y = in[x];
            const unsigned short* const s = base + from[x] + y / 16 * 16 * D + y % 16 * 8;
            unsigned short* const t = to + x / 16 * 16 * D + x % 16 * 8;
            Unit u[ROUNDS];
#pragma unroll
            for (int i = 0; i < ROUNDS; i++)
                if (i % parts == part) u[i] = __builtin_nontemporal_load((const Unit*)(s + (tid / KEYS + 8 * i) * 128));
#pragma unroll
            for (int i = 0; i < ROUNDS; i++)
                if (i % parts == part) *(Unit*)(t + (tid / KEYS + 8 * i) * 128) = u[i];
            continue;
        }
        // (a round is 256 units: of heads of 256 one group of positions, of 128 two, of 64 all four)
        Unit u[ROUNDS];
#pragma unroll
        for (int i = 0; i < ROUNDS; i++) {
            if (i % parts != part) continue;
            const int g = (tid + 256 * i) / D, d = (tid + 256 * i) % D;
#pragma unroll
            for (int z = 0; z < 8; z++) {
                const int x = min(16 * (z / 4) + 4 * g + z % 4, count - 1), y = in[x];
                u[i][z] = base[from[x] + (y % 16 / 4 * D + d) * 8 + y / 16 * 4 + y % 4];
            }
        }
#pragma unroll
        for (int i = 0; i < ROUNDS; i++) {
            if (i % parts != part) continue;
            const int g = (tid + 256 * i) / D;
            unsigned short* const o = to + (tid + 256 * i) * 8;
            if (16 + 4 * g + 3 < count) {
                *(Unit*)o = u[i];
            } else {
#pragma unroll
                for (int z = 0; z < 8; z++)
                    if (16 * (z / 4) + 4 * g + z % 4 < count) o[z] = u[i][z];
            }
        }
    }
}

// The weights that stay, from where the picks have put them: 20 x 16,384 5 us. (Gathered by position, in place, 14.5.)
__global__ void __launch_bounds__(256) pack_kernel(WeightsAt w, const Eviction* __restrict__ entries, const float* __restrict__ kept,
                                                   size_t stride, size_t all, int units) {
    for (size_t b = blockIdx.x; b < all; b += gridDim.x) {
        const int unit = (int)(b % units);
        const Eviction e = entries[b / units];
        float* const p = w.p + w.at(unit / w.kv_heads, e.seq, unit % w.kv_heads);
        const float* const from = kept + (size_t)unit * stride + e.off;
#pragma unroll 4
        for (int i = blockIdx.y * 256 + threadIdx.x; i < e.keep; i += gridDim.y * 256) p[i] = from[i];
    }
}

template <typename T, int D>
hipError_t weigh_as(const Args& a, const int* batch, const WeighLists& l, const int* grid, hipStream_t s) {
    hipError_t e = hipSuccess;
    auto go = [&](auto kernel, int list, auto* items, int threads = 256) {
        if (!grid[list] || e != hipSuccess) return;
        kernel<<<dim3(grid[list]), dim3(threads), 0, s>>>(a, items, batch + list);
        e = hipGetLastError();
    };
    go(score_few<T, D, 1>, SCORE_FEW, (const Score*)(batch + l.at[SCORE_FEW]));
    go(score_few<T, D, 2>, SCORE_SOME, (const Score*)(batch + l.at[SCORE_SOME]));
    go(score_rows<T, D>, SCORE_MANY, (const Score*)(batch + l.at[SCORE_MANY]));
    go(merge_kernel, MERGES, (const Merge*)(batch + l.at[MERGES]));
    go(sum_few, SUM_FEW, (const Sum*)(batch + l.at[SUM_FEW]));
    go(sum_rows<T, D>, SUM_MANY, (const Sum*)(batch + l.at[SUM_MANY]), 512);
    go(fade_kernel, FADES, (const Fade*)(batch + l.at[FADES]));
    return e;
}

template <typename T>
hipError_t weigh_dim(int dim, const Args& a, const int* batch, const WeighLists& l, const int* grid, hipStream_t s) {
    return dim == 64    ? weigh_as<T, 64>(a, batch, l, grid, s)
           : dim == 128 ? weigh_as<T, 128>(a, batch, l, grid, s)
                        : weigh_as<T, 256>(a, batch, l, grid, s);
}

template <bool COPY>
hipError_t change(const WeightsAt& w, const Change* c, int n, hipStream_t s) {
    for (int i = 0; i < n; i += CHANGES) {
        ChangeList list;
        const int m = std::min(CHANGES, n - i);
        int most = 0;
        for (int j = 0; j < CHANGES; j++) list.c[j] = j < m ? c[i + j] : Change{0, 0, 0, 0};
        for (int j = 0; j < m; j++) most = std::max(most, c[i + j].count);
        const int spans = (most + SPAN - 1) / SPAN;
        const size_t all = (size_t)w.layers * w.kv_heads * m * spans;
        change_kernel<COPY><<<dim3((unsigned)std::min<size_t>(all, MOST_GRID)), dim3(256), 0, s>>>(w, list, m, spans, all);
        if (const hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_clear(const WeightsAt& w, const Change* c, int n, hipStream_t s) { return change<false>(w, c, n, s); }
hipError_t launch_weights_copy(const WeightsAt& w, const Change* c, int n, hipStream_t s) { return change<true>(w, c, n, s); }

hipError_t launch_weigh(const Geometry& g, const WeightsAt& w, const WeighArgs& x, const int* batch, const WeighLists& l,
                        const int* grid, hipStream_t s) {
    Args a;
    a.table = x.table;
    a.most_pages = g.most_pages;
    a.page = g.page;
    a.page_shift = __builtin_ctz(g.page);
    a.kv_heads = g.kv_heads;
    a.group = g.q_heads / g.kv_heads;
    a.window = x.window;
    a.rows = x.rows;
    a.kpool = x.pool + (size_t)x.layer * 2 * g.plane_elems() * 2;
    a.q = x.q.p;
    a.q_tok = x.q.tok;
    a.q_head = x.q.head;
    a.sinks = x.sinks;
    a.scale2 = x.scale * LOG2E;
    a.decay = x.decay;
    a.stats = (float2*)x.stats;
    a.work = x.work;
    a.weights = w.p + w.at(x.layer, 0, 0);
    a.stride = w.stride;
    a.seq_stride = w.stride * w.kv_heads;
    return g.fmt == MKV_F16 ? weigh_dim<_Float16>(g.head_dim, a, batch, l, grid, s) : weigh_dim<__bf16>(g.head_dim, a, batch, l, grid, s);
}

hipError_t launch_pick(const Geometry& g, const WeightsAt& w, const Eviction* e, int n, int first, int recent, Eviction* entries,
                       int* picks, float* kept, size_t stride, hipStream_t s) {
    const int units = g.layers * g.kv_heads;
    for (int i = 0; i < n; i += EVICTIONS) {
        EvictionList list;
        const int m = std::min(EVICTIONS, n - i);
        for (int j = 0; j < EVICTIONS; j++) list.e[j] = j < m ? e[i + j] : Eviction{0, 0, 0, 0};
        pick_kernel<<<dim3((unsigned)std::min<long long>((long long)m * units, MOST_GRID)), dim3(1024), 0, s>>>(w, list, m, i, first, recent, entries,
                                                                                                    picks, kept, stride, units);
        if (const hipError_t err = hipGetLastError()) return err;
    }
    return hipSuccess;
}

hipError_t launch_gather(const Geometry& g, char* pool, const int* table, const Eviction* entries, const int* picks, size_t stride,
                         const NewPage* pages, int n, hipStream_t s) {
    const auto kernel = g.head_dim == 64 ? gather_kernel<64> : g.head_dim == 128 ? gather_kernel<128> : gather_kernel<256>;
    for (int i = 0; i < n; i += NEW_PAGES) {
        PageList list;
        const int m = std::min(NEW_PAGES, n - i);
        for (int j = 0; j < NEW_PAGES; j++) {
            const NewPage np = j < m ? pages[i + j] : NewPage{0, 0, 0};
            list.p[j][0] = (unsigned)np.page | (unsigned)np.entry << 27;
            list.p[j][1] = (unsigned)np.entry >> 5 | (unsigned)np.nth << 11;
        }
        const int units = g.layers * g.kv_heads;
        const long long groups = (long long)n * (g.page / KEYS) * units * 2;
        const int parts = groups >= 2048 ? 1 : std::min(g.head_dim / 64, groups >= 1024 ? 2 : 4);
        kernel<<<dim3(m * (g.page / KEYS), std::min(units, 1024), 2 * parts), dim3(256), 0, s>>>(
            (unsigned short*)pool, table, g.most_pages, g.page, g.kv_heads, units, g.plane_elems(), entries, picks, stride, parts, list);
        if (const hipError_t err = hipGetLastError()) return err;
    }
    return hipSuccess;
}

hipError_t launch_pack(const WeightsAt& w, const Eviction* entries, int n, int longest, const float* kept, size_t stride, hipStream_t s) {
    const int units = w.layers * w.kv_heads;
    const size_t all = (size_t)n * units;
    pack_kernel<<<dim3((unsigned)std::min<size_t>(all, MOST_GRID / 64), std::min((longest + 1023) / 1024, 64)), dim3(256), 0, s>>>(
        w, entries, kept, stride, all, units);
    return hipGetLastError();
}

}  // namespace paged
}  // namespace mkv

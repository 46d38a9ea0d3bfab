// q38b_attention.cu -- attention of a chunk of new tokens over a paged cache.
//
//   out[i][h] = sum_j softmax_j(scale q[i][h] . k[j][h / G]) v[j][h / G],  j <= length - new + i
//
// One pass over the keys with the running maximum m and sum l of a softmax.  The (token, head) pairs that read one key head of one sequence are the rows
// of a tile (128, or 256 in two), so that a group's heads and a chunk's tokens share what is read of the cache; 128 keys at a time:
//   S = Q K^T       tcgen05.mma, both operands in shared memory, 128 fp32 columns of tensor memory
//   P = 2^(S c - m) by a warpgroup, a thread a row, rounded to the cache's type and written over S; c = scale log2(e).  S has two places, for which two warpgroups take turns
//   O += P V        tcgen05.mma with P from tensor memory and V as it lies (its keys are the rows of an MN-major operand)
// The maximum that is taken off lags behind the true one by up to 2^8: O is rescaled in tensor memory only where a row's maximum has grown by
// more, which after the first tiles of a text is rare.  fp16 weights carry a factor of 2^7 (they end at 2^15), so that what is 2^-31 of the largest
// still counts; bf16 weights one of 2^-8 (they end at 1).
//
// The work is cut for all SMs whatever the batch is: tiles in the order (sequence, key head, rows), each of as many units as it sees tiles of keys, lie one behind the
// other and every CTA takes an equal range of the units, worked out on the device from the lengths, begins and table as they are when the kernel runs.  A tile of rows that
// two or more CTAs share leaves its sums in the work area, and a second kernel joins them, always in the same order.
//
// Three variants of one kernel.  Few rows: a CTA by itself; keys and values stream (32 sequences of 1600 to 32000 tokens, 24 + 4 heads of 256, a token each: 367 us = 6.5 TB/s).  Where
// no sequence has more than 8 rows a key head (the kernel finds out when it runs), the products are the warps' own: few_rows() below.
// Many rows: two tiles of 128 rows in a CTA (heads of at most 128 elements), whose keys and values then cross shared memory once; for heads of 193 to 256 a pair of CTAs that
// multiply as one (cta_group::2), each with half of the keys of a tile and half of the values' columns: one CTA by itself moves 128 KB into shared memory for 128 keys and
// the tensor core reads 192 KB of it, 2560 clocks at 128 bytes where the products need 2048 (measured 2700), the pair moves and reads half as much (4096 tokens behind 28672:
// 2.61 -> 2.26 ms, 1370 TFLOP/s; in calls one behind the other, at the power limit, 2.70 ms, 1145).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <type_traits>

#include "q38b_cache.cuh"
#include "q38b_internal.h"
#include "q38b_pipe.cuh"
#include "q38b_types.cuh"
#include "q38b_umma.cuh"

using namespace q38b;

namespace {

constexpr int KEYS = 128;                // keys of a tile
constexpr int BLOCK_BYTES = KEYS * 128;  // 64 elements of 128 rows, 128-byte swizzle
constexpr int HEAD = 3 * 1024;               // shared memory in front of the queries: barriers, the plan, maxima and sums of rows (no more, or D = 256 has a stage less)
constexpr int FEW = 8;                  // rows of a sequence and key head up to which few_rows() is taken
constexpr float GROWTH = 8.0f;           // how far, in powers of two, a row's maximum may grow before O is rescaled

// A tile of rows that several CTAs share, as the one that begins it leaves it for the joining kernel
struct Job { int n_parts, first, past, kv, row0, rows, pad[2]; };

struct AttnArgs {
    Batch batch;
    const void *q, *v;
    void* out;
    float* lse;
    float* slots;
    Job* jobs;
    int* status;
    long long q_row, q_head, out_row, out_head, v_page, v_slot, v_head;
    const void* k;
    long long k_page, k_slot, k_head;
    int q_kind, out_kind, n_heads, n_kv, group, D, box_rows, slot_rows, q_vec, out_vec, pdl;
    float c;       // scale log2(e)
    uint32_t group_mul;   // x / group = x group_mul >> group_shift for 0 <= x < 2^31
    int group_shift, ctas, q_shift, out_shift;   // log2 of the bytes of an element
};
__device__ __forceinline__ int by_group(const AttnArgs& a, int x) { return (int)((uint64_t)(uint32_t)x * a.group_mul >> a.group_shift); }

// Shapes of a variant: heads padded to DP elements, QT tiles of 128 rows, or PAIR: two CTAs that multiply as one, each with 128 of 256 rows, half of the keys of
// a tile and half of the values' columns
template <int DP, int QT, bool PAIR>
struct Shape {
    static constexpr int CW = DP % 128 == 0 ? 128 : 64;        // elements of a stage: 128 keys x CW (PAIR: 64 keys x DP, 128 values x DP / 2)
    static constexpr int NCH = PAIR ? 1 : DP / CW;             // stages of a tile of keys (or of values)
    static constexpr int STAGE = KEYS * CW * 2;
    static constexpr int Q_BYTES = QT * 128 * DP * 2;
    static constexpr int ROOM = (232448 - HEAD - Q_BYTES) / STAGE;
    static constexpr int STAGES = ROOM < 12 ? ROOM : 12;
    static constexpr int SMEM = HEAD + Q_BYTES + STAGES * STAGE;
    static constexpr int ROWS = (PAIR ? 2 : QT) * 128;
    static constexpr int THREADS = 384;                       // warps 0, 2, 3 load, warp 1 multiplies, two warpgroups make weights
    static_assert(256 + QT * DP <= 512 && (!PAIR || (QT == 1 && DP == 256)), "tensor memory; halves of whole blocks");
};

// positions of a tile's stages in the ring, in stages behind the item's first: in the order in which the tensor core takes them
template <int QT, int NCH> __device__ __forceinline__ uint32_t at_keys(int j) { return (uint32_t)((QT == 2 || j == 0 ? 2 * j : 2 * j - 1) * NCH); }
template <int QT, int NCH> __device__ __forceinline__ uint32_t at_values(int j, int n) { return (uint32_t)((QT == 2 || j == n - 1 ? 2 * j + 1 : 2 * j + 2) * NCH); }

// Boxes of a stage, `wide` elements of keys or values a row in pages of which a box takes box_rows slots, and the warps that load them: warp w of three takes boxes w, w + 3 ..  One
// that has none must not follow the ring: nothing waits for it, so it could miss a stage's phase and wait for one that does not come.
__host__ __device__ constexpr int stage_boxes(int box_rows, int wide) { return KEYS / box_rows * (wide / 64); }
__host__ __device__ constexpr int loading_warps(int boxes) { return boxes < 3 ? boxes : 3; }

// The walk of a CTA through its range of units.
struct Walk {
    int s, first, n_new, past, kv, tile, n_tiles;   // where it is: sequence, its rows and the tokens in front of them (negative: rows in front of the text), ..
    int row0, rows, seen, units;                   // of the tile of rows: first of the sequence's (token, head) rows, how many, keys the last of them sees, tiles of keys
    int from, to;                                  // of those, this CTA's
};
template <int ROWS>
__device__ __forceinline__ void walk_sequence(const AttnArgs& a, Walk& w) {
    const int next = a.batch.first(w.s + 1);
    w.first = a.batch.first(w.s);
    w.n_new = max(min(next, a.batch.rows) - w.first, 0);
    w.past = a.batch.length(w.s) - max(next - w.first, 0);   // (whether the call has all of the sequence's rows or not)
    w.n_tiles = (w.n_new * a.group + ROWS - 1) / ROWS;
}
template <int ROWS>
__device__ __forceinline__ int tile_seen(const AttnArgs& a, const Walk& w, int tile) {
    const int last = by_group(a, min((tile + 1) * ROWS, w.n_new * a.group) - 1);   // token
    return max(0, w.past + last + 1);
}
__device__ __forceinline__ int tile_units(int seen) { return max(1, (seen + KEYS - 1) / KEYS); }   // (a tile that sees nothing is one, too: its zeros are written)
// A tile of rows costs what it sees and a start (queries, first scores, outputs: 5900 to 9900 clocks where a tile of keys takes 2200 to 3600): three tiles of keys more, which
// lie in front of its first.  Without them 2048 tokens of a fresh text, whose first rows see little, were 103 us (one CTA with ten tiles of rows took 1.7 of the average's time).
constexpr int START = 3;
template <int ROWS>
__device__ __forceinline__ void walk_tile(const AttnArgs& a, Walk& w) {
    w.row0 = w.tile * ROWS;
    w.rows = min(ROWS, w.n_new * a.group - w.row0);
    w.seen = tile_seen<ROWS>(a, w, w.tile);
    w.units = tile_units(w.seen);
}
// the tile of rows behind this one; false: there is none
template <int ROWS>
__device__ __forceinline__ bool walk_on(const AttnArgs& a, Walk& w) {
    if (++w.tile == w.n_tiles) {
        w.tile = 0;
        if (++w.kv == a.n_kv) {
            w.kv = 0;
            do {
                if (++w.s >= a.batch.n_seqs) return false;
                walk_sequence<ROWS>(a, w);
            } while (w.n_tiles == 0);
        }
    }
    walk_tile<ROWS>(a, w);
    w.from = 0;
    return true;
}
// how far the CTA goes in the tile of rows where it is; `left`: units of its range that remain, starts included
__device__ __forceinline__ void walk_to(Walk& w, int& left) {
    if (w.from == 0) left -= START;
    w.to = min(w.units, w.from + left);
    left -= w.to - w.from;
}
// on to the next tile of rows.  false: none
template <int ROWS>
__device__ __forceinline__ bool walk_next(const AttnArgs& a, Walk& w, int& left) {
    if (left <= 0 || !walk_on<ROWS>(a, w)) return false;
    walk_to(w, left);
    return true;
}

// A part of a tile of rows that others finish costs about as much as a tile of keys for every 32 of its rows (its sums go out to memory and come back).  So a range that
// would begin or end within that of a tile's ends begins or ends there instead (5 sequences of 77 to 333 new tokens, 15 + 5 heads of 96: 56 us cut exactly, 39 so).
template <int DP> __device__ __forceinline__ int dear(const Walk& w) { return w.rows * DP / 8192; }
template <int DP>
__device__ __forceinline__ int moved_cut(const Walk& w, int in) {   // a cut `in` units behind the first of a tile's
    if (in > dear<DP>(w) && w.units - in > dear<DP>(w)) return in;
    return 2 * in <= w.units ? 0 : w.units;
}

// keys that all of a tile's rows see
__device__ __forceinline__ int least_seen(const AttnArgs& a, const Walk& w) { return max(0, w.past + by_group(a, w.row0) + 1); }

// Units of one key head of a sequence, by one thread or by the lanes of a warp together
template <int ROWS>
__device__ __forceinline__ int sequence_units(const AttnArgs& a, const Walk& w, int lane, int lanes) {
    int n = 0;
#pragma unroll 1
    for (int t = lane; t < w.n_tiles; t += lanes) n += START + tile_units(tile_seen<ROWS>(a, w, t));
    return n;
}

struct Plan {             // in shared memory
    int sums[16];
    int total, cut[2];         // units of all; this CTA's first and the one behind its last
    int active;                // CTAs among which the units are divided
    int found[2];              // whether a thread has placed the cut (begins that fall can make the units pass 32 bits: a cut then lies in several sequences, or in none)
    Walk walk;                 // the tile of rows it begins in
};
// where CTA c of `active` would begin if units were divided exactly: total c / active
__device__ __forceinline__ int exact_cut(int each, int rest, int active, int c) { return each * c + rest * c / active; }

// All threads: the batch's units, this CTA's range of them, and the tile of rows it begins in.  false: nothing to do
template <int DP, int ROWS, int THREADS>
__device__ __forceinline__ bool plan_work(const AttnArgs& a, Plan* p, int cta, int n_ctas, bool& few) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int WARPS = THREADS / 32;
    // few sequences: a warp each, its lanes along the tiles; many: a thread each
    const bool wide = a.batch.n_seqs <= WARPS;
    const int per_round = wide ? WARPS : THREADS, rounds = (a.batch.n_seqs + per_round - 1) / per_round;
    int most = 0;              // (token, head) rows of a sequence
    const auto units_of = [&](int s) {
        Walk w;
        w.s = s;
        w.n_tiles = 0;
        if (s < a.batch.n_seqs) {
            walk_sequence<ROWS>(a, w);
            most = max(most, w.n_new * a.group);
        }
        int n = sequence_units<ROWS>(a, w, wide ? lane : 0, wide ? 32 : 1);
        if (wide) {
            n = __reduce_add_sync(0xffffffffu, n);
            if (lane > 0) n = 0;
        }
        return a.n_kv * n;
    };
    int mine = 0, units = 0;   // units: of the last round
#pragma unroll 1
    for (int r = 0; r < rounds; r++) {
        units = units_of(r * per_round + (wide ? warp : (int)threadIdx.x));
        mine += units;
    }
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) p->sums[warp] = mine;
    few = !__syncthreads_or(most > FEW);
    const int total = __reduce_add_sync(0xffffffffu, lane < WARPS ? p->sums[lane] : 0);
    const int active = min(n_ctas, total);
    if (cta >= active) return false;
    const int each = total / active, rest = total - each * active, begin = exact_cut(each, rest, active, cta), end = exact_cut(each, rest, active, cta + 1);
    if (threadIdx.x == 0) {
        p->total = total;
        p->active = active;
        p->found[0] = p->found[1] = 0;
        p->cut[0] = 0;
        p->cut[1] = end == total ? total : 0;
    }
    int before = 0;            // units of the rounds before
#pragma unroll 1
    for (int r = 0; r < rounds; r++) {
        if (rounds > 1) units = units_of(r * per_round + (wide ? warp : (int)threadIdx.x));
        int upto = units;      // inclusive sums
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += o;
        }
        __syncthreads();       // (the sums before have been read)
        if (lane == 31) p->sums[warp] = upto;
        __syncthreads();
        const int sum = lane < WARPS ? p->sums[lane] : 0;
        const int at = before + __reduce_add_sync(0xffffffffu, lane < warp ? sum : 0) + upto - units;
        before += __reduce_add_sync(0xffffffffu, sum);
#pragma unroll 1
        for (int i = 0; i < 2; i++) {
            const int cut = i ? end : begin;
            if (!(units > 0 && cut >= at && cut < at + units) || atomicExch(&p->found[i], 1)) continue;   // one thread of the block goes on, for each of the two
            Walk w;
            w.s = r * per_round + (wide ? warp : (int)threadIdx.x);
            walk_sequence<ROWS>(a, w);
            const int per_head = units / a.n_kv;
            w.kv = min((cut - at) / per_head, a.n_kv - 1);
            int in = cut - at - w.kv * per_head;
#pragma unroll 1
            for (w.tile = 0;; w.tile++) {
                walk_tile<ROWS>(a, w);
                if (in < START + w.units || w.tile + 1 == w.n_tiles) break;
                in -= START + w.units;
            }
            in = max(0, min(in, START + w.units - 1));   // (begins that fall: whatever comes of them stays inside)
            const int to = moved_cut<DP>(w, max(0, in - START));
            p->cut[i] = cut - in + (to ? START + to : 0);
            if (i == 0) {
                w.from = to;
                if (to == w.units && !walk_on<ROWS>(a, w)) w.from = 0;   // (the last tile's end: nothing to do)
                p->walk = w;
            }
        }
    }
    __syncthreads();
    return p->found[0] && p->cut[1] > p->cut[0];
}

__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t smem_addr) {
    // MN-major, 128-byte swizzle: a row of 128 bytes is 64 of the operand's N, eight of them (K) a group, groups 1024 bytes apart (SBO); the next 64 of N a
    // block further (LBO)
    return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)(BLOCK_BYTES >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z),
                 "r"(w), "r"(bar)
                 : "memory");
}
// counted on a barrier of either CTA of a pair
__device__ __forceinline__ void tma_load_4d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map), "r"(x), "r"(y),
                 "r"(z), "r"(w), "r"(bar)
                 : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    if constexpr (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    if constexpr (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
// 16 columns of this warp's 32 rows, on their way until tmem_st_wait
__device__ __forceinline__ void tmem_st16_start(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
        "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// named_bar_sync that tells all of its threads whether each came with `yes`
__device__ __forceinline__ bool named_bar_all(int id, int nthreads, bool yes) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.and.pred p, %2, %3, q;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r) : "r"(yes ? 1u : 0u), "r"(id), "r"(nthreads) : "memory");
    return r != 0;
}
template <typename C> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if constexpr (std::is_same<C, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// fp16: weights up to 2^15.  bf16: up to 1, so that values as large as the type's, which a weight of 2^8 would take past fp32 before the division by l, stay inside.
template <typename C> constexpr float WEIGHT_BIAS = std::is_same<C, __half>::value ? 7.0f : -GROWTH;
// whether either 16-bit number of a word is an infinity or a NaN
template <typename C> __device__ __forceinline__ uint32_t no_number(uint32_t w) {
    constexpr uint32_t E = std::is_same<C, __half>::value ? 0x7C00u : 0x7F80u;
    return ((w & E) == E ? 0xFFFFu : 0u) | ((w >> 16 & E) == E ? 0xFFFF0000u : 0u);
}
template <typename C> __device__ __forceinline__ float bits_as(uint32_t bits) {
    if constexpr (std::is_same<C, __half>::value) return __half2float(__ushort_as_half((uint16_t)bits));
    else return __uint_as_float(bits << 16);
}
// 0 x + sum of either 16-bit number
template <typename C> __device__ __forceinline__ uint32_t add_zero_times(uint32_t x, uint32_t sum) {
    uint32_t r;
    if constexpr (std::is_same<C, __half>::value) asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(sum));
    else asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(sum));
    return r;
}
template <typename T> __device__ __forceinline__ float load_as(const void* p, long long at) { return to_f32(((const T*)p)[at]); }

template <typename C>
__device__ __forceinline__ float query_one(const AttnArgs& a, long long at) {
    return a.q_kind == Q38B_OUT_F32 ? to_f32(from_f32<C>(((const float*)a.q)[at])) : to_f32(((const C*)a.q)[at]);
}

__device__ __forceinline__ void store_one(const AttnArgs& a, long long at, float f) {
    if (a.out_kind == Q38B_OUT_F32) ((float*)a.out)[at] = f;
    else if (a.out_kind == Q38B_OUT_F16) ((__half*)a.out)[at] = __float2half_rn(f);
    else ((__nv_bfloat16*)a.out)[at] = __float2bfloat16_rn(f);
}

// Four elements of a head: f by, or nothing for a row that sees nothing
__device__ __forceinline__ void store_four(const AttnArgs& a, long long head, int e, const float* f, float by, bool sees) {
    if (e >= a.D) return;
    const float x[4] = {sees ? f[0] * by : 0.0f, sees ? f[1] * by : 0.0f, sees ? f[2] * by : 0.0f, sees ? f[3] * by : 0.0f};
    const long long to = head + e;
    if (a.out_kind == Q38B_OUT_F32) {
        if (a.out_vec) *(float4*)((float*)a.out + to) = make_float4(x[0], x[1], x[2], x[3]);
        else
#pragma unroll
            for (int i = 0; i < 4; i++) ((float*)a.out)[to + i] = x[i];
        return;
    }
    const uint32_t w0 = a.out_kind == Q38B_OUT_F16 ? pack2<__half>(x[0], x[1]) : pack2<__nv_bfloat16>(x[0], x[1]);
    const uint32_t w1 = a.out_kind == Q38B_OUT_F16 ? pack2<__half>(x[2], x[3]) : pack2<__nv_bfloat16>(x[2], x[3]);
    uint16_t* p = (uint16_t*)a.out + to;
    if (a.out_vec) {
        *(uint2*)p = make_uint2(w0, w1);
    } else {
        p[0] = (uint16_t)w0; p[1] = (uint16_t)(w0 >> 16); p[2] = (uint16_t)w1; p[3] = (uint16_t)(w1 >> 16);
    }
}

// ---- few rows: at most 8 (token, head) rows of each key head, a decoding batch ----
// The tensor core's 128 rows would be nearly empty, and what a tile of keys costs besides its bytes (scores to registers, weights back, three hand-overs) is more than these take to
// come.  So eight warps work by themselves on warp-wide products with keys, and values' columns, as the 16 rows and the queries as the 8 columns (m16n8k16): warp kg takes
// keys 16 kg .. 16 kg + 15 of every tile, with a maximum, a sum and outputs of its own in registers.  11 elements of the cache a clock and SM need 90 multiplications, these products have 975
// (measured).  Nothing is waited for but the memory; at the end of a tile of rows the eight warps' sums meet in shared memory while the ring fills.  A token each, this way and the other:
// 64 sequences of 1000 tokens, 32 + 8 heads of 128 56 / 68 us, of 64 37 / 57; 256 of 500 98 / 140 and 69 / 117; one of 500 10.0 / 11.5 and 9.7 / 10.8; 24 + 4 heads of 256: 59 / 60, 104 / 108, 11.6 / 12.6.
// For up to 16 rows (queries as the 16, keys as the 8, half of the columns a warp) heads of 128 gained less (59 / 68) and heads of 256 lost (86 / 60).
template <typename C>
__device__ __forceinline__ void mma_16x8x16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<C, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool TRANS>
__device__ __forceinline__ void load_matrices(uint32_t* r, uint32_t at) {
    if constexpr (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

template <typename C, int DP>
__device__ __forceinline__ void few_rows(const AttnArgs& a, Walk& w, int cta, uint8_t* q_at, uint8_t* ring, uint64_t* full, uint64_t* empty, uint64_t* meet, uint64_t* w_full,
                                         const Walk* walks, float2* ml, volatile int* abort_flag) {
    using Sh = Shape<DP, 1, false>;
    constexpr int CW = Sh::CW, NCH = Sh::NCH, STAGES = Sh::STAGES, STAGE = Sh::STAGE;
    constexpr int Q_BLOCK = FEW * 128, Q_PLACE = DP / 64 * Q_BLOCK;   // queries: two places, blocks of 8 rows x 64 elements
    constexpr int ROW = DP + 4;                                       // floats between a row's sums and the next's: those of 8 columns and 4 pairs of rows fall into different banks
    constexpr int PASS = 6;                                           // rows whose sums meet at once
    constexpr int MT = DP / 16, CT = CW / 16;                         // 16 columns each: of a head, of a stage
    static_assert(FEW == 8 && 2 * Q_PLACE + 8 * PASS * ROW * 4 <= Sh::Q_BYTES, "shared memory");
    const int kg = (int)(threadIdx.x >> 5) - 4, lane = threadIdx.x & 31, tid = threadIdx.x - 128, quad = lane >> 2, pair = lane & 3;
    float* sums = (float*)(q_at + 2 * Q_PLACE);   // [8 warps][PASS rows][ROW]
    const uint32_t ring_u = smem_u32(ring), full_u = smem_u32(full), empty_u = smem_u32(empty), meet_u = smem_u32(meet), read_u = meet_u + 8;
    // a lane's part in loading four times 8 x 8: keys or rows lie 128 bytes apart, 16-byte pieces are swizzled by the row's last three bits
    const int r8 = lane & 7, lo = lane >> 3 & 1, hi = lane >> 4;
    const uint32_t k_row = (uint32_t)((16 * kg + lo * 8 + r8) * 128), v_row = (uint32_t)((16 * kg + hi * 8 + r8) * 128);
    const auto piece = [&](int block_bytes, int e8) {   // of 8 elements, e8 of them in front
        return (uint32_t)(e8 / 8 * block_bytes + ((e8 % 8) ^ r8) * 16);
    };
    const auto walk_of = [&](int i) {   // (none where the wait was given up: the whole warp then ends)
        const bool there = __all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(&w_full[i & 7]), (uint32_t)i >> 3 & 1u, abort_flag, a.status, ST_WAIT_FULL_TIMEOUT));
        Walk v = walks[i & 7];
        if (!there) v.to = v.from;
        return v;
    };
    const auto load_queries = [&](const Walk& v, int place) {   // a row a warp; rows that are not there come as zeros
        const int e = lane * 8;
        if (e >= DP) return;
        C* to = (C*)(q_at + place * Q_PLACE + e / 64 * Q_BLOCK + kg * 128 + ((e % 64 / 8) ^ kg) * 16);
        uint4 x = make_uint4(0, 0, 0, 0);
        if (kg < v.rows && e < a.D) {
            const int in = by_group(a, v.row0 + kg);
            const long long at = (long long)(v.first + in) * a.q_row + (long long)(v.kv * a.group + v.row0 + kg - in * a.group) * a.q_head + e;
            if (a.q_vec && a.q_shift == 1) {
                x = *(const uint4*)((const uint16_t*)a.q + at);
            } else if (a.q_vec) {
                const float4 y = *(const float4*)((const float*)a.q + at), z = *(const float4*)((const float*)a.q + at + 4);
                x = make_uint4(pack2<C>(y.x, y.y), pack2<C>(y.z, y.w), pack2<C>(z.x, z.y), pack2<C>(z.z, z.w));
            } else {
#pragma unroll 1
                for (int i = 0; i < 8; i++) to[i] = from_f32<C>(query_one<C>(a, at + i));
                return;
            }
        }
        *(uint4*)to = x;
    };
    // all warps have come by (a barrier whose wait ends by itself)
    uint32_t met = 0;
    const auto all_here = [&] {
        __syncwarp();
        if (lane == 0) mbar_arrive(meet_u);
        mbar_wait_bounded(meet_u, met & 1u, abort_flag, a.status, ST_TMEM_TIMEOUT);
        met++;
    };
    const Walk start = walk_of(0);
    if (start.to <= start.from) return;
    w = start;
    load_queries(w, 0);
    all_here();
    uint32_t at = 0, wrote = 0;   // stages taken, uses of `sums`
    for (int item = 0;; item++) {
        int limit[2];   // keys that this lane's two rows, 2 pair and 2 pair + 1, see
#pragma unroll
        for (int r = 0; r < 2; r++) limit[r] = 2 * pair + r < w.rows ? max(0, w.past + by_group(a, w.row0 + 2 * pair + r) + 1) : w.seen;
        const int least = least_seen(a, w);
        uint32_t q[DP / 16][2];
#pragma unroll
        for (int k = 0; k < DP / 16; k += 2)
            load_matrices<false>(q[k], smem_u32(q_at) + (uint32_t)((item & 1) * Q_PLACE) + (uint32_t)(r8 * 128) + piece(Q_BLOCK, 2 * k + (lane >> 3)));
        float o[MT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};   // o: columns quad, quad + 8 of 16, this lane's rows; m: what is taken off, times c
#pragma unroll
        for (int n = 0; n < MT; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
#pragma unroll 1
        for (int tile = w.from; tile < w.to; tile++) {
            const int key0 = tile * KEYS + 16 * kg;
            const bool there = key0 < w.seen, masked = key0 + 16 > least;
            float s[2][4] = {};   // keys quad, quad + 8; in two sums
#pragma unroll
            for (int c = 0; c < NCH; c++, at++) {
                const uint32_t st = at % STAGES;
                mbar_wait_bounded(full_u + 8u * st, at / STAGES & 1u, abort_flag, a.status, ST_WAIT_FULL_TIMEOUT);
                if (there) {
#pragma unroll
                    for (int x0 = 0; x0 < CT; x0 += 4) {   // four loads at once, then their products
                        uint32_t k[4][4];
#pragma unroll
                        for (int x = 0; x < 4; x++) load_matrices<false>(k[x], ring_u + st * STAGE + k_row + piece(BLOCK_BYTES, 2 * (x0 + x) + hi));
#pragma unroll
                        for (int x = 0; x < 4; x++) mma_16x8x16<C>(s[x & 1], k[x], q[c * CT + x0 + x][0], q[c * CT + x0 + x][1]);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty_u + 8u * st);
            }
            uint32_t p[2] = {0, 0}, seen_by_any[2] = {0, 0}, seen_by_some[2] = {0, 0};   // (of values: bits of this lane's two keys, and of 8 further on)
            if (masked)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int key = key0 + 8 * i + 2 * pair;
                    seen_by_any[i] = (key < w.seen ? 0xFFFFu : 0u) | (key + 1 < w.seen ? 0xFFFF0000u : 0u);
                    seen_by_some[i] = (key >= least ? 0xFFFFu : 0u) | (key + 1 >= least ? 0xFFFF0000u : 0u);
                }
            if (there) {
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    s[0][x] += s[1][x];
                    if (masked && key0 + quad + 8 * (x >> 1) >= limit[x & 1]) s[0][x] = -INFINITY;
                }
                float now[2];
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    float top = fmaxf(s[0][r], s[0][2 + r]);
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    top *= a.c;
                    now[r] = m[r] == -INFINITY || top > m[r] + GROWTH ? top : m[r];
                }
                if (__any_sync(0xffffffffu, now[0] != m[0] || now[1] != m[1])) {
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const float by = now[r] == m[r] ? 1.0f : m[r] == -INFINITY ? 0.0f : exp2_fast(m[r] - now[r]);
                        l[r] *= by;
                        m[r] = now[r];
#pragma unroll
                        for (int n = 0; n < MT; n++) {
                            o[n][r] *= by;
                            o[n][2 + r] *= by;
                        }
                    }
                }
                float e[4];
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    e[x] = exp2_fast(fmaf(s[0][x], a.c, (m[x & 1] == -INFINITY ? 0.0f : -m[x & 1]) + WEIGHT_BIAS<C>));
                    l[x & 1] += e[x];
                }
                p[0] = transposed(pack2<C>(e[0], e[1]));   // row quad, keys 2 pair, 2 pair + 1 and 8 more
                p[1] = transposed(pack2<C>(e[2], e[3]));
            }
#pragma unroll
            for (int c = 0; c < NCH; c++, at++) {
                const uint32_t st = at % STAGES;
                mbar_wait_bounded(full_u + 8u * st, at / STAGES & 1u, abort_flag, a.status, ST_WAIT_FULL_TIMEOUT);
                if (there) {
#pragma unroll
                    for (int x0 = 0; x0 < CT; x0 += 4) {
                        const uint32_t v_u = ring_u + st * STAGE + v_row;
                        uint32_t v[4][4];
#pragma unroll
                        for (int x = 0; x < 4; x++) load_matrices<true>(v[x], v_u + piece(BLOCK_BYTES, 2 * (x0 + x) + lo));
                        if (masked) {
                            // Values of keys that none of the rows sees may be anything; those that only some see, and that are no numbers, go to these rows one by one.
                            uint32_t times0 = 0;   // a NaN for what is no number
#pragma unroll
                            for (int x = 0; x < 4; x++)
#pragma unroll
                                for (int i = 0; i < 4; i++) {
                                    v[x][i] &= seen_by_any[i >> 1];
                                    times0 = add_zero_times<C>(v[x][i] & seen_by_some[i >> 1], times0);
                                }
                            if (__any_sync(0xffffffffu, no_number<C>(times0) != 0)) {
                                uint32_t odd[4][4];
#pragma unroll
                                for (int x = 0; x < 4; x++)
#pragma unroll
                                    for (int i = 0; i < 4; i++) {
                                        odd[x][i] = v[x][i] & no_number<C>(v[x][i]) & seen_by_some[i >> 1];
                                        v[x][i] ^= odd[x][i];
                                    }
#pragma unroll 1
                                for (int j = 0; j < 16; j++) {
                                    const int shift = j & 1 ? 16 : 0, in = (j & 7) / 2;
                                    float weight[2];
#pragma unroll
                                    for (int y = 0; y < 2; y++)   // of row 2 pair + y
                                        weight[y] = bits_as<C>(__shfl_sync(0xffffffffu, j < 8 ? p[0] : p[1], (2 * pair + y) * 4 + in) >> shift & 0xFFFFu);
#pragma unroll
                                    for (int x = 0; x < 4; x++)
#pragma unroll
                                        for (int y = 0; y < 2; y++) {   // column quad + 8 y
                                            const uint32_t value = __shfl_sync(0xffffffffu, j < 8 ? odd[x][y] : odd[x][2 + y], (lane & ~3) + in) >> shift & 0xFFFFu;
#pragma unroll
                                            for (int r = 0; r < 2; r++)
                                                if (value != 0 && key0 + j < limit[r]) o[c * CT + x0 + x][2 * y + r] = fmaf(weight[r], bits_as<C>(value), o[c * CT + x0 + x][2 * y + r]);
                                        }
                                }
                            }
                        }
#pragma unroll
                        for (int x = 0; x < 4; x++) mma_16x8x16<C>(o[c * CT + x0 + x], v[x], p[0], p[1]);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty_u + 8u * st);
            }
        }
        // the eight warps' sums meet; the next tile's queries come in between
        const Walk next = walk_of(item + 1);
        const bool more = next.to > next.from;
        if (more) load_queries(next, (item + 1) & 1);
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], d);
        const bool whole = w.from == 0 && w.to == w.units;
#pragma unroll 1
        for (int row0 = 0; row0 < w.rows; row0 += PASS) {
            if (wrote) mbar_wait_bounded(read_u, (wrote - 1) & 1u, abort_flag, a.status, ST_TMEM_TIMEOUT);
            wrote++;
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int in = 2 * pair + r - row0;
                if (in < 0 || in >= PASS) continue;
                if (quad == 0) ml[8 * kg + in] = make_float2(m[r], l[r]);
#pragma unroll
                for (int n = 0; n < MT; n++) {
                    float* to = sums + (PASS * kg + in) * ROW + 16 * n + quad;
                    to[0] = o[n][r];
                    to[8] = o[n][2 + r];
                }
            }
            all_here();
            const int rows = min(PASS, w.rows - row0);
            for (int u = tid; u < rows * (DP / 4); u += 256) {
                const int r = u / (DP / 4), e = u % (DP / 4) * 4, row = row0 + r;
                float2 of[8];
#pragma unroll
                for (int k = 0; k < 8; k++) of[k] = ml[8 * k + r];
                float top = of[0].x;
#pragma unroll
                for (int k = 1; k < 8; k++) top = fmaxf(top, of[k].x);
                float sum = 0.0f, f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float by = of[k].x == -INFINITY ? 0.0f : exp2_fast(of[k].x - top);
                    const float4 x = *(const float4*)(sums + (PASS * k + r) * ROW + e);
                    sum = fmaf(of[k].y, by, sum);
                    f[0] = fmaf(x.x, by, f[0]);
                    f[1] = fmaf(x.y, by, f[1]);
                    f[2] = fmaf(x.z, by, f[2]);
                    f[3] = fmaf(x.w, by, f[3]);
                }
                if (whole) {
                    const int tok = by_group(a, w.row0 + row), head = w.kv * a.group + w.row0 + row - tok * a.group;
                    const long long out_row = w.first + tok;
                    const bool sees = w.past + tok + 1 > 0;
                    if (a.lse && e == 0) a.lse[out_row * a.n_heads + head] = sees ? 0.6931471805599453f * (top + (log2f(sum) - WEIGHT_BIAS<C>)) : -INFINITY;
                    store_four(a, out_row * a.out_row + (long long)head * a.out_head, e, f, sees ? 1.0f / sum : 0.0f, sees);
                } else {
                    float* to = a.slots + (long long)(2 * cta + (w.from == 0 ? 1 : 0)) * a.slot_rows * (DP + 4);
                    *(float4*)(to + (long long)(e / 4 * a.slot_rows + row) * 4) = make_float4(f[0], f[1], f[2], f[3]);
                    if (e == 0) *(float2*)(to + (long long)a.slot_rows * DP + 2 * row) = make_float2(top, sum);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(read_u);
        }
        if (!more) break;
        w = next;
    }
}

template <typename C, int DP, int QT, bool PAIR>
__global__ void __launch_bounds__(Shape<DP, QT, PAIR>::THREADS, 1)
attention_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using Sh = Shape<DP, QT, PAIR>;
    constexpr int CW = Sh::CW, NCH = Sh::NCH, STAGE = Sh::STAGE, STAGES = Sh::STAGES, ROWS = Sh::ROWS;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* full = (uint64_t*)smem;
    uint64_t* empty = full + 12;
    uint64_t* s_full = empty + 12;   // [2] scores are there
    uint64_t* p_full = s_full + 2;   // [2] weights are there
    uint64_t* o_done = p_full + 2;   // [2] ... have been multiplied with values
    uint64_t* m_full = o_done + 2;   // [2][4] QT = 1: the maxima that a warp of either warpgroup took off are known to the other
    uint64_t* q_full = m_full + 8;
    uint64_t* w_full = q_full + 1;   // [8] a tile of rows is known
    uint64_t* v_here = w_full + 8;   // [STAGES] PAIR: this CTA's values of a tile that some rows do not see all of
    uint64_t* o_free = v_here + 8;   // QT = 1: the outputs of a tile of rows have been read, by both warpgroups
    uint32_t* tmem_slot = (uint32_t*)(o_free + 1);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    volatile int* spoilt = abort_flag + 1;   // [2]: the item that met values that are no numbers among keys that not all of its rows see
    Plan* plan = (Plan*)(smem + 464);
    Walk* walks = (Walk*)(smem + 608);             // [8] the CTA's tiles of rows, as the first loading warp goes through them (it is at most half a ring ahead)
    float* m_rows = (float*)(smem + 1024);       // [2][128]
    float* l_rows = (float*)(smem + 2048);       // [2][128]
    static_assert(sizeof(Plan) <= 144 && 608 + 8 * sizeof(Walk) <= 1024 && (!PAIR || STAGES <= 8), "shared memory");
    uint8_t* q_at = smem + HEAD;
    uint8_t* ring = q_at + Sh::Q_BYTES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = PAIR ? (int)cluster_rank() : 0, cta = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;   // (a pair counts as one)

    if (threadIdx.x == 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
    }
    if (threadIdx.x == 64) {
        *abort_flag = 0;
        spoilt[0] = spoilt[1] = -1;
    }
    {   // a barrier a thread
        const int b = threadIdx.x;
        const auto is = [&](const uint64_t* first, int n) { return b >= (int)(first - full) && b < (int)(first - full) + n; };
        if (b < (int)(o_free + 1 - full)) {
            mbar_init(smem_u32(&full[b]), is(p_full, 2) ? (PAIR ? 8 : 4) : is(q_full, 1) || is(o_free, 1) ? (PAIR ? 16 : 8) : 1);
            mbar_fence_init();
            fence_proxy_async();
        }
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    bool few = false;
    const bool any = plan_work<DP, ROWS, Sh::THREADS>(a, plan, cta, PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x, few);   // (with barriers of the block)
    if (QT == 2 || PAIR) few = false;
    if (few) {   // eight warps arrive there, and nothing but warps: no fences for the copies' and products' sake as above
        if (threadIdx.x < 20) {
            const uint32_t bar = smem_u32(threadIdx.x < 12 ? &empty[threadIdx.x] : &m_full[threadIdx.x - 12]);
            asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
            mbar_init(bar, 8);
        }
        __syncthreads();
    }
    if constexpr (PAIR) cluster_sync_all();   // the other CTA's barriers are initialised
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    int left = any ? plan->cut[1] - plan->cut[0] : 0;
    Walk w = plan->walk;
    if (any) walk_to(w, left);

    const int boxes = stage_boxes(a.box_rows, CW);
    if (any && (warp == 0 || (warp >= 2 && warp <= loading_warps(boxes)))) {
        // ---------------- keys and values: a lane of one of three warps a box of at most 128 slots x 64 elements ----------------
        // (A warp issues its lanes' copies one by one, some 80 clocks each: the 64 of 128 keys and values in pages of 16 took it as long as the memory does.)
        // A box of keys: block `block[0]` of 64 elements, slots `in[0]` and on of the tile; of values: [1].
        const int loader = warp == 0 ? 0 : warp - 1, box = 3 * lane + loader, k_boxes = (PAIR ? KEYS / 2 : KEYS) / a.box_rows, v_boxes = KEYS / a.box_rows;
        const bool mine = box < boxes;   // lanes behind the last box do nothing
        const int k_block = box / k_boxes, k_part = box % k_boxes * a.box_rows, v_block = box / v_boxes, v_part = box % v_boxes * a.box_rows;
        const int in[2] = {k_part + (PAIR ? rank * (KEYS / 2) : 0), v_part}, x0[2] = {k_block * 64, v_block * 64 + (PAIR ? rank * 128 : 0)};
        const uint32_t to[2] = {(uint32_t)(k_block * (PAIR ? BLOCK_BYTES / 2 : BLOCK_BYTES) + k_part * 128), (uint32_t)(v_block * BLOCK_BYTES + v_part * 128)};
        const uint32_t ring_u = smem_u32(ring), full_u = PAIR ? peer_smem(smem_u32(full), 0u) : smem_u32(full), empty_u = smem_u32(empty);
        const int slots = (1 << a.batch.page_shift) - 1;
        const bool in_turn = QT == 2 || few;
        uint32_t at = 0;   // stages filled so far
        int item = 0;
        const auto publish = [&](const Walk& v) {
            if (threadIdx.x == 0) {
                walks[item & 7] = v;
                mbar_arrive(smem_u32(&w_full[item & 7]));
            }
            item++;
        };
        bool ended = false;   // a wait was given up: no tile of rows and no copy more, so that nobody finds a place of `walks` changed
        do {
            ended = __any_sync(0xffffffffu, *abort_flag != 0);
            if (ended) break;
            publish(w);
            const int n = w.to - w.from;
            // the steps in the order in which the tensor core takes them: keys K0 K1 V0 K2 V1 .. (QT = 1), K0 V0 K1 V1 .. (QT = 2, few rows); a step's page is looked up during the one before
            const auto tile_of = [&](int i, bool& values) {
                values = in_turn ? i & 1 : i == 2 * n - 1 || (i > 0 && !(i & 1));
                return in_turn ? i >> 1 : i == 2 * n - 1 ? n - 1 : values ? i / 2 - 1 : (i + 1) / 2;
            };
            const auto page_of = [&](int i) {   // of this lane's box; keys nobody sees come as zeros, from a page that is not there
                bool values;
                const int tile = tile_of(i, values), token = (w.from + tile) * KEYS + in[values];
                return i < 2 * n && token < w.seen ? a.batch.page(w.s, token) : a.batch.n_pages;
            };
            int page = page_of(0);
#pragma unroll 1
            for (int i = 0; i < 2 * n && !ended; i++) {
                bool values;
                const int j0 = (w.from + tile_of(i, values)) * KEYS, slot = (j0 + in[values]) & slots, next = page_of(i + 1);
                const CUtensorMap* map = values ? &vmap : &kmap;
                const bool looked_at = PAIR && values && j0 + KEYS > least_seen(a, w);   // these the other warps of this CTA wait for themselves
#pragma unroll 1
                for (int c = 0; c < NCH; c++, at++) {
                    const uint32_t st = at % STAGES, use = at / STAGES;
                    ended = !__all_sync(0xffffffffu, mbar_wait_bounded(empty_u + 8u * st, (use & 1u) ^ 1u, abort_flag, a.status, ST_WAIT_EMPTY_TIMEOUT));
                    if (ended) break;
                    if constexpr (PAIR) {
                        const uint32_t here = smem_u32(&v_here[st]);
                        if (threadIdx.x == 0) {
                            if (looked_at) mbar_arrive_expect_tx(here, STAGE);
                            if (rank == 0 && looked_at) mbar_arrive(smem_u32(&full[st]));
                            if (rank == 0 && !looked_at) mbar_arrive_expect_tx(smem_u32(&full[st]), 2 * STAGE);
                        }
                        __syncwarp();
                        if (mine && looked_at) tma_load_4d(ring_u + st * STAGE + to[values], map, x0[values], slot, w.kv, page, here);
                        if (mine && !looked_at) tma_load_4d_pair(ring_u + st * STAGE + to[values], map, x0[values], slot, w.kv, page, full_u + 8u * st);
                    } else {
                        if (threadIdx.x == 0) mbar_arrive_expect_tx(full_u + 8u * st, STAGE);
                        __syncwarp();
                        if (mine) tma_load_4d(ring_u + st * STAGE + to[values], map, c * CW + x0[values], slot, w.kv, page, full_u + 8u * st);
                    }
                }
                page = next;
            }
        } while (!ended && walk_next<ROWS>(a, w, left));
        w.to = w.from;   // no more
        if (!ended) publish(w);
    } else if (few) {
        if constexpr (QT == 1 && !PAIR)
            if (any && warp >= 4) few_rows<C, DP>(a, w, cta, q_at, ring, full, empty, m_full, w_full, walks, (float2*)m_rows, abort_flag);
    } else if (any && warp == 1 && rank == 0) {
        // ---------------- products (of a pair: for both) ----------------
        constexpr uint32_t TYPE = std::is_same<C, __half>::value ? 0u : 1u;
        constexpr uint32_t idesc_s = (1u << 4) | (TYPE << 7) | (TYPE << 10) | ((uint32_t)(KEYS >> 3) << 17) | ((uint32_t)((PAIR ? 256 : 128) >> 4) << 24);
        constexpr uint32_t idesc_o = (1u << 4) | (TYPE << 7) | (TYPE << 10) | (1u << 16) | ((uint32_t)((PAIR ? DP : CW) >> 3) << 17) | ((uint32_t)((PAIR ? 256 : 128) >> 4) << 24);
        const uint64_t kdesc0 = umma_desc_sw128(0), vdesc0 = umma_desc_mn_sw128(0);
        const uint32_t q_u = smem_u32(q_at), ring_u = smem_u32(ring), full_u = smem_u32(full), empty_u = smem_u32(empty);
        uint32_t ring0 = 0, p_phase = 0, item = 0;
        for (;;) {
            const bool there = __all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(&w_full[item & 7]), item >> 3 & 1u, abort_flag, a.status, ST_WAIT_FULL_TIMEOUT));
            const int tiles = walks[item & 7].to - walks[item & 7].from, n = QT * tiles;
            if (!there || tiles <= 0) break;
            mbar_wait_bounded(smem_u32(q_full), item & 1u, abort_flag, a.status, ST_WAIT_FULL_TIMEOUT);
            const auto scores = [&](int i) {
                const int tile = QT == 2 ? i >> 1 : i, t = QT == 2 ? i & 1 : 0;
                const uint32_t d = tmem + (uint32_t)((i & 1) * KEYS);
#pragma unroll
                for (int c = 0; c < NCH; c++) {
                    const uint32_t at = ring0 + at_keys<QT, NCH>(tile) + c, st = at % STAGES;
                    mbar_wait_bounded(full_u + 8u * st, at / STAGES & 1u, abort_flag, a.status, ST_WAIT_FULL_TIMEOUT);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t qd = kdesc0 + ((q_u + (uint32_t)(t * 128 * DP * 2 + c * CW / 64 * BLOCK_BYTES)) >> 4), kd = kdesc0 + ((ring_u + st * STAGE) >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < (PAIR ? DP : CW) / 16; k++)
                            mma_ss<PAIR>(d, qd + (uint64_t)((k / 4 * BLOCK_BYTES + k % 4 * 32) >> 4), kd + (uint64_t)((k / 4 * (PAIR ? BLOCK_BYTES / 2 : BLOCK_BYTES) + k % 4 * 32) >> 4), idesc_s,
                                         c > 0 || k > 0 ? 1u : 0u);
                        if (QT == 1 || t == 1) umma_commit<PAIR>(empty_u + 8u * st);
                        if (c == NCH - 1) umma_commit<PAIR>(smem_u32(&s_full[i & 1]));
                    }
                    __syncwarp();
                }
            };
            // two scores ahead of the products with values; one copy of either's code (a CTA of few tiles waits for its instructions)
#pragma unroll 1
            for (int i = -2; i < n; i++) {
                if (i >= 0) {
                    const int tile = QT == 2 ? i >> 1 : i, t = QT == 2 ? i & 1 : 0;
                    mbar_wait_bounded(smem_u32(&p_full[i & 1]), p_phase >> (i & 1) & 1u, abort_flag, a.status, ST_WAIT_FULL_TIMEOUT);
                    p_phase ^= 1u << (i & 1);
                    // A tile's first product writes over the outputs of the tile before.  QT = 2: those whose weights have just come have read them.  QT = 1: the other warpgroup
                    // stores the other half of them, and nothing else makes this one wait for it.
                    if (QT == 1 && i == 0 && item > 0) mbar_wait_bounded(smem_u32(o_free), (item - 1) & 1u, abort_flag, a.status, ST_TMEM_TIMEOUT);
#pragma unroll
                    for (int c = 0; c < NCH; c++) {
                        const uint32_t at = ring0 + at_values<QT, NCH>(tile, tiles) + c, st = at % STAGES;
                        mbar_wait_bounded(full_u + 8u * st, at / STAGES & 1u, abort_flag, a.status, ST_WAIT_FULL_TIMEOUT);
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t d = tmem + (uint32_t)(256 + t * DP + c * CW), p = tmem + (uint32_t)((i & 1) * KEYS);
                        const uint64_t vd = vdesc0 + ((ring_u + st * STAGE) >> 4);
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < KEYS / 16; k++) mma_ts<PAIR>(d, p + (uint32_t)(8 * k), vd + (uint64_t)(k * 2048 >> 4), idesc_o, k > 0 || tile > 0 ? 1u : 0u);
                            if (QT == 1 || t == 1) umma_commit<PAIR>(empty_u + 8u * st);
                            if (c == NCH - 1) umma_commit<PAIR>(smem_u32(&o_done[i & 1]));
                        }
                        __syncwarp();
                    }
                }
                if (i + 2 < n) scores(i + 2);
            }
            ring0 += (uint32_t)(2 * tiles * NCH);
            item++;
        }
    } else if (any && warp >= 4) {
        // ---------------- weights: warpgroup g takes the scores that lie in place g, a thread a row ----------------
        // QT = 2: those of its own 128 rows.  QT = 1: those of every other tile of keys; the maxima go from one warpgroup to the other, and each has a sum of its own.
        const int g = (warp >> 2) - 1, quad = warp & 3, qt = QT == 2 ? g : 0, t = PAIR ? rank : qt, row = 128 * t + 32 * quad + lane;   // row: of the tile of rows
        const uint32_t lanes = (uint32_t)(32 * quad) << 16, o_tm = tmem + lanes + (uint32_t)(256 + qt * DP), s_tm = tmem + lanes + (uint32_t)(g * KEYS);
        const uint32_t s_bar = smem_u32(&s_full[g]), p_bar = PAIR ? peer_smem(smem_u32(&p_full[g]), 0u) : smem_u32(&p_full[g]), done_u = smem_u32(o_done);
        constexpr int COLS = QT == 2 ? DP : DP / 2;     // of the outputs this warpgroup stores
        const int col0 = QT == 2 ? 0 : g * COLS;
        const auto arrive = [](uint32_t bar) {   // PAIR: at the CTA that issues
            if constexpr (PAIR) mbar_arrive_peer(bar);
            else mbar_arrive(bar);
        };
        const auto load_queries = [&](const Walk& v) {
            constexpr int UNITS = DP / 8, STEP = QT == 2 ? 32 : 64;    // 16-byte pieces of a row; (QT = 1: the two warps of these rows take turns)
            const int here = min(32, v.rows - (128 * t + 32 * quad)), pieces = here * UNITS;   // rows that are not there keep whatever they hold: it meets no other row
            uint8_t* to = q_at + qt * 128 * DP * 2 + 32 * quad * 128;
            if (here > 0) {
                const int flat = v.row0 + row, in = by_group(a, flat);
                const long long my_row = (long long)(v.first + in) * a.q_row + (long long)(v.kv * a.group + flat - in * a.group) * a.q_head;
                const auto put = [&](int u, const uint4& x) {
                    const int r = u / UNITS, e = u % UNITS * 8;
                    if (u < pieces) *(uint4*)(to + e / 64 * BLOCK_BYTES + r * 128 + ((e % 64 / 8) ^ (r & 7)) * 16) = x;
                };
                const auto ask = [&](int u, int half) {   // 16 bytes of a piece
                    const long long at = __shfl_sync(0xffffffffu, my_row, u / UNITS & 31) + u % UNITS * 8;
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (u < pieces && u % UNITS * 8 < a.D) x = ((const uint4*)((const uint8_t*)a.q + (at << a.q_shift)))[half];
                    return x;
                };
                const int u1 = (QT == 2 ? 0 : 32 * g) + lane;
                if (a.q_vec && a.q_shift == 1) {   // all of them on their way at once, past the registers
#pragma unroll 1
                    for (int u = u1; u - lane < pieces; u += STEP) {
                        const int r = u / UNITS, e = u % UNITS * 8;
                        const long long at = __shfl_sync(0xffffffffu, my_row, r & 31) + e;
                        if (u < pieces)
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to) + (uint32_t)(e / 64 * BLOCK_BYTES + r * 128 + ((e % 64 / 8) ^ (r & 7)) * 16)),
                                         "l"((const uint16_t*)a.q + (e < a.D ? at : 0)), "r"(e < a.D ? 16 : 0)
                                         : "memory");
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                } else if (a.q_vec) {
                    constexpr int AHEAD = 4;
#pragma unroll 1
                    for (int u0 = u1; u0 - lane < pieces; u0 += STEP * AHEAD) {
                        uint4 x[AHEAD], y[AHEAD];
#pragma unroll
                        for (int n = 0; n < AHEAD; n++) {
                            x[n] = ask(u0 + STEP * n, 0);
                            y[n] = ask(u0 + STEP * n, 1);
                        }
#pragma unroll
                        for (int n = 0; n < AHEAD; n++)
                            put(u0 + STEP * n, make_uint4(pack2<C>(__uint_as_float(x[n].x), __uint_as_float(x[n].y)), pack2<C>(__uint_as_float(x[n].z), __uint_as_float(x[n].w)),
                                                          pack2<C>(__uint_as_float(y[n].x), __uint_as_float(y[n].y)), pack2<C>(__uint_as_float(y[n].z), __uint_as_float(y[n].w))));
                    }
                }
                if (!a.q_vec) {
                    __syncwarp();
#pragma unroll 1
                    for (int u = (QT == 2 ? 0 : 32 * g) + lane; u - lane < pieces; u += STEP) {
                        const int r = u / UNITS, e = u % UNITS * 8;
                        const long long at = __shfl_sync(0xffffffffu, my_row, r & 31) + e;
                        if (u >= pieces) continue;
                        C* x = (C*)(to + e / 64 * BLOCK_BYTES + r * 128 + ((e % 64 / 8) ^ (r & 7)) * 16);
#pragma unroll 1
                        for (int i = 0; i < 8; i++) x[i] = from_f32<C>(e < a.D ? query_one<C>(a, at + i) : 0.0f);
                    }
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) arrive(PAIR ? peer_smem(smem_u32(q_full), 0u) : smem_u32(q_full));
        };
        uint32_t ring0 = 0, s_use = 0, m_use = 0, looked = 0, done[2] = {0, 0};   // done: products P V from either place up to this item
        int item;   // the tile of rows in front of the one that is worked on
        const auto walk_there = [&](int i) {
            return (bool)__all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(&w_full[i & 7]), (uint32_t)i >> 3 & 1u, abort_flag, a.status, ST_WAIT_FULL_TIMEOUT));
        };
        // A round ends a tile of rows: the next one's queries go in place while its last products run, its outputs leave, the next one's scores become weights.
        // Where a wait was given up there may be none for one warp and still one for another: the two warps that meet at the end of a tile go on together, or neither does.
        bool there = walk_there(0);
        if (QT == 1) there = named_bar_all(1 + quad, 64, there);
        Walk next = walks[0];
        float m = -INFINITY, l = 0.0f;   // m: what is taken off, times c
        int tiles = 0, n = 0, tok = 0, limit = 0, least_item = 0;
        bool idle = true;
        for (item = -1;; item++) {
            const bool more = there && next.to > next.from;
            if (more) load_queries(next);
            if (item >= 0) {
                {
                    const int last = QT == 2 ? n - 2 + g : n - 1;
                    mbar_wait_bounded(done_u + 8u * (uint32_t)(last & 1), (done[last & 1] + (uint32_t)(last >> 1)) & 1u, abort_flag, a.status, ST_TMEM_TIMEOUT);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                }
                done[0] += (uint32_t)((n + 1) >> 1);
                done[1] += (uint32_t)(n >> 1);
                if (least_item < w.seen && spoilt[item & 1] == item) {
                    // Rare: what was taken out of the products goes to the rows that see it, a value at a time.
                    const int lo = max(least_item, w.from * KEYS), hi = min(w.seen, w.to * KEYS);
                    const long long q_row = (long long)(w.first + tok) * a.q_row + (long long)(w.kv * a.group + w.row0 + row - tok * a.group) * a.q_head;
                    for (int j = lo; j < hi; j++) {
                        const int page = a.batch.page(w.s, j);
                        if (page >= a.batch.n_pages) continue;
                        const long long in = j & ((1 << a.batch.page_shift) - 1);
                        const long long v_at = page * a.v_page + in * a.v_slot + w.kv * a.v_head, k_at = page * a.k_page + in * a.k_slot + w.kv * a.k_head;
                        float weight = 0.0f;
                        bool known = false;
                        for (int e = col0; e < min(a.D, col0 + COLS); e++) {
                            const float x = load_as<C>(a.v, v_at + e);
                            if (fabsf(x) < INFINITY) continue;
                            if (!known) {
                                float dot = 0.0f;
                                if (row < w.rows)
                                    for (int d = 0; d < a.D; d++) dot = fmaf(query_one<C>(a, q_row + d), load_as<C>(a.k, k_at + d), dot);
                                weight = exp2_fast(fmaf(dot, a.c, (m == -INFINITY ? 0.0f : -m) + WEIGHT_BIAS<C>));
                                known = true;
                            }
                            uint32_t o;
                            __syncwarp();
                            asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(o) : "r"(o_tm + (uint32_t)e) : "memory");
                            tmem_ld_wait();
                            asm volatile("" : "+r"(o));
                            if (j < limit) o = __float_as_uint(fmaf(weight, x, __uint_as_float(o)));
                            asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(o_tm + (uint32_t)e), "r"(o) : "memory");
                            tmem_st_wait();
                        }
                    }
                }
                const bool whole = w.from == 0 && w.to == w.units;
                const int head = w.kv * a.group + w.row0 + row - tok * a.group;
                const long long out_row = w.first + tok;
                if (idle) {
                } else if (whole) {
                    const float by = limit > 0 ? 1.0f / l : 0.0f;
                    const long long out_at = out_row * a.out_row + (long long)head * a.out_head;
                    if (a.out_vec && (a.out_kind == Q38B_OUT_F32 || a.out_kind == (std::is_same<C, __half>::value ? Q38B_OUT_F16 : Q38B_OUT_BF16))) {
#pragma unroll 1
                        for (int k0 = col0; k0 < col0 + COLS; k0 += 32) {
                            uint32_t o[32];
                            tmem_ld16_start(o_tm + (uint32_t)k0, o);
                            tmem_ld16_start(o_tm + (uint32_t)k0 + 16, o + 16);
                            tmem_ld_wait();
                            tmem_ld_arrived(o);
                            tmem_ld_arrived(o + 16);
#pragma unroll
                            for (int e = 0; e < 32; e++) o[e] = limit > 0 ? __float_as_uint(__uint_as_float(o[e]) * by) : 0u;
                            if (a.out_kind != Q38B_OUT_F32)
#pragma unroll
                                for (int e = 0; e < 32; e += 2) o[e / 2] = pack2<C>(__uint_as_float(o[e]), __uint_as_float(o[e + 1]));
                            if (row >= w.rows) continue;
                            // whole sectors of 32 bytes where they are aligned: stores of 16 went to 32 lines each as well (128 rows of 256 in 5500 clocks)
                            uint8_t* to = (uint8_t*)a.out + ((out_at + k0) << a.out_shift);
                            const int bytes = min(32, a.D - k0) << a.out_shift;
                            if (a.out_vec == 2) {
#pragma unroll
                                for (int i = 0; i < 4; i++)
                                    if (32 * i < bytes)
                                        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to + 32 * i), "r"(o[8 * i]), "r"(o[8 * i + 1]), "r"(o[8 * i + 2]), "r"(o[8 * i + 3]),
                                                     "r"(o[8 * i + 4]), "r"(o[8 * i + 5]), "r"(o[8 * i + 6]), "r"(o[8 * i + 7])
                                                     : "memory");
                            } else {
#pragma unroll
                                for (int i = 0; i < 8; i++)
                                    if (16 * i < bytes) *(uint4*)(to + 16 * i) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                            }
                        }
                    } else {   // another type or alignment: a column at a time
#pragma unroll 1
                        for (int k = col0; k < min(a.D, col0 + COLS); k++) {
                            uint32_t o;
                            asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(o) : "r"(o_tm + (uint32_t)k) : "memory");
                            tmem_ld_wait();
                            asm volatile("" : "+r"(o));
                            if (row < w.rows) store_one(a, out_at + k, limit > 0 ? __uint_as_float(o) * by : 0.0f);
                        }
                    }
                    if (a.lse && row < w.rows && col0 == 0) a.lse[out_row * a.n_heads + head] = limit > 0 ? 0.6931471805599453f * (m + (log2f(l) - WEIGHT_BIAS<C>)) : -INFINITY;
                } else {
                    // a place in the work area: [4 columns][row] and each row's m and l behind
                    float* to = a.slots + (long long)(2 * cta + (w.from == 0 ? 1 : 0)) * a.slot_rows * (DP + 4);
#pragma unroll 1
                    for (int k = col0; k < col0 + COLS; k += 32) {
                        uint32_t o[32];
                        tmem_ld16_start(o_tm + (uint32_t)k, o);
                        tmem_ld16_start(o_tm + (uint32_t)k + 16, o + 16);
                        tmem_ld_wait();
                        tmem_ld_arrived(o);
                        tmem_ld_arrived(o + 16);
                        if (row < w.rows)
#pragma unroll
                            for (int e = 0; e < 32; e += 4) *(uint4*)(to + (long long)((k + e) / 4 * a.slot_rows + row) * 4) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    }
                    if (row < w.rows && col0 == 0) *(float2*)(to + (long long)a.slot_rows * DP + 2 * row) = make_float2(m, l);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                if constexpr (QT == 1) {
                    __syncwarp();
                    if (lane == 0) arrive(PAIR ? peer_smem(smem_u32(o_free), 0u) : smem_u32(o_free));
                }
            }
            if (!more) break;
            w = next;
            tiles = w.to - w.from;
            n = QT * tiles;
            tok = by_group(a, w.row0 + row);
            limit = row < w.rows ? max(0, w.past + tok + 1) : w.seen;                          // keys this row sees
            const int least = max(0, w.past + by_group(a, w.row0 + min(128 * t + 32 * quad, w.rows - 1)) + 1);   // ... the warp's first row
            least_item = least_seen(a, w);                                                                    // ... the item's first row
            idle = 128 * t + 32 * quad >= w.rows;   // no row of this warp's is there
            m = -INFINITY;
            l = 0.0f;
            for (int i = g; i < n; i += 2) {
                const int tile = QT == 2 ? i >> 1 : i, j0 = (w.from + tile) * KEYS;
                mbar_wait_bounded(s_bar, s_use & 1u, abort_flag, a.status, ST_TMEM_TIMEOUT);
                s_use++;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (!idle) {
                    // a half of the scores at a time (all of a row's in registers spilled a fifth of them); the first stays for the weights
                    constexpr int HALF = KEYS / 2;
                    uint32_t v[HALF];
                    const int seen = limit - j0;
                    const bool masked = j0 + KEYS > least;
                    const auto load_half = [&](int h) {
#pragma unroll
                        for (int k = 0; k < HALF; k += 16) tmem_ld16_start(s_tm + (uint32_t)(h * HALF + k), v + k);
                        tmem_ld_wait();
#pragma unroll
                        for (int k = 0; k < HALF; k += 16) tmem_ld_arrived(v + k);
                        if (masked)
#pragma unroll
                            for (int k = 0; k < HALF; k++) v[k] = h * HALF + k < seen ? v[k] : 0xFF800000u;
                    };
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                    for (int h = 1; h >= 0; h--) {
                        load_half(h);
#pragma unroll
                        for (int k = 0; k < HALF; k += 8)
#pragma unroll
                            for (int x = 0; x < 4; x++) top[x] = fmaxf(fmaxf(top[x], __uint_as_float(v[k + 2 * x])), __uint_as_float(v[k + 2 * x + 1]));
                    }
                    const float here = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * a.c;
                    float before = m;        // what the tile before took off
                    if (QT == 1 && i > 0) {
                        mbar_wait_bounded(smem_u32(&m_full[4 * (g ^ 1) + quad]), m_use & 1u, abort_flag, a.status, ST_TMEM_TIMEOUT);
                        m_use++;
                        before = m_rows[(g ^ 1) * 128 + 32 * quad + lane];
                    }
                    float now = before;
                    if (tile == 0) {
                        now = here;
                    } else if (__any_sync(0xffffffffu, here > before + GROWTH)) {
                        if (here > before + GROWTH) now = here;   // (a row by itself: what its neighbours see changes no bit of it)
                        const float by = now == -INFINITY ? 1.0f : exp2_fast(before - now);
                        const int last = i - (QT == 2 ? 2 : 1);   // the product that has to be there
                        mbar_wait_bounded(done_u + 8u * (uint32_t)(last & 1), (done[last & 1] + (uint32_t)(last >> 1)) & 1u, abort_flag, a.status, ST_TMEM_TIMEOUT);
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                        for (int k = 0; k < DP; k += 16) {
                            uint32_t o[16];
                            tmem_ld16(o_tm + (uint32_t)k, o);
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * by);
                            tmem_st16_start(o_tm + (uint32_t)k, o);
                        }
                        tmem_st_wait();
                    }
                    if (QT == 1 && i + 1 < n) {
                        m_rows[g * 128 + 32 * quad + lane] = now;
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&m_full[4 * g + quad]));
                    }
                    if (now != m) l *= m == -INFINITY ? 0.0f : exp2_fast(m - now);
                    m = now;
                    const float off = (m == -INFINITY ? 0.0f : -m) + WEIGHT_BIAS<C>;
                    const uint64_t c2 = pack_f32x2(a.c, a.c), off2 = pack_f32x2(off, off);
                    uint64_t sum[2] = {0, 0};
#pragma unroll 1
                    for (int h = 0; h < 2; h++) {
                        if (h) load_half(1);
#pragma unroll
                        for (int k = 0; k < HALF; k += 2) {
                            const float2 x = unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), c2, off2));
                            const float p = exp2_fast(x.x), r = exp2_fast(x.y);
                            sum[k / 2 % 2] = add_f32x2(sum[k / 2 % 2], pack_f32x2(p, r));
                            v[k / 2] = pack2<C>(p, r);
                        }
                        // (over scores that are in registers already)
#pragma unroll
                        for (int k = 0; k < HALF / 2; k += 16) tmem_st16_start(s_tm + (uint32_t)(h * HALF / 2 + k), v + k);
                    }
                    const float2 sums = unpack_f32x2(add_f32x2(sum[0], sum[1]));
                    l += sums.x + sums.y;
                }
                // Values of slots behind the last key that is seen may be anything, and so may values that some of the rows do not see: no product with
                // a weight of zero takes them away if they are no numbers.
                if (j0 + KEYS > least_item) {
                    // rows of this stage's values: from `lo` on some of the item's rows do not see them, from `seen` on none does; up to `rest` they came with a page
                    const int lo = max(0, least_item - j0), seen = w.seen - j0, rest = min(KEYS, (seen + a.box_rows - 1) / a.box_rows * a.box_rows);
#pragma unroll 1
                    for (int c = 0; c < NCH; c++) {
                        const uint32_t at = ring0 + at_values<QT, NCH>(tile, tiles) + c, st = at % STAGES;
                        mbar_wait_bounded(PAIR ? smem_u32(&v_here[st]) : smem_u32(&full[st]), (PAIR ? looked >> st : at / STAGES) & 1u, abort_flag, a.status, ST_WAIT_FULL_TIMEOUT);
                        // 16-byte pieces: eight to a row of a block of 64 elements, whose order in the row does not matter here
                        for (int u = 32 * quad + lane; u < (rest - lo) * (CW / 8); u += 128) {
                            const int j = lo + u / (CW / 8);
                            uint4* x = (uint4*)(ring + st * STAGE + u % (CW / 8) / 8 * BLOCK_BYTES + j * 128) + u % 8;
                            if (j >= seen) {
                                *x = make_uint4(0, 0, 0, 0);
                                continue;
                            }
                            const uint4 y = *x;
                            const uint4 bad = make_uint4(no_number<C>(y.x), no_number<C>(y.y), no_number<C>(y.z), no_number<C>(y.w));
                            if (bad.x | bad.y | bad.z | bad.w) {
                                spoilt[(item + 1) & 1] = item + 1;
                                if constexpr (PAIR) {    // (the other CTA's rows multiply these columns too)
                                    st_peer_f32(peer_smem(smem_u32((const void*)&spoilt[(item + 1) & 1]), (uint32_t)(rank ^ 1)), (uint32_t)(item + 1));
                                    asm volatile("fence.acq_rel.cluster;" ::: "memory");
                                }
                                __threadfence_block();   // (whoever finds these zeros finds the mark too)
                                *x = make_uint4(y.x & ~bad.x, y.y & ~bad.y, y.z & ~bad.z, y.w & ~bad.w);
                            }
                        }
                    }
                    fence_proxy_async();
                }
                tmem_st_wait();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive(p_bar);
            }
            if constexpr (PAIR)   // the stages whose values were waited for here, by either warpgroup
                for (int i = max(0, least_item / KEYS - w.from); i < tiles; i++) looked ^= 1u << ((ring0 + at_values<QT, NCH>(i, tiles)) % STAGES);
            ring0 += (uint32_t)(2 * tiles * NCH);
            there = walk_there(item + 2);
            if (QT == 1) {   // both warpgroups' maxima and sums: the later of the maxima is the larger
                m_rows[g * 128 + 32 * quad + lane] = m;
                l_rows[g * 128 + 32 * quad + lane] = l;
                named_bar_sync(1 + quad, 64);   // (the other warp of these rows; all scores of the item are there)
                const float m2 = m_rows[(g ^ 1) * 128 + 32 * quad + lane], l2 = l_rows[(g ^ 1) * 128 + 32 * quad + lane], top = fmaxf(m, m2);
                there = named_bar_all(1 + quad, 64, there);   // (both have read)
                l = l * (m == -INFINITY ? 0.0f : exp2_fast(m - top)) + l2 * (m2 == -INFINITY ? 0.0f : exp2_fast(m2 - top));   // (times zero: a sum that is no number stays none)
                m = top;
            }
            next = walks[(item + 2) & 7];
        }
    }
    // The last tile of rows, if others go on with it, is this CTA's to announce: its parts are this CTA's and those of the CTAs up to the one with its last unit.
    if (threadIdx.x == 128 && rank == 0) {
        Job job = {};
        if (any) {
            if (w.from == 0 && w.to < w.units) {
                // its parts: up to the last CTA that begins in it, no nearer to its end than a cut may lie
                const int last = plan->cut[1] + (w.units - w.to) - dear<DP>(w) - 1, each = plan->total / plan->active, rest = plan->total - each * plan->active;
                int c = min(plan->active - 1, (int)((float)last * (float)plan->active / (float)plan->total) + 1);   // (within one of it)
                while (c > cta && exact_cut(each, rest, plan->active, c) > last) c--;
                job.n_parts = c - cta + 1;
                job.first = w.first;
                job.past = w.past;
                job.kv = w.kv;
                job.row0 = w.row0;
                job.rows = w.rows;
            }
        }
        a.jobs[cta] = job;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (a.pdl) pdl_launch_dependents();
    if constexpr (PAIR) cluster_sync_all();   // both CTAs have read their sums, and nothing is on its way to the other's barriers
    if (warp == 1) {
        if (__builtin_expect(*abort_flag, 0)) settle_after_abort();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
    if constexpr (PAIR) cluster_sync_all();   // neither CTA leaves before both have given it back
}

// Joins the parts of tiles of rows.  A piece of work is 32 rows (the lanes: what a part left lies so) of one group of four elements where there are 16 parts or more, to
// which eight warps go with every eighth part, of two groups for four warps each from 8 parts on, of eight groups below.  The blocks share
// out the pieces of all tiles that were cut.  (A token behind 30000, 32 + 1 heads of 128, 148 parts: four warps 19.4 us in all, eight 16.7; six or eight parts on their way at once
// instead of four: larger tiles of rows 5 to 10 % slower.)
template <int DP>
__global__ void __launch_bounds__(256) attention_join_kernel(const AttnArgs a, float bias) {
    __shared__ int upto[256], sums[8];
    __shared__ float4 o_of[8][32];
    __shared__ float2 ml_of[8][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_jobs = a.ctas;
    if (a.pdl) pdl_wait_prior();
    // pieces of the jobs before and of each itself
    const auto warps_a_group = [](int n_parts) { return n_parts >= 16 ? 8 : n_parts >= 8 ? 4 : 1; };
    int n = 0;
    if ((int)threadIdx.x < n_jobs) {
        const Job j = a.jobs[threadIdx.x];
        if (j.n_parts > 0) n = (j.rows + 31) / 32 * (DP / 4 * warps_a_group(j.n_parts) / 8);
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, n, d);
        if (lane >= d) n += o;
    }
    if (lane == 31) sums[warp] = n;
    __syncthreads();
    for (int w = 0; w < warp; w++) n += sums[w];
    upto[threadIdx.x] = n;
    __syncthreads();
    const int total = upto[255];
    const long long slot = (long long)a.slot_rows * (DP + 4);
    for (int piece = (int)blockIdx.x; piece < total; piece += (int)gridDim.x) {
        int lo = 0;   // the first job whose pieces end behind this one
#pragma unroll
        for (int d = 128; d; d >>= 1)
            if (upto[lo + d - 1] <= piece) lo += d;
        const Job job = a.jobs[lo];
        const int in = piece - (lo ? upto[lo - 1] : 0), wpg = warps_a_group(job.n_parts), groups = 8 / wpg, chunks = DP / 4 / groups;
        const int row = in / chunks * 32 + lane, col = in % chunks * groups + warp / wpg, part = warp % wpg;
        const bool here = row < job.rows;
        float m = -INFINITY, l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const auto add = [&](float m2, float l2, const float4& o2) {
            const float top = fmaxf(m, m2), by = m == -INFINITY ? 0.0f : exp2_fast(m - top), by2 = m2 == -INFINITY ? 0.0f : exp2_fast(m2 - top);
            l = l * by + l2 * by2;
            o.x = o.x * by + o2.x * by2;
            o.y = o.y * by + o2.y * by2;
            o.z = o.z * by + o2.z * by2;
            o.w = o.w * by + o2.w * by2;
            m = top;
        };
        if (here) {
            constexpr int AHEAD = 4;
#pragma unroll 1
            for (int p0 = part; p0 < job.n_parts; p0 += wpg * AHEAD) {
                float2 ml[AHEAD];
                float4 x[AHEAD];
#pragma unroll
                for (int i = 0; i < AHEAD; i++) {
                    const int p = p0 + wpg * i;
                    ml[i] = make_float2(-INFINITY, 0.0f);
                    x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (p < job.n_parts) {
                        const float* s = a.slots + (p == 0 ? 2 * (long long)lo + 1 : 2 * ((long long)lo + p)) * slot;
                        ml[i] = *(const float2*)(s + (long long)a.slot_rows * DP + 2 * row);
                        x[i] = *(const float4*)(s + (long long)(col * a.slot_rows + row) * 4);
                    }
                }
#pragma unroll
                for (int i = 0; i < AHEAD; i++)
                    if (p0 + wpg * i < job.n_parts) add(ml[i].x, ml[i].y, x[i]);
            }
        }
        if (wpg > 1) {   // (the same for the whole block)
            o_of[warp][lane] = o;
            ml_of[warp][lane] = make_float2(m, l);
            __syncthreads();
            if (part == 0)
                for (int i = 1; i < wpg; i++) add(ml_of[warp + i][lane].x, ml_of[warp + i][lane].y, o_of[warp + i][lane]);
            __syncthreads();
        }
        if (part != 0 || !here) continue;
        const int tok = by_group(a, job.row0 + row), head = job.kv * a.group + job.row0 + row - tok * a.group, e = 4 * col;
        const long long out_row = job.first + tok;
        const bool sees = job.past + tok + 1 > 0;
        const float by = 1.0f / l;
        if (a.lse && e == 0) a.lse[out_row * a.n_heads + head] = sees ? 0.6931471805599453f * (m + (log2f(l) - bias)) : -INFINITY;
        const float f[4] = {o.x, o.y, o.z, o.w};
        store_four(a, out_row * a.out_row + (long long)head * a.out_head, e, f, by, sees);
    }
}

bool encode_pages(CUtensorMap* map, const q38b_paged_kv* c, const void* base, long long page, long long slot, long long head, int box_rows) {
    const cuuint64_t dims[4] = {(cuuint64_t)c->D, (cuuint64_t)c->page_size, (cuuint64_t)c->n_heads, (cuuint64_t)c->n_pages};
    // (the stride of one head or one page is never used: any that is allowed.  Heads of less than 256 bytes in [slot][head] pages: lines of 256
    // would fetch their neighbours', too: 64 sequences of 4000 tokens, 32 + 8 heads of 64, 142 us, 107 with lines of 128; heads of 256 elements are 1 % faster with 256)
    const cuuint64_t strides[3] = {(cuuint64_t)slot * 2, (cuuint64_t)(c->n_heads > 1 ? head : slot) * 2, (cuuint64_t)(c->n_pages > 1 ? page : slot) * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1}, estr[4] = {1, 1, 1, 1};
    EncodeTiledFn enc = encode_fn();
    return enc && enc(map, c->kind == Q38B_OUT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, (void*)base, dims, strides, box, estr,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, c->D < 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int ctas(const q38b_ctx* ctx) { return std::min(ctx->sm_count, 256); }   // (the joining kernel counts their work with a thread each)
int padded(int D) { return (D + 63) / 64 * 64; }
// rows of a place in the work area
int slot_rows(int group, int D, int rows) { return (int)std::min((long long)(padded(D) <= 128 ? 256 : 128), (long long)rows * group); }

template <typename C, int DP, int QT, bool PAIR = false>
int attention_as(q38b_ctx* ctx, const AttnArgs& a, const CUtensorMap& kmap, const CUtensorMap& vmap, cudaStream_t st) {
    using Sh = Shape<DP, QT, PAIR>;
    auto kern = attention_kernel<C, DP, QT, PAIR>;
    const int rc = q38b_ensure_kernel_smem(ctx, (const void*)kern, ctx->smem_optin, false);
    if (rc != Q38B_OK) return rc;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)(PAIR ? 2 * a.ctas : a.ctas));
    cfg.blockDim = dim3(Sh::THREADS);
    cfg.dynamicSmemBytes = Sh::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = PAIR ? 1 : 0;
    const int done = launch_status(ctx, cudaLaunchKernelEx(&cfg, kern, a, kmap, vmap));
    if (done != Q38B_OK) return done;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(4u * (unsigned)ctx->sm_count);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.pdl ? 1 : 0;
    return launch_status(ctx, cudaLaunchKernelEx(&cfg, attention_join_kernel<DP>, a, WEIGHT_BIAS<C>));
}
template <typename C>
int attention_for(q38b_ctx* ctx, const AttnArgs& a, bool two, const CUtensorMap& kmap, const CUtensorMap& vmap, cudaStream_t st) {
    switch (padded(a.D)) {
        case 64: return two ? attention_as<C, 64, 2>(ctx, a, kmap, vmap, st) : attention_as<C, 64, 1>(ctx, a, kmap, vmap, st);
        case 128: return two ? attention_as<C, 128, 2>(ctx, a, kmap, vmap, st) : attention_as<C, 128, 1>(ctx, a, kmap, vmap, st);
        case 192: return attention_as<C, 192, 1>(ctx, a, kmap, vmap, st);
        default: return two ? attention_as<C, 256, 1, true>(ctx, a, kmap, vmap, st) : attention_as<C, 256, 1>(ctx, a, kmap, vmap, st);
    }
}

bool known_kind(int kind) { return kind == Q38B_OUT_F32 || kind == Q38B_OUT_F16 || kind == Q38B_OUT_BF16; }
int kind_size(int kind) { return kind == Q38B_OUT_F32 ? 4 : 2; }

}  // namespace

extern "C" {

size_t q38b_attention_work_bytes(const q38b_ctx* ctx, int n_heads, int n_kv_heads, int D, int rows) {
    if (!ctx || n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads || D < 8 || D > 256 || D % 8 || rows < 1) return 0;
    return (size_t)ctas(ctx) * (sizeof(Job) + 2 * (size_t)slot_rows(n_heads / n_kv_heads, D, rows) * (padded(D) + 4) * 4);
}

int q38b_attention(q38b_ctx* ctx, const q38b_paged_kv* c, const void* q, int q_kind, long long q_row, long long q_head, int n_heads, float scale, void* out,
                   int out_kind, long long out_row, long long out_head, float* lse, int rows, void* work, size_t work_bytes, void* stream) {
    if (!ctx || !q || !out || !work || rows < 1 || !known_kind(q_kind) || !known_kind(out_kind) || !(scale > 0.0f) || !std::isfinite(scale)) return Q38B_ERR_ARG;
    int rc = paged_kv_check(c);
    if (rc != Q38B_OK) return rc;
    if (n_heads < 1 || n_heads % c->n_heads || q_row < 0 || q_head < 0 || out_row < 0 || out_head < 0) return Q38B_ERR_ARG;
    if ((n_heads > 1 && out_head < c->D) || (rows > 1 && out_row < c->D)) return Q38B_ERR_ARG;
    // rows lie outside heads, or heads outside rows
    if (n_heads > 1 && rows > 1 && out_row < (n_heads - 1) * out_head + c->D && out_head < (rows - 1) * out_row + c->D) return Q38B_ERR_ARG;
    if (q == out) return Q38B_ERR_ARG;   // (a row's queries may be read when another part of it is written)
    if (q_kind != Q38B_OUT_F32 && q_kind != c->kind) return Q38B_ERR_UNSUPPORTED;
    if (!attention_fits(c, n_heads, rows)) return Q38B_ERR_UNSUPPORTED;
    if ((uintptr_t)q % kind_size(q_kind) || (uintptr_t)out % kind_size(out_kind) || ((uintptr_t)lse & 3) || ((uintptr_t)work & 15)) return Q38B_ERR_ALIGN;
    if (work_bytes < 16 || work_bytes < q38b_attention_work_bytes(ctx, n_heads, c->n_heads, c->D, rows)) return Q38B_ERR_NOMEM;
    DeviceGuard on(ctx);
    AttnArgs a;
    memset(&a, 0, sizeof(a));
    a.batch = batch_of(c, rows);
    a.q = q; a.k = c->k; a.v = c->v; a.out = out; a.lse = lse;
    a.q_row = q_row; a.q_head = q_head; a.out_row = out_row; a.out_head = out_head;
    a.k_page = c->k_page; a.k_slot = c->k_slot; a.k_head = c->k_head; a.v_page = c->v_page; a.v_slot = c->v_slot; a.v_head = c->v_head;
    a.q_kind = q_kind; a.out_kind = out_kind; a.n_heads = n_heads; a.n_kv = c->n_heads; a.group = n_heads / c->n_heads; a.D = c->D;
    // Two tiles of rows share the keys' and values' way into shared memory, in one CTA (heads of at most 128) or in a pair of them (more than 192), where sequences fill
    // more than one on average and there are enough of them: of 12288 (row, head) pairs of 256 elements behind 2000 tokens 60.3 -> 51.8 us, 7512 pairs 40.5 -> 44.4; 32768 of 128
    // behind nothing 44.5 -> 36.2, 10016 14.0 -> 16.8.
    const bool two = ctx->attention_two ? ctx->attention_two > 0
                                        : (long long)rows * a.group > 128LL * c->n_seqs && (long long)rows * n_heads >= (padded(c->D) == 256 ? 80LL : 128LL) * ctx->sm_count;
    const bool pair = two && padded(c->D) == 256;
    a.box_rows = std::min(c->page_size, pair ? KEYS / 2 : KEYS);
    a.slot_rows = slot_rows(a.group, pair ? 128 : c->D, rows);
    a.ctas = pair ? ctas(ctx) / 2 : ctas(ctx);
    a.jobs = (Job*)work;
    a.slots = (float*)((uint8_t*)work + (size_t)ctas(ctx) * sizeof(Job));
    a.status = ctx->d_status;
    a.q_shift = q_kind == Q38B_OUT_F32 ? 2 : 1;
    a.q_vec = (((uintptr_t)q | (uintptr_t)(q_row * kind_size(q_kind)) | (uintptr_t)(q_head * kind_size(q_kind))) & 15) == 0;
    a.out_shift = out_kind == Q38B_OUT_F32 ? 2 : 1;
    const uintptr_t out_at = (uintptr_t)out | (uintptr_t)(out_row * kind_size(out_kind)) | (uintptr_t)(out_head * kind_size(out_kind)) | (uintptr_t)(c->D * kind_size(out_kind));
    a.out_vec = out_at % 32 == 0 ? 2 : out_at % 16 == 0 ? 1 : 0;
    a.pdl = ctx->pass_pdl ? 1 : 0;
    a.c = (float)((double)scale * 1.4426950408889634);
    int log = 0;
    while (1LL << log < a.group) log++;
    a.group_shift = 31 + log;
    a.group_mul = (uint32_t)(((1ULL << a.group_shift) + a.group - 1) / a.group);
    CUtensorMap kmap, vmap;
    if (!encode_pages(&kmap, c, c->k, c->k_page, c->k_slot, c->k_head, a.box_rows) || !encode_pages(&vmap, c, c->v, c->v_page, c->v_slot, c->v_head, a.box_rows)) return Q38B_ERR_ARG;
    return c->kind == Q38B_OUT_F16 ? attention_for<__half>(ctx, a, two, kmap, vmap, (cudaStream_t)stream) : attention_for<__nv_bfloat16>(ctx, a, two, kmap, vmap, (cudaStream_t)stream);
}

// Test hook (not in the public header): boxes of a stage and the warps that load them.
int q38b_debug_attention_loading(int D, int page_size, int pair, int* boxes, int* warps) {
    if (D < 8 || D > 256 || page_size < 8 || !boxes || !warps || (pair && padded(D) != 256)) return Q38B_ERR_ARG;
    *boxes = stage_boxes(std::min(page_size, pair ? KEYS / 2 : KEYS), padded(D) % 128 == 0 ? 128 : 64);
    *warps = loading_warps(*boxes);
    return Q38B_OK;
}

// Test hook (not in the public header): two tiles of rows together never (-1), wherever there is such a variant (1), by the rule (0).
int q38b_debug_set_attention_two(q38b_ctx* ctx, int mode) {
    if (!ctx || mode < -1 || mode > 1) return Q38B_ERR_ARG;
    ctx->attention_two = mode;
    return Q38B_OK;
}

}  // extern "C"

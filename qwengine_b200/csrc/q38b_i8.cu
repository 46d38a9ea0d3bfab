// q38b_i8.cu -- 8-bit integers with one scale a row: quantizer, and the product of two such matrices.
//
//   scale = max(fl32(amax / 127), 2^-126), code = x / scale rounded half to even (exactly)
//   Y[t][r] (+)= X_scales[t] W_scales[r] sum_k X[t][k] W[r][k]
//
// The sums are whole numbers below 2^31 (K <= 131071, codes of 8 bits): exact in any order, whatever splits K.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstring>
#include <type_traits>

#include "../../include/q38b200.h"
#include "q38b_host.h"
#include "q38b_internal.h"
#include "q38b_pipe.cuh"
#include "q38b_types.cuh"
#include "q38b_umma.cuh"

using namespace q38b;

namespace {

constexpr int I8_MAX_K = 131071;

// What a row's codes are made with.  inv is 1 / scale rounded: x inv is off by less than 2^-17 where the quotient is at most 127.5, so the nearest whole
// number n to it is the quotient's or, next to a half, one beside it.  x - n scale is exact in a fused operation (a multiple of the smaller of the two's last
// places, no larger than half a scale and a little), so comparing it with half the scale, itself exact, finds which, and ties.
struct RowScale { float scale, inv, half; uint32_t keep; };   // keep: the bits of the codes that stay
__device__ __forceinline__ RowScale row_scale(uint32_t top) {   // bit pattern of the largest magnitude; no number: a scale of NaN, codes of zero
    RowScale r;
    const bool bad = top >= 0x7F800000u;
    r.scale = bad ? __uint_as_float(0x7FC00000u) : fmaxf(__fdiv_rn(__uint_as_float(top), 127.0f), 1.17549435e-38f);
    r.inv = bad ? 0.0f : __fdiv_rn(1.0f, r.scale);
    r.half = bad ? INFINITY : 0.5f * r.scale;
    r.keep = bad ? 0u : ~0u;
    return r;
}
// Eight codes, each in the low byte of a word (rounding by an addition: conversions run at a quarter of the rate).  The remainders are looked at together: whether any of the
// eight may have to move is one branch (one for each made the kernel three times as long, and it waited for instructions).
constexpr float MAGIC = 12582912.0f;   // 1.5 * 2^23: whole numbers lie one apart
__device__ __forceinline__ void codes_of(const float (&x)[8], const RowScale& r, float (&t)[8]) {
    float worst = 0.0f;
    const uint64_t inv = pack_f32x2(r.inv, r.inv), scale = pack_f32x2(r.scale, r.scale), magic = pack_f32x2(MAGIC, MAGIC), minus = pack_f32x2(-1.0f, -1.0f);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint64_t v = pack_f32x2(x[i], x[i + 1]), u = fma_f32x2(v, inv, magic);
        const float2 rest = unpack_f32x2(fma_f32x2(fma_f32x2(u, minus, magic), scale, v)), c = unpack_f32x2(u);
        t[i] = c.x;
        t[i + 1] = c.y;
        worst = fmaxf(fmaxf(worst, fabsf(rest.x)), fabsf(rest.y));
    }
    if (worst >= r.half) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float rest = fmaf(MAGIC - t[i], r.scale, x[i]);
            const bool odd = (__float_as_uint(t[i]) & 1u) != 0u;
            t[i] += rest > r.half || (rest == r.half && odd) ? 1.0f : rest < -r.half || (rest == -r.half && odd) ? -1.0f : 0.0f;
        }
    }
}

// Eight neighbours of a row as they lie in memory
template <typename T> struct Raw8 { uint4 q[sizeof(T) / 2]; };
template <typename T> __device__ __forceinline__ void raw8_values(const Raw8<T>& r, float (&v)[8]) {
    const T* e = (const T*)r.q;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = to_f32(e[i]);
}
// the larger ones of two times two numbers, a NaN where either is one
template <typename T> __device__ __forceinline__ uint32_t max_nan2(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <typename T> __device__ __forceinline__ uint32_t raw8_top2(const Raw8<T>& r) {   // 16-bit types: the largest magnitudes of the even and of the odd four
    return max_nan2<T>(max_nan2<T>(r.q[0].x & 0x7FFF7FFFu, r.q[0].y & 0x7FFF7FFFu), max_nan2<T>(r.q[0].z & 0x7FFF7FFFu, r.q[0].w & 0x7FFF7FFFu));
}
template <typename T> __device__ __forceinline__ uint32_t top_of2(uint32_t m) {
    const unsigned short top = (unsigned short)max(m & 0x7FFFu, m >> 16 & 0x7FFFu);
    return __float_as_uint(to_f32(*(const T*)&top));
}
// the bit pattern (in fp32) of the largest magnitude: magnitudes compare like their bits, a NaN's exceeds them all
template <typename T> __device__ __forceinline__ uint32_t raw8_top(const Raw8<T>& r) {
    if constexpr (sizeof(T) == 2) {
        return top_of2<T>(raw8_top2<T>(r));
    } else {
        const float* v = (const float*)r.q;
        uint32_t top = 0u;
#pragma unroll
        for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
        return top;
    }
}

// A row to a warp, or to a block, whose threads have up to four pieces of eight neighbours each; they stay in registers between the largest magnitude and the
// codes, so that every value is read once.  What is longer than 20480 is read twice.  Bound by the issue of instructions (13 a value, 72 % of the issue slots) and memory: 17408 x
// 5120 from bf16 53 us (5.0 TB/s), 110 with single elements read twice; 77 x 5120 from fp32 2.3 us.
constexpr int PIECES = 4;
// VEC: whole pieces, aligned (the rest of a row's code, unused, took half of the instructions issued).  WARP: eight rows a block.
template <typename T, bool VEC, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 640, sizeof(T) == 2 && !WARP ? 2 : 1) i8_quantize_kernel(const T* x, long long x_ld, int K, int rows, int8_t* codes, long long codes_ld, float* scales) {
    pdl_launch_dependents();   // (a product behind it brings its first weights meanwhile)
    __shared__ uint32_t tops[32];
    const int threads = WARP ? 32 : (int)blockDim.x, t = WARP ? (int)threadIdx.x % 32 : (int)threadIdx.x;
    const long long row = WARP ? (long long)blockIdx.x * 8 + threadIdx.x / 32 : (long long)blockIdx.x;
    const int pieces = (K + 7) / 8;
    const bool here = row < rows;
    const T* p = x + row * x_ld;
    int8_t* to = codes + row * codes_ld;
    const auto load = [&](int u) {
        if constexpr (VEC) {
            return *(const Raw8<T>*)(p + 8 * u);
        } else {
            T e[8] = {};
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (8 * u + i < K) e[i] = p[8 * u + i];
            Raw8<T> r;
            memcpy(&r, e, sizeof(e));
            return r;
        }
    };
    Raw8<T> raw[PIECES] = {};
    uint32_t top = 0u;
#pragma unroll
    for (int j = 0; j < PIECES; j++)
        if (here && t + j * threads < pieces) raw[j] = load(t + j * threads);
    if constexpr (sizeof(T) == 2) {
        uint32_t m[PIECES];
#pragma unroll
        for (int j = 0; j < PIECES; j++) m[j] = raw8_top2<T>(raw[j]);
#pragma unroll
        for (int j = 1; j < PIECES; j++) m[0] = max_nan2<T>(m[0], m[j]);
        top = top_of2<T>(m[0]);
    } else {
#pragma unroll
        for (int j = 0; j < PIECES; j++) top = max(top, raw8_top<T>(raw[j]));
    }
    if (here)
        for (int u = t + PIECES * threads; u < pieces; u += threads) top = max(top, raw8_top<T>(load(u)));
    top = __reduce_max_sync(0xffffffffu, top);
    if constexpr (!WARP) {
        if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
        __syncthreads();
        top = __reduce_max_sync(0xffffffffu, (int)(threadIdx.x % 32) < threads / 32 ? tops[threadIdx.x % 32] : 0u);
    }
    if (!here) return;
    const RowScale s = row_scale(top);
    if (t == 0) scales[row] = s.scale;
    const auto store = [&](int u, const Raw8<T>& r) {
        float v[8], f[8];
        raw8_values<T>(r, v);
        codes_of(v, s, f);
        const uint32_t* c = (const uint32_t*)f;
        const uint2 w = make_uint2(__byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410) & s.keep,
                                   __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410) & s.keep);
        if (VEC || 8 * u + 8 <= K) {
            *(uint2*)(to + 8 * u) = w;
        } else {
#pragma unroll 1
            for (int i = 0; 8 * u + i < K; i++) to[8 * u + i] = (int8_t)((i < 4 ? w.x : w.y) >> (8 * (i % 4)));
        }
    };
#pragma unroll
    for (int j = 0; j < PIECES; j++)
        if (t + j * threads < pieces) store(t + j * threads, raw[j]);
    for (int u = t + PIECES * threads; u < pieces; u += threads) store(u, load(u));
}

// ---------------------------------------------------------------------------------------------------------------
// The product.  Weight rows are the MMA's M, tokens its N (as for the 4-bit product, whose stages of 128 bytes a row these are too), kind::i8, K = 32: exact sums in
// 32 bits of tensor memory.
//
// i8_gemm_kernel: a CTA owns 128 weight rows and up to 256 tokens.  One thread keeps a ring of stages of 128 K filled (tiled TMA, 128-byte swizzle, zeros behind the
// last K), one issues the MMAs, eight warps scale and store.  K may be shared by the CTAs of a cluster, whose sums meet in distributed shared memory.
// ---------------------------------------------------------------------------------------------------------------
constexpr int I8_ROWS = 128, I8_MAX_N = 256, I8_K = 128;
constexpr int I8_THREADS = 320, I8_MAX_STAGES = 12, I8_MAX_SPLITS = 8;
constexpr int I8_A_BYTES = I8_ROWS * I8_K;

struct I8Args {
    const float *w_scales, *x_scales;
    void* Y;
    long long ldy;
    int* status;
    int K, M, B, accumulate;
    int n_tile, stages, splits, pdl;
    int box_at;             // splits: where the others' sums come in shared memory; 0: over the ring
};
__host__ __device__ constexpr int i8_stage_bytes(int n_tile) { return I8_A_BYTES + n_tile * I8_K; }
__host__ __device__ constexpr uint32_t i8_tmem_cols(int n_tile) { return n_tile <= 32 ? 32u : n_tile <= 64 ? 64u : n_tile <= 128 ? 128u : 256u; }

// signed times signed, 32-bit sums, K-major
__device__ __forceinline__ uint32_t i8_idesc(int m, int n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
template <bool PAIR>
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    if constexpr (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}

template <typename T>
__global__ void __launch_bounds__(I8_THREADS, 2) i8_gemm_kernel(const I8Args a, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap) {
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* full = (uint64_t*)smem;
    uint64_t* empty = full + I8_MAX_STAGES;
    uint64_t* acc_done = empty + I8_MAX_STAGES;
    uint32_t* tmem_slot = (uint32_t*)(acc_done + 1);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    uint8_t* ring = smem + 1024;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = a.splits > 1 ? (int)cluster_rank() : 0;
    const int row0 = (int)(blockIdx.x / (unsigned)a.splits) * I8_ROWS, tok0 = (int)blockIdx.y * a.n_tile;
    const int n_tok = min(a.n_tile, a.B - tok0), n_mma = (n_tok + 15) / 16 * 16;
    const int steps = (a.K + I8_K - 1) / I8_K;
    const int s_begin = (int)((long long)steps * rank / a.splits), s_end = (int)((long long)steps * (rank + 1) / a.splits);
    const int stage_bytes = i8_stage_bytes(a.n_tile);
    const uint32_t tmem_cols = i8_tmem_cols(a.n_tile);
    auto ask_weights = [&](int s, int st) {   // and what the stage waits for altogether
        const uint32_t bar = smem_u32(&full[st]);
        mbar_arrive_expect_tx(bar, (uint32_t)stage_bytes);
        tma_load_2d(smem_u32(ring + st * stage_bytes), &wmap, s * I8_K, row0, bar);
    };
    auto ask_tokens = [&](int s, int st) { tma_load_2d(smem_u32(ring + st * stage_bytes) + I8_A_BYTES, &xmap, s * I8_K, tok0, smem_u32(&full[st])); };

    const int ahead = min(a.stages, s_end - s_begin);   // stages that need no waiting for
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < a.stages; s++) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        mbar_init(smem_u32(acc_done), 1);
        mbar_fence_init();
        fence_proxy_async();
        for (int i = 0; i < ahead; i++) ask_weights(s_begin + i, i);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = *tmem_slot;
    if (a.box_at) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");   // (this CTA has started; waited for in front of the exchange)
    if (a.pdl) pdl_wait_prior();

    if (warp == 0) {
        if (lane == 0) {
            for (int i = 0; i < ahead; i++) ask_tokens(s_begin + i, i);
            int st = 0;
            uint32_t use = 0;
            for (int s = s_begin + ahead; s < s_end; s++) {
                mbar_wait_bounded(smem_u32(&empty[st]), use, abort_flag, a.status, ST_WAIT_EMPTY_TIMEOUT);
                ask_weights(s, st);
                ask_tokens(s, st);
                if (++st == a.stages) { st = 0; use ^= 1u; }
            }
        }
    } else if (warp == 1) {
        int st = 0;
        uint32_t use = 0;
        const uint64_t desc0 = umma_desc_sw128(0);
        const uint32_t ring_at = smem_u32(ring), idesc = i8_idesc(I8_ROWS, n_mma);
        for (int s = s_begin; s < s_end; s++) {
            mbar_wait_bounded(smem_u32(&full[st]), use, abort_flag, a.status, ST_WAIT_FULL_TIMEOUT);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t at = ring_at + (uint32_t)(st * stage_bytes);
            const uint64_t ad = desc0 + (at >> 4), bd = desc0 + ((at + I8_A_BYTES) >> 4);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < I8_K / 32; k++) mma_i8<false>(tmem_base, ad + (uint64_t)(2 * k), bd + (uint64_t)(2 * k), idesc, k > 0 || s > s_begin ? 1u : 0u);
                umma_commit<false>(smem_u32(&empty[st]));
                if (s == s_end - 1) umma_commit<false>(smem_u32(acc_done));
            }
            __syncwarp();
            if (++st == a.stages) { st = 0; use ^= 1u; }
        }
    }

    // ---------------- warps 2..9 store: lanes 32 (warp % 4) .. + 31 of the accumulator are 32 rows; two warps share their tokens ----------------
    const int part = (warp - 2) >> 2;
    const int n_chunks = (n_tok + 15) / 16, quad = warp & 3, row = row0 + 32 * quad + lane;
    const uint32_t acc = tmem_base + ((uint32_t)(32 * quad) << 16);
    const float w_scale = row < a.M ? a.w_scales[row] : 0.0f;
    T* Y = (T*)a.Y;
    auto store = [&](int chunk, const int (&v)[16]) {
        if (row >= a.M) return;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const int t = 16 * chunk + j;
            if (t < n_tok) {
                T* y = Y + (size_t)(tok0 + t) * a.ldy + row;
                const float f = __int2float_rn(v[j]) * a.x_scales[tok0 + t] * w_scale;
                *y = from_f32<T>(a.accumulate ? to_f32(*y) + f : f);
            }
        }
    };
    if (warp >= 2) {
        mbar_wait_bounded(smem_u32(acc_done), 0u, abort_flag, a.status, ST_TMEM_TIMEOUT);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    }
    if (a.splits == 1) {
        if (warp >= 2)
            for (int chunk = part; chunk < n_chunks; chunk += 2) {
                uint32_t v[16];
                int f[16];
                tmem_ld16(acc + (uint32_t)(16 * chunk), v);
#pragma unroll
                for (int j = 0; j < 16; j++) f[j] = (int)v[j];
                store(chunk, f);
            }
    } else {
        // Chunk c of the tile is finished by rank c % splits: the others put their sums of it into that CTA's shared memory,
        // [source][c / splits][16 tokens][128 rows].  Few tokens have a place of their own there; more go over the ring, which every CTA's tensor core has read
        // by then.
        const int own_chunks = (n_chunks + a.splits - 1) / a.splits;
        const uint8_t* boxes = a.box_at ? smem + a.box_at : ring;
        const uint32_t box = smem_u32(boxes);
        __syncwarp();
        if (a.box_at) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
        else cluster_sync_all();
        if (warp >= 2)
            for (int chunk = part; chunk < n_chunks; chunk += 2) {
                const int owner = chunk % a.splits;
                if (owner == rank) continue;
                uint32_t v[16];
                tmem_ld16(acc + (uint32_t)(16 * chunk), v);
                const int src = rank - (rank > owner ? 1 : 0);
                const uint32_t to = peer_smem(box + (uint32_t)((src * own_chunks + chunk / a.splits) * (16 * I8_ROWS) + 32 * quad + lane) * 4u, (uint32_t)owner);
#pragma unroll
                for (int j = 0; j < 16; j++)
                    if (16 * chunk + j < n_tok) st_peer_f32(to + (uint32_t)(j * I8_ROWS * 4), v[j]);
            }
        cluster_sync_all();   // all sums have arrived; nobody touches another CTA's memory after this
        if (warp >= 2)
            for (int own = part; own * a.splits + rank < n_chunks; own += 2) {
                uint32_t v[16];
                int f[16];
                tmem_ld16(acc + (uint32_t)(16 * (own * a.splits + rank)), v);
#pragma unroll
                for (int j = 0; j < 16; j++) f[j] = (int)v[j];
                for (int r = 0; r < a.splits - 1; r++) {
                    const int* in = (const int*)boxes + (size_t)(r * own_chunks + own) * (16 * I8_ROWS) + 32 * quad + lane;
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        if (16 * (own * a.splits + rank) + j < n_tok) f[j] += in[j * I8_ROWS];
                }
                store(own * a.splits + rank, f);
            }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        if (__builtin_expect(*abort_flag, 0)) settle_after_abort();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(tmem_cols) : "memory");
    }
}

// ---------------------------------------------------------------------------------------------------------------
// Many tokens: two CTAs (a cluster of two) multiply as one, M = 256, each with 128 weight rows and half of the tokens.  The pairs stay and walk the tiles (tokens
// fastest: neighbours read the same weights out of L2), the ring runs on across tiles, two accumulators take turns, and eight warps bring one
// to registers and hand it back before they scale and store.  Outputs leave through shared memory and TMA stores where Y's base and row stride are multiples of 16 bytes.
// ---------------------------------------------------------------------------------------------------------------
constexpr int I8P_EPI_WARPS = 8;
constexpr int I8P_OUT_BYTES = 4096;   // one TMA store: 16 tokens (8 in 32 bits) x 128 rows; two halves of the storing warps with two buffers each
constexpr int I8P_FIXED_SMEM = 1024 + 4 * I8P_OUT_BYTES;

struct I8PairArgs {
    const float *w_scales, *x_scales;
    void* Y;
    long long ldy;
    int* status;
    int K, M, B, accumulate;
    int n_tile, stages, tok_tiles, n_tiles, pdl, tma_out;
};
__host__ __device__ constexpr int i8p_stage_bytes(int n_tile) { return I8_A_BYTES + n_tile / 2 * I8_K; }

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(I8_THREADS, 1)
i8_pair_kernel(const I8PairArgs a, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap ymap) {
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* full = (uint64_t*)smem;                // CTA 0's: the bytes of both CTAs
    uint64_t* empty = full + I8_MAX_STAGES;          // each CTA's
    uint64_t* acc_full = empty + I8_MAX_STAGES;      // [2] each CTA's
    uint64_t* acc_empty = acc_full + 2;              // [2] CTA 0's: the storing warps of both
    uint32_t* tmem_slot = (uint32_t*)(acc_empty + 2);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    uint8_t* ring = smem + I8P_FIXED_SMEM;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, side = (int)cluster_rank();
    const int pair = (int)(blockIdx.x >> 1), n_pairs = (int)(gridDim.x >> 1);
    const int steps = (a.K + I8_K - 1) / I8_K;
    const int stage_bytes = i8p_stage_bytes(a.n_tile);

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < a.stages; s++) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(smem_u32(&acc_full[i]), 1);
            mbar_init(smem_u32(&acc_empty[i]), 2 * I8P_EPI_WARPS);
        }
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync_all();   // the other CTA's barriers are initialised
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = *tmem_slot;
    if (a.pdl) pdl_wait_prior();

    if (warp == 0) {
        // (the whole warp walks and one elected lane issues, as for the MMA: the addresses stay in uniform registers)
        int st = 0;
        uint32_t use = 0;
        const uint32_t ring_at = smem_u32(ring), full_at = peer_smem(smem_u32(full), 0u);
        for (int tile = pair; tile < a.n_tiles; tile += n_pairs) {
            const int row0 = tile / a.tok_tiles * 256 + side * I8_ROWS, tok0 = tile % a.tok_tiles * a.n_tile;
            const int tok = tok0 + side * ((min(a.n_tile, a.B - tok0) + 31) / 32 * 16);
            for (int s = 0; s < steps; s++) {
                mbar_wait_bounded(smem_u32(&empty[st]), use ^ 1u, abort_flag, a.status, ST_WAIT_EMPTY_TIMEOUT);
                const uint32_t bar = full_at + 8u * (uint32_t)st, at = ring_at + (uint32_t)(st * stage_bytes);
                if (elect_one()) {
                    if (side == 0) mbar_arrive_expect_tx(smem_u32(&full[st]), 2u * (uint32_t)stage_bytes);
                    tma_load_2d_pair(at, &wmap, s * I8_K, row0, bar);
                    tma_load_2d_pair(at + I8_A_BYTES, &xmap, s * I8_K, tok, bar);
                }
                __syncwarp();
                if (++st == a.stages) { st = 0; use ^= 1u; }
            }
        }
    } else if (warp == 1) {
        if (side == 0) {
            int st = 0, acc = 0;
            uint32_t use = 0, acc_use = 0;
            const uint64_t desc0 = umma_desc_sw128(0);
            const uint32_t ring_at = smem_u32(ring);
            for (int tile = pair; tile < a.n_tiles; tile += n_pairs) {
                const int tok0 = tile % a.tok_tiles * a.n_tile, n_mma = (min(a.n_tile, a.B - tok0) + 31) / 32 * 32;
                const uint32_t d = tmem_base + (uint32_t)(acc * 256), idesc = i8_idesc(256, n_mma);
                mbar_wait_bounded(smem_u32(&acc_empty[acc]), acc_use ^ 1u, abort_flag, a.status, ST_TMEM_TIMEOUT);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int s = 0; s < steps; s++) {
                    mbar_wait_bounded(smem_u32(&full[st]), use, abort_flag, a.status, ST_WAIT_FULL_TIMEOUT);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t at = ring_at + (uint32_t)(st * stage_bytes);
                    const uint64_t ad = desc0 + (at >> 4), bd = desc0 + ((at + I8_A_BYTES) >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < I8_K / 32; k++) mma_i8<true>(d, ad + (uint64_t)(2 * k), bd + (uint64_t)(2 * k), idesc, k > 0 || s > 0 ? 1u : 0u);
                        umma_commit<true>(smem_u32(&empty[st]));
                        if (s == steps - 1) umma_commit<true>(smem_u32(&acc_full[acc]));
                    }
                    __syncwarp();
                    if (++st == a.stages) { st = 0; use ^= 1u; }
                }
                acc ^= 1;
                if (acc == 0) acc_use ^= 1u;
            }
        }
    } else {
        // a warp reads the 16-token chunks 2 i + part of its quarter of the rows
        const int quad = warp & 3, part = (warp - 2) >> 2;
        constexpr int OUT_TOK = I8P_OUT_BYTES / (I8_ROWS * (int)sizeof(T));
        uint8_t* out = smem + 1024 + part * 2 * I8P_OUT_BYTES;
        const bool storer = quad == 0 && lane == 0;
        int acc = 0, buf = 0;
        uint32_t acc_use = 0;
        T* Y = (T*)a.Y;
        for (int tile = pair; tile < a.n_tiles; tile += n_pairs) {
            const int row0 = tile / a.tok_tiles * 256 + side * I8_ROWS, row = row0 + 32 * quad + lane, tok0 = tile % a.tok_tiles * a.n_tile, n_tok = min(a.n_tile, a.B - tok0);
            const float w_scale = row < a.M ? a.w_scales[row] : 0.0f;
            mbar_wait_bounded(smem_u32(&acc_full[acc]), acc_use, abort_flag, a.status, ST_TMEM_TIMEOUT);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t from = tmem_base + ((uint32_t)(32 * quad) << 16) + (uint32_t)(acc * 256 + 16 * part);
            uint32_t v[8][16] = {};
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (16 * (2 * i + part) < n_tok) tmem_ld16_start(from + (uint32_t)(32 * i), v[i]);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; i++) tmem_ld_arrived(v[i]);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                if (side == 0) mbar_arrive(smem_u32(&acc_empty[acc]));
                else mbar_arrive_peer(peer_smem(smem_u32(&acc_empty[acc]), 0u));
            }
            acc ^= 1;
            if (acc == 0) acc_use ^= 1u;
            auto value = [&](int i, int j) {
                const int t = 16 * (2 * i + part) + j;
                const float f = __int2float_rn((int)v[i][j]) * (t < n_tok ? a.x_scales[tok0 + t] : 0.0f) * w_scale;
                if (!a.accumulate) return from_f32<T>(f);
                return row < a.M && t < n_tok ? from_f32<T>(to_f32(Y[(size_t)(tok0 + t) * a.ldy + row]) + f) : from_f32<T>(f);
            };
            // (a store is clipped in whole 16-byte units only: a last tile that ends inside one goes by plain stores)
            if (a.tma_out && (row0 + I8_ROWS <= a.M || a.M % (16 / (int)sizeof(T)) == 0)) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (16 * (2 * i + part) >= n_tok) break;
#pragma unroll
                    for (int h = 0; h < 16 / OUT_TOK; h++) {
                        if (storer) tma_store_wait_read<1>();
                        named_bar_sync(1 + part, 128);   // the buffer of two stores before is free
                        T* to = (T*)(out + buf * I8P_OUT_BYTES) + 32 * quad + lane;
#pragma unroll
                        for (int j = 0; j < OUT_TOK; j++) to[j * I8_ROWS] = value(i, OUT_TOK * h + j);
                        fence_proxy_async();
                        named_bar_sync(1 + part, 128);
                        if (storer && row0 < a.M) {
                            tma_store_2d(&ymap, smem_u32(out + buf * I8P_OUT_BYTES), row0, tok0 + 16 * (2 * i + part) + OUT_TOK * h);
                            tma_store_commit();
                        }
                        buf ^= 1;
                    }
                }
            } else if (row < a.M) {
#pragma unroll
                for (int i = 0; i < 8; i++)
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        const int t = 16 * (2 * i + part) + j;
                        if (t < n_tok) Y[(size_t)(tok0 + t) * a.ldy + row] = value(i, j);
                    }
            }
        }
        if (storer) tma_store_wait_all();
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync_all();   // both CTAs have read their accumulators, and nothing is on its way to the other's barriers
    if (warp == 1) {
        if (__builtin_expect(*abort_flag, 0)) settle_after_abort();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
    }
    cluster_sync_all();   // neither CTA leaves before both have given it back
}

// How a product is cut: tokens in tiles of n_tile, K in `splits` parts, few tokens with two CTAs to an SM, each with half of its shared memory.
struct I8Cut { int n_tile, stages, splits, box, per_sm; };   // box: bytes of shared memory for the others' sums (0: over the ring)

int exchange_bytes(const I8Cut& c) {
    const int chunks = c.n_tile / 16;
    return (c.splits - 1) * ((chunks + c.splits - 1) / c.splits) * 16 * I8_ROWS * 4;
}
int i8_ring_bytes(int smem_optin, const I8Cut& c) { return (c.per_sm == 2 ? (smem_optin + 1024) / 2 - 1024 : smem_optin) - 1024 - c.box; }

// ... by their time in SM clocks, of one wave of CTAs after the other: what starts and drains a CTA, the exchange of split sums, and stages, each as long as a CTA
// takes alone (two of an SM: twice) or, if that is longer, as its bytes take out of L2 (8600 a clock for all SMs; pairs 6450) and its weights out of DRAM
// (3200).  Fitted to 105 sizes (7 matrices, 1 to 2048 tokens) in every cut: the taken one is 1.7 % behind the best on average, 10 % at most (17408 x 5120, 256 tokens 32.4 us in single
// CTAs, 29.4 in pairs; 4096 x 4096, 1024 tokens 26.3 and 24.1).
I8Cut i8_cut(int sm_count, int smem_optin, int K, int M, int B, int forced_splits, int forced_per_sm, double* cost_of) {
    I8Cut best = {};
    double best_cost = 0.0;
    const int steps = (K + I8_K - 1) / I8_K, whole = B <= I8_MAX_N ? (B + 15) / 16 * 16 : I8_MAX_N;
    const auto rate = [&](int n, int per_sm) {
        if (forced_per_sm && per_sm != forced_per_sm) return;
        I8Cut c = {};
        c.n_tile = n;
        c.per_sm = per_sm;
        const long long tok_tiles = (B + n - 1) / n, tiles = (long long)((M + I8_ROWS - 1) / I8_ROWS) * tok_tiles;
        for (c.splits = 1; c.splits <= std::min(I8_MAX_SPLITS, steps); c.splits++) {
            if (forced_splits && c.splits != std::min(forced_splits, steps)) continue;
            const int own_steps = (steps + c.splits - 1) / c.splits;
            c.box = c.splits > 1 && n <= 32 ? exchange_bytes(c) : 0;
            c.stages = std::min(I8_MAX_STAGES, i8_ring_bytes(smem_optin, c) / i8_stage_bytes(n));
            if (c.splits > 1 && !c.box && exchange_bytes(c) > c.stages * i8_stage_bytes(n)) break;
            const int sms = c.splits <= 2 ? sm_count : c.splits <= 6 ? sm_count * 7 / 8 : sm_count * 7 / 10;
            const long long ctas = tiles * c.splits, once = std::max(1, sms / c.splits) * (long long)c.splits, slots = per_sm * once, waves = (ctas + slots - 1) / slots;
            if (per_sm == 2 && !forced_per_sm && (ctas <= once || own_steps < 4)) continue;
            const double active = (double)std::min(ctas, slots);
            const double stage = std::max({per_sm * (590.0 + 0.5 * n), active * i8_stage_bytes(n) / 8600.0, active / (double)tok_tiles * I8_A_BYTES / 3200.0});
            const double cost = 3600.0 + (double)waves * (own_steps * stage + (per_sm == 2 ? 0.0 : 2000.0) + 28.0 * n + (c.splits > 1 ? 1900.0 : 0.0));
            if (!best.n_tile || cost < best_cost) { best = c; best_cost = cost; }
        }
    };
    rate(whole, 1);
    if (whole > 128) rate(128, 1);
    if (whole <= 64) rate(whole, 2);
    if (cost_of) *cost_of = best_cost;
    return best;
}

// Tiles of a product in pairs: 64, 128, 192 or 256 tokens, by their time in SM clocks as above: rounds of tiles over the pairs.
struct I8PairCut { int n_tile, stages, tok_tiles, n_tiles; };
I8PairCut i8_pair_cut(int sm_count, int smem_optin, int K, int M, int B, int forced, double* cost_of) {
    I8PairCut best = {};
    double best_cost = 0.0;
    const int row_tiles = (M + 255) / 256, steps = (K + I8_K - 1) / I8_K;
    for (int n = 64; n <= 256; n += 64) {
        if (forced && n != forced) continue;
        I8PairCut c;
        c.n_tile = n;
        c.tok_tiles = (B + n - 1) / n;
        if ((long long)row_tiles * c.tok_tiles > 0x7FFFFFFF) continue;
        c.n_tiles = row_tiles * c.tok_tiles;
        c.stages = std::min(I8_MAX_STAGES, (smem_optin - I8P_FIXED_SMEM) / i8p_stage_bytes(n));
        const int pairs = sm_count / 2;
        const double active = (double)std::min(c.n_tiles, pairs);
        const double stage = std::max(310.0 + 1.2 * n, active * 2.0 * i8p_stage_bytes(n) / 6450.0), weights = active / c.tok_tiles * 2.0 * I8_A_BYTES / 3200.0;
        const double cost = 7800.0 + 25.0 * n + (double)((c.n_tiles + pairs - 1) / pairs) * std::max(steps * stage + 2200.0, steps * weights);
        if (!best.n_tile || cost < best_cost) { best = c; best_cost = cost; }
    }
    if (cost_of) *cost_of = best_cost;
    return best;
}

bool known_kind(int kind) { return kind == Q38B_OUT_F32 || kind == Q38B_OUT_F16 || kind == Q38B_OUT_BF16; }
size_t kind_size(int kind) { return kind == Q38B_OUT_F32 ? 4 : 2; }
bool i8_shape(int K, int rows) { return K >= 1 && K <= I8_MAX_K && rows >= 1 && rows <= 1 << 30; }
long long padded(int K) { return (K + 15) / 16 * 16; }

int check_operand(const void* codes, long long ld, const float* scales, int K, int rows) {
    if (!codes || !scales || !i8_shape(K, rows) || ld < K) return Q38B_ERR_ARG;
    return ((uintptr_t)codes & 15) || (ld & 15) || ((uintptr_t)scales & 3) ? Q38B_ERR_ALIGN : Q38B_OK;
}

template <typename T>
int quantize_as(q38b_ctx* ctx, const void* x, long long x_ld, int K, int rows, int8_t* codes, long long codes_ld, float* scales, cudaStream_t st) {
    // a warp a row and eight rows a block where that is enough, otherwise a block a row
    const int pieces = (K + 7) / 8, warps = std::min(20, (pieces + 32 * PIECES - 1) / (32 * PIECES));
    const bool vec = K % 8 == 0 && (((uintptr_t)x | (uintptr_t)(x_ld * (long long)sizeof(T))) & 15) == 0;
    const T* p = (const T*)x;
    if (warps == 1) {
        const unsigned grid = (unsigned)((rows + 7LL) / 8);
        if (vec) i8_quantize_kernel<T, true, true><<<grid, 256, 0, st>>>(p, x_ld, K, rows, codes, codes_ld, scales);
        else i8_quantize_kernel<T, false, true><<<grid, 256, 0, st>>>(p, x_ld, K, rows, codes, codes_ld, scales);
    } else {
        if (vec) i8_quantize_kernel<T, true, false><<<(unsigned)rows, (unsigned)(32 * warps), 0, st>>>(p, x_ld, K, rows, codes, codes_ld, scales);
        else i8_quantize_kernel<T, false, false><<<(unsigned)rows, (unsigned)(32 * warps), 0, st>>>(p, x_ld, K, rows, codes, codes_ld, scales);
    }
    return launch_status(ctx, cudaSuccess);
}

bool encode_codes(CUtensorMap* map, const void* codes, long long ld, int K, int rows, int box_rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {I8_K, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    EncodeTiledFn enc = encode_fn();
    return enc && enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)codes, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// the outputs, stored in pieces of I8P_OUT_BYTES; false: they go there by plain stores
bool encode_out(CUtensorMap* map, void* Y, int kind, long long ldy, int M, int B) {
    const int size = (int)kind_size(kind);
    if (((uintptr_t)Y & 15) || (ldy * size) % 16) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)M, (cuuint64_t)B};
    const cuuint64_t strides[1] = {(cuuint64_t)ldy * size};
    const cuuint32_t box[2] = {I8_ROWS, (cuuint32_t)(I8P_OUT_BYTES / (I8_ROWS * size))}, estr[2] = {1, 1};
    EncodeTiledFn enc = encode_fn();
    return enc && enc(map, kind == Q38B_OUT_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : kind == Q38B_OUT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, Y,
                      dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T>
int pair_as(q38b_ctx* ctx, const I8PairArgs& a, const CUtensorMap& wmap, const CUtensorMap& xmap, const CUtensorMap& ymap, cudaStream_t st) {
    auto kern = i8_pair_kernel<T>;
    const int rc = q38b_ensure_kernel_smem(ctx, (const void*)kern, ctx->smem_optin, false);
    if (rc != Q38B_OK) return rc;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(2u * (unsigned)std::min(ctx->sm_count / 2, a.n_tiles));
    cfg.blockDim = dim3(I8_THREADS);
    cfg.dynamicSmemBytes = (size_t)(I8P_FIXED_SMEM + a.stages * i8p_stage_bytes(a.n_tile));
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.pdl ? 1 : 0;
    return launch_status(ctx, cudaLaunchKernelEx(&cfg, kern, a, wmap, xmap, ymap));
}

template <typename T>
int gemm_as(q38b_ctx* ctx, const I8Args& a, int box, const CUtensorMap& wmap, const CUtensorMap& xmap, cudaStream_t st) {
    auto kern = i8_gemm_kernel<T>;
    const int rc = q38b_ensure_kernel_smem(ctx, (const void*)kern, ctx->smem_optin, false);
    if (rc != Q38B_OK) return rc;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)((a.M + I8_ROWS - 1) / I8_ROWS * a.splits), (unsigned)((a.B + a.n_tile - 1) / a.n_tile));
    cfg.blockDim = dim3(I8_THREADS);
    cfg.dynamicSmemBytes = (size_t)(1024 + a.stages * i8_stage_bytes(a.n_tile) + box);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (a.splits > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = (unsigned)a.splits;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        n++;
    }
    if (a.pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        n++;
    }
    cfg.attrs = attr;
    cfg.numAttrs = (unsigned)n;
    return launch_status(ctx, cudaLaunchKernelEx(&cfg, kern, a, wmap, xmap));
}

// the product of two such matrices; behind_quantizer: launched while the kernel that makes X still runs, where the context allows it
int gemm_i8(q38b_ctx* ctx, const void* W, long long W_ld, const float* W_scales, int K, int M, const void* X, long long X_ld, const float* X_scales, int B, void* Y, int y_kind,
            long long ldy, int accumulate, void* stream, bool behind_quantizer) {
    if (!ctx || !Y || !known_kind(y_kind) || ldy < M) return Q38B_ERR_ARG;
    int rc = check_operand(W, W_ld, W_scales, K, M);
    if (rc == Q38B_OK) rc = check_operand(X, X_ld, X_scales, K, B);
    if (rc != Q38B_OK) return rc;
    if ((uintptr_t)Y % kind_size(y_kind)) return Q38B_ERR_ALIGN;
    DeviceGuard on(ctx);
    cudaStream_t st = (cudaStream_t)stream;
    const int pdl = behind_quantizer && ctx->pass_pdl ? 1 : 0;
    const int forced_pairs = ctx->i8_cut > 0 && ctx->i8_cut >= 64 ? ctx->i8_cut : 0, forced_one = ctx->i8_cut < 0 ? -ctx->i8_cut : 0;   // test hook
    double cost = 0.0, pair_cost = 0.0;
    const I8Cut one = i8_cut(ctx->sm_count, ctx->smem_optin, K, M, B, forced_one % 10, forced_one / 10, &cost);
    const I8PairCut cut = i8_pair_cut(ctx->sm_count, ctx->smem_optin, K, M, B, forced_pairs, &pair_cost);
    const bool too_many = !one.n_tile || (B + one.n_tile - 1) / one.n_tile > 65535;   // token tiles, for a grid's second dimension
    if (forced_pairs || too_many || (!forced_one && M > I8_ROWS && pair_cost < cost)) {
        if (!cut.n_tile) return Q38B_ERR_UNSUPPORTED;
        CUtensorMap wmap, xmap, ymap;
        memset(&ymap, 0, sizeof(ymap));
        const int tma_out = encode_out(&ymap, Y, y_kind, ldy, M, B) ? 1 : 0;
        if (!encode_codes(&wmap, W, W_ld, K, M, I8_ROWS) || !encode_codes(&xmap, X, X_ld, K, B, cut.n_tile / 2)) return Q38B_ERR_ARG;
        const I8PairArgs a = {W_scales, X_scales, Y, ldy, ctx->d_status, K, M, B, accumulate ? 1 : 0, cut.n_tile, cut.stages, cut.tok_tiles, cut.n_tiles, pdl, tma_out};
        return y_kind == Q38B_OUT_F32 ? pair_as<float>(ctx, a, wmap, xmap, ymap, st)
             : y_kind == Q38B_OUT_F16 ? pair_as<__half>(ctx, a, wmap, xmap, ymap, st)
                                      : pair_as<__nv_bfloat16>(ctx, a, wmap, xmap, ymap, st);
    }
    CUtensorMap wmap, xmap;
    if (!encode_codes(&wmap, W, W_ld, K, M, I8_ROWS) || !encode_codes(&xmap, X, X_ld, K, B, one.n_tile)) return Q38B_ERR_ARG;
    const I8Args a = {W_scales, X_scales, Y, ldy, ctx->d_status, K, M, B, accumulate ? 1 : 0, one.n_tile, one.stages, one.splits, pdl,
                      one.box ? 1024 + one.stages * i8_stage_bytes(one.n_tile) : 0};
    return y_kind == Q38B_OUT_F32 ? gemm_as<float>(ctx, a, one.box, wmap, xmap, st)
         : y_kind == Q38B_OUT_F16 ? gemm_as<__half>(ctx, a, one.box, wmap, xmap, st)
                                  : gemm_as<__nv_bfloat16>(ctx, a, one.box, wmap, xmap, st);
}

}  // namespace

extern "C" {

int q38b_quantize_i8(q38b_ctx* ctx, const void* x, int x_kind, long long x_ld, int K, int rows, void* codes, long long codes_ld, float* scales, void* stream) {
    if (!ctx || !x || !known_kind(x_kind) || x_ld < K) return Q38B_ERR_ARG;
    const int rc = check_operand(codes, codes_ld, scales, K, rows);
    if (rc != Q38B_OK) return rc;
    if ((uintptr_t)x % kind_size(x_kind)) return Q38B_ERR_ALIGN;
    DeviceGuard on(ctx);
    cudaStream_t st = (cudaStream_t)stream;
    return x_kind == Q38B_OUT_F32 ? quantize_as<float>(ctx, x, x_ld, K, rows, (int8_t*)codes, codes_ld, scales, st)
         : x_kind == Q38B_OUT_F16 ? quantize_as<__half>(ctx, x, x_ld, K, rows, (int8_t*)codes, codes_ld, scales, st)
                                  : quantize_as<__nv_bfloat16>(ctx, x, x_ld, K, rows, (int8_t*)codes, codes_ld, scales, st);
}

int q38b_gemm_i8(q38b_ctx* ctx, const void* W, long long W_ld, const float* W_scales, int K, int M, const void* X, long long X_ld, const float* X_scales, int B,
                 void* Y, int y_kind, long long ldy, int accumulate, void* stream) {
    return gemm_i8(ctx, W, W_ld, W_scales, K, M, X, X_ld, X_scales, B, Y, y_kind, ldy, accumulate, stream, false);
}

size_t q38b_gemm_i8_scratch_bytes(int K, int B) { return i8_shape(K, B) ? (size_t)B * (size_t)padded(K) + ((size_t)B * 4 + 15) / 16 * 16 : 0; }

int q38b_gemm_i8_x(q38b_ctx* ctx, const void* W, long long W_ld, const float* W_scales, int K, int M, const void* x, int x_kind, long long x_ld, int B, void* Y,
                   int y_kind, long long ldy, int accumulate, void* scratch, size_t scratch_bytes, void* stream) {
    if (!ctx || !x || !Y || !known_kind(x_kind) || !known_kind(y_kind) || x_ld < K || !i8_shape(K, B)) return Q38B_ERR_ARG;
    int rc = check_operand(W, W_ld, W_scales, K, M);
    if (rc != Q38B_OK) return rc;
    if (ldy < M || !scratch) return Q38B_ERR_ARG;
    if ((uintptr_t)x % kind_size(x_kind) || (uintptr_t)Y % kind_size(y_kind) || ((uintptr_t)scratch & 15)) return Q38B_ERR_ALIGN;
    if (scratch_bytes < q38b_gemm_i8_scratch_bytes(K, B)) return Q38B_ERR_NOMEM;
    uint8_t* codes = (uint8_t*)scratch;
    float* scales = (float*)(codes + (size_t)B * (size_t)padded(K));
    rc = q38b_quantize_i8(ctx, x, x_kind, x_ld, K, B, codes, padded(K), scales, stream);
    if (rc != Q38B_OK) return rc;
    return gemm_i8(ctx, W, W_ld, W_scales, K, M, codes, padded(K), scales, B, Y, y_kind, ldy, accumulate, stream, true);
}

// Test hook (not in the public header): products in pairs of CTAs with tiles of `mode` tokens (64, 128, 192, 256); never in pairs and K in -mode % 10 parts, -mode / 10
// CTAs to an SM (0 in either place: by the rule); everything by the rule (0).
int q38b_debug_set_i8_cut(q38b_ctx* ctx, int mode) {
    if (!ctx || mode > 256 || (mode > 0 && mode % 64) || mode < -28 || -mode % 10 == 9) return Q38B_ERR_ARG;
    ctx->i8_cut = mode;
    return Q38B_OK;
}

}  // extern "C"

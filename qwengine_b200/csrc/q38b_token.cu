// q38b_token.cu -- the element-wise steps of a token between its products: norms and rotation of the query and key heads, and
// the rules that shape the logits before the top-k.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "../../include/q38b200.h"
#include "q38b_host.h"
#include "q38b_internal.h"
#include "q38b_pipe.cuh"
#include "q38b_types.cuh"

using namespace q38b;

namespace {

// ---------------------------------------------------------------------------------------------------------------
// Query and key heads.  z = x / sqrt(mean(x^2) + eps) * w;  y_a = z_a c - z_b n, y_b = z_b c + z_a n over the pairs of the first R
// elements, c = s cos(pos f_j), n = s sin(pos f_j).  A position times a frequency loses the angle in 32 bits (from position 2^17
// on its error passes 0.01), so the angle is taken in turns as a 64-bit fraction: F = frac(f / 2 pi) 2^64 once per pair, pos * F modulo
// 2^64 exactly in integers.  Its upper 32 bits less their nearest quarter turn become a float, which holds that remainder to 2^-28 turns (all of a half turn
// only to 2^-26: cosines were off by up to 1.1e-7).
// ---------------------------------------------------------------------------------------------------------------
struct HeadsArgs {
    q38b_heads t[2];
    const int* positions;
    const double* inv_freq;
    int D, rot, adjacent, rows;
    float eps, scale, inv_d;
};

__device__ __forceinline__ unsigned long long turn_fraction(double inv_freq) {
    const double t = inv_freq * 0.15915494309189533577;   // 1 / (2 pi)
    return __double2ull_rz((t - floor(t)) * 18446744073709551616.0);
}
// (Taylor series on an eighth of a turn; all 2^30 + 1 remainders compared: sines within 6.1e-8, cosines within 7.8e-8, the float in them.  sincospif of the same
// remainder, with its own reduction, 5e-8, but 4096 rows of 16 + 4 heads of 512, all rotated, 101 us against 86 in the kernel that has an angle a lane.)
__device__ __forceinline__ void turn_sincos(unsigned long long f, int pos, float scale, float& s, float& c) {
    // the angle in turns, 2^-32 each, and half a quarter: the upper two bits are the nearest quarter's number, what lies below them is the remainder
    const uint32_t t = (uint32_t)(((unsigned long long)(long long)pos * f) >> 32) + 0x20000000u;
    const float x = (float)((int)(t & 0x3FFFFFFFu) - 0x20000000) * 4.656612873077393e-10f, z = x * x;   // in half turns (2^-31): -1/4 .. 1/4
    // sin pi x = pi x - (pi x)^3 / 3! + .. + (pi x)^9 / 9! with pi in two parts, cos pi x = 1 - (pi x)^2 / 2! + .. - (pi x)^10 / 10!
    const float sn = fmaf(x, 3.14159274f, x * fmaf(z, fmaf(z, fmaf(z, fmaf(z, 0.0821458866f, -0.599264529f), 2.55016404f), -5.16771278f), -8.74227766e-8f));
    const float cs = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -0.0258068913f, 0.235330630f), -1.33526277f), 4.05871213f), -4.93480220f), 1.0f);
    const bool odd = t & 0x40000000u;
    s = __uint_as_float(__float_as_uint(odd ? cs : sn) ^ (t & 0x80000000u)) * scale;
    c = __uint_as_float(__float_as_uint(odd ? sn : cs) ^ ((t + 0x40000000u) & 0x80000000u)) * scale;
}

// Any size, stride and alignment: one warp per (row, head), element by element; every head computes its row's angles anew.  Bound by the issue of instructions
// and by waiting for its own loads: 4096 rows of 16 + 4 heads of 512 in 16 bits, all rotated, 88 us, of 8 + 2 heads of 1024 85 (floor 26); 8192 rows of 24 + 4
// heads of 256 at odd strides, fp32 to bf16, 104 (floor 55).  Six CTAs an SM (40 registers; 48 as the compiler would have it: 109 at the latter);
// only the sum's loop unrolled, whose loads then overlap (by two: 110 for 512, by one 126).
template <typename Tin, typename Tout>
__global__ void __launch_bounds__(256, 6) heads_kernel(const HeadsArgs a) {
    const int lane = threadIdx.x & 31, n_heads = a.t[0].n_heads + a.t[1].n_heads;
    const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= (long long)a.rows * n_heads) return;
    const int row = (int)(item / n_heads);
    int h = (int)(item % n_heads);
    const q38b_heads& t = a.t[h >= a.t[0].n_heads];
    if (h >= a.t[0].n_heads) h -= a.t[0].n_heads;
    const Tin* src = (const Tin*)t.src + row * t.src_row + h * t.src_head;
    Tout* dst = (Tout*)t.dst + row * t.dst_row + h * t.dst_head;
    float ss = 0.0f;
    for (int i = lane; i < a.D; i += 32) {
        const float v = to_f32(src[i]);
        ss = fmaf(v, v, ss);
    }
#pragma unroll
    for (int s = 16; s; s >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, s);
    const float r = rsqrtf(ss * a.inv_d + a.eps);
    const int half = a.rot / 2;
#pragma unroll 1
    for (int j = lane; j < half; j += 32) {
        const int ia = a.adjacent ? 2 * j : j, ib = a.adjacent ? 2 * j + 1 : j + half;
        float sn, cs;
        turn_sincos(turn_fraction(a.inv_freq[j]), a.positions[row], a.scale, sn, cs);
        const float za = to_f32(src[ia]) * r * (t.weight ? t.weight[ia] : 1.0f), zb = to_f32(src[ib]) * r * (t.weight ? t.weight[ib] : 1.0f);
        dst[ia] = from_f32<Tout>(za * cs - zb * sn);
        dst[ib] = from_f32<Tout>(zb * cs + za * sn);
    }
#pragma unroll 1
    for (int i = a.rot + lane; i < a.D; i += 32) dst[i] = from_f32<Tout>(to_f32(src[i]) * r * (t.weight ? t.weight[i] : 1.0f));
}

// Heads of up to 256 elements whose rows allow it move four elements a lane at a time.  A CTA has one row (its sines and cosines are computed
// once, into shared memory) and up to HEADS_BATCH heads a warp, whose loads are all issued first; a head's L lanes add its squares by
// shuffles and swap partners of the rotation through shared memory.  Bound by memory: 8192 rows of 24 + 4 heads of 256, fp32 to bf16, 62 us =
// 5.7 TB/s (four heads a warp, eight warps a CTA, three CTAs an SM 77) against 104 us element by element, where every head's warp computes its own angles.
constexpr int HEADS_BATCH = 2, HEADS_WARPS = 4, HEADS_MAX_D = 256;

template <typename T> __device__ __forceinline__ float4 load4(const T* p) {
    if constexpr (sizeof(T) == 4) return *(const float4*)p;
    const uint2 q = *(const uint2*)p;
    T e[4];
    memcpy(e, &q, 8);
    return make_float4(to_f32(e[0]), to_f32(e[1]), to_f32(e[2]), to_f32(e[3]));
}
template <typename T> __device__ __forceinline__ void store4(T* p, float4 v) {
    if constexpr (sizeof(T) == 4) {
        *(float4*)p = v;
    } else {
        const T e[4] = {from_f32<T>(v.x), from_f32<T>(v.y), from_f32<T>(v.z), from_f32<T>(v.w)};
        uint2 q;
        memcpy(&q, e, 8);
        *(uint2*)p = q;
    }
}

// Two 32-bit products or sums of products an instruction (8192 rows of 32 + 8 heads of 128 in 16 bits 47.3 us, 48.7 one by one)
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 w, {%6, %7};\n\tfma.rn.f32x2 z, x, y, w;\n\tmov.b64 {%0, %1}, z;\n\t}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 lo2(float4 v) { return make_float2(v.x, v.y); }
__device__ __forceinline__ float2 hi2(float4 v) { return make_float2(v.z, v.w); }
__device__ __forceinline__ float4 both(float2 a, float2 b) { return make_float4(a.x, a.y, b.x, b.y); }
__device__ __forceinline__ float4 mul4(float4 a, float4 b) { return both(mul2(lo2(a), lo2(b)), mul2(hi2(a), hi2(b))); }
__device__ __forceinline__ float4 fma4(float4 a, float4 b, float4 c) { return both(fma2(lo2(a), lo2(b), lo2(c)), fma2(hi2(a), hi2(b), hi2(c))); }
// L lanes a head (two heads a warp where 16 do, four where 8), NV vectors of four elements a lane: two, so that what a head costs beside its
// elements is paid half as often (4096 rows of 32 + 8 heads of 128, 16 bits, all rotated, 24.8 us, with one vector 30; four vectors
// 37; more heads a CTA, one batch after the other, 28).  A CTA has heads of one tensor: its pointers and weights
// are the same for all of them (with heads of both in a CTA 68 us, bound by the issue of instructions: 232 a head, 74 % of the slots).
template <typename Tin, typename Tout, int L, int NV>
__global__ void __launch_bounds__(32 * HEADS_WARPS, 10) heads4_kernel(const HeadsArgs a, int heads_per_cta, int q_ctas, int ctas_per_row) {
    constexpr int SUB = 32 / L, STEP = HEADS_WARPS * SUB;
    __shared__ float cs[HEADS_MAX_D / 2], sn[HEADS_MAX_D / 2];
    __shared__ float4 swap[HEADS_WARPS][32 * NV];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, l = lane % L, half = a.rot / 2;
    const int row = (int)(blockIdx.x / (unsigned)ctas_per_row), c = (int)(blockIdx.x % (unsigned)ctas_per_row);
    const q38b_heads& t = a.t[c >= q_ctas];
    const int h0 = (c >= q_ctas ? c - q_ctas : c) * heads_per_cta, h_end = min(t.n_heads, h0 + heads_per_cta), h_mine = h0 + warp * SUB + lane / L;
    const Tin* src = (const Tin*)t.src + row * t.src_row + h_mine * t.src_head + 4 * l;
    float4 x[HEADS_BATCH][NV];
#pragma unroll
    for (int b = 0; b < HEADS_BATCH; b++)
#pragma unroll
        for (int i = 0; i < NV; i++)
            x[b][i] = h_mine + b * STEP < h_end && 4 * (l + L * i) < a.D ? load4(src + b * STEP * t.src_head + 4 * L * i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (tid < half) turn_sincos(turn_fraction(a.inv_freq[tid]), a.positions[row], a.scale, sn[tid], cs[tid]);
    float4 w[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) w[i] = t.weight && 4 * (l + L * i) < a.D ? __ldg((const float4*)(t.weight + 4 * (l + L * i))) : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
    Tout* dst = (Tout*)t.dst + row * t.dst_row + h_mine * t.dst_head + 4 * l;
    __syncthreads();
#pragma unroll
    for (int b = 0; b < HEADS_BATCH; b++) {
        if (h0 + warp * SUB + b * STEP >= h_end) break;   // (the whole warp)
        float2 s2 = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < NV; i++) s2 = fma2(hi2(x[b][i]), hi2(x[b][i]), fma2(lo2(x[b][i]), lo2(x[b][i]), s2));
        float ss = s2.x + s2.y;
#pragma unroll
        for (int s = L / 2; s; s >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, s);
        const float r = rsqrtf(ss * a.inv_d + a.eps);
#pragma unroll
        for (int i = 0; i < NV; i++) {
            float4& z = x[b][i];
            z = mul4(mul4(z, make_float4(r, r, r, r)), w[i]);
        }
        if (a.adjacent) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int j = 2 * (l + L * i);   // pairs j and j + 1
                float4& z = x[b][i];
                if (j < half) {
                    const float2 c2 = *(const float2*)(cs + j), n2 = *(const float2*)(sn + j);   // (behind the last pair: whatever is there)
                    const float2 p = make_float2(z.x, z.z), o = make_float2(z.y, z.w), u = fma2(o, make_float2(-n2.x, -n2.y), mul2(p, c2)), q = fma2(p, n2, mul2(o, c2));
                    z = j + 1 < half ? make_float4(u.x, q.x, u.y, q.y) : make_float4(u.x, q.x, z.z, z.w);
                }
            }
        } else if (half) {
            float4* mine = swap[warp] + lane / L * L * NV;
#pragma unroll
            for (int i = 0; i < NV; i++)
                if (4 * (l + L * i) < a.rot) mine[l + L * i] = x[b][i];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int e = 4 * (l + L * i);
                if (e < a.rot) {
                    const bool second = e >= half;
                    const int other = second ? e - half : e + half, j = second ? other : e;
                    const float4 o = mine[other / 4], cj = *(const float4*)(cs + j);
                    float4 n = *(const float4*)(sn + j);
                    if (!second) n = make_float4(-n.x, -n.y, -n.z, -n.w);
                    float4& z = x[b][i];
                    z = fma4(o, n, mul4(z, cj));
                }
            }
            __syncwarp();
        }
        if (h_mine + b * STEP < h_end) {
#pragma unroll
            for (int i = 0; i < NV; i++)
                if (4 * (l + L * i) < a.D) store4(dst + b * STEP * t.dst_head + 4 * L * i, x[b][i]);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------
// Logits.  count_v: times token v occurs among the generated tokens of the row, seen_v: in prompt or generated ones.
//   seen: l = l > 0 ? l / rep : l * rep;  l -= freq * count_v;  count_v > 0: l -= pres;  l += bias_v;  mask bit clear: l = -inf
// A CTA owns CHUNK logits of a row.  Their loads are issued first (four neighbours a lane where rows are aligned to 16 bytes, else one: any
// stride will do; in place nothing is loaded and only masked logits are written).  While they are on their way the CTA counts the row's tokens
// that fall among them in shared memory (whole numbers, so the order of the atomics does not matter): a bit for each that occurs, a count for
// each generated one.  Then the logits pass through the mask, and those that occur, few, are mended from where they were read: a lane has the bits of
// the logits 512 apart, so that a warp's share of a bit is 32 neighbours, and places are packed so that no warp computes for one lane.  Biases
// come last, the last entry of each token found in the same shared words.
// Every CTA of a row reads the whole text, so a CTA takes many logits where there are many rows (logits_in), and an id costs
// six instructions (difference, comparison, address, bit, predicated atomics).  128 rows of 248320: nothing but the counting of one token each
// 41.5 us = 6.1 TB/s, 16000 tokens of prompt 60, 4000 generated ones 50, both with masks and 32 biases 73.7 = 3.6 TB/s; where the ends of a row were
// asked for at every place and texts had lengths instead of ends (registers spilled) 43.5, 61, 53 and 77.5.  Before that, without the bits, every word of
// the counts looked through, 49, 76, 62 and 90; bits of 32 neighbours to a lane, whose 32 places at a time lie in 32 lines, 44, 76, 63 and 93; 32 places
// mended at a time instead of 64, read back from where they were written, 44, 63, 53 and 79.5.  What was slower there: clusters that
// share a text by atomics in each other's memory (101 alone, 111 in twos, 161 in eights, all with 8192 logits a CTA); CTAs that stay and bring
// the next piece's logits ahead (138); half of the warps counting a piece ahead of the others (112 mending in memory, 156 in registers): a warp
// then waits too often for too few others; logits mended in registers before their only store, which then waits (95); logits read after
// the counting, with three CTAs to an SM (81 to 86); text of the next step on its way during this one's counting (89, registers spilled).
// ---------------------------------------------------------------------------------------------------------------
constexpr int LG_THREADS = 512, LG_WARPS = LG_THREADS / 32, LG_MAX_N = 1 << 30;

struct LogitsArgs {
    const float* x;
    float* y;
    long long x_ld, y_ld;
    q38b_logit_rules r;
    int n, index_offset;
};

// Counts those of [ids, end) that are among the n logits from `first` on: a bit for each that occurs, a count for each generated one.
// (Unsigned: ids below the first and negative ones fall out with those behind the last.)
template <bool GENERATED>
__device__ __forceinline__ void count_id(uint32_t words, uint32_t occurs, int id, uint32_t first, uint32_t n) {
    const uint32_t at = (uint32_t)id - first, word = occurs + at % LG_THREADS * 4u, bit = 1u << (at / LG_THREADS & 31u);
    if constexpr (GENERATED)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.u32 p, %0, %1;\n\t@p red.shared.or.b32 [%2], %3;\n\t@p red.shared.add.u32 [%4], 1;\n\t}" ::"r"(at), "r"(n), "r"(word), "r"(bit), "r"(words + 4u * at) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.u32 p, %0, %1;\n\t@p red.shared.or.b32 [%2], %3;\n\t}" ::"r"(at), "r"(n), "r"(word), "r"(bit) : "memory");
}
template <bool GENERATED>
__device__ __forceinline__ void count_ids(uint32_t words, uint32_t occurs, const int* ids, const int* end, uint32_t first, uint32_t n, int tid) {
    if (end <= ids) return;
    // four ids a load, two loads of a thread ahead of their atomics; the ends that are no whole 16 bytes by themselves
    const int head = (int)min((long long)(end - ids), (long long)((16 - ((uintptr_t)ids & 15)) & 15) / 4);
    if (tid < head) count_id<GENERATED>(words, occurs, ids[tid], first, n);
    const int4* q = (const int4*)(ids + head) + tid;
    const int4* q_end = (const int4*)((uintptr_t)end & ~(uintptr_t)15);   // (behind a head that reaches the end: before q)
    for (; q + LG_THREADS < q_end; q += 2 * LG_THREADS) {
        const int4 a = __ldg(q), b = __ldg(q + LG_THREADS);
        count_id<GENERATED>(words, occurs, a.x, first, n);
        count_id<GENERATED>(words, occurs, a.y, first, n);
        count_id<GENERATED>(words, occurs, a.z, first, n);
        count_id<GENERATED>(words, occurs, a.w, first, n);
        count_id<GENERATED>(words, occurs, b.x, first, n);
        count_id<GENERATED>(words, occurs, b.y, first, n);
        count_id<GENERATED>(words, occurs, b.z, first, n);
        count_id<GENERATED>(words, occurs, b.w, first, n);
    }
    if (q < q_end) {
        const int4 a = __ldg(q);
        count_id<GENERATED>(words, occurs, a.x, first, n);
        count_id<GENERATED>(words, occurs, a.y, first, n);
        count_id<GENERATED>(words, occurs, a.z, first, n);
        count_id<GENERATED>(words, occurs, a.w, first, n);
    }
    // (a head that reaches the end leaves no tail)
    const int* tail = (const int*)q_end + tid;
    if (tid < 4 && tail >= ids + head && tail < end) count_id<GENERATED>(words, occurs, *tail, first, n);
}

// VEC: rows of x and y are aligned to 16 bytes, a lane has four neighbours at a time.
template <int CHUNK, bool VEC>
__global__ void __launch_bounds__(LG_THREADS, CHUNK <= 4096 ? 3 : 2) logits_kernel(const LogitsArgs a) {
    constexpr int E = VEC ? 4 : 1, WARP = 32 * E, STEP = LG_THREADS * E;   // logits of a lane, a warp, the block at a time
    constexpr int UN = CHUNK / STEP;                                       // ... of a lane altogether
    extern __shared__ __align__(16) uint32_t times[];                      // [CHUNK] of generated tokens, where there are texts or biases
    __shared__ uint32_t occurs[LG_THREADS];                                // bit b: the token of logit 512 b + the thread occurs
    __shared__ uint16_t packed[LG_WARPS][96];
    const int row = blockIdx.y, c0 = blockIdx.x * CHUNK, n = min(CHUNK, a.n - c0), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t first = (uint32_t)(a.index_offset + c0);
    const bool counts = a.r.history != nullptr, in_place = a.x == a.y;
    const float* x = a.x + row * a.x_ld + c0;
    float* y = a.y + row * a.y_ld + c0;
    // what the later parts need, on its way before the logits
    const int *text = nullptr, *generated_text = nullptr, *text_end = nullptr;
    long long bias0 = 0;
    int n_bias = 0;
    if (counts) {
        const long long begin = a.r.history_begin[row], end = a.r.history_begin[row + 1];
        text = a.r.history + begin;
        text_end = a.r.history + end;
        generated_text = text + (a.r.prompt_len ? max(0LL, min((long long)a.r.prompt_len[row], end - begin)) : 0LL);
    }
    if (a.r.bias_ids) {
        bias0 = a.r.bias_begin[row];
        n_bias = (int)(a.r.bias_begin[row + 1] - bias0);
    }
    const int m = !a.r.masks ? -1 : a.r.mask_of_row ? a.r.mask_of_row[row] : row;
    const uint32_t* mask = a.r.masks + (m >= 0 ? m * a.r.mask_ld : 0);
    const uint32_t mask_end = (uint32_t)(a.index_offset + a.n - 1) >> 5;
    auto allowed = [&](uint32_t at) { return m < 0 || (mask[(first + at) >> 5] >> ((first + at) & 31u) & 1u); };
    // the logits on their way
    float v[UN][E];
    const bool whole = VEC && n == CHUNK && !in_place;   // nothing to ask of a place
    if (whole) {
        if constexpr (VEC) {
#pragma unroll
            for (int u = 0; u < UN; u++) {
                const float4 q = *(const float4*)(x + STEP * u + E * tid);
                v[u][0] = q.x; v[u][1] = q.y; v[u][2] = q.z; v[u][3] = q.w;
            }
        }
    } else if (!in_place) {
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const int i = STEP * u + E * tid;
            if constexpr (VEC) {
                const float4 q = i + 3 < n ? *(const float4*)(x + i)   // (or the row's last one to three)
                                           : make_float4(i < n ? x[i] : 0.0f, i + 1 < n ? x[i + 1] : 0.0f, i + 2 < n ? x[i + 2] : 0.0f, 0.0f);
                v[u][0] = q.x; v[u][1] = q.y; v[u][2] = q.z; v[u][3] = q.w;
            } else {
                v[u][0] = i < n ? x[i] : 0.0f;
            }
        }
    }
    // the mask bits of the warp's logits: lane E u + k has those of the k-th 32 of its u-th WARP
    uint32_t bits = 0xFFFFFFFFu;
    const int masked_at = STEP * (lane / E) + WARP * warp + 32 * (lane % E);
    if (m >= 0 && lane < E * UN && masked_at < n) {
        const uint32_t at = first + (uint32_t)masked_at;
        bits = __funnelshift_r(mask[at >> 5], mask[min((at >> 5) + 1u, mask_end)], at & 31u);
    }
    // biases among the block's logits; a thread keeps its first one's place
    const uint32_t bias_at = tid < n_bias ? (uint32_t)a.r.bias_ids[bias0 + tid] - first : 0xFFFFFFFFu;
    bool any = bias_at < (uint32_t)n;
    for (int j = tid + LG_THREADS; j < n_bias; j += LG_THREADS) any |= (uint32_t)a.r.bias_ids[bias0 + j] - first < (uint32_t)n;
    if (counts)
        for (int i = 4 * tid; i < CHUNK; i += 4 * LG_THREADS) *(uint4*)(times + i) = make_uint4(0, 0, 0, 0);
    if (counts) {
        occurs[tid] = 0u;
        __syncthreads();
        count_ids<false>(smem_u32(times), smem_u32(occurs), text, generated_text, first, (uint32_t)n, tid);
        count_ids<true>(smem_u32(times), smem_u32(occurs), generated_text, text_end, first, (uint32_t)n, tid);
    }
    // ... and through
    const float minus_inf = __int_as_float(0xFF800000);
    if (whole) {
        if constexpr (VEC) {
#pragma unroll
            for (int u = 0; u < UN; u++) {
                const uint32_t keep = __shfl_sync(0xffffffffu, bits, E * u + E * lane / 32) >> (E * lane % 32);
                *(float4*)(y + STEP * u + E * tid) = make_float4(keep & 1u ? v[u][0] : minus_inf, keep & 2u ? v[u][1] : minus_inf, keep & 4u ? v[u][2] : minus_inf, keep & 8u ? v[u][3] : minus_inf);
            }
        }
    } else if (!in_place || m >= 0) {
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const int i = STEP * u + E * tid;
            const uint32_t keep = __shfl_sync(0xffffffffu, bits, E * u + E * lane / 32) >> (E * lane % 32);
            if constexpr (VEC) {
                if (i + 3 < n && !in_place) {
                    *(float4*)(y + i) = make_float4(keep & 1u ? v[u][0] : minus_inf, keep & 2u ? v[u][1] : minus_inf, keep & 4u ? v[u][2] : minus_inf, keep & 8u ? v[u][3] : minus_inf);
                } else {   // in place, and the row's last one to three
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        if (i + k >= n) break;
                        if (!(keep >> k & 1u)) y[i + k] = minus_inf;
                        else if (!in_place) y[i + k] = v[u][k];
                    }
                }
            } else if (i < n) {
                if (!(keep & 1u)) y[i] = minus_inf;
                else if (!in_place) y[i] = v[u][0];
            }
        }
    }
    if (!counts && !a.r.bias_ids) return;
    any = __syncthreads_or(any);   // (every id is counted, and every logit through)
    if (counts) {
        const float repetition = a.r.penalties[3 * row], frequency = a.r.penalties[3 * row + 1], presence = a.r.penalties[3 * row + 2];
        // a lane has the bits of its logits and gives one at a time; places are packed and mended 64 at a time, two to a lane
        uint16_t* mine = packed[warp];
        int waiting = 0;
        auto mend = [&](int from, int k) {   // k of the packed places
            uint32_t at[2];
            float l[2];
            bool on[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                on[h] = lane + 32 * h < k;
                at[h] = on[h] ? mine[from + lane + 32 * h] : 0u;
                if (on[h]) l[h] = x[at[h]];
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if (on[h] && allowed(at[h])) {
                    const uint32_t generated = times[at[h]];
                    float z = l[h] > 0.0f ? __fdiv_rn(l[h], repetition) : l[h] * repetition;
                    if (generated) z = z - frequency * (float)generated - presence;
                    y[at[h]] = z;
                }
            }
            __syncwarp();
        };
        uint32_t left = occurs[tid];
        while (const uint32_t giving = __ballot_sync(0xffffffffu, left != 0u)) {
            if (left) mine[waiting + __popc(giving & ((1u << lane) - 1u))] = (uint16_t)(LG_THREADS * (__ffs(left) - 1) + tid);
            left &= left - 1u;
            waiting += __popc(giving);
            __syncwarp();
            if (waiting >= 64) {   // the last 64
                waiting -= 64;
                mend(waiting, 64);
            }
        }
        mend(0, waiting);
    }
    if (!any) return;
    const long long from = a.r.bias_begin[row], count = a.r.bias_begin[row + 1] - from;   // (again: not kept in registers)
    const int* ids = a.r.bias_ids + from;
    auto each = [&](auto&& f) {   // f(entry, place) for this thread's biases among the block's logits
        if (bias_at < (uint32_t)n) f((uint32_t)tid, bias_at);
        for (long long j = tid + LG_THREADS; j < count; j += LG_THREADS) {
            const uint32_t at = (uint32_t)ids[j] - first;
            if (at < (uint32_t)n) f((uint32_t)j, at);
        }
    };
    __syncthreads();
    each([&](uint32_t, uint32_t at) { times[at] = 0u; });
    __syncthreads();
    each([&](uint32_t j, uint32_t at) { atomicMax(&times[at], j + 1u); });
    __syncthreads();
    each([&](uint32_t j, uint32_t at) {
        if (times[at] == j + 1u && allowed(at)) y[at] += a.r.bias_values[from + j];
    });
}

bool known_kind(int kind) { return kind == Q38B_OUT_F32 || kind == Q38B_OUT_F16 || kind == Q38B_OUT_BF16; }
uintptr_t kind_size(int kind) { return kind == Q38B_OUT_F32 ? 4 : 2; }

// whether four elements can move at a time
bool heads_by_four(const HeadsArgs& a, uintptr_t in_size, uintptr_t out_size) {
    if (a.D > HEADS_MAX_D || a.D % 4 || (!a.adjacent && a.rot / 2 % 4)) return false;
    for (const q38b_heads& t : a.t) {
        if (!t.n_heads) continue;
        if ((uintptr_t)t.src % (4 * in_size) || (uintptr_t)t.dst % (4 * out_size) || (uintptr_t)t.weight % 16) return false;
        if ((t.src_head | t.dst_head) % 4 || (a.rows > 1 && (t.src_row | t.dst_row) % 4)) return false;
    }
    return true;
}

template <typename Tin, typename Tout>
int heads_as(q38b_ctx* ctx, const HeadsArgs& a, cudaStream_t st) {
    const int n_heads = a.t[0].n_heads + a.t[1].n_heads;
    if (heads_by_four(a, sizeof(Tin), sizeof(Tout))) {
        // as many heads a CTA as its warps take at once, fewer where rows alone leave SMs idle
        const int once = HEADS_WARPS * (a.D <= 64 ? 4 : a.D <= 128 ? 2 : 1);
        int per = once * HEADS_BATCH;
        const auto ctas = [&](int n, int of) { return (n + of - 1) / of; };
        while (per > once && (long long)a.rows * (ctas(a.t[0].n_heads, per) + ctas(a.t[1].n_heads, per)) < 2 * ctx->sm_count) per -= once;
        const int q = ctas(a.t[0].n_heads, per), all = q + ctas(a.t[1].n_heads, per);
        const long long grid = (long long)a.rows * all;
        if (grid > 0x7FFFFFFF) return Q38B_ERR_UNSUPPORTED;
        if (a.D <= 64) heads4_kernel<Tin, Tout, 8, 2><<<(unsigned)grid, 32 * HEADS_WARPS, 0, st>>>(a, per, q, all);
        else if (a.D <= 128) heads4_kernel<Tin, Tout, 16, 2><<<(unsigned)grid, 32 * HEADS_WARPS, 0, st>>>(a, per, q, all);
        else heads4_kernel<Tin, Tout, 32, 2><<<(unsigned)grid, 32 * HEADS_WARPS, 0, st>>>(a, per, q, all);
        return launch_status(ctx, cudaSuccess);
    }
    const long long blocks = ((long long)a.rows * n_heads + 7) / 8;
    if (blocks > 0x7FFFFFFF) return Q38B_ERR_UNSUPPORTED;
    heads_kernel<Tin, Tout><<<(unsigned)blocks, 256, 0, st>>>(a);
    return launch_status(ctx, cudaSuccess);
}
template <typename Tin>
int heads_from(q38b_ctx* ctx, const HeadsArgs& a, int out_kind, cudaStream_t st) {
    return out_kind == Q38B_OUT_F32 ? heads_as<Tin, float>(ctx, a, st) : out_kind == Q38B_OUT_F16 ? heads_as<Tin, __half>(ctx, a, st) : heads_as<Tin, __nv_bfloat16>(ctx, a, st);
}

template <int CHUNK, bool VEC>
int logits_as(q38b_ctx* ctx, const LogitsArgs& a, int n_rows, cudaStream_t st) {
    const int rc = q38b_ensure_kernel_smem(ctx, (const void*)logits_kernel<CHUNK, VEC>, CHUNK * 4, false);
    if (rc != Q38B_OK) return rc;
    const size_t smem = a.r.history || a.r.bias_ids ? CHUNK * 4 : 0;
    logits_kernel<CHUNK, VEC><<<dim3((unsigned)((a.n + CHUNK - 1) / CHUNK), (unsigned)n_rows), LG_THREADS, smem, st>>>(a);
    return launch_status(ctx, cudaSuccess);
}
template <bool VEC>
int logits_in(q38b_ctx* ctx, const LogitsArgs& a, int n_rows, cudaStream_t st) {
    // The least time by waves of CTAs, three to an SM (two of 8192 and 16384 logits): what a wave takes beside what every call takes, in parts
    // of some 0.3 us, more where each CTA reads a text; a last wave that is not full counts half, but for the largest.  (Before, the most logits that
    // left three CTAs to every SM: 4 rows of 248320 then were 488 CTAs for 444 places and took 5.1 us, 11.6 with 20000 tokens, biases and masks; so
    // 4.3 and 10.6, 16 rows 8.1 -> 7.4 and 17.6 -> 15.2.)
    const int chunks[] = {16384, 8192, 4096, 2048}, per_sm[] = {2, 2, 3, 3}, wave[] = {30, 20, 18, 12}, wave_of_texts[] = {30, 21, 22, 18};
    int best = 0;
    double least = 0.0;
    for (int i = 0; i < 4; i++) {
        if (i < 3 && a.n <= chunks[i] / 2) continue;   // (half of its threads would have nothing)
        const double waves = (double)n_rows * ((a.n + chunks[i] - 1) / chunks[i]) / (per_sm[i] * ctx->sm_count), whole = std::ceil(waves);
        const double time = (i == 0 ? whole : std::max(1.0, (whole + waves) / 2.0)) * (a.r.history ? wave_of_texts[i] : wave[i]);
        if (!best || time < least) { best = chunks[i]; least = time; }
    }
    return best == 16384 ? logits_as<16384, VEC>(ctx, a, n_rows, st) : best == 8192 ? logits_as<8192, VEC>(ctx, a, n_rows, st)
         : best == 4096  ? logits_as<4096, VEC>(ctx, a, n_rows, st) : logits_as<2048, VEC>(ctx, a, n_rows, st);
}

}  // namespace

int q38b_logit_rules_check(const q38b_logit_rules* rules, int n, int index_offset) {
    if (n > LG_MAX_N) return Q38B_ERR_UNSUPPORTED;
    if (!rules->penalties != !rules->history || !rules->history != !rules->history_begin || (rules->prompt_len && !rules->history)) return Q38B_ERR_ARG;
    if (!rules->bias_ids != !rules->bias_values || !rules->bias_ids != !rules->bias_begin) return Q38B_ERR_ARG;
    if ((rules->mask_of_row && !rules->masks) || (rules->masks && rules->mask_ld < ((long long)index_offset + n + 31) / 32)) return Q38B_ERR_ARG;
    if (((uintptr_t)rules->penalties | (uintptr_t)rules->history | (uintptr_t)rules->prompt_len | (uintptr_t)rules->bias_ids | (uintptr_t)rules->bias_values |
         (uintptr_t)rules->masks | (uintptr_t)rules->mask_of_row) & 3)
        return Q38B_ERR_ALIGN;
    return ((uintptr_t)rules->history_begin | (uintptr_t)rules->bias_begin) & 7 ? Q38B_ERR_ALIGN : Q38B_OK;
}

extern "C" {

int q38b_qk_norm_rope(q38b_ctx* ctx, const q38b_heads* q, const q38b_heads* k, int D, int rot, int adjacent, float eps, float scale, const int* positions,
                      const double* inv_freq, int in_kind, int out_kind, int rows, void* stream) {
    if (!ctx || !q || D < 1 || D > 1024 || rot < 0 || rot > D || rot % 2 || rows < 1 || !known_kind(in_kind) || !known_kind(out_kind)) return Q38B_ERR_ARG;
    if (rot > 0 && (!positions || !inv_freq)) return Q38B_ERR_ARG;
    HeadsArgs a;
    memset(&a, 0, sizeof(a));
    a.t[0] = *q;
    if (k) a.t[1] = *k;
    for (int i = 0; i < (k ? 2 : 1); i++) {
        const q38b_heads& t = a.t[i];
        if (!t.src || !t.dst || t.n_heads < 1 || t.src_head < 0 || t.dst_head < 0 || t.src_row < 0 || t.dst_row < 0) return Q38B_ERR_ARG;
        // no two heads of one destination share elements: rows lie outside heads, or heads outside rows
        const long long in_row = (t.n_heads - 1) * t.dst_head + D, in_head = (rows - 1) * t.dst_row + D;
        if ((t.n_heads > 1 && t.dst_head < D) || (rows > 1 && t.dst_row < D)) return Q38B_ERR_ARG;
        if (t.n_heads > 1 && rows > 1 && t.dst_row < in_row && t.dst_head < in_head) return Q38B_ERR_ARG;
        if ((uintptr_t)t.src % kind_size(in_kind) || (uintptr_t)t.dst % kind_size(out_kind) || ((uintptr_t)t.weight & 3)) return Q38B_ERR_ALIGN;
        // in place only element over element (the strides of one head, of one row say nothing)
        if (t.src == t.dst && (in_kind != out_kind || (t.n_heads > 1 && t.src_head != t.dst_head) || (rows > 1 && t.src_row != t.dst_row))) return Q38B_ERR_ARG;
    }
    if (((uintptr_t)positions & 3) || ((uintptr_t)inv_freq & 7)) return Q38B_ERR_ALIGN;
    a.D = D;
    a.rot = rot;
    a.adjacent = adjacent ? 1 : 0;
    a.rows = rows;
    a.eps = eps;
    a.scale = scale;
    a.inv_d = 1.0f / (float)D;
    a.positions = positions;
    a.inv_freq = inv_freq;
    DeviceGuard on(ctx);
    cudaStream_t st = (cudaStream_t)stream;
    return in_kind == Q38B_OUT_F32 ? heads_from<float>(ctx, a, out_kind, st) : in_kind == Q38B_OUT_F16 ? heads_from<__half>(ctx, a, out_kind, st)
                                                                                                     : heads_from<__nv_bfloat16>(ctx, a, out_kind, st);
}

int q38b_adjust_logits(q38b_ctx* ctx, const float* x, long long x_ld, int n, int n_rows, int index_offset, const q38b_logit_rules* rules, float* y, long long y_ld,
                       void* stream) {
    if (!ctx || !x || !y || !rules || n < 1 || n_rows < 1 || n_rows > 65535 || index_offset < 0 || index_offset > 0x7FFFFFFF - n) return Q38B_ERR_ARG;
    if (n > LG_MAX_N) return Q38B_ERR_UNSUPPORTED;
    if (n_rows > 1 && (x_ld < n || y_ld < n)) return Q38B_ERR_ARG;
    if (x == y && n_rows > 1 && x_ld != y_ld) return Q38B_ERR_ARG;
    if (((uintptr_t)x | (uintptr_t)y) & 3) return Q38B_ERR_ALIGN;
    const int rc = q38b_logit_rules_check(rules, n, index_offset);
    if (rc != Q38B_OK) return rc;
    LogitsArgs a;
    a.x = x;
    a.y = y;
    a.x_ld = x_ld;
    a.y_ld = y_ld;
    a.r = *rules;
    a.n = n;
    a.index_offset = index_offset;
    DeviceGuard on(ctx);
    cudaStream_t st = (cudaStream_t)stream;
    const bool vec = (((uintptr_t)x | (uintptr_t)y) & 15) == 0 && (n_rows == 1 || ((x_ld | y_ld) & 3) == 0);
    return vec ? logits_in<true>(ctx, a, n_rows, st) : logits_in<false>(ctx, a, n_rows, st);
}

}  // extern "C"

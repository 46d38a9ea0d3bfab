// q38b_token.cu -- the element-wise steps of a token between its products: norms and rotation of the query and key heads, and
// the rules that shape the logits before the top-k.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

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
// 2^64 exactly in integers, its upper 32 bits to sin and cos of pi x.
// ---------------------------------------------------------------------------------------------------------------
struct HeadsArgs {
    q38b_heads t[2];
    const int* positions;
    const double* inv_freq;
    int D, rot, adjacent, rows;
    float eps, scale;
};

__device__ __forceinline__ unsigned long long turn_fraction(double inv_freq) {
    const double t = inv_freq * 0.15915494309189533577;   // 1 / (2 pi)
    return __double2ull_rz((t - floor(t)) * 18446744073709551616.0);
}
__device__ __forceinline__ void turn_sincos(unsigned long long f, int pos, float scale, float& s, float& c) {
    const int top = (int)(((unsigned long long)(long long)pos * f) >> 32);   // the angle in turns, 2^-32 each, -1/2 .. 1/2
    sincospif((float)top * 4.656612873077393e-10f, &s, &c);                  // 2^-31: half turns
    s *= scale;
    c *= scale;
}

// One warp per (row, head).
template <typename Tin, typename Tout>
__global__ void __launch_bounds__(256) heads_kernel(const HeadsArgs a) {
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
    const float r = rsqrtf(ss / (float)a.D + a.eps);
    const int half = a.rot / 2;
    for (int j = lane; j < half; j += 32) {
        const int ia = a.adjacent ? 2 * j : j, ib = a.adjacent ? 2 * j + 1 : j + half;
        float sn, cs;
        turn_sincos(turn_fraction(a.inv_freq[j]), a.positions[row], a.scale, sn, cs);
        const float za = to_f32(src[ia]) * r * (t.weight ? t.weight[ia] : 1.0f), zb = to_f32(src[ib]) * r * (t.weight ? t.weight[ib] : 1.0f);
        dst[ia] = from_f32<Tout>(za * cs - zb * sn);
        dst[ib] = from_f32<Tout>(zb * cs + za * sn);
    }
    for (int i = a.rot + lane; i < a.D; i += 32) dst[i] = from_f32<Tout>(to_f32(src[i]) * r * (t.weight ? t.weight[i] : 1.0f));
}

// ---------------------------------------------------------------------------------------------------------------
// Logits.  count_v: times token v occurs among the generated tokens of the row, seen_v: in prompt or generated ones.
//   seen: l = l > 0 ? l / rep : l * rep;  l -= freq * count_v;  count_v > 0: l -= pres;  l += bias_v;  mask bit clear: l = -inf
// A CTA owns LG_CHUNK logits of a row, counts the row's tokens that fall into them in shared memory (whole numbers, so the
// order of the atomics does not matter), notes the last bias entry of each, and passes over its logits once.
// ---------------------------------------------------------------------------------------------------------------
constexpr int LG_CHUNK = 4096, LG_THREADS = 512;
constexpr uint32_t LG_PROMPT = 0x80000000u;   // seen in the prompt; the other bits count generated tokens

struct LogitsArgs {
    const float* x;
    float* y;
    long long x_ld, y_ld;
    q38b_logit_rules r;
    int n, index_offset;
};

__global__ void __launch_bounds__(LG_THREADS) logits_kernel(const LogitsArgs a) {
    __shared__ uint32_t seen[LG_CHUNK], last[LG_CHUNK];
    const int row = blockIdx.y, c0 = blockIdx.x * LG_CHUNK, n = min(LG_CHUNK, a.n - c0), first = a.index_offset + c0;
    const bool counts = a.r.history && a.r.penalties, biases = a.r.bias_ids != nullptr;
    for (int i = threadIdx.x; i < LG_CHUNK; i += LG_THREADS) {
        seen[i] = 0u;
        last[i] = 0u;
    }
    __syncthreads();
    if (counts) {
        const long long b = a.r.history_begin[row], e = a.r.history_begin[row + 1], made = b + (a.r.prompt_len ? a.r.prompt_len[row] : 0);
        for (long long i = b + threadIdx.x; i < e; i += LG_THREADS) {
            const unsigned at = (unsigned)a.r.history[i] - (unsigned)first;
            if (a.r.history[i] >= 0 && at < (unsigned)n) {
                if (i < made) atomicOr(&seen[at], LG_PROMPT);
                else atomicAdd(&seen[at], 1u);
            }
        }
    }
    long long bias0 = 0;
    if (biases) {
        bias0 = a.r.bias_begin[row];
        const long long e = a.r.bias_begin[row + 1];
        for (long long i = bias0 + threadIdx.x; i < e; i += LG_THREADS) {
            const unsigned at = (unsigned)a.r.bias_ids[i] - (unsigned)first;
            if (a.r.bias_ids[i] >= 0 && at < (unsigned)n) atomicMax(&last[at], (uint32_t)(i - bias0) + 1u);
        }
    }
    __syncthreads();
    const float rep = counts ? a.r.penalties[3 * row] : 1.0f, freq = counts ? a.r.penalties[3 * row + 1] : 0.0f, pres = counts ? a.r.penalties[3 * row + 2] : 0.0f;
    const int m = !a.r.masks ? -1 : a.r.mask_of_row ? a.r.mask_of_row[row] : row;
    const uint32_t* mask = m >= 0 ? a.r.masks + m * a.r.mask_ld : nullptr;
    for (int i = threadIdx.x; i < n; i += LG_THREADS) {
        float v = a.x[row * a.x_ld + c0 + i];
        const uint32_t s = seen[i];
        if (s) {
            v = v > 0.0f ? __fdiv_rn(v, rep) : v * rep;
            const uint32_t count = s & ~LG_PROMPT;
            if (count) v = v - freq * (float)count - pres;
        }
        if (last[i]) v += a.r.bias_values[bias0 + last[i] - 1];
        const int id = first + i;
        if (mask && !((mask[id >> 5] >> (id & 31)) & 1u)) v = __int_as_float(0xFF800000);
        a.y[row * a.y_ld + c0 + i] = v;
    }
}

bool known_kind(int kind) { return kind == Q38B_OUT_F32 || kind == Q38B_OUT_F16 || kind == Q38B_OUT_BF16; }
uintptr_t kind_size(int kind) { return kind == Q38B_OUT_F32 ? 4 : 2; }

template <typename Tin, typename Tout>
int heads_as(q38b_ctx* ctx, const HeadsArgs& a, cudaStream_t st) {
    const long long items = (long long)a.rows * (a.t[0].n_heads + a.t[1].n_heads);
    heads_kernel<Tin, Tout><<<(unsigned)((items + 7) / 8), 256, 0, st>>>(a);
    return launch_status(ctx, cudaSuccess);
}
template <typename Tin>
int heads_from(q38b_ctx* ctx, const HeadsArgs& a, int out_kind, cudaStream_t st) {
    return out_kind == Q38B_OUT_F32 ? heads_as<Tin, float>(ctx, a, st) : out_kind == Q38B_OUT_F16 ? heads_as<Tin, __half>(ctx, a, st) : heads_as<Tin, __nv_bfloat16>(ctx, a, st);
}

}  // namespace

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
        // two heads, or two rows, of one destination must not share elements
        if ((t.n_heads > 1 && t.dst_head < D) || (rows > 1 && t.dst_row < D)) return Q38B_ERR_ARG;
        if ((uintptr_t)t.src % kind_size(in_kind) || (uintptr_t)t.dst % kind_size(out_kind) || ((uintptr_t)t.weight & 3)) return Q38B_ERR_ALIGN;
        // in place only element over element
        if (t.src == t.dst && (in_kind != out_kind || t.src_head != t.dst_head || t.src_row != t.dst_row)) return Q38B_ERR_ARG;
    }
    if (((uintptr_t)positions & 3) || ((uintptr_t)inv_freq & 7)) return Q38B_ERR_ALIGN;
    a.D = D;
    a.rot = rot;
    a.adjacent = adjacent ? 1 : 0;
    a.rows = rows;
    a.eps = eps;
    a.scale = scale;
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
    if (n_rows > 1 && (x_ld < n || y_ld < n)) return Q38B_ERR_ARG;
    if (x == y && n_rows > 1 && x_ld != y_ld) return Q38B_ERR_ARG;
    if (!rules->penalties != !rules->history || !rules->history != !rules->history_begin || (rules->prompt_len && !rules->history)) return Q38B_ERR_ARG;
    if (!rules->bias_ids != !rules->bias_values || !rules->bias_ids != !rules->bias_begin) return Q38B_ERR_ARG;
    if ((rules->mask_of_row && !rules->masks) || (rules->masks && rules->mask_ld < ((long long)index_offset + n + 31) / 32)) return Q38B_ERR_ARG;
    if (((uintptr_t)x | (uintptr_t)y | (uintptr_t)rules->penalties | (uintptr_t)rules->history | (uintptr_t)rules->prompt_len | (uintptr_t)rules->bias_ids |
         (uintptr_t)rules->bias_values | (uintptr_t)rules->masks | (uintptr_t)rules->mask_of_row) & 3)
        return Q38B_ERR_ALIGN;
    if (((uintptr_t)rules->history_begin | (uintptr_t)rules->bias_begin) & 7) return Q38B_ERR_ALIGN;
    LogitsArgs a;
    a.x = x;
    a.y = y;
    a.x_ld = x_ld;
    a.y_ld = y_ld;
    a.r = *rules;
    a.n = n;
    a.index_offset = index_offset;
    DeviceGuard on(ctx);
    logits_kernel<<<dim3((unsigned)((n + LG_CHUNK - 1) / LG_CHUNK), (unsigned)n_rows), LG_THREADS, 0, (cudaStream_t)stream>>>(a);
    return launch_status(ctx, cudaSuccess);
}

}  // extern "C"

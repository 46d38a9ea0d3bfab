// q38b_attention.cu -- attention of a chunk of new tokens over a paged cache.
//
//   out[i][h] = sum_j softmax_j(scale q[i][h] . k[j][h / G]) v[j][h / G],  j <= length - new + i
//
// One pass over the keys with the running maximum m and sum l of a softmax: a new maximum scales what was summed before by exp(m_old - m_new).
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstring>

#include "q38b_cache.cuh"
#include "q38b_internal.h"
#include "q38b_pipe.cuh"
#include "q38b_types.cuh"

using namespace q38b;

namespace {

struct AttnArgs {
    Batch batch;
    const void *q, *k, *v;
    void* out;
    float* lse;
    long long q_row, q_head, out_row, out_head, k_page, k_slot, k_head, v_page, v_slot, v_head;
    int q_kind, out_kind, n_heads, n_kv, group, D;
    float scale;
};

__device__ __forceinline__ float load_kind(const void* p, int kind, long long at) {
    return kind == Q38B_OUT_F32 ? ((const float*)p)[at] : kind == Q38B_OUT_F16 ? __half2float(((const __half*)p)[at]) : __bfloat162float(((const __nv_bfloat16*)p)[at]);
}
__device__ __forceinline__ void store_kind(void* p, int kind, long long at, float v) {
    if (kind == Q38B_OUT_F32) ((float*)p)[at] = v;
    else if (kind == Q38B_OUT_F16) ((__half*)p)[at] = __float2half_rn(v);
    else ((__nv_bfloat16*)p)[at] = __float2bfloat16_rn(v);
}

// A block: 64 (token, head) pairs of one key head of one sequence, 32 keys at a time through shared memory; four threads a pair.
constexpr int SR = 64, SK = 32;
template <typename C>
__global__ void __launch_bounds__(256) attention_simple_kernel(const AttnArgs a) {
    extern __shared__ float sm[];
    const int W = a.D + 1;
    float *qs = sm, *ks = qs + SR * W, *vs = ks + SK * W, *ps = vs + SK * W;
    const int s = (int)blockIdx.z, kvh = (int)blockIdx.y;
    const int first = a.batch.first(s), n_new = max(a.batch.first(s + 1) - first, 0);
    const int r0 = (int)blockIdx.x * SR, n_rows = n_new * a.group;
    if (r0 >= n_rows) return;
    const int len = a.batch.length(s), r = threadIdx.x / 4, c = threadIdx.x % 4;
    const int mine = r0 + r, tok = mine / a.group, head = kvh * a.group + mine % a.group;
    const int seen = mine < n_rows ? max(0, len - n_new + tok + 1) : 0;
    const int last = min(r0 + SR, n_rows) - 1, most = max(0, len - n_new + last / a.group + 1);
    for (int i = threadIdx.x; i < SR * a.D; i += 256) {
        const int rr = r0 + i / a.D, e = i % a.D;
        float x = 0.0f;
        if (rr < n_rows) x = load_kind(a.q, a.q_kind, (first + rr / a.group) * a.q_row + (kvh * a.group + rr % a.group) * a.q_head + e);
        qs[i / a.D * W + e] = to_f32(from_f32<C>(x));
    }
    float m = -INFINITY, l = 0.0f, acc[64] = {};
    for (int j0 = 0; j0 < most; j0 += SK) {
        __syncthreads();
        for (int i = threadIdx.x; i < SK * a.D; i += 256) {
            const int j = j0 + i / a.D, e = i % a.D, page = j < most ? a.batch.page(s, j) : a.batch.n_pages;
            const long long slot = j & ((1 << a.batch.page_shift) - 1);
            const bool there = page < a.batch.n_pages;
            ks[i / a.D * W + e] = there ? to_f32(((const C*)a.k)[page * a.k_page + slot * a.k_slot + kvh * a.k_head + e]) : 0.0f;
            vs[i / a.D * W + e] = there ? to_f32(((const C*)a.v)[page * a.v_page + slot * a.v_slot + kvh * a.v_head + e]) : 0.0f;
        }
        __syncthreads();
        float p[SK / 4], top = m;
        for (int n = 0; n < SK / 4; n++) {
            const int j = c * (SK / 4) + n;
            float dot = 0.0f;
            for (int e = 0; e < a.D; e++) dot = fmaf(qs[r * W + e], ks[j * W + e], dot);
            p[n] = j0 + j < seen ? dot * a.scale : -INFINITY;
            top = fmaxf(top, p[n]);
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float at = top == -INFINITY ? 0.0f : top, by = __expf(m - at);
        float sum = 0.0f;
        for (int n = 0; n < SK / 4; n++) {
            p[n] = __expf(p[n] - at);
            sum += p[n];
            ps[r * SK + c * (SK / 4) + n] = p[n];
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        l = l * by + sum;
        m = top;
        __syncwarp();
        for (int n = 0; n < 64; n++) {
            const int e = c + 4 * n;
            if (e >= a.D) break;
            float x = acc[n] * by;
            for (int j = 0; j < SK; j++)
                if (j0 + j < seen) x = fmaf(ps[r * SK + j], vs[j * W + e], x);
            acc[n] = x;
        }
    }
    if (mine >= n_rows) return;
    const float inv = seen > 0 ? 1.0f / l : 0.0f;
    for (int n = 0; n < 64; n++)
        if (c + 4 * n < a.D) store_kind(a.out, a.out_kind, (first + tok) * a.out_row + head * a.out_head + c + 4 * n, seen > 0 ? acc[n] * inv : 0.0f);
    if (a.lse && c == 0) a.lse[(long long)(first + tok) * a.n_heads + head] = seen > 0 ? m + logf(l) : -INFINITY;
}

template <typename C>
int attention_as(q38b_ctx* ctx, const AttnArgs& a, int rows, cudaStream_t st) {
    auto kern = attention_simple_kernel<C>;
    const int smem = ((SR + 2 * SK) * (a.D + 1) + SR * SK) * 4;
    const int rc = q38b_ensure_kernel_smem(ctx, (const void*)kern, ctx->smem_optin, false);
    if (rc != Q38B_OK) return rc;
    kern<<<dim3((unsigned)(((long long)rows * a.group + SR - 1) / SR), (unsigned)a.n_kv, (unsigned)a.batch.n_seqs), 256, smem, st>>>(a);
    return launch_status(ctx, cudaSuccess);
}

bool known_kind(int kind) { return kind == Q38B_OUT_F32 || kind == Q38B_OUT_F16 || kind == Q38B_OUT_BF16; }
int kind_size(int kind) { return kind == Q38B_OUT_F32 ? 4 : 2; }

}  // namespace

extern "C" {

size_t q38b_attention_work_bytes(const q38b_ctx* ctx, int n_heads, int n_kv_heads, int D, int rows) { return 16; }

int q38b_attention(q38b_ctx* ctx, const q38b_paged_kv* c, const void* q, int q_kind, long long q_row, long long q_head, int n_heads, float scale, void* out,
                   int out_kind, long long out_row, long long out_head, float* lse, int rows, void* work, size_t work_bytes, void* stream) {
    if (!ctx || !q || !out || !work || rows < 1 || !known_kind(q_kind) || !known_kind(out_kind) || !(scale > 0.0f) || !std::isfinite(scale)) return Q38B_ERR_ARG;
    int rc = paged_kv_check(c);
    if (rc != Q38B_OK) return rc;
    if (n_heads < 1 || n_heads % c->n_heads || q_row < 0 || q_head < 0 || out_row < 0 || out_head < 0) return Q38B_ERR_ARG;
    if ((n_heads > 1 && out_head < c->D) || (rows > 1 && out_row < c->D)) return Q38B_ERR_ARG;
    if (q_kind != Q38B_OUT_F32 && q_kind != c->kind) return Q38B_ERR_UNSUPPORTED;
    if ((uintptr_t)q % kind_size(q_kind) || (uintptr_t)out % kind_size(out_kind) || ((uintptr_t)lse & 3) || ((uintptr_t)work & 15)) return Q38B_ERR_ALIGN;
    if (work_bytes < q38b_attention_work_bytes(ctx, n_heads, c->n_heads, c->D, rows)) return Q38B_ERR_NOMEM;
    DeviceGuard on(ctx);
    const AttnArgs a = {batch_of(c, rows), q, c->k, c->v, out, lse, q_row, q_head, out_row, out_head, c->k_page, c->k_slot, c->k_head, c->v_page, c->v_slot, c->v_head,
                        q_kind, out_kind, n_heads, c->n_heads, n_heads / c->n_heads, c->D, scale};
    return c->kind == Q38B_OUT_F16 ? attention_as<__half>(ctx, a, rows, (cudaStream_t)stream) : attention_as<__nv_bfloat16>(ctx, a, rows, (cudaStream_t)stream);
}

}  // extern "C"

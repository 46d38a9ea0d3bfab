// q38b_cache.cu -- new keys and values into the pages of a cache.
//
//   cache[page of token j][j mod page size][head] = row, j = length - new + i for the i-th of a sequence's `new` rows
//
// Bound by memory: each row is read once and written once.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "q38b_cache.cuh"
#include "q38b_internal.h"
#include "q38b_pipe.cuh"
#include "q38b_types.cuh"

using namespace q38b;

namespace {

struct AppendArgs {
    Batch batch;
    const void* src[2];
    long long src_row[2], src_head[2];
    void* dst[2];
    long long dst_page[2], dst_slot[2], dst_head[2];
    int n_heads, D;
};

// A warp moves one row of keys or of values, eight elements (16 bytes of the cache) a lane at a time.  The row's elements are asked for before its
// place is known, which takes three loads one behind the other (first rows, length, page).
template <typename T, typename C, bool VEC>
__global__ void __launch_bounds__(256) cache_append_kernel(const AppendArgs a) {
    constexpr int AHEAD = 4;
    const int lane = threadIdx.x & 31, what = (int)blockIdx.y;
    const int row = (int)(blockIdx.x * 8 + (threadIdx.x >> 5));
    if (row >= a.batch.rows) return;
    const int per_head = a.D / 8, units = a.n_heads * per_head;
    const T* src = (const T*)a.src[what] + row * a.src_row[what];
    struct alignas(16) Eight { T e[8]; };
    Eight v[AHEAD];
    const auto load = [&](int u, Eight& to) {
        const T* p = src + u / per_head * a.src_head[what] + u % per_head * 8;
        if constexpr (VEC) {
            to = *(const Eight*)p;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) to.e[i] = p[i];
        }
    };
#pragma unroll
    for (int n = 0; n < AHEAD; n++)
        if (lane + 32 * n < units) load(lane + 32 * n, v[n]);
    const int s = sequence_of_row(a.batch, row), first = a.batch.first(s), next = a.batch.first(s + 1);
    if (row < first || row >= next) return;   // (nobody's row)
    // (of the length as it is: with one past the table, counted as the table's, the chunk would go over tokens that are there)
    const long long j = (long long)max(a.batch.lengths[s], 0) - (next - first) + (row - first);
    if (j < 0 || j >= (long long)a.batch.table_n << a.batch.page_shift) return;
    const int page = a.batch.page(s, (int)j);
    if (page >= a.batch.n_pages) return;
    C* dst = (C*)a.dst[what] + page * a.dst_page[what] + (j & ((1 << a.batch.page_shift) - 1)) * a.dst_slot[what];
    for (int u0 = lane; u0 < units; u0 += 32 * AHEAD) {
#pragma unroll
        for (int n = 0; n < AHEAD; n++) {
            const int u = u0 + 32 * n;
            if (u >= units) break;
            struct alignas(16) Out { C e[8]; } o;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if constexpr (sizeof(T) == sizeof(C)) memcpy(&o.e[i], &v[n].e[i], 2);   // (the same type: infinities, NaN and all as they are)
                else o.e[i] = from_f32<C>(to_f32(v[n].e[i]));
            }
            *(Out*)(dst + u / per_head * a.dst_head[what] + u % per_head * 8) = o;
        }
#pragma unroll
        for (int n = 0; n < AHEAD; n++)
            if (u0 + 32 * (AHEAD + n) < units) load(u0 + 32 * (AHEAD + n), v[n]);
    }
}

template <typename T, typename C>
int append_as(q38b_ctx* ctx, const AppendArgs& a, bool vec, cudaStream_t st) {
    const dim3 grid((unsigned)((a.batch.rows + 7) / 8), 2);
    if (vec) cache_append_kernel<T, C, true><<<grid, 256, 0, st>>>(a);
    else cache_append_kernel<T, C, false><<<grid, 256, 0, st>>>(a);
    return launch_status(ctx, cudaSuccess);
}

}  // namespace

extern "C" int q38b_cache_append(q38b_ctx* ctx, const q38b_paged_kv* c, const void* k, const void* v, int in_kind, long long k_row, long long k_head,
                                 long long v_row, long long v_head, int rows, void* stream) {
    if (!ctx || !k || !v || rows < 1 || k_row < 0 || k_head < 0 || v_row < 0 || v_head < 0) return Q38B_ERR_ARG;
    const int rc = paged_kv_check(c);
    if (rc != Q38B_OK) return rc;
    if (in_kind != Q38B_OUT_F32 && in_kind != c->kind) return in_kind == Q38B_OUT_F16 || in_kind == Q38B_OUT_BF16 ? Q38B_ERR_UNSUPPORTED : Q38B_ERR_ARG;
    const int size = in_kind == Q38B_OUT_F32 ? 4 : 2;
    if (((uintptr_t)k | (uintptr_t)v) % size) return Q38B_ERR_ALIGN;
    DeviceGuard on(ctx);
    cudaStream_t st = (cudaStream_t)stream;
    AppendArgs a = {batch_of(c, rows), {k, v}, {k_row, v_row}, {k_head, v_head}, {c->k, c->v}, {c->k_page, c->v_page}, {c->k_slot, c->v_slot}, {c->k_head, c->v_head}, c->n_heads, c->D};
    const bool vec = (((uintptr_t)k | (uintptr_t)v | (uintptr_t)((k_row | k_head | v_row | v_head) * size)) & 15) == 0;
    if (in_kind == Q38B_OUT_F32) return c->kind == Q38B_OUT_F16 ? append_as<float, __half>(ctx, a, vec, st) : append_as<float, __nv_bfloat16>(ctx, a, vec, st);
    return append_as<__half, __half>(ctx, a, vec, st);   // (16 bits to the same 16 bits)
}

// q38b_cache.cuh -- the paged cache of keys and values as its kernels see it: which sequence a row belongs to, where a token lies.
#pragma once
#include <cuda_runtime.h>

#include "../../include/q38b200.h"
#include "q38b_host.h"

namespace q38b {

// The batch of a q38b_paged_kv; lengths and pages are clamped to what there is, and whoever goes through a sequence's rows to the rows there are.
struct Batch {
    const int *table, *lengths, *begin;
    long long table_ld;
    int table_n, n_seqs, n_pages, page_shift, rows;

    // first of sequence s's rows (s <= n_seqs), which may lie behind the rows there are: a call for fewer rows than the lists say takes the first of them, and each has the token
    // that it would have with all
    __device__ __forceinline__ int first(int s) const { return max(begin[s], 0); }
    __device__ __forceinline__ int length(int s) const {   // (whole pages of at most 2^31 - 1 slots)
        return (int)min((long long)max(lengths[s], 0), (long long)table_n << page_shift);
    }
    // page of token j of sequence s; a number that is no page's: n_pages
    __device__ __forceinline__ int page(int s, int j) const {
        const int p = table[(long long)s * table_ld + (j >> page_shift)];
        return (unsigned)p < (unsigned)n_pages ? p : n_pages;
    }
};

// The last sequence whose first row is at or before `row`, found by a whole warp, 32 candidates at a time (one look for 32 sequences, two for 1024).
__device__ __forceinline__ int sequence_of_row(const Batch& b, int row) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = b.n_seqs;   // the answer lies in [lo, lo + n)
    while (n > 1) {
        const int step = (n + 31) / 32, at = lo + lane * step;
        const bool here = lane * step < n && (at == 0 || b.first(at) <= row);
        const int last = 31 - __clz(__ballot_sync(0xffffffffu, here) | 1u);
        n = min(step, lo + n - (lo + last * step));
        lo += last * step;
    }
    return lo;
}

}  // namespace q38b

// whether a q38b_paged_kv is whole and aligned: a q38b_status
inline int paged_kv_check(const q38b_paged_kv* c) {
    if (!c || !c->k || !c->v || !c->table || !c->lengths || !c->begin) return Q38B_ERR_ARG;
    if (c->kind != Q38B_OUT_F16 && c->kind != Q38B_OUT_BF16) return Q38B_ERR_ARG;
    if (c->n_pages < 1 || c->page_size < 8 || (c->page_size & (c->page_size - 1)) || (long long)c->n_pages * c->page_size > 0x7FFFFFFF) return Q38B_ERR_ARG;
    if (c->n_heads < 1 || c->n_heads > 65535 || c->D < 8 || c->D > 256 || c->D % 8 || c->n_seqs < 1 || c->n_seqs > 65535) return Q38B_ERR_ARG;
    if (c->table_n < 1 || c->table_ld < c->table_n || (long long)c->table_n * c->page_size > 0x7FFFFFFF) return Q38B_ERR_ARG;
    const long long strides[6] = {c->k_page, c->k_slot, c->k_head, c->v_page, c->v_slot, c->v_head};
    for (int i = 0; i < 6; i++) {
        const bool used = i % 3 == 0 ? c->n_pages > 1 : i % 3 == 1 || c->n_heads > 1;
        if (!used) continue;
        if (strides[i] < c->D || strides[i] >= 1LL << 38) return Q38B_ERR_ARG;
        if (strides[i] % 8) return Q38B_ERR_ALIGN;
    }
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return Q38B_ERR_ALIGN;
    if (((uintptr_t)c->table | (uintptr_t)c->lengths | (uintptr_t)c->begin) & 3) return Q38B_ERR_ALIGN;
    return Q38B_OK;
}

// whether the attention counts such a batch's work in 32 bits: the end of the last tile of 128 keys, (row, head) pairs, and tiles of 128 of them times tiles of keys (and three
// more for a start)
inline bool attention_fits(const q38b_paged_kv* c, int n_heads, int rows) {
    return (long long)c->table_n * c->page_size <= 0x7FFFFFFF - 127 && (long long)rows * n_heads <= 0x3FFFFFFF &&
           ((long long)rows * n_heads / 128 + (long long)c->n_seqs * c->n_heads) * ((long long)c->table_n * c->page_size / 128 + 4) <= 0x7FFFFFFF;
}

inline q38b::Batch batch_of(const q38b_paged_kv* c, int rows) {
    int shift = 0;
    while (1 << shift < c->page_size) shift++;
    return {c->table, c->lengths, c->begin, c->table_ld, c->table_n, c->n_seqs, c->n_pages, shift, rows};
}

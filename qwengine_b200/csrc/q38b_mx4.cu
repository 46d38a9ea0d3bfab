// q38b_mx4.cu -- microscaled 4-bit floating point (OCP MX: E2M1 elements, one E8M0 scale per 32): quantizer, dequantizer
// and the product of two such matrices on the block-scaled tensor-core instructions.
//
//   e = clamp(floor(log2 amax) - 2, -127, 127) over 32 values; code = x / 2^e rounded half to even to {0 .5 1 1.5 2 3 4 6}
//   Y[t][r] (+)= sum_k X[t][k] W[r][k] over the values the codes and scales stand for
//
// A matrix is held as the tensor core reads it: codes [rows][K/2], two per byte (even element low), rows `ld` bytes apart;
// scale bytes in tiles of 128 rows x 4 blocks (512 bytes: byte 16 (r % 32) + 4 (r / 32) + b), tile (i, j) at (i ceil(K/128) + j) 512,
// which is what one copy into tensor memory takes; bytes behind the last row and block are zero.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
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

constexpr int MX_TILE = 512;   // scale bytes of 128 rows x 4 blocks

__host__ __device__ inline long long mx_tiles_k(int K) { return (K + 127) / 128; }

// Eight values to E2M1 codes in a word, the first in its low four bits: half to even, saturated at 6 (one block: the conversions then merge their bytes themselves)
__device__ __forceinline__ uint32_t e2m1_eight(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\tcvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\tmov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// The scale byte of a block whose largest magnitude has the bit pattern `top`, and the power of two its values are multiplied
// with.  The byte is the exponent field less two (the exponent of 4, the largest power of two an element holds), never below 0;
// a block that holds a NaN or an infinity gets 255, the scale that is NaN, and codes of its own zeros (0 times anything but NaN).
__device__ __forceinline__ uint32_t mx_scale(uint32_t top, float& inv) {
    const uint32_t field = top >> 23;
    if (field == 255u) { inv = 0.0f; return 255u; }
    const uint32_t byte = field > 2u ? field - 2u : 0u;
    inv = __uint_as_float((254u - byte) << 23);
    return byte;
}

// Quantizer and dequantizer walk a matrix alike: a warp owns 256 values (two K tiles) of the four rows r, r + 32, r + 64, r + 96 whose
// scales lie together in a tile, 16 bytes for each K tile, so that scales move in whole pieces; a lane has eight neighbours of each row
// (four lanes are a block) and all four rows' loads in flight.  Bound by memory: what is read and written once.  17408 x 5120 bf16 122 ->
// 40 us (5.7 TB/s; fp32 58 us, 7.0 TB/s), back to bf16 179 -> 37 us (6.1 TB/s), against one row and four values a lane with a byte store per block.
struct MxWalk {
    long long row;   // the first of the four rows
    int k;           // this lane's first value
    long long tile;  // the scales' first K tile of the warp, in tiles
};
__host__ __device__ inline long long mx_walk_warps(int K, int rows) { return (long long)(rows + 127) / 128 * 32 * ((K + 255) / 256); }
__device__ __forceinline__ bool mx_walk(int K, int rows, MxWalk& w) {
    const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), kc = (K + 255) / 256;
    if (item >= mx_walk_warps(K, rows)) return false;
    // the eight warps of a block: neighbouring rows, so that their scales are one piece of 128 bytes
    const long long group = item / 8, at = group / kc, c = group % kc;
    w.row = at / 4 * 128 + at % 4 * 8 + (item & 7);
    w.k = (int)c * 256 + 8 * (int)(threadIdx.x & 31);
    w.tile = at / 4 * mx_tiles_k(K) + 2 * c;
    return true;
}

// Eight values as they lie in memory (16-bit types keep all four rows in half the registers until they are needed) and as floats
template <typename T> struct Raw8 { uint4 q[sizeof(T) / 2]; };
template <typename T> __device__ __forceinline__ void raw8_values(const Raw8<T>& r, float (&v)[8]) {
    const T* e = (const T*)r.q;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = to_f32(e[i]);
}
// 16-bit types: the largest magnitudes of the even and of the odd four (magnitudes compare like their bits, a NaN's exceeds them all)
template <typename T> __device__ __forceinline__ uint32_t raw8_top16(const Raw8<T>& r) {
    return __vmaxu2(__vmaxu2(r.q[0].x & 0x7FFF7FFFu, r.q[0].y & 0x7FFF7FFFu), __vmaxu2(r.q[0].z & 0x7FFF7FFFu, r.q[0].w & 0x7FFF7FFFu));
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) mx4_quantize_kernel(const T* x, long long x_ld, int K, int rows, uint8_t* codes, long long codes_ld, uint8_t* scales) {
    pdl_launch_dependents();   // (a product behind it brings its first weights meanwhile)
    MxWalk w;
    if (!mx_walk(K, rows, w)) return;
    const int lane = threadIdx.x & 31, here = w.k < K ? (int)min(4LL, (rows - w.row + 31) / 32) : 0;   // of the four rows, those that are there
    const T* p = x + w.row * x_ld + w.k;
    uint8_t* to = codes + w.row * codes_ld + w.k / 2;
    Raw8<T> raw[4] = {};
#pragma unroll
    for (int j = 0; j < 4; j++, p += 32 * x_ld)
        if (j < here) {
            if constexpr (VEC) {
                raw[j] = *(const Raw8<T>*)p;
            } else {
                T e[8];
#pragma unroll
                for (int i = 0; i < 8; i++) e[i] = p[i];
                memcpy(&raw[j], e, sizeof(e));
            }
        }
    // the largest magnitudes of the four rows' blocks (16-bit types: two rows a word, which compare and travel together)
    uint32_t top[4];
    if constexpr (sizeof(T) == 2) {
        uint32_t pair[2];
#pragma unroll
        for (int p = 0; p < 2; p++) {
            const uint32_t a = raw8_top16<T>(raw[2 * p]), b = raw8_top16<T>(raw[2 * p + 1]);
            pair[p] = __vmaxu2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
            pair[p] = __vmaxu2(pair[p], __shfl_xor_sync(0xffffffffu, pair[p], 1));
            pair[p] = __vmaxu2(pair[p], __shfl_xor_sync(0xffffffffu, pair[p], 2));
            const unsigned short lo = (unsigned short)(pair[p] & 0xFFFFu), hi = (unsigned short)(pair[p] >> 16);
            top[2 * p] = __float_as_uint(to_f32(*(const T*)&lo));
            top[2 * p + 1] = __float_as_uint(to_f32(*(const T*)&hi));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float* v = (const float*)raw[j].q;
            top[j] = 0u;
#pragma unroll
            for (int i = 0; i < 8; i++) top[j] = max(top[j], __float_as_uint(v[i]) & 0x7FFFFFFFu);
            top[j] = max(top[j], __shfl_xor_sync(0xffffffffu, top[j], 1));
            top[j] = max(top[j], __shfl_xor_sync(0xffffffffu, top[j], 2));
        }
    }
    uint32_t bytes = 0u;   // of the four rows' blocks here
#pragma unroll
    for (int j = 0; j < 4; j++, to += 32 * codes_ld) {
        float v[8], inv;
        raw8_values<T>(raw[j], v);
        bytes |= mx_scale(top[j], inv) << (8 * j);   // (zeros behind the last row and block: byte 0)
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= inv;
        if (j < here) *(uint32_t*)to = e2m1_eight(v);
    }
    // four rows of this block to four blocks of a row: a transposition of 4 x 4 bytes between the K tile's four blocks
    const int q = lane / 4 % 4;
    uint32_t other = __shfl_xor_sync(0xffffffffu, bytes, 4);
    bytes = __byte_perm(bytes, other, q & 1 ? 0x3715 : 0x6240);
    other = __shfl_xor_sync(0xffffffffu, bytes, 8);
    bytes = __byte_perm(bytes, other, q & 2 ? 0x3276 : 0x5410);
    if (lane % 4 == 0 && w.k - 8 * (lane % 16) < K)   // (the K tile is there)
        *(uint32_t*)(scales + (w.tile + lane / 16) * MX_TILE + 16 * (w.row % 32) + 4 * q) = bytes;
}

// Scale bytes of another producer, row by row, into the tiles.
__global__ void __launch_bounds__(256) mx4_tile_kernel(const uint8_t* src, long long src_ld, int K, int rows, uint8_t* scales) {
    const long long kt = mx_tiles_k(K), n = (long long)(rows + 127) / 128 * kt * MX_TILE;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int in = (int)(i % MX_TILE);
    const long long row = i / MX_TILE / kt * 128 + in / 16 + 32 * (in % 16 / 4), block = i / MX_TILE % kt * 4 + in % 4;
    scales[i] = row < rows && block < K / 32 ? src[row * src_ld + block] : (uint8_t)0;
}

__device__ __forceinline__ float mx_scale_value(uint32_t byte) {   // 2^(byte - 127); 255: NaN
    return byte == 255u ? __uint_as_float(0x7FC00000u) : byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}
// the two values of a byte, which halves hold exactly
__device__ __forceinline__ float2 e2m1_values(uint32_t byte) {
    uint32_t h;
    asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "r"(byte));
    return __half22float2(*(const __half2*)&h);
}

// A lane writes 16 bytes at a time: eight values of 16 bits, or four of 32 bits in each of the warp's two K tiles (eight neighbours in two
// stores of 16 bytes, 32 apart, left half-written sectors: 17408 x 5120 to fp32 92 us, 64 so).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) mx4_dequant_kernel(const uint8_t* codes, long long codes_ld, const uint8_t* scales, int K, int rows, T* out, long long out_ld) {
    constexpr int E = 16 / (int)sizeof(T), PARTS = 256 / (32 * E);
    using Code = typename std::conditional<E == 8, uint32_t, uint16_t>::type;
    MxWalk w;
    if (!mx_walk(K, rows, w)) return;
    const int lane = threadIdx.x & 31;
    w.k = w.k - 8 * lane + E * lane;
    uint32_t code[PARTS][4], word[PARTS][4];
#pragma unroll
    for (int p = 0; p < PARTS; p++) {
        const int in = 32 * E * p + E * lane;   // of the warp's 256
        const bool any = w.k + 32 * E * p < K;
        const uint4 q = any ? *(const uint4*)(scales + (w.tile + in / 128) * MX_TILE + 16 * (w.row % 32)) : make_uint4(0, 0, 0, 0);
        word[p][0] = q.x; word[p][1] = q.y; word[p][2] = q.z; word[p][3] = q.w;
#pragma unroll
        for (int j = 0; j < 4; j++) code[p][j] = any && w.row + 32 * j < rows ? *(const Code*)(codes + (w.row + 32 * j) * codes_ld + (w.k + 32 * E * p) / 2) : (Code)0;
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
        for (int p = 0; p < PARTS; p++) {
            if (w.row + 32 * j >= rows || w.k + 32 * E * p >= K) continue;
            const float s = mx_scale_value(word[p][j] >> (8 * ((32 * E * p + E * lane) % 128 / 32)) & 255u);
            T r[E];
#pragma unroll
            for (int i = 0; i < E / 2; i++) {
                const float2 v = e2m1_values(code[p][j] >> (8 * i) & 255u);
                r[2 * i] = from_f32<T>(v.x * s);
                r[2 * i + 1] = from_f32<T>(v.y * s);
            }
            T* to = out + (w.row + 32 * j) * out_ld + w.k + 32 * E * p;
            if constexpr (VEC) {
                uint4 q;
                memcpy(&q, r, 16);
                *(uint4*)to = q;
            } else {
#pragma unroll
                for (int i = 0; i < E; i++) to[i] = r[i];
            }
        }
}

// ---------------------------------------------------------------------------------------------------------------
// The product.  A CTA owns 128 weight rows (MMA M) and up to 256 tokens (MMA N).  One thread keeps a ring of stages of 256 K filled
// (codes by tiled TMA with the 128-byte swizzle, scale tiles by bulk copies), one issues per stage the copies of the scale tiles into
// tensor memory and the MMA (kind::mxf4, K = 64, one scale per 32), four warps store the accumulator.  Nothing is expanded: the
// tensor core multiplies the codes and applies the scales.  Products of two elements are multiples of 1/4 up to 36 and the scales
// are powers of two, so only the 32-bit sum rounds.
// ---------------------------------------------------------------------------------------------------------------
constexpr int MX_ROWS = 128, MX_MAX_N = 256, MX_K = 256;
constexpr int MX_THREADS = 320, MX_MAX_STAGES = 12, MX_MAX_SPLITS = 8;
constexpr int MX_FUSE_MAX_K = 8192;   // one token: every CTA quantizes its part of the activations itself, of at most so many K
constexpr int MX_A_BYTES = MX_ROWS * MX_K / 2, MX_SFA_BYTES = 2 * MX_TILE;

struct MxArgs {
    const uint8_t *w_scales, *x_scales;
    void* Y;
    long long ldy;
    int* status;
    int K, M, B, accumulate;
    int n_tile, stages, splits, pdl;
    const void* x;          // FUSED: the token's activations as they are
    int x_kind, x_steps;    // x_steps: stages of K a CTA holds, at most
    int box_at;             // splits: where the others' sums come in shared memory; 0: over the ring
};
__host__ __device__ constexpr int mx_groups(int n_tile) { return (n_tile + 127) / 128; }
__host__ __device__ constexpr int mx_stage_bytes(int n_tile) { return MX_A_BYTES + n_tile * (MX_K / 2) + MX_SFA_BYTES * (1 + mx_groups(n_tile)); }
// FUSED: a stage is weights only; the activations' codes (16 rows) and scales of every stage lie in front of the ring
constexpr int MX_FUSED_STAGE = MX_A_BYTES + MX_SFA_BYTES, MX_FUSED_X = 16 * (MX_K / 2);
__host__ __device__ constexpr int mx_fused_x_bytes(int steps) { return steps * (MX_FUSED_X + MX_SFA_BYTES); }
// accumulator, then the scales of each stage (a stage's columns are free when its shared memory is): 4 columns per tile of 128 rows x 128 K
__host__ __device__ constexpr int mx_acc_cols(int n_tile) { return (n_tile + 31) / 32 * 32; }
__host__ __device__ constexpr int mx_scale_cols(int n_tile) { return 8 * (1 + mx_groups(n_tile)); }
__host__ __device__ constexpr uint32_t mx_tmem_cols(int n_tile, int stages) {
    const int n = mx_acc_cols(n_tile) + stages * mx_scale_cols(n_tile);
    return n <= 64 ? 64u : n <= 128 ? 128u : n <= 256 ? 256u : 512u;
}

__device__ __forceinline__ uint64_t umma_desc_flat(uint32_t smem_addr) {   // no swizzle, groups of eight 16-byte rows 128 bytes apart
    return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}
// one scale tile (32 x 16 bytes) to four columns of tensor memory, repeated for the four quarters of the lanes
// (of a pair: in each CTA from its own shared memory)
template <bool PAIR>
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint32_t smem_addr) {
    if constexpr (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(umma_desc_flat(smem_addr)) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(umma_desc_flat(smem_addr)) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t add) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
            "r"(sfa), "r"(sfb), "r"(add)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
            "r"(sfa), "r"(sfb), "r"(add)
            : "memory");
}
// E2M1 times E2M1, E8M0 scales, K-major; the first two of a column's four scales (K 0..63 of a tile; 2 in both scale fields: K 64..127)
__device__ __forceinline__ uint32_t mx_idesc(int m, int n) { return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24); }

// What the tensor core does with a stage that is there: NK steps of 64 K (four but for the last stage).  The counts are constants and the
// addresses come from outside the elected branch, the same in every lane: in uniform registers a step issues in tens of clocks, out of
// vector registers in a hundred and more (with loops over run-time counts a stage took some 1200 clocks whatever its tokens: 2048 x
// 17408 x 5120 110 us).
template <bool PAIR, int GROUPS, int NK>
__device__ __forceinline__ void mx_issue(uint32_t d, uint64_t ad, uint64_t bd, uint32_t sfa, uint32_t sfb, uint32_t cols, uint32_t first_col, uint32_t idesc, uint32_t add) {
#pragma unroll
    for (int c = 0; 2 * c < NK; c++) {
        tmem_copy_scales<PAIR>(cols + (uint32_t)(4 * c), sfa + (uint32_t)(c * MX_TILE));
#pragma unroll
        for (int g = 0; g < GROUPS; g++)
            tmem_copy_scales<PAIR>(cols + (uint32_t)(8 + 4 * (c * GROUPS + g)), sfb + (uint32_t)(g * MX_SFA_BYTES + c * MX_TILE));
    }
#pragma unroll
    for (int k = 0; k < NK; k++)
        mma_mxf4<PAIR>(d, ad + (uint64_t)(2 * k), bd + (uint64_t)(2 * k), idesc + (k & 1 ? (2u << 4) | (2u << 29) : 0u), cols + (uint32_t)(4 * (k >> 1)),
                       cols + first_col + (uint32_t)(4 * (k >> 1) * GROUPS), k > 0 ? 1u : add);
}
template <bool PAIR, int GROUPS>
__device__ __forceinline__ void mx_issue_stage(int n_k, uint32_t d, uint64_t ad, uint64_t bd, uint32_t sfa, uint32_t sfb, uint32_t cols, uint32_t first_col, uint32_t idesc, uint32_t add) {
    if (n_k >= 4) mx_issue<PAIR, GROUPS, 4>(d, ad, bd, sfa, sfb, cols, first_col, idesc, add);
    else if (n_k == 3) mx_issue<PAIR, GROUPS, 3>(d, ad, bd, sfa, sfb, cols, first_col, idesc, add);
    else if (n_k == 2) mx_issue<PAIR, GROUPS, 2>(d, ad, bd, sfa, sfb, cols, first_col, idesc, add);
    else mx_issue<PAIR, GROUPS, 1>(d, ad, bd, sfa, sfb, cols, first_col, idesc, add);
}

// Eight neighbours of a row of activations, of whatever kind and alignment
__device__ __forceinline__ void load_x8(const void* x, int kind, long long at, bool vec, float (&v)[8]) {
    if (kind == Q38B_OUT_F32) {
        const float* p = (const float*)x + at;
        if (vec) {
            const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = p[i];
        }
        return;
    }
    const uint16_t* p = (const uint16_t*)x + at;
    alignas(16) uint16_t h[8];
    if (vec) {
        *(uint4*)h = *(const uint4*)p;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = kind == Q38B_OUT_F16 ? __half2float(__ushort_as_half(h[i])) : __uint_as_float((uint32_t)h[i] << 16);
}

// FUSED (one token): warps 2..9 quantize the activations of this CTA's K into operand B and its scales while the first weights are on
// their way; one launch instead of two: 17408 x 5120 12.2 us against 13.4, 5120 x 17408 14.6 against 15.2, both a CTA to an SM.  (With two tokens 13.6 and 13.4,
// with eight 18.5 and 13.5: every CTA quantizes what one kernel does once, and the weights' ring stands full meanwhile.)
// The weights of the first stages are asked for before anything else, also before the quantizer's kernel in front has ended.
template <typename T, int GROUPS, bool FUSED>
__global__ void __launch_bounds__(MX_THREADS, GROUPS == 1 ? 2 : 1) mx4_gemm_kernel(const MxArgs a, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap) {
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* full = (uint64_t*)smem;
    uint64_t* empty = full + MX_MAX_STAGES;
    uint64_t* acc_done = empty + MX_MAX_STAGES;
    uint64_t* x_there = acc_done + 1;
    uint32_t* tmem_slot = (uint32_t*)(x_there + 1);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    uint8_t* x_codes = smem + 1024;                                                       // FUSED: [steps][16 rows x 128 bytes], swizzled
    uint8_t* x_sf = x_codes + (FUSED ? a.x_steps * MX_FUSED_X : 0);                       // FUSED: [steps][two scale tiles]
    uint8_t* ring = smem + 1024 + (FUSED ? mx_fused_x_bytes(a.x_steps) : 0);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = a.splits > 1 ? (int)cluster_rank() : 0;
    const int row0 = (int)(blockIdx.x / (unsigned)a.splits) * MX_ROWS, tok0 = (int)blockIdx.y * a.n_tile;
    const int n_tok = min(a.n_tile, a.B - tok0), n_mma = (n_tok + 15) / 16 * 16;
    const int kt = (int)mx_tiles_k(a.K), steps = (a.K + MX_K - 1) / MX_K;
    const int s_begin = (int)((long long)steps * rank / a.splits), s_end = (int)((long long)steps * (rank + 1) / a.splits);
    const int stage_bytes = FUSED ? MX_FUSED_STAGE : mx_stage_bytes(a.n_tile), sf_at = FUSED ? MX_A_BYTES : MX_A_BYTES + a.n_tile * (MX_K / 2);
    const uint32_t tmem_cols = mx_tmem_cols(a.n_tile, a.stages);
    const int used = (n_tok + 127) / 128;   // groups of 128 tokens that hold any
    const uint8_t* wsc = a.w_scales + (size_t)(row0 / 128) * kt * MX_TILE;
    auto scale_bytes = [&](int s) { return (uint32_t)min(2, kt - 2 * s) * MX_TILE; };
    auto ask_weights = [&](int s, int st) {   // and what the stage waits for altogether
        const uint32_t bar = smem_u32(&full[st]), at = smem_u32(ring + st * stage_bytes);
        mbar_arrive_expect_tx(bar, (uint32_t)(FUSED ? MX_A_BYTES : sf_at) + scale_bytes(s) * (uint32_t)(FUSED ? 1 : 1 + used));
        tma_load_2d(at, &wmap, s * (MX_K / 2), row0, bar);
        bulk_copy_g2s(at + (uint32_t)sf_at, wsc + (size_t)s * MX_SFA_BYTES, scale_bytes(s), bar);
    };
    auto ask_tokens = [&](int s, int st) {
        const uint32_t bar = smem_u32(&full[st]), at = smem_u32(ring + st * stage_bytes);
        tma_load_2d(at + MX_A_BYTES, &xmap, s * (MX_K / 2), tok0, bar);
        for (int g = 0; g < used; g++)
            bulk_copy_g2s(at + (uint32_t)(sf_at + (1 + g) * MX_SFA_BYTES), a.x_scales + ((size_t)(tok0 / 128 + g) * kt + 2 * s) * MX_TILE, scale_bytes(s), bar);
    };

    const int ahead = min(a.stages, s_end - s_begin);   // stages that need no waiting for
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < a.stages; s++) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        mbar_init(smem_u32(acc_done), 1);
        mbar_init(smem_u32(x_there), 8);
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
            if constexpr (!FUSED)
                for (int i = 0; i < ahead; i++) ask_tokens(s_begin + i, i);
            int st = 0;
            uint32_t use = 0;
            for (int s = s_begin + ahead; s < s_end; s++) {
                mbar_wait_bounded(smem_u32(&empty[st]), use, abort_flag, a.status, ST_WAIT_EMPTY_TIMEOUT);
                ask_weights(s, st);
                if constexpr (!FUSED) ask_tokens(s, st);
                if (++st == a.stages) { st = 0; use ^= 1u; }
            }
        }
    } else if (warp == 1) {
        int st = 0;
        uint32_t use = 0;
        const uint64_t desc0 = umma_desc_sw128(0);
        const uint32_t sf_cols = tmem_base + (uint32_t)mx_acc_cols(a.n_tile), ring_at = smem_u32(ring), idesc = mx_idesc(MX_ROWS, n_mma);
        uint32_t xc = smem_u32(x_codes), xs = smem_u32(x_sf);
        if constexpr (FUSED) mbar_wait_bounded(smem_u32(x_there), 0u, abort_flag, a.status, ST_WAIT_FULL_TIMEOUT);
        for (int s = s_begin; s < s_end; s++) {
            mbar_wait_bounded(smem_u32(&full[st]), use, abort_flag, a.status, ST_WAIT_FULL_TIMEOUT);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t at = ring_at + (uint32_t)(st * stage_bytes), sfa = at + (uint32_t)sf_at;
            const uint32_t b_at = FUSED ? xc : at + MX_A_BYTES, sfb = FUSED ? xs : sfa + MX_SFA_BYTES;
            const uint32_t cols = sf_cols + (uint32_t)(st * mx_scale_cols(a.n_tile));
            const int n_k = (a.K - s * MX_K + 63) / 64;   // steps of 64 K that hold any; codes behind K are zero
            if (elect_one()) {
                mx_issue_stage<false, GROUPS>(n_k, tmem_base, desc0 + (at >> 4), desc0 + (b_at >> 4), sfa, sfb, cols, 8u, idesc, s > s_begin ? 1u : 0u);
                umma_commit<false>(smem_u32(&empty[st]));
                if (s == s_end - 1) umma_commit<false>(smem_u32(acc_done));
            }
            __syncwarp();
            xc += MX_FUSED_X;
            xs += MX_SFA_BYTES;
            if (++st == a.stages) { st = 0; use ^= 1u; }
        }
    } else if constexpr (FUSED) {
        // units of eight values, four lanes a block; behind K zeros as far as the last step of 64 K reaches
        const int k0 = s_begin * MX_K, units = (min(s_end * MX_K, (a.K + 63) / 64 * 64) - k0) / 8;
        const bool vec = ((uintptr_t)a.x & 15) == 0;
        constexpr int AHEAD = 3;   // units of a lane on their way at a time (5120 K: all of them)
        for (int u0 = 32 * (warp - 2); u0 < units; u0 += 256 * AHEAD) {
            float v[AHEAD][8] = {};
#pragma unroll
            for (int g = 0; g < AHEAD; g++) {
                const int k = 8 * (u0 + 256 * g + lane);
                if (k < 8 * units && k0 + k < a.K) load_x8(a.x, a.x_kind, k0 + k, vec, v[g]);
            }
#pragma unroll
            for (int g = 0; g < AHEAD; g++) {
                if (u0 + 256 * g >= units) break;   // (the whole warp)
                const int k = 8 * (u0 + 256 * g + lane);
                uint32_t top = 0u;
#pragma unroll
                for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(v[g][i]) & 0x7FFFFFFFu);
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                float inv;
                const uint32_t byte = mx_scale(top, inv);
#pragma unroll
                for (int i = 0; i < 8; i++) v[g][i] *= inv;
                const uint32_t code = e2m1_eight(v[g]);
                if (k < 8 * units) {   // row 0 of operand B: 128 bytes a stage hold 256 K, in order (the swizzle moves rows 1 to 7)
                    const int s = k / MX_K, b = k % MX_K / 2;
                    *(uint32_t*)(x_codes + s * MX_FUSED_X + b) = code;
                    if (lane % 4 == 0) x_sf[s * MX_SFA_BYTES + b / 64 * MX_TILE + b / 16 % 4] = (uint8_t)byte;
                }
            }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(x_there));
    }

    // ---------------- warps 2..9 store: lanes 32 (warp % 4) .. + 31 of the accumulator are 32 rows; two warps share their tokens ----------------
    const int part = (warp - 2) >> 2;
    const int n_chunks = (n_tok + 15) / 16, quad = warp & 3, row = row0 + 32 * quad + lane;
    const uint32_t acc = tmem_base + ((uint32_t)(32 * quad) << 16);
    T* Y = (T*)a.Y;
    auto store = [&](int chunk, const float (&v)[16]) {
        if (row >= a.M) return;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const int t = 16 * chunk + j;
            if (t < n_tok) {
                T* y = Y + (size_t)(tok0 + t) * a.ldy + row;
                *y = from_f32<T>(a.accumulate ? to_f32(*y) + v[j] : v[j]);
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
                float f[16];
                tmem_ld16(acc + (uint32_t)(16 * chunk), v);
#pragma unroll
                for (int j = 0; j < 16; j++) f[j] = __uint_as_float(v[j]);
                store(chunk, f);
            }
    } else {
        // Chunk c of the tile is finished by rank c % splits: the others put their sums of it into that CTA's shared memory,
        // [source][c / splits][16 tokens][128 rows]; sums are added in rank order.  Few tokens have a place of their own there; more go over
        // the ring, which every CTA's tensor core has read by then.
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
                const uint32_t to = peer_smem(box + (uint32_t)((src * own_chunks + chunk / a.splits) * (16 * MX_ROWS) + 32 * quad + lane) * 4u, (uint32_t)owner);
#pragma unroll
                for (int j = 0; j < 16; j++) st_peer_f32(to + (uint32_t)(j * MX_ROWS * 4), v[j]);
            }
        cluster_sync_all();   // all sums have arrived; nobody touches another CTA's memory after this
        if (warp >= 2)
            for (int own = part; own * a.splits + rank < n_chunks; own += 2) {
                uint32_t v[16];
                float f[16] = {};
                tmem_ld16(acc + (uint32_t)(16 * (own * a.splits + rank)), v);
                for (int r = 0; r < a.splits; r++) {
                    const float* in = (const float*)boxes + (size_t)((r - (r > rank ? 1 : 0)) * own_chunks + own) * (16 * MX_ROWS) + 32 * quad + lane;
#pragma unroll
                    for (int j = 0; j < 16; j++) f[j] += r == rank ? __uint_as_float(v[j]) : in[j * MX_ROWS];
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
// Many tokens: two CTAs (a cluster of two on neighbouring SMs) multiply as one, M = 256: each holds 128 weight rows and half of
// the tokens' codes, so that a stage costs an SM 16 + 16 KB of codes for 256 x 256 instead of 16 + 32 for 128 x 256.  The pairs
// stay and walk the tiles (tokens fastest: neighbours read the same weights out of L2), the ring runs on across tiles, and eight warps
// bring the accumulator to registers and hand it back before they store: the tensor core goes on meanwhile.  Bound by shared memory: a
// stage of 256 tokens writes 35 KB there and the tensor cores of both SMs read 48 KB of it, 650 clocks at 128 bytes, of which the MMA need 512;
// it takes 870 (2048 x 17408 x 5120 in 73 us = 5.0 PFLOP/s; without stores 61, loads alone 44).  Outputs leave through
// shared memory and TMA stores (a token's 128 rows are one piece of 256 or 512 bytes) where Y's base and row stride are multiples of 16
// bytes; plain stores, 64 bytes of a token a warp in 16 bits, stood in the way of the loads: 2048 x 17408 x 5120 76 us, 61 without them.
// ---------------------------------------------------------------------------------------------------------------
constexpr int MXP_THREADS = 320, MXP_EPI_WARPS = 8;
constexpr int MXP_OUT_BYTES = 4096;   // one TMA store: 16 tokens (8 in 32 bits) x 128 rows; two halves of the storing warps with two buffers each
constexpr int MXP_FIXED_SMEM = 1024 + 4 * MXP_OUT_BYTES;

struct MxPairArgs {
    void* Y;
    long long ldy;
    int* status;
    int K, M, B, accumulate;
    int n_tile, stages, n_acc, tok_tiles, n_tiles, pdl, tma_out;
};
__host__ __device__ constexpr int mxp_stage_bytes(int n_tile) { return MX_A_BYTES + n_tile / 2 * (MX_K / 2) + MX_SFA_BYTES * (1 + mx_groups(n_tile)); }

template <typename T, int GROUPS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(MXP_THREADS, 1)
mx4_pair_kernel(const MxPairArgs a, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wsmap,
                const __grid_constant__ CUtensorMap xsmap, const __grid_constant__ CUtensorMap ymap) {
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* full = (uint64_t*)smem;                // CTA 0's: the bytes of both CTAs
    uint64_t* empty = full + MX_MAX_STAGES;          // each CTA's
    uint64_t* acc_full = empty + MX_MAX_STAGES;      // [2] each CTA's
    uint64_t* acc_empty = acc_full + 2;              // [2] CTA 0's: the storing warps of both
    uint32_t* tmem_slot = (uint32_t*)(acc_empty + 2);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    uint8_t* ring = smem + MXP_FIXED_SMEM;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, side = (int)cluster_rank();
    const int pair = (int)(blockIdx.x >> 1), n_pairs = (int)(gridDim.x >> 1);
    const int steps = (a.K + MX_K - 1) / MX_K;
    const int stage_bytes = mxp_stage_bytes(a.n_tile);

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < a.stages; s++) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(smem_u32(&acc_full[i]), 1);
            mbar_init(smem_u32(&acc_empty[i]), 2 * MXP_EPI_WARPS);
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
        // The whole warp walks and one elected lane issues, as for the MMA: the addresses stay in uniform registers (under `if (lane == 0)`
        // four copies and a wait took some 700 clocks a stage: 2048 x 17408 x 5120 in tiles of 192 tokens 85 -> 78 us, 128 tokens 107 -> 93).
        int st = 0;
        uint32_t use = 0;
        const uint32_t ring_at = smem_u32(ring), full_at = peer_smem(smem_u32(full), 0u);
        for (int tile = pair; tile < a.n_tiles; tile += n_pairs) {
            const int row0 = tile / a.tok_tiles * 256 + side * MX_ROWS, tok0 = tile % a.tok_tiles * a.n_tile;
            const int tok = tok0 + side * ((min(a.n_tile, a.B - tok0) + 31) / 32 * 16);
            for (int s = 0; s < steps; s++) {
                mbar_wait_bounded(smem_u32(&empty[st]), use ^ 1u, abort_flag, a.status, ST_WAIT_EMPTY_TIMEOUT);
                const uint32_t bar = full_at + 8u * (uint32_t)st, at = ring_at + (uint32_t)(st * stage_bytes), sf = at + MX_A_BYTES + (uint32_t)(a.n_tile / 2) * (MX_K / 2);
                if (elect_one()) {
                    if (side == 0) mbar_arrive_expect_tx(smem_u32(&full[st]), 2u * (uint32_t)stage_bytes);
                    tma_load_2d_pair(at, &wmap, s * (MX_K / 2), row0, bar);
                    tma_load_2d_pair(at + MX_A_BYTES, &xmap, s * (MX_K / 2), tok, bar);
                    tma_load_3d_pair(sf, &wsmap, 0, 2 * s, row0 / 128, bar);
                    tma_load_3d_pair(sf + MX_SFA_BYTES, &xsmap, 0, 2 * s, tok0 / 128, bar);
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
            const uint32_t sf_cols = tmem_base + (uint32_t)(a.n_acc * mx_acc_cols(a.n_tile)), ring_at = smem_u32(ring);
            for (int tile = pair; tile < a.n_tiles; tile += n_pairs) {
                const int tok0 = tile % a.tok_tiles * a.n_tile, n_mma = (min(a.n_tile, a.B - tok0) + 31) / 32 * 32;
                const uint32_t first_col = (uint32_t)(8 + (tok0 & 127) / 32), d = tmem_base + (uint32_t)(acc * mx_acc_cols(a.n_tile)), idesc = mx_idesc(256, n_mma);
                mbar_wait_bounded(smem_u32(&acc_empty[acc]), acc_use ^ 1u, abort_flag, a.status, ST_TMEM_TIMEOUT);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int s = 0; s < steps; s++) {
                    mbar_wait_bounded(smem_u32(&full[st]), use, abort_flag, a.status, ST_WAIT_FULL_TIMEOUT);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t at = ring_at + (uint32_t)(st * stage_bytes), sf = at + MX_A_BYTES + (uint32_t)(a.n_tile / 2) * (MX_K / 2);
                    const uint32_t cols = sf_cols + (uint32_t)(st * mx_scale_cols(a.n_tile));
                    const int n_k = (a.K - s * MX_K + 63) / 64;
                    if (elect_one()) {
                        mx_issue_stage<true, GROUPS>(n_k, d, desc0 + (at >> 4), desc0 + ((at + MX_A_BYTES) >> 4), sf, sf + MX_SFA_BYTES, cols, first_col, idesc, s > 0 ? 1u : 0u);
                        umma_commit<true>(smem_u32(&empty[st]));
                        if (s == steps - 1) umma_commit<true>(smem_u32(&acc_full[acc]));
                    }
                    __syncwarp();
                    if (++st == a.stages) { st = 0; use ^= 1u; }
                }
                if (++acc == a.n_acc) { acc = 0; acc_use ^= 1u; }
            }
        }
    } else {
        // a warp reads the 16-token chunks 2 i + part of its quarter of the rows
        const int quad = warp & 3, part = (warp - 2) >> 2;
        constexpr int OUT_TOK = MXP_OUT_BYTES / (MX_ROWS * (int)sizeof(T));
        uint8_t* out = smem + 1024 + part * 2 * MXP_OUT_BYTES;
        const bool storer = quad == 0 && lane == 0;
        int acc = 0, buf = 0;
        uint32_t acc_use = 0;
        T* Y = (T*)a.Y;
        for (int tile = pair; tile < a.n_tiles; tile += n_pairs) {
            const int row0 = tile / a.tok_tiles * 256 + side * MX_ROWS, row = row0 + 32 * quad + lane, tok0 = tile % a.tok_tiles * a.n_tile, n_tok = min(a.n_tile, a.B - tok0);
            mbar_wait_bounded(smem_u32(&acc_full[acc]), acc_use, abort_flag, a.status, ST_TMEM_TIMEOUT);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t from = tmem_base + ((uint32_t)(32 * quad) << 16) + (uint32_t)(acc * mx_acc_cols(a.n_tile) + 16 * part);
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
            if (++acc == a.n_acc) { acc = 0; acc_use ^= 1u; }
            auto value = [&](int i, int j) {
                const float f = __uint_as_float(v[i][j]);
                if (!a.accumulate) return from_f32<T>(f);
                const int t = 16 * (2 * i + part) + j;
                return row < a.M && t < n_tok ? from_f32<T>(to_f32(Y[(size_t)(tok0 + t) * a.ldy + row]) + f) : from_f32<T>(f);
            };
            // (a store is clipped in whole 16-byte units only: a last tile that ends inside one goes by plain stores)
            if (a.tma_out && (row0 + MX_ROWS <= a.M || a.M % (16 / (int)sizeof(T)) == 0)) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (16 * (2 * i + part) >= n_tok) break;
#pragma unroll
                    for (int h = 0; h < 16 / OUT_TOK; h++) {
                        if (storer) tma_store_wait_read<1>();
                        named_bar_sync(1 + part, 128);   // the buffer of two stores before is free
                        T* to = (T*)(out + buf * MXP_OUT_BYTES) + 32 * quad + lane;
#pragma unroll
                        for (int j = 0; j < OUT_TOK; j++) to[j * MX_ROWS] = value(i, OUT_TOK * h + j);
                        fence_proxy_async();
                        named_bar_sync(1 + part, 128);
                        if (storer) {
                            tma_store_2d(&ymap, smem_u32(out + buf * MXP_OUT_BYTES), row0, tok0 + 16 * (2 * i + part) + OUT_TOK * h);
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

// How a product is cut: tokens in tiles of n_tile (one tile, or several of 128 or 256: a tile starts on a scale tile's border), K in
// `splits` parts, few tokens with two CTAs to an SM, each with half of its shared memory.
struct MxCut { int n_tile, stages, splits, box, per_sm; };   // box: bytes of shared memory for the others' sums (0: over the ring)

int exchange_bytes(const MxCut& c) {
    const int chunks = c.n_tile / 16;
    return (c.splits - 1) * ((chunks + c.splits - 1) / c.splits) * 16 * MX_ROWS * 4;
}
// what a CTA has for its ring and what stands behind it
int mx_ring_bytes(int smem_optin, const MxCut& c) { return (c.per_sm == 2 ? (smem_optin + 1024) / 2 - 1024 : smem_optin) - 1024 - c.box; }
// stages of weights beside one token's codes
int mx_fused_stages(int smem_optin, const MxCut& c, int x_steps) { return std::min(MX_MAX_STAGES, (mx_ring_bytes(smem_optin, c) - mx_fused_x_bytes(x_steps)) / MX_FUSED_STAGE); }

// ... by their time in SM clocks, of one wave of CTAs after the other: what starts and drains a CTA, the exchange of split sums, and stages, each as
// long as a CTA takes alone (two of an SM: twice) or, if that is longer, as its bytes take out of L2 (6400 a clock for all SMs) and its weights out of
// DRAM (3300).  Fitted to 1024, 5120 and 17408 rows, 16 to 768 tokens, in every number of parts and tiles: the taken cut is within 4 % of the best
// there, but for one token (below).  1024 x 5120: 256 tokens 11.1 -> 8.2 us, 512 tokens 20.5 -> 9.0; 5120 x 17408, 256 tokens 24.1 -> 20.8 (before,
// a stage counted 600 clocks and 5 a token, whoever else ran).
// Two CTAs of an SM overlap their ends, and parts fill all SMs: 7 x 5120 x 17408 in six parts 13.7 us, in three of whole SMs 14.8; 7 x 12288 x 5120 in two
// 11.5 and 12.5; one token x 248320 x 5120 112 and 130.  One token's codes take shared memory too, of which a ring of three stages has to remain.  And
// where not all CTAs run at once each wave quantizes its part anew: more than two parts, six at most, pay in one wave (1 x 6144 x 10240 in five 10.8 us, in two
// of whole SMs 12.7; 10752 x 10240 in three 14.5, undivided 18.1; 55 of 59 drawn sizes gained, up to a quarter, 3200 x 5632 in six lost 0.5 us; in seven 21 of
// 25 lost) and not in several (24576 x 10240 in four 32.7, undivided 26.3; 19 of 24 lost).  Two such CTAs hold at most 256 columns of tensor memory
// each, and no other kernel here that allocates columns fits beside one (registers, shared memory): no cluster waits for columns that another waiting
// one holds.
// Clusters of three to six leave an eighth of the SMs unused, larger ones three tenths (45, 33, 26, 22, 15 and 15 clusters were there at a time).
MxCut mx_cut(int sm_count, int smem_optin, int K, int M, int B, double* cost_of) {
    MxCut best = {};
    double best_cost = 0.0;
    const int steps = (K + MX_K - 1) / MX_K, whole = B <= MX_MAX_N ? (B + 15) / 16 * 16 : MX_MAX_N;
    const auto rate = [&](int n, int per_sm) {
        MxCut c = {};
        c.n_tile = n;
        c.per_sm = per_sm;
        const long long tok_tiles = (B + n - 1) / n, tiles = (long long)((M + MX_ROWS - 1) / MX_ROWS) * tok_tiles;
        for (c.splits = 1; c.splits <= std::min(MX_MAX_SPLITS, steps); c.splits++) {
            const int own_steps = (steps + c.splits - 1) / c.splits;
            c.box = c.splits > 1 && n <= 32 ? exchange_bytes(c) : 0;
            c.stages = std::min(std::min(MX_MAX_STAGES, mx_ring_bytes(smem_optin, c) / mx_stage_bytes(n)), (512 / per_sm - mx_acc_cols(n)) / mx_scale_cols(n));
            if (c.splits > 1 && !c.box && exchange_bytes(c) > c.stages * mx_stage_bytes(n)) break;
            const int sms = c.splits <= 2 ? sm_count : c.splits <= 6 ? sm_count * 7 / 8 : sm_count * 7 / 10;
            const long long ctas = tiles * c.splits, once = std::max(1, sms / c.splits) * (long long)c.splits, slots = per_sm * once, waves = (ctas + slots - 1) / slots;
            if (per_sm == 2) {
                if (ctas <= once || c.stages < 3 || own_steps < 4) continue;   // (shorter ones are all ends: 16 x 2048 x 2048 in eight parts 6.5 us, 5.6 otherwise)
                if (B == 1 && own_steps * MX_K <= MX_FUSE_MAX_K && ((c.splits > 2 && (waves > 1 || c.splits > 6)) || mx_fused_stages(smem_optin, c, own_steps) < 3)) continue;
            }
            const double active = (double)std::min(ctas, slots);
            const double stage = std::max({per_sm * (590.0 + 0.45 * n), active * mx_stage_bytes(n) / 6400.0, active / (double)tok_tiles * (MX_A_BYTES + MX_SFA_BYTES) / 3300.0});
            const double cost = 3600.0 + (double)waves * (own_steps * stage + (per_sm == 2 ? 0.0 : 3000.0) + 37.0 * n + (c.splits > 1 ? 1900.0 : 0.0));
            if (!best.n_tile || cost < best_cost) { best = c; best_cost = cost; }
        }
    };
    rate(whole, 1);
    if (whole > 128) rate(128, 1);
    if (whole <= 32) rate(whole, 2);
    if (cost_of) *cost_of = best_cost;
    return best;
}

// Tiles of a product in pairs: 64, 128, 192 or 256 tokens (a tile starts on half a scale tile), by their time in SM clocks as above: rounds of
// tiles over the pairs (2048 x 17408 x 5120 in tiles of 128, 192 and 256 tokens: 93, 78 and 74 us; 333 x 16384 x 5120: 22, 21 and 26), what starts and
// drains a pair, and what a tile costs beside its stages, less where two accumulators take turns.
struct MxPairCut { int n_tile, stages, n_acc, tok_tiles, n_tiles; };
MxPairCut mx_pair_cut(int sm_count, int smem_optin, int K, int M, int B, int forced, double* cost_of) {
    MxPairCut best = {};
    double best_cost = 0.0;
    const int row_tiles = (M + 255) / 256, steps = (K + MX_K - 1) / MX_K;
    for (int n = 64; n <= 256; n += 64) {
        if (forced && n != forced) continue;
        MxPairCut c;
        c.n_tile = n;
        c.tok_tiles = (B + n - 1) / n;
        if ((long long)row_tiles * c.tok_tiles > 0x7FFFFFFF) continue;
        c.n_tiles = row_tiles * c.tok_tiles;
        c.stages = std::min(MX_MAX_STAGES, (smem_optin - MXP_FIXED_SMEM) / mxp_stage_bytes(n));
        c.n_acc = 1;
        const int two = (512 - 2 * mx_acc_cols(n)) / mx_scale_cols(n);   // stages whose scales fit beside two accumulators
        if (two >= 4) {
            c.n_acc = 2;
            c.stages = std::min(c.stages, two);
        }
        const int pairs = sm_count / 2;
        const double active = (double)std::min(c.n_tiles, pairs);
        const double stage = std::max(400.0 + 0.87 * n, active * 2.0 * mxp_stage_bytes(n) / 6200.0), weights = active / c.tok_tiles * 2.0 * (MX_A_BYTES + MX_SFA_BYTES) / 3300.0;
        const double cost = 7800.0 + 24.0 * n + (double)((c.n_tiles + pairs - 1) / pairs) * std::max(steps * stage + (c.n_acc == 2 ? 1700.0 : 2700.0), steps * weights);
        if (!best.n_tile || cost < best_cost) { best = c; best_cost = cost; }
    }
    if (cost_of) *cost_of = best_cost;
    return best;
}

size_t kind_size(int kind) { return kind == Q38B_OUT_F32 ? 4 : 2; }
bool known_kind(int kind) { return kind == Q38B_OUT_F32 || kind == Q38B_OUT_F16 || kind == Q38B_OUT_BF16; }
// (sizes that leave room for rounding up in 32 bits)
bool mx_shape(int K, int rows) { return K >= 32 && K % 32 == 0 && K <= 1 << 30 && rows >= 1 && rows <= 1 << 30; }

template <typename T>
int quantize_as(q38b_ctx* ctx, const void* x, long long x_ld, int K, int rows, uint8_t* codes, long long codes_ld, uint8_t* scales, cudaStream_t st) {
    const long long blocks = (mx_walk_warps(K, rows) + 7) / 8;
    if (blocks > 0x7FFFFFFF) return Q38B_ERR_UNSUPPORTED;
    const unsigned grid = (unsigned)blocks;
    const bool vec = (((uintptr_t)x | (uintptr_t)(x_ld * (long long)sizeof(T))) & 15) == 0;
    if (vec) mx4_quantize_kernel<T, true><<<grid, 256, 0, st>>>((const T*)x, x_ld, K, rows, codes, codes_ld, scales);
    else mx4_quantize_kernel<T, false><<<grid, 256, 0, st>>>((const T*)x, x_ld, K, rows, codes, codes_ld, scales);
    return launch_status(ctx, cudaSuccess);
}

template <typename T>
int dequant_as(q38b_ctx* ctx, const uint8_t* codes, long long codes_ld, const uint8_t* scales, int K, int rows, void* out, long long out_ld, cudaStream_t st) {
    const long long blocks = (mx_walk_warps(K, rows) + 7) / 8;
    if (blocks > 0x7FFFFFFF) return Q38B_ERR_UNSUPPORTED;
    const bool vec = (((uintptr_t)out | (uintptr_t)(out_ld * (long long)sizeof(T))) & 15) == 0;
    if (vec) mx4_dequant_kernel<T, true><<<(unsigned)blocks, 256, 0, st>>>(codes, codes_ld, scales, K, rows, (T*)out, out_ld);
    else mx4_dequant_kernel<T, false><<<(unsigned)blocks, 256, 0, st>>>(codes, codes_ld, scales, K, rows, (T*)out, out_ld);
    return launch_status(ctx, cudaSuccess);
}

bool encode_codes(CUtensorMap* map, const void* codes, long long ld, int K, int rows, int box_rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)K / 2, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {MX_K / 2, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    EncodeTiledFn enc = encode_fn();
    return enc && enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)codes, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// the scale tiles of a matrix as they lie: 512 bytes x K tiles x row tiles
bool encode_scales(CUtensorMap* map, const void* scales, int K, int rows, int groups) {
    const cuuint64_t kt = (cuuint64_t)mx_tiles_k(K);
    const cuuint64_t dims[3] = {MX_TILE / 4, kt, (cuuint64_t)((rows + 127) / 128)};
    const cuuint64_t strides[2] = {MX_TILE, kt * MX_TILE};
    const cuuint32_t box[3] = {MX_TILE / 4, 2, (cuuint32_t)groups}, estr[3] = {1, 1, 1};
    EncodeTiledFn enc = encode_fn();
    return enc && enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, (void*)scales, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// the outputs, stored in pieces of MXP_OUT_BYTES; false: they go there by plain stores
bool encode_out(CUtensorMap* map, void* Y, int kind, long long ldy, int M, int B) {
    const int size = kind == Q38B_OUT_F32 ? 4 : 2;
    if (((uintptr_t)Y & 15) || (ldy * size) % 16) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)M, (cuuint64_t)B};
    const cuuint64_t strides[1] = {(cuuint64_t)ldy * size};
    const cuuint32_t box[2] = {MX_ROWS, (cuuint32_t)(MXP_OUT_BYTES / (MX_ROWS * size))}, estr[2] = {1, 1};
    EncodeTiledFn enc = encode_fn();
    return enc && enc(map, kind == Q38B_OUT_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : kind == Q38B_OUT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, Y,
                      dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T>
int pair_as(q38b_ctx* ctx, const MxPairArgs& a, const CUtensorMap& wmap, const CUtensorMap& xmap, const CUtensorMap& wsmap, const CUtensorMap& xsmap, const CUtensorMap& ymap,
            cudaStream_t st) {
    auto kern = mx_groups(a.n_tile) == 1 ? mx4_pair_kernel<T, 1> : mx4_pair_kernel<T, 2>;
    const int rc = q38b_ensure_kernel_smem(ctx, (const void*)kern, ctx->smem_optin, false);
    if (rc != Q38B_OK) return rc;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(2u * (unsigned)std::min(ctx->sm_count / 2, a.n_tiles));
    cfg.blockDim = dim3(MXP_THREADS);
    cfg.dynamicSmemBytes = (size_t)(MXP_FIXED_SMEM + a.stages * mxp_stage_bytes(a.n_tile));
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.pdl ? 1 : 0;
    return launch_status(ctx, cudaLaunchKernelEx(&cfg, kern, a, wmap, xmap, wsmap, xsmap, ymap));
}

// where the shared memory behind the ring begins
template <bool FUSED> int mx_box_at(const MxArgs& a) { return 1024 + (FUSED ? mx_fused_x_bytes(a.x_steps) + a.stages * MX_FUSED_STAGE : a.stages * mx_stage_bytes(a.n_tile)); }

template <typename T, int GROUPS, bool FUSED>
int gemm_as(q38b_ctx* ctx, const MxArgs& a, int box, const CUtensorMap& wmap, const CUtensorMap& xmap, cudaStream_t st) {
    auto kern = mx4_gemm_kernel<T, GROUPS, FUSED>;
    const int rc = q38b_ensure_kernel_smem(ctx, (const void*)kern, ctx->smem_optin, false);
    if (rc != Q38B_OK) return rc;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)((a.M + MX_ROWS - 1) / MX_ROWS * a.splits), (unsigned)((a.B + a.n_tile - 1) / a.n_tile));
    cfg.blockDim = dim3(MX_THREADS);
    cfg.dynamicSmemBytes = (size_t)mx_box_at<FUSED>(a) + box;
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
template <int GROUPS, bool FUSED>
int gemm_kind(q38b_ctx* ctx, MxArgs a, int box, const CUtensorMap& wmap, const CUtensorMap& xmap, int y_kind, cudaStream_t st) {
    a.box_at = box ? mx_box_at<FUSED>(a) : 0;
    return y_kind == Q38B_OUT_F32 ? gemm_as<float, GROUPS, FUSED>(ctx, a, box, wmap, xmap, st)
         : y_kind == Q38B_OUT_F16 ? gemm_as<__half, GROUPS, FUSED>(ctx, a, box, wmap, xmap, st)
                                  : gemm_as<__nv_bfloat16, GROUPS, FUSED>(ctx, a, box, wmap, xmap, st);
}

MxArgs mx_args(q38b_ctx* ctx, const MxCut& cut, const void* W_scales, int K, int M, int B, void* Y, long long ldy, int accumulate) {
    MxArgs a;
    memset(&a, 0, sizeof(a));
    a.w_scales = (const uint8_t*)W_scales;
    a.Y = Y;
    a.ldy = ldy;
    a.status = ctx->d_status;
    a.K = K;
    a.M = M;
    a.B = B;
    a.accumulate = accumulate ? 1 : 0;
    a.n_tile = cut.n_tile;
    a.stages = cut.stages;
    a.splits = cut.splits;
    return a;
}

// arguments of one operand
int check_operand(const void* codes, long long ld, const void* scales, int K, int rows) {
    if (!codes || !scales || !mx_shape(K, rows) || ld < K / 2) return Q38B_ERR_ARG;
    return ((uintptr_t)codes & 15) || (ld & 15) || ((uintptr_t)scales & 15) ? Q38B_ERR_ALIGN : Q38B_OK;
}

// the product of two such matrices; behind_quantizer: launched while the kernel that makes X still runs, where the context allows it
int gemm_mx4(q38b_ctx* ctx, const void* W, long long W_ld, const void* W_scales, int K, int M, const void* X, long long X_ld, const void* X_scales, int B,
             void* Y, int y_kind, long long ldy, int accumulate, void* stream, bool behind_quantizer) {
    if (!ctx || !Y || !known_kind(y_kind) || ldy < M) return Q38B_ERR_ARG;
    int rc = check_operand(W, W_ld, W_scales, K, M);
    if (rc == Q38B_OK) rc = check_operand(X, X_ld, X_scales, K, B);
    if (rc != Q38B_OK) return rc;
    if ((uintptr_t)Y % kind_size(y_kind)) return Q38B_ERR_ALIGN;
    DeviceGuard on(ctx);
    cudaStream_t st = (cudaStream_t)stream;
    const int pdl = behind_quantizer && ctx->pass_pdl ? 1 : 0;
    double cost = 0.0, pair_cost = 0.0;
    const MxCut one = mx_cut(ctx->sm_count, ctx->smem_optin, K, M, B, &cost);
    const MxPairCut cut = mx_pair_cut(ctx->sm_count, ctx->smem_optin, K, M, B, ctx->mx4_pairs > 0 ? ctx->mx4_pairs : 0, &pair_cost);
    const bool too_many = (B + one.n_tile - 1) / one.n_tile > 65535;   // token tiles, for a grid's second dimension
    if (ctx->mx4_pairs > 0 || (ctx->mx4_pairs == 0 && (too_many || (B > 1 && M > MX_ROWS && pair_cost < cost)))) {
        if (!cut.n_tile) return Q38B_ERR_UNSUPPORTED;
        CUtensorMap wmap, xmap, wsmap, xsmap, ymap;
        memset(&ymap, 0, sizeof(ymap));
        const int tma_out = encode_out(&ymap, Y, y_kind, ldy, M, B) ? 1 : 0;
        if (!encode_codes(&wmap, W, W_ld, K, M, MX_ROWS) || !encode_codes(&xmap, X, X_ld, K, B, cut.n_tile / 2) || !encode_scales(&wsmap, W_scales, K, M, 1) ||
            !encode_scales(&xsmap, X_scales, K, B, mx_groups(cut.n_tile)))
            return Q38B_ERR_ARG;
        const MxPairArgs a = {Y, ldy, ctx->d_status, K, M, B, accumulate ? 1 : 0, cut.n_tile, cut.stages, cut.n_acc, cut.tok_tiles, cut.n_tiles, pdl, tma_out};
        return y_kind == Q38B_OUT_F32 ? pair_as<float>(ctx, a, wmap, xmap, wsmap, xsmap, ymap, st)
             : y_kind == Q38B_OUT_F16 ? pair_as<__half>(ctx, a, wmap, xmap, wsmap, xsmap, ymap, st)
                                      : pair_as<__nv_bfloat16>(ctx, a, wmap, xmap, wsmap, xsmap, ymap, st);
    }
    if (too_many) return Q38B_ERR_UNSUPPORTED;
    CUtensorMap wmap, xmap;
    if (!encode_codes(&wmap, W, W_ld, K, M, MX_ROWS) || !encode_codes(&xmap, X, X_ld, K, B, one.n_tile)) return Q38B_ERR_ARG;
    MxArgs a = mx_args(ctx, one, W_scales, K, M, B, Y, ldy, accumulate);
    a.x_scales = (const uint8_t*)X_scales;
    a.pdl = pdl;
    return mx_groups(a.n_tile) == 1 ? gemm_kind<1, false>(ctx, a, one.box, wmap, xmap, y_kind, st) : gemm_kind<2, false>(ctx, a, one.box, wmap, xmap, y_kind, st);
}

}  // namespace

extern "C" {

size_t q38b_mx4_scale_bytes(int K, int rows) { return mx_shape(K, rows) ? (size_t)((rows + 127) / 128) * (size_t)mx_tiles_k(K) * MX_TILE : 0; }

int q38b_quantize_mx4(q38b_ctx* ctx, const void* x, int x_kind, long long x_ld, int K, int rows, void* codes, long long codes_ld, void* scales, void* stream) {
    if (!ctx || !x || !known_kind(x_kind) || x_ld < K) return Q38B_ERR_ARG;
    const int rc = check_operand(codes, codes_ld, scales, K, rows);
    if (rc != Q38B_OK) return rc;
    if ((uintptr_t)x % kind_size(x_kind)) return Q38B_ERR_ALIGN;
    DeviceGuard on(ctx);
    cudaStream_t st = (cudaStream_t)stream;
    uint8_t *c = (uint8_t*)codes, *s = (uint8_t*)scales;
    return x_kind == Q38B_OUT_F32 ? quantize_as<float>(ctx, x, x_ld, K, rows, c, codes_ld, s, st)
         : x_kind == Q38B_OUT_F16 ? quantize_as<__half>(ctx, x, x_ld, K, rows, c, codes_ld, s, st)
                                  : quantize_as<__nv_bfloat16>(ctx, x, x_ld, K, rows, c, codes_ld, s, st);
}

int q38b_mx4_tile_scales(q38b_ctx* ctx, const void* src, long long src_ld, int K, int rows, void* scales, void* stream) {
    if (!ctx || !src || !scales || !mx_shape(K, rows) || src_ld < K / 32) return Q38B_ERR_ARG;
    if ((uintptr_t)scales & 15) return Q38B_ERR_ALIGN;
    DeviceGuard on(ctx);
    const size_t n = q38b_mx4_scale_bytes(K, rows);
    if ((n + 255) / 256 > 0x7FFFFFFF) return Q38B_ERR_UNSUPPORTED;
    mx4_tile_kernel<<<(unsigned)((n + 255) / 256), 256, 0, (cudaStream_t)stream>>>((const uint8_t*)src, src_ld, K, rows, (uint8_t*)scales);
    return launch_status(ctx, cudaSuccess);
}

int q38b_dequant_mx4(q38b_ctx* ctx, const void* codes, long long codes_ld, const void* scales, int K, int rows, void* out, int out_kind, long long out_ld,
                     void* stream) {
    if (!ctx || !out || !known_kind(out_kind) || out_ld < K) return Q38B_ERR_ARG;
    const int rc = check_operand(codes, codes_ld, scales, K, rows);
    if (rc != Q38B_OK) return rc;
    if ((uintptr_t)out % kind_size(out_kind)) return Q38B_ERR_ALIGN;
    DeviceGuard on(ctx);
    cudaStream_t st = (cudaStream_t)stream;
    const uint8_t *c = (const uint8_t*)codes, *s = (const uint8_t*)scales;
    return out_kind == Q38B_OUT_F32 ? dequant_as<float>(ctx, c, codes_ld, s, K, rows, out, out_ld, st)
         : out_kind == Q38B_OUT_F16 ? dequant_as<__half>(ctx, c, codes_ld, s, K, rows, out, out_ld, st)
                                    : dequant_as<__nv_bfloat16>(ctx, c, codes_ld, s, K, rows, out, out_ld, st);
}

int q38b_gemm_mx4(q38b_ctx* ctx, const void* W, long long W_ld, const void* W_scales, int K, int M, const void* X, long long X_ld, const void* X_scales, int B,
                  void* Y, int y_kind, long long ldy, int accumulate, void* stream) {
    return gemm_mx4(ctx, W, W_ld, W_scales, K, M, X, X_ld, X_scales, B, Y, y_kind, ldy, accumulate, stream, false);
}

size_t q38b_gemm_mx4_scratch_bytes(int K, int B) {
    if (!mx_shape(K, B) || (B == 1 && K <= MX_FUSE_MAX_K)) return 0;
    return (size_t)B * (K / 2) + q38b_mx4_scale_bytes(K, B) + 16;
}

int q38b_gemm_mx4_x(q38b_ctx* ctx, const void* W, long long W_ld, const void* W_scales, int K, int M, const void* x, int x_kind, long long x_ld, int B, void* Y,
                    int y_kind, long long ldy, int accumulate, void* scratch, size_t scratch_bytes, void* stream) {
    if (!ctx || !x || !Y || !known_kind(x_kind) || !known_kind(y_kind) || x_ld < K || B < 1) return Q38B_ERR_ARG;
    int rc = check_operand(W, W_ld, W_scales, K, M);
    if (rc != Q38B_OK) return rc;
    if (ldy < M) return Q38B_ERR_ARG;
    if ((uintptr_t)x % kind_size(x_kind) || (uintptr_t)Y % kind_size(y_kind)) return Q38B_ERR_ALIGN;
    const size_t need = q38b_gemm_mx4_scratch_bytes(K, B);
    if (need && !scratch) return Q38B_ERR_ARG;
    if ((uintptr_t)scratch & 15) return Q38B_ERR_ALIGN;
    if (scratch_bytes < need) return Q38B_ERR_NOMEM;
    if (B == 1 && ctx->mx4_pairs <= 0 && !ctx->mx4_two_launches) {
        MxCut cut = mx_cut(ctx->sm_count, ctx->smem_optin, K, M, B, nullptr);   // (the same cut as of the two calls: the same sums)
        const int steps = (K + MX_K - 1) / MX_K, x_steps = (steps + cut.splits - 1) / cut.splits;
        if (x_steps * MX_K <= MX_FUSE_MAX_K) {
            DeviceGuard on(ctx);
            cut.stages = mx_fused_stages(ctx->smem_optin, cut, x_steps);
            CUtensorMap wmap, none;
            memset(&none, 0, sizeof(none));
            if (!encode_codes(&wmap, W, W_ld, K, M, MX_ROWS)) return Q38B_ERR_ARG;
            MxArgs a = mx_args(ctx, cut, W_scales, K, M, B, Y, ldy, accumulate);
            a.x = x;
            a.x_kind = x_kind;
            a.x_steps = x_steps;
            return gemm_kind<1, true>(ctx, a, cut.box, wmap, none, y_kind, (cudaStream_t)stream);
        }
    }
    if (!scratch) return Q38B_ERR_ARG;
    uint8_t* scales = (uint8_t*)scratch;
    uint8_t* codes = scales + q38b_mx4_scale_bytes(K, B);
    if (scratch_bytes < (size_t)(codes - scales) + (size_t)B * (K / 2)) return Q38B_ERR_NOMEM;
    rc = q38b_quantize_mx4(ctx, x, x_kind, x_ld, K, B, codes, K / 2, scales, stream);
    if (rc != Q38B_OK) return rc;
    return gemm_mx4(ctx, W, W_ld, W_scales, K, M, codes, K / 2, scales, B, Y, y_kind, ldy, accumulate, stream, true);
}

// Test hook (not in the public header): products in pairs of CTAs never (-1), with tiles of `mode` tokens (64, 128, 192, 256), by the rule (0).
int q38b_debug_set_mx4_pairs(q38b_ctx* ctx, int mode) {
    if (!ctx || mode < -1 || mode > 256 || (mode > 0 && mode % 64)) return Q38B_ERR_ARG;
    ctx->mx4_pairs = mode;
    return Q38B_OK;
}

// Test hook (not in the public header): q38b_gemm_mx4_x quantizes in a launch of its own whatever the tokens.
int q38b_debug_set_mx4_two_launches(q38b_ctx* ctx, int enabled) {
    if (!ctx) return Q38B_ERR_ARG;
    ctx->mx4_two_launches = enabled ? 1 : 0;
    return Q38B_OK;
}

}  // extern "C"

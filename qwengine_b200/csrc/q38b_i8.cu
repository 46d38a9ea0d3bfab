// q38b_i8.cu -- 8-bit integers with one scale a row: quantizer, and the product of two such matrices.
//
//   scale = max(fl32(amax / 127), 2^-126), code = x / scale rounded half to even (exactly)
//   Y[t][r] (+)= X_scales[t] W_scales[r] sum_k X[t][k] W[r][k]
//
// The sums are whole numbers below 2^31 (K <= 131071, codes of 8 bits): exact in any order, whatever splits K.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "../../include/q38b200.h"
#include "q38b_host.h"
#include "q38b_internal.h"
#include "q38b_pipe.cuh"
#include "q38b_types.cuh"

using namespace q38b;

namespace {

constexpr int I8_MAX_K = 131071;

// What a row's codes are made with.  inv is 1 / scale rounded: x * inv is off by less than 2^-22 of the quotient, which is at most 127.5, so its
// nearest whole number n is the quotient's or, next to a half, one beside it.  x - n scale is exact in a fused operation (a multiple of the smaller
// of the two's last places, no larger than half a scale and a little), so comparing it with half the scale, itself exact, finds which, and ties.
struct RowScale { float scale, inv, half; bool bad; };
__device__ __forceinline__ RowScale row_scale(uint32_t top) {   // bit pattern of the largest magnitude
    RowScale r;
    r.bad = top >= 0x7F800000u;
    r.scale = r.bad ? __uint_as_float(0x7FC00000u) : fmaxf(__fdiv_rn(__uint_as_float(top), 127.0f), 1.17549435e-38f);
    r.inv = r.bad ? 0.0f : __fdiv_rn(1.0f, r.scale);
    r.half = 0.5f * r.scale;
    return r;
}
__device__ __forceinline__ int code_of(float x, const RowScale& r) {
    if (r.bad) return 0;
    float n = rintf(x * r.inv);
    const float rest = fmaf(-n, r.scale, x);
    const bool odd = ((int)n & 1) != 0;
    if (rest > r.half || (rest == r.half && odd)) n += 1.0f;
    else if (rest < -r.half || (rest == -r.half && odd)) n -= 1.0f;
    return (int)n;
}

// A block a row: the largest magnitude, then the codes.
template <typename T>
__global__ void __launch_bounds__(256) i8_quantize_kernel(const T* x, long long x_ld, int K, int8_t* codes, long long codes_ld, float* scales) {
    __shared__ uint32_t tops[8];
    const long long row = blockIdx.x;
    const T* p = x + row * x_ld;
    uint32_t top = 0u;
    for (int k = threadIdx.x; k < K; k += 256) top = max(top, __float_as_uint(to_f32(p[k])) & 0x7FFFFFFFu);
    top = __reduce_max_sync(0xffffffffu, top);
    if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) top = max(top, tops[w]);
    const RowScale r = row_scale(top);
    if (threadIdx.x == 0) scales[row] = r.scale;
    for (int k = threadIdx.x; k < K; k += 256) codes[row * codes_ld + k] = (int8_t)code_of(to_f32(p[k]), r);
}

struct I8Args {
    const int8_t *W, *X;
    const float *w_scales, *x_scales;
    void* Y;
    long long W_ld, X_ld, ldy;
    int K, M, B, accumulate;
};

// 64 x 64 outputs a block, 64 K at a time through shared memory, 4 x 4 outputs a thread.
template <typename T>
__global__ void __launch_bounds__(256) i8_simple_kernel(const I8Args a) {
    __shared__ int ws[64][17], xs[64][17];
    const int r0 = (int)blockIdx.x * 64, t0 = (int)blockIdx.y * 64, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < a.K; k0 += 64) {
        __syncthreads();
        for (int i = threadIdx.x; i < 64 * 64; i += 256) {
            const int r = i / 64, k = k0 + i % 64;
            ((int8_t*)&ws[r][0])[i % 64] = r0 + r < a.M && k < a.K ? a.W[(r0 + r) * a.W_ld + k] : (int8_t)0;
            ((int8_t*)&xs[r][0])[i % 64] = t0 + r < a.B && k < a.K ? a.X[(t0 + r) * a.X_ld + k] : (int8_t)0;
        }
        __syncthreads();
        for (int k = 0; k < 16; k++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __dp4a(ws[tx + 16 * i][k], xs[ty + 16 * j][k], acc[i][j]);
    }
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            const int r = r0 + tx + 16 * i, t = t0 + ty + 16 * j;
            if (r >= a.M || t >= a.B) continue;
            T* y = (T*)a.Y + (long long)t * a.ldy + r;
            const float v = (float)acc[i][j] * a.x_scales[t] * a.w_scales[r];
            *y = from_f32<T>(a.accumulate ? to_f32(*y) + v : v);
        }
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
    i8_quantize_kernel<T><<<(unsigned)rows, 256, 0, st>>>((const T*)x, x_ld, K, codes, codes_ld, scales);
    return launch_status(ctx, cudaSuccess);
}

template <typename T>
int gemm_as(q38b_ctx* ctx, const I8Args& a, cudaStream_t st) {
    i8_simple_kernel<T><<<dim3((unsigned)((a.M + 63) / 64), (unsigned)((a.B + 63) / 64)), 256, 0, st>>>(a);
    return launch_status(ctx, cudaSuccess);
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
    if (!ctx || !Y || !known_kind(y_kind) || ldy < M) return Q38B_ERR_ARG;
    int rc = check_operand(W, W_ld, W_scales, K, M);
    if (rc == Q38B_OK) rc = check_operand(X, X_ld, X_scales, K, B);
    if (rc != Q38B_OK) return rc;
    if ((uintptr_t)Y % kind_size(y_kind)) return Q38B_ERR_ALIGN;
    if ((B + 63) / 64 > 65535) return Q38B_ERR_UNSUPPORTED;
    DeviceGuard on(ctx);
    cudaStream_t st = (cudaStream_t)stream;
    const I8Args a = {(const int8_t*)W, (const int8_t*)X, W_scales, X_scales, Y, W_ld, X_ld, ldy, K, M, B, accumulate ? 1 : 0};
    return y_kind == Q38B_OUT_F32 ? gemm_as<float>(ctx, a, st) : y_kind == Q38B_OUT_F16 ? gemm_as<__half>(ctx, a, st) : gemm_as<__nv_bfloat16>(ctx, a, st);
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
    return q38b_gemm_i8(ctx, W, W_ld, W_scales, K, M, codes, padded(K), scales, B, Y, y_kind, ldy, accumulate, stream);
}

}  // extern "C"

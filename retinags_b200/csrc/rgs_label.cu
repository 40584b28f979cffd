// Label loss: softmax cross entropy of linear scores over a vocabulary, without the scores in memory.
//
//   s_nv = x_n . w_v + b_v,  lse_n = log sum_v exp s_nv,  loss_n = lse_n - s_n,y_n
//   G_nv = g_n (exp(s_nv - lse_n) - [v = y_n]),  dX = G W,  dW = G^T X,  db_v = sum_n G_nv
//
// First form: a warp owns a row (of X, or of W for the gradients of W and b) and walks the rows of the other matrix;
// the scores are recomputed in the backward pass from the kept lse.
#include <cuda_runtime.h>
#include <stdint.h>
#include "rgs_cuda_common.cuh"
#include "rgs_field_math.h"

#define LB_WARPS 8

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

__device__ __forceinline__ float row_dot(const void* a, int64_t ia, const void* b, int64_t ib, int c, int dtype, int lane) {
    float s = 0.f;
    for (int j = lane; j < c; j += 32) s = fmaf(rgs_load_as_float(a, ia + j, dtype), rgs_load_as_float(b, ib + j, dtype), s);
    return warp_sum(s);
}

__global__ void __launch_bounds__(LB_WARPS * 32) rgs_label_fwd_kernel(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                                                                      const void* labels, int label_bytes, int64_t n, int c, int64_t vocab,
                                                                      int dtype, int b_dtype, float* lse, float* losses) {
    const int lane = threadIdx.x & 31;
    for (int64_t i = (int64_t)blockIdx.x * LB_WARPS + (threadIdx.x >> 5); i < n; i += (int64_t)gridDim.x * LB_WARPS) {
        const int64_t y = rgs_label(labels, i, label_bytes, vocab);
        float m = -INFINITY, s = 0.f, at = 0.f;
        for (int64_t v = 0; v < vocab; ++v) {
            const float l = row_dot(x, i * ldx, w, v * ldw, c, dtype, lane) + (bias ? rgs_load_as_float(bias, v, b_dtype) : 0.f);
            if (v == y) at = l;
            if (l > m || l != l) { s *= expf(m - l); m = l; }
            if (!(l == -INFINITY && m == -INFINITY)) s += expf(l - m);
        }
        if (lane == 0) {
            const float z = logf(s);
            lse[i] = m;
            lse[n + i] = z;
            losses[i] = y < 0 ? 0.f : z + (m - at);
        }
    }
}

__global__ void __launch_bounds__(1024) rgs_label_sum_kernel(const float* losses, const void* labels, int label_bytes, int64_t n,
                                                             int64_t vocab, int mean, float* result, float* count) {
    __shared__ double part[32];
    __shared__ unsigned long long rows[32];
    double t = 0;
    unsigned long long k = 0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        t += losses[i];
        k += rgs_label(labels, i, label_bytes, vocab) >= 0;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) { t += __shfl_xor_sync(0xffffffffu, t, d); k += __shfl_xor_sync(0xffffffffu, k, d); }
    if ((threadIdx.x & 31) == 0) { part[threadIdx.x >> 5] = t; rows[threadIdx.x >> 5] = k; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 32; ++i) { t += part[i]; k += rows[i]; }
        *count = (float)k;
        if (result) *result = (float)(mean ? t / (double)(k > 0 ? k : 1) : t);
    }
}

// rows_of_w = 0: out = dX, walks W; 1: out = dW (and db), walks X
__global__ void __launch_bounds__(LB_WARPS * 32) rgs_label_bwd_kernel(const void* a, int64_t lda, const void* b, int64_t ldb, const void* bias,
                                                                      const void* labels, int label_bytes, int64_t na, int64_t nb, int c,
                                                                      int64_t vocab, int dtype, int b_dtype, const float* lse,
                                                                      const float* gout, int per_row, const float* count, int rows_of_w,
                                                                      void* out, void* db) {
    extern __shared__ float acc_all[];
    const int lane = threadIdx.x & 31;
    float* acc = acc_all + (size_t)(threadIdx.x >> 5) * c;
    const float scale = count ? 1.f / fmaxf(*count, 1.f) : 1.f;
    for (int64_t i = (int64_t)blockIdx.x * LB_WARPS + (threadIdx.x >> 5); i < na; i += (int64_t)gridDim.x * LB_WARPS) {
        for (int j = lane; j < c; j += 32) acc[j] = 0.f;
        float sb = 0.f;
        const int64_t ya = rows_of_w ? 0 : rgs_label(labels, i, label_bytes, vocab);
        for (int64_t k = 0; k < nb && ya >= 0; ++k) {
            const int64_t n = rows_of_w ? k : i, v = rows_of_w ? i : k;
            const int64_t y = rows_of_w ? rgs_label(labels, k, label_bytes, vocab) : ya;
            if (y < 0) continue;
            const float l = row_dot(a, i * lda, b, k * ldb, c, dtype, lane) + (bias ? rgs_load_as_float(bias, v, b_dtype) : 0.f);
            const float g = (expf((l - lse[n]) - lse[(rows_of_w ? nb : na) + n]) - (v == y ? 1.f : 0.f)) * gout[per_row ? n : 0] * scale;
            sb += g;
            for (int j = lane; j < c; j += 32) acc[j] = fmaf(g, rgs_load_as_float(b, k * ldb + j, dtype), acc[j]);
        }
        if (out)
            for (int j = lane; j < c; j += 32) rgs_store_float(out, i * c + j, dtype, acc[j]);
        if (db && lane == 0) rgs_store_float(db, i, b_dtype, sb);
    }
}

static inline unsigned label_grid(int64_t rows) {
    const int64_t want = (rows + LB_WARPS - 1) / LB_WARPS, most = RGS_SMS * 8;
    return (unsigned)(want < 1 ? 1 : (want > most ? most : want));
}

extern "C" {

int64_t rgs_cuda_label_scratch_bytes(int64_t n, int64_t, int64_t, int64_t, int64_t) { return n * 4 + 16; }

int rgs_cuda_label_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* labels, int64_t label_bytes,
                       int64_t n, int64_t c, int64_t vocab, int64_t dtype, int64_t b_dtype, int64_t mean, void* scratch, float* lse,
                       float* losses, float* result, float* count, void* stream) {
    float* row_loss = losses ? losses : static_cast<float*>(scratch);
    rgs_label_fwd_kernel<<<label_grid(n), LB_WARPS * 32, 0, (cudaStream_t)stream>>>(x, ldx, w, ldw, bias, labels, (int)label_bytes, n, (int)c,
                                                                                    vocab, (int)dtype, (int)b_dtype, lse, row_loss);
    rgs_label_sum_kernel<<<1, 1024, 0, (cudaStream_t)stream>>>(row_loss, labels, (int)label_bytes, n, vocab, (int)mean, result, count);
    return (int)cudaGetLastError();
}

int rgs_cuda_label_bwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* labels, int64_t label_bytes,
                       int64_t n, int64_t c, int64_t vocab, int64_t dtype, int64_t b_dtype, const float* lse, const float* gout,
                       int64_t per_row, const float* count, void* scratch, void* dx, void* dw, void* db, void* stream) {
    const size_t smem = (size_t)LB_WARPS * c * 4;
    if (dx)
        rgs_label_bwd_kernel<<<label_grid(n), LB_WARPS * 32, smem, (cudaStream_t)stream>>>(
            x, ldx, w, ldw, bias, labels, (int)label_bytes, n, vocab, (int)c, vocab, (int)dtype, (int)b_dtype, lse, gout, (int)per_row, count,
            0, dx, nullptr);
    if (dw || db)
        rgs_label_bwd_kernel<<<label_grid(vocab), LB_WARPS * 32, smem, (cudaStream_t)stream>>>(
            w, ldw, x, ldx, bias, labels, (int)label_bytes, vocab, n, (int)c, vocab, (int)dtype, (int)b_dtype, lse, gout, (int)per_row, count,
            1, dw, db);
    return (int)cudaGetLastError();
}

}  // extern "C"

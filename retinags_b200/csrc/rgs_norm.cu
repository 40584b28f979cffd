// Layer norm over the channels of feature rows (forward, backward, reduction of the weight's gradient) and the 8-bit
// form in which its input can wait for the backward pass.
//
//   xhat = (x - mean) rstd,  y = xhat w + b;   a = dy w,  dx = rstd (a - mean(a) - xhat mean(a xhat)),
//   dw = sum_n dy xhat,  db = sum_n dy
// With codes in place of x the backward pass is that of the norm at the values the codes stand for.
// First form: a warp per row, elements re-read for every sum.
#include <cuda_runtime.h>
#include <stdint.h>
#include "rgs_cuda_common.cuh"
#include "rgs_field_math.h"

#define NR_WARPS 8

struct NormArgs {
    const void* x; int dtype; int64_t ld; int planes;
    const int8_t* codes; const uint8_t* expo;
    int64_t n, c;
};

__device__ __forceinline__ float norm_warp_sum(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

__device__ __forceinline__ float norm_value(const NormArgs& a, int64_t i, int64_t j) {
    if (!a.codes) return rgs_load_as_float(a.x, a.planes ? j * a.ld + i : i * a.ld + j, a.dtype);
    const int64_t blocks = (a.c + RGS_PACK_BLOCK - 1) / RGS_PACK_BLOCK, b = j / RGS_PACK_BLOCK;
    return (float)a.codes[a.planes ? j * a.n + i : i * a.c + j] * rgs_pack_step(a.expo[a.planes ? b * a.n + i : i * blocks + b]);
}

__device__ __forceinline__ void norm_stats(const NormArgs& a, int64_t i, float eps, int lane, float& mu, float& rstd) {
    float s = 0.f;
    for (int64_t j = lane; j < a.c; j += 32) s += norm_value(a, i, j);
    mu = norm_warp_sum(s) / (float)a.c;
    s = 0.f;
    for (int64_t j = lane; j < a.c; j += 32) { const float d = norm_value(a, i, j) - mu; s = fmaf(d, d, s); }
    rstd = 1.0f / sqrtf(norm_warp_sum(s) / (float)a.c + eps);
}

__global__ void __launch_bounds__(NR_WARPS * 32) rgs_norm_fwd_kernel(NormArgs a, const void* w, const void* b, int p_dtype, float eps, void* y,
                                                                     int y_dtype) {
    const int lane = threadIdx.x & 31;
    for (int64_t i = (int64_t)blockIdx.x * NR_WARPS + (threadIdx.x >> 5); i < a.n; i += (int64_t)gridDim.x * NR_WARPS) {
        float mu, rstd;
        norm_stats(a, i, eps, lane, mu, rstd);
        for (int64_t j = lane; j < a.c; j += 32)
            rgs_store_float(y, i * a.c + j, y_dtype,
                            fmaf((norm_value(a, i, j) - mu) * rstd, w ? rgs_load_as_float(w, j, p_dtype) : 1.f,
                                 b ? rgs_load_as_float(b, j, p_dtype) : 0.f));
    }
}

__global__ void __launch_bounds__(NR_WARPS * 32) rgs_norm_bwd_kernel(NormArgs a, const void* dy, int dy_dtype, int64_t ldy, const void* w,
                                                                     int p_dtype, float eps, float2* stats, void* dx, int x_dtype) {
    const int lane = threadIdx.x & 31;
    for (int64_t i = (int64_t)blockIdx.x * NR_WARPS + (threadIdx.x >> 5); i < a.n; i += (int64_t)gridDim.x * NR_WARPS) {
        float mu, rstd, sa = 0.f, sax = 0.f;
        norm_stats(a, i, eps, lane, mu, rstd);
        if (lane == 0) stats[i] = make_float2(mu, rstd);
        if (!dx) continue;
        for (int64_t j = lane; j < a.c; j += 32) {
            const float g = rgs_load_as_float(dy, i * ldy + j, dy_dtype) * (w ? rgs_load_as_float(w, j, p_dtype) : 1.f);
            sa += g;
            sax = fmaf(g, (norm_value(a, i, j) - mu) * rstd, sax);
        }
        sa = norm_warp_sum(sa) / (float)a.c;
        sax = norm_warp_sum(sax) / (float)a.c;
        for (int64_t j = lane; j < a.c; j += 32) {
            const float g = rgs_load_as_float(dy, i * ldy + j, dy_dtype) * (w ? rgs_load_as_float(w, j, p_dtype) : 1.f);
            rgs_store_float(dx, a.planes ? j * a.n + i : i * a.c + j, x_dtype, rstd * (g - sa - (norm_value(a, i, j) - mu) * rstd * sax));
        }
    }
}

__global__ void __launch_bounds__(256) rgs_norm_dw_kernel(NormArgs a, const void* dy, int dy_dtype, int64_t ldy, const float2* stats,
                                                          int p_dtype, void* dw, void* db) {
    __shared__ double sw[256], sb[256];
    const int64_t j = blockIdx.x;
    double tw = 0, tb = 0;
    for (int64_t i = threadIdx.x; i < a.n; i += 256) {
        const float g = rgs_load_as_float(dy, i * ldy + j, dy_dtype);
        const float2 s = stats[i];
        tw += (double)(g * (norm_value(a, i, j) - s.x) * s.y);
        tb += (double)g;
    }
    sw[threadIdx.x] = tw;
    sb[threadIdx.x] = tb;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < 256; ++k) { tw += sw[k]; tb += sb[k]; }
        if (dw) rgs_store_float(dw, j, p_dtype, (float)tw);
        if (db) rgs_store_float(db, j, p_dtype, (float)tb);
    }
}

__global__ void __launch_bounds__(256) rgs_pack8_kernel(NormArgs a, int8_t* codes, uint8_t* expo) {
    const int64_t blocks = (a.c + RGS_PACK_BLOCK - 1) / RGS_PACK_BLOCK, total = a.n * blocks;
    const int lane = threadIdx.x & 31;
    for (int64_t t = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5; t < total; t += (int64_t)gridDim.x * 8) {
        const int64_t i = t / blocks, b = t % blocks, j = b * RGS_PACK_BLOCK + lane;
        const float v = j < a.c ? norm_value(a, i, j) : 0.f;
        const uint32_t top = __reduce_max_sync(0xffffffffu, rgs_f2u(v) & 0x7fffffffu);
        const uint32_t e = rgs_pack_exponent(rgs_u2f(top));
        if (lane == 0) expo[a.planes ? b * a.n + i : t] = (uint8_t)e;
        if (j < a.c) codes[a.planes ? j * a.n + i : i * a.c + j] = (int8_t)(e == RGS_PACK_NAN ? 0 : rgs_pack_code(v, rgs_pack_inverse(e)));
    }
}

__global__ void __launch_bounds__(256) rgs_unpack8_kernel(NormArgs a, void* out, int dtype) {
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < a.n * a.c; t += (int64_t)gridDim.x * 256) {
        const int64_t i = a.planes ? t % a.n : t / a.c, j = a.planes ? t / a.n : t % a.c;
        rgs_store_float(out, t, dtype, norm_value(a, i, j));
    }
}

static inline unsigned norm_grid(int64_t n, int per_block) {
    const int64_t want = (n + per_block - 1) / per_block, most = RGS_SMS * 16;
    return (unsigned)(want < 1 ? 1 : (want > most ? most : want));
}

extern "C" {

int64_t rgs_cuda_norm_scratch_bytes(int64_t n, int64_t) { return n * 8 + 16; }

int rgs_cuda_pack8(const void* x, int64_t dtype, int64_t ld, int64_t planes, int64_t n, int64_t c, int8_t* codes, uint8_t* expo, void* stream) {
    const NormArgs a{x, (int)dtype, ld, (int)planes, nullptr, nullptr, n, c};
    rgs_pack8_kernel<<<norm_grid(n * ((c + 31) / 32), 8), 256, 0, (cudaStream_t)stream>>>(a, codes, expo);
    return (int)cudaGetLastError();
}

int rgs_cuda_unpack8(const int8_t* codes, const uint8_t* expo, int64_t planes, int64_t n, int64_t c, void* out, int64_t dtype, void* stream) {
    const NormArgs a{nullptr, 0, 0, (int)planes, codes, expo, n, c};
    rgs_unpack8_kernel<<<norm_grid(n * c, 256), 256, 0, (cudaStream_t)stream>>>(a, out, (int)dtype);
    return (int)cudaGetLastError();
}

int rgs_cuda_norm_fwd(const void* x, int64_t dtype, int64_t ld, int64_t planes, const void* w, const void* b, int64_t p_dtype, int64_t n,
                      int64_t c, double eps, void* y, int64_t y_dtype, int8_t* codes, uint8_t* expo, void* stream) {
    const NormArgs a{x, (int)dtype, ld, (int)planes, nullptr, nullptr, n, c};
    rgs_norm_fwd_kernel<<<norm_grid(n, NR_WARPS), NR_WARPS * 32, 0, (cudaStream_t)stream>>>(a, w, b, (int)p_dtype, (float)eps, y, (int)y_dtype);
    RGS_CUDA_CHECK(cudaGetLastError());
    return codes ? rgs_cuda_pack8(x, dtype, ld, planes, n, c, codes, expo, stream) : 0;
}

int rgs_cuda_norm_bwd(const void* x, int64_t dtype, int64_t ld, int64_t planes, const int8_t* codes, const uint8_t* expo, const void* dy,
                      int64_t dy_dtype, int64_t ldy, const void* w, int64_t p_dtype, int64_t n, int64_t c, double eps, void* scratch,
                      void* dx, void* dw, void* db, void* stream) {
    const NormArgs a{x, (int)dtype, ld, (int)planes, codes, expo, n, c};
    float2* stats = static_cast<float2*>(scratch);
    rgs_norm_bwd_kernel<<<norm_grid(n, NR_WARPS), NR_WARPS * 32, 0, (cudaStream_t)stream>>>(a, dy, (int)dy_dtype, ldy, w, (int)p_dtype,
                                                                                            (float)eps, stats, dx, (int)dtype);
    if (dw || db)
        rgs_norm_dw_kernel<<<(unsigned)c, 256, 0, (cudaStream_t)stream>>>(a, dy, (int)dy_dtype, ldy, stats, (int)p_dtype, dw, db);
    return (int)cudaGetLastError();
}

}  // extern "C"

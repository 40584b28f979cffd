// Layer norm over the channels of feature rows (forward, backward, reduction of the weight's gradient) and the 8-bit
// form in which its input can wait for the backward pass.
//
//   xhat = (x - mean) rstd,  y = xhat w + b;   a = dy w,  dx = rstd (a - mean(a) - xhat mean(a xhat)),
//   dw = sum_n dy xhat,  db = sum_n dy
// With codes in place of x the backward pass is that of the norm at the values the codes stand for.
//
// All of it is bound by memory, so every tensor is read and written once: a group of 1 to 32 lanes holds a row in registers,
// the two sums of each pass are shuffles, and in the backward pass the mean and rstd are computed anew from the row (four
// shuffles) instead of being kept.  Lanes keep the sums of their own channels for dw and db over all the rows they meet;
// blocks write them once and a second kernel adds the blocks in order, so results do not depend on timing.
// Rows of 4 n channels on aligned boundaries are read in vectors of four, others element by element.  Channel planes (the
// renderer's images) pass through shared memory 32 pixels at a time.  Beyond 1024 channels a warp re-reads its row.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <atomic>
#include "rgs_cuda_common.cuh"
#include "rgs_field_math.h"

#define NT 256            // threads of a block
#define NR_MAX 1024       // channels that a group holds in registers
#define PT 32             // pixels of a tile of planes

enum { SRC_F32 = 0, SRC_BF16 = 1, SRC_CODES = 2 };

struct NormArgs {
    const void* x; int src, planes; int64_t ld;
    const int8_t* codes; const uint8_t* expo;      // kept input (backward)
    const void* w; const void* b; int p_dtype;
    int64_t n; int c, blocks;                      // rows, channels, 32-channel blocks of a row
    float eps, inv_c;
    void* y; int y_dtype;
    int8_t* codes_out; uint8_t* expo_out;          // forward with an 8-bit copy
    const void* dy; int dy_dtype; int64_t ldy;
    void* dx; int dx_dtype;
    float* part;                                   // (blocks of the grid, 2, c)
};

// The switch on a type stands outside the loops over a row's vectors, so that all loads of a row are in flight together
// (inside, every load waited for the one before: 3 to 4 times slower on wide or odd rows).
template <int VEC, int DT>
__device__ __forceinline__ void load_vec(const void* p, int64_t i, float (&f)[VEC]) {
    if constexpr (VEC == 4 && DT == RGS_BF16) {
        const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
        f[0] = __uint_as_float(u.x << 16); f[1] = __uint_as_float(u.x & 0xffff0000u);
        f[2] = __uint_as_float(u.y << 16); f[3] = __uint_as_float(u.y & 0xffff0000u);
    } else if constexpr (VEC == 4) {
        const float4 u = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
        f[0] = u.x; f[1] = u.y; f[2] = u.z; f[3] = u.w;
    } else if constexpr (DT == RGS_BF16) {
        f[0] = __uint_as_float((uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
    } else {
        f[0] = static_cast<const float*>(p)[i];
    }
}
// vectors k of a lane, (k lanes + l) VEC, of the row that starts at element i; zero behind the last channel
template <int VEC, int NV, int LANES, int DT>
__device__ __forceinline__ void load_all(const void* p, int64_t i, int l, int c, float (&x)[NV][VEC]) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int at = (k * LANES + l) * VEC;
        if (at < c) load_vec<VEC, DT>(p, i + at, x[k]);
        else
#pragma unroll
            for (int q = 0; q < VEC; ++q) x[k][q] = 0.f;
    }
}
template <int VEC, int NV, int LANES>
__device__ __forceinline__ void load_typed(const void* p, int dtype, int64_t i, int l, int c, float (&x)[NV][VEC]) {
    if (dtype == RGS_BF16) load_all<VEC, NV, LANES, RGS_BF16>(p, i, l, c, x);
    else load_all<VEC, NV, LANES, RGS_F32>(p, i, l, c, x);
}
__device__ __forceinline__ uint32_t pair_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <int VEC>
__device__ __forceinline__ void store_vec(void* p, int64_t i, int dtype, const float (&f)[VEC]) {
    if constexpr (VEC == 4) {
        if (dtype == RGS_BF16) *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = make_uint2(pair_bf16(f[0], f[1]), pair_bf16(f[2], f[3]));
        else *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
        if (dtype == RGS_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(f[0]);
        else static_cast<float*>(p)[i] = f[0];
    }
}
// codes of four channels (one word) or of one, from values scaled by the inverse step of their block
template <int VEC>
__device__ __forceinline__ void store_codes(int8_t* p, int64_t i, const float (&f)[VEC], uint32_t e) {
    const float inv = rgs_pack_inverse(e);
    if constexpr (VEC == 4) {
        uint32_t u = 0;
        if (e != RGS_PACK_NAN)
#pragma unroll
            for (int k = 0; k < 4; ++k) u |= (uint32_t)(rgs_pack_code(f[k], inv) & 0xff) << (8 * k);
        *reinterpret_cast<uint32_t*>(p + i) = u;
    } else {
        p[i] = (int8_t)(e == RGS_PACK_NAN ? 0 : rgs_pack_code(f[0], inv));
    }
}
template <int VEC>
__device__ __forceinline__ void load_codes(const int8_t* p, int64_t i, float step, float (&f)[VEC]) {
    if constexpr (VEC == 4) {
        const uint32_t u = *reinterpret_cast<const uint32_t*>(p + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = (float)(int8_t)(u >> (8 * k)) * step;
    } else {
        f[0] = (float)p[i] * step;
    }
}

// sum, or maximum, over the LANES lanes (a power of two) that share a row
template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int d = LANES >> 1; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
template <int LANES>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
    for (int d = LANES >> 1; d > 0; d >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}

// mean and 1 / sqrt(var + eps) of a row; vector k of a lane starts at channel (k lanes + lane) VEC
template <int VEC, int NV, int LANES>
__device__ __forceinline__ void row_stats(const float (&x)[NV][VEC], int l, int c, float inv_c, float eps, float& mu, float& rstd) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int q = 0; q < VEC; ++q) s += x[k][q];   // zero behind the last channel
    mu = group_sum<LANES>(s) * inv_c;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if ((k * LANES + l) * VEC < c)
#pragma unroll
            for (int q = 0; q < VEC; ++q) s = fmaf(x[k][q] - mu, x[k][q] - mu, s);
    rstd = 1.0f / sqrtf(group_sum<LANES>(s) * inv_c + eps);
}

// the part of the backward pass that rows and planes share: a row's x, dy -> dx (over x), sums of dw and db
template <int VEC, int NV, int LANES>
__device__ __forceinline__ void row_bwd(float (&x)[NV][VEC], float (&g)[NV][VEC], const float (&w)[NV][VEC], float (&sw)[NV][VEC], float (&sb)[NV][VEC],
                                        int l, int c, float inv_c, float eps) {
    float mu, rstd, sa = 0.f, sax = 0.f;
    row_stats<VEC, NV, LANES>(x, l, c, inv_c, eps, mu, rstd);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
            const bool in = (k * LANES + l) * VEC < c;
            x[k][q] = in ? (x[k][q] - mu) * rstd : 0.f;
            sw[k][q] = fmaf(g[k][q], x[k][q], sw[k][q]);
            sb[k][q] += g[k][q];
            g[k][q] *= w[k][q];
            sa += g[k][q];
            sax = fmaf(g[k][q], x[k][q], sax);
        }
    sa = group_sum<LANES>(sa) * inv_c;
    sax = group_sum<LANES>(sax) * inv_c;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int q = 0; q < VEC; ++q) x[k][q] = rstd * (g[k][q] - sa - x[k][q] * sax);
}

template <int VEC, int NV, int LANES>
__device__ __forceinline__ void load_params(const NormArgs& a, int l, const void* p, float none, float (&w)[NV][VEC]) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
            const int c = (k * LANES + l) * VEC + q;
            w[k][q] = none;
            if (p && c < a.c) w[k][q] = a.p_dtype == RGS_BF16 ? rgs_bf16_value(static_cast<const uint16_t*>(p)[c]) : static_cast<const float*>(p)[c];
        }
}

// sums of a block's groups, in the order of the groups, to the block's row of the partial sums
template <int VEC, int NV, int LANES>
__device__ __forceinline__ void block_sums(const NormArgs& a, int l, const float (&sw)[NV][VEC], const float (&sb)[NV][VEC], float* sh) {
    // sh: (groups of the block, channels) of one of the two sums at a time, 64 channels a turn
    const int group = threadIdx.x / LANES, groups = NT / LANES;
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (k * LANES * VEC >= a.c) break;
            __syncthreads();
#pragma unroll
            for (int q = 0; q < VEC; ++q) sh[group * (LANES * VEC) + l * VEC + q] = which ? sb[k][q] : sw[k][q];
            __syncthreads();
            for (int j = threadIdx.x; j < LANES * VEC; j += NT) {
                float t = 0.f;
                for (int r = 0; r < groups; ++r) t += sh[r * (LANES * VEC) + j];
                const int c = k * LANES * VEC + j;
                if (c < a.c) a.part[((int64_t)blockIdx.x * 2 + which) * a.c + c] = t;
            }
        }
}

// ---------------------------------------------------------------------------------------------------------------------
// rows
// ---------------------------------------------------------------------------------------------------------------------
template <int VEC, int NV, int LANES>
__device__ __forceinline__ void load_row(const NormArgs& a, int64_t i, int l, float (&x)[NV][VEC]) {
    if (a.src == SRC_CODES) {
        float step[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int at = (k * LANES + l) * VEC;
            step[k] = at < a.c ? rgs_pack_step(a.expo[i * a.blocks + at / RGS_PACK_BLOCK]) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int at = (k * LANES + l) * VEC;
            if (at < a.c) load_codes<VEC>(a.codes, i * a.c + at, step[k], x[k]);
            else
#pragma unroll
                for (int q = 0; q < VEC; ++q) x[k][q] = 0.f;
        }
    } else {
        load_typed<VEC, NV, LANES>(a.x, a.src, i * a.ld, l, a.c, x);
    }
}

template <int VEC, int NV, int LANES, int R, bool PACK>
__global__ void __launch_bounds__(NT) rgs_norm_rows_fwd_kernel(const __grid_constant__ NormArgs a) {
    const int l = threadIdx.x % LANES, groups = NT / LANES;
    const int64_t stride = (int64_t)gridDim.x * groups;
    float w[NV][VEC], b[NV][VEC];
    load_params<VEC, NV, LANES>(a, l, a.w, 1.f, w);
    load_params<VEC, NV, LANES>(a, l, a.b, 0.f, b);
    // all lanes of a warp take the same number of turns: shuffles need them
    for (int64_t i0 = (int64_t)blockIdx.x * groups; i0 < a.n; i0 += R * stride) {
        const int64_t i = i0 + threadIdx.x / LANES;
        float x[R][NV][VEC];
#pragma unroll
        for (int r = 0; r < R; ++r)
            load_row<VEC, NV, LANES>(a, min(i + r * stride, a.n - 1), l, x[r]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = i + r * stride;
            float mu, rstd;
            row_stats<VEC, NV, LANES>(x[r], l, a.c, a.inv_c, a.eps, mu, rstd);
            uint32_t top[NV];
            if (PACK) {
                // a block of 32 channels is 32 / VEC vectors: KB of every lane of the row, or one of some of its lanes
                constexpr int LB = RGS_PACK_BLOCK / VEC, KB = LANES < LB ? LB / LANES : 1;
#pragma unroll
                for (int k = 0; k < NV; k += KB) {
                    uint32_t m = 0;
#pragma unroll
                    for (int e = k; e < k + KB && e < NV; ++e)
#pragma unroll
                        for (int q = 0; q < VEC; ++q) m = max(m, __float_as_uint(x[r][e][q]) & 0x7fffffffu);
                    m = rgs_pack_exponent(__uint_as_float(group_max<(LANES < LB ? LANES : LB)>(m)));
#pragma unroll
                    for (int e = k; e < k + KB && e < NV; ++e) top[e] = m;
                }
            }
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int c = (k * LANES + l) * VEC;
                if (PACK && row < a.n && c < a.c) {
                    if (c % RGS_PACK_BLOCK == 0) a.expo_out[row * a.blocks + c / RGS_PACK_BLOCK] = (uint8_t)top[k];
                    store_codes<VEC>(a.codes_out, row * a.c + c, x[r][k], top[k]);
                }
                if (a.y && row < a.n && c < a.c) {
                    float f[VEC];
#pragma unroll
                    for (int q = 0; q < VEC; ++q) f[q] = fmaf((x[r][k][q] - mu) * rstd, w[k][q], b[k][q]);
                    store_vec<VEC>(a.y, row * a.c + c, a.y_dtype, f);
                }
            }
        }
    }
}

template <int VEC, int NV, int LANES, int R>
__global__ void __launch_bounds__(NT) rgs_norm_rows_bwd_kernel(const __grid_constant__ NormArgs a) {
    __shared__ float sh[NT * VEC];
    const int l = threadIdx.x % LANES, groups = NT / LANES;
    const int64_t stride = (int64_t)gridDim.x * groups;
    float w[NV][VEC], sw[NV][VEC], sb[NV][VEC];
    load_params<VEC, NV, LANES>(a, l, a.w, 1.f, w);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int q = 0; q < VEC; ++q) sw[k][q] = sb[k][q] = 0.f;
    for (int64_t i0 = (int64_t)blockIdx.x * groups; i0 < a.n; i0 += R * stride) {
        const int64_t i = i0 + threadIdx.x / LANES;
        float x[R][NV][VEC], g[R][NV][VEC];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = min(i + r * stride, a.n - 1);
            load_row<VEC, NV, LANES>(a, row, l, x[r]);
            load_typed<VEC, NV, LANES>(a.dy, a.dy_dtype, row * a.ldy, l, i + r * stride < a.n ? a.c : 0, g[r]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = i + r * stride;
            if (row >= a.n) {  // the last row again, in place of one behind the end: nothing of it counts, whatever it holds
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int q = 0; q < VEC; ++q) x[r][k][q] = 0.f;
            }
            row_bwd<VEC, NV, LANES>(x[r], g[r], w, sw, sb, l, a.c, a.inv_c, a.eps > 0.f ? a.eps : (row >= a.n ? 1.f : 0.f));
            if (a.dx && row < a.n)
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const int c = (k * LANES + l) * VEC;
                    if (c < a.c) store_vec<VEC>(a.dx, row * a.c + c, a.dx_dtype, x[r][k]);
                }
        }
    }
    if (a.part) block_sums<VEC, NV, LANES>(a, l, sw, sb, sh);
}

// ---------------------------------------------------------------------------------------------------------------------
// channel planes: 32 pixels at a time through shared memory, (channel, pixel) with rows of 33
// ---------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float plane_value(const NormArgs& a, int64_t i, int c) {
    if (a.src == SRC_CODES)
        return (float)a.codes[(int64_t)c * a.n + i] * rgs_pack_step(a.expo[(int64_t)(c / RGS_PACK_BLOCK) * a.n + i]);
    return rgs_load_as_float(a.x, (int64_t)c * a.ld + i, a.src);
}
// channels c0, c0 + 8, ... of pixel i to shared memory
template <int SRC>
__device__ __forceinline__ void load_plane(const NormArgs& a, int64_t i, int c0, int p, float* sm) {
#pragma unroll 8
    for (int c = c0; c < a.c; c += NT / 32) {
        float f[1];
        if constexpr (SRC == SRC_CODES) load_codes<1>(a.codes, (int64_t)c * a.n + i, rgs_pack_step(a.expo[(int64_t)(c / RGS_PACK_BLOCK) * a.n + i]), f);
        else load_vec<1, SRC>(a.x, (int64_t)c * a.ld + i, f);
        sm[c * 33 + p] = f[0];
    }
}

template <int NV, int LANES, bool BWD>
__global__ void __launch_bounds__(NT) rgs_norm_planes_kernel(const __grid_constant__ NormArgs a) {
    extern __shared__ float sm[];                // (c, 33); behind it room for the sums of a block
    constexpr int WR = 32 / LANES;               // rows of a warp, LANES apart: their words lie in different banks
    const int l = threadIdx.x % LANES;
    const int p = threadIdx.x & 31, c0 = threadIdx.x >> 5;
    float w[NV][1], b[NV][1], sw[NV][1], sb[NV][1];
    load_params<1, NV, LANES>(a, l, a.w, 1.f, w);
    if (!BWD) load_params<1, NV, LANES>(a, l, a.b, 0.f, b);
#pragma unroll
    for (int k = 0; k < NV; ++k) sw[k][0] = sb[k][0] = 0.f;
    const int64_t tiles = (a.n + PT - 1) / PT;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int64_t base = t * PT;
        __syncthreads();
        if (base + p < a.n) {
            if (a.src == SRC_CODES) load_plane<SRC_CODES>(a, base + p, c0, p, sm);
            else if (a.src == SRC_BF16) load_plane<SRC_BF16>(a, base + p, c0, p, sm);
            else load_plane<SRC_F32>(a, base + p, c0, p, sm);
        } else {
            for (int c = c0; c < a.c; c += NT / 32) sm[c * 33 + p] = 0.f;
        }
        __syncthreads();
        if (!BWD && a.codes_out && base + p < a.n) {
            for (int k = c0; k < a.blocks; k += NT / 32) {
                const int end = min(a.c, (k + 1) * RGS_PACK_BLOCK);
                uint32_t top = 0;
                for (int c = k * RGS_PACK_BLOCK; c < end; ++c) top = max(top, __float_as_uint(sm[c * 33 + p]) & 0x7fffffffu);
                const uint32_t e = rgs_pack_exponent(__uint_as_float(top));
                a.expo_out[(int64_t)k * a.n + base + p] = (uint8_t)e;
                for (int c = k * RGS_PACK_BLOCK; c < end; ++c) {
                    const float f[1] = {sm[c * 33 + p]};
                    store_codes<1>(a.codes_out, (int64_t)c * a.n + base + p, f, e);
                }
            }
        }
        for (int r0 = threadIdx.x >> 5; r0 < PT / WR; r0 += NT / 32) {
            const int r = r0 + (threadIdx.x & 31) / LANES * (PT / WR);
            const int64_t row = base + r;
            float x[NV][1];
#pragma unroll
            for (int k = 0; k < NV; ++k) x[k][0] = k * LANES + l < a.c ? sm[(k * LANES + l) * 33 + r] : 0.f;
            if (!BWD) {
                float mu, rstd;
                row_stats<1, NV, LANES>(x, l, a.c, a.inv_c, a.eps, mu, rstd);
                if (row < a.n)
#pragma unroll
                    for (int k = 0; k < NV; ++k) {
                        const int c = k * LANES + l;
                        const float f[1] = {fmaf((x[k][0] - mu) * rstd, w[k][0], b[k][0])};
                        if (c < a.c) store_vec<1>(a.y, row * a.c + c, a.y_dtype, f);
                    }
            } else {
                float g[NV][1];
                load_typed<1, NV, LANES>(a.dy, a.dy_dtype, row * a.ldy, l, row < a.n ? a.c : 0, g);
                row_bwd<1, NV, LANES>(x, g, w, sw, sb, l, a.c, a.inv_c, row < a.n ? a.eps : 1.f);
#pragma unroll
                for (int k = 0; k < NV; ++k)
                    if (k * LANES + l < a.c) sm[(k * LANES + l) * 33 + r] = x[k][0];
            }
        }
        if (BWD && a.dx) {
            __syncthreads();
            if (base + p < a.n)
                for (int c = c0; c < a.c; c += NT / 32) {
                    const float f[1] = {sm[c * 33 + p]};
                    store_vec<1>(a.dx, (int64_t)c * a.n + base + p, a.dx_dtype, f);
                }
        }
    }
    if (BWD && a.part) {
        __syncthreads();
        block_sums<1, NV, LANES>(a, l, sw, sb, sm);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// more channels than a group holds: a warp re-reads its row; a block of threads per 32 channels sums dw and db
// ---------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float wide_value(const NormArgs& a, int64_t i, int c) {
    if (a.planes) return plane_value(a, i, c);
    if (a.src == SRC_CODES) return (float)a.codes[i * a.c + c] * rgs_pack_step(a.expo[i * a.blocks + c / RGS_PACK_BLOCK]);
    return rgs_load_as_float(a.x, i * a.ld + c, a.src);
}

__global__ void __launch_bounds__(NT) rgs_norm_wide_kernel(const __grid_constant__ NormArgs a, int backward, float2* stats) {
    const int lane = threadIdx.x & 31;
    for (int64_t i = (int64_t)blockIdx.x * (NT / 32) + (threadIdx.x >> 5); i < a.n; i += (int64_t)gridDim.x * (NT / 32)) {
        float s = 0.f;
        for (int j = lane; j < a.c; j += 32) s += wide_value(a, i, j);
        const float mu = group_sum<32>(s) * a.inv_c;
        s = 0.f;
        for (int j = lane; j < a.c; j += 32) { const float d = wide_value(a, i, j) - mu; s = fmaf(d, d, s); }
        const float rstd = 1.0f / sqrtf(group_sum<32>(s) * a.inv_c + a.eps);
        if (!backward) {
            for (int j = lane; j < a.c; j += 32)
                rgs_store_float(a.y, i * a.c + j, a.y_dtype,
                                fmaf((wide_value(a, i, j) - mu) * rstd, a.w ? rgs_load_as_float(a.w, j, a.p_dtype) : 1.f,
                                     a.b ? rgs_load_as_float(a.b, j, a.p_dtype) : 0.f));
            continue;
        }
        if (lane == 0) stats[i] = make_float2(mu, rstd);
        if (!a.dx) continue;
        float sa = 0.f, sax = 0.f;
        for (int j = lane; j < a.c; j += 32) {
            const float g = rgs_load_as_float(a.dy, i * a.ldy + j, a.dy_dtype) * (a.w ? rgs_load_as_float(a.w, j, a.p_dtype) : 1.f);
            sa += g;
            sax = fmaf(g, (wide_value(a, i, j) - mu) * rstd, sax);
        }
        sa = group_sum<32>(sa) * a.inv_c;
        sax = group_sum<32>(sax) * a.inv_c;
        for (int j = lane; j < a.c; j += 32) {
            const float g = rgs_load_as_float(a.dy, i * a.ldy + j, a.dy_dtype) * (a.w ? rgs_load_as_float(a.w, j, a.p_dtype) : 1.f);
            rgs_store_float(a.dx, a.planes ? j * a.n + i : i * a.c + j, a.dx_dtype, rstd * (g - sa - (wide_value(a, i, j) - mu) * rstd * sax));
        }
    }
}

__global__ void __launch_bounds__(NT) rgs_norm_wide_sums_kernel(const __grid_constant__ NormArgs a, const float2* stats) {
    const int j = blockIdx.x * 32 + (threadIdx.x & 31), rows = gridDim.y * (NT / 32);
    float sw = 0.f, sb = 0.f;
    if (j < a.c)
        for (int64_t i = (int64_t)blockIdx.y * (NT / 32) + (threadIdx.x >> 5); i < a.n; i += rows) {
            const float g = rgs_load_as_float(a.dy, i * a.ldy + j, a.dy_dtype);
            const float2 s = stats[i];
            sw = fmaf(g, (wide_value(a, i, j) - s.x) * s.y, sw);
            sb += g;
        }
    __shared__ float sh[2][NT / 32][32];
    sh[0][threadIdx.x >> 5][threadIdx.x & 31] = sw;
    sh[1][threadIdx.x >> 5][threadIdx.x & 31] = sb;
    __syncthreads();
    if (threadIdx.x < 64) {
        const int which = threadIdx.x >> 5, c = blockIdx.x * 32 + (threadIdx.x & 31);
        float t = 0.f;
        for (int r = 0; r < NT / 32; ++r) t += sh[which][r][threadIdx.x & 31];
        if (c < a.c) a.part[((int64_t)blockIdx.y * 2 + which) * a.c + c] = t;
    }
}

// adds the blocks' sums in order: 32 channels to a block, 32 interleaved chains each
__global__ void __launch_bounds__(1024) rgs_norm_reduce_kernel(const float* __restrict__ part, int parts, int c, void* dw, void* db, int p_dtype) {
    __shared__ float sh[32][33];
    const int lane = threadIdx.x & 31, chain = threadIdx.x >> 5, j = blockIdx.x * 32 + lane, which = blockIdx.y;
    float t = 0.f;
    if (j < c)
#pragma unroll 4
        for (int k = chain; k < parts; k += 32) t += part[((int64_t)k * 2 + which) * c + j];
    sh[chain][lane] = t;
    __syncthreads();
    if (chain == 0 && j < c) {
        t = 0.f;
        for (int k = 0; k < 32; ++k) t += sh[k][lane];
        void* out = which ? db : dw;
        if (out) rgs_store_float(out, j, p_dtype, t);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// the 8-bit form by itself
// ---------------------------------------------------------------------------------------------------------------------
// Rows: 32 / VEC lanes to a 32-channel block, so that a warp reads and writes what lies together; four blocks in flight.
// `flat`: whole blocks that follow one another without a gap, no division.
template <int VEC, int DT>
__global__ void __launch_bounds__(NT) rgs_pack8_rows_kernel(const __grid_constant__ NormArgs a, int flat) {
    constexpr int LB = RGS_PACK_BLOCK / VEC, U = 4;
    const int l = threadIdx.x % LB;
    const int64_t total = a.n * a.blocks, per = NT / LB;
    for (int64_t t0 = (int64_t)blockIdx.x * (per * U); t0 < total; t0 += (int64_t)gridDim.x * (per * U)) {
        float x[U][VEC];
        int64_t row[U];
        int c[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t t = t0 + u * per + threadIdx.x / LB;
            if (flat) { row[u] = t; c[u] = l * VEC; }
            else {
                row[u] = total < ((int64_t)1 << 31) ? (int64_t)((uint32_t)t / (uint32_t)a.blocks) : t / a.blocks;
                c[u] = (int)(t - row[u] * a.blocks) * RGS_PACK_BLOCK + l * VEC;
            }
#pragma unroll
            for (int q = 0; q < VEC; ++q) x[u][q] = 0.f;
            if (t < total && (flat || c[u] < a.c)) load_vec<VEC, DT>(a.x, flat ? t * RGS_PACK_BLOCK + c[u] : row[u] * a.ld + c[u], x[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t t = t0 + u * per + threadIdx.x / LB;
            uint32_t top = 0;
#pragma unroll
            for (int q = 0; q < VEC; ++q) top = max(top, __float_as_uint(x[u][q]) & 0x7fffffffu);
            const uint32_t e = rgs_pack_exponent(__uint_as_float(group_max<LB>(top)));
            if (t >= total) continue;
            if (l == 0) a.expo_out[t] = (uint8_t)e;
            if (flat) store_codes<VEC>(a.codes_out, t * RGS_PACK_BLOCK + c[u], x[u], e);
            else if (c[u] < a.c) store_codes<VEC>(a.codes_out, row[u] * a.c + c[u], x[u], e);
        }
        __syncwarp();
    }
}

// planes: a thread per pixel and block
template <int DT>
__global__ void __launch_bounds__(NT) rgs_pack8_planes_kernel(const __grid_constant__ NormArgs a) {
    const int64_t tiles = (a.n + NT - 1) / NT;
    for (int64_t t = blockIdx.x; t < tiles * a.blocks; t += gridDim.x) {
        const int64_t k = t / tiles, i = (t - k * tiles) * NT + threadIdx.x;
        if (i >= a.n) continue;
        const int c = (int)k * RGS_PACK_BLOCK;
        float x[RGS_PACK_BLOCK];
        uint32_t top = 0;
#pragma unroll
        for (int q = 0; q < RGS_PACK_BLOCK; ++q) {
            float f[1] = {0.f};
            if (c + q < a.c) load_vec<1, DT>(a.x, (int64_t)(c + q) * a.ld + i, f);
            x[q] = f[0];
            top = max(top, __float_as_uint(x[q]) & 0x7fffffffu);
        }
        const uint32_t e = rgs_pack_exponent(__uint_as_float(top));
        a.expo_out[k * a.n + i] = (uint8_t)e;
#pragma unroll
        for (int q = 0; q < RGS_PACK_BLOCK; ++q)
            if (c + q < a.c) {
                const float f[1] = {x[q]};
                store_codes<1>(a.codes_out, (int64_t)(c + q) * a.n + i, f, e);
            }
    }
}

// VEC codes to a thread, four such in flight; rows (VEC divides a row) or planes (VEC divides a plane)
template <int VEC>
__global__ void __launch_bounds__(NT) rgs_unpack8_kernel(const __grid_constant__ NormArgs a, int flat, void* out, int dtype) {
    constexpr int U = 4;
    const int64_t total = a.n * a.c / VEC;
    const uint32_t per = (uint32_t)((a.planes ? a.n : a.c) / VEC);  // (below 2^31: rows and channels are)
    for (int64_t t0 = (int64_t)blockIdx.x * (NT * U) + threadIdx.x; t0 < total; t0 += (int64_t)gridDim.x * (NT * U)) {
        float f[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t t = t0 + u * NT;
            if (t >= total) break;
            if (a.planes) {
                const int64_t c = total < ((int64_t)1 << 31) ? (int64_t)((uint32_t)t / per) : t / per, i = (t - c * per) * VEC;
                float e[VEC];
#pragma unroll
                for (int q = 0; q < VEC; ++q) e[q] = rgs_pack_step(a.expo[c / RGS_PACK_BLOCK * a.n + i + q]);
                load_codes<VEC>(a.codes, t * VEC, 1.f, f[u]);
#pragma unroll
                for (int q = 0; q < VEC; ++q) f[u][q] *= e[q];
            } else {
                int64_t k;
                if (flat) k = t / (RGS_PACK_BLOCK / VEC);
                else {
                    const int64_t i = total < ((int64_t)1 << 31) ? (int64_t)((uint32_t)t / per) : t / per;
                    k = i * a.blocks + (t - i * per) * VEC / RGS_PACK_BLOCK;
                }
                load_codes<VEC>(a.codes, t * VEC, rgs_pack_step(a.expo[k]), f[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (t0 + u * NT < total) store_vec<VEC>(out, (t0 + u * NT) * VEC, dtype, f[u]);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------------
static inline int64_t norm_grid(int64_t want, int64_t per_sm) {
    const int64_t most = RGS_SMS * per_sm;
    return want < 1 ? 1 : (want > most ? most : want);
}
static inline bool aligned_to(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes) == 0; }
static inline int64_t four(int dtype) { return dtype == RGS_BF16 ? 8 : 16; }  // bytes of four elements

#define NORM_PARTS 1184   // most blocks that leave partial sums

// blocks of a kernel that fit on the device together: persistent grids, so that a block reads the parameters once
template <typename K>
static int64_t norm_resident(K kernel, int smem) {
    int per_sm = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, NT, (size_t)smem) != cudaSuccess || per_sm < 1) per_sm = 1;
    return RGS_SMS * per_sm;
}
static inline int64_t at_most(int64_t want, int64_t most) { return want < 1 ? 1 : (want > most ? most : want); }

template <int VEC, int NV, int LANES, int R>
static int norm_rows_launch(const NormArgs& a, bool backward, cudaStream_t st) {
    const int64_t want = (a.n + (NT / LANES) * R - 1) / ((NT / LANES) * R);
    if (backward) {
        static std::atomic<int64_t> most{0};
        if (!most) most = norm_resident(rgs_norm_rows_bwd_kernel<VEC, NV, LANES, R>, 0);
        const int64_t grid = at_most(at_most(want, most), NORM_PARTS);
        rgs_norm_rows_bwd_kernel<VEC, NV, LANES, R><<<(unsigned)grid, NT, 0, st>>>(a);
        return (int)grid;
    }
    static std::atomic<int64_t> most[2];
    const int pack = a.codes_out != nullptr;
    if (!most[pack]) most[pack] = pack ? norm_resident(rgs_norm_rows_fwd_kernel<VEC, NV, LANES, R, true>, 0) : norm_resident(rgs_norm_rows_fwd_kernel<VEC, NV, LANES, R, false>, 0);
    const unsigned grid = (unsigned)at_most(want, most[pack]);
    if (pack) rgs_norm_rows_fwd_kernel<VEC, NV, LANES, R, true><<<grid, NT, 0, st>>>(a);
    else rgs_norm_rows_fwd_kernel<VEC, NV, LANES, R, false><<<grid, NT, 0, st>>>(a);
    return 0;
}

// Few lanes to a row and several vectors to a lane: the shuffles of a row's sums are what narrow rows cost most (one lane
// to a vector: 1.4 TB/s at 33 channels, 3.4 at 64 backward).
static int norm_rows(const NormArgs& a, bool vec, bool backward, cudaStream_t st) {
    const int u = vec ? a.c / 4 : a.c;
    if (vec) {
        if (u <= 2) return norm_rows_launch<4, 2, 1, 2>(a, backward, st);
        if (u <= 4) return norm_rows_launch<4, 2, 2, 2>(a, backward, st);
        if (u <= 8) return norm_rows_launch<4, 2, 4, 2>(a, backward, st);
        if (u <= 16) return norm_rows_launch<4, 2, 8, 2>(a, backward, st);
        if (u <= 32) return norm_rows_launch<4, 2, 16, 2>(a, backward, st);
        if (u <= 64) return norm_rows_launch<4, 2, 32, 2>(a, backward, st);
        if (u <= 128) return norm_rows_launch<4, 4, 32, 1>(a, backward, st);
        return norm_rows_launch<4, 8, 32, 1>(a, backward, st);
    }
    if (u <= 4) return norm_rows_launch<1, 4, 1, 2>(a, backward, st);
    if (u <= 8) return norm_rows_launch<1, 4, 2, 2>(a, backward, st);
    if (u <= 16) return norm_rows_launch<1, 4, 4, 2>(a, backward, st);
    if (u <= 32) return norm_rows_launch<1, 4, 8, 2>(a, backward, st);
    if (u <= 64) return norm_rows_launch<1, 4, 16, 2>(a, backward, st);
    if (u <= 128) return norm_rows_launch<1, 4, 32, 2>(a, backward, st);
    if (u <= 256) return norm_rows_launch<1, 8, 32, 1>(a, backward, st);
    if (u <= 512) return norm_rows_launch<1, 16, 32, 1>(a, backward, st);
    if (u <= 640) return norm_rows_launch<1, 20, 32, 1>(a, backward, st);
    if (u <= 768) return norm_rows_launch<1, 24, 32, 1>(a, backward, st);
    if (u <= 896) return norm_rows_launch<1, 28, 32, 1>(a, backward, st);
    return norm_rows_launch<1, 32, 32, 1>(a, backward, st);
}

template <int NV, int LANES, bool BWD>
static int norm_planes_launch(const NormArgs& a, int* parts, cudaStream_t st) {
    const int smem = (a.c * 33 > NT ? a.c * 33 : NT) * 4;  // (block_sums takes NT floats of it)
    if (smem > 48 * 1024) RGS_CUDA_CHECK(cudaFuncSetAttribute(rgs_norm_planes_kernel<NV, LANES, BWD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    *parts = (int)at_most(at_most((a.n + PT - 1) / PT, norm_resident(rgs_norm_planes_kernel<NV, LANES, BWD>, smem)), NORM_PARTS);
    rgs_norm_planes_kernel<NV, LANES, BWD><<<(unsigned)*parts, NT, smem, st>>>(a);
    return (int)cudaGetLastError();
}

template <bool BWD>
static int norm_planes(const NormArgs& a, int* parts, cudaStream_t st) {
    if (a.c <= 8) return norm_planes_launch<8, 1, BWD>(a, parts, st);
    if (a.c <= 16) return norm_planes_launch<8, 2, BWD>(a, parts, st);
    if (a.c <= 32) return norm_planes_launch<8, 4, BWD>(a, parts, st);
    if (a.c <= 64) return norm_planes_launch<8, 8, BWD>(a, parts, st);
    if (a.c <= 128) return norm_planes_launch<8, 16, BWD>(a, parts, st);
    if (a.c <= 256) return norm_planes_launch<8, 32, BWD>(a, parts, st);
    if (a.c <= 512) return norm_planes_launch<16, 32, BWD>(a, parts, st);
    return norm_planes_launch<32, 32, BWD>(a, parts, st);
}

extern "C" {

int64_t rgs_cuda_norm_scratch_bytes(int64_t n, int64_t c) { return (int64_t)NORM_PARTS * 2 * c * 4 + (c > NR_MAX ? n * 8 : 0) + 16; }

int rgs_cuda_pack8(const void* x, int64_t dtype, int64_t ld, int64_t planes, int64_t n, int64_t c, int8_t* codes, uint8_t* expo, void* stream) {
    cudaStream_t st = (cudaStream_t)stream;
    NormArgs a{};
    a.x = x; a.src = (int)dtype; a.ld = ld; a.planes = (int)planes; a.n = n; a.c = (int)c; a.blocks = (int)((c + 31) / 32);
    a.codes_out = codes; a.expo_out = expo;
    if (planes) {
        const unsigned grid = (unsigned)norm_grid((n + NT - 1) / NT * a.blocks, 16);
        if (a.src == SRC_BF16) rgs_pack8_planes_kernel<RGS_BF16><<<grid, NT, 0, st>>>(a);
        else rgs_pack8_planes_kernel<RGS_F32><<<grid, NT, 0, st>>>(a);
    } else if (c % 4 == 0 && ld % 4 == 0 && aligned_to(x, four(a.src))) {
        const unsigned grid = (unsigned)norm_grid((n * a.blocks * 8 + NT * 4 - 1) / (NT * 4), 32);
        const int flat = c % 32 == 0 && ld == c;
        if (a.src == SRC_BF16) rgs_pack8_rows_kernel<4, RGS_BF16><<<grid, NT, 0, st>>>(a, flat);
        else rgs_pack8_rows_kernel<4, RGS_F32><<<grid, NT, 0, st>>>(a, flat);
    } else {
        const unsigned grid = (unsigned)norm_grid((n * a.blocks * 32 + NT * 4 - 1) / (NT * 4), 32);
        if (a.src == SRC_BF16) rgs_pack8_rows_kernel<1, RGS_BF16><<<grid, NT, 0, st>>>(a, 0);
        else rgs_pack8_rows_kernel<1, RGS_F32><<<grid, NT, 0, st>>>(a, 0);
    }
    return (int)cudaGetLastError();
}

int rgs_cuda_unpack8(const int8_t* codes, const uint8_t* expo, int64_t planes, int64_t n, int64_t c, void* out, int64_t dtype, void* stream) {
    cudaStream_t st = (cudaStream_t)stream;
    NormArgs a{};
    a.codes = codes; a.expo = expo; a.planes = (int)planes; a.n = n; a.c = (int)c; a.blocks = (int)((c + 31) / 32);
    if ((planes ? n : c) % 4 == 0)
        rgs_unpack8_kernel<4><<<(unsigned)norm_grid((n * c / 4 + NT * 4 - 1) / (NT * 4), 32), NT, 0, st>>>(a, !planes && c % 32 == 0, out, (int)dtype);
    else
        rgs_unpack8_kernel<1><<<(unsigned)norm_grid((n * c + NT * 4 - 1) / (NT * 4), 32), NT, 0, st>>>(a, 0, out, (int)dtype);
    return (int)cudaGetLastError();
}

int rgs_cuda_norm_fwd(const void* x, int64_t dtype, int64_t ld, int64_t planes, const void* w, const void* b, int64_t p_dtype, int64_t n,
                      int64_t c, double eps, void* y, int64_t y_dtype, int8_t* codes, uint8_t* expo, void* stream) {
    cudaStream_t st = (cudaStream_t)stream;
    NormArgs a{};
    a.x = x; a.src = (int)dtype; a.ld = ld; a.planes = (int)planes;
    a.w = w; a.b = b; a.p_dtype = (int)p_dtype;
    a.n = n; a.c = (int)c; a.blocks = (int)((c + 31) / 32); a.eps = (float)eps; a.inv_c = 1.f / (float)c;
    a.y = y; a.y_dtype = (int)y_dtype;
    a.codes_out = codes; a.expo_out = expo;
    if (c > NR_MAX) {
        rgs_norm_wide_kernel<<<(unsigned)norm_grid((n + 7) / 8, 16), NT, 0, st>>>(a, 0, nullptr);
        RGS_CUDA_CHECK(cudaGetLastError());
        return codes ? rgs_cuda_pack8(x, dtype, ld, planes, n, c, codes, expo, stream) : 0;
    }
    if (planes) {
        int parts;
        return norm_planes<false>(a, &parts, st);
    }
    const bool vec = c % 4 == 0 && ld % 4 == 0 && aligned_to(x, four(a.src));
    norm_rows(a, vec, false, st);
    return (int)cudaGetLastError();
}

int rgs_cuda_norm_bwd(const void* x, int64_t dtype, int64_t ld, int64_t planes, const int8_t* codes, const uint8_t* expo, const void* dy,
                      int64_t dy_dtype, int64_t ldy, const void* w, int64_t p_dtype, int64_t n, int64_t c, double eps, void* scratch,
                      void* dx, void* dw, void* db, void* stream) {
    cudaStream_t st = (cudaStream_t)stream;
    NormArgs a{};
    a.x = x; a.src = codes ? SRC_CODES : (int)dtype; a.ld = ld; a.planes = (int)planes;
    a.codes = codes; a.expo = expo;
    a.w = w; a.p_dtype = (int)p_dtype;
    a.n = n; a.c = (int)c; a.blocks = (int)((c + 31) / 32); a.eps = (float)eps; a.inv_c = 1.f / (float)c;
    a.dy = dy; a.dy_dtype = (int)dy_dtype; a.ldy = ldy;
    a.dx = dx; a.dx_dtype = (int)dtype;
    a.part = dw || db ? static_cast<float*>(scratch) : nullptr;
    int parts = 0;
    if (c > NR_MAX) {
        float2* stats = reinterpret_cast<float2*>(static_cast<float*>(scratch) + (int64_t)NORM_PARTS * 2 * c);
        rgs_norm_wide_kernel<<<(unsigned)norm_grid((n + 7) / 8, 16), NT, 0, st>>>(a, 1, stats);
        if (a.part) {
            parts = (int)norm_grid((n + 63) / 64, 1);
            rgs_norm_wide_sums_kernel<<<dim3((unsigned)((c + 31) / 32), (unsigned)parts), NT, 0, st>>>(a, stats);
        }
    } else if (planes) {
        const int rc = norm_planes<true>(a, &parts, st);
        if (rc) return rc;
    } else {
        const bool vec = c % 4 == 0 && ldy % 4 == 0 && aligned_to(dy, four(a.dy_dtype)) &&
                         (codes || (ld % 4 == 0 && aligned_to(x, four((int)dtype))));
        parts = norm_rows(a, vec, true, st);
    }
    RGS_CUDA_CHECK(cudaGetLastError());
    if (a.part)
        rgs_norm_reduce_kernel<<<dim3((unsigned)((c + 31) / 32), 2), 1024, 0, st>>>(a.part, parts, (int)c, dw, db, (int)p_dtype);
    return (int)cudaGetLastError();
}

}  // extern "C"

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
// Rows are read in aligned vectors of four.  Where a row does not begin on such a boundary (a width that four does not
// divide) its vectors begin up to three elements before it: a group takes rows a multiple of four apart, so that this shift
// and with it the channels of a lane stay the same; the first and last vector of a row are then read element by element.
// Codes of such rows are read element by element throughout.  Channel planes (the renderer's images) are read with a lane to
// a pixel and turned into rows in shared memory.  Beyond 1024 channels a warp re-reads its row.
//
// Measured (a copy moves 6.5 TB/s): 1657600 rows x 64 channels, float32 in, bf16 out: forward 108 us (5.9 TB/s), with the
// 8-bit copy 127 us (5.8 TB/s), backward 189 us (5.6 TB/s), from codes 206 us (3.6 TB/s: the arithmetic of decoding shares
// the time); the same from planes 193 and 306 us, in 8 bits 317 and 364 us (instructions: two thirds of the issue slots, most of
// them addresses and the sums over warps); 40003 x 771 bf16 47 and 134 us (backward: 255 registers, one block to an SM, a quarter
// of the issue slots: waiting, with no registers left to fetch the next row ahead), in 8 bits, codes one by one, 103 and 439 us;
// packing 95, unpacking 118 us.  Beyond 1024 channels nothing is kept in registers: 40003 x 2000, a step, 1.0 ms.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <atomic>
#include <type_traits>
#include "rgs_cuda_common.cuh"
#include "rgs_field_math.h"

#define NT 256            // threads of a block
#define NR_MAX 1024       // channels that a group holds in registers
#define NP_MAX 512        // channels of planes that a block holds

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
    void* dw; void* db;                            // written at once when the grid is one block
};

// Whether vector k of a lane can reach outside the row.  The widths that a kernel of vectors of four takes fill all but its
// last vectors (norm_rows_vec), so only these, and the first one of shifted rows, are tested and masked.
template <int VEC, int NV, int LANES, bool SHIFT>
__device__ __forceinline__ constexpr bool maybe_out(int k) {
    return VEC == 1 || (LANES == 1 && NV == 3) || (SHIFT && k == 0) || k >= NV - (SHIFT ? 2 : 1);
}
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
// vectors k of a lane, from channel (k lanes + l) VEC - s on, of the row that starts at element i; zero outside the row
// (EDGE: the last row, whose last vector may reach behind the tensor)
template <int VEC, int NV, int LANES, int DT, bool SHIFT, bool EDGE>
__device__ __forceinline__ void load_all(const void* p, int64_t i, int l, int s, int c, float (&x)[NV][VEC]) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int at = (k * LANES + l) * VEC - (SHIFT ? s : 0);
        if (!maybe_out<VEC, NV, LANES, SHIFT>(k)) {
            load_vec<VEC, DT>(p, i + at, x[k]);
        } else if (EDGE && at < c && at + VEC > c) {
#pragma unroll
            for (int q = 0; q < VEC; ++q) {
                float f[1] = {0.f};
                if (at + q >= 0 && at + q < c) load_vec<1, DT>(p, i + at + q, f);
                x[k][q] = f[0];
            }
        } else if (at < c) {
            load_vec<VEC, DT>(p, i + at, x[k]);
        } else {
#pragma unroll
            for (int q = 0; q < VEC; ++q) x[k][q] = 0.f;
        }
    }
    if (SHIFT) {  // the first and the last vector of the row hold elements of its neighbours
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (maybe_out<VEC, NV, LANES, SHIFT>(k))
#pragma unroll
                for (int q = 0; q < VEC; ++q) {
                    const int at = (k * LANES + l) * VEC - s + q;
                    x[k][q] = at >= 0 && at < c ? x[k][q] : 0.f;
                }
    }
}
template <int VEC, int NV, int LANES, bool SHIFT, bool EDGE>
__device__ __forceinline__ void load_typed(const void* p, int dtype, int64_t i, int l, int s, int c, float (&x)[NV][VEC]) {
    if (dtype == RGS_BF16) load_all<VEC, NV, LANES, RGS_BF16, SHIFT, EDGE>(p, i, l, s, c, x);
    else load_all<VEC, NV, LANES, RGS_F32, SHIFT, EDGE>(p, i, l, s, c, x);
}
__device__ __forceinline__ uint32_t pair_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <int VEC, int DT>
__device__ __forceinline__ void store_vec(void* p, int64_t i, const float (&f)[VEC]) {
    if constexpr (VEC == 4 && DT == RGS_BF16) *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = make_uint2(pair_bf16(f[0], f[1]), pair_bf16(f[2], f[3]));
    else if constexpr (VEC == 4) *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(f[0], f[1], f[2], f[3]);
    else if constexpr (DT == RGS_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(f[0]);
    else static_cast<float*>(p)[i] = f[0];
}
template <int VEC, int NV, int LANES, int DT, bool SHIFT>
__device__ __forceinline__ void store_all(void* p, int64_t i, int l, int s, int c, const float (&x)[NV][VEC]) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int at = (k * LANES + l) * VEC - (SHIFT ? s : 0);
        if (!maybe_out<VEC, NV, LANES, SHIFT>(k) || (SHIFT ? at >= 0 && at + VEC <= c : at < c)) store_vec<VEC, DT>(p, i + at, x[k]);
    }
    if (SHIFT) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (maybe_out<VEC, NV, LANES, SHIFT>(k)) {
                const int at = (k * LANES + l) * VEC - s;
                if (at < 0 || (at + VEC > c && at < c))
#pragma unroll
                    for (int q = 0; q < VEC; ++q) {
                        const float f[1] = {x[k][q]};
                        if (at + q >= 0 && at + q < c) store_vec<1, DT>(p, i + at + q, f);
                    }
            }
    }
}
template <int VEC, int NV, int LANES, bool SHIFT>
__device__ __forceinline__ void store_typed(void* p, int dtype, int64_t i, int l, int s, int c, const float (&x)[NV][VEC]) {
    if (dtype == RGS_BF16) store_all<VEC, NV, LANES, RGS_BF16, SHIFT>(p, i, l, s, c, x);
    else store_all<VEC, NV, LANES, RGS_F32, SHIFT>(p, i, l, s, c, x);
}
// Codes of four channels (one word) or of one.  v * inv + 1.5 * 2^23 leaves the code in the low byte (two's complement); only
// the topmost exponent needs the bound of rgs_pack_code.
template <int VEC>
__device__ __forceinline__ void store_codes(int8_t* p, int64_t i, const float (&f)[VEC], uint32_t e) {
    const float inv = rgs_pack_inverse(e);
    uint32_t u[VEC];
    if (e < 249u) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) u[k] = __float_as_uint(fmaf(f[k], inv, 12582912.f));
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) u[k] = e == RGS_PACK_NAN ? 0u : (uint32_t)rgs_pack_code(f[k], inv);
    }
    if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(p + i) = __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
    else p[i] = (int8_t)u[0];
}
// The value of byte k: 2^23 + (code + 128) is the float with that byte in its mantissa; the offset comes off and the step on,
// both exactly (a conversion instruction runs at a quarter of the rate; the offset times the largest steps would overflow).
template <int VEC>
__device__ __forceinline__ void load_codes(const int8_t* p, int64_t i, float step, float (&f)[VEC]) {
    if constexpr (VEC == 4) {
        const uint32_t u = *reinterpret_cast<const uint32_t*>(p + i) ^ 0x80808080u;
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + k)) - 8388736.f) * step;
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

// whether element q of vector k of a lane is a channel
template <int VEC, int LANES, bool SHIFT>
__device__ __forceinline__ bool in_row(int k, int q, int l, int s, int c) {
    const int at = (k * LANES + l) * VEC;
    return SHIFT ? at + q >= s && at + q < c + s : at < c;
}

// mean and 1 / sqrt(var + eps) of a row
template <int VEC, int NV, int LANES, bool SHIFT>
__device__ __forceinline__ void row_stats(const float (&x)[NV][VEC], int l, int s0, int c, float inv_c, float eps, float& mu, float& rstd) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int q = 0; q < VEC; ++q) s += x[k][q];   // zero outside the row
    mu = group_sum<LANES>(s) * inv_c;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
            const float d = !maybe_out<VEC, NV, LANES, SHIFT>(k) || in_row<VEC, LANES, SHIFT>(k, q, l, s0, c) ? x[k][q] - mu : 0.f;
            s = fmaf(d, d, s);
        }
    rstd = rsqrtf(group_sum<LANES>(s) * inv_c + eps);  // within two units in the last place (the kernel of wide rows: root and quotient)
}

template <int VEC>
__device__ __forceinline__ void load_param(const float* sh, int at, float (&w)[VEC]) {
    if constexpr (VEC == 4) {
        const float4 u = *reinterpret_cast<const float4*>(sh + at);
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else {
        w[0] = sh[at];
    }
}

// the backward pass of a row: x, dy -> dx (over x), sums of dw and db
template <int VEC, int NV, int LANES, bool SHIFT>
__device__ __forceinline__ void row_bwd(float (&x)[NV][VEC], float (&g)[NV][VEC], const float* w, float (&sw)[NV][VEC], float (&sb)[NV][VEC],
                                        int l, int s0, int c, float inv_c, float eps) {
    float mu, rstd, sa = 0.f, sax = 0.f;
    row_stats<VEC, NV, LANES, SHIFT>(x, l, s0, c, inv_c, eps, mu, rstd);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        float wk[VEC];
        load_param<VEC>(w, (k * LANES + l) * VEC, wk);
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
            // (outside the row dy is zero, and so is what x adds to the sums)
            x[k][q] = (x[k][q] - mu) * rstd;
            sw[k][q] = fmaf(g[k][q], x[k][q], sw[k][q]);
            sb[k][q] += g[k][q];
            g[k][q] *= wk[q];
            sa += g[k][q];
            sax = fmaf(g[k][q], x[k][q], sax);
        }
    }
    sa = group_sum<LANES>(sa) * inv_c;
    sax = group_sum<LANES>(sax) * inv_c;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int q = 0; q < VEC; ++q) x[k][q] = rstd * (g[k][q] - sa - x[k][q] * sax);
}

// A parameter in shared memory as the vectors of a row see it: one copy for each shift, channel c of copy s at c + s.
template <int VEC, int NV, int LANES, bool SHIFT>
__device__ __forceinline__ void stage_param(const NormArgs& a, const void* p, float none, float* sh) {
    constexpr int ROW = NV * LANES * VEC;
    for (int j = threadIdx.x; j < (SHIFT ? 4 : 1) * ROW; j += NT) {
        const int c = SHIFT ? j % ROW - j / ROW : j;
        sh[j] = p && c >= 0 && c < a.c ? rgs_load_as_float(p, c, a.p_dtype) : none;
    }
}
// Sums of a block's groups, in the order of the groups, to the block's row of the partial sums; a vector of every lane at a
// time, and with shifted rows the three elements that its groups' vectors reach into the one before.
template <int VEC, int NV, int LANES, bool SHIFT>
__device__ __forceinline__ void block_sums(const NormArgs& a, int l, int s, const float (&sw)[NV][VEC], const float (&sb)[NV][VEC], float* sh) {
    constexpr int GROUPS = NT / LANES, W = LANES * VEC, ROW = SHIFT ? W + 3 : W;
    const int group = threadIdx.x / LANES;
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
        if (SHIFT && l == 0)
            for (int q = 0; q < 3; ++q) sh[group * ROW + q] = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (k * W >= a.c + (SHIFT ? 3 : 0)) break;
            __syncthreads();
            // position 3 + channel - k W: channels of this turn, and behind a shift the last ones of the turn before
#pragma unroll
            for (int q = 0; q < VEC; ++q) sh[group * ROW + l * VEC + q + (SHIFT ? 3 - s : 0)] = which ? sb[k][q] : sw[k][q];
            __syncthreads();
            const bool end = k + 1 == NV || (k + 1) * W >= a.c + (SHIFT ? 3 : 0);
            for (int j = threadIdx.x; j < (SHIFT && !end ? W : ROW); j += NT) {
                const int c = k * W + j - (SHIFT ? 3 : 0);
                if (c < 0 || c >= a.c) continue;
                float t = 0.f;
                for (int r = 0; r < GROUPS; ++r) t += sh[r * ROW + j];
                if (gridDim.x > 1) a.part[((int64_t)blockIdx.x * 2 + which) * a.c + c] = t;
                else if (which ? a.db : a.dw) rgs_store_float(which ? a.db : a.dw, c, a.p_dtype, t);
            }
            if (SHIFT) {  // what reaches into the next turn's first three places (a group overwrites those it does not reach into)
                __syncthreads();
                for (int q = l; q < 3; q += LANES) sh[group * ROW + q] = sh[group * ROW + W + q];
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// rows
// ---------------------------------------------------------------------------------------------------------------------
template <int VEC, int NV, int LANES, bool SHIFT, bool EDGE>
__device__ __forceinline__ void load_row(const NormArgs& a, int64_t i, int l, int s, float (&x)[NV][VEC]) {
    if (!SHIFT && a.src == SRC_CODES) {
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
        load_typed<VEC, NV, LANES, SHIFT, EDGE>(a.x, a.src, i * a.ld, l, s, a.c, x);
    }
}

template <int VEC, int NV, int LANES, bool SHIFT, bool PACK>
__global__ void __launch_bounds__(NT, NV * VEC <= 16 ? 4 : NV * VEC <= 24 ? 3 : 2) rgs_norm_rows_fwd_kernel(const __grid_constant__ NormArgs a) {
    constexpr int GROUPS = NT / LANES;
    const int l = threadIdx.x % LANES;
    const int64_t stride = (int64_t)gridDim.x * GROUPS;  // a multiple of four rows: the shift stays
    const int s = SHIFT ? (int)(((int64_t)blockIdx.x * GROUPS + threadIdx.x / LANES) * a.c & 3) : 0;
    constexpr int ROW = NV * LANES * VEC, COPIES = SHIFT ? 4 : 1;
    __shared__ __align__(16) float params[2 * COPIES * ROW];
    stage_param<VEC, NV, LANES, SHIFT>(a, a.w, 1.f, params);
    stage_param<VEC, NV, LANES, SHIFT>(a, a.b, 0.f, params + COPIES * ROW);
    __syncthreads();
    const float *w = params + s * ROW, *b = params + (COPIES + s) * ROW;
    // all lanes of a warp take the same number of turns: shuffles need them.  A row that is not there is zeros.
    auto turn = [&](int64_t row, bool there, auto edge) {
        float x[NV][VEC];
        if (there) {
            load_row<VEC, NV, LANES, SHIFT, decltype(edge)::value>(a, row, l, s, x);
        } else {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int q = 0; q < VEC; ++q) x[k][q] = 0.f;
        }
        __syncwarp();
        float mu, rstd;
        row_stats<VEC, NV, LANES, SHIFT>(x, l, s, a.c, a.inv_c, a.eps, mu, rstd);
        if (PACK) {
            // a block of 32 channels is 32 / VEC vectors: KB of every lane of the row, or one of some of its lanes
            constexpr int LB = RGS_PACK_BLOCK / VEC, KB = LANES < LB ? LB / LANES : 1;
#pragma unroll
            for (int k = 0; k < NV; k += KB) {
                uint32_t m = 0;
#pragma unroll
                for (int e = k; e < k + KB && e < NV; ++e)
#pragma unroll
                    for (int q = 0; q < VEC; ++q) m = max(m, __float_as_uint(x[e][q]) & 0x7fffffffu);
                m = rgs_pack_exponent(__uint_as_float(group_max<(LANES < LB ? LANES : LB)>(m)));
                if (there)
#pragma unroll
                    for (int e = k; e < k + KB && e < NV; ++e) {
                        const int c = (e * LANES + l) * VEC;
                        if (c >= a.c) break;
                        if (c % RGS_PACK_BLOCK == 0) a.expo_out[row * a.blocks + c / RGS_PACK_BLOCK] = (uint8_t)m;
                        store_codes<VEC>(a.codes_out, row * a.c + c, x[e], m);
                    }
                __syncwarp();
            }
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float wk[VEC], bk[VEC];
            load_param<VEC>(w, (k * LANES + l) * VEC, wk);
            load_param<VEC>(b, (k * LANES + l) * VEC, bk);
#pragma unroll
            for (int q = 0; q < VEC; ++q) x[k][q] = fmaf((x[k][q] - mu) * rstd, wk[q], bk[q]);
        }
        if (there) store_typed<VEC, NV, LANES, SHIFT>(a.y, a.y_dtype, row * a.c, l, s, a.c, x);
        __syncwarp();
    };
    const int64_t rows = SHIFT ? a.n - 1 : a.n;
    for (int64_t i = (int64_t)blockIdx.x * GROUPS; i < rows; i += stride) turn(i + threadIdx.x / LANES, i + threadIdx.x / LANES < rows, std::false_type());
    // the last row by itself: its last vector may reach behind the tensor (a group of the first block with its shift)
    if (SHIFT && blockIdx.x == 0) turn(rows, threadIdx.x / LANES == (rows & 3), std::true_type());
}

template <int VEC, int NV, int LANES, bool SHIFT>
__global__ void __launch_bounds__(NT, NV * VEC <= 12 ? 3 : NV * VEC <= (SHIFT ? 24 : 16) ? 2 : 1) rgs_norm_rows_bwd_kernel(const __grid_constant__ NormArgs a) {
    constexpr int GROUPS = NT / LANES;
    constexpr int ROW = NV * LANES * VEC, COPIES = SHIFT ? 4 : 1, SUMS = NT * VEC + (SHIFT ? 3 * GROUPS : 0);
    __shared__ __align__(16) float sh[COPIES * ROW > SUMS ? COPIES * ROW : SUMS];
    const int l = threadIdx.x % LANES;
    const int64_t stride = (int64_t)gridDim.x * GROUPS;
    const int s = SHIFT ? (int)(((int64_t)blockIdx.x * GROUPS + threadIdx.x / LANES) * a.c & 3) : 0;
    float sw[NV][VEC], sb[NV][VEC];
    stage_param<VEC, NV, LANES, SHIFT>(a, a.w, 1.f, sh);
    __syncthreads();
    const float* w = sh + s * ROW;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int q = 0; q < VEC; ++q) sw[k][q] = sb[k][q] = 0.f;
    auto fetch = [&](int64_t row, bool there, auto edge, float (&x)[NV][VEC], float (&g)[NV][VEC]) {
        if (there) {
            load_row<VEC, NV, LANES, SHIFT, decltype(edge)::value>(a, row, l, s, x);
            load_typed<VEC, NV, LANES, SHIFT, decltype(edge)::value>(a.dy, a.dy_dtype, row * a.ldy, l, s, a.c, g);
        } else {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int q = 0; q < VEC; ++q) x[k][q] = g[k][q] = 0.f;
        }
    };
    auto turn = [&](int64_t row, bool there, float (&x)[NV][VEC], float (&g)[NV][VEC]) {
        __syncwarp();
        // (a row that is not there adds none to the sums: with eps = 0 its rstd would be infinite)
        row_bwd<VEC, NV, LANES, SHIFT>(x, g, w, sw, sb, l, s, a.c, a.inv_c, there ? a.eps : 1.f);
        if (a.dx && there) store_typed<VEC, NV, LANES, SHIFT>(a.dx, a.dx_dtype, row * a.c, l, s, a.c, x);
        __syncwarp();
    };
    const int64_t rows = SHIFT ? a.n - 1 : a.n, mine = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LANES;
    float x[NV][VEC], g[NV][VEC];
    if constexpr (NV * VEC >= 20 && !SHIFT) {
        // one block to an SM: the next row is on its way while this one is worked on (771 shifted channels have no registers
        // left for it: 177 -> 284 us; 772 channels 114 -> 99 us)
        fetch(mine, mine < rows, std::false_type(), x, g);
        for (int64_t i = mine - threadIdx.x / LANES, row = mine; i < rows; i += stride, row += stride) {
            float nx[NV][VEC], ng[NV][VEC];
            fetch(row + stride, row + stride < rows, std::false_type(), nx, ng);
            turn(row, row < rows, x, g);
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int q = 0; q < VEC; ++q) { x[k][q] = nx[k][q]; g[k][q] = ng[k][q]; }
        }
    } else {
        for (int64_t i = mine - threadIdx.x / LANES, row = mine; i < rows; i += stride, row += stride) {
            fetch(row, row < rows, std::false_type(), x, g);
            turn(row, row < rows, x, g);
        }
    }
    if (SHIFT && blockIdx.x == 0) {
        const bool there = threadIdx.x / LANES == (rows & 3);
        fetch(rows, there, std::true_type(), x, g);
        turn(rows, there, x, g);
    }
    if (a.part) block_sums<VEC, NV, LANES, SHIFT>(a, l, s, sw, sb, sh);
}

// ---------------------------------------------------------------------------------------------------------------------
// channel planes: 32 or 64 pixels at a time, a lane to one or two; warp v of V holds channels v, v + V, ... of them, so planes are read
// and written where they lie, sums run over the warps, and only rows (y, dy) are turned around in shared memory
// ---------------------------------------------------------------------------------------------------------------------
// off: the lane's pixels relative to the tile (behind the last pixel: the last pixel again, which then counts nowhere)
template <int NV, int V, int Q, int SRC>
__device__ __forceinline__ void load_plane(const NormArgs& a, int64_t base, const int (&off)[Q], int v, float (&x)[Q][NV]) {
    constexpr int SIZE = SRC == SRC_CODES ? 1 : SRC == SRC_BF16 ? 2 : 4;
    const int64_t ld = SRC == SRC_CODES ? a.n : a.ld;
    const char* p = static_cast<const char*>(SRC == SRC_CODES ? static_cast<const void*>(a.codes) : a.x) + (v * ld + base) * SIZE;
    const uint8_t* expo = a.expo + base;
    float step[Q];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (SRC == SRC_CODES && k * V % RGS_PACK_BLOCK == 0) {  // (V divides 32: the warps' channels of a step lie in one block)
#pragma unroll
            for (int q = 0; q < Q; ++q) step[q] = k * V < a.c ? rgs_pack_step(expo[off[q]]) : 0.f;
            expo += a.n;
        }
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            float f[1] = {0.f};
            if (v + k * V < a.c) {
                if constexpr (SRC == SRC_CODES) load_codes<1>(reinterpret_cast<const int8_t*>(p), off[q], step[q], f);
                else load_vec<1, SRC>(p, off[q], f);
            }
            x[q][k] = f[0];
        }
        p += V * ld * SIZE;
    }
}
template <int NV, int V, int Q, typename T>
__device__ __forceinline__ void store_plane(const NormArgs& a, int64_t i, int v, const bool (&in)[Q], const float (&x)[Q][NV]) {
    T* out = static_cast<T*>(a.dx) + v * a.n + i;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (v + k * V < a.c)
#pragma unroll
            for (int q = 0; q < Q; ++q)
                if (in[q]) {
                    if constexpr (sizeof(T) == 2) out[q * 32] = __float2bfloat16_rn(x[q][k]);
                    else out[q * 32] = x[q][k];
                }
        out += V * a.n;
    }
}

// sums over the V warps of what each holds for its Q pixels; red: (V, 32 Q)
template <int V, int Q>
__device__ __forceinline__ void warps_sum(float (&t)[Q], float* red, int v, int p) {
#pragma unroll
    for (int q = 0; q < Q; ++q) red[(v * Q + q) * 32 + p] = t[q];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        t[q] = 0.f;
#pragma unroll
        for (int k = 0; k < V; ++k) t[q] += red[(k * Q + q) * 32 + p];
    }
}

// rows of `from` to rows of `to`, B at a time: all are read before the first is written (one row after the other waits once
// a row: 76 us of 213 forward)
template <int B, typename T>
__device__ __forceinline__ void copy_batch(T* to, int64_t to_ld, const T* from, int64_t from_ld, int first, int step, int count) {
    T t[B];
    for (int r = first; r < count; r += step * B) {
        const T* p = from + r * from_ld;
        T* q = to + r * to_ld;
        if (r + (B - 1) * step < count) {
#pragma unroll
            for (int k = 0; k < B; ++k) t[k] = p[k * step * from_ld];
#pragma unroll
            for (int k = 0; k < B; ++k) q[k * step * to_ld] = t[k];
        } else {
            for (int k = 0; r + k * step < count; ++k) q[k * step * to_ld] = p[k * step * from_ld];
        }
    }
}
template <typename T>
__device__ __forceinline__ void copy_rows(T* to, int64_t to_ld, const T* from, int64_t from_ld, int r0, int step, int l, int wide, int count, int units) {
    if (count > 7 * step) {
        for (int u = l; u < units; u += wide) copy_batch<8>(to + u, to_ld, from + u, from_ld, r0, step, count);
    } else if (count > 3 * step) {
        for (int u = l; u < units; u += wide) copy_batch<4>(to + u, to_ld, from + u, from_ld, r0, step, count);
    } else {  // fewer rows to a warp: places of a row
        for (int r = r0; r < count; r += step) {
            if (units > 7 * wide) copy_batch<8>(to + r * to_ld, 1, from + r * from_ld, 1, l, wide, units);
            else copy_batch<4>(to + r * to_ld, 1, from + r * from_ld, 1, l, wide, units);
        }
    }
}

// (32 Q, pitch) of T in shared memory <-> rows of c elements, ld apart; T2: two of them
template <int V, bool STORE, typename T, typename T2>
__device__ __forceinline__ void tile_rows(T* tile, int pitch, T* rows, int64_t ld, int count, int c, bool pairs) {
    const int units = pairs ? c / 2 : c, lane = threadIdx.x & 31;
    const int wide = units > 16 ? 32 : units > 8 ? 16 : units > 4 ? 8 : units > 2 ? 4 : 2;  // lanes to a row
    const int per = 32 / wide, l = lane & (wide - 1);
    const int r0 = (threadIdx.x >> 5) * per + lane / wide;
    if constexpr (STORE) {
        if (pairs) copy_rows<T2>(reinterpret_cast<T2*>(rows), ld / 2, reinterpret_cast<const T2*>(tile), pitch / 2, r0, V * per, l, wide, count, units);
        else copy_rows<T>(rows, ld, tile, pitch, r0, V * per, l, wide, count, units);
    } else {
        if (pairs) copy_rows<T2>(reinterpret_cast<T2*>(tile), pitch / 2, reinterpret_cast<const T2*>(rows), ld / 2, r0, V * per, l, wide, count, units);
        else copy_rows<T>(tile, pitch, rows, ld, r0, V * per, l, wide, count, units);
    }
}

template <int NV, int V, int Q, bool BWD>
__global__ void __launch_bounds__(V * 32, V == 4 ? (BWD ? 5 : 8) : V == 8 ? (NV == 16 ? (BWD ? 2 : 3) : (BWD ? 3 : 4)) : V == 16 ? (BWD ? 1 : 2) : 1) rgs_norm_planes_kernel(const __grid_constant__ NormArgs a) {
    extern __shared__ float sm[];
    constexpr int T = 32 * Q;                           // pixels of a tile
    float* red = sm;                                    // three sums of V x T, w and b, then the tile of y or dy
    float *w = sm + 3 * V * T, *b = w + NV * V;
    void* tile = b + NV * V;
    const int p = threadIdx.x & 31, v = threadIdx.x >> 5;
    const int dt = BWD ? a.dy_dtype : a.y_dtype;
    // words between pixels: odd, or half a word off, so that 32 pixels of a channel lie in different banks
    const int pitch = dt == RGS_BF16 ? (a.c % 4 == 0 ? a.c + 2 : a.c) : (a.c % 2 == 0 ? a.c + 1 : a.c);
    const int64_t ld = BWD ? a.ldy : a.c;
    const bool pairs = dt == RGS_BF16 && a.c % 2 == 0 && ld % 2 == 0 && (!BWD || (reinterpret_cast<uintptr_t>(a.dy) & 3) == 0);
    for (int c = threadIdx.x; c < NV * V; c += V * 32) {
        w[c] = a.w && c < a.c ? rgs_load_as_float(a.w, c, a.p_dtype) : 1.f;
        b[c] = a.b && c < a.c ? rgs_load_as_float(a.b, c, a.p_dtype) : 0.f;
    }
    w += v;
    b += v;
    float sw[NV], sb[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) sw[k] = sb[k] = 0.f;
    const int64_t tiles = (a.n + T - 1) / T;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int64_t base = t * T, i = base + p;
        const int count = (int)(a.n - base < T ? a.n - base : T);
        float x[Q][NV], s[Q], mu[Q], rstd[Q];
        int off[Q];
        bool in[Q];
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            in[q] = p + q * 32 < count;
            off[q] = min(p + q * 32, count - 1);
        }
        if (a.src == SRC_CODES) load_plane<NV, V, Q, SRC_CODES>(a, base, off, v, x);
        else if (a.src == SRC_BF16) load_plane<NV, V, Q, SRC_BF16>(a, base, off, v, x);
        else load_plane<NV, V, Q, SRC_F32>(a, base, off, v, x);
        if (BWD) {
            if (dt == RGS_BF16) tile_rows<V, false, uint16_t, uint32_t>(static_cast<uint16_t*>(tile), pitch, const_cast<uint16_t*>(static_cast<const uint16_t*>(a.dy)) + base * ld, ld, count, a.c, pairs);
            else tile_rows<V, false, float, float2>(static_cast<float*>(tile), pitch, const_cast<float*>(static_cast<const float*>(a.dy)) + base * ld, ld, count, a.c, false);
        }
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            s[q] = 0.f;
#pragma unroll
            for (int k = 0; k < NV; ++k) s[q] += x[q][k];
        }
        warps_sum<V, Q>(s, red, v, p);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            mu[q] = s[q] * a.inv_c;
            s[q] = 0.f;
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (v + k * V < a.c) s[q] = fmaf(x[q][k] - mu[q], x[q][k] - mu[q], s[q]);
        }
        warps_sum<V, Q>(s, red + V * T, v, p);
#pragma unroll
        for (int q = 0; q < Q; ++q) rstd[q] = rsqrtf(s[q] * a.inv_c + a.eps);
        if (!BWD) {
            if (a.codes_out) {
                // largest magnitude of a block of 32 channels: those of every warp lie in 32 / V of its steps
                constexpr int KB = V < RGS_PACK_BLOCK ? RGS_PACK_BLOCK / V : 1;
                uint32_t* top = reinterpret_cast<uint32_t*>(red + 2 * V * T);
#pragma unroll
                for (int k = 0; k < NV; k += KB) {
                    if (k * V >= a.c) break;
                    __syncthreads();
#pragma unroll
                    for (int q = 0; q < Q; ++q) {
                        uint32_t m = 0;
#pragma unroll
                        for (int e = k; e < k + KB && e < NV; ++e) m = max(m, __float_as_uint(x[q][e]) & 0x7fffffffu);
                        top[(v * Q + q) * 32 + p] = m;
                    }
                    __syncthreads();
#pragma unroll
                    for (int q = 0; q < Q; ++q) {
                        uint32_t m = 0;
#pragma unroll
                        for (int e = 0; e < V; ++e) m = max(m, top[(e * Q + q) * 32 + p]);
                        m = rgs_pack_exponent(__uint_as_float(m));
                        const int64_t iq = i + q * 32;
                        if (in[q]) {
                            if (v == 0) a.expo_out[(int64_t)(k * V / RGS_PACK_BLOCK) * a.n + iq] = (uint8_t)m;
#pragma unroll
                            for (int e = k; e < k + KB && e < NV; ++e) {
                                const float f[1] = {x[q][e]};
                                if (v + e * V < a.c) store_codes<1>(a.codes_out, (int64_t)(v + e * V) * a.n + iq, f, m);
                            }
                        }
                    }
                }
            }
            // (the last tile's rows were read before the barriers of these sums)
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const float wk = w[k * V], bk = b[k * V];
#pragma unroll
                for (int q = 0; q < Q; ++q) x[q][k] = fmaf((x[q][k] - mu[q]) * rstd[q], wk, bk);
            }
            if (dt == RGS_BF16) {
                __nv_bfloat16* o = static_cast<__nv_bfloat16*>(tile) + p * pitch + v;
#pragma unroll
                for (int q = 0; q < Q; ++q)
#pragma unroll
                    for (int k = 0; k < NV; ++k)
                        if (v + k * V < a.c) o[q * 32 * pitch + k * V] = __float2bfloat16_rn(x[q][k]);
            } else {
                float* o = static_cast<float*>(tile) + p * pitch + v;
#pragma unroll
                for (int q = 0; q < Q; ++q)
#pragma unroll
                    for (int k = 0; k < NV; ++k)
                        if (v + k * V < a.c) o[q * 32 * pitch + k * V] = x[q][k];
            }
            __syncthreads();
            if (dt == RGS_BF16) tile_rows<V, true, uint16_t, uint32_t>(static_cast<uint16_t*>(tile), pitch, static_cast<uint16_t*>(a.y) + base * ld, ld, count, a.c, pairs);
            else tile_rows<V, true, float, float2>(static_cast<float*>(tile), pitch, static_cast<float*>(a.y) + base * ld, ld, count, a.c, false);
        } else {
            float g[Q][NV], sa[Q], sax[Q];
            if (dt == RGS_BF16) {
                const uint16_t* o = static_cast<const uint16_t*>(tile) + p * pitch + v;
#pragma unroll
                for (int q = 0; q < Q; ++q)
#pragma unroll
                    for (int k = 0; k < NV; ++k) g[q][k] = v + k * V < a.c ? rgs_bf16_value(o[q * 32 * pitch + k * V]) : 0.f;
            } else {
                const float* o = static_cast<const float*>(tile) + p * pitch + v;
#pragma unroll
                for (int q = 0; q < Q; ++q)
#pragma unroll
                    for (int k = 0; k < NV; ++k) g[q][k] = v + k * V < a.c ? o[q * 32 * pitch + k * V] : 0.f;
            }
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                sa[q] = sax[q] = 0.f;
                if (count < T && !in[q]) {  // the last pixel again: none of it counts, whatever it holds
                    mu[q] = rstd[q] = 0.f;
#pragma unroll
                    for (int k = 0; k < NV; ++k) x[q][k] = g[q][k] = 0.f;
                }
#pragma unroll
                for (int k = 0; k < NV; ++k) {  // (outside dy is zero, and so is what x adds to the sums)
                    x[q][k] = (x[q][k] - mu[q]) * rstd[q];
                    sw[k] = fmaf(g[q][k], x[q][k], sw[k]);
                    sb[k] += g[q][k];
                    g[q][k] *= w[k * V];
                    sa[q] += g[q][k];
                    sax[q] = fmaf(g[q][k], x[q][k], sax[q]);
                }
            }
            warps_sum<V, Q>(sax, red + 2 * V * T, v, p);
            warps_sum<V, Q>(sa, red, v, p);  // (every warp has read the first sum before the barrier of the second)
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                sa[q] *= a.inv_c;
                sax[q] *= a.inv_c;
#pragma unroll
                for (int k = 0; k < NV; ++k) x[q][k] = rstd[q] * (g[q][k] - sa[q] - x[q][k] * sax[q]);
            }
            if (a.dx) {
                if (a.dx_dtype == RGS_BF16) store_plane<NV, V, Q, __nv_bfloat16>(a, i, v, in, x);
                else store_plane<NV, V, Q, float>(a, i, v, in, x);
            }
            __syncthreads();  // the sums' words have been read before the next tile's are written
        }
    }
    if (BWD && a.part)
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = v + k * V;
            const float tw = group_sum<32>(sw[k]), tb = group_sum<32>(sb[k]);
            if (p == 0 && c < a.c) {
                if (gridDim.x > 1) {
                    a.part[((int64_t)blockIdx.x * 2) * a.c + c] = tw;
                    a.part[((int64_t)blockIdx.x * 2 + 1) * a.c + c] = tb;
                } else {
                    if (a.dw) rgs_store_float(a.dw, c, a.p_dtype, tw);
                    if (a.db) rgs_store_float(a.db, c, a.p_dtype, tb);
                }
            }
        }
}

// ---------------------------------------------------------------------------------------------------------------------
// more channels than a group holds: a warp re-reads its row; a block of threads per 32 channels sums dw and db
// ---------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float wide_value(const NormArgs& a, int64_t i, int c) {
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
            rgs_store_float(a.dx, i * a.c + j, a.dx_dtype, rstd * (g - sa - (wide_value(a, i, j) - mu) * rstd * sax));
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
// Rows: eight lanes to a 32-channel block, four channels each (together, or eight apart where rows are not aligned), so that a
// warp reads and writes what lies together; four blocks in flight.  `flat`: whole blocks that follow one another without a
// gap, no division.
template <int VEC, int DT>
__global__ void __launch_bounds__(NT) rgs_pack8_rows_kernel(const __grid_constant__ NormArgs a, int flat) {
    constexpr int LB = 8, U = 4;
    const int l = threadIdx.x % LB;
    const int64_t total = a.n * a.blocks, per = NT / LB;
    for (int64_t t0 = (int64_t)blockIdx.x * (per * U); t0 < total; t0 += (int64_t)gridDim.x * (per * U)) {
        float x[U][4];
        int64_t row[U];
        int c[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t t = t0 + u * per + threadIdx.x / LB;
            if (flat) { row[u] = t; c[u] = 0; }
            else {
                row[u] = total < ((int64_t)1 << 31) ? (int64_t)((uint32_t)t / (uint32_t)a.blocks) : t / a.blocks;
                c[u] = (int)(t - row[u] * a.blocks) * RGS_PACK_BLOCK;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) x[u][q] = 0.f;
            if (t >= total) continue;
            const int64_t at = flat ? t * RGS_PACK_BLOCK : row[u] * a.ld + c[u];
            if constexpr (VEC == 4) {
                if (flat || c[u] + l * 4 < a.c) load_vec<4, DT>(a.x, at + l * 4, x[u]);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float f[1] = {0.f};
                    if (c[u] + q * 8 + l < a.c) load_vec<1, DT>(a.x, at + q * 8 + l, f);
                    x[u][q] = f[0];
                }
            }
        }
        __syncwarp();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t t = t0 + u * per + threadIdx.x / LB;
            uint32_t top = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) top = max(top, __float_as_uint(x[u][q]) & 0x7fffffffu);
            const uint32_t e = rgs_pack_exponent(__uint_as_float(group_max<LB>(top)));
            if (t < total) {
                if (l == 0) a.expo_out[t] = (uint8_t)e;
                const int64_t at = flat ? t * RGS_PACK_BLOCK : row[u] * a.c + c[u];
                if constexpr (VEC == 4) {
                    if (flat || c[u] + l * 4 < a.c) store_codes<4>(a.codes_out, at + l * 4, x[u], e);
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float f[1] = {x[u][q]};
                        if (c[u] + q * 8 + l < a.c) store_codes<1>(a.codes_out, at + q * 8 + l, f, e);
                    }
                }
            }
            __syncwarp();
        }
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
            if (t0 + u * NT < total) {
                if (dtype == RGS_BF16) store_vec<VEC, RGS_BF16>(out, (t0 + u * NT) * VEC, f[u]);
                else store_vec<VEC, RGS_F32>(out, (t0 + u * NT) * VEC, f[u]);
            }
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

template <int VEC, int NV, int LANES, bool SHIFT>
static int norm_rows_launch(const NormArgs& a, bool backward, cudaStream_t st) {
    const int64_t want = (a.n + NT / LANES - 1) / (NT / LANES);
    if (backward) {
        static std::atomic<int64_t> most{0};
        if (!most) most = norm_resident(rgs_norm_rows_bwd_kernel<VEC, NV, LANES, SHIFT>, 0);
        // a few rows: one block, no partial sums, one launch
        const int64_t grid = want <= 4 ? 1 : at_most(at_most(want, most), NORM_PARTS);
        rgs_norm_rows_bwd_kernel<VEC, NV, LANES, SHIFT><<<(unsigned)grid, NT, 0, st>>>(a);
        rgs_cuda_field_launches(1);
        return (int)grid;
    }
    static std::atomic<int64_t> most[2];
    const int pack = !SHIFT && a.codes_out != nullptr;
    if (!most[pack])
        most[pack] = pack ? norm_resident(rgs_norm_rows_fwd_kernel<VEC, NV, LANES, SHIFT, !SHIFT>, 0) : norm_resident(rgs_norm_rows_fwd_kernel<VEC, NV, LANES, SHIFT, false>, 0);
    const unsigned grid = (unsigned)at_most(want, most[pack]);
    if (pack) rgs_norm_rows_fwd_kernel<VEC, NV, LANES, SHIFT, !SHIFT><<<grid, NT, 0, st>>>(a);
    else rgs_norm_rows_fwd_kernel<VEC, NV, LANES, SHIFT, false><<<grid, NT, 0, st>>>(a);
    rgs_cuda_field_launches(1);
    return 0;
}

// Few lanes to a row and several vectors to a lane: the shuffles of a row's sums are what narrow rows cost most (one lane
// to a vector: 1.4 TB/s at 33 channels, 3.4 at 64 backward).
template <bool SHIFT>
static int norm_rows_vec(const NormArgs& a, bool backward, cudaStream_t st) {
    const int u = (a.c + (SHIFT ? 6 : 0)) / 4;  // vectors of a row
    if (u <= 3) return norm_rows_launch<4, 3, 1, SHIFT>(a, backward, st);
    if (u <= 4) return norm_rows_launch<4, 4, 1, SHIFT>(a, backward, st);
    if (u <= 6) return norm_rows_launch<4, 3, 2, SHIFT>(a, backward, st);
    if (u <= 8) return norm_rows_launch<4, 4, 2, SHIFT>(a, backward, st);
    if (u <= 12) return norm_rows_launch<4, 3, 4, SHIFT>(a, backward, st);
    if (u <= 16) return norm_rows_launch<4, 4, 4, SHIFT>(a, backward, st);
    if (u <= 24) return norm_rows_launch<4, 3, 8, SHIFT>(a, backward, st);
    if (u <= 32) return norm_rows_launch<4, 4, 8, SHIFT>(a, backward, st);
    if (u <= 48) return norm_rows_launch<4, 3, 16, SHIFT>(a, backward, st);
    if (u <= 64) return norm_rows_launch<4, 4, 16, SHIFT>(a, backward, st);
    if (u <= 96) return norm_rows_launch<4, 3, 32, SHIFT>(a, backward, st);
    if (u <= 128) return norm_rows_launch<4, 4, 32, SHIFT>(a, backward, st);
    if (u <= 160) return norm_rows_launch<4, 5, 32, SHIFT>(a, backward, st);
    if (u <= 192) return norm_rows_launch<4, 6, 32, SHIFT>(a, backward, st);
    if (u <= 224) return norm_rows_launch<4, 7, 32, SHIFT>(a, backward, st);
    return norm_rows_launch<4, 8, 32, SHIFT>(a, backward, st);
}
// element by element: rows apart by a stride that four does not divide, codes of an odd width
static int norm_rows_single(const NormArgs& a, bool backward, cudaStream_t st) {
    const int u = a.c;
    if (u <= 8) return norm_rows_launch<1, 8, 1, false>(a, backward, st);
    if (u <= 16) return norm_rows_launch<1, 8, 2, false>(a, backward, st);
    if (u <= 32) return norm_rows_launch<1, 8, 4, false>(a, backward, st);
    if (u <= 64) return norm_rows_launch<1, 8, 8, false>(a, backward, st);
    if (u <= 128) return norm_rows_launch<1, 8, 16, false>(a, backward, st);
    if (u <= 256) return norm_rows_launch<1, 8, 32, false>(a, backward, st);
    if (u <= 512) return norm_rows_launch<1, 16, 32, false>(a, backward, st);
    if (u <= 768) return norm_rows_launch<1, 24, 32, false>(a, backward, st);
    return norm_rows_launch<1, 32, 32, false>(a, backward, st);
}

template <int NV, int V, int Q, bool BWD>
static int norm_planes_launch(const NormArgs& a, int* parts, cudaStream_t st) {
    const int smem = (3 * V * 32 * Q + 2 * NV * V + 32 * Q * (a.c + 2)) * 4;
    if (smem > 48 * 1024) RGS_CUDA_CHECK(cudaFuncSetAttribute(rgs_norm_planes_kernel<NV, V, Q, BWD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    int per_sm = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, rgs_norm_planes_kernel<NV, V, Q, BWD>, V * 32, (size_t)smem) != cudaSuccess || per_sm < 1) per_sm = 1;
    *parts = (int)at_most(at_most((a.n + 32 * Q - 1) / (32 * Q), RGS_SMS * per_sm), NORM_PARTS);
    rgs_norm_planes_kernel<NV, V, Q, BWD><<<(unsigned)*parts, V * 32, smem, st>>>(a);
    rgs_cuda_field_launches(1);
    return (int)cudaGetLastError();
}

template <bool BWD>
static int norm_planes(const NormArgs& a, int* parts, cudaStream_t st) {
    // few warps to a pixel: what the sums over the warps cost is what narrow planes cost most
    if (a.c <= 8) return norm_planes_launch<4, 2, 4, BWD>(a, parts, st);
    if (a.c <= 16) return norm_planes_launch<8, 2, 2, BWD>(a, parts, st);
    if (a.c <= 32) return norm_planes_launch<8, 4, 2, BWD>(a, parts, st);
    if (a.c <= 64) return norm_planes_launch<8, 8, 2, BWD>(a, parts, st);
    if (a.c <= 128) return norm_planes_launch<16, 8, 1, BWD>(a, parts, st);
    if (a.c <= 256) return norm_planes_launch<16, 16, 1, BWD>(a, parts, st);
    return norm_planes_launch<16, 32, 1, BWD>(a, parts, st);
}

extern "C" {

int64_t rgs_cuda_field_launches(int64_t more) {
    static std::atomic<int64_t> count{0};
    return count.fetch_add(more) + more;
}

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
    rgs_cuda_field_launches(1);
    return (int)cudaGetLastError();
}

int rgs_cuda_unpack8(const int8_t* codes, const uint8_t* expo, int64_t planes, int64_t n, int64_t c, void* out, int64_t dtype, void* stream) {
    cudaStream_t st = (cudaStream_t)stream;
    NormArgs a{};
    a.codes = codes; a.expo = expo; a.planes = (int)planes; a.n = n; a.c = (int)c; a.blocks = (int)((c + 31) / 32);
    if ((planes ? n : c) % 4 == 0 && aligned_to(codes, 4))  // (codes may be a slice that begins at any byte)
        rgs_unpack8_kernel<4><<<(unsigned)norm_grid((n * c / 4 + NT * 4 - 1) / (NT * 4), 32), NT, 0, st>>>(a, !planes && c % 32 == 0, out, (int)dtype);
    else
        rgs_unpack8_kernel<1><<<(unsigned)norm_grid((n * c + NT * 4 - 1) / (NT * 4), 32), NT, 0, st>>>(a, 0, out, (int)dtype);
    rgs_cuda_field_launches(1);
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
    if (planes && c > NP_MAX) return 23;
    if (c > NR_MAX) {
        rgs_norm_wide_kernel<<<(unsigned)norm_grid((n + 7) / 8, 16), NT, 0, st>>>(a, 0, nullptr);
        rgs_cuda_field_launches(1);
        RGS_CUDA_CHECK(cudaGetLastError());
        return codes ? rgs_cuda_pack8(x, dtype, ld, planes, n, c, codes, expo, stream) : 0;
    }
    if (planes) {
        int parts;
        return norm_planes<false>(a, &parts, st);
    }
    const bool start = aligned_to(x, four(a.src));
    if (start && c % 4 == 0 && ld % 4 == 0) norm_rows_vec<false>(a, false, st);
    else if (start && rgs_rows_shifted(c, ld)) {
        norm_rows_vec<true>(a, false, st);  // its blocks of 32 channels begin anywhere in a vector: packed by themselves
        RGS_CUDA_CHECK(cudaGetLastError());
        if (codes) return rgs_cuda_pack8(x, dtype, ld, planes, n, c, codes, expo, stream);
    } else norm_rows_single(a, false, st);
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
    a.dw = dw; a.db = db;
    int parts = 0;
    if (planes && c > NP_MAX) return 23;
    if (c > NR_MAX) {
        float2* stats = reinterpret_cast<float2*>(static_cast<float*>(scratch) + (int64_t)NORM_PARTS * 2 * c);
        rgs_norm_wide_kernel<<<(unsigned)norm_grid((n + 7) / 8, 16), NT, 0, st>>>(a, 1, stats);
        rgs_cuda_field_launches(1);
        if (a.part) {
            parts = (int)norm_grid((n + 63) / 64, 1);
            rgs_norm_wide_sums_kernel<<<dim3((unsigned)((c + 31) / 32), (unsigned)parts), NT, 0, st>>>(a, stats);
            rgs_cuda_field_launches(1);
        }
    } else if (planes) {
        const int rc = norm_planes<true>(a, &parts, st);
        if (rc) return rc;
    } else {
        // (codes that were kept elsewhere in between may come back at any byte)
        const bool start = aligned_to(dy, four(a.dy_dtype)) && (codes ? aligned_to(codes, 4) : aligned_to(x, four((int)dtype)));
        if (start && c % 4 == 0 && ldy % 4 == 0 && (codes || ld % 4 == 0)) parts = norm_rows_vec<false>(a, true, st);
        else if (start && !codes && rgs_rows_shifted(c, ld) && rgs_rows_shifted(c, ldy)) parts = norm_rows_vec<true>(a, true, st);
        else parts = norm_rows_single(a, true, st);
    }
    RGS_CUDA_CHECK(cudaGetLastError());
    if (a.part && (parts > 1 || c > NR_MAX)) {
        rgs_norm_reduce_kernel<<<dim3((unsigned)((c + 31) / 32), 2), 1024, 0, st>>>(a.part, parts, (int)c, dw, db, (int)p_dtype);
        rgs_cuda_field_launches(1);
    }
    return (int)cudaGetLastError();
}

}  // extern "C"

// Scalar math of the label-field operators (label loss, layer norm, 8-bit kept features), shared by the sm_100a kernels
// and the native CPU backend.
//
// 8-bit blocks: 32 consecutive channels of a row share the power of two 2^e, e the smallest integer with
// 127 * 2^e >= max|x| (at least -126); a value is kept as round-half-even(x * 2^-e).  Scaling by a power of two and
// rounding to an integer are both exact in 32 bits, so every implementation produces the same codes.  A block that
// holds an infinity or a NaN gets the exponent byte 255 and stands for NaN throughout.
#pragma once
#include <math.h>
#include <stdint.h>
#include <string.h>
#include "rgs_math.h"

#define RGS_F32 0
#define RGS_BF16 1
#define RGS_PACK_BLOCK 32
#define RGS_PACK_NAN 255

RGS_HD uint32_t rgs_f2u(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }
RGS_HD float rgs_u2f(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }

// Exponent byte (e + 127) of a block whose largest magnitude is m (m >= 0, NaN and infinity included).
RGS_HD uint32_t rgs_pack_exponent(float m) {
    const uint32_t u = rgs_f2u(m);
    if (u >= 0x7f800000u) return RGS_PACK_NAN;
    if (u == 0u) return 127u;
    // m = 1.f * 2^q with q = (u >> 23) - 127; 127 * 2^(q-6) covers it unless the mantissa is above 127/64
    const int q = (int)(u >> 23) - 6 + ((u & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    return (uint32_t)(q < 1 ? 1 : q);
}
RGS_HD float rgs_pack_step(uint32_t expo) { return expo >= 254u ? rgs_u2f(0x7fc00000u) : rgs_u2f(expo << 23); }
RGS_HD float rgs_pack_inverse(uint32_t expo) { return expo >= 254u ? 0.f : rgs_u2f((254u - expo) << 23); }
// |v * inv| <= 127 for members of the block, so adding 1.5 * 2^23 rounds it half to even into the low mantissa bits.
// Magnitudes above 63 * 2^122 count as that: the next code would stand for 2^128, which is no finite float.
RGS_HD int rgs_pack_code(float v, float inv) {
    const float top = 334965454937798799971759379190646833152.f;  // 63 * 2^122
    v = v > top ? top : (v < -top ? -top : v);
    return (int)(rgs_f2u(v * inv + 12582912.f) - 0x4b400000u);
}

// Round a 32-bit float to bf16, half to even (host twin of the device conversion).
RGS_HD uint16_t rgs_bf16_bits(float f) {
    const uint32_t u = rgs_f2u(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)0x7fffu;
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
RGS_HD float rgs_bf16_value(uint16_t b) { return rgs_u2f((uint32_t)b << 16); }

// Whether rows of c channels, ld apart and the first of them aligned, may be read in aligned vectors of four that begin inside
// the row in front (rgs_norm.cu; the last row is read by itself).  The shift repeats where ld = c modulo 4, and a lane holds
// 1024 channels with it.  Of the other rows the vectors end up to three elements behind the row: with ld >= 2 that is inside the
// tensor (row n-2 ends at (n-1) ld - ld + c; 2 and 3 channels: the multiple of four behind it is at most (n-1) ld + c), with
// single elements it is not: row n-3 or n-2 would be read up to element n.
RGS_HD bool rgs_rows_shifted(int64_t c, int64_t ld) { return (ld - c) % 4 == 0 && c <= 1024 - 6 && ld > 1; }

RGS_HD float rgs_load_as_float(const void* p, int64_t i, int dtype) {
    return dtype == RGS_BF16 ? rgs_bf16_value(static_cast<const uint16_t*>(p)[i]) : static_cast<const float*>(p)[i];
}
RGS_HD void rgs_store_float(void* p, int64_t i, int dtype, float v) {
    if (dtype == RGS_BF16) static_cast<uint16_t*>(p)[i] = rgs_bf16_bits(v);
    else static_cast<float*>(p)[i] = v;
}
// Label of a row, or -1 when the row does not count (any label outside [0, vocab)).
RGS_HD int64_t rgs_label(const void* labels, int64_t i, int label_bytes, int64_t vocab) {
    const int64_t y = label_bytes == 8 ? static_cast<const int64_t*>(labels)[i] : (int64_t)static_cast<const int32_t*>(labels)[i];
    return y >= 0 && y < vocab ? y : -1;
}

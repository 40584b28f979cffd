// CPU twins of the label-field operators (rgs_label.cu, rgs_norm.cu): OpenMP loops with 64-bit sums.
#include <math.h>
#include <stdint.h>
#include <string.h>
#include <new>
#include <vector>
#include "rgs_field_math.h"

static inline int64_t field_at(int64_t n, int64_t c, int64_t ld, int64_t planes) { return planes ? c * ld + n : n * ld + c; }

extern "C" {

int64_t rgs_cpu_norm_scratch_bytes(int64_t, int64_t) { return 16; }
int64_t rgs_cpu_label_scratch_bytes(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) { return 16; }
int64_t rgs_cpu_rows_shifted(int64_t c, int64_t ld) { return rgs_rows_shifted(c, ld); }  // the rule of rgs_norm.cu

int rgs_cpu_pack8(const void* x, int64_t dtype, int64_t ld, int64_t planes, int64_t n, int64_t c, int8_t* codes, uint8_t* expo, void*) {
    const int64_t blocks = (c + RGS_PACK_BLOCK - 1) / RGS_PACK_BLOCK;
#pragma omp parallel for schedule(static)
    for (int64_t i = 0; i < n; ++i)
        for (int64_t b = 0; b < blocks; ++b) {
            const int64_t c0 = b * RGS_PACK_BLOCK, c1 = c0 + RGS_PACK_BLOCK < c ? c0 + RGS_PACK_BLOCK : c;
            uint32_t top = 0;  // magnitudes compare as their bits, NaN above infinity
            for (int64_t j = c0; j < c1; ++j) {
                const uint32_t u = rgs_f2u(rgs_load_as_float(x, field_at(i, j, ld, planes), (int)dtype)) & 0x7fffffffu;
                if (u > top) top = u;
            }
            const uint32_t e = rgs_pack_exponent(rgs_u2f(top));
            const float inv = rgs_pack_inverse(e);
            expo[planes ? b * n + i : i * blocks + b] = (uint8_t)e;
            for (int64_t j = c0; j < c1; ++j) {
                const float v = rgs_load_as_float(x, field_at(i, j, ld, planes), (int)dtype);
                codes[planes ? j * n + i : i * c + j] = (int8_t)(e == RGS_PACK_NAN ? 0 : rgs_pack_code(v, inv));
            }
        }
    return 0;
}

int rgs_cpu_unpack8(const int8_t* codes, const uint8_t* expo, int64_t planes, int64_t n, int64_t c, void* out, int64_t dtype, void*) {
    const int64_t blocks = (c + RGS_PACK_BLOCK - 1) / RGS_PACK_BLOCK;
#pragma omp parallel for schedule(static)
    for (int64_t i = 0; i < n; ++i)
        for (int64_t j = 0; j < c; ++j) {
            const int64_t b = j / RGS_PACK_BLOCK, at = planes ? j * n + i : i * c + j;
            rgs_store_float(out, at, (int)dtype, (float)codes[at] * rgs_pack_step(expo[planes ? b * n + i : i * blocks + b]));
        }
    return 0;
}

int rgs_cpu_norm_fwd(const void* x, int64_t dtype, int64_t ld, int64_t planes, const void* w, const void* b, int64_t p_dtype, int64_t n,
                     int64_t c, double eps, void* y, int64_t y_dtype, int8_t* codes, uint8_t* expo, void*) {
#pragma omp parallel for schedule(static)
    for (int64_t i = 0; i < n; ++i) {
        double mu = 0, var = 0;
        for (int64_t j = 0; j < c; ++j) mu += rgs_load_as_float(x, field_at(i, j, ld, planes), (int)dtype);
        mu /= (double)c;
        for (int64_t j = 0; j < c; ++j) { const double d = rgs_load_as_float(x, field_at(i, j, ld, planes), (int)dtype) - mu; var += d * d; }
        const double rstd = 1.0 / sqrt(var / (double)c + eps);
        for (int64_t j = 0; j < c; ++j) {
            double v = (rgs_load_as_float(x, field_at(i, j, ld, planes), (int)dtype) - mu) * rstd;
            if (w) v *= rgs_load_as_float(w, j, (int)p_dtype);
            if (b) v += rgs_load_as_float(b, j, (int)p_dtype);
            rgs_store_float(y, i * c + j, (int)y_dtype, (float)v);
        }
    }
    return codes ? rgs_cpu_pack8(x, dtype, ld, planes, n, c, codes, expo, nullptr) : 0;
}

int rgs_cpu_norm_bwd(const void* x, int64_t dtype, int64_t ld, int64_t planes, const int8_t* codes, const uint8_t* expo, const void* dy,
                     int64_t dy_dtype, int64_t ldy, const void* w, int64_t p_dtype, int64_t n, int64_t c, double eps, void*, void* dx,
                     void* dw, void* db, void*) {
    const int64_t blocks = (c + RGS_PACK_BLOCK - 1) / RGS_PACK_BLOCK;
    auto kept = [&](int64_t i, int64_t j) -> double {
        if (!codes) return rgs_load_as_float(x, field_at(i, j, ld, planes), (int)dtype);
        const int64_t b = j / RGS_PACK_BLOCK;
        return (float)codes[planes ? j * n + i : i * c + j] * rgs_pack_step(expo[planes ? b * n + i : i * blocks + b]);
    };
    auto stats = [&](int64_t i, double& mu, double& rstd) {
        double var = 0;
        mu = 0;
        for (int64_t j = 0; j < c; ++j) mu += kept(i, j);
        mu /= (double)c;
        for (int64_t j = 0; j < c; ++j) { const double d = kept(i, j) - mu; var += d * d; }
        rstd = 1.0 / sqrt(var / (double)c + eps);
    };
    if (dx) {
#pragma omp parallel for schedule(static)
        for (int64_t i = 0; i < n; ++i) {
            double mu, rstd, sa = 0, sax = 0;
            stats(i, mu, rstd);
            for (int64_t j = 0; j < c; ++j) {
                const double a = (double)rgs_load_as_float(dy, i * ldy + j, (int)dy_dtype) * (w ? rgs_load_as_float(w, j, (int)p_dtype) : 1.f);
                sa += a;
                sax += a * (kept(i, j) - mu) * rstd;
            }
            sa /= (double)c;
            sax /= (double)c;
            for (int64_t j = 0; j < c; ++j) {
                const double a = (double)rgs_load_as_float(dy, i * ldy + j, (int)dy_dtype) * (w ? rgs_load_as_float(w, j, (int)p_dtype) : 1.f);
                rgs_store_float(dx, planes ? j * n + i : i * c + j, (int)dtype, (float)(rstd * (a - sa - (kept(i, j) - mu) * rstd * sax)));
            }
        }
    }
    if (dw || db) {
        std::vector<double> ms;  // mean and rstd of every row, once (anew for every channel: quadratic in the channels)
        if (dw) {
            try {
                ms.resize(2 * (size_t)n);
            } catch (const std::exception&) {
                return 12;
            }
#pragma omp parallel for schedule(static)
            for (int64_t i = 0; i < n; ++i) stats(i, ms[2 * i], ms[2 * i + 1]);
        }
#pragma omp parallel for schedule(static)
        for (int64_t j = 0; j < c; ++j) {
            double sw = 0, sb = 0;
            for (int64_t i = 0; i < n; ++i) {
                const double g = rgs_load_as_float(dy, i * ldy + j, (int)dy_dtype);
                sb += g;
                if (dw) sw += g * (kept(i, j) - ms[2 * i]) * ms[2 * i + 1];
            }
            if (dw) rgs_store_float(dw, j, (int)p_dtype, (float)sw);
            if (db) rgs_store_float(db, j, (int)p_dtype, (float)sb);
        }
    }
    return 0;
}

// Score of a row and a label, rounded to 32 bits as on the GPU: the largest one is kept for the backward pass as a float, and only
// of numbers that it holds exactly do the differences stay (a 64-bit score of 1e9 differs from its float by up to 32, and exp of
// that is not at most one).
static inline double label_score(const void* x, int64_t xi, const void* w, int64_t wi, const void* bias, int64_t v, int64_t c, int dtype,
                                 int b_dtype) {
    double l = bias ? rgs_load_as_float(bias, v, b_dtype) : 0.f;
    for (int64_t j = 0; j < c; ++j) l += (double)rgs_load_as_float(x, xi + j, dtype) * rgs_load_as_float(w, wi + j, dtype);
    return (double)(float)l;
}

// lse (2,n): largest score and log sum exp(score - largest) of a row, two numbers so that scores of any size (all labels at
// the lowest value of the type, say) keep their differences; losses[i] per row, result[0] = sum / max(count, 1) or sum, count[0] = rows that count
int rgs_cpu_label_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* labels, int64_t label_bytes,
                      int64_t n, int64_t c, int64_t vocab, int64_t dtype, int64_t b_dtype, int64_t mean, void*, int64_t, float* lse, float* losses,
                      float* result, float* count, void*) {
    double total = 0;
    int64_t rows = 0;
#pragma omp parallel for schedule(static) reduction(+ : total, rows)
    for (int64_t i = 0; i < n; ++i) {
        const int64_t y = rgs_label(labels, i, (int)label_bytes, vocab);
        double m = -INFINITY, s = 0, at = 0;
        for (int64_t v = 0; v < vocab; ++v) {
            const double l = label_score(x, i * ldx, w, v * ldw, bias, v, c, (int)dtype, (int)b_dtype);
            if (v == y) at = l;
            if (l > m || l != l) { s *= exp(m - l); m = l; }
            s += l == -INFINITY && m == -INFINITY ? 0.0 : exp(l - m);
        }
        const double z = log(s), loss = y < 0 ? 0.0 : z + (m - at);
        lse[i] = (float)m;
        lse[n + i] = (float)z;
        if (losses) losses[i] = (float)loss;
        total += loss;
        rows += y >= 0;
    }
    *count = (float)rows;
    if (result) *result = (float)(mean ? total / (double)(rows > 0 ? rows : 1) : total);
    return 0;
}

// gout: one gradient for all rows (per_row = 0; divided by max(count, 1) for the mean) or one per row
int rgs_cpu_label_bwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* labels, int64_t label_bytes,
                      int64_t n, int64_t c, int64_t vocab, int64_t dtype, int64_t b_dtype, const float* lse, const float* gout,
                      int64_t per_row, int64_t mean, const float* count, void*, int64_t, void* dx, void* dw, void* db, void*) {
    const double scale = mean ? 1.0 / (*count > 1.f ? *count : 1.f) : 1.0;
    auto grad = [&](int64_t i, int64_t v, int64_t y) -> double {
        const double l = label_score(x, i * ldx, w, v * ldw, bias, v, c, (int)dtype, (int)b_dtype);
        return (exp((l - lse[i]) - lse[n + i]) - (v == y)) * gout[per_row ? i : 0] * scale;
    };
    if (dx) {
#pragma omp parallel
        {
            double acc[4096];
#pragma omp for schedule(static)
            for (int64_t i = 0; i < n; ++i)
                for (int64_t c0 = 0; c0 < c; c0 += 4096) {
                    const int64_t cn = c - c0 < 4096 ? c - c0 : 4096, y = rgs_label(labels, i, (int)label_bytes, vocab);
                    for (int64_t j = 0; j < cn; ++j) acc[j] = 0;
                    for (int64_t v = 0; v < vocab && y >= 0; ++v) {
                        const double g = grad(i, v, y);
                        for (int64_t j = 0; j < cn; ++j) acc[j] += g * rgs_load_as_float(w, v * ldw + c0 + j, (int)dtype);
                    }
                    for (int64_t j = 0; j < cn; ++j) rgs_store_float(dx, i * c + c0 + j, (int)dtype, (float)acc[j]);
                }
        }
    }
    if (dw || db) {
#pragma omp parallel
        {
            double acc[4096];
#pragma omp for schedule(static)
            for (int64_t v = 0; v < vocab; ++v) {
                double sb = 0;
                for (int64_t c0 = 0; c0 < c; c0 += 4096) {
                    const int64_t cn = c - c0 < 4096 ? c - c0 : 4096;
                    for (int64_t j = 0; j < cn; ++j) acc[j] = 0;
                    for (int64_t i = 0; i < n; ++i) {
                        const int64_t y = rgs_label(labels, i, (int)label_bytes, vocab);
                        if (y < 0) continue;
                        const double g = grad(i, v, y);
                        if (c0 == 0) sb += g;
                        for (int64_t j = 0; j < cn; ++j) acc[j] += g * rgs_load_as_float(x, i * ldx + c0 + j, (int)dtype);
                    }
                    if (dw)
                        for (int64_t j = 0; j < cn; ++j) rgs_store_float(dw, v * c + c0 + j, (int)dtype, (float)acc[j]);
                }
                if (db) rgs_store_float(db, v, (int)b_dtype, (float)sb);
            }
        }
    }
    return 0;
}

}  // extern "C"

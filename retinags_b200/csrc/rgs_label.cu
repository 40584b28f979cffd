// Label loss: softmax cross entropy of linear scores over a vocabulary, without the scores in memory.
//
//   s_nv = x_n . w_v + b_v,  m_n = max_v s_nv,  z_n = sum_v exp(s_nv - m_n),  loss_n = log z_n + (m_n - s_n,y_n)
//   G_nv = exp(s_nv - m_n) / z_n - [v = y_n],  dX = g G W,  dW = (g G)^T X,  db_v = sum_n g_n G_nv
//
// One persistent kernel on the fifth-generation tensor cores does all the products.  A CTA holds a tile of 128 rows of
// one matrix (A: rows of X for the loss and dX, rows of W for dW) and walks tiles of 128 rows of the other (B):
//   TMA brings tiles of 128 rows x 64 channels (bf16, 128-byte swizzle; up to 32 channels: 64 bytes) into a ring in shared memory
//   S = A B^T: tcgen05.mma into one of two to four score buffers in TMEM
//   four warpgroups, two to a score buffer with 64 of its columns each (one thread per row of A: no shuffles), form the
//   running maximum and sum (forward) or G (backward); G goes back over the scores in TMEM as a bf16 operand
//   O += G B: tcgen05.mma with G from TMEM and the same B tile, read with its channels as the N side
// so a B tile is fetched once for both products and the scores never leave the SM.  The gradient kernel walks the items of
// dX and dW in one launch.  For dW the roles are swapped (rows of A are labels, columns are pixels); the scores are
// computed anew there: five products of 2NVC operations in all against four with scores kept, and no N x V traffic.
//
// What depends on a row alone rides along in the product: sixteen extra channels hold (b in three bf16 pieces, 1, 1, 1) of a
// label and (1, 1, 1, -lse in three pieces) of a pixel, so S is the score with its bias and, backward, minus lse: the
// warpgroups need nothing per column but the labels of dW (constants per column read from shared memory cost as much of its
// bandwidth as half of the products' operands).  Columns behind the last label and pixels without one have -inf there.
// Where scores are so large that log z would vanish beside m (a mask of the type's lowest value over all labels), only the bias
// rides along: the scores are then formed in the very steps of the forward pass, m is taken off them in registers and 1/z is
// multiplied.  (With -m in the product x.w + b - m is rounded in other places than m was: 64 apart at scores of 1e9, and exp of
// that is no probability.)  The same factor serves gradients that differ from pixel to pixel.
//
// 32-bit inputs: every operand is split into three bf16 pieces (8 + 8 + 8 bits of mantissa) and six of the nine piece
// products are kept; what is dropped is below 2^-24 of a product.  G is split the same way in registers.
//
// What bounds it, per 128 x 128 scores: 1024 clocks for the exponentials (16 per clock and SM) and 4 C clocks for a product,
// so the exponentials up to about 128 channels (forward; two products backward), the products beyond.  Measured on 148 SMs, whole
// passes with preparation, joining and reduction (events, L2 flushed):
//   1657600 pixels x 64 channels x 1024 labels, bf16: forward 0.62 ms (1.7 times the exponentials alone, 0.37 ms), both gradients
//     1.53 ms (2.1 times); the rest is waiting between the two products and the label terms
//   66560 x 256 x 32771, bf16: forward 1.02 ms (1.1 PFLOP/s), gradients 3.8 ms (1.2 PFLOP/s of the 4.5 TFLOP done): the first
//     product reads 128 bytes of operands a clock, all that shared memory gives, while TMA writes the next block there
//   1657600 x 32 x 512, 32 bits: forward 0.50 ms, gradients 1.41 ms: the split of G in three and six products for one; splitting the
//     features into pieces is 0.1 ms of each pass
// Gradients of wide features: an item gives 256 output channels (64 in 32 bits) and forms the scores anew, and beyond 8 chunks of
// pieces A is fetched with every block of B.  66560 pixels x 4096 labels, a step: bf16 0.69 ms at 256 channels, 2.1 at 512, 9.3 at
// 1024; 32 bits 0.86 at 64, 2.2 at 128, 7.4 at 256, 26 at 512, 108 at 1024 (products with the scores in memory: 18 and 31 ms).
//
// All waits are bounded.  A warp whose wait runs out says so in shared memory (fail) before anything else it does.  From then on
// barriers may complete for work that is not whole: the MMA warp goes through its motions to the end of its item.  So the
// warpgroups look at fail behind the last wait that an output hangs on, and write NaN; one whose own wait ran out arrives
// nowhere any more, so that no buffer of it is used again.  A loss or gradient is right or NaN (a forward pass that gave up makes
// its backward pass NaN).  Copies in flight land before the CTA leaves, and its TMEM is freed.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>
#include <atomic>
#include <type_traits>
#include "rgs_cuda_common.cuh"
#include "rgs_field_math.h"

#define LT 128                      // rows of a tile of either matrix
#define LROOM (25 * 8192)           // bytes of staged tiles: 128 rows x 64 (or 32) channels bf16 each
#define LSTAGES 13                  // most stages of the ring
#define LE 4096                     // bytes of a tile of the extra channels, 128 x 16 bf16
#define LESLOTS 3                   // such tiles of B (of A there are two)
#define LKSLOTS 3                   // staged blocks of what dW needs of 128 pixels: label, g, factor
#define LKBYTES (3 * LT * 4)
#define LTHREADS 576                // warp 0 TMA, warp 1 MMA, warps 2-17 four warpgroups on the scores
#define LWAIT (1u << 20)
#define LOG2E 1.4426950408889634f

enum { LF_DIRTY = 1,   // a pixel without a label has a score that is not finite (its features, or a row of the weight)
       LF_LARGE = 2 }; // a largest score above 2^10: m and log z are not added up, and m stays out of the product

struct LabelArgs {
    int64_t n, v;
    int c, nk;                       // channels, chunks of 64 (32) channels
    int noc, nrange;                 // chunks of output channels per item, ranges of them
    int a_slots;                     // blocks of A that stay in shared memory (0: A goes through the ring)
    int whole, stages;               // stages of B are kept for both products; stages of the ring
    int nbuf, nob;                   // score and output buffers in TMEM
    int nmx, nmw;                    // tiles of 128 pixels, of 128 labels
    int nsx, nsw;                    // partial sums of the walk over labels (forward, dX) and over pixels (dW)
    int subx, subw, sub;             // pieces added into a partial sum, one a launch; those of this launch
    int perx, restx, perw, restw;    // tiles of a piece: per, one more in the first rest pieces
    unsigned items_x, items_w;
    const float* kn;                 // (nmx, 3, 128) per pixel: label (bits; -1: none), g, factor; backward only
    const float* lse;                // (2, n) m and log z
    const float* gs;                 // g of all pixels where they share it
    int per_row;                     // a gradient to a pixel
    const void* labels; int label_bytes;
    const float* flags;              // [1]: LF_ bits
    float* pm; float* ps; float* at; // forward: (4 nsx, n) partial maximum and sum, (n) score of the label
    float* part_x; float* part_w;    // (nsx, nmx*128, cq), (nsw, nmw*128, cq) when split
    float* part_b;                   // (4 nsw, nmw*128)
    int cq;
    void* dx; void* dw; int dtype;
    uint32_t wait, loads;            // limits: tries of a wait; stages that the producer of a CTA fills before it gives up
};

// ---------------------------------------------------------------------------------------------------------------------
// PTX
// ---------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

__device__ __forceinline__ bool lb_try(unsigned long long* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(rgs_smem_addr(bar)), "r"(parity) : "memory");
    return ok;
}
__device__ __forceinline__ bool lb_wait(unsigned long long* bar, uint32_t parity, volatile int* fail, uint32_t limit) {
    for (uint32_t it = 0; it < limit; ++it) {
        if (lb_try(bar, parity)) return true;
        if ((it & 15u) == 15u && *fail) break;
    }
    *fail = 1;
    __threadfence_block();  // seen before what this warp issues next
    return false;
}
// the same by a whole warp, with one answer for all of it
__device__ __forceinline__ bool lb_wait_warp(unsigned long long* bar, uint32_t parity, volatile int* fail, uint32_t limit) {
    return __all_sync(0xffffffffu, lb_wait(bar, parity, fail, limit));
}
// The MMA warp's.  It goes on either way: every answer that its loop looks at costs (votes 3 % of a pass, a lane that gives up
// issuing 20 to 50 %), and so does anything between a try that succeeds and the return (codebook forward 1033 -> 1093 us).
__device__ __noinline__ void lb_wait_slow(unsigned long long* bar, uint32_t parity, volatile int* fail, uint32_t limit) {
    if (*fail) {
        __threadfence_block();
        return;
    }
    for (uint32_t it = 0; it < limit; ++it) {
        if (lb_try(bar, parity)) return;
        if ((it & 15u) == 15u && *fail) return;
    }
    *fail = 1;
    __threadfence_block();  // seen before what this warp issues next
}
__device__ __forceinline__ void lb_wait_quiet(unsigned long long* bar, uint32_t parity, volatile int* fail, uint32_t limit) {
    if (!lb_try(bar, parity)) lb_wait_slow(bar, parity, fail, limit);
    __syncwarp();
}
// all roles of a CTA have come to their end
__device__ __forceinline__ void lb_end_of_role() {
    __syncwarp();
    asm volatile("barrier.sync 1, %0;" ::"n"(LTHREADS) : "memory");
}
// One lane of a converged warp.  The producer and MMA warps run their loops with all lanes and let this one issue (a single
// thread in the loop: codebook forward 2.53 instead of 1.99 ms).  Asked once: to elect anew costs more than a product.
__device__ __forceinline__ bool lb_elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void lb_tma(void* dst, const CUtensorMap* map, int x, int y, int z, unsigned long long* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
                 "r"(rgs_smem_addr(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(rgs_smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void lb_commit(uint32_t lead, unsigned long long* bar) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(rgs_smem_addr(bar)), "r"(lead) : "memory");
}
// Shared-memory descriptors: rows of KC channels under the swizzle of their length (128, 64 or 32 bytes), eight rows to a
// pattern; both strides are that of the pattern, so a tile reads as K-major rows or as steps of K.  The low word holds the
// address (in 16 bytes), the high word never changes: the products below take the low words alone.
template <int KC> constexpr uint32_t lb_desc_lo = (uint32_t)KC << 16;
template <int KC> constexpr uint32_t lb_desc_hi = (uint32_t)KC | (1u << 14) | ((KC == 64 ? 2u : KC == 32 ? 4u : 6u) << 29);

template <int KC>
__device__ __forceinline__ void lb_mma_ss(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\tmov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)acc), "n"(lb_desc_hi<KC>), "r"(lead) : "memory");
}
template <int KC>
__device__ __forceinline__ void lb_mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\tmov.b64 y, {%2, %5};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)acc), "n"(lb_desc_hi<KC>), "r"(lead) : "memory");
}
#define LB_R16(r, o) "+r"(r[o]), "+r"(r[o + 1]), "+r"(r[o + 2]), "+r"(r[o + 3]), "+r"(r[o + 4]), "+r"(r[o + 5]), "+r"(r[o + 6]), "+r"(r[o + 7]), \
    "+r"(r[o + 8]), "+r"(r[o + 9]), "+r"(r[o + 10]), "+r"(r[o + 11]), "+r"(r[o + 12]), "+r"(r[o + 13]), "+r"(r[o + 14]), "+r"(r[o + 15])
#define LB_O16(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7]), \
    "=r"(r[o + 8]), "=r"(r[o + 9]), "=r"(r[o + 10]), "=r"(r[o + 11]), "=r"(r[o + 12]), "=r"(r[o + 13]), "=r"(r[o + 14]), "=r"(r[o + 15])

__device__ __forceinline__ void tm_ld32(uint32_t a, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
                 "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : LB_O16(r, 0), LB_O16(r, 16) : "r"(a) : "memory");
}
__device__ __forceinline__ void tm_wait_ld32(uint32_t (&r)[32]) {  // the registers pass through, so nothing reads them before
    asm volatile("tcgen05.wait::ld.sync.aligned;" : LB_R16(r, 0), LB_R16(r, 16)::"memory");
}
__device__ __forceinline__ void tm_ld16(uint32_t a, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : LB_O16(r, 0) : "r"(a) : "memory");
}
__device__ __forceinline__ void tm_wait_ld16(uint32_t (&r)[16]) { asm volatile("tcgen05.wait::ld.sync.aligned;" : LB_R16(r, 0)::"memory"); }
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void tm_st8(uint32_t a, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(a) : "memory");
}
// two floats to a register pair: one instruction for both
typedef unsigned long long f2;
__device__ __forceinline__ f2 mk2(float a, float b) { f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ f2 mk2u(uint32_t a, uint32_t b) { f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ void un2(f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ f2 add2(f2 a, f2 b) { f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) { f2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
// v -= g where a == b.  Written out: the compiler turns a chain of such conditions over an array into an index, and the
// array into local memory (the backward pass then took twice as long).
__device__ __forceinline__ void sub_if(float& v, float g, int a, int b) {
    asm("{\n\t.reg .pred p;\n\tsetp.eq.s32 p, %2, %3;\n\t@p sub.f32 %0, %0, %1;\n\t}" : "+f"(v) : "f"(g), "r"(a), "r"(b));
}
__device__ __forceinline__ float bf_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// ---------------------------------------------------------------------------------------------------------------------
// items of the persistent loop: rows of A, range of output channels, piece of the walk over B
// ---------------------------------------------------------------------------------------------------------------------
struct LabelItem { int dw, m, oc0, noc, split, j0, j1; };

// single threads run this between products: no division where there is nothing to divide
template <bool GRAD>
__device__ __forceinline__ LabelItem lb_item(const LabelArgs& a, unsigned i) {
    LabelItem it;
    it.dw = i >= a.items_x;
    if (it.dw) i -= a.items_x;
    const unsigned nm = it.dw ? a.nmw : a.nmx, base = it.dw ? a.perw : a.perx, rest = it.dw ? a.restw : a.restx;
    unsigned q = 0;
    if (i >= nm) { q = i / nm; i -= q * nm; }
    it.m = (int)i;
    unsigned range = 0;
    if (a.nrange > 1) { range = q % (unsigned)a.nrange; q /= (unsigned)a.nrange; }
    it.oc0 = (int)range * a.noc;
    it.noc = min(a.noc, a.nk - it.oc0);
    it.split = (int)q;
    if (GRAD) q = q * (unsigned)(it.dw ? a.subw : a.subx) + (unsigned)a.sub;  // its piece
    it.j0 = (int)(q * base + min(q, rest));  // the first `rest` pieces are one tile longer
    it.j1 = it.j0 + (int)base + (q < rest);
    return it;
}

// place in a ring of buffers and the parity of its current use
struct LabelCursor {
    uint32_t slot = 0, phase = 0;
    __device__ __forceinline__ void next(uint32_t size) {
        if (++slot == size) { slot = 0; phase ^= 1; }
    }
};

// sixteen channels of a row of the output, rounded to its type; vector stores where rows keep their alignment
// (add: on top of what is there, 32 bits only)
__device__ __forceinline__ void lb_store16(void* out, int64_t r, int c, int channels, int dtype, bool add, float (&f)[16]) {
    if (dtype == RGS_BF16) {
        __nv_bfloat16* p = static_cast<__nv_bfloat16*>(out) + r * channels + c;
        if ((channels & 7) == 0) {
#pragma unroll
            for (int q = 0; q < 16; q += 8)
                if (c + q < channels)
                    *reinterpret_cast<uint4*>(p + q) = make_uint4(bf16x2(f[q], f[q + 1]), bf16x2(f[q + 2], f[q + 3]), bf16x2(f[q + 4], f[q + 5]), bf16x2(f[q + 6], f[q + 7]));
        } else {
#pragma unroll
            for (int q = 0; q < 16; ++q)
                if (c + q < channels) p[q] = __float2bfloat16_rn(f[q]);
        }
    } else {
        float* p = static_cast<float*>(out) + r * channels + c;
        if (add)
#pragma unroll
            for (int q = 0; q < 16; ++q) f[q] += c + q < channels ? p[q] : 0.f;
        if ((channels & 3) == 0) {
#pragma unroll
            for (int q = 0; q < 16; q += 4)
                if (c + q < channels) *reinterpret_cast<float4*>(p + q) = make_float4(f[q], f[q + 1], f[q + 2], f[q + 3]);
        } else {
#pragma unroll
            for (int q = 0; q < 16; ++q)
                if (c + q < channels) p[q] = f[q];
        }
    }
}

struct LabelShared {
    unsigned long long full[LSTAGES], empty[LSTAGES], a_full[2], a_empty[2], k_full[LKSLOTS], k_empty[LKSLOTS];
    unsigned long long ea_full[2], ea_empty[2], e_empty[LESLOTS];
    unsigned long long s_full[4], s_done[4], o_full[2], o_free[2], drain;
    uint32_t tmem;
    int fail;
};
#define LSMEM (1024 + LROOM + (2 + LESLOTS) * LE + LKSLOTS * LKBYTES + (int)sizeof(LabelShared))
static_assert(LSMEM <= 232448, "shared memory of an SM");

// WHOLE: A stays in shared memory and, backward, so do the stages of B between the two products
template <int P, bool GRAD, int KC, int CS, bool WHOLE>
__global__ void __launch_bounds__(LTHREADS, 1) rgs_label_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                                   const __grid_constant__ CUtensorMap map_ex, const __grid_constant__ CUtensorMap map_ew,
                                                                   const __grid_constant__ LabelArgs a) {
    constexpr int SB = GRAD && P == 3 ? 192 : 128;  // TMEM columns of a score buffer (scores; over them G, its third piece behind)
    // 32-bit outputs are summed in two buffers: the leading products, eight steps to a tile, and the small ones.  The tensor
    // core truncates where it adds (2^-27 of the sum a step, measured), which the 40 other steps would do to the large sum.
    constexpr int LO = KC;                        // columns between the two
    const int OUT = a.nbuf * SB;                  // first column of the outputs
    constexpr int OB = 64;                        // columns of an output buffer when there are two
    constexpr int COMBOS = P == 1 ? 1 : 6;
    // smallest products first; the piece of X first where S = X W^T, and the same pairs in the same order where S = W X^T
    constexpr int CA[6] = {P == 1 ? 0 : 2, 0, 1, 1, 0, 0}, CB[6] = {0, 2, 1, 0, 1, 0};
    constexpr int TB = KC * 2 * LT;               // bytes of a staged tile
    extern __shared__ unsigned char raw[];
    unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    unsigned char *ea_tiles = tiles + LROOM, *e_tiles = ea_tiles + 2 * LE;
    float* kbuf = reinterpret_cast<float*>(e_tiles + LESLOTS * LE);
    LabelShared* sh = reinterpret_cast<LabelShared*>(e_tiles + LESLOTS * LE + LKSLOTS * LKBYTES);
    volatile int* fail = &sh->fail;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t na = P * a.nk;                 // tiles of one block of 128 rows, chunk by chunk, its pieces together
    unsigned char* ring = tiles + a.a_slots * na * TB;
    constexpr uint32_t stage = CS * P * TB;       // bytes of a stage of the ring: CS chunks of A or B, their pieces
    const int nst = GRAD && WHOLE && CS != 2 ? 1 : a.nk / CS;  // stages of a block of 128 rows

    if (warp == 0) {
        if (lane == 0) {
            for (int i = 0; i < LSTAGES; ++i) { rgs_mbar_init(&sh->full[i], 1); rgs_mbar_init(&sh->empty[i], 1); }
            for (int i = 0; i < 2; ++i) {
                rgs_mbar_init(&sh->a_full[i], 1); rgs_mbar_init(&sh->a_empty[i], 1);
                rgs_mbar_init(&sh->ea_full[i], 1); rgs_mbar_init(&sh->ea_empty[i], 1);
                rgs_mbar_init(&sh->o_full[i], 1); rgs_mbar_init(&sh->o_free[i], 512);
            }
            for (int i = 0; i < 4; ++i) { rgs_mbar_init(&sh->s_full[i], 1); rgs_mbar_init(&sh->s_done[i], 256); }
            for (int i = 0; i < LKSLOTS; ++i) { rgs_mbar_init(&sh->k_full[i], 1); rgs_mbar_init(&sh->k_empty[i], 256); }
            for (int i = 0; i < LESLOTS; ++i) rgs_mbar_init(&sh->e_empty[i], 1);
            rgs_mbar_init(&sh->drain, 1);
            sh->fail = 0;
            rgs_fence_mbar_init();
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(rgs_smem_addr(&sh->tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = sh->tmem;
    const unsigned items = a.items_x + a.items_w;

    if (warp == 0) {
        // ------------------------------------------------------------------------------------------------ TMA
        const bool lead = lb_elect();
        LabelCursor rc, ac, kc, eac, ec;
        uint32_t loads = 0, labels = 0;
        bool ok = true;
        auto load = [&](const CUtensorMap* map, int k, int row, const CUtensorMap* extra) {
            if (ok && loads >= a.loads) { *fail = 1; ok = false; }
            ok = ok && lb_wait_warp(&sh->empty[rc.slot], rc.phase ^ 1, fail, a.wait);
            if (!ok) return;
            if (lead) {
                unsigned char* dst = ring + rc.slot * stage;
                rgs_mbar_expect_tx(&sh->full[rc.slot], extra ? stage + LE : stage);
                if (extra) lb_tma(e_tiles + ec.slot * LE, extra, 0, row * LT, 0, &sh->full[rc.slot]);
#pragma unroll
                for (int u = 0; u < CS * P; ++u) lb_tma(dst + u * TB, map, (k * CS + u / P) * KC, row * LT, u % P, &sh->full[rc.slot]);
            }
            rc.next(a.stages);
            ++loads;
        };
        // the order of stages is the order in which the MMA warp takes them: S(0), S(1), O(0), S(2), O(1), ...; with B kept
        // for both products O takes nothing from the ring
        bool have_prev = false;
        int prev_j = 0, prev_oc0 = 0, prev_noc = 0, prev_dw = 0;
        auto out_tiles = [&]() {
            if (!GRAD || WHOLE || !have_prev) return;
            for (int oc = 0; oc < prev_noc && ok; oc += CS) load(prev_dw ? &map_x : &map_w, (prev_oc0 + oc) / CS, prev_j, nullptr);
        };
        for (unsigned i = blockIdx.x; i < items && ok; i += gridDim.x) {
            const LabelItem it = lb_item<GRAD>(a, i);
            const CUtensorMap *ma = it.dw ? &map_w : &map_x, *mb = it.dw ? &map_x : &map_w;
            // (forward: the pixels' extra channels are the same for all, one tile of them)
            ok = lb_wait_warp(&sh->ea_empty[eac.slot], eac.phase ^ 1, fail, a.wait);
            if (!ok) break;
            if (lead) {
                rgs_mbar_expect_tx(&sh->ea_full[eac.slot], LE);
                lb_tma(ea_tiles + eac.slot * LE, it.dw ? &map_ew : &map_ex, 0, GRAD ? it.m * LT : 0, 0, &sh->ea_full[eac.slot]);
            }
            eac.next(2);
            if (WHOLE || a.a_slots) {
                ok = lb_wait_warp(&sh->a_empty[ac.slot], ac.phase ^ 1, fail, a.wait);
                if (!ok) break;
                if (lead) {
                    unsigned char* dst = tiles + ac.slot * na * TB;
                    rgs_mbar_expect_tx(&sh->a_full[ac.slot], na * TB);
                    for (int k = 0; k < a.nk; ++k)
#pragma unroll
                        for (int p = 0; p < P; ++p) lb_tma(dst + (k * P + p) * TB, ma, k * KC, it.m * LT, p, &sh->a_full[ac.slot]);
                }
                ac.next(a.a_slots);
            }
            for (int j = it.j0; j < it.j1 && ok; ++j) {
                ok = lb_wait_warp(&sh->e_empty[ec.slot], ec.phase ^ 1, fail, a.wait);
                if (!ok) break;
                if (GRAD && it.dw) {
                    ok = lb_wait_warp(&sh->k_empty[kc.slot], kc.phase ^ 1, fail, a.wait);
                    if (!ok) break;
                    if (lead) {
                        rgs_mbar_expect_tx(&sh->k_full[kc.slot], LKBYTES);
                        rgs_bulk_g2s(kbuf + kc.slot * (LKBYTES / 4), a.kn + (size_t)j * (3 * LT), LKBYTES, &sh->k_full[kc.slot]);
                    }
                    kc.next(LKSLOTS);
                    ++labels;
                }
                for (int k = 0; k < nst && ok; ++k) {
                    if (!WHOLE && !a.a_slots) load(ma, k, it.m, nullptr);
                    load(mb, k, j, k == 0 ? (it.dw ? &map_ex : &map_ew) : nullptr);  // the extra channels come with the first stage
                }
                ec.next(LESLOTS);
                out_tiles();
                have_prev = true; prev_j = j; prev_oc0 = it.oc0; prev_noc = it.noc; prev_dw = it.dw;
            }
        }
        if (ok) out_tiles();
        lb_end_of_role();
        if (*fail) {  // copies still in flight land before the CTA leaves (all were consumed unless a wait ran out)
            const uint32_t live = loads < (uint32_t)a.stages ? loads : a.stages;
            for (uint32_t k = 0; k < live; ++k) {
                if (rc.slot == 0) { rc.slot = a.stages; rc.phase ^= 1; }
                --rc.slot;
                rgs_mbar_wait(&sh->full[rc.slot], rc.phase, 1u << 12);
            }
            for (uint32_t k = 0; k < LKSLOTS && k < labels; ++k) {
                if (kc.slot == 0) { kc.slot = LKSLOTS; kc.phase ^= 1; }
                --kc.slot;
                rgs_mbar_wait(&sh->k_full[kc.slot], kc.phase, 1u << 12);
            }
            for (int k = 0; k < 2; ++k) {
                if (eac.slot == 0) { eac.slot = 2; eac.phase ^= 1; }
                --eac.slot;
                rgs_mbar_wait(&sh->ea_full[eac.slot], eac.phase, 1u << 12);
            }
            for (int k = 0; k < a.a_slots; ++k) {
                if (ac.slot == 0) { ac.slot = a.a_slots; ac.phase ^= 1; }
                --ac.slot;
                rgs_mbar_wait(&sh->a_full[ac.slot], ac.phase, 1u << 12);
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------------------------------------ MMA
        const uint32_t lead = lb_elect();
        // one product after the other by predicate (several chunks to a stage), or a branch around all of them: each the
        // faster one (256 channels backward 4.09 -> 3.85 ms with predicates, 32 channels in 32 bits 1.74 -> 1.86 ms)
        const uint32_t issue = P == 3 || CS == 1 ? 1u : lead;
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(LT >> 4) << 24);
        LabelCursor rc, ac, oc_, gc, sc, pc, eac, ec;        // ring, A, outputs; oldest stage not given back; S, its G; extra channels
        const uint32_t ea16 = lb_desc_lo<16> + (rgs_smem_addr(ea_tiles) >> 4), e16 = lb_desc_lo<16> + (rgs_smem_addr(e_tiles) >> 4);
        const uint32_t dlo = lb_desc_lo<KC>, ring16 = dlo + (rgs_smem_addr(ring) >> 4), tiles16 = dlo + (rgs_smem_addr(tiles) >> 4);
        constexpr uint32_t T16 = TB >> 4, stage16 = stage >> 4;
        auto take = [&]() {
            lb_wait_quiet(&sh->full[rc.slot], rc.phase, fail, a.wait);
            const uint32_t d = ring16 + rc.slot * stage16;
            rc.next(a.stages);
            return d;
        };
        // the chunks of a stage; channels behind the last one are zeros in shared memory
        auto stage_s = [&](uint32_t d, uint32_t at, uint32_t bt, bool more, bool swap) {
            // pairs (2,0) (0,2) (1,1) (1,0) (0,1) (0,0) of pieces of A and B, or with their members swapped
            const uint32_t a2 = swap ? 0 : 2 * T16, a1 = swap ? 0 : T16;
            const uint32_t oa[6] = {P == 1 ? 0 : a2, 2 * T16 - a2, T16, a1, T16 - a1, 0}, ob[6] = {P == 1 ? 0 : 2 * T16 - a2, a2, T16, T16 - a1, a1, 0};
#pragma unroll
            for (int k = 0; k < CS; ++k)
#pragma unroll
                for (int q = 0; q < COMBOS; ++q)
#pragma unroll
                    for (int ks = 0; ks < KC / 16; ++ks)
                        lb_mma_ss<KC>(issue, d, at + k * P * T16 + oa[q] + ks * 2, bt + k * P * T16 + ob[q] + ks * 2, idesc | ((LT >> 3) << 17), k || q || ks ? true : more);
        };
        auto issue_s = [&](const LabelItem& it, int j) {
            const uint32_t d = tmem + sc.slot * SB;
            // forward: the scores there before have been read; backward: the product with their G was issued before, and runs before
            if (!GRAD) lb_wait_quiet(&sh->s_done[sc.slot], sc.phase ^ 1, fail, a.wait);
            if (j == it.j0) {
                lb_wait_quiet(&sh->ea_full[eac.slot], eac.phase, fail, a.wait);
                if (WHOLE || a.a_slots) lb_wait_quiet(&sh->a_full[ac.slot], ac.phase, fail, a.wait);
            }
            const uint32_t abase = tiles16 + ac.slot * (na * T16);
            const bool last = j == it.j1 - 1;
            for (int k = 0; k < nst; ++k) {
                const uint32_t at = WHOLE || a.a_slots ? abase + k * stage16 : take();
                const uint32_t bt = take();
                const uint32_t g0 = gc.slot;
                if (!GRAD || !WHOLE) {
                    gc.next(a.stages);
                    if (!WHOLE && !a.a_slots) gc.next(a.stages);
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if ((P == 1 && CS > 1) || lead) {
                    stage_s(d, at, bt, k != 0, GRAD && it.dw);
                    if (!GRAD || !WHOLE) {
                        lb_commit(issue, &sh->empty[g0]);
                        if (!WHOLE && !a.a_slots) lb_commit(issue, &sh->empty[g0 + 1 == (uint32_t)a.stages ? 0 : g0 + 1]);
                    }
                    if (k == nst - 1) {
                        // last: where b is huge and -(m + log z) cancels it, what is small beside them is gone, as it is from the scores
                        lb_mma_ss<16>(issue, d, ea16 + eac.slot * (LE >> 4), e16 + ec.slot * (LE >> 4), idesc | ((LT >> 3) << 17), true);
                        lb_commit(issue, &sh->s_full[sc.slot]);
                        lb_commit(issue, &sh->e_empty[ec.slot]);
                        if (last) {
                            lb_commit(issue, &sh->ea_empty[eac.slot]);
                            if (WHOLE || a.a_slots) lb_commit(issue, &sh->a_empty[ac.slot]);
                        }
                    }
                }
                __syncwarp();
            }
            sc.next(a.nbuf);
            ec.next(LESLOTS);
            if (last) {
                eac.next(2);
                if (WHOLE || a.a_slots) ac.next(a.a_slots);
            }
        };
        // G B; B as the K x N operand with its channels as N, 16 rows a step
        auto stage_o = [&](uint32_t s, uint32_t o, uint32_t bt, bool more) {
            // 16 bits: the chunks of a stage lie a tile apart and are one operand of CS KC columns, so that G is read once for them
            constexpr int W = P == 1 ? CS * KC : KC;
            constexpr uint32_t id = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(W >> 3) << 17) | ((uint32_t)(LT >> 4) << 24);
            if (P == 1) bt += (T16 - KC) << 16;
#pragma unroll
            for (int q = 0; q < COMBOS; ++q)
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    // 16 columns of G are 8 words: the first two pieces lie over the 16 scores, the third behind all
                    const uint32_t g = CA[q] == 2 ? s + 128 + ks * 8 : s + ks * 16 + CA[q] * 8;
                    const bool first = ks == 0 && (q == 0 || q == COMBOS - 1);
                    lb_mma_ts<KC>(issue, o + (q < COMBOS - 1 ? LO : 0), g, bt + CB[q] * T16 + ks * (KC * 2), id, first ? more : true);
                }
        };
        auto issue_o = [&](const LabelItem& it, int j) {
            lb_wait_quiet(&sh->s_done[pc.slot], pc.phase, fail, a.wait);
            if (j == it.j0) lb_wait_quiet(&sh->o_free[oc_.slot], oc_.phase ^ 1, fail, a.wait);
            const uint32_t s = tmem + pc.slot * SB, o = tmem + OUT + oc_.slot * OB;
            pc.next(a.nbuf);
            const bool last = j == it.j1 - 1;
            for (int oc = 0; oc < it.noc; oc += CS) {
                // kept stages: those that S took are the oldest ones still held (all chunks are output channels then)
                const uint32_t bt = WHOLE ? ring16 + gc.slot * stage16 : take();
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if ((P == 1 && CS > 1) || lead) {
                    stage_o(s, o + oc * KC, bt, j != it.j0);
                    lb_commit(issue, &sh->empty[gc.slot]);
                    if (last && oc + CS == it.noc) lb_commit(issue, &sh->o_full[oc_.slot]);
                }
                __syncwarp();
                gc.next(a.stages);
            }
            if (last) oc_.next(a.nob);
        };
        // walks over the score tiles: S runs nbuf - 1 tiles ahead of G B, so that a warpgroup finds its next scores ready
        unsigned si = blockIdx.x, oi = blockIdx.x;
        LabelItem is, io;
        int sj = 0, oj = 0;
        if (si < items) { is = io = lb_item<GRAD>(a, si); sj = oj = is.j0; }
        auto step_s = [&]() {
            issue_s(is, sj);
            if (++sj == is.j1) {
                si += gridDim.x;
                if (si < items) { is = lb_item<GRAD>(a, si); sj = is.j0; }
            }
        };
        auto failed = [&]() { return __any_sync(0xffffffffu, *fail); };
        if (GRAD) {
            for (int l = 1; l < a.nbuf; ++l)
                if (si < items) step_s();
            while (oi < items) {
                if (si < items) step_s();
                issue_o(io, oj);
                if (++oj == io.j1) {
                    if (failed()) break;
                    oi += gridDim.x;
                    if (oi < items) { io = lb_item<GRAD>(a, oi); oj = io.j0; }
                }
            }
        } else {
            while (si < items) {
                const unsigned i = si;
                step_s();
                if (si != i && failed()) break;
            }
        }
        lb_commit(lead, &sh->drain);  // what was issued is done before TMEM goes
        __syncwarp();
        rgs_mbar_wait(&sh->drain, 0, LWAIT);
        lb_end_of_role();
    } else {
        // ------------------------------------------------------------------------------------------------ scores
        const int wg = (warp - 2) >> 2;                      // warpgroup: score tiles t with t % 2 == wg % 2,
        const int half = (wg >> 1) * 64;                     // 64 of their columns
        const int wrow = (warp & 3) * 32, row = wrow + lane; // row of A
        const uint32_t lanes = (uint32_t)wrow << 16;
        const float nan = __int_as_float(0x7fc00000);
        const f2 log2e = mk2(LOG2E, LOG2E);
        uint32_t t = 0, kept = 0;                            // score tiles seen; ring stage where the B block of tile t begins
        LabelCursor oc_, sc, kc;
        bool dead = false;
        const int flags = GRAD ? (int)a.flags[1] : 0;
        const bool large = flags & LF_LARGE, scaled = GRAD && (large || a.per_row);  // factors to dW's columns
        const float gshare = GRAD && !scaled ? *a.gs : 1.f;
        unsigned out_i = blockIdx.x;                         // next item whose output this warpgroup writes
        // what a row of A brings to an item, fetched an item ahead: from memory at its start it would cost as much as a score tile
        auto row_label = [&](unsigned i) -> int {
            if (i >= items) return -1;
            const LabelItem it = lb_item<GRAD>(a, i);
            if (it.dw) return 0;
            if (GRAD) return __float_as_int(a.kn[(size_t)it.m * (3 * LT) + row]);
            const int64_t r = (int64_t)it.m * LT + row;
            return r < a.n ? (int)rgs_label(a.labels, r, a.label_bytes, a.v) : -1;
        };
        auto row_scale = [&](unsigned i) -> float {
            if (!GRAD || i >= items) return 1.f;
            const LabelItem it = lb_item<GRAD>(a, i);
            return it.dw ? gshare : a.kn[(size_t)it.m * (3 * LT) + LT + row];
        };
        auto write_out = [&](unsigned i, float scale, int label) {
            const LabelItem it = lb_item<GRAD>(a, i);
            if (!dead) dead = __any_sync(0xffffffffu, !lb_wait(&sh->o_full[oc_.slot], oc_.phase, fail, a.wait));
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t o = tmem + lanes + OUT + oc_.slot * OB;
            const int64_t r = (int64_t)it.m * LT + row, rows = it.dw ? a.v : a.n;
            float* part = it.dw ? a.part_w : a.part_x;
            for (int c0 = wg * 16; c0 < it.noc * KC; c0 += 64) {
                const int c = it.oc0 * KC + c0;
                if (c >= a.c) break;
                uint32_t u[16], lo[16];
                tm_ld16(o + c0, u);
                if (P == 3) {
                    tm_ld16(o + LO + c0, lo);
                    tm_wait_ld16(lo);
                }
                tm_wait_ld16(u);
                const bool lost = dead || *fail;  // behind the loads: a buffer is given to other work only after fail is set
                if (r < rows && (!it.dw || a.dw)) {
                    float f[16];
#pragma unroll
                    for (int q = 0; q < 16; ++q) f[q] = lost ? nan : P == 3 ? __uint_as_float(u[q]) + __uint_as_float(lo[q]) : __uint_as_float(u[q]);
                    if (part) {
                        if (it.dw)
#pragma unroll
                            for (int q = 0; q < 16; ++q) f[q] *= scale;
                        float* p = part + ((int64_t)it.split * (it.dw ? a.nmw : a.nmx) * LT + r) * a.cq + c;
                        if (a.sub)
#pragma unroll
                            for (int q = 0; q < 16; ++q) f[q] += p[q];
#pragma unroll
                        for (int q = 0; q < 16; q += 4) *reinterpret_cast<float4*>(p + q) = make_float4(f[q], f[q + 1], f[q + 2], f[q + 3]);
                    } else {
#pragma unroll
                        for (int q = 0; q < 16; ++q) f[q] = label < 0 ? 0.f : f[q] * scale;
                        lb_store16(it.dw ? a.dw : a.dx, r, c, a.c, a.dtype, a.sub != 0, f);
                    }
                }
                __syncwarp();
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            if (!dead) rgs_mbar_arrive(&sh->o_free[oc_.slot]);
            oc_.next(a.nob);
        };
        const bool dirty = GRAD && (flags & LF_DIRTY);
        const bool rare = dirty || scaled;
        int next_label = row_label(blockIdx.x), out_label = 0;
        float next_scale = row_scale(blockIdx.x), out_scale = 1.f;  // out_: of the first item whose output is not written
        for (unsigned i = blockIdx.x; i < items; i += gridDim.x) {
            const LabelItem it = lb_item<GRAD>(a, i);
            const int64_t r = (int64_t)it.m * LT + row;
            const int label = next_label;
            const float scale = next_scale;
            next_label = row_label(i + gridDim.x);
            next_scale = row_scale(i + gridDim.x);
            if (out_i == i) { out_label = label; out_scale = scale; }
            const int64_t y = it.dw ? -1 : label;
            float m = -INFINITY, sum = 0.f;
            for (int j = it.j0; j < it.j1; ++j, ++t) {
                const uint32_t bstage = kept, buf = sc.slot, parity = sc.phase;
                if (GRAD && P == 1 && (kept += nst) >= (uint32_t)a.stages) kept -= a.stages;
                const uint32_t kslot = kc.slot, kparity = kc.phase;
                sc.next(a.nbuf);
                if (GRAD && it.dw) kc.next(LKSLOTS);
                if ((int)(t & 1) != (wg & 1)) continue;
                const uint32_t s = tmem + lanes + buf * SB + half;
                if (!dead) {  // the whole warp goes on or none of it: TMEM accesses are warp-wide
                    dead = !lb_wait(&sh->s_full[buf], parity, fail, a.wait) || (GRAD && it.dw && !lb_wait(&sh->k_full[kslot], kparity, fail, a.wait));
                    dead = __any_sync(0xffffffffu, dead);
                }
                if (dead) continue;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const float* kb = kbuf + kslot * (LKBYTES / 4) + half;
                const int64_t yt = y - (int64_t)j * LT - half;
                const int yl = y >= 0 && yt >= 0 && yt < 64 ? (int)yt : -1;  // the row's label among these columns
                if (!GRAD) {
                    uint32_t u[2][32];
                    tm_ld32(s, u[0]);
                    tm_ld32(s + 32, u[1]);
                    tm_wait_ld32(u[0]);
                    tm_wait_ld32(u[1]);
                    // all scores are in registers: the buffer is free for the product after the next
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    rgs_mbar_arrive(&sh->s_done[buf]);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float f[32];
#pragma unroll
                        for (int q = 0; q < 32; ++q) f[q] = __uint_as_float(u[h][q]);
                        float top[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            top[q] = fmaxf(f[q], f[q + 4]);
#pragma unroll
                            for (int e = 8; e < 32; e += 8) top[q] = fmaxf(top[q], fmaxf(f[q + e], f[q + e + 4]));
                        }
                        if ((yl >> 5) == h) {  // one of the 32 by the bits of its index
                            float z[16];
#pragma unroll
                            for (int q = 0; q < 16; ++q) z[q] = yl & 16 ? f[q + 16] : f[q];
#pragma unroll
                            for (int w = 8; w > 0; w >>= 1)
#pragma unroll
                                for (int q = 0; q < w; ++q) z[q] = yl & w ? z[q + w] : z[q];
                            a.at[r] = z[0];
                        }
                        const float best = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
                        const float ref = best == -INFINITY ? 0.f : best;
                        const f2 minus = mk2(-ref, -ref);
                        f2 acc[2] = {0ull, 0ull};
#pragma unroll
                        for (int q = 0; q < 16; ++q) {  // (the difference first: scores at the type's lowest value times log2 e are none)
                            float e0, e1;
                            un2(mul2(add2(mk2(f[2 * q], f[2 * q + 1]), minus), log2e), e0, e1);
                            acc[q & 1] = add2(acc[q & 1], mk2(ex2(e0), ex2(e1)));
                        }
                        float s0, s1;
                        un2(add2(acc[0], acc[1]), s0, s1);
                        sum = fmaf(sum, ex2((m - ref) * LOG2E), s0 + s1);
                        m = best;
                    }
                    continue;
                }
                // factors and pixels to be kept out are in a copy of their own: their tests alone, never met, cost a fifth
                auto gradient = [&](auto rare_) {
                constexpr bool RARE = decltype(rare_)::value;
                float row_m = 0.f, inv_z = 1.f;
                if (RARE && large && !it.dw && label >= 0) { row_m = a.lse[r]; inv_z = ex2(-a.lse[a.n + r] * LOG2E); }
#pragma unroll 1
                for (int h = 0; h < 64; h += 32) {
                    uint32_t u[32];
                    __syncwarp();
                    tm_ld32(s + h, u);
                    tm_wait_ld32(u);
                    if (RARE && large && it.dw) {  // m of the pixels of the columns; of a row: above (no label: -infinity stays)
                        const int lab = reinterpret_cast<const int*>(kb)[h + lane];
                        row_m = lab >= 0 ? a.lse[(int64_t)j * LT + half + h + lane] : 0.f;
                    }
#pragma unroll
                    for (int o = 0; o < 32; o += 16) {  // 16 columns: one step of the product's inner dimension
                        float e[16];
                        if (RARE && large)  // (all 32 at once cost registers: codebook gradients 3.79 -> 3.95 ms, though never run there)
#pragma unroll
                            for (int q = 0; q < 16; ++q) u[o + q] = __float_as_uint(__uint_as_float(u[o + q]) - __shfl_sync(0xffffffffu, row_m, it.dw ? o + q : lane));
#pragma unroll
                        for (int q = 0; q < 16; q += 2) {
                            un2(mul2(mk2u(u[o + q], u[o + q + 1]), log2e), e[q], e[q + 1]);
                            e[q] = ex2(e[q]);
                            e[q + 1] = ex2(e[q + 1]);
                        }
                        if (!it.dw) {
                            if (RARE && large) {
#pragma unroll
                                for (int q = 0; q < 16; ++q) e[q] *= inv_z;
                            }
                            if ((yl >> 4) == ((h + o) >> 4)) {  // before the rounding: p - 1 of a pixel that is nearly certain is small
#pragma unroll
                                for (int q = 0; q < 16; ++q) sub_if(e[q], 1.f, yl & 15, q);
                            }
                        } else {
                            if (RARE && scaled) {
#pragma unroll
                                for (int q = 0; q < 16; ++q) e[q] *= kb[2 * LT + h + o + q];
                            }
                            // pixels of these 16 whose label is one of the warp's 32 rows
                            const int* lab = reinterpret_cast<const int*>(kb + h + o);
                            if (__any_sync(0xffffffffu, (unsigned)(lab[lane & 15] - it.m * LT - wrow) < 32u)) {
#pragma unroll
                                for (int q = 0; q < 16; q += 4) {
                                    const int4 l = *reinterpret_cast<const int4*>(lab + q);
                                    float4 g = make_float4(1.f, 1.f, 1.f, 1.f);
                                    if (RARE && scaled) g = *reinterpret_cast<const float4*>(kb + LT + h + o + q);
                                    sub_if(e[q], g.x, l.x, (int)r);
                                    sub_if(e[q + 1], g.y, l.y, (int)r);
                                    sub_if(e[q + 2], g.z, l.z, (int)r);
                                    sub_if(e[q + 3], g.w, l.w, (int)r);
                                }
                            }
                            if (RARE && dirty) {
#pragma unroll
                                for (int q = 0; q < 16; ++q)
                                    if (lab[q] < 0) e[q] = 0.f;
                            }
                            if (a.part_b) {
                                f2 acc = mk2(e[0], e[1]);
#pragma unroll
                                for (int q = 2; q < 16; q += 2) acc = add2(acc, mk2(e[q], e[q + 1]));
                                float s0, s1;
                                un2(acc, s0, s1);
                                sum += s0 + s1;
                            }
                        }
                        uint32_t w0[8];
#pragma unroll
                        for (int q = 0; q < 8; ++q) w0[q] = bf16x2(e[2 * q], e[2 * q + 1]);
                        __syncwarp();
                        tm_st8(s + h + o, w0);
                        if (P == 3) {
                            uint32_t w1[8];
#pragma unroll
                            for (int q = 0; q < 8; ++q) {
                                e[2 * q] -= bf_lo(w0[q]);
                                e[2 * q + 1] -= bf_hi(w0[q]);
                                w1[q] = bf16x2(e[2 * q], e[2 * q + 1]);
                            }
                            tm_st8(s + h + o + 8, w1);
#pragma unroll
                            for (int q = 0; q < 8; ++q) w0[q] = bf16x2(e[2 * q] - bf_lo(w1[q]), e[2 * q + 1] - bf_hi(w1[q]));
                            tm_st8(s - half + 128 + ((half + h + o) >> 1), w0);
                        }
                    }
                }
                };
                if (rare) gradient(std::true_type());
                else gradient(std::false_type());
                if (P == 1 && WHOLE && dirty && it.dw) {
                    // pixels without a label whose features are not finite: 0 * inf must not reach dW, so their rows of the
                    // staged block are cleared (row n of every chunk, whole, whatever the swizzle)
                    if (__float_as_int(kb[row - half]) < 0) {
                        for (int k = 0; k < a.nk; ++k) {
                            uint32_t slot = bstage + k / CS;
                            if (slot >= (uint32_t)a.stages) slot -= a.stages;
                            uint4* p = reinterpret_cast<uint4*>(ring + slot * stage + (k % CS) * TB + row * (KC * 2));
#pragma unroll
                            for (int q = 0; q < KC / 8; ++q) p[q] = make_uint4(0, 0, 0, 0);
                        }
                    }
                    rgs_fence_proxy_async();
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                if (it.dw) rgs_mbar_arrive(&sh->k_empty[kslot]);
                rgs_mbar_arrive(&sh->s_done[buf]);
                if (out_i < i) {  // outputs of earlier items, behind the first scores of this one
                    write_out(out_i, out_scale, out_label);
                    for (out_i += gridDim.x; out_i < i; out_i += gridDim.x) write_out(out_i, row_scale(out_i), row_label(out_i));
                    out_label = label;
                    out_scale = scale;
                }
            }
            if (!GRAD) {
                dead = __any_sync(0xffffffffu, dead || *fail);
                if (r < a.n) {
                    a.pm[((int64_t)it.split * 4 + wg) * a.n + r] = dead ? nan : m;
                    a.ps[((int64_t)it.split * 4 + wg) * a.n + r] = dead ? nan : sum;
                }
            } else if (it.dw && a.part_b && it.oc0 == 0) {
                dead = __any_sync(0xffffffffu, dead || *fail);
                // which warpgroup takes the even tiles of an item hangs on the items before it: the sums go by even and odd, so
                // that their order, and db, do not hang on what else is asked for
                const int place = wg ^ (int)((t - (uint32_t)(it.j1 - it.j0)) & 1u);
                float* p = a.part_b + ((int64_t)it.split * 4 + place) * a.nmw * LT + r;
                *p = (dead ? nan : sum * gshare) + (a.sub ? *p : 0.f);
            }
        }
        if (GRAD && out_i < items) {
            write_out(out_i, out_scale, out_label);
            for (out_i += gridDim.x; out_i < items; out_i += gridDim.x) write_out(out_i, row_scale(out_i), row_label(out_i));
        }
        lb_end_of_role();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// ---------------------------------------------------------------------------------------------------------------------
// before: operands that TMA cannot read as they are, column constants
// ---------------------------------------------------------------------------------------------------------------------
struct LabelPrep {
    const void* x; int64_t ldx; const void* w; int64_t ldw; const void* bias; const void* labels;
    int label_bytes, dtype, b_dtype, backward, per_row, mean, pieces;
    int64_t n, v;
    int c, cp, nmx, nmw;
    __nv_bfloat16* xs; __nv_bfloat16* ws;  // (pieces, rows, cp) or null where the tensor itself is read
    __nv_bfloat16* ew; __nv_bfloat16* ex;  // extra channels, (nmw * 128, 16) and (nmx * 128, 16); forward: ex (128, 16)
    float* kn; float* gs;
    const float* lse; const float* gout; const float* count;
    unsigned* ticket;
};

// eight channels of a row in one or three bf16 pieces whose sum is the value (to 2^-25 of it; infinities in the first alone)
__device__ __forceinline__ void lb_split8(const void* src, int64_t ld, int dtype, int64_t rows, int64_t r, int c0, int c, int cp, int pieces,
                                          bool clear, __nv_bfloat16* dst) {
    float f[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) f[q] = !clear && c0 + q < c ? rgs_load_as_float(src, r * ld + c0 + q, dtype) : 0.f;
    for (int p = 0; p < pieces; ++p) {
        uint32_t u[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            u[q] = bf16x2(f[2 * q], f[2 * q + 1]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float& e = f[2 * q + h];
                float k = h ? bf_hi(u[q]) : bf_lo(u[q]);
                if (!(fabsf(k) <= 3.3e38f)) {      // infinity, NaN, or a finite value that rounds up to infinity
                    if (fabsf(e) <= 3.402823466e38f) {
                        k = __uint_as_float(__float_as_uint(e) & 0xffff0000u);
                        u[q] = h ? (u[q] & 0xffffu) | (__float_as_uint(k) & 0xffff0000u) : (u[q] & 0xffff0000u) | (__float_as_uint(k) >> 16);
                    } else {
                        k = 0.f;
                        e = 0.f;
                    }
                }
                e -= k;
            }
        }
        *reinterpret_cast<uint4*>(dst + ((int64_t)p * rows + r) * cp + c0) = make_uint4(u[0], u[1], u[2], u[3]);
    }
}

// a value in three bf16 pieces (an infinity, or what rounds to one, whole in the first where it cannot be split)
__device__ __forceinline__ void lb_split3(float v, uint32_t (&p)[3]) {
#pragma unroll
    for (int q = 0; q < 3; ++q) {
        uint32_t u = bf16x2(v, 0.f) & 0xffffu;
        if ((u & 0x7fffu) >= 0x7f80u) {
            if (fabsf(v) <= 3.402823466e38f) u = __float_as_uint(v) >> 16;
            else { p[q] = u; v = 0.f; continue; }
        }
        p[q] = u;
        v -= __uint_as_float(u << 16);
    }
}
// sixteen extra channels of a row: three values and three more, zeros behind
__device__ __forceinline__ void lb_extra(__nv_bfloat16* dst, const uint32_t (&a)[3], const uint32_t (&b)[3]) {
    uint4* d = reinterpret_cast<uint4*>(dst);
    d[0] = make_uint4(a[0] | (a[1] << 16), a[2] | (b[0] << 16), b[1] | (b[2] << 16), 0u);
    d[1] = make_uint4(0u, 0u, 0u, 0u);
}

__global__ void __launch_bounds__(256) rgs_label_prep_kernel(const __grid_constant__ LabelPrep a) {
    const int groups = a.cp / 8;
    const int64_t gx = a.xs ? a.n * groups : 0, gw = a.ws ? a.v * groups : 0, gb = (int64_t)a.nmw * LT;
    const int64_t gk = a.backward ? (int64_t)a.nmx * LT : LT;
    const uint32_t ones[3] = {0x3f80u, 0x3f80u, 0x3f80u}, none[3] = {0xff80u, 0u, 0u};  // 1; -infinity
    const bool large = a.backward && ((int)a.count[1] & LF_LARGE);
    const float mean = a.mean ? 1.f / fmaxf(a.count[0], 1.f) : 1.f;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        if (a.ticket) *a.ticket = 0u;
        if (a.gs) *a.gs = a.gout[0] * mean;
    }
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < gx + gw + gb + gk; i += (int64_t)gridDim.x * 256) {
        int64_t k = i;
        if (k < gx) {
            const int64_t r = k / groups;
            const bool clear = a.backward && rgs_label(a.labels, r, a.label_bytes, a.v) < 0;
            lb_split8(a.x, a.ldx, a.dtype, a.n, r, (int)(k - r * groups) * 8, a.c, a.cp, a.pieces, clear, a.xs);
            continue;
        }
        k -= gx;
        if (k < gw) {
            const int64_t r = k / groups;
            lb_split8(a.w, a.ldw, a.dtype, a.v, r, (int)(k - r * groups) * 8, a.c, a.cp, a.pieces, false, a.ws);
            continue;
        }
        k -= gw;
        if (k < gb) {
            uint32_t b[3] = {0u, 0u, 0u};
            if (k < a.v) {
                if (a.bias) lb_split3(rgs_load_as_float(a.bias, k, a.b_dtype), b);
                lb_extra(a.ew + k * 16, b, ones);
            } else {
                lb_extra(a.ew + k * 16, none, ones);
            }
            continue;
        }
        k -= gb;
        uint32_t c[3] = {0u, 0u, 0u};
        if (!a.backward) {
            lb_extra(a.ex + k * 16, ones, c);
            continue;
        }
        const int64_t y = k < a.n ? rgs_label(a.labels, k, a.label_bytes, a.v) : -1;
        float g = 0.f, f = 0.f;
        if (y >= 0) {
            g = a.gout[a.per_row ? k : 0] * mean;
            const float m = a.lse[k], lz = a.lse[a.n + k];
            if (!large) lb_split3(-(m + lz), c);
            f = large ? g * expf(-lz) : g;
            lb_extra(a.ex + k * 16, ones, c);
        } else {
            lb_extra(a.ex + k * 16, ones, none);
        }
        float* o = a.kn + (k / LT) * (3 * LT) + k % LT;
        o[0] = __int_as_float((int)y); o[LT] = g; o[2 * LT] = f;
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// after the forward pass: joins the pieces of the walk over the labels; the last block adds up the blocks in order
// ---------------------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) rgs_label_join_kernel(const float* __restrict__ pm, const float* __restrict__ ps, const float* __restrict__ at,
                                                             const void* labels, int label_bytes, int64_t n, int64_t vocab, int parts, int mean,
                                                             float* lse, float* losses, float* result, float* count, double* bsum,
                                                             unsigned long long* bcount, unsigned* ticket) {
    __shared__ double ssum[8];
    __shared__ unsigned long long scount[8];
    __shared__ int sdirty, last;
    double total = 0;
    unsigned long long rows = 0;
    int dirty = 0;
    if (threadIdx.x == 0) sdirty = 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t y = rgs_label(labels, i, label_bytes, vocab);
        float m = pm[i];
        for (int k = 1; k < parts; ++k) m = fmaxf(m, pm[(int64_t)k * n + i]);
        const float ref = m == -INFINITY ? 0.f : m;
        float z = 0.f;
        for (int k = 0; k < parts; ++k) z = fmaf(ps[(int64_t)k * n + i], expf(pm[(int64_t)k * n + i] - ref), z);
        const float lz = logf(z);
        lse[i] = m;
        lse[n + i] = lz;
        float loss = 0.f;
        if (y >= 0) {
            loss = lz + (m - at[i]);
            ++rows;
            if (fabsf(m) > 1024.f) dirty |= LF_LARGE;
        } else if (!(fabsf(m) <= 3.402823466e38f) || !(fabsf(lz) <= 3.402823466e38f)) {
            dirty |= LF_DIRTY;
        }
        if (losses) losses[i] = loss;
        total += (double)loss;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) { total += __shfl_xor_sync(0xffffffffu, total, d); rows += __shfl_xor_sync(0xffffffffu, rows, d); }
    __syncthreads();
    if (dirty) atomicOr(&sdirty, dirty);
    if ((threadIdx.x & 31) == 0) { ssum[threadIdx.x >> 5] = total; scount[threadIdx.x >> 5] = rows; }
    __syncthreads();
    if (threadIdx.x == 0) {
        total = 0; rows = 0;
        for (int k = 0; k < 8; ++k) { total += ssum[k]; rows += scount[k]; }
        bsum[blockIdx.x] = total;
        bcount[blockIdx.x] = rows * 4 + (unsigned)sdirty;
        __threadfence();
        last = atomicAdd(ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    total = 0; rows = 0; dirty = 0;
    for (unsigned k = threadIdx.x; k < gridDim.x; k += 256) {
        total += __ldcg(&bsum[k]);
        const unsigned long long u = __ldcg(&bcount[k]);
        rows += u >> 2;
        dirty |= (int)(u & 3);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) { total += __shfl_xor_sync(0xffffffffu, total, d); rows += __shfl_xor_sync(0xffffffffu, rows, d); }
    if ((threadIdx.x & 31) == 0) { ssum[threadIdx.x >> 5] = total; scount[threadIdx.x >> 5] = rows; }
    if (threadIdx.x == 0) sdirty = 0;
    __syncthreads();
    if (dirty) atomicOr(&sdirty, dirty);
    __syncthreads();
    if (threadIdx.x == 0) {
        total = 0; rows = 0;
        for (int k = 0; k < 8; ++k) { total += ssum[k]; rows += scount[k]; }
        count[0] = (float)rows;
        count[1] = (float)sdirty;
        if (result) *result = (float)(mean ? total / (double)(rows > 0 ? rows : 1) : total);
    }
}

// After the backward pass: adds up the pieces of dX, in order, a thread to four channels (few pieces, many rows).
__global__ void __launch_bounds__(256) rgs_label_reduce_x_kernel(const __grid_constant__ LabelArgs a) {
    const int per = a.cq / 4;
    const int64_t stride = (int64_t)a.nmx * LT * a.cq;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.n * per; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per;
        const int c = (int)(i - r * per) * 4;
        if (c >= a.c) continue;
        const float* p = a.part_x + r * a.cq + c;
        float4 s = *reinterpret_cast<const float4*>(p);
        for (int k = 1; k < a.nsx; ++k) {
            const float4 t = *reinterpret_cast<const float4*>(p + k * stride);
            s.x += t.x; s.y += t.y; s.z += t.z; s.w += t.w;
        }
        const float f[4] = {s.x, s.y, s.z, s.w};
        const float* k = a.kn + (r / LT) * (3 * LT) + r % LT;
        const float scale = k[LT];
        const bool zero = __float_as_int(k[0]) < 0;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (c + q < a.c) rgs_store_float(a.dx, r * a.c + c + q, a.dtype, zero ? 0.f : f[q] * scale);
    }
}

// The pieces of dW and db are many and the sums few (810 pieces of 512 x 32 in the 32-bit view): sixteen chains of every
// sum side by side, 32 sums of four channels (of one label for db) to a block, joined in order.  A thread to a sum: 220 us.
__global__ void __launch_bounds__(512) rgs_label_reduce_w_kernel(const __grid_constant__ LabelArgs a, int blocks_w, void* db, int b_dtype) {
    __shared__ float4 sh[16][32];
    const int lane = threadIdx.x & 31, chain = threadIdx.x >> 5;
    if ((int)blockIdx.x < blocks_w) {
        const int64_t i = (int64_t)blockIdx.x * 32 + lane, total = a.v * (a.cq / 4), stride = (int64_t)a.nmw * LT * a.cq;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < total)
#pragma unroll 4
            for (int k = chain; k < a.nsw; k += 16) {
                const float4 t = *reinterpret_cast<const float4*>(a.part_w + k * stride + i * 4);
                s.x += t.x; s.y += t.y; s.z += t.z; s.w += t.w;
            }
        sh[chain][lane] = s;
        __syncthreads();
        if (chain == 0 && i < total) {
            const int chains = a.nsw < 16 ? a.nsw : 16;
            for (int k = 1; k < chains; ++k) {
                const float4 t = sh[k][lane];
                s.x += t.x; s.y += t.y; s.z += t.z; s.w += t.w;
            }
            const int64_t r = i / (a.cq / 4);
            const int c = (int)(i - r * (a.cq / 4)) * 4;
            const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (c + q < a.c) rgs_store_float(a.dw, r * a.c + c + q, a.dtype, f[q]);
        }
        return;
    }
    const int64_t v = (int64_t)(blockIdx.x - blocks_w) * 32 + lane;
    float s = 0.f;
    if (v < a.v)
#pragma unroll 8
        for (int k = chain; k < 4 * a.nsw; k += 16) s += a.part_b[(int64_t)k * a.nmw * LT + v];
    sh[chain][lane].x = s;
    __syncthreads();
    if (chain == 0 && v < a.v) {
        for (int k = 1; k < 16; ++k) s += sh[k][lane].x;
        rgs_store_float(db, v, b_dtype, s);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------------
typedef CUresult (*LabelEncode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static LabelEncode label_encode() {
    static std::atomic<LabelEncode> cached{nullptr};
    LabelEncode fn = cached.load();
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return nullptr;
        fn = reinterpret_cast<LabelEncode>(p);
        cached.store(fn);
    }
    return fn;
}

// (channels, rows, pieces) of bf16; boxes of kc channels x 128 rows; what lies outside reads as zero
static int label_map(CUtensorMap* map, const void* base, int64_t c, int64_t rows, int64_t ld, int64_t pieces, int kc) {  // kc: 64, 32, 16
    LabelEncode enc = label_encode();
    if (!enc) return 20;
    const cuuint64_t dims[3] = {(cuuint64_t)c, (cuuint64_t)rows, (cuuint64_t)pieces};
    const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)ld * 2 * (cuuint64_t)rows};
    const cuuint32_t box[3] = {(cuuint32_t)kc, LT, 1}, estr[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               kc == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : kc == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : 21;
}

// Limits: [0] tries of a wait, [1] stages that the producer of a CTA fills before it gives up, [2] bytes of partial sums of dX and
// of dW (and one sum more).  Tests lower them.
static const int64_t label_defaults[3] = {LWAIT, 0xffffffffll, (int64_t)1 << 31};
static std::atomic<int64_t> label_limits[3] = {{label_defaults[0]}, {label_defaults[1]}, {label_defaults[2]}};

static inline int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// A walk over nj tiles made by `tiles` row tiles, in `slots` partial sums of `subs` pieces each.  One piece where there are three
// row tiles or more to an SM; else pieces short enough for six items to an SM.  No piece is longer than `run` tiles, the most
// that one accumulator may sum; there is room for `most` partial sums, and where that is too few the pieces of one follow each
// other in launches of their own, each adding to what the ones before left (1657600 pixels x 64 channels x 32771 labels in 32 bits:
// with pieces of 43 tiles in place of eight dX was off by 1.5e-5 of its absolute sum, with one sign throughout, instead of 1.9e-6).
static void label_pieces(int64_t tiles, int64_t nj, int64_t sms, int64_t run, int64_t most, int* slots, int* subs) {
    int64_t per = nj;
    if (tiles < 3 * sms) per = (tiles * nj + sms * 6 - 1) / (sms * 6);
    if (per > run) per = run;
    if (per < 1) per = 1;
    int64_t ns = (nj + per - 1) / per, k = 1;
    if (ns > most) {
        ns = most < 1 ? 1 : most;
        k = ((nj + run - 1) / run + ns - 1) / ns;
        if (ns * k > nj) ns = nj / k;  // no empty pieces
    }
    *slots = (int)(ns < 1 ? 1 : ns);
    *subs = (int)k;
}

struct LabelPlan {
    LabelArgs a;
    int pieces, kc, cs, direct_x, direct_w, cp, parts_x, parts_w;
    int64_t o_xs, o_ws, o_ew, o_ex, o_kn, o_gs, o_pm, o_ps, o_at, o_px, o_pw, o_pb, o_bsum, o_bcount, o_ticket, bytes;
};

#define LJOIN 592  // most blocks of the joining kernel

// what a backward pass is to give: bits of `backward`, 0 for the forward pass
enum { LB_ANY = 1, LB_DX = 2, LB_DW = 4, LB_DB = 8 };

static void label_plan(LabelPlan& p, int64_t n, int64_t c, int64_t v, int dtype, int direct, int backward) {
    LabelArgs& a = p.a;
    memset(&p, 0, sizeof(p));
    const int64_t sms = RGS_SMS;
    p.pieces = dtype == RGS_BF16 ? 1 : 3;
    p.kc = c <= 32 ? 32 : 64;
    a.n = n; a.v = v; a.c = (int)c; a.nk = (int)((c + p.kc - 1) / p.kc);
    a.nmx = (int)((n + LT - 1) / LT); a.nmw = (int)((v + LT - 1) / LT);
    a.dtype = dtype;
    const int na = p.pieces * a.nk, room = LROOM / (256 * p.kc);
    // TMEM: 512 columns.  Up to 128 output channels leave room for three score buffers in 16 bits, more for two; the two sums
    // of 32-bit outputs and the third piece of G leave room for two and one chunk of channels.  The forward pass takes four.
    const int cols = p.pieces == 1 ? 256 / p.kc : 1;
    a.noc = a.nk < cols ? a.nk : cols;
    a.nrange = backward ? (a.nk + a.noc - 1) / a.noc : 1;
    a.nbuf = !backward ? 4 : (p.pieces == 1 && a.nk * p.kc <= 128 ? 3 : 2);
    a.nob = (p.pieces == 1 ? a.nk * p.kc : 2 * p.kc) <= 64 ? 2 : 1;
    // Stages of B are kept for both products where the ring holds one block to a score buffer beside the block (better two)
    // of A and one range covers the channels; else they are fetched for each product, and A stays where half the room holds it.
    a.a_slots = na <= 8 ? 1 : 0;
    a.whole = backward && a.nrange == 1 && room >= na * (a.nbuf + 1);
    if (room >= na * ((backward ? a.nbuf : 2) + 3)) a.a_slots = 2;
    // chunks of a stage: few barriers to a block where the ring is deep enough
    p.cs = 1;
    if (p.pieces == 1 && p.kc == 64 && a.a_slots && a.nk <= 4) p.cs = a.nk == 2 || a.nk == 4 ? 2 : (a.nk == 3 ? 3 : 1);
    a.stages = (room - a.a_slots * na) / (p.pieces * p.cs);
    if (a.stages > LSTAGES) a.stages = LSTAGES;
    a.cq = (int)up(c, 16);
    // where B is fetched anew for the second product its rows cannot be cleared in place: X goes through the copy
    p.direct_x = p.pieces == 1 && (direct & 1) && (!backward || a.whole);
    p.direct_w = p.pieces == 1 && (direct & 2);
    p.cp = (int)up(c, 8);
    // an accumulator that adds 8 tiles of leading products is off by 1.0e-6 of its sum in 32 bits (16 tiles: 2.0e-6; the pieces
    // take 1 % of the time); beside 16-bit outputs 512 tiles are far below their rounding
    const int64_t run = p.pieces == 1 ? 512 : 8;
    const int64_t rows_x = (int64_t)a.nmx * LT, rows_w = (int64_t)a.nmw * LT;
    if (backward) {
        const int64_t room = label_limits[2].load();
        label_pieces((int64_t)a.nmx * a.nrange, a.nmw, sms, run, room / (rows_x * a.cq * 4) + 1, &a.nsx, &a.subx);
        label_pieces((int64_t)a.nmw * a.nrange, a.nmx, sms, run, room / (rows_w * a.cq * 4) + 1, &a.nsw, &a.subw);
    } else {
        label_pieces(a.nmx, a.nmw, sms, a.nmw, a.nmw, &a.nsx, &a.subx);
        a.nsw = a.subw = 1;
    }
    const int px = a.nsx * a.subx, pw = a.nsw * a.subw;
    a.perx = a.nmw / px; a.restx = a.nmw % px;
    a.perw = a.nmx / pw; a.restw = a.nmx % pw;
    // one partial sum: 32-bit outputs are added up where they lie
    p.parts_x = !(backward & LB_DX) ? 0 : a.nsx > 1 || (a.subx > 1 && dtype == RGS_BF16);
    p.parts_w = !(backward & LB_DW) ? 0 : a.nsw > 1 || (a.subw > 1 && dtype == RGS_BF16);
    int64_t o = 0;
    auto take = [&](int64_t bytes) { const int64_t at = o; o = up(o + bytes, 1024); return at; };
    p.o_xs = p.direct_x ? -1 : take(n * p.cp * 2 * p.pieces);
    p.o_ws = p.direct_w ? -1 : take(v * p.cp * 2 * p.pieces);
    p.o_ew = take(rows_w * 32);
    p.o_ex = take((backward ? rows_x : LT) * 32);
    if (backward) {
        p.o_kn = take(rows_x * 12);
        p.o_gs = take(4);
        p.o_px = p.parts_x ? take(a.nsx * rows_x * a.cq * 4) : -1;
        p.o_pw = p.parts_w ? take(a.nsw * rows_w * a.cq * 4) : -1;
        p.o_pb = backward & LB_DB ? take(4 * a.nsw * rows_w * 4) : -1;
    } else {
        p.o_pm = take(4 * a.nsx * n * 4);
        p.o_ps = take(4 * a.nsx * n * 4);
        p.o_at = take(n * 4);
        p.o_bsum = take(LJOIN * 8);
        p.o_bcount = take(LJOIN * 8);
        p.o_ticket = take(4);
    }
    p.bytes = o + 1024;
}

static int label_direct(const void* x, int64_t ldx, const void* w, int64_t ldw) {
    const int dx = ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0, dw = ldw % 8 == 0 && (reinterpret_cast<uintptr_t>(w) & 15) == 0;
    return dx | (dw << 1);
}

struct LabelMaps { CUtensorMap x, w, ex, ew; };

template <int P, bool GRAD, int KC, int CS, bool WHOLE>
static int label_launch(const LabelMaps& m, LabelArgs a, cudaStream_t stream) {
    static std::atomic<uint64_t> ready{0};  // devices whose limit on dynamic shared memory was raised
    int dev = 0;
    RGS_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev > 63 || !((ready.load() >> dev) & 1)) {
        RGS_CUDA_CHECK(cudaFuncSetAttribute(rgs_label_tc_kernel<P, GRAD, KC, CS, WHOLE>, cudaFuncAttributeMaxDynamicSharedMemorySize, LSMEM));
        if (dev <= 63) ready.fetch_or((uint64_t)1 << dev);
    }
    const int64_t items = (int64_t)a.items_x + a.items_w, sms = RGS_SMS;
    a.wait = (uint32_t)label_limits[0].load();
    a.loads = (uint32_t)label_limits[1].load();
    rgs_label_tc_kernel<P, GRAD, KC, CS, WHOLE><<<(unsigned)(items < sms ? items : sms), LTHREADS, LSMEM, stream>>>(m.x, m.w, m.ex, m.ew, a);
    rgs_cuda_field_launches(1);
    return (int)cudaGetLastError();
}

template <bool GRAD>
static int label_run(const LabelPlan& p, const LabelMaps& m, cudaStream_t stream) {
    const bool whole = GRAD ? p.a.whole != 0 : p.a.a_slots > 0;
    if (p.kc == 32) return p.pieces == 3 ? label_launch<3, GRAD, 32, 1, true>(m, p.a, stream) : label_launch<1, GRAD, 32, 1, true>(m, p.a, stream);
    if (p.pieces == 3) return whole ? label_launch<3, GRAD, 64, 1, true>(m, p.a, stream) : label_launch<3, GRAD, 64, 1, false>(m, p.a, stream);
    if (!whole) return label_launch<1, GRAD, 64, 1, false>(m, p.a, stream);
    if (p.cs == 3) return label_launch<1, GRAD, 64, 3, true>(m, p.a, stream);
    return p.cs == 2 ? label_launch<1, GRAD, 64, 2, true>(m, p.a, stream) : label_launch<1, GRAD, 64, 1, true>(m, p.a, stream);
}

static inline unsigned label_grid(int64_t work, int64_t most) {
    const int64_t want = (work + 255) / 256;
    return (unsigned)(want < 1 ? 1 : (want > most ? most : want));
}

static int label_operands(const LabelPlan& p, const LabelPrep& q, LabelMaps* m) {
    // autograd runs the backward pass on a thread of its own, where the driver has no context yet: cudaSetDevice binds it
    int dev = 0;
    RGS_CUDA_CHECK(cudaGetDevice(&dev));
    RGS_CUDA_CHECK(cudaSetDevice(dev));
    int rc = p.direct_x ? label_map(&m->x, q.x, q.c, q.n, q.ldx, 1, p.kc) : label_map(&m->x, q.xs, p.cp, q.n, p.cp, p.pieces, p.kc);
    if (!rc) rc = p.direct_w ? label_map(&m->w, q.w, q.c, q.v, q.ldw, 1, p.kc) : label_map(&m->w, q.ws, p.cp, q.v, p.cp, p.pieces, p.kc);
    if (!rc) rc = label_map(&m->ex, q.ex, 16, q.backward ? (int64_t)q.nmx * LT : LT, 16, 1, 16);
    return rc ? rc : label_map(&m->ew, q.ew, 16, (int64_t)q.nmw * LT, 16, 1, 16);
}

static void label_prep(const LabelPlan& p, const LabelPrep& q, cudaStream_t stream) {
    const int64_t work = ((q.xs ? q.n : 0) + (q.ws ? q.v : 0)) * (q.cp / 8) + (int64_t)q.nmw * LT + (q.backward ? (int64_t)q.nmx * LT : LT);
    rgs_label_prep_kernel<<<label_grid(work, RGS_SMS * 16), 256, 0, stream>>>(q);
    rgs_cuda_field_launches(1);
}

static void label_fill(LabelPrep& q, const LabelPlan& p, unsigned char* s, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                       const void* labels, int label_bytes, int dtype, int b_dtype) {
    q.x = x; q.ldx = ldx; q.w = w; q.ldw = ldw; q.bias = bias; q.labels = labels;
    q.label_bytes = label_bytes; q.dtype = dtype; q.b_dtype = b_dtype; q.pieces = p.pieces;
    q.n = p.a.n; q.v = p.a.v; q.c = p.a.c; q.cp = p.cp; q.nmx = p.a.nmx; q.nmw = p.a.nmw;
    q.xs = p.direct_x ? nullptr : reinterpret_cast<__nv_bfloat16*>(s + p.o_xs);
    q.ws = p.direct_w ? nullptr : reinterpret_cast<__nv_bfloat16*>(s + p.o_ws);
    q.ew = reinterpret_cast<__nv_bfloat16*>(s + p.o_ew);
    q.ex = reinterpret_cast<__nv_bfloat16*>(s + p.o_ex);
}

extern "C" {

// Sets limit `which` of label_limits to `value`, a negative one to its default, for calls from now on; returns the value before, or
// -1 for a limit that there is not.
int64_t rgs_cuda_label_limit(int64_t which, int64_t value) {
    if (which < 0 || which > 2) return -1;
    return label_limits[which].exchange(value < 0 ? label_defaults[which] : value);
}

// direct: bit 0 / 1: rows of x / w start on 16-byte boundaries; backward: 0, or LB_ bits of the gradients wanted
int64_t rgs_cuda_label_scratch_bytes(int64_t n, int64_t c, int64_t vocab, int64_t dtype, int64_t direct, int64_t backward) {
    LabelPlan p;
    label_plan(p, n, c, vocab, (int)dtype, (int)direct, (int)backward);
    return p.bytes;
}

int rgs_cuda_label_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* labels, int64_t label_bytes,
                       int64_t n, int64_t c, int64_t vocab, int64_t dtype, int64_t b_dtype, int64_t mean, void* scratch, int64_t scratch_bytes,
                       float* lse, float* losses, float* result, float* count, void* stream) {
    cudaStream_t st = (cudaStream_t)stream;
    LabelPlan p;
    label_plan(p, n, c, vocab, (int)dtype, label_direct(x, ldx, w, ldw), 0);
    if (p.bytes > scratch_bytes) return 24;
    LabelArgs& a = p.a;
    unsigned char* s = reinterpret_cast<unsigned char*>(up((int64_t)reinterpret_cast<uintptr_t>(scratch), 1024));
    LabelPrep q{};
    label_fill(q, p, s, x, ldx, w, ldw, bias, labels, (int)label_bytes, (int)dtype, (int)b_dtype);
    q.ticket = reinterpret_cast<unsigned*>(s + p.o_ticket);
    LabelMaps m;
    int rc = label_operands(p, q, &m);
    if (rc) return rc;
    label_prep(p, q, st);
    RGS_CUDA_CHECK(cudaGetLastError());
    a.items_x = (unsigned)a.nmx * a.nsx;
    a.labels = labels; a.label_bytes = (int)label_bytes;
    a.flags = count;
    a.pm = reinterpret_cast<float*>(s + p.o_pm);
    a.ps = reinterpret_cast<float*>(s + p.o_ps);
    a.at = reinterpret_cast<float*>(s + p.o_at);
    rc = label_run<false>(p, m, st);
    if (rc) return rc;
    rgs_label_join_kernel<<<label_grid(n, LJOIN), 256, 0, st>>>(a.pm, a.ps, a.at, labels, (int)label_bytes, n, vocab, 4 * a.nsx, (int)mean, lse, losses,
                                                                result, count, reinterpret_cast<double*>(s + p.o_bsum),
                                                                reinterpret_cast<unsigned long long*>(s + p.o_bcount), q.ticket);
    rgs_cuda_field_launches(1);
    return (int)cudaGetLastError();
}

int rgs_cuda_label_bwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* labels, int64_t label_bytes,
                       int64_t n, int64_t c, int64_t vocab, int64_t dtype, int64_t b_dtype, const float* lse, const float* gout,
                       int64_t per_row, int64_t mean, const float* count, void* scratch, int64_t scratch_bytes, void* dx, void* dw, void* db, void* stream) {
    cudaStream_t st = (cudaStream_t)stream;
    LabelPlan p;
    label_plan(p, n, c, vocab, (int)dtype, label_direct(x, ldx, w, ldw), LB_ANY | (dx ? LB_DX : 0) | (dw ? LB_DW : 0) | (db ? LB_DB : 0));
    if (p.bytes > scratch_bytes) return 24;
    LabelArgs& a = p.a;
    unsigned char* s = reinterpret_cast<unsigned char*>(up((int64_t)reinterpret_cast<uintptr_t>(scratch), 1024));
    LabelPrep q{};
    label_fill(q, p, s, x, ldx, w, ldw, bias, labels, (int)label_bytes, (int)dtype, (int)b_dtype);
    q.backward = 1; q.per_row = (int)per_row; q.mean = (int)mean;
    q.lse = lse; q.gout = gout; q.count = count;
    q.kn = reinterpret_cast<float*>(s + p.o_kn);
    q.gs = reinterpret_cast<float*>(s + p.o_gs);
    LabelMaps m;
    int rc = label_operands(p, q, &m);
    if (rc) return rc;
    label_prep(p, q, st);
    RGS_CUDA_CHECK(cudaGetLastError());
    a.kn = q.kn; a.lse = lse; a.gs = q.gs; a.per_row = (int)per_row;
    a.labels = labels; a.label_bytes = (int)label_bytes;
    a.flags = count;
    a.part_x = p.parts_x ? reinterpret_cast<float*>(s + p.o_px) : nullptr;
    a.part_w = p.parts_w ? reinterpret_cast<float*>(s + p.o_pw) : nullptr;
    a.part_b = db ? reinterpret_cast<float*>(s + p.o_pb) : nullptr;
    a.dx = dx; a.dw = dw;
    const int subx = dx ? a.subx : 0, subw = dw || db ? a.subw : 0;
    for (a.sub = 0; a.sub < subx || a.sub < subw; ++a.sub) {
        a.items_x = a.sub < subx ? (unsigned)a.nmx * a.nrange * a.nsx : 0;
        a.items_w = a.sub < subw ? (unsigned)a.nmw * a.nrange * a.nsw : 0;
        rc = label_run<true>(p, m, st);
        if (rc) return rc;
    }
    if (a.part_x) rgs_label_reduce_x_kernel<<<label_grid(n * (a.cq / 4), RGS_SMS * 16), 256, 0, st>>>(a);
    const int64_t blocks_w = a.part_w ? (vocab * (a.cq / 4) + 31) / 32 : 0, blocks_b = db ? (vocab + 31) / 32 : 0;
    rgs_cuda_field_launches((a.part_x ? 1 : 0) + (blocks_w + blocks_b ? 1 : 0));
    if (blocks_w + blocks_b) rgs_label_reduce_w_kernel<<<(unsigned)(blocks_w + blocks_b), 512, 0, st>>>(a, (int)blocks_w, db, (int)b_dtype);
    return (int)cudaGetLastError();
}

}  // extern "C"

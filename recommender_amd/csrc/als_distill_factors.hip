// The distillation loss (als_distill.hip) straight from the factors: scores s_ui = <x_u, y_i>, loss and both gradients
//     dX_u = sum_i slope_ui y_i,   dY_i = sum_u slope_ui x_u,   slope_ui = c_u (q_ui - t_ui),  c_u = weight_u / T
// without a score matrix.  Two passes over the pairs (user, item), each a pair of chained matrix products on the fp16 matrix
// cores with the exponential between them in registers:
//   pass 1  users stationary, items streaming: s = x y^T, p = exp(s - running maximum), O += p y, Z += p; a user's O / Z is
//           sum_i q_ui y_i.  Split over the items; the parts are joined afterwards.
//   lists   per user: joins the parts, ln Z, the teacher's softmax, the loss, dX; and the list in item order.
//   pass 2  items stationary, users streaming: s again, q = exp(s - ln Z_u), minus the listed t, dY += (q - t) (c_u x_u).
// 8 n M f multiplications and additions, of which three products each: operands are two fp16 pieces of a value scaled by a
// power of two (22 mantissa bits) and hi hi + hi lo + lo hi are accumulated in float32 - about the accuracy of float32 products
// at several times their rate.  A power of two for each factor, and where the values' range is not the factors' own each has its
// own: a user's weights exp(s - maximum) in pass 1, a user's c x, and an item's q - t in pass 2 (cut to pieces times a power that
// follows its largest; user_exp, and g in pass_kernel).
//
// A handful of users leaves such tiles mostly empty: they take als_distill_few.inc's vector kernels instead.
//
// Layout.  v_mfma_f32_32x32x16_f16: operand A lane (h, i), h = lane / 32, holds row i, k = 8 h .. 8 h + 7; B lane (h, j)
// column j, the same k; the result's register r in lane (h, j) is row 8 (r / 4) + 4 h + r % 4, column j.  A 32 x 32 tile of
// scores [streaming row, stationary column] leaves a lane with 16 values of ONE column; taken as two k-steps of 8 they are
// the B operand of the second product, if the other operand's k runs over the streaming rows in the same order.  So nothing
// is exchanged between lanes, and both factors are laid out beforehand (prepare_kernel) as the lanes read them, per tile of
// 32 rows: row form (KS = F / 16 k-steps x 2 pieces) and transposed form (F / 32 feature tiles x 2 k-steps x 2 pieces), each
// 64 lanes x 16 bytes.  A stage is one tile: F / 4 KB, contiguous, copied to LDS by LDS-DMA.
//
// What bounds it (one MI355X).  24 n M f operations at the 1.18 PFLOP/s a large fp16 library product reaches here (at 1.6 GHz:
// power) are 315 us at 4096 x 59047, f = 64, and 666 us at 1023 x 250001, f = 128; whole calls take 423 to 436 and 873 to 882
// from card to card.  Under a profiler, which makes them 497 and 1018, the passes are 178 + 247 and 396 + 479 us: the matrix pipe is
// busy 66 and 44 % of their cycles at f = 64, 57 and 44 % at 128, and
// vector instructions take the rest (per tile and wave at f = 64: 24 matrix instructions of 32 cycles, 16 exponentials of 16,
// some 100 others of 4, which do not overlap them).  Pass 2 has the lists on top, and 231 blocks of items for 256 compute units.
// The other launches are memory: laying out 14 and 86 us, lists 42 and 25, the maxima 6 and 32.  Small calls are launches
// and latency: 64 x 9724, f = 20, 36 us in five launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "als_hip.h"

int als_fail_(int code, const char *fmt, ...);  // defined in als_kernels.hip

#define ALS_HIP_CHECK6(expr)                                                                      \
    do {                                                                                          \
        hipError_t e_ = (expr);                                                                   \
        if (e_ != hipSuccess) return als_fail_(ALS_ERR_HIP, "%s: %s", #expr, hipGetErrorString(e_)); \
    } while (0)

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
#include "als_fp16.inc"

constexpr int LIST_MAX = 1024;
constexpr int MAX_SPLITS = 512;
constexpr int TILE = 32;                // rows per tile, of either factor
constexpr int Y_MAX_BLOCKS = 1024, X_MAX_BLOCKS = 256;
constexpr int64_t ROWS_MAX = 1 << 27;   // of either factor: a launch takes fewer than 2^32 threads along x, here 256 per tile
constexpr int64_t GRID_X = 1 << 21;     // a workgroup per user: beyond that along y
constexpr float P_OFFSET = 9.f;         // pass 1: p 2^9, and at most 2^6 above the running maximum's: below 2^16, fp16's largest
constexpr float LAZY = 6.f;             // the running maximum follows when it lags by more than 2^6.  The lower piece holds a user's
                                        // weights to 2^-34 of the largest in its part, which a part's 32768 items make 2^-19 of the
                                        // sum.  (12 and 3, with more corrections: 2^-22 and 1 to 2 % more time)
constexpr int Q_TOP = 15, Q_ROOM = 6;   // pass 2: an item's q - t times a power of two that keeps them below 2^Q_TOP; when one passes
                                        // that, the power is set so that Q_ROOM bits are free above it
constexpr float NEVER = 1e30f;          // bias of a padding user: q = 0
constexpr int NO_SHARE = -(1 << 20);    // in place of an exponent: a user whose row adds nothing to dY
constexpr int CX_TOP = 15;              // a user's c x, as an operand, times the power of two that keeps it below 2^CX_TOP
constexpr int T_STRIDE = 36;            // floats per item column of the list tile: 16-byte aligned, columns on different banks

struct FactorArgs {
    const float *X, *Y;
    int64_t ldx, ldy;
    const int64_t *users;
    int64_t n, M, x_rows;
    int32_t f;
    const int32_t *t_idx;
    const float *t_val;
    int64_t ldt;
    int32_t k;
    float inv_t;
    const float *weight;
    float *loss, *dX, *dY;
    // workspace
    float *maxima;        // Y_MAX_BLOCKS of |y|, X_MAX_BLOCKS of |x|, X_MAX_BLOCKS of user_exp
    float *scales;        // {1 / (s_x s_y), 1 / s_y, exponent of dY's unit, largest user_exp}
    int32_t *user_exp;    // |c_u x_uk| < 2^user_exp[u], or NO_SHARE; NULL in the form for few users
    char *xt, *yt;        // the factors as tiles
    float *o_part;        // [split, user, F]
    float *stat_part;     // [split, user, 2]: running maximum (log2), sum
    float *bias;          // log2 Z_u less what the user's q carries, NEVER for padding
    int32_t *s_item;      // lists in item order [user, k]
    float *s_t;           // t, times what it carries
    uint16_t *offs;       // [user, item blocks + 1] first list entry at or behind the block
    float *dy_part;       // [split, item, F]
    int64_t n_tiles, m_tiles;
    int32_t splits1, splits2, item_blocks, block_items;
};

__device__ __forceinline__ float exp2_fast(const float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float finite_abs(const float v) { const float a = fabsf(v); return a < 3e38f ? a : 0.f; }

// The factor row of output row u, or NULL for a user id outside X.
__device__ __forceinline__ const float *user_row(const FactorArgs &a, const int64_t u) {
    const int64_t id = a.users ? a.users[u] : u;
    return id >= 0 && id < a.x_rows ? a.X + id * a.ldx : nullptr;
}

// Four factors of a row, zero beyond f.  VEC: one 16-byte load.
template <bool VEC>
__device__ __forceinline__ f32x4 load4(const float *row, const int c, const int f) {
    if constexpr (VEC) return c < f ? *reinterpret_cast<const f32x4 *>(row + c) : f32x4{0.f, 0.f, 0.f, 0.f};
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = c + e < f ? row[c + e] : 0.f;
    return v;
}
// v of another lane of the wave by a DPP move; lanes without a source get `none`
template <int CTRL, int ROWS>
__device__ __forceinline__ float moved(const float v, const float none) {
    return __uint_as_float((unsigned)__builtin_amdgcn_update_dpp((int)__float_as_uint(none), (int)__float_as_uint(v), CTRL, ROWS, 0xf, false));
}
// Over the workgroup's 256 threads.  In a wave: towards lane 63 (a row's 16 lanes, then across rows).
__device__ __forceinline__ float block_max256(float v, float *red) {
    const float none = -__builtin_inff();
    asm volatile("s_nop 1" : "+v"(v));      // a DPP move reads its register two states after the write, wherever that was
    v = fmaxf(v, moved<0x111, 0xf>(v, none));
    v = fmaxf(v, moved<0x112, 0xf>(v, none));
    v = fmaxf(v, moved<0x114, 0xf>(v, none));
    v = fmaxf(v, moved<0x118, 0xf>(v, none));
    v = fmaxf(v, moved<0x142, 0xa>(v, none));
    v = fmaxf(v, moved<0x143, 0xc>(v, none));
    __syncthreads();
    if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}
__device__ __forceinline__ float block_sum256(float v, float *red) {
    asm volatile("s_nop 1" : "+v"(v));
    v += moved<0x111, 0xf>(v, 0.f);
    v += moved<0x112, 0xf>(v, 0.f);
    v += moved<0x114, 0xf>(v, 0.f);
    v += moved<0x118, 0xf>(v, 0.f);
    v += moved<0x142, 0xa>(v, 0.f);
    v += moved<0x143, 0xc>(v, 0.f);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// ----------------------------------------------------------------------------- laying the factors out
// Over the sixteen lanes that share a row, in all of them.
__device__ __forceinline__ float max16(float v) {
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ bool any16(const bool v) { return (__ballot(v) >> (threadIdx.x & 48) & 0xffffu) != 0; }

// Whether a user's list has an entry that counts: of an item listed twice the first stands.  By the sixteen lanes of its row.
// first / first_val: entries l, l + 16, .., which the caller has loaded (-1 behind the list's end).
constexpr int FIRST = 8;
__device__ bool list_counts(const FactorArgs &a, const int64_t u, const int l, const int32_t (&first)[FIRST], const float (&first_val)[FIRST]) {
    const int32_t *idx = a.t_idx + u * a.ldt;
    const float *val = a.t_val + u * a.ldt;
    bool good = false, masked = false;
    auto see = [&](const int32_t i, const float v) {
        const bool in = i >= 0 && i < a.M, low = v == -__builtin_inff();
        good |= in && !low;
        masked |= in && low;
    };
#pragma unroll
    for (int q = 0; q < FIRST; ++q) see(first[q], first_val[q]);
#pragma unroll 4
    for (int p = l + 16 * FIRST; p < a.k; p += 16) see(idx[p], val[p]);
    good = any16(good);
    if (!good || !any16(masked)) return good;
    good = false;                                        // rare: only an item's first entry may count, and that may be a masked one
    for (int p = l; p < a.k && !good; p += 16) {
        if (idx[p] < 0 || idx[p] >= a.M || val[p] == -__builtin_inff()) continue;
        good = true;
        for (int q = 0; q < p && good; ++q) good = idx[q] != idx[p];
    }
    return any16(good);
}

// Exponents of the parts of c x: v = m 2^e, 0.5 <= |m| < 1; 0 for what is 0 or not finite.
__device__ __forceinline__ int exponent(const float v) {
    int e = 0;
    if (fabsf(v) < __builtin_inff() && v != 0.f) (void)frexpf(v, &e);
    return e;
}

// Largest |y| and |x| (finite ones) and largest user_exp, one value per block: the reader takes the maximum over blocks.
//
// A user's weight, and with it the size of c_u x_u, is the caller's choice: one power of two for all users would let the
// largest weight, which may be that of an empty list, take the others' bits.  So every user has its own, which pass 2 carries in
// q and t instead: (q - t) 2^(user_exp - largest) times c x 2^-user_exp.
template <bool VEC>
__global__ __launch_bounds__(256) void maxima_kernel(const FactorArgs a) {
    __shared__ float red[4];
    // the users' blocks first: theirs are chains of loads, beside which the items stream
    const bool is_y = blockIdx.x >= X_MAX_BLOCKS;
    const int b = is_y ? blockIdx.x - X_MAX_BLOCKS : blockIdx.x, nb = is_y ? Y_MAX_BLOCKS : X_MAX_BLOCKS;
    const int64_t rows = is_y ? a.M : a.n;
    float m = 0.f, mc = (float)NO_SHARE;
    // rows without gaps are one long row (500 000 x 33: 36 us otherwise); of others sixteen lanes take a row at a time
    const bool flat = is_y && a.ldy == a.f && (uintptr_t)a.Y % 16 == 0;
    if (flat) {
        const int64_t quads = a.M * a.f / 4, rest = 4 * quads + threadIdx.x;
        const f32x4 *y = reinterpret_cast<const f32x4 *>(a.Y);
#pragma unroll 4
        for (int64_t q = (int64_t)b * 256 + threadIdx.x; q < quads; q += (int64_t)nb * 256) {
            const f32x4 v = y[q];
#pragma unroll
            for (int e = 0; e < 4; ++e) m = fmaxf(m, finite_abs(v[e]));
        }
        if (b == 0 && rest < a.M * a.f) m = fmaxf(m, finite_abs(a.Y[rest]));
    }
    if (!flat) for (int64_t r = (int64_t)b * 16 + (threadIdx.x >> 4); r < rows; r += (int64_t)nb * 16) {
        const int l = threadIdx.x & 15;
        const float w = !is_y && a.weight ? a.weight[r] : 1.f;
        int32_t first[FIRST];
        float first_val[FIRST];
        if (!is_y) {                                     // under way beside the user's id
#pragma unroll
            for (int q = 0; q < FIRST; ++q) {
                const int p = l + 16 * q;
                first[q] = p < a.k ? a.t_idx[r * a.ldt + p] : -1;
                first_val[q] = p < a.k ? a.t_val[r * a.ldt + p] : 0.f;
            }
        }
        const float *row = is_y ? a.Y + r * a.ldy : user_row(a, r);
        float mr = 0.f;
        if (row)
            for (int k = 4 * (threadIdx.x & 15); k < a.f; k += 64) {
                const f32x4 v = load4<VEC>(row, k, a.f);
#pragma unroll
                for (int e = 0; e < 4; ++e) mr = fmaxf(mr, finite_abs(v[e]));
            }
        m = fmaxf(m, mr);
        if (!is_y) {                                     // all sixteen lanes: r is one for them
            mr = max16(mr);
            const bool share = list_counts(a, r, l, first, first_val) && row && mr > 0.f && w != 0.f;
            const int e = share ? exponent(mr) + exponent(w) + exponent(a.inv_t) : NO_SHARE;
            if (l == 0) a.user_exp[r] = e;
            if (fabsf(w) < __builtin_inff()) mc = fmaxf(mc, (float)e);
        }
    }
    m = block_max256(m, red);
    mc = block_max256(mc, red);
    if (threadIdx.x == 0) {
        a.maxima[is_y ? b : Y_MAX_BLOCKS + b] = m;
        if (!is_y) a.maxima[Y_MAX_BLOCKS + X_MAX_BLOCKS + b] = mc;
    }
}

// hi and lo fp16 pieces of v.  (Of the float32 v: left to itself the compiler takes a product into the conversion, and hi is
// then that of another rounding than the v whose rest is lo.)
__device__ __forceinline__ void cut(float v, _Float16 &hi, _Float16 &lo) {
    asm volatile("" : "+v"(v));
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

__device__ __forceinline__ int within(const int e) { return e < -126 ? -126 : e > 126 ? 126 : e; }
__device__ __forceinline__ float power(const int e) { return ldexpf(1.f, within(e)); }      // 2^e

// One tile of 32 rows per workgroup: through LDS, then both forms.  Tiles of Y first, then of X (whose row form carries
// log2(e) / T and whose transposed form carries c_u 2^-user_exp).
template <int F>
__global__ __launch_bounds__(256) void prepare_kernel(const FactorArgs a) {
    constexpr int KS = F / 16, FT = F / 32;
    __shared__ float tile[TILE][F + 1];
    __shared__ float red[4], cs[TILE];
    __shared__ int xe[TILE];
    const int tid = threadIdx.x;
    const bool is_y = blockIdx.x < a.m_tiles;
    const int64_t T = is_y ? blockIdx.x : blockIdx.x - a.m_tiles;
    const int64_t rows = is_y ? a.M : a.n;
    float my = 0.f, mx = a.maxima[Y_MAX_BLOCKS + tid], mc = a.maxima[Y_MAX_BLOCKS + X_MAX_BLOCKS + tid];      // X_MAX_BLOCKS = 256
#pragma unroll
    for (int q = 0; q < Y_MAX_BLOCKS; q += 256) my = fmaxf(my, a.maxima[q + tid]);
    for (int q = tid; q < TILE * F; q += 256) {
        const int i = q / F, k = q % F;
        const int64_t r = T * TILE + i;
        const float *row = r >= rows ? nullptr : is_y ? a.Y + r * a.ldy : user_row(a, r);
        tile[i][k] = row && k < a.f ? row[k] : 0.f;
    }
    if (tid < TILE) {
        const int64_t r = T * TILE + tid;
        const bool user = !is_y && r < rows;
        const int own_exp = user ? a.user_exp[r] : NO_SHARE;
        const float w = user && a.weight ? a.weight[r] : 1.f;
        const int ew = exponent(w), et = exponent(a.inv_t);
        float c = 0.f;                                   // users without a share, whatever their weight: 0
        int e = 0;
        if (own_exp != NO_SHARE) {
            e = ew + et - own_exp;                       // of x alone
            c = ldexpf(w, -ew) * ldexpf(a.inv_t, CX_TOP - et);
        }
        cs[tid] = c;
        xe[tid] = e;
    }
    my = block_max256(my, red);                          // the first of them waits for the tile as well
    mx = block_max256(mx, red);
    mc = block_max256(mc, red);
    // both factors times a power of two that keeps them below 2^15, X times log2(e) / T besides
    const float to_log2 = a.inv_t * 1.44269504f;
    const int ex = within(15 - exponent(mx)), ey = within(15 - exponent(my)), el = exponent(to_log2);
    const float sy = power(ey), sx = ldexpf(to_log2, -el) * power(ex);
    if (blockIdx.x == 0 && tid == 0) {
        const int top = mc > (float)NO_SHARE ? (int)mc : 0;
        a.scales[0] = power(el - ex - ey);
        a.scales[1] = power(-ey);
        a.scales[2] = (float)(top - CX_TOP);
        a.scales[3] = (float)top;
    }
    char *out = (is_y ? a.yt : a.xt) + T * (F * 256);
    const float s_row = is_y ? sy : sx;
    for (int q = tid; q < KS * 64; q += 256) {
        const int ks = q >> 6, lane = q & 63, h = lane >> 5, i = lane & 31;
        f16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            _Float16 x, y;
            cut(tile[i][16 * ks + 8 * h + e] * s_row, x, y);
            hi[e] = x; lo[e] = y;
        }
        *reinterpret_cast<f16x8 *>(out + (2 * ks) * 1024 + lane * 16) = hi;
        *reinterpret_cast<f16x8 *>(out + (2 * ks + 1) * 1024 + lane * 16) = lo;
    }
    for (int q = tid; q < FT * 2 * 64; q += 256) {
        const int fk = q >> 6, ft = fk >> 1, kk = fk & 1, lane = q & 63, h = lane >> 5, i = lane & 31;
        f16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int row = 16 * kk + 8 * (e / 4) + 4 * h + e % 4;
            _Float16 x, y;
            cut(is_y ? tile[row][32 * ft + i] * sy : ldexpf(tile[row][32 * ft + i], xe[row]) * cs[row], x, y);
            hi[e] = x; lo[e] = y;
        }
        *reinterpret_cast<f16x8 *>(out + (2 * KS + 2 * fk) * 1024 + lane * 16) = hi;
        *reinterpret_cast<f16x8 *>(out + (2 * KS + 2 * fk + 1) * 1024 + lane * 16) = lo;
    }
}

// ----------------------------------------------------------------------------- the two passes
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"      // m0 is reserved, and written here on purpose: the LDS address of the DMA
// 64 lanes x 16 bytes from g (per lane) to LDS bytes [lds, lds + 1024), lane l at 16 l
__device__ __forceinline__ void dma16(const void *g, const unsigned lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                 :: "v"(g), "s"(__builtin_amdgcn_readfirstlane((int)lds)) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ f32x16 mfma32(const u32x4 &a, const u32x4 &b, const f32x16 &c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// p0 g and p1 g, g a power of two, as fp16 pairs of both pieces, each rounded to nearest: what is lost of p g is unbiased and at
// most 2^-22 of it or 2^-25.  g is in a register that the compiler does not look into, so that p g - hi is one instruction
// also where g is 1; and the rests are made opaque too: taken into the conversion, as two instructions that leave a half each, they
// take longer (443 us for 437 at f = 64).
__device__ __forceinline__ void cut_rest(const float p0, const float p1, const float g, const unsigned hi, unsigned &lo) {
    float r0 = __builtin_fmaf(p0, g, -f16_lo(hi)), r1 = __builtin_fmaf(p1, g, -f16_hi(hi));
    asm volatile("" : "+v"(r0), "+v"(r1));
    lo = pack_f16(r0, r1);
}
__device__ __forceinline__ float power_inverse(const float p) { return __uint_as_float(0x7f000000u - __float_as_uint(p)); }

// BACK = false: pass 1 (stationary X, streaming Y).  BACK = true: pass 2 (stationary Y, streaming X, lists).
// A wave owns one stationary tile (32 rows: operands and result in registers); the WAVES waves of a workgroup share the
// streaming tiles in LDS.  RING tiles are kept: the copy of tile t + RING - 1 starts while tile t is worked on.
// Workgroup (split, block): the ids of one split go to one XCD, so that the blocks that stream the same tiles share its L2.
template <int F, int WAVES, int RING, bool BACK>
__global__ __launch_bounds__(WAVES * 64, F <= 64 ? 4 : 1) void pass_kernel(const FactorArgs a) {
    constexpr int KS = F / 16, FT = F / 32, CHUNKS = F / 4, PER_WAVE = CHUNKS / WAVES;
    constexpr int LPR = WAVES * 2;                       // lanes that write one user's row of the list tile
    static_assert(CHUNKS % WAVES == 0, "every wave copies the same number of chunks");
    constexpr int LDS_BYTES = RING * CHUNKS * 1024 + (BACK ? (WAVES * T_STRIDE + 1) * 32 * 4 : 0);
    static_assert(LDS_BYTES <= 160 * 1024, "LDS");
    __shared__ __attribute__((aligned(16))) char lds[LDS_BYTES];
    u32x4 *ring = reinterpret_cast<u32x4 *>(lds);                                   // RING x CHUNKS x 64
    float *t_tile = reinterpret_cast<float *>(lds + RING * CHUNKS * 1024);          // BACK: WAVES * 32 x T_STRIDE
    float *bias = t_tile + WAVES * 32 * T_STRIDE;                                   // BACK: 32
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, j = lane & 31;
    const int splits = BACK ? a.splits2 : a.splits1;
    const int64_t stat_tiles = BACK ? a.m_tiles : a.n_tiles, stream_tiles = BACK ? a.n_tiles : a.m_tiles;
    const int64_t blocks = (stat_tiles + WAVES - 1) / WAVES;
    const int64_t w = blockIdx.x;
    const int group = splits >= 8 ? 8 : 1;               // splits is a multiple of 8 from 8 on
    const int64_t block = (w / group) % blocks;
    const int split = (int)(w / (group * blocks)) * group + (int)(w % group);
    const int64_t per = (stream_tiles + splits - 1) / splits;
    const int64_t t0 = split * per, t1 = t0 + per < stream_tiles ? t0 + per : stream_tiles;       // the host leaves no split empty
    const char *stat = (BACK ? a.yt : a.xt);
    const char *stream = (BACK ? a.xt : a.yt);
    const int64_t tile = block * WAVES + wave;
    const bool active = tile < stat_tiles;

    const unsigned ring_base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    auto copy = [&](const int64_t t, const int slot) {
        // past the range's end the last tile is copied again: every stage issues the same number of copies
        const char *src = stream + (t < t1 ? t : t1 - 1) * (F * 256) + lane * 16;
#pragma unroll
        for (int q = 0; q < PER_WAVE; ++q) {
            const int c = wave * PER_WAVE + q;
            dma16(src + c * 1024, ring_base + (slot * CHUNKS + c) * 1024);
        }
    };

    // under way while the rest is set up (F = 128: 365 us, 420 with the copies behind that; in pass 2, where they are less of the
    // work, 474 and 430)
    constexpr bool EARLY = !BACK || F <= 64;
    if constexpr (EARLY) {
#pragma unroll
        for (int q = 0; q < RING - 1; ++q) copy(t0 + q, q);
    }
    u32x4 BH[KS], BL[KS];
    {
        const u32x4 *src = reinterpret_cast<const u32x4 *>(stat + (active ? tile : 0) * (F * 256)) + lane;
#pragma unroll
        for (int s = 0; s < KS; ++s) { BH[s] = src[(2 * s) * 64]; BL[s] = src[(2 * s + 1) * 64]; }
    }
    // waited for before the loop (pin): in it, their waits would also wait, every time, for the copies under way
    auto pin = [&]() {
#pragma unroll
        for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(BH[s]), "+v"(BL[s]));
    };
    f32x16 O[FT];
#pragma unroll
    for (int q = 0; q < FT; ++q)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[q][r] = 0.f;
    const float k = a.scales[0];
    float m = -__builtin_inff();
    double z = 0.0;                                      // of a lane: up to half of all items, a tile's sixteen in float32
    float one = 1.f;
    asm volatile("" : "+s"(one));
    // pass 2: O is sum_u (q - t) g x_u.  One g for all items would leave the q of a large catalogue, 10^-6 of the t's, few bits
    // (16 at a million items); so each item (a lane and its other half's lane) has its own, which follows its largest
    // |q - t| downwards and leaves that one its 22 bits (f = 64: 433 us a call, 425 with one g; f = 128: 887 and 875).
    float g = 0x1p126f;                                  // |q - t| <= 1: a new one is 2^8 at the least

    // ---- pass 2: the lists of the streaming users, as a dense tile [item of the block, user of the stage] that is zero but
    // for the listed pairs.  LPR lanes of a wave own a user's row: between two barriers they clear what they wrote there for
    // the last stage and write the new entries, which they loaded a stage ahead.  A second tile in place of the second barrier
    // leaves room for one workgroup per compute unit (f = 64: 276 us, 237 with one tile).  Also measured there: each wave on
    // its own 32 items without that barrier 254-270, entries loaded a stage after their ranges 246, 32-bit addresses 258.
    const int row = BACK ? tid / LPR : 0, sub = BACK ? tid % LPR : 0;
    const int64_t i_first = block * WAVES * 32;
    const uint16_t *offs = BACK ? a.offs + block : nullptr;
    struct Entries { int b, e, item; float t, bias; };
    Entries now{0, 0, 0, 0.f, NEVER}, old = now;
    auto fetch = [&](const int64_t t) {                  // the first LPR entries of the row's user in stage t
        Entries x{0, 0, 0, 0.f, NEVER};
        const int64_t u = t * TILE + row;
        if (t < t1 && sub == 0) x.bias = a.bias[u];      // padding users have one too
        if (t < t1 && u < a.n) {
            const uint16_t *o = offs + (uint64_t)(uint32_t)u * (uint32_t)(a.item_blocks + 1);
            x.b = o[0]; x.e = o[1];
            const uint64_t at = (uint64_t)(uint32_t)u * (uint32_t)a.k + (uint32_t)(x.b + sub);
            if (x.b + sub < x.e) { x.item = a.s_item[at]; x.t = a.s_t[at]; }
        }
        return x;
    };
    auto place = [&](const int64_t t) {                  // writes `now`, the entries of stage t
        if (old.b + sub < old.e) t_tile[(old.item - i_first) * T_STRIDE + row] = 0.f;
        const int64_t u = t * TILE + row;
        for (int q = old.b + sub + LPR; q < old.e; q += LPR) t_tile[(a.s_item[(u - TILE) * a.k + q] - i_first) * T_STRIDE + row] = 0.f;
        if (now.b + sub < now.e) t_tile[(now.item - i_first) * T_STRIDE + row] = now.t;
        for (int q = now.b + sub + LPR; q < now.e; q += LPR)
            t_tile[(a.s_item[u * a.k + q] - i_first) * T_STRIDE + row] = a.s_t[u * a.k + q];
        old = now;
        if (sub == 0) bias[row] = now.bias;
    };

    if constexpr (BACK) {
        for (int q = tid; q < WAVES * 32 * T_STRIDE / 4; q += WAVES * 64) reinterpret_cast<f32x4 *>(t_tile)[q] = f32x4{0.f, 0.f, 0.f, 0.f};
        now = fetch(t0);
        pin();
        __syncthreads();
        place(t0);
        now = fetch(t0 + 1);
    } else {
        pin();
    }
    if constexpr (!EARLY) {
#pragma unroll
        for (int q = 0; q < RING - 1; ++q) copy(t0 + q, q);
    }
    int slot = 0;
    for (int64_t t = t0; t < t1; ++t) {
        // this wave's copies of tile t have landed (behind them it issued RING - 2 further tiles, and maybe list loads, which
        // only make the count stricter); after the barrier everyone's have, and everyone is done with tile t - 1
        asm volatile("s_waitcnt vmcnt(%0)" :: "n"((RING - 2) * PER_WAVE) : "memory");
        __syncthreads();
        copy(t + RING - 1, slot == 0 ? RING - 1 : slot - 1);
        const u32x4 *st = ring + slot * CHUNKS * 64 + lane;
        slot = slot + 1 == RING ? 0 : slot + 1;
        if (active) {
        f32x16 S;
#pragma unroll
        for (int r = 0; r < 16; ++r) S[r] = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const u32x4 ah = st[(2 * s) * 64], al = st[(2 * s + 1) * 64];
            S = mfma32(al, BH[s], S);
            S = mfma32(ah, BL[s], S);
            S = mfma32(ah, BH[s], S);
        }
        unsigned PH[8], PL[8];
        if constexpr (!BACK) {
            if ((t + 1) * TILE > a.M) {                  // the last tile's padding rows
                const int rows = (int)(a.M - t * TILE) - 4 * h;
                asm volatile("" ::: "memory");           // stays a branch: taken into the loop, it is 48 instructions a tile
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (8 * (r / 4) + r % 4 >= rows) S[r] = -__builtin_inff();
            }
            float top = S[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) top = fmaxf(top, S[r]);
            top *= k;
            if (__any(top > m + LAZY)) {
                // only where it lags: a user's sums must not depend on what else its wave works on
                top = fmaxf(top, __shfl_xor(top, 32));
                const float next = top > m + LAZY ? top : m;
                const float scale = m == -__builtin_inff() ? 0.f : exp2_fast(m - next);
                m = next;
                z *= (double)scale;
#pragma unroll
                for (int q = 0; q < FT; ++q)
#pragma unroll
                    for (int r = 0; r < 16; ++r) O[q][r] *= scale;
            }
            const float c = P_OFFSET - m;
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float p0 = exp2_fast(__builtin_fmaf(S[r], k, c)), p1 = exp2_fast(__builtin_fmaf(S[r + 1], k, c));
                sum += p0 + p1;
                PH[r / 2] = pack_f16_pinned(p0, p1);
                cut_rest(p0, p1, one, PH[r / 2], PL[r / 2]);
            }
            z += (double)sum;
        } else {
            const f32x4 *tt = reinterpret_cast<const f32x4 *>(t_tile + (wave * 32 + j) * T_STRIDE) + h;
            const f32x4 *bb = reinterpret_cast<const f32x4 *>(bias) + h;
            float top = 0.f;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const f32x4 tv = tt[2 * b], bv = bb[2 * b];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    S[4 * b + e] = exp2_fast(__builtin_fmaf(S[4 * b + e], k, -bv[e])) - tv[e];
                    top = fmaxf(top, fabsf(S[4 * b + e]));
                }
                if (F == 64) __builtin_amdgcn_sched_barrier(0);     // these two keep the form of four waves per SIMD from spilling
            }
            if (__any(top * g > (float)(1 << Q_TOP))) {
                top = fmaxf(top, __shfl_xor(top, 32));
                // 2^(Q_TOP - Q_ROOM - 1) <= top next < twice that; the power from the exponent's bits
                const float next = __uint_as_float((unsigned)(253 + Q_TOP - Q_ROOM) * 0x800000u - (__float_as_uint(top) & 0x7f800000u));
                const float scale = top * g > (float)(1 << Q_TOP) ? next * power_inverse(g) : 1.f;
                g *= scale;
#pragma unroll
                for (int q = 0; q < FT; ++q)
#pragma unroll
                    for (int r = 0; r < 16; ++r) O[q][r] *= scale;
            }
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                PH[r / 2] = pack_f16_pinned(S[r] * g, S[r + 1] * g);
                cut_rest(S[r], S[r + 1], g, PH[r / 2], PL[r / 2]);
                if (F == 64) __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int q = 0; q < FT; ++q)
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const u32x4 vh = st[(2 * KS + 4 * q + 2 * kk) * 64], vl = st[(2 * KS + 4 * q + 2 * kk + 1) * 64];
                const u32x4 ph{PH[4 * kk], PH[4 * kk + 1], PH[4 * kk + 2], PH[4 * kk + 3]};
                const u32x4 pl{PL[4 * kk], PL[4 * kk + 1], PL[4 * kk + 2], PL[4 * kk + 3]};
                O[q] = mfma32(vl, ph, O[q]);
                O[q] = mfma32(vh, pl, O[q]);
                O[q] = mfma32(vh, ph, O[q]);
            }
        }
        if constexpr (BACK) {                            // the next entries go in when everyone has read these
            __syncthreads();
            place(t + 1);
            now = fetch(t + 2);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // no copy is left in flight
    if (!active) return;
    const int64_t r = tile * TILE + j;                   // this lane's stationary row
    if constexpr (!BACK) {
        z += __shfl_xor(z, 32);
        if (r < a.n) {
            const int64_t at = (int64_t)split * a.n + r;
            if (h == 0) { a.stat_part[2 * at] = m; a.stat_part[2 * at + 1] = (float)z; }
#pragma unroll
            for (int q = 0; q < FT; ++q)
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    *reinterpret_cast<f32x4 *>(a.o_part + at * F + 32 * q + 8 * b + 4 * h) =
                        f32x4{O[q][4 * b], O[q][4 * b + 1], O[q][4 * b + 2], O[q][4 * b + 3]};
        }
    } else if (r < a.M) {
        const float inv_g = power_inverse(g);
        if (splits == 1) {
            const int unit = (int)a.scales[2];
            const bool quads = a.f % 4 == 0 && (uintptr_t)a.dY % 16 == 0;
#pragma unroll
            for (int q = 0; q < FT; ++q)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int c = 32 * q + 8 * b + 4 * h;
                    const f32x4 v{ldexpf(O[q][4 * b] * inv_g, unit), ldexpf(O[q][4 * b + 1] * inv_g, unit),
                                  ldexpf(O[q][4 * b + 2] * inv_g, unit), ldexpf(O[q][4 * b + 3] * inv_g, unit)};
                    float *dst = a.dY + r * a.f + c;
                    if (quads) {
                        if (c < a.f) *reinterpret_cast<f32x4 *>(dst) = v;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (c + e < a.f) dst[e] = v[e];
                    }
                }
        } else {
            const int64_t at = (int64_t)split * a.M + r;
#pragma unroll
            for (int q = 0; q < FT; ++q)
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    *reinterpret_cast<f32x4 *>(a.dy_part + at * F + 32 * q + 8 * b + 4 * h) =
                        f32x4{O[q][4 * b] * inv_g, O[q][4 * b + 1] * inv_g, O[q][4 * b + 2] * inv_g, O[q][4 * b + 3] * inv_g};
        }
    }
}

// dY from the parts of pass 2, in split order.
__global__ __launch_bounds__(256) void join_items_kernel(const FactorArgs a, const int F) {
    const int unit = (int)a.scales[2];
    const int64_t total = a.M * a.f;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total; q += (int64_t)gridDim.x * 256) {
        const int64_t i = q / a.f;
        const int c = (int)(q - i * a.f);
        float v = 0.f;
        for (int s = 0; s < a.splits2; ++s) v += a.dy_part[((int64_t)s * a.M + i) * F + c];
        a.dY[q] = ldexpf(v, unit);
    }
}

// ----------------------------------------------------------------------------- lists
// One workgroup per user (and per padding user of the last tile, which only gets its bias).  Sixteen lanes work on one
// listed item, sixteen items at a time, four floats per lane and 64 factors; VEC: the rows allow 16-byte loads.  K_MAX: lists of up to
// 256 items leave room for eight workgroups per compute unit (4096 x 59047, f = 64, k = 100: 439 us for all of distill_topk, 448
// with room for 1024).
__device__ __forceinline__ float sum16(float v) {
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

template <int F, bool VEC, int K_MAX>
__global__ __launch_bounds__(256) void lists_kernel(const FactorArgs a) {
    constexpr int NC = F <= 64 ? 1 : F / 64;        // float4 per lane and item
    constexpr int QUADS = F / 4, GROUPS = 256 / QUADS;
    __shared__ uint64_t key[K_MAX];              // item << 32 | position, ~0 for padding
    __shared__ int32_t sorted[K_MAX];
    __shared__ float sorted_t[K_MAX];
    __shared__ f32x4 part[16][QUADS], o_sum[GROUPS][QUADS];
    __shared__ float x[F], red[4], loss_part[16], scale[MAX_SPLITS];
    __shared__ int32_t n_kept, n_again;
    const int tid = threadIdx.x;
    const int64_t u = (int64_t)blockIdx.y * GRID_X + blockIdx.x;
    if (u >= a.n) {
        if (tid == 0 && u < a.n_tiles * TILE) a.bias[u] = NEVER;
        return;
    }
    const int f = a.f;
    const float *xrow = user_row(a, u);
    if (!xrow) {                                         // no such user: NaN for it, nothing for the items
        if (tid == 0) { a.bias[u] = NEVER; a.loss[u] = __builtin_nanf(""); }
        if (tid < f) a.dX[u * f + tid] = __builtin_nanf("");
        for (int64_t b = tid; b <= a.item_blocks; b += 256) a.offs[u * (a.item_blocks + 1) + b] = 0;
        return;
    }
    // everything that is read whatever the list holds, at once
    constexpr int OWN = K_MAX / 256, S_OWN = MAX_SPLITS / 256;
    const int quad = tid % QUADS, o_first = tid / QUADS;
    const float *o_src = a.o_part + u * F + 4 * quad;
    const float x_own = tid < f ? xrow[tid] : 0.f;
    // what the user's row of the c x operand carries less than the largest, its q and t in pass 2 carry
    const int own_exp = a.user_exp ? a.user_exp[u] : 0;
    const int shift = a.user_exp && own_exp != NO_SHARE ? own_exp - (int)a.scales[3] : 0;
    uint64_t own[OWN];
    float own_val[OWN], m_own[S_OWN], z_own[S_OWN];
#pragma unroll
    for (int b = 0; b < OWN; ++b) {
        const int p = tid + 256 * b;
        const int32_t i = p < a.k ? a.t_idx[u * a.ldt + p] : -1;
        own_val[b] = p < a.k ? a.t_val[u * a.ldt + p] : 0.f;
        own[b] = i >= 0 && i < a.M ? (uint64_t)(uint32_t)i << 32 | (uint32_t)p : ~0ull;
    }
#pragma unroll
    for (int b = 0; b < S_OWN; ++b) {
        const int64_t at = (int64_t)(tid + 256 * b) * a.n + u;
        m_own[b] = tid + 256 * b < a.splits1 ? a.stat_part[2 * at] : -__builtin_inff();
        z_own[b] = tid + 256 * b < a.splits1 ? a.stat_part[2 * at + 1] : 0.f;
    }
    f32x4 o{0.f, 0.f, 0.f, 0.f};
    if (o_first < a.splits1) o = *reinterpret_cast<const f32x4 *>(o_src + (int64_t)o_first * a.n * F);
    if (tid < F) x[tid] = x_own;
#pragma unroll
    for (int b = 0; b < OWN; ++b)
        if (tid + 256 * b < a.k) key[tid + 256 * b] = own[b];
    if (tid == 0) { n_kept = 0; n_again = 0; }
    // the parts of pass 1
    float hi = fmaxf(m_own[0], m_own[S_OWN - 1]);
    hi = block_max256(hi, red);
    float z = 0.f;
#pragma unroll
    for (int b = 0; b < S_OWN; ++b) {
        const float c = exp2_fast(m_own[b] - hi);
        if (tid + 256 * b < a.splits1) {
            scale[tid + 256 * b] = c;
            z += z_own[b] * c;
        }
    }
    z = block_sum256(z, red);
    // of an item listed twice the first entry stands
    float top = -__builtin_inff();
    int rank[OWN];                                       // entries in front of the own one in item order
    bool keep[OWN];
#pragma unroll
    for (int b = 0; b < OWN; ++b) {
        rank[b] = 0; keep[b] = false;
        if (tid + 256 * b >= a.k || own[b] == ~0ull) continue;
        bool again = false;
#pragma unroll 8
        for (int q = 0; q < a.k; ++q) {
            const uint64_t other = key[q];
            const bool before = other < own[b];
            rank[b] += before;
            again |= before & ((other ^ own[b]) >> 32 == 0);
        }
        keep[b] = !again;
        if (again) n_again = 1;
        else top = fmaxf(top, own_val[b] == own_val[b] ? own_val[b] : __builtin_inff());      // NaN: not an empty list
    }
    top = block_max256(top, red);
    const bool any = top != -__builtin_inff();           // a list without weight asks for nothing
    float sum = 0.f, share[OWN];
#pragma unroll
    for (int b = 0; b < OWN; ++b) {
        keep[b] = keep[b] && any;
        share[b] = keep[b] ? expf((own_val[b] - top) * a.inv_t) : 0.f;
        sum += share[b];
        if (keep[b]) atomicAdd(&n_kept, 1);
        else if (tid + 256 * b < a.k) key[tid + 256 * b] = ~0ull;
    }
    sum = block_sum256(sum, red);
    const int n_list = n_kept;
    // item order, by rank among the kept
#pragma unroll
    for (int b = 0; b < OWN; ++b) {
        if (!keep[b]) continue;
        if (n_again) {
            rank[b] = 0;
            for (int q = 0; q < a.k; ++q) rank[b] += key[q] < own[b];
        }
        const float t = share[b] / sum;
        sorted[rank[b]] = (int32_t)(own[b] >> 32);
        sorted_t[rank[b]] = t;
        a.s_item[u * a.k + rank[b]] = (int32_t)(own[b] >> 32);
        a.s_t[u * a.k + rank[b]] = own_exp != NO_SHARE ? ldexpf(t, shift) : 0.f * t;
    }
    __syncthreads();
    for (int64_t b = tid; b <= a.item_blocks; b += 256) {
        const int64_t first = b * a.block_items;
        int lo = 0, end = n_list;
        while (lo < end) {
            const int mid = (lo + end) >> 1;
            if (sorted[mid] < first) lo = mid + 1;
            else end = mid;
        }
        a.offs[u * (a.item_blocks + 1) + b] = (uint16_t)lo;
    }
    // a list without weight: c (q - t) must be 0 for all items, so its user's q is switched off
    if (tid == 0) a.bias[u] = any && own_exp != NO_SHARE ? hi + log2f(z) - P_OFFSET - (float)shift : NEVER;
    const float lse = (hi + log2f(z) - P_OFFSET) * 0.69314718f;      // ln Z of s / T
    // the listed items: t y summed, <x, y> for the loss
    const int group = tid >> 4, l = tid & 15;
    f32x4 acc[NC];
    float loss = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    constexpr int AHEAD = NC == 1 ? 4 : 2;               // items whose rows are under way together
    for (int p0 = group; p0 < n_list; p0 += 16 * AHEAD) {
        f32x4 v[AHEAD][NC];
        float ts[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int p = p0 + 16 * i < n_list ? p0 + 16 * i : p0;
            const float *y = a.Y + (int64_t)sorted[p] * a.ldy;
            ts[i] = p0 + 16 * i < n_list ? sorted_t[p] : 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c) v[i][c] = 64 * c + 4 * l < F ? load4<VEC>(y, 64 * c + 4 * l, f) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const float t = ts[i];
            float dot = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int k0 = 64 * c + 4 * l;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    dot = fmaf(v[i][c][e], k0 < F ? x[k0 + e] : 0.f, dot);
                    acc[c][e] = fmaf(t, v[i][c][e], acc[c][e]);
                }
            }
            dot = sum16(dot);
            if (t != 0.f) loss += t * (logf(t) - (dot * a.inv_t - lse));
        }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
        if (64 * c + 4 * l < F) part[group][16 * c + l] = acc[c];
    if (l == 0) loss_part[group] = loss;
    // O, its parts dealt out over the threads by four factors and split
    {
        if (o_first < a.splits1) o *= scale[o_first];
#pragma unroll 4
        for (int s = o_first + GROUPS; s < a.splits1; s += GROUPS)
            o += *reinterpret_cast<const f32x4 *>(o_src + (int64_t)s * a.n * F) * scale[s];
        o_sum[o_first][quad] = o;
    }
    __syncthreads();
    if (tid < 16) {
        const float all = sum16(loss_part[tid]);
        if (tid == 0) a.loss[u] = any ? all : 0.f;
    }
    if (tid < QUADS && 4 * tid < f) {
        f32x4 o = o_sum[0][tid], listed = part[0][tid];
#pragma unroll 3
        for (int g = 1; g < GROUPS; ++g) o += o_sum[g][tid];
#pragma unroll 3
        for (int g = 1; g < 16; ++g) listed += part[g][tid];
        const float c = (a.weight ? a.weight[u] : 1.f) * a.inv_t, inv = 1.f / z, unit = a.scales[1];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (4 * tid + e < f) a.dX[u * f + 4 * tid + e] = any ? c * (o[e] * inv * unit - listed[e]) : 0.f;
    }
}

#include "als_distill_few.inc"

// ----------------------------------------------------------------------------- host
int padded_factors(const int32_t f) { return f <= 32 ? 32 : f <= 64 ? 64 : f <= 128 ? 128 : 256; }
// Up to how many users take als_distill_few's kernels, which hold their rows and O in registers.  Few / tiles in us: 1 x 9724,
// f = 20, 22 / 31, four users 29 / 31, eight 40 / 32; 8 x 59047, f = 64, 47 / 50; 8 x 1000003, f = 20, 201 / 249, f = 128, 389 / 1007;
// 4 x 1000003, f = 256, 515 / 2269.
int few_users(const int F, const int64_t M) { return F == 256 || M < 65536 ? 4 : 8; }
int waves_of(const int F) { return F == 256 ? 4 : 8; }

struct Plan {
    int F, waves, splits1, splits2, item_blocks;
    bool few;
    int64_t n_tiles, m_tiles;
    size_t off_scales, off_xt, off_yt, off_o, off_stat, off_bias, off_item, off_t, off_offs, off_dy, off_exp, total;
};

// Splits of a pass over `stream` tiles for `blocks` workgroups: enough workgroups for 512 (two per compute unit), at least
// 8 tiles each (fewer do not end sooner: a workgroup's start takes as long as 8 tiles), a multiple of 8 from 8 on (one XCD
// per split), none empty.  And at most SPLIT_TILES each, as long as a launch takes them: a float32 sum that has grown long loses
// whatever small terms follow.
constexpr int64_t SPLIT_TILES = 1024;
int split_count(const int64_t blocks, const int64_t stream) {
    int64_t s = std::max<int64_t>(1, std::min<int64_t>(MAX_SPLITS / std::max<int64_t>(blocks, 1), stream / 8));
    if (s > 8) s = s / 8 * 8;
    int64_t least = std::min<int64_t>({MAX_SPLITS, (stream + SPLIT_TILES - 1) / SPLIT_TILES, (1 << 22) / std::max<int64_t>(blocks, 1)});
    if (least > 8) least = (least + 7) / 8 * 8;
    s = std::max(s, least);
    while (s > 1) {
        const int64_t per = (stream + s - 1) / s;
        if ((s - 1) * per < stream) break;
        s = s > 8 ? s - 8 : s - 1;
    }
    return (int)s;
}

Plan make_plan(const int64_t n, const int64_t M, const int32_t f, const int32_t k) {
    Plan p;
    p.F = padded_factors(f);
    p.waves = waves_of(p.F);
    p.n_tiles = (n + TILE - 1) / TILE;
    p.m_tiles = (M + TILE - 1) / TILE;
    p.few = n <= few_users(p.F, M);
    p.splits1 = split_count((p.n_tiles + p.waves - 1) / p.waves, p.m_tiles);
    p.splits2 = split_count((p.m_tiles + p.waves - 1) / p.waves, p.n_tiles);
    p.item_blocks = (int)((M + p.waves * TILE - 1) / (p.waves * TILE));
    if (p.few) {                                         // eight items per row of lanes or more, none without items
        const int64_t s = std::min<int64_t>(MAX_SPLITS, (M + 255) / 256), per = (M + s - 1) / s;
        p.splits1 = (int)((M + per - 1) / per);
        p.splits2 = 1;
    }
    size_t at = 0;
    auto take = [&](const size_t bytes) { const size_t here = at; at += (bytes + 255) / 256 * 256; return here; };
    take((Y_MAX_BLOCKS + 2 * X_MAX_BLOCKS) * 4);
    p.off_scales = take(16);
    p.off_xt = take(p.few ? 0 : (size_t)p.n_tiles * p.F * 256);
    p.off_yt = take(p.few ? (size_t)n * M * 4 : (size_t)p.m_tiles * p.F * 256);       // few: the scores
    p.off_o = take((size_t)p.splits1 * n * p.F * 4);
    p.off_stat = take((size_t)p.splits1 * n * 8);
    p.off_bias = take((size_t)p.n_tiles * TILE * 4);
    p.off_item = take((size_t)n * k * 4);
    p.off_t = take((size_t)n * k * 4);
    p.off_offs = take((size_t)n * (p.item_blocks + 1) * 2);
    p.off_dy = take(p.splits2 > 1 ? (size_t)p.splits2 * M * p.F * 4 : 0);
    p.off_exp = take(p.few ? 0 : (size_t)n * 4);
    p.total = at;
    return p;
}

template <int F, int WAVES, int RING, bool BACK>
int32_t launch_pass(const FactorArgs &a, hipStream_t st) {
    const int64_t stat_tiles = BACK ? a.m_tiles : a.n_tiles;
    const int64_t grid = (stat_tiles + WAVES - 1) / WAVES * (BACK ? a.splits2 : a.splits1);      // below 2^23 (ROWS_MAX)
    hipLaunchKernelGGL((pass_kernel<F, WAVES, RING, BACK>), dim3((unsigned)grid), dim3(WAVES * 64), 0, st, a);
    ALS_HIP_CHECK6(hipGetLastError());
    return ALS_OK;
}

template <int F>
void launch_lists(const FactorArgs &a, const bool vec, hipStream_t st) {
    const int64_t n_users = a.n_tiles * TILE;
    const dim3 users((unsigned)std::min(n_users, GRID_X), (unsigned)((n_users + GRID_X - 1) / GRID_X));
    if (a.k <= 256) {
        if (vec) hipLaunchKernelGGL((lists_kernel<F, true, 256>), users, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((lists_kernel<F, false, 256>), users, dim3(256), 0, st, a);
    } else {
        if (vec) hipLaunchKernelGGL((lists_kernel<F, true, LIST_MAX>), users, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((lists_kernel<F, false, LIST_MAX>), users, dim3(256), 0, st, a);
    }
}
bool vector_rows(const FactorArgs &a) {
    return a.f % 4 == 0 && a.ldy % 4 == 0 && a.ldx % 4 == 0 && ((uintptr_t)a.Y | (uintptr_t)a.X) % 16 == 0;
}

template <int F, int NU, bool VEC>
int32_t run_few(const FactorArgs &a, hipStream_t st) {
    float *scores = (float *)a.yt;
    hipLaunchKernelGGL((few_scan_kernel<F, NU, VEC>), dim3((unsigned)a.splits1), dim3(512), 0, st, a, scores);
    launch_lists<F>(a, VEC, st);
    const int64_t blocks = std::min<int64_t>((a.M + 63) / 64, 2048);      // four items per row of lanes or more
    hipLaunchKernelGGL((few_back_kernel<F, NU, VEC>), dim3((unsigned)blocks), dim3(256), 0, st, a, scores);
    hipLaunchKernelGGL((few_listed_kernel<NU>), dim3((unsigned)(a.n * a.k)), dim3(64), 0, st, a, scores);
    ALS_HIP_CHECK6(hipGetLastError());
    return ALS_OK;
}
template <int F>
int32_t run_few(const FactorArgs &a, hipStream_t st) {
    const bool vec = vector_rows(a);
    if (a.n <= 2) return vec ? run_few<F, 2, true>(a, st) : run_few<F, 2, false>(a, st);
    if (F == 256 || a.n <= 4) return vec ? run_few<F, 4, true>(a, st) : run_few<F, 4, false>(a, st);
    if constexpr (F < 256) return vec ? run_few<F, 8, true>(a, st) : run_few<F, 8, false>(a, st);
    return ALS_OK;
}

template <int F, int WAVES, int RING1, int RING2>
int32_t run(const FactorArgs &a, const bool few, hipStream_t st) {
    if (few) return run_few<F>(a, st);
    const bool vec = vector_rows(a);
    const dim3 blocks(Y_MAX_BLOCKS + X_MAX_BLOCKS);
    if (vec) hipLaunchKernelGGL((maxima_kernel<true>), blocks, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((maxima_kernel<false>), blocks, dim3(256), 0, st, a);
    hipLaunchKernelGGL((prepare_kernel<F>), dim3((unsigned)(a.m_tiles + a.n_tiles)), dim3(256), 0, st, a);
    ALS_HIP_CHECK6(hipGetLastError());
    int32_t rc = launch_pass<F, WAVES, RING1, false>(a, st);
    if (rc) return rc;
    launch_lists<F>(a, vec, st);
    ALS_HIP_CHECK6(hipGetLastError());
    rc = launch_pass<F, WAVES, RING2, true>(a, st);
    if (rc) return rc;
    if (a.splits2 > 1) {
        const int64_t n_blocks = std::min<int64_t>((a.M * a.f + 255) / 256, 4096);
        hipLaunchKernelGGL(join_items_kernel, dim3((unsigned)n_blocks), dim3(256), 0, st, a, F);
        ALS_HIP_CHECK6(hipGetLastError());
    }
    return ALS_OK;
}

bool sizes_ok(const int64_t n, const int64_t M, const int32_t f, const int32_t k) {
    return n >= 1 && M >= 1 && M <= ROWS_MAX && n <= ROWS_MAX && f >= 1 && f <= ALS_MAX_FACTORS && k >= 1 && k <= LIST_MAX;
}

}  // namespace

extern "C" {

size_t als_distill_topk_workspace_bytes(int64_t n_users, int64_t M, int32_t f, int32_t k) {
    return sizes_ok(n_users, M, f, k) ? make_plan(n_users, M, f, k).total : 0;
}

int32_t als_distill_topk_f32(const float *X, int64_t x_rows, int64_t ldx, const int64_t *user_ids, int64_t n_users, const float *Y,
                             int64_t ldy, int64_t M, int32_t f, const int32_t *teacher_idx, const float *teacher_val, int64_t ld_teacher,
                             int32_t k, float temperature, const float *weight, float *loss_out, float *dX_out, float *dY_out,
                             void *workspace, size_t ws_bytes, void *stream) {
    if (!X || !Y || !teacher_idx || !teacher_val || !loss_out || !dX_out || !dY_out)
        return als_fail_(ALS_ERR_INVALID_ARG, "als_distill_topk_f32: null pointer");
    if (f > ALS_MAX_FACTORS || k > LIST_MAX)
        return als_fail_(ALS_ERR_UNSUPPORTED, "als_distill_topk_f32: f=%d (at most %d), k=%d (at most %d)", f, ALS_MAX_FACTORS, k, LIST_MAX);
    if (!sizes_ok(n_users, M, f, k) || x_rows < 1 || (!user_ids && n_users > x_rows) || ldx < f || ldy < f || ld_teacher < k)
        return als_fail_(ALS_ERR_INVALID_ARG, "als_distill_topk_f32: bad sizes (n_users=%lld M=%lld f=%d k=%d)", (long long)n_users,
                         (long long)M, f, k);
    if (!(temperature >= 1e-6f && temperature <= 1e6f))
        return als_fail_(ALS_ERR_INVALID_ARG, "als_distill_topk_f32: temperature %g outside [1e-6, 1e6]", (double)temperature);
    const Plan p = make_plan(n_users, M, f, k);
    if (!workspace || ws_bytes < p.total || (uintptr_t)workspace % 16)
        return als_fail_(ALS_ERR_WORKSPACE, "als_distill_topk_f32: workspace too small or not 16-byte aligned: %zu < %zu", ws_bytes, p.total);
    FactorArgs a;
    a.X = X; a.Y = Y; a.ldx = ldx; a.ldy = ldy; a.users = user_ids; a.n = n_users; a.M = M; a.f = f; a.x_rows = x_rows;
    a.t_idx = teacher_idx; a.t_val = teacher_val; a.ldt = ld_teacher; a.k = k; a.inv_t = 1.f / temperature; a.weight = weight;
    a.loss = loss_out; a.dX = dX_out; a.dY = dY_out;
    char *ws = (char *)workspace;
    a.maxima = (float *)ws;
    a.scales = (float *)(ws + p.off_scales);
    a.xt = ws + p.off_xt; a.yt = ws + p.off_yt;
    a.o_part = (float *)(ws + p.off_o); a.stat_part = (float *)(ws + p.off_stat); a.bias = (float *)(ws + p.off_bias);
    a.s_item = (int32_t *)(ws + p.off_item); a.s_t = (float *)(ws + p.off_t); a.offs = (uint16_t *)(ws + p.off_offs);
    a.dy_part = (float *)(ws + p.off_dy);
    a.user_exp = p.few ? nullptr : (int32_t *)(ws + p.off_exp);
    a.n_tiles = p.n_tiles; a.m_tiles = p.m_tiles; a.splits1 = p.splits1; a.splits2 = p.splits2; a.item_blocks = p.item_blocks;
    a.block_items = p.waves * TILE;
    hipStream_t st = (hipStream_t)stream;
    switch (p.F) {
        case 32: return run<32, 8, 4, 2>(a, p.few, st);
        case 64: return run<64, 8, 4, 2>(a, p.few, st);
        case 128: return run<128, 8, 3, 2>(a, p.few, st);
        default: return run<256, 4, 2, 2>(a, p.few, st);
    }
}

}  // extern "C"

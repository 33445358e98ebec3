// Random draws from rows of scores: temperature, min-p, top-k, top-p and the draw itself, from given random numbers.
//
// The operator.  For one row s of M scores, T its temperature, x_i = (s_i - max s) / T, w_i = exp(x_i):
//   1. items with w_i < min_p are dropped;
//   2. of the rest, in rank order (score descending, ties by ascending column), the first top_k stay;
//   3. of those the shortest prefix stays whose weight reaches top_p times theirs;
//   4. with W the weight of what is left and u in [0, 1): the draw is the first item in rank order at which the running
//      weight exceeds u W; its ln(w_i / W) is returned beside it.
// Every step asks the same question - at which item, in rank order, does a running sum (of ones, or of weights) pass a
// target - and the kernels have one answer to it (find): a histogram of the row over 512 or 2048 buckets of equal width in
// the score gives the bucket, the bucket's few items are collected in LDS and ranked against each other.  Rows are not sorted.
//
// Weights are held as integers, round(w 2^Q) with Q = min(51, 62 - ceil(log2 M)): their sums are exact whatever the order,
// so integer atomics do not make the result depend on timing, and a draw differs from the definition's only where u W lies
// within the summed roundings of a border.  With M = 59 047 (Q = 46) that is a part in 10^11 of W; float32 sums would
// decide one draw in a hundred wrongly on a catalogue of a million.  An item whose weight rounds to 0 (below 2^-47 of the
// largest) counts as dropped.  exp is computed in float64 (which this chip multiplies at the float32 rate): x 256 / ln 2 =
// k + r, 2^(k mod 256 / 256) from a table, a polynomial of degree 4 in r; error below 1e-15.
//
// Two forms.  sample_rows_kernel: one workgroup per row, one launch; the row is read from memory for its maximum and for the
// items that can matter, in one pass if they are few (filtered rows), and otherwise, mostly from the caches, twice more (and
// once or more per window of the rank order where those are too many for LDS).
// Few long rows are cut into parts, one workgroup each, in four launches: maximum; histogram; items of the buckets the
// answers can lie in, collected in a list; the answers from the list.
//
// What bounds it (whole calls on one MI355X).  Filtered rows: the read, 4096 x 59047 float32 in 181 us = 5.3 TB/s (a plain
// sum over them reads 4.0).  Rows of which much counts: vector instructions and LDS atomics; 1021 x 131071 bfloat16 with
// 8 draws each takes 190 us, 185 000 cycles a row with two rows on a compute unit: about 40 000 for the maximum, 55 000 for
// counting the values, 40 000 for collecting, 40 000 for the draws.  Single rows: a chain of memory round trips and some
// forty barriers, 19 us for 59 047 items; 10^6 items in four launches 37 us (under a profiler 5 + 9 + 11 + 13).  Rows of which
// thousands of items matter to many draws: windows, see there.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "als_hip.h"

int als_fail_(int code, const char *fmt, ...);  // defined in als_kernels.hip

#define ALS_HIP_CHECK4(expr)                                                                      \
    do {                                                                                          \
        hipError_t e_ = (expr);                                                                   \
        if (e_ != hipSuccess) return als_fail_(ALS_ERR_HIP, "%s: %s", #expr, hipGetErrorString(e_)); \
    } while (0)

namespace {

#include "als_rows.inc"

typedef unsigned long long u64;

// A workgroup's size.  The steps between the passes are short and alike for all waves, so a workgroup has few threads, and
// a compute unit several workgroups (launch says which group a row gets).
template <int T, int B>
struct Group {
    static constexpr int THREADS = T, WAVES = T / 64, BUCKETS = B;
    static constexpr int OWN = B / T;             // buckets per thread
    static constexpr int EDGE = B / 100 + 1;      // bucket_of takes scores 1 % beyond the last bucket's width into it
    static constexpr bool BY_VALUE = T > 256;     // 16-bit rows: see count_values
    static constexpr int RANKED = T / 4;          // items that are ranked against each other directly, four threads each
    static constexpr int WAVE_ITEMS = T > 256 ? 192 : 64;      // ... by one wave
};
typedef Group<256, 512> Small;
typedef Group<512, 2048> Large;
constexpr int CUT_BUCKETS = Large::BUCKETS;
constexpr int LISTED = 2048;          // items collected in LDS
constexpr int SR_LISTED = 16384;      // cut rows: items collected per row
// A row's draws: some microseconds each from a list in LDS, several of them side by side; where thousands of items matter, a share
// of the passes over the row that a window takes (draw_from_windows).  65 536 draws, ms: 13 of a row of 1 000 003 equal scores,
// 23 of five different ones, 210 of a normal distribution's, 1500 where all of it lies within one bucket of the histogram.
// A window takes a pass of one workgroup, 0.3 ns an item (1.2 at the worst), and there are no more windows than draws or some
// M / 1024: so that a launch ends within seconds, rows of more than 2^22 items are drawn from 2^34 / M times a call.
constexpr int32_t DRAWS_MAX = 1 << 16;
int32_t draws_max(const int64_t M) { return M <= (1 << 22) ? DRAWS_MAX : (int32_t)std::max<int64_t>(1, (1LL << 34) / M); }

struct Found {            // an item collected by a workgroup of a cut row
    float score;
    int32_t index;
};
struct PartStat {
    u64 best;             // rank key of the largest score << 32 | ~column: the best item of the part
    float low, pad;       // smallest score that is no mask value
};

struct SampleArgs {
    void *scores;
    int64_t lds, n, M;
    const int64_t *ex_rowptr;
    const int32_t *ex_col;
    const int64_t *ex_rows;
    als_sample_opts_t o;
    const void *u;
    int32_t u_f64, n_draws, q_bits;
    int32_t *idx;
    float *logp;
    // cut rows
    int32_t n_parts, per_part;        // chunks per part
    PartStat *stats;                  // [row, part]
    u64 *wsum;                        // [row, bucket]
    uint32_t *cnt;                    // [row, bucket]
    uint32_t *n_found;                // [row]
    Found *found;                     // [row, SR_LISTED]
};

// A value that is the same in all lanes of a wave, told to the compiler: it then lives in scalar registers.
__device__ __forceinline__ uint32_t uniform(const uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ int32_t uniform(const int32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float uniform(const float v) { return __uint_as_float(uniform(__float_as_uint(v))); }
__device__ __forceinline__ u64 uniform(const u64 v) { return (u64)uniform((uint32_t)(v >> 32)) << 32 | uniform((uint32_t)v); }

// floats as unsigned keys of the same order
__device__ __forceinline__ uint32_t rank_key(const float s) {
    const uint32_t b = __float_as_uint(s + 0.f);            // -0 and +0 are one score: -0 + 0 = +0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_score(const uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct Picked {
    u64 before, weight;       // running weight in front of the item, its own
    int32_t index;
    float score;
};

template <class G>
struct SampleShared {
    u64 wsum[G::BUCKETS];
    uint32_t cnt[G::BUCKETS];
    static constexpr int VALUES = G::BY_VALUE ? (G::BUCKETS * 12 + LISTED * 8) / 4 : 1;
    union {
        struct {
            union {
                struct { u64 wsub[G::BUCKETS]; uint32_t csub[G::BUCKETS]; };
                u64 ranked[G::RANKED][2];           // (key << 32 | ~column, weight)
                u64 wave_ranked[G::WAVES][G::WAVE_ITEMS][2];
            };
            union {
                Found found[LISTED];
                u64 sorted[LISTED];                 // rank key << 32 | ~column
            };
        };
        uint32_t values[VALUES];                    // how often a 16-bit value and its negative occur
    };
    double pow2[256];               // 2^(i / 256)
    u64 wave_w[G::WAVES];
    uint32_t wave_c[G::WAVES];
    float wave_f[G::WAVES], wave_g[G::WAVES];
    Picked picked;
    uint32_t bucket, n_list, k_lo, k_hi;
    u64 base_w, kept;
    uint32_t base_c, in_bucket;
};

// A row's parameters.
struct RowParams {
    float T, top_p, min_p;
    int32_t top_k;
};
__device__ __forceinline__ RowParams row_params(const SampleArgs &a, const int64_t r) {
    RowParams p;
    p.T = a.o.temperature_rows ? a.o.temperature_rows[r] : a.o.temperature;
    p.top_k = a.o.top_k_rows ? a.o.top_k_rows[r] : a.o.top_k;
    p.top_p = a.o.top_p_rows ? a.o.top_p_rows[r] : a.o.top_p;
    const float m = a.o.min_p_rows ? a.o.min_p_rows[r] : a.o.min_p;
    p.min_p = m > 0.f ? fminf(m, 1.f) : 0.f;                  // NaN: off
    return p;
}

// Whether top-k can take part, and the histogram needs counts.
__device__ __forceinline__ bool top_k_asked(const SampleArgs &a, const RowParams &p) { return p.top_k > 0 && p.top_k < a.M; }

// How scores become weights and buckets.  (The largest score is finite here: rows with +inf are answered apart.)
struct RowScale {
    double top;         // the largest score
    double steps;       // 256 / (T ln 2): a score's x in 256ths of a power of two
    double cut;         // ... and how many of those below the top an item has no weight, or is below min_p
    double min_w;       // min_p 2^Q
    float top_f, per_score;    // buckets per unit of score
    float reject;       // scores this many buckets or more below the top are beyond the cut
};
// How far below the largest x an item can be and count: beyond it a weight rounds to 0, or is below min_p.
__device__ __forceinline__ double item_cut(const RowParams &p, const int q_bits) {
    const double cut = 0.6931471805599453 * (q_bits + 1);
    return p.min_p > 0.f ? fmin(cut, -log((double)p.min_p) + 1e-6) : cut;
}
// The same in scores; +inf where that exceeds what scores can differ by.
__device__ __forceinline__ float score_reach(const double cut, const float T) {
    const double reach = cut * (double)T;
    return reach < 1e38 ? (float)reach : __builtin_inff();
}
// low: a low score of the row that is no mask value (+inf if there is none).  It only sets the buckets' width.
__device__ __forceinline__ RowScale row_scale(const float top, const float low, const double cut, const RowParams &p, const int q_bits,
                                              const int buckets) {
    RowScale c;
    c.top = (double)top;
    c.steps = 256.0 * 1.4426950408889634074 / (double)p.T;
    c.cut = cut * (256.0 * 1.4426950408889634074);
    c.min_w = ldexp((double)p.min_p, q_bits);
    const float reach = score_reach(cut, p.T);
    const float width = fminf(fmaxf(low <= top ? fminf(reach, top - low) : reach, 1e-30f), 3e38f);
    c.top_f = uniform(top);
    c.per_score = uniform((float)buckets / width);
    c.reject = uniform((float)buckets * fmaxf(1.f, reach / width) * 1.01f);
    return c;
}

// pow2: 2^(Q + i / 256), i < 256.  2^(y / 256 + Q) for y <= 0, y = k + f with k an integer: table and a polynomial of degree 4.
__device__ __forceinline__ double exp_table(const double y, const double *pow2) {
    constexpr double MAGIC = 6755399441055744.0;              // 1.5 2^52: adds, rounds to an integer
    const double kd = y + MAGIC;
    const int k = (int)(uint32_t)__double_as_longlong(kd);
    const double r = (y - (kd - MAGIC)) * (0.69314718055994530942 / 256.0);
    const double p = fma(r, fma(r, fma(r, 1.0 / 24, 1.0 / 6), 0.5), 1.0);
    const double t = pow2[k & 255];
    const double m = fma(t * r, p, t);
    return __hiloint2double(__double2hiint(m) + ((k >> 8) << 20), __double2loint(m));
}
// The integer weight of a score; false if it has none.  Without branches: four at a time keep the float64 units busy.
__device__ __forceinline__ bool weigh(const float s, const RowScale &c, const double *pow2, u64 &w) {
    const double y = ((double)s - c.top) * c.steps;
    const double m = exp_table(y, pow2);                      // w 2^Q
    // + 2^52: the mantissa's low bits are the integer, rounded to nearest even
    w = (u64)__double_as_longlong(m + 4503599627370496.0) & 0xfffffffffffffull;
    return y >= -c.cut && m >= c.min_w && w != 0;             // not so for NaN scores and NaN products (-inf x 0)
}
// ln of a weight's integer: float32's logarithm of the mantissa and one Newton step with the exponential at hand (the
// library's float64 logarithm would cost the kernels the registers of a second resident workgroup).
__device__ __forceinline__ double log_of(const u64 w, const double *pow2, const int q_bits) {
    const int e = 63 - __clzll((long long)w);
    const double m = ldexp((double)w, -e);
    const double y = (double)logf((float)m);
    const double t = ldexp(exp_table(y * (-256.0 * 1.4426950408889634074), pow2), -q_bits);       // e^-y
    return 0.69314718055994530942 * e + (y + fma(m, t, -1.0));
}
// Bucket of a score, B if it is certainly beyond the cut.  Falls with the score (every operation is monotone), so
// buckets are runs of the rank order.  NaN scores get some bucket or none: they have no weight.
template <int B>
__device__ __forceinline__ uint32_t bucket_of(const float s, const RowScale &c) {
    const float t = (c.top_f - s) * c.per_score;
    return t <= c.reject ? (uint32_t)(int)fminf(t, (float)(B - 1)) : B;
}

// Inclusive running sums over a wave's lanes by DPP moves (rows of 16 lanes, then across rows).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(const uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, true);      // lanes without a source get 0
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 moved(const u64 v) {
    return (u64)moved<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | moved<CTRL, ROWS>((uint32_t)v);
}
template <class V>
__device__ __forceinline__ V wave_scan(V v) {
    asm volatile("s_nop 1" : "+v"(v));      // a DPP move reads its register two states after the write, wherever that was
    v += moved<0x111, 0xf>(v);        // row_shr:1
    v += moved<0x112, 0xf>(v);        // row_shr:2
    v += moved<0x114, 0xf>(v);        // row_shr:4
    v += moved<0x118, 0xf>(v);        // row_shr:8
    v += moved<0x142, 0xa>(v);        // row_bcast:15 into rows 1 and 3
    v += moved<0x143, 0xc>(v);        // row_bcast:31 into rows 2 and 3
    return v;
}

// The wave's largest `hi` (returned) and smallest `low`, in lane 63.
template <int CTRL, int ROWS>
__device__ __forceinline__ float moved(const float v, const float none) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp((int)__float_as_uint(none), (int)__float_as_uint(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float wave_ends(float hi, float &low) {
    const float inf = __builtin_inff();
    asm volatile("s_nop 1" : "+v"(hi), "+v"(low));
    hi = fmaxf(hi, moved<0x111, 0xf>(hi, -inf)); low = fminf(low, moved<0x111, 0xf>(low, inf));
    hi = fmaxf(hi, moved<0x112, 0xf>(hi, -inf)); low = fminf(low, moved<0x112, 0xf>(low, inf));
    hi = fmaxf(hi, moved<0x114, 0xf>(hi, -inf)); low = fminf(low, moved<0x114, 0xf>(low, inf));
    hi = fmaxf(hi, moved<0x118, 0xf>(hi, -inf)); low = fminf(low, moved<0x118, 0xf>(low, inf));
    hi = fmaxf(hi, moved<0x142, 0xa>(hi, -inf)); low = fminf(low, moved<0x142, 0xa>(low, inf));
    hi = fmaxf(hi, moved<0x143, 0xc>(hi, -inf)); low = fminf(low, moved<0x143, 0xc>(low, inf));
    return hi;
}

// Sum of the first `n` of the per-wave values: a lane loads one each (a loop over them costs its unrolled registers).
template <class G, class V>
__device__ __forceinline__ V sum_of_first(const V *v, const int n) {
    const int l = threadIdx.x & (G::WAVES - 1);
    V s = l < n ? v[l] : 0;
#pragma unroll
    for (int o = G::WAVES / 2; o >= 1; o >>= 1) {
        if constexpr (sizeof(V) == 4) {
            s += (V)__shfl_xor((int)s, o);
        } else {
            const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)s, o), hi = (uint32_t)__shfl_xor((int)(uint32_t)(s >> 32), o);
            s += (u64)hi << 32 | lo;
        }
    }
    return s;
}

// Inclusive running sums over the buckets of (cnt, wsum), in place; every thread has OWN neighbours.
template <class G>
__device__ __forceinline__ void scan_buckets(uint32_t *cnt, u64 *wsum, SampleShared<G> &sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t c[G::OWN];
    u64 w[G::OWN];
#pragma unroll
    for (int q = 0; q < G::OWN; ++q) {
        c[q] = cnt[G::OWN * tid + q] + (q ? c[q - 1] : 0);
        w[q] = wsum[G::OWN * tid + q] + (q ? w[q - 1] : 0);
    }
    uint32_t bc = wave_scan(c[G::OWN - 1]);
    u64 bw = wave_scan(w[G::OWN - 1]);
    if (lane == 63) { sh.wave_c[wave] = bc; sh.wave_w[wave] = bw; }
    __syncthreads();
    bc += sum_of_first<G>(sh.wave_c, wave) - c[G::OWN - 1];          // in front of the thread's buckets
    bw += sum_of_first<G>(sh.wave_w, wave) - w[G::OWN - 1];
#pragma unroll
    for (int q = 0; q < G::OWN; ++q) { cnt[G::OWN * tid + q] = bc + c[q]; wsum[G::OWN * tid + q] = bw + w[q]; }
    __syncthreads();
}

// The bucket at which the running sum (of ones or of weights) passes `target`; base sums in front of it.
template <class G>
__device__ __forceinline__ void pick_bucket(const uint32_t *cnt, const u64 *wsum, const bool by_count, const u64 target, const uint32_t base_c,
                            const u64 base_w, SampleShared<G> &sh) {
#pragma unroll
    for (int q = 0; q < G::OWN; ++q) {
        const int b = G::OWN * threadIdx.x + q;
        const uint32_t pc = b ? cnt[b - 1] : 0, cc = cnt[b];
        const u64 pw = b ? wsum[b - 1] : 0, cw = wsum[b];
        const u64 lo = by_count ? base_c + pc : base_w + pw, hi = by_count ? base_c + cc : base_w + cw;
        if (lo <= target && target < hi) {
            sh.bucket = b; sh.in_bucket = cc - pc; sh.base_c = base_c + pc; sh.base_w = base_w + pw;
        }
    }
    __syncthreads();
}

// ----------------------------------------------------------------------------- where a row's items come from
// f(score, column) for the calling thread's share of the items; columns outside the row are never passed on, but scores
// of -inf may stand for nothing.

// Four items at a time, if any of them has a bucket: f(scores, column of the first, buckets), false to stop.
template <int B, class F>
__device__ __forceinline__ bool four_buckets(const float s0, const float s1, const float s2, const float s3, const int32_t i0,
                                             const RowScale &c, F f) {
    const float s[4] = {s0, s1, s2, s3};
    const uint32_t b[4] = {bucket_of<B>(s0, c), bucket_of<B>(s1, c), bucket_of<B>(s2, c), bucket_of<B>(s3, c)};
    return min(min(b[0], b[1]), min(b[2], b[3])) >= B || f(s, i0, b);
}
// Adds the four to the histogram.  Counts are only kept where they are asked for: by top-k, and in cut rows, where knowing how
// many items a bucket has saves its answer a look at all of them (47.7 -> 43.5 us for one row of a million).
template <int B>
__device__ __forceinline__ void count_four(const float (&s)[4], const uint32_t (&b)[4], const RowScale &c, const double *pow2,
                                           uint32_t *cnt, u64 *wsum, const bool counted) {
    u64 w[4];
    bool in[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) in[q] = weigh(s[q], c, pow2, w[q]) && b[q] < B;
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (in[q]) {
            atomicAdd(&wsum[b[q]], w[q]);
            if (counted) atomicAdd(&cnt[b[q]], 1u);
        }
}

// Read from memory, four chunks in flight per thread: f(chunk, column of its first element), false to stop the wave's walk.
// v: the thread's first four, which the caller has loaded (load_four).
template <class G, int TYPE>
__device__ __forceinline__ void load_four(const RowView<TYPE> &view, const int32_t q, const int32_t q1, row_u32x4 (&v)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        v[k] = RowView<TYPE>::nothing();
        if (q + k * G::THREADS < q1) v[k] = view.load(q + k * G::THREADS);
    }
}
template <class G, int TYPE, class F>
__device__ __forceinline__ void each_chunk(const RowView<TYPE> &view, const int32_t q0, const int32_t q1, row_u32x4 (&v)[4], F f) {
#pragma unroll 1
    for (int32_t q = q0 + threadIdx.x; q < q1;) {
        bool go = true;
#pragma unroll
        for (int k = 0; k < 4; ++k) go = f(v[k], view.index0(q + k * G::THREADS)) && go;
        if (!__all(go)) break;
        q += 4 * G::THREADS;
        load_four<G>(view, q, q1, v);
    }
}
// The same, the four chunks together: f(chunks, column of the first one's first element); the others follow 4 THREADS
// elements apart.
template <class G, int TYPE, class F>
__device__ __forceinline__ void each_quad(const RowView<TYPE> &view, const int32_t q0, const int32_t q1, F f) {
#pragma unroll 1
    for (int32_t q = q0 + threadIdx.x; q < q1; q += 4 * G::THREADS) {
        row_u32x4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[k] = RowView<TYPE>::nothing();
            if (q + k * G::THREADS < q1) v[k] = view.load(q + k * G::THREADS);
        }
        if (!f(v, view.index0(q))) break;
    }
}
// The items that have a bucket, four at a time (see four_buckets).
template <class G, int TYPE, class F>
__device__ __forceinline__ void each_bucket(const RowView<TYPE> &view, const int32_t q0, const int32_t q1, const bool extra,
                                            row_u32x4 (&first)[4], const RowScale &c, F f) {
    each_chunk<G>(view, q0, q1, first, [&](const row_u32x4 &v, const int32_t i0) {
        bool go = true;
#pragma unroll
        for (int e = 0; e < RowView<TYPE>::VEC; e += 4)
            go = four_buckets<G::BUCKETS>(RowView<TYPE>::value(v, e), RowView<TYPE>::value(v, e + 1), RowView<TYPE>::value(v, e + 2),
                                          RowView<TYPE>::value(v, e + 3), i0 + e, c, f) && go;
        return go;
    });
    const int32_t x = extra ? view.extra(threadIdx.x) : -1;
    if (x >= 0) four_buckets<G::BUCKETS>(view.at(x), -__builtin_inff(), -__builtin_inff(), -__builtin_inff(), x, c, f);
}

// The same for the rare passes over a whole row: not unrolled, it would take the registers of a resident workgroup.
template <class G, int TYPE, class F>
__device__ __forceinline__ void each_again(const RowView<TYPE> &view, F f) {
#pragma unroll 1
    for (int32_t i = threadIdx.x; i < view.M; i += G::THREADS) f(view.at(i), i);
}

// The items the answers can be, in LDS.
struct Listed {
    const Found *found;
    uint32_t n;
    template <class F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll 1
        for (uint32_t q = threadIdx.x; q < n; q += blockDim.x) f(found[q].score, found[q].index);
    }
};
// The same where LDS does not hold them: a list in memory or, if that does not either (whole), the row itself.
template <class G, int TYPE>
struct Unlisted {
    const RowView<TYPE> &view;
    const Found *found;
    uint32_t n;
    bool whole;
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        if (!whole) {
#pragma unroll 1
            for (uint32_t q = threadIdx.x; q < n; q += G::THREADS) f(found[q].score, found[q].index);
            return;
        }
        row_u32x4 v, next = RowView<TYPE>::nothing();
        if ((int32_t)threadIdx.x < view.n_chunks) next = view.load(threadIdx.x);
#pragma unroll 1
        for (int32_t q = threadIdx.x; q < view.n_chunks; q += G::THREADS) {
            v = next;
            if (q + G::THREADS < view.n_chunks) next = view.load(q + G::THREADS);
#pragma unroll
            for (int e = 0; e < RowView<TYPE>::VEC; ++e) f(RowView<TYPE>::value(v, e), view.index0(q) + e);
        }
        const int32_t x = view.extra(threadIdx.x);
        if (x >= 0) f(view.at(x), x);
    }
};

// Items of one score stand in column order.  Counted once per block of columns (running sums in sh.csub; returns their log2
// width, at least a wave's 64), any number of draws among them cost a look at one block each.
template <class G, int TYPE>
__device__ __forceinline__ int count_columns(const RowView<TYPE> &view, const uint32_t key, SampleShared<G> &sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int shift = 6;
    while ((view.M - 1) >> shift >= G::BUCKETS) ++shift;
#pragma unroll
    for (int q = 0; q < G::OWN; ++q) { sh.csub[G::OWN * tid + q] = 0; sh.wsub[G::OWN * tid + q] = 0; }
    __syncthreads();
#pragma unroll 1
    for (int32_t i0 = 64 * wave; i0 < view.M; i0 += 4 * G::THREADS) {       // a wave's 64 columns lie in one block
        u64 mask[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int32_t i = i0 + k * G::THREADS + lane;
            mask[k] = __ballot(i < view.M && rank_key(view.at(i)) == key);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (lane == 0 && mask[k]) atomicAdd(&sh.csub[(i0 + k * G::THREADS) >> shift], (uint32_t)__popcll(mask[k]));
    }
    __syncthreads();
    scan_buckets(sh.csub, sh.wsub, sh);
    return shift;
}
// Column of the m-th of them, from 0; by one wave, m below their number.
template <class G, int TYPE>
__device__ __forceinline__ int32_t nth_column(const RowView<TYPE> &view, const uint32_t key, const int shift, uint32_t m,
                                              const SampleShared<G> &sh) {
    constexpr int SEGMENT = G::BUCKETS / 64;
    const int lane = threadIdx.x & 63;
    const int seg = __ffsll(__ballot(sh.csub[SEGMENT * lane + SEGMENT - 1] > m)) - 1;
    if (seg < 0) return -1;                                  // not so: m is below the last sum
    const int b = SEGMENT * seg + __ffsll(__ballot(sh.csub[SEGMENT * seg + (lane & (SEGMENT - 1))] > m)) - 1;
    m -= b ? sh.csub[b - 1] : 0;
    const int64_t end = min((int64_t)view.M, (int64_t)(b + 1) << shift);
#pragma unroll 1
    for (int64_t i0 = (int64_t)b << shift; i0 < end; i0 += 256) {
        u64 mask[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t i = i0 + 64 * k + lane;
            mask[k] = __ballot(i < end && rank_key(view.at(i)) == key);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t here = (uint32_t)__popcll(mask[k]);
            if (m < here) {
                const uint32_t before = __builtin_amdgcn_mbcnt_hi((uint32_t)(mask[k] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask[k], 0u));
                return (int32_t)(i0 + 64 * k + __ffsll(__ballot((mask[k] >> lane & 1) != 0 && before == m)) - 1);
            }
            m -= here;
        }
    }
    return -1;
}

// ----------------------------------------------------------------------------- the question
// The item, in rank order, at which the running sum of ones (by_count) or of weights passes `target`; the caller has
// made sure that it does.  Every thread returns the same.
template <class G, int TYPE>
__device__ __forceinline__ Picked find(const Listed &row, const RowView<TYPE> &view, const RowScale &c, const bool by_count, const u64 target,
                       const bool counted, SampleShared<G> &sh) {
    const int tid = threadIdx.x;
    pick_bucket(sh.cnt, sh.wsum, by_count, target, 0, 0, sh);
    const uint32_t b = uniform(sh.bucket);
    uint32_t n = counted ? uniform(sh.in_bucket) : 0, base_c = uniform(sh.base_c);      // 0: not known, tried
    u64 base_w = uniform(sh.base_w);
    // the bucket's keys [k_lo, k_hi] that are still in question: to begin with its scores and a bucket's width more on either
    // side, for roundings (the last bucket is open downwards)
    const float width = 1.f / c.per_score;
    uint32_t k_hi = rank_key(fminf(c.top_f - (float)((int)b - 1) * width, c.top_f));
    uint32_t k_lo = b == G::BUCKETS - 1 ? 0 : rank_key(c.top_f - (float)(b + 2) * width);
    k_lo = uniform(k_lo); k_hi = uniform(k_hi);
    uint32_t i_lo = 0, i_hi = (uint32_t)view.M - 1;          // once they share one key: their columns
    auto mine = [&](const float s, const uint32_t i, u64 &w) {           // an item in question, and its weight
        if (bucket_of<G::BUCKETS>(s, c) != b) return false;
        const uint32_t key = rank_key(s);
        return key >= k_lo && key <= k_hi && i >= i_lo && i <= i_hi && weigh(s, c, sh.pow2, w);
    };
    // More items than are ranked directly: of BUCKETS parts of the range the part with the answer, and of one key's columns
    // likewise, until few are left (they are taken into LDS).
    int shift = 0;
    for (;;) {
        __syncthreads();
        const bool rank_them = n <= G::RANKED, by_column = k_lo == k_hi;
        if (!rank_them) {
            const int bits = 32 - __clz(by_column ? i_hi - i_lo : k_hi - k_lo), part_bits = 31 - __clz(G::BUCKETS);
            shift = bits > part_bits ? bits - part_bits : 0;
#pragma unroll
            for (int q = 0; q < G::OWN; ++q) { sh.csub[G::OWN * tid + q] = 0; sh.wsub[G::OWN * tid + q] = 0; }
        } else if (tid == 0) {
            sh.n_list = 0;
        }
        __syncthreads();
        row.each([&](const float s, const int32_t i) {
            u64 w;
            if (!mine(s, (uint32_t)i, w)) return;
            const uint32_t key = rank_key(s);
            if (!rank_them) {
                const uint32_t d = (by_column ? (uint32_t)i - i_lo : k_hi - key) >> shift;       // in rank order
                atomicAdd(&sh.csub[d], 1u);
                atomicAdd(&sh.wsub[d], w);
            } else {
                const uint32_t at = atomicAdd(&sh.n_list, 1u);
                if (at < (uint32_t)G::RANKED) {
                    sh.ranked[at][0] = (u64)key << 32 | (uint32_t)~(uint32_t)i;
                    sh.ranked[at][1] = w;
                }
            }
        });
        __syncthreads();
        if (rank_them) {
            n = uniform(sh.n_list);
            if (n <= G::RANKED) break;
            continue;
        }
        scan_buckets(sh.csub, sh.wsub, sh);
        pick_bucket(sh.csub, sh.wsub, by_count, target, base_c, base_w, sh);
        const uint32_t d = uniform(sh.bucket);
        const uint64_t behind = (uint64_t)(d + 1) << shift;                // keys down to the part's end
        if (by_column) {
            i_hi = behind > i_hi - i_lo ? i_hi : i_lo + (uint32_t)behind - 1;
            i_lo += d << shift;
        } else {
            k_lo = behind > k_hi - k_lo ? k_lo : k_hi - (uint32_t)behind + 1;
            k_hi = k_hi - (d << shift);
        }
        n = uniform(sh.in_bucket); base_c = uniform(sh.base_c); base_w = uniform(sh.base_w);
    }
    // The few that are left are ranked against each other, four threads to an item.
    const int e = tid >> 2;
    const u64 own = e < (int)n ? sh.ranked[e][0] : 0, w = e < (int)n ? sh.ranked[e][1] : 0;
    u64 before = 0;
    uint32_t rank = 0;
#pragma unroll 2
    for (uint32_t q = tid & 3; q < n; q += 4)
        if (sh.ranked[q][0] > own) { before += sh.ranked[q][1]; ++rank; }
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
        const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)before, o), hi = (uint32_t)__shfl_xor((int)(uint32_t)(before >> 32), o);
        before += (u64)hi << 32 | lo;
        rank += (uint32_t)__shfl_xor((int)rank, o);
    }
    before += base_w;
    rank += base_c;
    if (e < (int)n && (by_count ? rank == target : (before <= target && target < before + w))) {
        sh.picked.before = before; sh.picked.weight = w; sh.picked.index = (int32_t)~(uint32_t)own;
        sh.picked.score = key_score((uint32_t)(own >> 32));
    }
    __syncthreads();
    const Picked out{uniform(sh.picked.before), uniform(sh.picked.weight), uniform(sh.picked.index), uniform(sh.picked.score)};
    __syncthreads();
    return out;
}

// The same by one wave, from a list in LDS: without barriers, so that draws are made side by side.  False if the bucket has
// more items than a wave ranks.
template <class G>
__device__ __forceinline__ bool wave_find(const Found *list, const uint32_t n, const RowScale &c, const bool by_count, const u64 target,
                                          SampleShared<G> &sh, Picked &out) {
    constexpr int SEGMENT = G::BUCKETS / 64;
    const int lane = threadIdx.x & 63;
    u64(*items)[2] = sh.wave_ranked[threadIdx.x >> 6];
    auto sum_at = [&](const int b) { return by_count ? (u64)sh.cnt[b] : sh.wsum[b]; };
    const int seg = __ffsll(__ballot(sum_at(SEGMENT * lane + SEGMENT - 1) > target)) - 1;
    const int b = SEGMENT * seg + __ffsll(__ballot(sum_at(SEGMENT * seg + (lane & (SEGMENT - 1))) > target)) - 1;
    const u64 base_w = b ? sh.wsum[b - 1] : 0;
    const uint32_t base_c = b ? sh.cnt[b - 1] : 0;
    uint32_t m = 0;
    for (uint32_t q0 = 0; q0 < n; q0 += 64) {
        const uint32_t q = q0 + lane;
        const Found f = list[q < n ? q : n - 1];
        bool hit = q < n && bucket_of<G::BUCKETS>(f.score, c) == (uint32_t)b;
        if (__ballot(hit) == 0) continue;
        u64 w;
        hit = weigh(f.score, c, sh.pow2, w) && hit;
        const u64 mask = __ballot(hit);
        const uint32_t at = m + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
        if (hit && at < (uint32_t)G::WAVE_ITEMS) {
            items[at][0] = (u64)rank_key(f.score) << 32 | (uint32_t)~(uint32_t)f.index;
            items[at][1] = w;
        }
        m += (uint32_t)__popcll(mask);
    }
    if (m > (uint32_t)G::WAVE_ITEMS) return false;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    auto of_lane = [&](const u64 v, const int from) {
        return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), from) << 32 |
               (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, from);
    };
    auto picked = [&](const u64 before, const u64 w, const u64 key) {
        return Picked{before, w, (int32_t)~(uint32_t)key, key_score((uint32_t)(key >> 32))};
    };
    if (m <= 64) {                                           // each against all
        const uint32_t e = (uint32_t)lane < m ? (uint32_t)lane : m - 1;
        const u64 own = items[e][0], w = items[e][1];
        u64 before = base_w;
        uint32_t rank = base_c;
#pragma unroll 4
        for (uint32_t q = 0; q < m; ++q)
            if (items[q][0] > own) { before += items[q][1]; ++rank; }
        const u64 found = __ballot(by_count ? rank == target : before <= target && target < before + w);
        if (found == 0) return false;
        const int from = __ffsll(found) - 1;
        out = picked(of_lane(before, from), of_lane(w, from), of_lane(own, from));
        return true;
    }
    if constexpr (G::WAVE_ITEMS > 64) {                      // halving what is in question by one of its items, about ten times
        constexpr int SLOTS = G::WAVE_ITEMS / 64;
        u64 key[SLOTS], w[SLOTS];
        bool in[SLOTS];
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) {
            const uint32_t e = lane + 64 * k;
            in[k] = e < m;
            key[k] = items[in[k] ? e : 0][0]; w[k] = items[in[k] ? e : 0][1];
        }
        u64 before = base_w;
        uint32_t rank = base_c;
        for (uint32_t round = 1; round <= m; ++round) {      // a round takes one item out at least
            u64 pivot = 0, pivot_w = 0;
            bool have = false;
#pragma unroll
            for (int k = 0; k < SLOTS; ++k) {                // any item: the list is in no order that matters, but not shuffled
                const u64 mask = __ballot(in[k]);
                if (mask == 0 || (have && (round + k) % 2)) continue;
                const uint32_t turn = 37 * round & 63;
                const u64 turned = mask >> turn | mask << (64 - turn & 63);
                const int from = (int)((__ffsll(turned) - 1 + turn) & 63);
                pivot = of_lane(key[k], from); pivot_w = of_lane(w[k], from);
                have = true;
            }
            if (!have) return false;
            u64 front_w = 0;
            uint32_t front_c = 0;
#pragma unroll
            for (int k = 0; k < SLOTS; ++k) {
                const bool front = in[k] && key[k] > pivot;
                front_w += front ? w[k] : 0;
                front_c += (uint32_t)__popcll(__ballot(front));
            }
            front_w = of_lane(wave_scan(front_w), 63);
            if (by_count ? target < rank + front_c : target < before + front_w) {
#pragma unroll
                for (int k = 0; k < SLOTS; ++k) in[k] = in[k] && key[k] > pivot;
                continue;
            }
            before += front_w;
            rank += front_c;
            if (by_count ? target == rank : target < before + pivot_w) {
                out = picked(before, pivot_w, pivot);
                return true;
            }
            before += pivot_w;
            rank += 1;
#pragma unroll
            for (int k = 0; k < SLOTS; ++k) in[k] = in[k] && key[k] < pivot;
        }
    }
    return false;
}

// Targets of the three steps (find passes a target: the first item whose running sum exceeds it).
__device__ __forceinline__ u64 top_p_target(const float top_p, const u64 W) {
    const double want = ceil((double)fmaxf(top_p, 0.f) * (double)W);
    const u64 need = want < 1.0 ? 1 : want >= (double)W ? W : (u64)want;
    return need - 1;
}
__device__ __forceinline__ double drawn_number(const SampleArgs &a, const int64_t at) {
    const double u = a.u_f64 ? ((const double *)a.u)[at] : (double)((const float *)a.u)[at];
    return u > 0.0 ? fmin(u, 1.0) : 0.0;                      // NaN: 0
}
__device__ __forceinline__ u64 draw_target(const double u, const u64 W) {
    const double t = u * (double)W;
    const u64 target = t >= (double)W ? W - 1 : (u64)t;
    return target < W ? target : W - 1;
}

// First bucket whose running sum exceeds the target (the last one if none does).
template <class G, class V>
__device__ __forceinline__ int bucket_passing(const V *sums, const u64 target) {
    int lo = 0, hi = G::BUCKETS - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] > target) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}
// The same for two targets, all threads together (every thread looks at its own buckets): a fifth of the search's time.
template <class G, class V>
__device__ __forceinline__ void buckets_passing(const V *sums, const u64 t0, const u64 t1, SampleShared<G> &sh, int &b0, int &b1) {
    if (threadIdx.x == 0) { sh.k_lo = G::BUCKETS - 1; sh.k_hi = G::BUCKETS - 1; }
    __syncthreads();
    u64 before = threadIdx.x ? (u64)sums[G::OWN * threadIdx.x - 1] : 0;
#pragma unroll
    for (int q = 0; q < G::OWN; ++q) {
        const int b = G::OWN * threadIdx.x + q;
        const u64 last = (u64)sums[b];
        if (before <= t0 && t0 < last) sh.k_lo = b;
        if (before <= t1 && t1 < last) sh.k_hi = b;
        before = last;
    }
    __syncthreads();
    b0 = uniform((int32_t)sh.k_lo); b1 = uniform((int32_t)sh.k_hi);
    __syncthreads();
}
// The buckets the answers can lie in, a byte each: top-k's is known; what it leaves of the weight, and so top-p's target, is
// known to within that bucket, and so on.
template <class G>
__device__ __forceinline__ void wanted_buckets(const SampleArgs &a, const int64_t r, const RowParams &p, const bool open_end, SampleShared<G> &sh,
                                               unsigned char (&want)[G::BUCKETS + G::EDGE + 1]) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // ranges of buckets, +1 where one begins and -1 behind its end: the running sum is the number of ranges over a bucket
    uint32_t *edge = sh.csub;
#pragma unroll
    for (int q = 0; q < G::OWN; ++q) edge[G::OWN * tid + q] = 0;
    __syncthreads();
    auto mark = [&](const int b0, const int b1) {
        atomicAdd(&edge[b0], 1u);
        if (b1 + 1 < G::BUCKETS) atomicAdd(&edge[b1 + 1], ~0u);
    };
    u64 w_lo = sh.wsum[G::BUCKETS - 1], w_hi = w_lo;
    if (top_k_asked(a, p) && (uint32_t)p.top_k < sh.cnt[G::BUCKETS - 1]) {
        int b, same;
        buckets_passing(sh.cnt, (u64)p.top_k - 1, (u64)p.top_k - 1, sh, b, same);
        if (tid == 0) mark(b, b);
        w_lo = (b ? sh.wsum[b - 1] : 0) + 1; w_hi = sh.wsum[b];
    }
    if (p.top_p < 1.f) {
        int b0, b1;
        buckets_passing(sh.wsum, top_p_target(p.top_p, w_lo), top_p_target(p.top_p, w_hi), sh, b0, b1);
        if (tid == 0) mark(b0, b1);
        w_lo = (b0 ? sh.wsum[b0 - 1] : 0) + 1; w_hi = sh.wsum[b1];
    }
    if (a.n_draws <= 2) {
        for (int d = 0; d < a.n_draws; ++d) {
            const double u = drawn_number(a, r * a.n_draws + d);
            int b0, b1;
            buckets_passing(sh.wsum, draw_target(u, w_lo), draw_target(u, w_hi), sh, b0, b1);
            if (tid == 0) mark(b0, b1);
        }
    } else for (int d = tid; d < a.n_draws; d += G::THREADS) {
        const double u = drawn_number(a, r * a.n_draws + d);
        mark(bucket_passing<G>(sh.wsum, draw_target(u, w_lo)), bucket_passing<G>(sh.wsum, draw_target(u, w_hi)));
    }
    __syncthreads();
    uint32_t own[G::OWN], sum = 0;
#pragma unroll
    for (int q = 0; q < G::OWN; ++q) own[q] = sum += edge[G::OWN * tid + q];
    uint32_t front = wave_scan(sum);
    if (lane == 63) sh.wave_c[wave] = front;
    __syncthreads();
    front += sum_of_first<G>(sh.wave_c, wave) - sum;
#pragma unroll
    for (int q = 0; q < G::OWN; ++q) want[G::OWN * tid + q] = front + own[q] != 0;
    // behind them scores beyond the last bucket's width, which bucket_of may take into it: EDGE widths, and all the rest
    if (tid == G::THREADS - 1)
        for (int q = 0; q <= G::EDGE; ++q) want[G::BUCKETS + q] = front + own[G::OWN - 1] != 0 && (q < G::EDGE || open_end);
    __syncthreads();
}

// ----------------------------------------------------------------------------- rows that LDS has no list of
// Thousands of items can matter: many draws of a flat row, equal scores, a temperature far above the scores' spread.  An answer
// then takes passes over the list in memory or the row; but what they find is a whole window of the rank order around it - as
// many items as are sorted in LDS, or all items of one score -, and every other draw that falls into it is answered with it.
// A row of M items has some M / BUCKETS such windows, however many draws.
struct Window {
    u64 base_w, end_w;        // running weight in front of it and behind it
    u64 each;                 // 0: items sorted in sh.sorted, their running weights in sh.wsub; else the weight of every item of score `key`
    uint32_t base_c, n, key;
    int shift;                // of count_columns
};
// sh.sorted[0, n) in descending order, and their running weights.
template <class G>
__device__ __forceinline__ void sort_window(const uint32_t n, const RowScale &c, SampleShared<G> &sh) {
    const int tid = threadIdx.x;
    uint32_t size = 2;
    while (size < n) size *= 2;                              // at most BUCKETS
    for (uint32_t q = n + tid; q < size; q += G::THREADS) sh.sorted[q] = 0;
    __syncthreads();
#pragma unroll 1
    for (uint32_t run = 2; run <= size; run *= 2)
#pragma unroll 1
        for (uint32_t step = run / 2; step > 0; step /= 2) {
            for (uint32_t q = tid; q < size / 2; q += G::THREADS) {
                const uint32_t lo = 2 * q - (q & (step - 1)), hi = lo + step;
                const u64 x = sh.sorted[lo], y = sh.sorted[hi];
                if ((lo & run) == 0 ? x < y : x > y) { sh.sorted[lo] = y; sh.sorted[hi] = x; }
            }
            // a wave's 64 pairs of up to 64 apart are 128 neighbours: until pairs are further apart no other wave touches them
            if (step > 64 || (step == 1 && run > 64)) __syncthreads();
            else {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
        }
    __syncthreads();
#pragma unroll 1
    for (int q = tid; q < G::BUCKETS; q += G::THREADS) {
        u64 w = 0;
        if ((uint32_t)q < n) weigh(key_score((uint32_t)(sh.sorted[q] >> 32)), c, sh.pow2, w);
        sh.wsub[q] = w; sh.csub[q] = 0;
    }
    __syncthreads();
    scan_buckets(sh.csub, sh.wsub, sh);
}
// From bucket (or part) b on, the last one up to which all items are sorted together; b itself if not even its own are.
template <class G>
__device__ __forceinline__ uint32_t sorted_with(const uint32_t *cnt, const uint32_t b) {
    const uint32_t before = b ? cnt[b - 1] : 0;
    const uint32_t e = (uint32_t)bucket_passing<G>(cnt, (u64)before + G::BUCKETS);
    return cnt[e] - before <= (uint32_t)G::BUCKETS ? e : max(b, e ? e - 1 : 0);
}
// The items of the bucket that `target` lies in, into sh.found; more than LISTED: too many.
template <class G, int TYPE>
__device__ __forceinline__ uint32_t bucket_into_lds(const Unlisted<G, TYPE> &row, const RowScale &c, const bool by_count, const u64 target,
                                                    SampleShared<G> &sh) {
    if (threadIdx.x == 0) sh.n_list = 0;
    pick_bucket(sh.cnt, sh.wsum, by_count, target, 0, 0, sh);
    const uint32_t b = uniform(sh.bucket);
    row.each([&](const float s, const int32_t i) {
        if (bucket_of<G::BUCKETS>(s, c) != b) return;
        const uint32_t at = atomicAdd(&sh.n_list, 1u);
        if (at < (uint32_t)LISTED) sh.found[at] = Found{s, i};
    });
    __syncthreads();
    return uniform(sh.n_list);
}
// The window that holds the item at which the running sum passes `target` (see find).
template <class G, int TYPE>
__device__ __forceinline__ Window window_of(const Unlisted<G, TYPE> &row, const RowView<TYPE> &view, const RowScale &c, const bool by_count,
                                            const u64 target, const bool counted, const bool wide, SampleShared<G> &sh) {
    const int tid = threadIdx.x;
    pick_bucket(sh.cnt, sh.wsum, by_count, target, 0, 0, sh);
    const uint32_t b = uniform(sh.bucket);
    uint32_t n = 0, base_c = uniform(sh.base_c);             // 0: not known, tried
    u64 base_w = uniform(sh.base_w);
    uint32_t last = b;                                       // buckets b to last
    if (counted) {
        // as many buckets as are sorted, where a look at the items costs more than that: of the row, a list need not have them all
        if (wide) last = uniform(sorted_with<G>(sh.cnt, b));
        n = uniform(sh.cnt[last] - (b ? sh.cnt[b - 1] : 0));
    }
    const float width = 1.f / c.per_score;                   // keys in question as in find
    uint32_t k_hi = uniform(rank_key(fminf(c.top_f - (float)((int)b - 1) * width, c.top_f)));
    uint32_t k_lo = uniform(last == G::BUCKETS - 1 ? 0 : rank_key(c.top_f - (float)(last + 2) * width));
    // Scores well above the cut have a weight.  (2 % above it, and a min_p that is not within 10^-4 of 1: then 0.98 of the way to
    // it leaves more than min_p.)
    const bool all_weigh = last < (uint32_t)(G::BUCKETS * 49 / 50) && c.cut > 0.1;
#pragma unroll 1
    for (;;) {
        __syncthreads();
        const bool take = n <= (uint32_t)G::BUCKETS;
        if (!take && k_lo == k_hi) break;
        const int bits = 32 - __clz(k_hi - k_lo), part_bits = 31 - __clz(G::BUCKETS), shift = bits > part_bits ? bits - part_bits : 0;
#pragma unroll
        for (int q = 0; q < G::OWN; ++q) { sh.csub[G::OWN * tid + q] = 0; sh.wsub[G::OWN * tid + q] = 0; }
        if (tid == 0) sh.n_list = 0;
        __syncthreads();
        // by the scores first, which is the same as by their keys: two comparisons are all that most items of a pass cost
        float lo = k_lo > rank_key(-__builtin_inff()) ? key_score(k_lo) : -__builtin_inff();
        const float hi = key_score(k_hi);
        row.each([&](const float s, const int32_t i) {
            if (!(s >= lo && s <= hi)) return;
            u64 w;
            if (bucket_of<G::BUCKETS>(s, c) - b > last - b || (!(take && all_weigh) && !weigh(s, c, sh.pow2, w))) return;
            const uint32_t key = rank_key(s);
            if (take) {
                const uint32_t at = atomicAdd(&sh.n_list, 1u);
                if (at >= (uint32_t)G::BUCKETS) lo = __builtin_inff();      // one item too many says enough
                else sh.sorted[at] = (u64)key << 32 | (uint32_t)~(uint32_t)i;
            } else {
                const uint32_t d = (k_hi - key) >> shift;    // in rank order
                atomicAdd(&sh.csub[d], 1u);
                atomicAdd(&sh.wsub[d], w);
            }
        });
        __syncthreads();
        if (take) {
            n = uniform(sh.n_list);
            if (n > (uint32_t)G::BUCKETS) continue;
            sort_window(n, c, sh);
            return Window{base_w, base_w + sh.wsub[G::BUCKETS - 1], 0, base_c, n, 0, 0};
        }
        scan_buckets(sh.csub, sh.wsub, sh);
        pick_bucket(sh.csub, sh.wsub, by_count, target, base_c, base_w, sh);
        const uint32_t d = uniform(sh.bucket), d_last = uniform(sorted_with<G>(sh.csub, d));
        const uint64_t behind = (uint64_t)(d_last + 1) << shift;           // keys down to the last part's end
        k_lo = behind > k_hi - k_lo ? k_lo : k_hi - (uint32_t)behind + 1;
        k_hi = k_hi - (d << shift);
        n = uniform(sh.csub[d_last] - (d ? sh.csub[d - 1] : 0)); base_c = uniform(sh.base_c); base_w = uniform(sh.base_w);
    }
    u64 each;
    weigh(key_score(k_lo), c, sh.pow2, each);
    const int shift = count_columns<G>(view, k_lo, sh);
    n = sh.csub[G::BUCKETS - 1];
    return Window{base_w, base_w + n * each, each, base_c, n, k_lo, shift};
}
// The item of a sorted window at place e.
template <class G>
__device__ __forceinline__ Picked item_at(const Window &x, const uint32_t e, const SampleShared<G> &sh) {
    const u64 before = e ? sh.wsub[e - 1] : 0, key = sh.sorted[e];
    return Picked{x.base_w + before, sh.wsub[e] - before, (int32_t)~(uint32_t)key, key_score((uint32_t)(key >> 32))};
}
// A threshold's item (its column only if the window is a sorted one).
template <class G>
__device__ __forceinline__ Picked threshold_in(const Window &x, const bool by_count, const u64 target, const SampleShared<G> &sh) {
    const u64 over = target - (by_count ? x.base_c : x.base_w);
    if (x.each) return Picked{x.base_w + (by_count ? over : over / x.each) * x.each, x.each, -1, key_score(x.key)};
    return item_at(x, min(by_count ? (uint32_t)over : (uint32_t)bucket_passing<G>(sh.wsub, over), x.n - 1), sh);
}
// The draws from `from` on.  target_of(draw), finish(draw, item); a draw that is still open has column OPEN.
constexpr int32_t OPEN = -2;
template <class G, int TYPE, class T, class F>
__device__ __forceinline__ void draw_from_windows(const SampleArgs &a, const int64_t r, const int from, const Unlisted<G, TYPE> &row, const RowView<TYPE> &view,
                                                  const RowScale &c, const bool counted, T target_of, F finish, SampleShared<G> &sh) {
    const int tid = threadIdx.x;
    int32_t *idx = a.idx + r * a.n_draws;                    // thread t writes and reads the draws from + t, from + t + THREADS, ...
    for (int d = from + tid; d < a.n_draws; d += G::THREADS) idx[d] = OPEN;
#pragma unroll 1
    for (int d0 = from; d0 < a.n_draws;) {
        __syncthreads();
        if (tid == 0) sh.k_lo = ~0u;
        __syncthreads();
        if (d0 + tid < a.n_draws && idx[d0 + tid] == OPEN) atomicMin(&sh.k_lo, (uint32_t)(d0 + tid));
        __syncthreads();
        const uint32_t first = uniform(sh.k_lo);
        if (first == ~0u) {
            d0 += G::THREADS;
            continue;
        }
        const Window x = window_of(row, view, c, false, target_of((int)first), counted, row.whole, sh);
#pragma unroll 1
        for (int d = d0 + tid; d - tid < a.n_draws; d += G::THREADS) {
            u64 over = 0;
            bool in = d < a.n_draws && idx[d] == OPEN;
            if (in) {
                const u64 target = target_of(d);
                in = (target >= x.base_w && target < x.end_w) || d == (int)first;        // the first is: it ends the loop
                over = target - x.base_w;
            }
            if (x.each == 0) {
                if (in) finish(d, item_at(x, min((uint32_t)bucket_passing<G>(sh.wsub, over), x.n - 1), sh));
                continue;
            }
            const uint32_t m = in ? (uint32_t)min(over / x.each, (u64)x.n - 1) : 0;
            int32_t column = -1;
            for (u64 mask = __ballot(in); mask; mask &= mask - 1) {      // a wave for one of its draws at a time
                const int lane = __ffsll(mask) - 1;
                const int32_t i = nth_column<G>(view, x.key, x.shift, (uint32_t)__builtin_amdgcn_readlane((int)m, lane), sh);
                if ((tid & 63) == lane) column = i;
            }
            if (in) finish(d, Picked{x.base_w + (u64)m * x.each, x.each, column, key_score(x.key)});
        }
    }
}

// Steps 2 to 4 from the running sums in sh.cnt / sh.wsum.  in_lds: the row's items are a list in LDS; then of several draws a
// wave makes one each, and the workgroup together those that a wave does not (one alone takes a wave as long: 19.7 and 20.2 us
// for a row of 59 047 at n = 1, but 36 against 31 for 300 rows of 9 724).
template <class G, int TYPE, bool CUT>
__device__ __forceinline__ void answer(const SampleArgs &a, const int64_t r, const Unlisted<G, TYPE> &row, const bool in_lds, const bool counted,
                                       const RowView<TYPE> &view, const RowScale &c, const RowParams &p, SampleShared<G> &sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    u64 W = uniform(sh.wsum[G::BUCKETS - 1]);
    const bool by_k = top_k_asked(a, p) && (uint32_t)p.top_k < sh.cnt[G::BUCKETS - 1], by_p = p.top_p < 1.f;
    auto target_of = [&](const int step) {
        return step == -2 ? (u64)p.top_k - 1 : step == -1 ? top_p_target(p.top_p, W) : draw_target(drawn_number(a, r * a.n_draws + step), W);
    };
    auto finish = [&](const int step, const Picked &f) {     // one thread
        if (step < 0) {
            sh.kept = f.before + f.weight;
            return;
        }
        const int64_t at = r * a.n_draws + step;             // ln (w / W) = x - ln W
        const double x = ((double)f.score - c.top) * c.steps * (0.69314718055994530942 / 256.0);
        a.idx[at] = f.index;
        a.logp[at] = (float)(x - (log_of(W, sh.pow2, a.q_bits) - 0.69314718055994530942 * a.q_bits));
    };
    // Few answers from a list in memory: of each one's bucket alone, as from a list in LDS, if that holds it (64 draws of
    // a row of a million: 438 us, 780 from windows; 1000, whose list does not fit: 116 ms so, 15 from windows).
    auto from_windows = [&](int step) {                      // this and all later steps
        for (; step < 0; ++step) {
            if (step == -1 && !by_p) continue;
            const u64 target = target_of(step);
            const Window x = window_of(row, view, c, step == -2, target, counted, false, sh);
            const Picked f = threshold_in(x, step == -2, target, sh);
            W = uniform(f.before + f.weight);
        }
        draw_from_windows(a, r, step, row, view, c, counted, target_of, finish, sh);
    };
    int step = by_k ? -2 : by_p ? -1 : 0;
    if (!in_lds && (!CUT || row.whole || a.n_draws > 256)) {
        from_windows(step);
        return;
    }
    Listed list{sh.found, row.n};
    while (step < a.n_draws) {                               // uniform
        if (step == -1 && !by_p) {
            step = 0;
            continue;
        }
        if (CUT && !in_lds) {
            list.n = bucket_into_lds(row, c, step == -2, target_of(step), sh);
            if (list.n > (uint32_t)LISTED) {
                from_windows(step);
                return;
            }
        }
        const int many = step < 0 || (CUT && !in_lds) ? 1 : min(G::WAVES, a.n_draws - step);
        uint32_t open = (1u << many) - 1;
        if (many > 1) {
            bool done = true;
            if (wave < many) {
                Picked f;
                done = wave_find<G>(list.found, list.n, c, step == -2, target_of(step + wave), sh, f);
                if (done && lane == 0) finish(step + wave, f);
            }
            if (lane == 0) sh.wave_c[wave] = !done;
            __syncthreads();
            open = (uint32_t)__ballot(lane < G::WAVES && sh.wave_c[lane & (G::WAVES - 1)]);
        }
        while (open) {
            const int mine = step + __ffs(open) - 1;
            open &= open - 1;
            const Picked f = find<G>(list, view, c, step == -2, target_of(mine), counted, sh);
            if (threadIdx.x == 0) finish(mine, f);
        }
        __syncthreads();
        if (step < 0) W = uniform(sh.kept);
        step += many;
    }
}
__device__ __forceinline__ void answer_all(const SampleArgs &a, const int64_t r, const int32_t index, const float logp) {
    for (int d = threadIdx.x; d < a.n_draws; d += blockDim.x) { a.idx[r * a.n_draws + d] = index; a.logp[r * a.n_draws + d] = logp; }
}

// A row whose largest score is +inf: n items share everything, in column order.
template <class G, int TYPE>
__device__ __forceinline__ void answer_infinite(const SampleArgs &a, const int64_t r, const RowView<TYPE> &view, const RowParams &p,
                                SampleShared<G> &sh) {
    const uint32_t key = rank_key(__builtin_inff());
    const int shift = count_columns<G>(view, key, sh);
    u64 n = sh.csub[G::BUCKETS - 1];
    if (p.top_k > 0 && (u64)p.top_k < n) n = (u64)p.top_k;
    if (p.top_p < 1.f) n = top_p_target(p.top_p, n) + 1;
    for (int d = threadIdx.x >> 6; d < a.n_draws; d += G::WAVES) {
        const int64_t at = r * a.n_draws + d;
        const int32_t i = nth_column<G>(view, key, shift, (uint32_t)draw_target(drawn_number(a, at), n), sh);
        if ((threadIdx.x & 63) == 0) { a.idx[at] = i; a.logp[at] = -logf((float)n); }
    }
}

__device__ __forceinline__ u64 wave_max64(u64 v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)v, o), hi = (uint32_t)__shfl_xor((int)(uint32_t)(v >> 32), o);
        const u64 x = (u64)hi << 32 | lo;
        v = x > v ? x : v;
    }
    return v;
}

template <int TYPE>
__device__ __forceinline__ void exclude_items(const SampleArgs &a, const int64_t r, const RowView<TYPE> &view) {
    const int64_t er = a.ex_rows ? a.ex_rows[r] : r;
    for (int64_t q = a.ex_rowptr[er] + threadIdx.x; q < a.ex_rowptr[er + 1]; q += blockDim.x) {
        const int32_t i = a.ex_col[q];
        if (i >= 0 && i < a.M) RowView<TYPE>::put((char *)view.base, i, -__builtin_inff());
    }
}

// ----------------------------------------------------------------------------- 16-bit rows
// The histogram of a row by its values: 16-bit scores have few (a few thousand where a catalogue has 10^5 items), so they are
// counted, 16 bits for a value and 16 for its negative in one word of LDS, and weighed once each - eight instructions and an
// LDS atomic per item instead of forty and two.  A word per magnitude from the largest that can count downwards; the few
// items of smaller magnitude are listed.  False, with sh.wsum and sh.cnt in disorder, if their list or a count overflows
// (a row of equal scores, or most scores 2^-8 of the largest or less): the caller weighs item by item.
template <class G, int TYPE>
__device__ __forceinline__ bool count_values(const RowView<TYPE> &view, const RowScale &c, const float reach, const float low,
                                             const bool counted, SampleShared<G> &sh) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    constexpr int FEW = 2048;
    __shared__ unsigned short few[FEW];
    __shared__ uint32_t n_few;
    constexpr uint32_t INF = TYPE == ROW_F16 ? 0x7c00u : 0x7f80u;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    auto bits_above = [](const float v) {                    // of a 16-bit value above v >= 0
        if constexpr (TYPE == ROW_BF16) return (__float_as_uint(v) >> 16) + 1;
        return v < 65504.f ? (uint32_t)__builtin_bit_cast(unsigned short, (_Float16)v) + 1 : INF;
    };
    auto value_of = [](const uint32_t bits) { return RowView<TYPE>::value(row_u32x4{bits, 0, 0, 0}, 0); };
    const float floor = c.top_f - reach;
    const uint32_t most = min(INF - 1, max(bits_above(fabsf(c.top_f)), floor < 0.f ? bits_above(-floor) : 0u));
    const uint32_t cap = min((uint32_t)SampleShared<G>::VALUES - 1, most + 1), first = most + 1 - cap;       // word t: magnitude first + t
    // how many those few may be: of scores spread like a normal distribution's, |s| < v has 0.8 v / sigma, and a row eight sigma
    if (first != 0 && value_of(first) * (float)view.M * 6.4f > 0.75f * (float)FEW * (c.top_f - low)) return false;
    for (uint32_t t = tid; t < cap; t += G::THREADS) sh.values[t] = 0;
    if (tid == 0) n_few = 0;
    __syncthreads();
    const u16x2 first2{(unsigned short)first, (unsigned short)first}, cap2{(unsigned short)cap, (unsigned short)cap};
    uint32_t n_in = 0, zeros = 0;                            // n_in: of the wave; its first lane has all of it
    auto add = [&](const uint32_t t4, const uint32_t sign) {
        const bool in = t4 < 4 * cap;
        n_in += (uint32_t)__popcll(__ballot(in));
        if (in) atomicAdd((uint32_t *)((char *)sh.values + t4), sign ? 0x10000u : 1u);
    };
    auto add_few = [&](const uint32_t bits) {
        if ((bits & 0x7fff) == 0) ++zeros;
        else {
            const uint32_t at = atomicAdd(&n_few, 1u);
            if (at < (uint32_t)FEW) few[at] = (unsigned short)bits;
        }
    };
    each_quad<G>(view, 0, view.n_chunks, [&](const row_u32x4 (&v)[4], const int32_t) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            u16x2 least = cap2;
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const uint32_t w = v[k][d];
                const u16x2 t = __builtin_elementwise_min(
                    __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, w & 0x7fff7fffu), first2), cap2);
                least = __builtin_elementwise_min(least, t);
                const uint32_t t4 = __builtin_bit_cast(uint32_t, (u16x2)(t << (unsigned short)2));
                add(t4 & 0xffffu, w & 0x8000u);
                add(t4 >> 16, w & 0x80000000u);
            }
            if (first != 0 && (least[0] == 0 || least[1] == 0)) {
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const uint32_t w = v[k][d];
                    if ((w & 0x7fffu) <= first) add_few(w & 0xffffu);
                    if ((w >> 16 & 0x7fffu) <= first) add_few(w >> 16);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        return true;
    });
    __syncthreads();
    auto put = [&](const float s, const uint32_t n) {        // n items of score s
        const uint32_t b = bucket_of<G::BUCKETS>(s, c);
        u64 w;
        if (weigh(s, c, sh.pow2, w) && b < (uint32_t)G::BUCKETS) {
            atomicAdd(&sh.wsum[b], w * n);
            if (counted) atomicAdd(&sh.cnt[b], n);
        }
    };
    uint32_t sum = lane == 0 ? 0u - n_in : 0u;
#pragma unroll 1
    for (uint32_t t = tid; t < cap; t += 2 * G::THREADS) {   // two words, four values, at a time
        const uint32_t t1 = t + G::THREADS;
        uint32_t n0 = sh.values[t], n1 = t1 < cap ? sh.values[t1] : 0;
        sum += (n0 & 0xffffu) + (n0 >> 16) + (n1 & 0xffffu) + (n1 >> 16);
        if (t == 0 && first != 0) n0 = 0;
        if ((n0 | n1) == 0) continue;
        const float s0 = value_of(first + t), s1 = value_of(first + t1);
        const float s[4] = {s0, -s0, s1, -s1};
        const uint32_t n[4] = {n0 & 0xffffu, n0 >> 16, n1 & 0xffffu, n1 >> 16};
        u64 w[4];
        bool in[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) in[q] = weigh(s[q], c, sh.pow2, w[q]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t b = bucket_of<G::BUCKETS>(s[q], c);
            if (in[q] && n[q] && b < (uint32_t)G::BUCKETS) {
                atomicAdd(&sh.wsum[b], w[q] * n[q]);
                if (counted) atomicAdd(&sh.cnt[b], n[q]);
            }
        }
    }
    if (zeros) put(0.f, zeros);
    const uint32_t n = n_few;
    for (uint32_t q = tid; q < min(n, (uint32_t)FEW); q += G::THREADS) put(value_of(few[q]), 1);
    {
        const int32_t x = view.extra(tid);
        if (x >= 0) put(view.at(x), 1);
    }
    sum = wave_scan(sum);
    __syncthreads();
    if (lane == 63) sh.wave_c[wave] = sum;
    __syncthreads();
    return sum_of_first<G>(sh.wave_c, G::WAVES) == 0 && n <= (uint32_t)FEW;
}

// ----------------------------------------------------------------------------- one workgroup per row
template <class G, int TYPE>
__global__ __launch_bounds__(G::THREADS, 4) void sample_rows_kernel(const SampleArgs a) {
    __shared__ SampleShared<G> sh;
    __shared__ unsigned char want[G::BUCKETS + G::EDGE + 1];
    __shared__ uint32_t n_found;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r = row_of_block();
    if (r >= a.n) return;
    const RowView<TYPE> view(a.scores, r, a.lds, a.M);
    if (a.ex_rowptr) {
        exclude_items<TYPE>(a, r, view);
        __syncthreads();
    }
    constexpr int VEC = RowView<TYPE>::VEC, STEP = G::THREADS * VEC;
    constexpr int AHEAD = TYPE == ROW_F32 ? 2 : 1;           // quads under way (4096 x 59047 f32: 234 us, 238 with one; 16-bit: spills)
    auto load_quad = [&](row_u32x4 (&v)[4], const int32_t q) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[k] = RowView<TYPE>::nothing();
            if (q + k * G::THREADS < view.n_chunks) v[k] = view.load(q + k * G::THREADS);
        }
    };
    row_u32x4 v[4], next[AHEAD][4];
    load_quad(v, tid);                                       // under way while the tables are made
    const int32_t x = view.extra(tid);
    const float x_score = x >= 0 ? view.at(x) : -__builtin_inff();
    const RowParams p = row_params(a, r);
    if (tid < 256) sh.pow2[tid] = exp2((double)tid / 256.0 + a.q_bits);
#pragma unroll
    for (int q = 0; q < G::OWN; ++q) { sh.cnt[q * G::THREADS + tid] = 0; sh.wsum[q * G::THREADS + tid] = 0; }
    if (tid == 0) { sh.base_w = ~0ull; n_found = 0; }

    // One pass over the row finds its maximum and, on the way, collects the items that can matter, unweighed: those within
    // the cut below the maximum so far, and at or above a score that some more than top_k items are likely to reach.  (A
    // filtered row has a few per cent of them, spread over all waves: weighed where they are found they would cost a whole
    // wave's weighing each.)  A row whose items do not fit the list is read again, see below.
    auto collect = [&](const row_u32x4 (&v)[4], const int32_t i0, auto wanted) {
        bool go = true;
#pragma unroll
        for (int half = 0; half < (VEC == 4 ? 1 : 2); ++half) {                // 16 elements per lane, one counter step per wave
            constexpr int CHUNKS = VEC == 4 ? 4 : 2;
            u64 taken[16];
            uint32_t total = 0;
#pragma unroll
            for (int q = 0; q < 16; ++q) {
                taken[q] = __ballot(wanted(RowView<TYPE>::value(v[half * CHUNKS + q / VEC], q % VEC)));
                total += (uint32_t)__popcll(taken[q]);
            }
            if (total == 0) continue;                        // uniform, as `total` is
            uint32_t base = 0;
            if (__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)) == (uint32_t)__ffsll(__ballot(1)) - 1)
                base = atomicAdd(&n_found, total);           // the first active lane, for the wave
            base = uniform(base);
            if (base >= (uint32_t)LISTED) return false;
#pragma unroll
            for (int q = 0; q < 16; ++q) {
                if (taken[q] == 0) continue;                 // uniform: most of them in a filtered row
                const float s = RowView<TYPE>::value(v[half * CHUNKS + q / VEC], q % VEC);
                const uint32_t at = base + __builtin_amdgcn_mbcnt_hi((uint32_t)(taken[q] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)taken[q], 0u));
                if (wanted(s) && at < (uint32_t)LISTED) sh.found[at] = Found{s, i0 + (half * CHUNKS + q / VEC) * STEP + q % VEC};
                base += (uint32_t)__popcll(taken[q]);
            }
            go = go && base <= (uint32_t)LISTED;
        }
        return go;
    };
    auto collect_one = [&](const float s, const int32_t i) {
        const uint32_t at = atomicAdd(&n_found, 1u);
        if (at < (uint32_t)LISTED) sh.found[at] = Found{s, i};
    };
    float hi = -__builtin_inff(), low = __builtin_inff();     // low: of the first chunks, it only sets the buckets' width
    auto top_of = [&](const row_u32x4 (&v)[4]) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) hi = fmaxf(hi, RowView<TYPE>::value(v[k], e));
    };
    // over the workgroup
    auto join_seen = [&]() {
        hi = wave_ends(hi, low);
        if (lane == 63) { sh.wave_f[wave] = hi; sh.wave_g[wave] = low; }
        __syncthreads();
        hi = sh.wave_f[0]; low = sh.wave_g[0];
#pragma unroll
        for (int q = 1; q < G::WAVES; ++q) { hi = fmaxf(hi, sh.wave_f[q]); low = fminf(low, sh.wave_g[q]); }
        __syncthreads();
    };
    const double cut = item_cut(p, a.q_bits);
    const bool drawn = p.T > 0.f;
    const float reach = drawn ? score_reach(cut, p.T) * 1.0001f : 0.f;         // items further below the top do not count
    float at_least = -__builtin_inff();                                        // top-k: a score to start from
    const bool counted = top_k_asked(a, p);
    {
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) load_quad(next[d], tid + 4 * (d + 1) * G::THREADS);
        top_of(v);
        hi = fmaxf(hi, x_score);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float s = RowView<TYPE>::value(v[k], e);
                low = fminf(low, s > -1e30f ? s : __builtin_inff());
            }
        join_seen();
        const float seen = fminf(2.f * STEP, (float)a.M), share = seen / (float)a.M, expect = share * (float)p.top_k;
        const float enough = 1.5f * expect + 4.f * sqrtf(expect) + 8.f;        // of the first two chunks' items
        if (counted && drawn && fabsf(hi) < __builtin_inff() && enough < 0.8f * share * (float)LISTED && hi > low) {
            const float per = (float)G::BUCKETS / (hi - low), top = hi;
            auto count = [&](const float s) {
                const float t = (top - s) * per;
                if (t < (float)G::BUCKETS) atomicAdd(&sh.cnt[(int)t], 1u);
            };
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) count(RowView<TYPE>::value(v[k], e));
            __syncthreads();
            scan_buckets(sh.cnt, sh.wsum, sh);
            int b, same;
            buckets_passing(sh.cnt, (u64)enough, (u64)enough, sh, b, same);
            at_least = uniform(hi - (float)(b + 1) / per);
#pragma unroll
            for (int q = 0; q < G::OWN; ++q) sh.cnt[q * G::THREADS + tid] = 0;
            __syncthreads();
        }
        bool collecting = hi < __builtin_inff();
        float floor = fmaxf(fmaxf(hi - reach, at_least), -3.402823466e38f);    // at the least everything but -inf
        auto wanted = [&](const float s) { return s >= floor; };
        if (collecting) {
            if (wanted(x_score)) collect_one(x_score, x);
            collecting = __all(collect(v, view.index0(tid), wanted));
        }
#pragma unroll 1
        for (int32_t q = tid + 4 * G::THREADS; q - tid < view.n_chunks; q += 4 * G::THREADS) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[k] = next[0][k];
#pragma unroll
                for (int d = 0; d + 1 < AHEAD; ++d) next[d][k] = next[d + 1][k];
            }
            load_quad(next[AHEAD - 1], q + 4 * AHEAD * G::THREADS);
            top_of(v);
            if (collecting) {                                // per wave
                floor = fmaxf(floor, hi - reach);            // the lane's own maximum: never above the row's
                collecting = __all(collect(v, view.index0(q), wanted));
            }
        }
        join_seen();
    }

    if (hi == -__builtin_inff()) {                            // nothing to draw from
        answer_all(a, r, -1, -__builtin_inff());
        return;
    }
    if (!drawn) {                                             // the best item: lowest column of the largest score
        auto see = [&](const float s, const int32_t i) { if (s == hi) atomicMin(&sh.base_w, (u64)i); };
        const uint32_t n = n_found;                           // 0: +inf among the first items
        if (n == 0 || n > (uint32_t)LISTED) each_again<G>(view, see);
        else for (uint32_t q = tid; q < n; q += G::THREADS) see(sh.found[q].score, sh.found[q].index);
        __syncthreads();
        answer_all(a, r, (int32_t)sh.base_w, 0.f);
        return;
    }
    if (hi == __builtin_inff()) {
        answer_infinite<G>(a, r, view, p, sh);
        return;
    }
    const RowScale c = row_scale(hi, low, cut, p, a.q_bits, G::BUCKETS);
    bool fits = n_found <= (uint32_t)LISTED;
    if (fits) {
        const uint32_t n = n_found;
#pragma unroll 1
        for (uint32_t q = tid; q < n; q += G::THREADS) {
            const float s = sh.found[q].score;
            const uint32_t b = bucket_of<G::BUCKETS>(s, c);
            u64 w;
            if (weigh(s, c, sh.pow2, w)) {
                atomicAdd(&sh.wsum[b], w);
                if (counted) atomicAdd(&sh.cnt[b], 1u);
            }
        }
        __syncthreads();
        scan_buckets(sh.cnt, sh.wsum, sh);
        // started from a score that fewer than top_k reach, although items below it count
        if (counted && at_least > hi - reach && sh.cnt[G::BUCKETS - 1] < (uint32_t)p.top_k) {
            fits = false;
            __syncthreads();
#pragma unroll
            for (int q = 0; q < G::OWN; ++q) { sh.cnt[q * G::THREADS + tid] = 0; sh.wsum[q * G::THREADS + tid] = 0; }
            __syncthreads();
        }
    }
    if (!fits) {
        // a row of which much counts: weighed as it is read; one more pass collects whatever the answers can be
        bool weighed = false;
        if constexpr (TYPE != ROW_F32 && G::BY_VALUE) {
            // bfloat16 has few values in any row of this group (161 against 182 us at 33 001 items); float16 eight times as
            // many, worth it from about 80 000 items on (257 against 279 us at 131 071, but 292 against 276 at 65 535)
            const bool by_value = TYPE == ROW_BF16 || view.M >= 81920;
            if (by_value) weighed = count_values<G>(view, c, reach, low, counted, sh);
            if (by_value && !weighed) {
                __syncthreads();
#pragma unroll
                for (int q = 0; q < G::OWN; ++q) { sh.cnt[q * G::THREADS + tid] = 0; sh.wsum[q * G::THREADS + tid] = 0; }
                __syncthreads();
            }
        }
        if (!weighed) {
            load_quad(v, tid);
            each_bucket<G>(view, 0, view.n_chunks, true, v, c, [&](const float (&s)[4], const int32_t, const uint32_t (&b)[4]) {
                count_four<G::BUCKETS>(s, b, c, sh.pow2, sh.cnt, sh.wsum, counted);
                return true;
            });
        }
        __syncthreads();
        scan_buckets(sh.cnt, sh.wsum, sh);
        wanted_buckets(a, r, p, c.reject > (float)G::BUCKETS * 1.02f, sh, want);
        if (tid == 0) n_found = 0;
        __syncthreads();
        auto wanted = [&](const float s) {
            // bucket_of without the cut: an item beyond it is in the list for nothing
            return want[(uint32_t)fminf((c.top_f - s) * c.per_score, (float)(G::BUCKETS + G::EDGE))] != 0;
        };
        each_quad<G>(view, 0, view.n_chunks, [&](const row_u32x4 (&v)[4], const int32_t i0) { return collect(v, i0, wanted); });
        const int32_t x = view.extra(tid);
        if (x >= 0 && wanted(view.at(x))) collect_one(view.at(x), x);
        __syncthreads();
    }
    const bool whole = n_found > (uint32_t)LISTED;           // more than the list holds: the answers come from memory
    const Unlisted<G, TYPE> list{view, sh.found, n_found, whole};
    answer<G, TYPE, false>(a, r, list, !whole, counted, view, c, p, sh);
}

// ----------------------------------------------------------------------------- cut rows
typedef Large G;
template <int TYPE>
__global__ __launch_bounds__(256) void exclude_kernel(const SampleArgs a) {
    const RowView<TYPE> view(a.scores, blockIdx.x, a.lds, a.M);
    exclude_items<TYPE>(a, blockIdx.x, view);
}

// 1. Every part's best item and smallest scores; clears the row's histogram and list.
template <int TYPE>
__global__ __launch_bounds__(G::THREADS) void part_stats_kernel(const SampleArgs a) {
    __shared__ u64 best_[G::WAVES];
    __shared__ float low_[G::WAVES];
    const int64_t r = blockIdx.x / a.n_parts;
    const int part = blockIdx.x % a.n_parts, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int b = part * G::THREADS + tid; b < G::BUCKETS; b += a.n_parts * G::THREADS) { a.cnt[r * G::BUCKETS + b] = 0; a.wsum[r * G::BUCKETS + b] = 0; }
    if (part == 0 && tid == 0) a.n_found[r] = 0;
    const RowView<TYPE> view(a.scores, r, a.lds, a.M);
    const int32_t q0 = part * a.per_part, q1 = min(q0 + a.per_part, view.n_chunks);
    float hi = -__builtin_inff(), low = __builtin_inff();
    int32_t at = 0x7fffffff;
    auto see = [&](const float s, const int32_t i) {
        if (s > hi || (s == hi && i < at)) { hi = s; at = i; }
        low = fminf(low, s > -1e30f ? s : __builtin_inff());
    };
    row_u32x4 first[4];
    load_four<G>(view, q0 + tid, q1, first);
    each_chunk<G>(view, q0, q1, first, [&](const row_u32x4 &v, const int32_t i0) {
#pragma unroll
        for (int e = 0; e < RowView<TYPE>::VEC; ++e) see(RowView<TYPE>::value(v, e), i0 + e);
        return true;
    });
    {
        const int32_t x = part == 0 ? view.extra(tid) : -1;
        if (x >= 0) see(view.at(x), x);
    }
    u64 best = wave_max64((u64)rank_key(hi) << 32 | (uint32_t)~(uint32_t)at);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) low = fminf(low, __shfl_xor(low, o));
    if (lane == 0) { best_[wave] = best; low_[wave] = low; }
    __syncthreads();
    if (tid == 0) {
        for (int v = 1; v < G::WAVES; ++v) {
            best = best_[v] > best ? best_[v] : best; low = fminf(low, low_[v]);
        }
        a.stats[blockIdx.x] = PartStat{best, low, 0.f};
    }
}
// The row's, from its parts'.  Every wave computes it.
__device__ __forceinline__ PartStat join_stats(const SampleArgs &a, const int64_t r) {
    PartStat s{0, __builtin_inff(), 0.f};
    for (int q = threadIdx.x & 63; q < a.n_parts; q += 64) {
        const PartStat x = a.stats[r * a.n_parts + q];
        s.best = x.best > s.best ? x.best : s.best;
        s.low = fminf(s.low, x.low);
    }
    s.best = wave_max64(s.best);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s.low = fminf(s.low, __shfl_xor(s.low, o));
    return s;
}

// 2. Every part's histogram, added to the row's by integer atomics.
template <int TYPE>
__global__ __launch_bounds__(G::THREADS) void part_histogram_kernel(const SampleArgs a) {
    __shared__ u64 wsum[G::BUCKETS];
    __shared__ uint32_t cnt[G::BUCKETS];
    __shared__ double pow2[256];
    const int64_t r = blockIdx.x / a.n_parts;
    const int part = blockIdx.x % a.n_parts, tid = threadIdx.x;
    const RowView<TYPE> view(a.scores, r, a.lds, a.M);
    const int32_t q0 = part * a.per_part, q1 = min(q0 + a.per_part, view.n_chunks);
    row_u32x4 first[4];
    load_four<G>(view, q0 + tid, q1, first);                  // under way while the parts' maxima are joined
    const RowParams p = row_params(a, r);
    const PartStat st = join_stats(a, r);
    const float hi = key_score((uint32_t)(st.best >> 32));
    if (!(fabsf(hi) < __builtin_inff()) || !(p.T > 0.f)) return;      // answered apart
    if (tid < 256) pow2[tid] = exp2((double)tid / 256.0 + a.q_bits);
    for (int b = tid; b < G::BUCKETS; b += G::THREADS) { cnt[b] = 0; wsum[b] = 0; }
    const RowScale c = row_scale(hi, st.low, item_cut(p, a.q_bits), p, a.q_bits, G::BUCKETS);
    __syncthreads();
    each_bucket<G>(view, q0, q1, part == 0, first, c, [&](const float (&s)[4], const int32_t, const uint32_t (&b)[4]) {
        count_four<G::BUCKETS>(s, b, c, pow2, cnt, wsum, true);
        return true;
    });
    __syncthreads();
    for (int b = tid; b < G::BUCKETS; b += G::THREADS)
        if (wsum[b]) { atomicAdd(&a.cnt[r * G::BUCKETS + b], cnt[b]); atomicAdd(&a.wsum[r * G::BUCKETS + b], wsum[b]); }
}

// The row's histogram, loaded early and turned into running sums.
struct Histogram {
    uint32_t cnt[G::OWN];
    u64 wsum[G::OWN];
    __device__ __forceinline__ void load(const SampleArgs &a, const int64_t r) {
#pragma unroll
        for (int h = 0; h < G::OWN; ++h) {
            const int b = threadIdx.x + h * G::THREADS;
            cnt[h] = a.cnt[r * G::BUCKETS + b];
            wsum[h] = a.wsum[r * G::BUCKETS + b];
        }
    }
    __device__ __forceinline__ void scan(SampleShared<G> &sh) const {
#pragma unroll
        for (int h = 0; h < G::OWN; ++h) { sh.cnt[threadIdx.x + h * G::THREADS] = cnt[h]; sh.wsum[threadIdx.x + h * G::THREADS] = wsum[h]; }
        __syncthreads();
        scan_buckets(sh.cnt, sh.wsum, sh);
    }
};
// 3. The items of those buckets.
template <int TYPE>
__global__ __launch_bounds__(G::THREADS) void part_collect_kernel(const SampleArgs a) {
    __shared__ SampleShared<G> sh;
    __shared__ unsigned char want[G::BUCKETS + G::EDGE + 1];
    __shared__ uint32_t n_local, base;
    if (threadIdx.x == 0) n_local = 0;
    const int64_t r = blockIdx.x / a.n_parts;
    const int part = blockIdx.x % a.n_parts;
    const RowView<TYPE> view(a.scores, r, a.lds, a.M);
    const int32_t q0 = part * a.per_part, q1 = min(q0 + a.per_part, view.n_chunks);
    row_u32x4 first[4];
    load_four<G>(view, q0 + threadIdx.x, q1, first);
    Histogram h;
    h.load(a, r);
    const RowParams p = row_params(a, r);
    const PartStat st = join_stats(a, r);
    const float hi = key_score((uint32_t)(st.best >> 32));
    if (!(fabsf(hi) < __builtin_inff()) || !(p.T > 0.f)) return;      // answered apart
    const RowScale c = row_scale(hi, st.low, item_cut(p, a.q_bits), p, a.q_bits, G::BUCKETS);
    h.scan(sh);
    wanted_buckets(a, r, p, false, sh, want);
    each_bucket<G>(view, q0, q1, part == 0, first, c, [&](const float (&s)[4], const int32_t i, const uint32_t (&b)[4]) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (b[q] >= (uint32_t)G::BUCKETS || !want[b[q]]) continue;
            uint32_t at = atomicAdd(&n_local, 1u);
            if (at < (uint32_t)LISTED) sh.found[at] = Found{s[q], i + q};
            else {                                           // more than LDS holds
                at = atomicAdd(&a.n_found[r], 1u);
                if (at < SR_LISTED) a.found[r * SR_LISTED + at] = Found{s[q], i + q};
            }
        }
        return true;
    });
    // one step of the row's counter per workgroup (11.1 us for one row of a million; 13.6 with a step per item)
    __syncthreads();
    const uint32_t n = min(n_local, (uint32_t)LISTED);
    if (threadIdx.x == 0 && n) base = atomicAdd(&a.n_found[r], n);
    __syncthreads();
    for (uint32_t q = threadIdx.x; q < n; q += G::THREADS)
        if (base + q < SR_LISTED) a.found[r * SR_LISTED + base + q] = sh.found[q];
}

// 4. The answers.
template <int TYPE>
__global__ __launch_bounds__(G::THREADS) void part_answer_kernel(const SampleArgs a) {
    __shared__ SampleShared<G> sh;
    const int64_t r = blockIdx.x;
    Histogram h;
    h.load(a, r);
    const uint32_t n = a.n_found[r];
    const RowParams p = row_params(a, r);
    const PartStat st = join_stats(a, r);
    const float hi = key_score((uint32_t)(st.best >> 32));
    if (hi == -__builtin_inff()) {
        answer_all(a, r, -1, -__builtin_inff());
        return;
    }
    if (!(p.T > 0.f)) {
        answer_all(a, r, (int32_t)~(uint32_t)st.best, 0.f);
        return;
    }
    const RowView<TYPE> view(a.scores, r, a.lds, a.M);
    if (hi == __builtin_inff()) {
        answer_infinite<G>(a, r, view, p, sh);
        return;
    }
    if (threadIdx.x < 256) sh.pow2[threadIdx.x] = exp2((double)threadIdx.x / 256.0 + a.q_bits);
    const RowScale c = row_scale(hi, st.low, item_cut(p, a.q_bits), p, a.q_bits, G::BUCKETS);
    h.scan(sh);
    const bool in_lds = n <= (uint32_t)LISTED;                // it is read once per step and round
    if (in_lds) {
        for (uint32_t q = threadIdx.x; q < n; q += G::THREADS) sh.found[q] = a.found[r * SR_LISTED + q];
        __syncthreads();
    }
    const Unlisted<G, TYPE> row{view, a.found + r * SR_LISTED, n, n > SR_LISTED};       // more than the list holds: from the row
    answer<G, TYPE, true>(a, r, row, in_lds, true, view, c, p, sh);
}

// ----------------------------------------------------------------------------- host
// Rows of 65 536 items and more (32-bit; 131 072 of 16 bits) are cut while they are few: 64 at 131 072 items, 128 from 262 144 on.
// Cut or not, in us (float32, top-p): 1 x 131071 31 / 75, 64 x 131071 54 / 82, 256 x 131071 120 / 98; 1 x 1000003 37 / 470,
// 128 x 1000003 398 / 658.  Filtered rows need one pass: 28 / 28, 48 / 32 at 64 x 131071, 319 / 441 at 128 x 1000003.
constexpr int64_t CUT_CHUNKS = 16384;
int64_t cut_rows(const int64_t M) { return std::min<int64_t>(128, M / 2048); }
// The small workgroup, of which four are resident per compute unit instead of two: for short rows, and for longer ones if
// there are more of them than the large workgroups that are resident.  Small / large in us (float32, all filters; none):
// 2000 x 9724 38 / 72; 57 / 80, 2000 x 32768 61 / 86; 136 / 145, 4096 x 59047 190 / 218; 461 / 476, 1000 x 100003 87 / 92; 225 / 217,
// 300 x 24576 21 / 24; 37 / 32.  With more draws per row the wider buckets of the small one overflow the list: 8 draws of
// 600 x 65000, all filters 44 / 53, none 146 / 116, every row its own 301 / 126.
constexpr int64_t SMALL_CHUNKS = 4096, SMALL_ITEMS = 65536, LARGE_RESIDENT = 512;
struct CutPlan {
    int32_t n_parts, per_part;        // n_parts == 0: one workgroup per row
    size_t off_wsum, off_cnt, off_nfound, off_found, total;
};
CutPlan cut_plan(const int32_t dtype, const int64_t n, const int64_t M) {
    CutPlan p{0, 0, 0, 0, 0, 0, 0};
    const int64_t chunks = M / (dtype == ALS_DTYPE_F32 ? 4 : 8);
    if (chunks <= CUT_CHUNKS || n > cut_rows(M)) return p;
    // about 512 workgroups, of two chunks per thread or more each
    const int64_t want = std::max<int64_t>((512 + n - 1) / n, 4);
    p.n_parts = (int32_t)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, 128), chunks / (4 * G::THREADS)));
    p.per_part = (int32_t)((chunks + p.n_parts - 1) / p.n_parts + 1);        // + 1: the row's alignment may add none, but cover all
    size_t at = 0;
    auto take = [&](const size_t bytes) { const size_t here = at; at += (bytes + 255) / 256 * 256; return here; };
    take((size_t)n * p.n_parts * sizeof(PartStat));
    p.off_wsum = take((size_t)n * CUT_BUCKETS * 8);
    p.off_cnt = take((size_t)n * CUT_BUCKETS * 4);
    p.off_nfound = take((size_t)n * 4);
    p.off_found = take((size_t)n * SR_LISTED * sizeof(Found));
    p.total = at;
    return p;
}

template <int TYPE>
void launch(const SampleArgs &a, const int64_t n, hipStream_t st) {
    const dim3 rows = grid_of_rows(n), block(G::THREADS);
    if (a.n_parts == 0) {
        const int64_t chunks = a.M / RowView<TYPE>::VEC;
        if (chunks <= SMALL_CHUNKS || (n > LARGE_RESIDENT && a.M <= SMALL_ITEMS && a.n_draws <= 2)) hipLaunchKernelGGL((sample_rows_kernel<Small, TYPE>), rows, dim3(Small::THREADS), 0, st, a);
        else hipLaunchKernelGGL((sample_rows_kernel<Large, TYPE>), rows, block, 0, st, a);
        return;
    }
    const dim3 parts((unsigned)(n * a.n_parts));
    if (a.ex_rowptr) hipLaunchKernelGGL((exclude_kernel<TYPE>), rows, dim3(256), 0, st, a);
    hipLaunchKernelGGL((part_stats_kernel<TYPE>), parts, block, 0, st, a);
    hipLaunchKernelGGL((part_histogram_kernel<TYPE>), parts, block, 0, st, a);
    hipLaunchKernelGGL((part_collect_kernel<TYPE>), parts, block, 0, st, a);
    hipLaunchKernelGGL((part_answer_kernel<TYPE>), rows, block, 0, st, a);
}

}  // namespace

extern "C" {

size_t als_sample_rows_workspace_bytes(int32_t dtype, int64_t n_rows, int64_t M) {
    if (dtype < ALS_DTYPE_F32 || dtype > ALS_DTYPE_BF16 || n_rows < 1 || M < 1 || M > ROW_MAX) return 0;
    return cut_plan(dtype, n_rows, M).total;
}

int32_t als_sample_rows_max_draws(int64_t M) { return M < 1 || M > ROW_MAX ? 0 : draws_max(M); }

int32_t als_sample_rows(void *scores, int32_t dtype, int64_t lds, int64_t n_rows, int64_t M, const int64_t *ex_rowptr,
                        const int32_t *ex_col, const int64_t *ex_row_ids, const als_sample_opts_t *opts, const void *u,
                        int32_t u_is_f64, int32_t n_draws, int32_t *idx_out, float *logp_out, void *workspace, size_t ws_bytes,
                        void *stream) {
    if (!scores || !opts || !u || !idx_out || !logp_out)
        return als_fail_(ALS_ERR_INVALID_ARG, "als_sample_rows: null pointer");
    if (n_rows < 1 || M < 1 || lds < M || M > ROW_MAX || n_rows > INT32_MAX || n_draws < 1 || n_draws > draws_max(M))
        return als_fail_(ALS_ERR_INVALID_ARG, "als_sample_rows: bad sizes (n_rows=%lld M=%lld lds=%lld n_draws=%d)", (long long)n_rows,
                         (long long)M, (long long)lds, n_draws);
    if (dtype < ALS_DTYPE_F32 || dtype > ALS_DTYPE_BF16)
        return als_fail_(ALS_ERR_UNSUPPORTED, "als_sample_rows: dtype %d (0 float32, 1 float16, 2 bfloat16)", dtype);
    if ((uintptr_t)scores % (dtype == ALS_DTYPE_F32 ? 4 : 2))
        return als_fail_(ALS_ERR_INVALID_ARG, "als_sample_rows: scores are not aligned to their type");
    if ((ex_rowptr == nullptr) != (ex_col == nullptr))
        return als_fail_(ALS_ERR_INVALID_ARG, "als_sample_rows: pass both exclusion arrays or neither");
    const CutPlan plan = cut_plan(dtype, n_rows, M);
    if (plan.total && (!workspace || ws_bytes < plan.total || (uintptr_t)workspace % 16))
        return als_fail_(ALS_ERR_WORKSPACE, "als_sample_rows: workspace too small or not 16-byte aligned: %zu < %zu", ws_bytes, plan.total);
    SampleArgs a;
    a.scores = scores; a.lds = lds; a.n = n_rows; a.M = M;
    a.ex_rowptr = ex_rowptr; a.ex_col = ex_col; a.ex_rows = ex_rowptr ? ex_row_ids : nullptr;
    a.o = *opts;
    a.u = u; a.u_f64 = u_is_f64 != 0; a.n_draws = n_draws;
    int bits = 0;
    while ((1LL << bits) < M) ++bits;
    a.q_bits = std::min(51, 62 - bits);
    a.idx = idx_out; a.logp = logp_out;
    char *ws = (char *)workspace;
    a.n_parts = plan.n_parts; a.per_part = plan.per_part;
    a.stats = (PartStat *)ws; a.wsum = (u64 *)(ws + plan.off_wsum); a.cnt = (uint32_t *)(ws + plan.off_cnt);
    a.n_found = (uint32_t *)(ws + plan.off_nfound); a.found = (Found *)(ws + plan.off_found);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ALS_DTYPE_F32) launch<ROW_F32>(a, n_rows, st);
    else if (dtype == ALS_DTYPE_F16) launch<ROW_F16>(a, n_rows, st);
    else launch<ROW_BF16>(a, n_rows, st);
    ALS_HIP_CHECK4(hipGetLastError());
    return ALS_OK;
}

}  // extern "C"

// Random draws from rows of scores: temperature, min-p, top-k, top-p and the draw itself, from given random numbers.
//
// The operator.  For one row s of M scores, T its temperature, x_i = (s_i - max s) / T, w_i = exp(x_i):
//   1. items with w_i < min_p are dropped;
//   2. of the rest, in rank order (score descending, ties by ascending column), the first top_k stay;
//   3. of those the shortest prefix stays whose weight reaches top_p times theirs;
//   4. with W the weight of what is left and u in [0, 1): the draw is the first item in rank order at which the running
//      weight exceeds u W; its ln(w_i / W) is returned beside it.
// Every step asks the same question - at which item, in rank order, does a running sum (of ones, or of weights) pass a
// target - and the kernel has one answer to it (find): a histogram of the row over 2048 buckets of equal width in the
// score gives the bucket, the bucket's few items are collected in LDS and ranked against each other.  Nothing is sorted.
//
// Weights are held as integers, round(w 2^Q) with Q = min(51, 62 - ceil(log2 M)): their sums are exact whatever the order,
// so LDS atomics do not make the result depend on timing, and a draw differs from the definition's only where u W lies
// within the summed roundings of a border.  With M = 59 047 (Q = 46) that is a part in 10^11 of W; float32 sums would
// decide one draw in a hundred wrongly on a catalogue of a million.  An item whose weight rounds to 0 (below 2^-47 of the
// largest) counts as dropped.  exp is computed in float64 (which this chip multiplies at the float32 rate): x 256 / ln 2 =
// k + r, 2^(k mod 256 / 256) from a table, a polynomial of degree 4 in r; error below 1e-15.
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

constexpr int SR_THREADS = 1024;
constexpr int SR_BUCKETS = 2048;      // 2 per thread
constexpr int SR_LIST = 1024;         // items of one bucket that are ranked directly
constexpr int SR_WAVES = SR_THREADS / 64;

struct SampleArgs {
    void *scores;
    int64_t lds, M;
    const int64_t *ex_rowptr;
    const int32_t *ex_col;
    const int64_t *ex_rows;
    als_sample_opts_t o;
    const void *u;
    int32_t u_f64, n_draws, q_bits;
    int32_t *idx;
    float *logp;
};

// floats as unsigned keys of the same order
__device__ __forceinline__ uint32_t rank_key(const float s) {
    const uint32_t b = __float_as_uint(s + 0.f);            // -0 and +0 are one score: -0 + 0 = +0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Picked {
    u64 before, weight;       // running weight in front of the item, its own
    int32_t index;
};

struct SampleShared {
    u64 wsum[SR_BUCKETS], wsub[SR_BUCKETS];
    uint32_t cnt[SR_BUCKETS], csub[SR_BUCKETS];
    u64 list[SR_LIST][2];           // (key << 32 | ~index, weight)
    double pow2[256];               // 2^(i / 256)
    u64 wave_w[SR_WAVES];
    uint32_t wave_c[SR_WAVES];
    float wave_f[SR_WAVES], wave_g[SR_WAVES];
    Picked picked;
    uint32_t bucket, n_list;
    u64 base_w;
    uint32_t base_c, in_bucket;
};

// What the steps of one row share.
struct RowScale {
    float top;          // the largest score
    double inv_t;       // 1 / T
    double cut;         // items with x < -cut have no weight
    float min_p;
    float per_score;    // buckets per unit of score
    int q_bits;
};

// exp(x) for x in [-cut, 0], and its integer weight
__device__ __forceinline__ double exp_table(const double x, const double *pow2, int &k256) {
    constexpr double C = 256.0 * 1.4426950408889634074, MAGIC = 6755399441055744.0;      // 1.5 2^52: adds, rounds to an integer
    const double kd = fma(x, C, MAGIC);
    const int k = (int)(uint32_t)__double_as_longlong(kd);
    const double r = fma(x, C, -(kd - MAGIC)) * (0.69314718055994530942 / 256.0);
    const double p = fma(r, fma(r, fma(r, 1.0 / 24, 1.0 / 6), 0.5), 1.0);
    k256 = k >> 8;
    const double t = pow2[k & 255];
    return fma(t * r, p, t);
}
__device__ __forceinline__ bool weigh(const float s, const RowScale &c, const double *pow2, u64 &w) {
    const double d = s == c.top ? 0.0 : (double)s - (double)c.top;
    const double x = d * c.inv_t;
    if (!(x >= -c.cut)) return false;                       // NaN scores and NaN products (inf x 0) among them
    int e;
    const double m = exp_table(x, pow2, e);                 // w = m 2^e, m in [1, 2)
    const double w1 = __longlong_as_double(__double_as_longlong(m) + ((int64_t)e << 52));
    if (!(w1 >= (double)c.min_p)) return false;
    // w 2^Q + 2^52: the mantissa's low bits are the integer, rounded to nearest even
    const double q = __longlong_as_double(__double_as_longlong(w1) + ((int64_t)c.q_bits << 52)) + 4503599627370496.0;
    w = (u64)__double_as_longlong(q) & 0xfffffffffffffull;
    return w != 0;
}
// Bucket of a score: falls with the score (each operation is monotone), so buckets are runs of the rank order.
__device__ __forceinline__ uint32_t bucket_of(const float s, const RowScale &c) {
    const float b = (c.top - s) * c.per_score;
    return (uint32_t)(int)fminf(b, (float)(SR_BUCKETS - 1));
}

__device__ __forceinline__ u64 shfl_up64(const u64 v, const int o) {
    const uint32_t lo = (uint32_t)__shfl_up((int)(uint32_t)v, o), hi = (uint32_t)__shfl_up((int)(uint32_t)(v >> 32), o);
    return (u64)hi << 32 | lo;
}

// Inclusive running sums over the 2048 buckets of (cnt, wsum), in place; every thread owns two.
__device__ void scan_buckets(uint32_t *cnt, u64 *wsum, SampleShared &sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t c0 = cnt[2 * tid], c1 = cnt[2 * tid + 1];
    const u64 w0 = wsum[2 * tid], w1 = wsum[2 * tid + 1];
    uint32_t c = c0 + c1;
    u64 w = w0 + w1;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t cc = (uint32_t)__shfl_up((int)c, o);
        const u64 ww = shfl_up64(w, o);
        if (lane >= o) { c += cc; w += ww; }
    }
    if (lane == 63) { sh.wave_c[wave] = c; sh.wave_w[wave] = w; }
    __syncthreads();
    uint32_t bc = 0;
    u64 bw = 0;
    for (int v = 0; v < wave; ++v) { bc += sh.wave_c[v]; bw += sh.wave_w[v]; }
    cnt[2 * tid] = bc + c - c1; cnt[2 * tid + 1] = bc + c;
    wsum[2 * tid] = bw + w - w1; wsum[2 * tid + 1] = bw + w;
    __syncthreads();
}

// The bucket at which the running sum (of ones or of weights) passes `target`; base sums in front of it.
__device__ void pick_bucket(const uint32_t *cnt, const u64 *wsum, const bool by_count, const u64 target, const uint32_t base_c,
                            const u64 base_w, SampleShared &sh) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int b = 2 * threadIdx.x + h;
        const uint32_t pc = b ? cnt[b - 1] : 0, cc = cnt[b];
        const u64 pw = b ? wsum[b - 1] : 0, cw = wsum[b];
        const u64 lo = by_count ? base_c + pc : base_w + pw, hi = by_count ? base_c + cc : base_w + cw;
        if (lo <= target && target < hi) {
            sh.bucket = b; sh.in_bucket = cc - pc; sh.base_c = base_c + pc; sh.base_w = base_w + pw;
        }
    }
    __syncthreads();
}

// The row, either held in registers (NV chunks per thread) or read from memory again at every pass (NV = 0).
template <int TYPE, int NV>
struct RowStore {
    RowView<TYPE> view;
    row_u32x4 held[NV ? NV : 1];
    float extra;
    int32_t extra_at;

    __device__ __forceinline__ RowStore(const RowView<TYPE> &v) : view(v) {
        if constexpr (NV > 0) {
#pragma unroll
            for (int q = 0; q < NV; ++q) {
                held[q] = RowView<TYPE>::nothing();
                if (q * SR_THREADS + (int)threadIdx.x < view.n_chunks) held[q] = view.load(q * SR_THREADS + threadIdx.x);
            }
        }
        extra_at = view.extra(threadIdx.x);
        extra = extra_at >= 0 ? view.at(extra_at) : -__builtin_inff();
    }
    // f(score, index) for this thread's elements; what lies outside the row comes as -inf
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        if constexpr (NV > 0) {
#pragma unroll
            for (int q = 0; q < NV; ++q) {
                const int32_t i0 = view.index0(q * SR_THREADS + threadIdx.x);
#pragma unroll
                for (int e = 0; e < RowView<TYPE>::VEC; ++e) f(RowView<TYPE>::value(held[q], e), i0 + e);
            }
        } else {
            for (int32_t q = threadIdx.x; q < view.n_chunks; q += SR_THREADS) {
                const row_u32x4 v = view.load(q);
                const int32_t i0 = view.index0(q);
#pragma unroll
                for (int e = 0; e < RowView<TYPE>::VEC; ++e) f(RowView<TYPE>::value(v, e), i0 + e);
            }
        }
        if ((int)threadIdx.x < view.head + view.tail) f(extra, extra_at);
    }
};

// Index of the m-th element (from 0, in index order) whose key is `key`; the rarest path: more than SR_LIST items of one
// bucket share one score.  An element per thread and round.
template <int TYPE>
__device__ int32_t nth_of_key(const RowView<TYPE> &view, const uint32_t key, const u64 m, SampleShared &sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid == 0) sh.picked.index = -1;
    u64 seen = 0;
    for (int64_t i0 = 0; i0 < view.M; i0 += SR_THREADS) {
        const int64_t i = i0 + tid;
        const bool hit = i < view.M && rank_key(view.at(i)) == key;
        const u64 mask = __ballot(hit);
        __syncthreads();                                     // the last round's wave sums have been read
        if (lane == 0) sh.wave_c[wave] = __popcll(mask);
        __syncthreads();
        u64 before = seen + __popcll(mask & ((1ull << lane) - 1));
        for (int x = 0; x < SR_WAVES; ++x) {
            if (x < wave) before += sh.wave_c[x];
            seen += sh.wave_c[x];
        }
        if (hit && before == m) sh.picked.index = (int32_t)i;
        if (m < seen) break;                                 // uniform: `seen` is the same in every thread
    }
    __syncthreads();
    return sh.picked.index;
}

// The item, in rank order, at which the running sum of ones (by_count) or of weights passes `target`; the caller has
// made sure that it does.  Every thread returns the same.
template <int TYPE, int NV>
__device__ Picked find(const RowStore<TYPE, NV> &row, const RowScale &c, const bool by_count, const u64 target,
                       SampleShared &sh) {
    const int tid = threadIdx.x;
    pick_bucket(sh.cnt, sh.wsum, by_count, target, 0, 0, sh);
    const uint32_t b = sh.bucket;
    uint32_t n = sh.in_bucket, base_c = sh.base_c;
    u64 base_w = sh.base_w;
    // A bucket with more items than the list holds (many equal scores, or an outlier that stretches the buckets) is cut
    // by its keys' digits, 11, 11 and 10 bits, until its part is short enough or a single key is left.
    int shift = 32;
    uint32_t prefix = 0;
    while (n > SR_LIST && shift > 0) {
        const int next = shift == 32 ? 21 : shift == 21 ? 10 : 0;
        __syncthreads();
        sh.csub[2 * tid] = sh.csub[2 * tid + 1] = 0;
        sh.wsub[2 * tid] = sh.wsub[2 * tid + 1] = 0;
        __syncthreads();
        row.each([&](const float s, const int32_t) {
            if (bucket_of(s, c) != b) return;
            const uint32_t key = rank_key(s);
            if (shift < 32 && (key >> shift) != prefix) return;
            u64 w;
            if (!weigh(s, c, sh.pow2, w)) return;
            const uint32_t d = SR_BUCKETS - 1 - ((key >> next) & (next ? 2047u : 1023u));     // large keys first
            atomicAdd(&sh.csub[d], 1u);
            atomicAdd(&sh.wsub[d], w);
        });
        __syncthreads();
        scan_buckets(sh.csub, sh.wsub, sh);
        pick_bucket(sh.csub, sh.wsub, by_count, target, base_c, base_w, sh);
        const uint32_t digit = SR_BUCKETS - 1 - sh.bucket;
        prefix = shift == 32 ? digit : next ? (prefix << 11 | digit) : (prefix << 10 | digit);
        n = sh.in_bucket; base_c = sh.base_c; base_w = sh.base_w;
        shift = next;
    }
    __syncthreads();
    Picked out;
    if (n > SR_LIST) {                                       // one score, n items
        const float s = __uint_as_float(prefix & 0x80000000u ? prefix & 0x7fffffffu : ~prefix);
        u64 w = 1;
        weigh(s, c, sh.pow2, w);
        const u64 m = by_count ? target - base_c : (target - base_w) / w;
        out.index = nth_of_key<TYPE>(row.view, prefix, m, sh);
        out.before = base_w + m * w;
        out.weight = w;
        __syncthreads();
        return out;
    }
    if (tid == 0) sh.n_list = 0;
    __syncthreads();
    row.each([&](const float s, const int32_t i) {
        if (bucket_of(s, c) != b) return;
        const uint32_t key = rank_key(s);
        if (shift < 32 && (key >> shift) != prefix) return;
        u64 w;
        if (!weigh(s, c, sh.pow2, w)) return;
        const uint32_t at = atomicAdd(&sh.n_list, 1u);
        if (at < SR_LIST) {
            sh.list[at][0] = (u64)key << 32 | (uint32_t)~(uint32_t)i;
            sh.list[at][1] = w;
        }
    });
    __syncthreads();
    if (tid < (int)n) {
        const u64 mine = sh.list[tid][0], w = sh.list[tid][1];
        u64 before = base_w;
        uint32_t rank = base_c;
        for (uint32_t q = 0; q < n; ++q)
            if (sh.list[q][0] > mine) { before += sh.list[q][1]; ++rank; }
        const bool here = by_count ? rank == target : (before <= target && target < before + w);
        if (here) { sh.picked.before = before; sh.picked.weight = w; sh.picked.index = (int32_t)~(uint32_t)mine; }
    }
    __syncthreads();
    out = sh.picked;
    __syncthreads();
    return out;
}

// One workgroup per row.
template <int TYPE, int NV>
__global__ __launch_bounds__(SR_THREADS) void sample_rows_kernel(const SampleArgs a) {
    __shared__ SampleShared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r = blockIdx.x;
    const RowView<TYPE> view(a.scores, r, a.lds, a.M);
    if (a.ex_rowptr) {
        const int64_t er = a.ex_rows ? a.ex_rows[r] : r;
        for (int64_t q = a.ex_rowptr[er] + tid; q < a.ex_rowptr[er + 1]; q += SR_THREADS) {
            const int32_t i = a.ex_col[q];
            if (i >= 0 && i < a.M) RowView<TYPE>::put((char *)view.base, i, -__builtin_inff());
        }
        __syncthreads();
    }
    if (tid < 256) sh.pow2[tid] = exp2((double)tid / 256.0);
    sh.cnt[2 * tid] = sh.cnt[2 * tid + 1] = 0;
    sh.wsum[2 * tid] = sh.wsum[2 * tid + 1] = 0;
    const RowStore<TYPE, NV> row(view);

    // the largest score, and the smallest that is no mask value (it only sets the buckets' width)
    float hi = -__builtin_inff(), lo = __builtin_inff();
    row.each([&](const float s, const int32_t) {
        hi = fmaxf(hi, s);
        lo = s > -1e30f ? fminf(lo, s) : lo;
    });
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) { hi = fmaxf(hi, __shfl_xor(hi, o)); lo = fminf(lo, __shfl_xor(lo, o)); }
    if (lane == 0) { sh.wave_f[wave] = hi; sh.wave_g[wave] = lo; }
    __syncthreads();
    for (int v = 0; v < SR_WAVES; ++v) { hi = fmaxf(hi, sh.wave_f[v]); lo = fminf(lo, sh.wave_g[v]); }

    const float T = a.o.temperature_rows ? a.o.temperature_rows[r] : a.o.temperature;
    const int32_t top_k = a.o.top_k_rows ? a.o.top_k_rows[r] : a.o.top_k;
    const float top_p = a.o.top_p_rows ? a.o.top_p_rows[r] : a.o.top_p;
    const float min_p = a.o.min_p_rows ? a.o.min_p_rows[r] : a.o.min_p;
    int32_t *idx = a.idx + r * a.n_draws;
    float *logp = a.logp + r * a.n_draws;
    if (hi == -__builtin_inff()) {                            // nothing to draw from
        for (int d = tid; d < a.n_draws; d += SR_THREADS) { idx[d] = -1; logp[d] = -__builtin_inff(); }
        return;
    }
    if (!(T > 0.f)) {                                         // the best item: lowest column of the largest score
        if (tid == 0) sh.base_w = ~0ull;
        __syncthreads();
        row.each([&](const float s, const int32_t i) { if (s == hi) atomicMin(&sh.base_w, (u64)i); });
        __syncthreads();
        for (int d = tid; d < a.n_draws; d += SR_THREADS) { idx[d] = (int32_t)sh.base_w; logp[d] = 0.f; }
        return;
    }
    RowScale c;
    c.top = hi;
    c.inv_t = 1.0 / (double)T;
    c.q_bits = a.q_bits;
    c.min_p = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;
    c.cut = 0.6931471805599453 * (a.q_bits + 1);              // beyond it a weight rounds to 0
    {
        // buckets span the scores that can matter: down to the lowest, the cut, or min-p's threshold
        double span = c.cut;
        if (c.min_p > 0.f) span = fmin(span, -log((double)c.min_p) + 1e-6);
        const float width = fminf((float)fmin(span * (double)T, 3e38), hi - lo);
        c.per_score = (float)SR_BUCKETS / fmaxf(width, 1e-30f);
    }
    row.each([&](const float s, const int32_t) {
        u64 w;
        if (!weigh(s, c, sh.pow2, w)) return;
        const uint32_t b = bucket_of(s, c);
        atomicAdd(&sh.cnt[b], 1u);
        atomicAdd(&sh.wsum[b], w);
    });
    __syncthreads();
    scan_buckets(sh.cnt, sh.wsum, sh);
    const uint32_t n = sh.cnt[SR_BUCKETS - 1];
    u64 W = sh.wsum[SR_BUCKETS - 1];
    if (top_k > 0 && (uint32_t)top_k < n) {
        const Picked p = find<TYPE, NV>(row, c, true, (u64)top_k - 1, sh);
        W = p.before + p.weight;
    }
    if (top_p < 1.f) {
        const double want = ceil((double)fmaxf(top_p, 0.f) * (double)W);
        const u64 need = want < 1.0 ? 1 : (u64)want;
        const Picked p = find<TYPE, NV>(row, c, false, (need < W ? need : W) - 1, sh);
        W = p.before + p.weight;
    }
    for (int d = 0; d < a.n_draws; ++d) {
        const int64_t at = r * a.n_draws + d;
        const double u = a.u_f64 ? ((const double *)a.u)[at] : (double)((const float *)a.u)[at];
        const double t = u > 0.0 ? fmin(u, 1.0) * (double)W : 0.0;
        const u64 target = t >= (double)W ? W - 1 : (u64)t;
        const Picked p = find<TYPE, NV>(row, c, false, target < W ? target : W - 1, sh);
        if (tid == 0) { idx[d] = p.index; logp[d] = (float)log((double)p.weight / (double)W); }
    }
}

}  // namespace

extern "C" {

int32_t als_sample_rows(void *scores, int32_t dtype, int64_t lds, int64_t n_rows, int64_t M, const int64_t *ex_rowptr,
                        const int32_t *ex_col, const int64_t *ex_row_ids, const als_sample_opts_t *opts, const void *u,
                        int32_t u_is_f64, int32_t n_draws, int32_t *idx_out, float *logp_out, void *stream) {
    if (!scores || !opts || !u || !idx_out || !logp_out) return als_fail_(ALS_ERR_INVALID_ARG, "als_sample_rows: null pointer");
    if (n_rows < 1 || M < 1 || lds < M || M > INT32_MAX || n_draws < 1)
        return als_fail_(ALS_ERR_INVALID_ARG, "als_sample_rows: bad sizes (n_rows=%lld M=%lld lds=%lld n_draws=%d)", (long long)n_rows,
                         (long long)M, (long long)lds, n_draws);
    if (n_rows > INT32_MAX) return als_fail_(ALS_ERR_UNSUPPORTED, "als_sample_rows: more than 2^31 - 1 rows per call");
    if (dtype < ALS_DTYPE_F32 || dtype > ALS_DTYPE_BF16)
        return als_fail_(ALS_ERR_UNSUPPORTED, "als_sample_rows: dtype %d (0 float32, 1 float16, 2 bfloat16)", dtype);
    if ((uintptr_t)scores % (dtype == ALS_DTYPE_F32 ? 4 : 2))
        return als_fail_(ALS_ERR_INVALID_ARG, "als_sample_rows: scores are not aligned to their type");
    if ((ex_rowptr == nullptr) != (ex_col == nullptr))
        return als_fail_(ALS_ERR_INVALID_ARG, "als_sample_rows: pass both exclusion arrays or neither");
    SampleArgs a;
    a.scores = scores; a.lds = lds; a.M = M;
    a.ex_rowptr = ex_rowptr; a.ex_col = ex_col; a.ex_rows = ex_rowptr ? ex_row_ids : nullptr;
    a.o = *opts;
    a.u = u; a.u_f64 = u_is_f64 != 0; a.n_draws = n_draws;
    int bits = 0;
    while ((1LL << bits) < M) ++bits;
    a.q_bits = std::min(51, 62 - bits);
    a.idx = idx_out; a.logp = logp_out;
    const dim3 grid((unsigned)n_rows), block(SR_THREADS);
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case ALS_DTYPE_F32: hipLaunchKernelGGL((sample_rows_kernel<ROW_F32, 0>), grid, block, 0, st, a); break;
        case ALS_DTYPE_F16: hipLaunchKernelGGL((sample_rows_kernel<ROW_F16, 0>), grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL((sample_rows_kernel<ROW_BF16, 0>), grid, block, 0, st, a); break;
    }
    ALS_HIP_CHECK4(hipGetLastError());
    return ALS_OK;
}

}  // extern "C"

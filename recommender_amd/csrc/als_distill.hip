// Following a teacher's ranked list: the loss of a softmax over all items against the list's, and its gradient.
//
// For one row of M student scores s, a list of up to 1024 teacher items j with scores z_j, and a temperature T:
//     t_j = exp(z_j / T) / sum over the list            (the teacher, on its list)
//     q_i = exp(s_i / T) / sum over all M items         (the student)
//     loss = sum_j t_j (ln t_j - ln q_j),      d loss / d s_i = (q_i - t_i) / T      (t_i = 0 off the list)
// The gradient leaves multiplied by the row's weight.
//
// als_distill_rows works on score rows and is bound by memory: a row is read once, kept in registers over its three
// passes (maximum, sum, gradient) and its gradient written once.  1024 threads hold 65 536 float32 or 131 072 16-bit items;
// longer rows are cut into parts of half that and take two launches, the second of which reads them again.  Whole calls on one
// MI355X: 4096 x 59047 float32 398 us = 4.9 TB/s, what a copy of them takes; 2048 x 59047 bfloat16 119 us = 4.1 TB/s (a copy
// 101: the exponentials of 16-bit rows cost twice as much per byte, two workgroups per compute unit hide most of it, and at the
// 64 registers that takes 7 to 9 of them spill, 32 to 40 bytes of scratch a lane);
// 61 x 1000003 float32 124 us where one read and one write take 102.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "als_hip.h"

int als_fail_(int code, const char *fmt, ...);  // defined in als_kernels.hip

#define ALS_HIP_CHECK5(expr)                                                                      \
    do {                                                                                          \
        hipError_t e_ = (expr);                                                                   \
        if (e_ != hipSuccess) return als_fail_(ALS_ERR_HIP, "%s: %s", #expr, hipGetErrorString(e_)); \
    } while (0)

namespace {

#include "als_rows.inc"

constexpr int DR_THREADS = 1024;
constexpr int DR_WAVES = DR_THREADS / 64;
constexpr int LIST_MAX = 1024;              // one list entry per thread
constexpr int HASH_SLOTS = 2048;

__device__ __forceinline__ float exp2_fast(const float x) { return __builtin_amdgcn_exp2f(x); }     // 1 ulp, subnormals to 0

struct RowsArgs {
    const void *scores;
    int64_t lds, n, M;
    const int32_t *t_idx;
    const float *t_val;
    int64_t ldt;
    int32_t k;
    float inv_t;
    const float *weight;
    float *loss;
    void *grad;
    int64_t ldg;
};

struct ListShared {
    int32_t key[HASH_SLOTS], first[HASH_SLOTS];
    double red[DR_WAVES];
    float redf[DR_WAVES];
};

// Reductions over the workgroup: per wave by shuffles, the 16 waves' values by the shuffles of every wave's first 16 lanes.
__device__ __forceinline__ float block_max(float v, ListShared &sh) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    __syncthreads();
    if (lane == 0) sh.redf[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh.redf[lane & (DR_WAVES - 1)];
#pragma unroll
    for (int o = DR_WAVES / 2; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ double block_sum(double v, ListShared &sh) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if (lane == 0) sh.red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh.red[lane & (DR_WAVES - 1)];
#pragma unroll
    for (int o = DR_WAVES / 2; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// Thread p < k: entry p of the row's list.  An entry outside [0, M) is padding; of an item listed twice the first entry
// stands (a hash table in LDS holds every item's lowest position, set by integer atomics: the same whatever the timing).
// item: the thread's item or -1.  t: its share of the teacher's softmax.  A list without weight is empty.
__device__ void teacher_entry(const RowsArgs &a, const int64_t r, ListShared &sh, int32_t &item, float &t) {
    const int tid = threadIdx.x;
    for (int q = tid; q < HASH_SLOTS; q += DR_THREADS) { sh.key[q] = -1; sh.first[q] = LIST_MAX; }
    item = -1;
    float z = 0.f;
    if (tid < a.k) {
        item = a.t_idx[r * a.ldt + tid];
        if (item < 0 || item >= a.M) item = -1;
        else z = a.t_val[r * a.ldt + tid];
    }
    __syncthreads();
    uint32_t slot = 0;
    if (item >= 0) {
        slot = ((uint32_t)item * 2654435761u) >> 21;
        for (;;) {                              // at most 1024 of the 2048 slots are ever taken
            const int32_t was = atomicCAS(&sh.key[slot], -1, item);
            if (was == -1 || was == item) break;
            slot = (slot + 1) & (HASH_SLOTS - 1);
        }
        atomicMin(&sh.first[slot], tid);
    }
    __syncthreads();
    if (item >= 0 && sh.first[slot] != tid) item = -1;
    // a NaN counts as the largest: the list is not an empty one, and its sum and shares become NaN
    const float top = block_max(item < 0 ? -__builtin_inff() : z == z ? z : __builtin_inff(), sh);
    float e = 0.f;
    if (item >= 0 && top != -__builtin_inff()) e = expf((z - top) * a.inv_t);
    const double sum = block_sum((double)e, sh);
    if (top == -__builtin_inff()) item = -1;
    t = item >= 0 ? (float)((double)e / sum) : 0.f;
}

// One term of the loss: ln t - ln q with ln q = (s - top) / T - ln Z (float32 logarithms: float64's would cost the kernels
// the registers of a second resident workgroup)
__device__ __forceinline__ float loss_term(const float t, const float s, const float top, const float log_z, const float inv_t) {
    if (s == -__builtin_inff()) return t == 0.f ? 0.f : t * __builtin_inff();       // also where the whole row is masked, Z = 0
    return t == 0.f ? 0.f : t * (logf(t) - ((s - top) * inv_t - log_z));            // a NaN share stays one
}

// Chunk q of the gradient row.  Its address has the alignment of the type only where scores and gradient lie differently.
// STREAM: past the caches, which keep the scores instead.
struct __attribute__((packed, aligned(2))) Chunk16 { row_u32x4 v; };
typedef unsigned loose_u32x4 __attribute__((ext_vector_type(4), aligned(2)));
template <int TYPE, bool STREAM>
__device__ __forceinline__ void put_chunk(char *out, const RowView<TYPE> &view, const int32_t q, const float (&g)[8]) {
    Chunk16 c;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (TYPE == ROW_F32) c.v[e] = __float_as_uint(g[e]);
        else c.v[e] = RowView<TYPE>::narrow(g[2 * e]) | RowView<TYPE>::narrow(g[2 * e + 1]) << 16;
    }
    char *at = out + (int64_t)view.index0(q) * RowView<TYPE>::BYTES;
    if constexpr (STREAM) __builtin_nontemporal_store((loose_u32x4)c.v, reinterpret_cast<loose_u32x4 *>(at));
    else *reinterpret_cast<Chunk16 *>(at) = c;
}

// A part of a row - NV chunks per thread from chunk q0 on, in registers - and this thread's element outside the body.
template <int TYPE, int NV>
struct RowPart {
    static constexpr int VEC = RowView<TYPE>::VEC;
    row_u32x4 held[NV];
    float extra;
    int32_t extra_at;
    __device__ __forceinline__ void load(const RowView<TYPE> &view, const int32_t q0, const bool with_extra) {
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            const int32_t at = q0 + q * DR_THREADS + threadIdx.x;
            held[q] = RowView<TYPE>::nothing();
            if (at < view.n_chunks) held[q] = view.load(at);
        }
        extra_at = with_extra ? view.extra(threadIdx.x) : -1;
        extra = extra_at >= 0 ? view.at(extra_at) : -__builtin_inff();
    }
    // The raw words are what stays in registers: made opaque between the passes, so that the compiler decodes them again
    // instead of keeping every decoded value (twice the registers for 16-bit rows, and spills).
    __device__ __forceinline__ void pin() {
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                unsigned w = held[q][e];
                asm volatile("" : "+v"(w));
                held[q][e] = w;
            }
    }
    __device__ __forceinline__ float top() {
        pin();
        float t = extra;
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
            for (int e = 0; e < VEC; ++e) t = fmaxf(t, RowView<TYPE>::value(held[q], e));
        return t;
    }
    // sum of exp((s - m) / T): float32 within a chunk, float64 above
    __device__ __forceinline__ double sum(const float m, const float c2) {
        pin();
        double z = (double)exp2_fast((extra - m) * c2);
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            float part = 0.f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) part += exp2_fast((RowView<TYPE>::value(held[q], e) - m) * c2);
            z += (double)part;
            __builtin_amdgcn_sched_barrier(0);          // a chunk at a time: unrolled together they spill more (NV = 8 spills 7 to 9 even so)
        }
        return z;
    }
    template <bool STREAM>
    __device__ __forceinline__ void put_slopes(char *out, const RowView<TYPE> &view, const int32_t q0, const float m, const float c2,
                                               const float cq, const bool any) {
        pin();
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            const int32_t at = q0 + q * DR_THREADS + threadIdx.x;
            if (at < view.n_chunks) {
                float g[8];
#pragma unroll
                for (int e = 0; e < VEC; ++e) g[e] = any ? cq * exp2_fast((RowView<TYPE>::value(held[q], e) - m) * c2) : 0.f;
                put_chunk<TYPE, STREAM>(out, view, at, g);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (extra_at >= 0) RowView<TYPE>::put(out, extra_at, any ? cq * exp2_fast((extra - m) * c2) : 0.f);
    }
};

// What a row's gradient needs of its sums.
struct RowScale {
    float cq, scale, inv_z;
    bool any;
};
__device__ __forceinline__ RowScale row_scale(const RowsArgs &a, const int64_t r, const double z, const bool any) {
    RowScale c;
    c.any = any;                             // a list without entries asks for nothing: loss and gradient 0
    c.scale = any ? (a.weight ? a.weight[r] : 1.f) * a.inv_t : 0.f;
    c.inv_z = z > 0.0 ? (float)(1.0 / z) : z == z ? 0.f : (float)z;
    c.cq = c.scale * c.inv_z;
    return c;
}

// One workgroup per row, the row in registers: read once, written once.
template <int TYPE, int NV>
__global__ __launch_bounds__(DR_THREADS, NV <= 8 ? 8 : 4) void distill_rows_kernel(const RowsArgs a) {
    __shared__ ListShared sh;
    const int64_t r = row_of_block();
    if (r >= a.n) return;
    const RowView<TYPE> view(a.scores, r, a.lds, a.M);
    RowPart<TYPE, NV> part;
    part.load(view, 0, true);
    int32_t item;
    float t;
    teacher_entry(a, r, sh, item, t);
    const float s_item = item >= 0 ? view.at(item) : 0.f;      // before the gradient may overwrite it
    const float c2 = a.inv_t * 1.44269504f;
    const float hi = block_max(part.top(), sh), top = hi == -__builtin_inff() ? 0.f : hi;
    const double z = block_sum(part.sum(top, c2), sh);
    const double loss = block_sum(item >= 0 ? (double)loss_term(t, s_item, top, logf((float)z), a.inv_t) : 0.0, sh);
    const RowScale c = row_scale(a, r, z, block_max(item >= 0 ? 1.f : 0.f, sh) > 0.f);
    if (threadIdx.x == 0) a.loss[r] = c.any ? (float)loss : 0.f;
    char *out = (char *)a.grad + r * a.ldg * RowView<TYPE>::BYTES;
    part.template put_slopes<false>(out, view, 0, top, c2, c.cq, c.any);
    __syncthreads();
    if (item >= 0) RowView<TYPE>::put(out, item, c.scale * (exp2_fast((s_item - top) * c2) * c.inv_z - t));
}

// Rows that one workgroup does not hold, in two launches of n_parts workgroups per row: the first leaves each part's
// maximum and sum and the scores of the listed items, the second joins them and writes the gradient.
struct PartStat { double z; float top; float pad; };
constexpr int DR_PART_NV = 8;
template <int TYPE>
__global__ __launch_bounds__(DR_THREADS, 8) void distill_parts_kernel(const RowsArgs a, const int n_parts, PartStat *__restrict__ stats,
                                                                   float *__restrict__ listed) {
    __shared__ ListShared sh;
    const int64_t r = blockIdx.x / n_parts;
    const int part_no = blockIdx.x % n_parts;
    const RowView<TYPE> view(a.scores, r, a.lds, a.M);
    RowPart<TYPE, DR_PART_NV> part;
    part.load(view, part_no * DR_PART_NV * DR_THREADS, part_no == 0);
    if (part_no == 0 && (int)threadIdx.x < a.k) {
        const int32_t item = a.t_idx[r * a.ldt + threadIdx.x];
        listed[r * a.k + threadIdx.x] = item >= 0 && item < a.M ? view.at(item) : 0.f;
    }
    const float hi = block_max(part.top(), sh), top = hi == -__builtin_inff() ? 0.f : hi;
    const double z = block_sum(part.sum(top, a.inv_t * 1.44269504f), sh);
    if (threadIdx.x == 0) stats[blockIdx.x] = PartStat{z, hi, 0.f};
}
template <int TYPE>
__global__ __launch_bounds__(DR_THREADS, 8) void distill_slopes_kernel(const RowsArgs a, const int n_parts,
                                                                    const PartStat *__restrict__ stats,
                                                                    const float *__restrict__ listed) {
    __shared__ ListShared sh;
    // Backwards, and the gradient past the caches: what the launch before read last may be in the last-level cache still
    // (61 x 1000003 float32: 124 us, 150 without the second, 153 without either; in the form of one launch, which reads
    // nothing twice, streaming stores cost float32 rows 3 %).
    const unsigned w = gridDim.x - 1 - blockIdx.x;
    const int64_t r = w / n_parts;
    const int part_no = w % n_parts;
    const RowView<TYPE> view(a.scores, r, a.lds, a.M);
    RowPart<TYPE, DR_PART_NV> part;
    const int32_t q0 = part_no * DR_PART_NV * DR_THREADS;
    int32_t item;
    float t;
    teacher_entry(a, r, sh, item, t);
    const float s_item = item >= 0 ? listed[r * a.k + threadIdx.x] : 0.f;
    const float c2 = a.inv_t * 1.44269504f;
    float hi = -__builtin_inff();
    for (int p = threadIdx.x; p < n_parts; p += DR_THREADS) hi = fmaxf(hi, stats[r * n_parts + p].top);
    hi = block_max(hi, sh);
    const float top = hi == -__builtin_inff() ? 0.f : hi;
    double z = 0.0;
    for (int p = threadIdx.x; p < n_parts; p += DR_THREADS) {
        // a part of nothing but -inf has no weight: its stand-in maximum 0 may lie any distance above the row's (0 x inf)
        const PartStat s = stats[r * n_parts + p];
        if (s.z != 0.0) z += s.z * (double)exp2_fast(((s.top == -__builtin_inff() ? 0.f : s.top) - top) * c2);
    }
    z = block_sum(z, sh);
    const RowScale c = row_scale(a, r, z, block_max(item >= 0 ? 1.f : 0.f, sh) > 0.f);
    if (part_no == 0) {
        const double loss = block_sum(item >= 0 ? (double)loss_term(t, s_item, top, logf((float)z), a.inv_t) : 0.0, sh);
        if (threadIdx.x == 0) a.loss[r] = c.any ? (float)loss : 0.f;
    }
    char *out = (char *)a.grad + r * a.ldg * RowView<TYPE>::BYTES;
    part.load(view, q0, part_no == 0);          // not earlier: two workgroups per unit overlap, and their registers do not spill
    part.template put_slopes<true>(out, view, q0, top, c2, c.cq, c.any);
    __syncthreads();
    // the listed items of this part
    if (item >= 0) {
        const int32_t q = (item - view.head) / RowView<TYPE>::VEC;
        const bool body = item >= view.head && q < view.n_chunks;
        if (body ? q / (DR_PART_NV * DR_THREADS) == part_no : part_no == 0)
            RowView<TYPE>::put(out, item, c.scale * (exp2_fast((s_item - top) * c2) * c.inv_z - t));
    }
}

int64_t row_parts(const int32_t dtype, const int64_t M) {
    const int64_t vec = dtype == ALS_DTYPE_F32 ? 4 : 8;
    return (M / vec + DR_PART_NV * DR_THREADS - 1) / (DR_PART_NV * DR_THREADS);
}

template <int TYPE>
void launch_rows(const RowsArgs &a, const int64_t n, void *ws, hipStream_t st) {
    const int64_t chunks = a.M / RowView<TYPE>::VEC;
    const dim3 block(DR_THREADS);
    if (chunks <= 4 * DR_THREADS) hipLaunchKernelGGL((distill_rows_kernel<TYPE, 4>), grid_of_rows(n), block, 0, st, a);
    else if (chunks <= 8 * DR_THREADS) hipLaunchKernelGGL((distill_rows_kernel<TYPE, 8>), grid_of_rows(n), block, 0, st, a);
    else if (chunks <= 16 * DR_THREADS) hipLaunchKernelGGL((distill_rows_kernel<TYPE, 16>), grid_of_rows(n), block, 0, st, a);
    else {
        const int parts = (int)row_parts(TYPE, a.M);
        PartStat *stats = (PartStat *)ws;
        float *listed = (float *)(stats + n * parts);
        hipLaunchKernelGGL((distill_parts_kernel<TYPE>), dim3((unsigned)(n * parts)), block, 0, st, a, parts, stats, listed);
        hipLaunchKernelGGL((distill_slopes_kernel<TYPE>), dim3((unsigned)(n * parts)), block, 0, st, a, parts, stats, listed);
    }
}

}  // namespace

extern "C" {

size_t als_distill_rows_workspace_bytes(int32_t dtype, int64_t n_rows, int64_t M, int32_t k) {
    if (dtype < ALS_DTYPE_F32 || dtype > ALS_DTYPE_BF16 || n_rows < 1 || M < 1 || M > ROW_MAX || k < 1 || k > LIST_MAX) return 0;
    const int64_t chunks = M / (dtype == ALS_DTYPE_F32 ? 4 : 8);
    if (chunks <= 16 * DR_THREADS) return 0;                  // held by one workgroup: nothing is kept between launches
    return (size_t)n_rows * ((size_t)row_parts(dtype, M) * sizeof(PartStat) + (size_t)k * 4) + 16;
}

int32_t als_distill_rows(const void *scores, int32_t dtype, int64_t lds, int64_t n_rows, int64_t M, const int32_t *teacher_idx,
                         const float *teacher_val, int64_t ld_teacher, int32_t k, float temperature, const float *weight,
                         float *loss_out, void *grad_out, int64_t ldg, void *workspace, size_t ws_bytes, void *stream) {
    if (!scores || !teacher_idx || !teacher_val || !loss_out || !grad_out)
        return als_fail_(ALS_ERR_INVALID_ARG, "als_distill_rows: null pointer");
    if (n_rows < 1 || M < 1 || lds < M || ldg < M || M > ROW_MAX || n_rows > INT32_MAX || ld_teacher < k)
        return als_fail_(ALS_ERR_INVALID_ARG, "als_distill_rows: bad sizes (n_rows=%lld M=%lld lds=%lld ldg=%lld)", (long long)n_rows,
                         (long long)M, (long long)lds, (long long)ldg);
    if (k < 1 || k > LIST_MAX) return als_fail_(ALS_ERR_UNSUPPORTED, "als_distill_rows: k=%d outside [1, %d]", k, LIST_MAX);
    if (dtype < ALS_DTYPE_F32 || dtype > ALS_DTYPE_BF16)
        return als_fail_(ALS_ERR_UNSUPPORTED, "als_distill_rows: dtype %d (0 float32, 1 float16, 2 bfloat16)", dtype);
    if (((uintptr_t)scores | (uintptr_t)grad_out) % (dtype == ALS_DTYPE_F32 ? 4 : 2))
        return als_fail_(ALS_ERR_INVALID_ARG, "als_distill_rows: scores or gradient are not aligned to their type");
    if (!(temperature >= 1e-30f && temperature <= 1e30f))     // 1 / T and its product with log2(e) are ordinary numbers
        return als_fail_(ALS_ERR_INVALID_ARG, "als_distill_rows: temperature %g outside [1e-30, 1e30]", (double)temperature);
    const size_t need = als_distill_rows_workspace_bytes(dtype, n_rows, M, k);
    if (need && (!workspace || ws_bytes < need || (uintptr_t)workspace % 8))
        return als_fail_(ALS_ERR_WORKSPACE, "als_distill_rows: workspace too small or not 8-byte aligned: %zu < %zu", ws_bytes, need);
    if (need && n_rows * row_parts(dtype, M) > GRID_X)
        return als_fail_(ALS_ERR_UNSUPPORTED, "als_distill_rows: too many rows of this length for one launch");
    RowsArgs a;
    a.scores = scores; a.lds = lds; a.n = n_rows; a.M = M; a.t_idx = teacher_idx; a.t_val = teacher_val; a.ldt = ld_teacher; a.k = k;
    a.inv_t = 1.f / temperature; a.weight = weight; a.loss = loss_out; a.grad = grad_out; a.ldg = ldg;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ALS_DTYPE_F32) launch_rows<ROW_F32>(a, n_rows, workspace, st);
    else if (dtype == ALS_DTYPE_F16) launch_rows<ROW_F16>(a, n_rows, workspace, st);
    else launch_rows<ROW_BF16>(a, n_rows, workspace, st);
    ALS_HIP_CHECK5(hipGetLastError());
    return ALS_OK;
}

}  // extern "C"

// Plans of ragged attention batches, and the selection of key blocks by a
// cheap score.
//
//   s3dsp_attn_plan_create  cuts every sequence into query blocks of 128 rows and key blocks of 64
//   s3dsp_block_select      per (query block, head): the key blocks of its sequence with the
//                           largest <mean of the block's q rows, mean of the key block's k rows>
//
// A selection is whole numbers: two scores that differ by less than f32
// rounding would swap blocks between two ways of adding the same rows, so the
// sums, means and scores are f64 (exact sums of 16-bit rows, in practice). The
// f64 work is 1 / (128 * 64) of the attention it steers.
//
//   block_mean_kernel   one pass over q and k (memory bound): a warp lane owns eight columns, eight
//                       warps share the block's rows, f64 sums joined in warp order
//   block_score_kernel  one CTA per (up to kGroup query blocks of a sequence, head): scores into shared
//                       memory, then one warp per row finds the top-th largest key by bisection over
//                       the ordered bits and writes the chosen indices in ascending order
#include "s3dsp_internal.h"

using namespace s3dsp;

namespace {

constexpr int kMeanThreads = 256;
constexpr int kMeanCols = 256;  // columns per CTA of the mean kernel: 32 lanes x 8
constexpr int kScoreThreads = 256;
constexpr int kGroup = kAttnGroupRows;  // most query blocks per CTA of the score kernel

template <typename T>
__device__ __forceinline__ double to_d(T v);
template <>
__device__ __forceinline__ double to_d<float>(float v) {
    return (double)v;
}
template <>
__device__ __forceinline__ double to_d<__nv_bfloat16>(__nv_bfloat16 v) {
    return (double)__bfloat162float(v);
}
template <>
__device__ __forceinline__ double to_d<__half>(__half v) {
    return (double)__half2float(v);
}

struct MeanParams {
    const void* q;
    const void* k;
    int64_t qs, ks;  // row strides in elements
    int qw, kw;      // columns: heads * d, kv_heads * d
    int n_qb, n_kb;
    const int4* q_blocks;
    const int2* k_blocks;
    double* q_mean;   // [n_qb][qw]
    double* k_mean;   // [kw][n_kb]: a score CTA's threads read neighbouring blocks
};

template <typename T, bool kVec>
__global__ void __launch_bounds__(kMeanThreads) block_mean_kernel(MeanParams p) {
    __shared__ double part[8][kMeanCols];
    pdl_wait();
    pdl_trigger();
    const bool is_k = (int)blockIdx.x >= p.n_qb;
    const int b = is_k ? blockIdx.x - p.n_qb : blockIdx.x;
    const int width = is_k ? p.kw : p.qw;
    const int c0 = blockIdx.y * kMeanCols;
    if (c0 >= width) return;
    int64_t row0;
    int rows;
    if (is_k) {
        const int2 kb = p.k_blocks[b];
        row0 = kb.x, rows = kb.y;
    } else {
        const int4 qb = p.q_blocks[b];
        row0 = qb.x, rows = qb.y & kAttnRowsMask;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c = c0 + 8 * lane;
    const int64_t ld = is_k ? p.ks : p.qs;
    const T* base = static_cast<const T*>(is_k ? p.k : p.q) + row0 * ld + c;
    double acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = 0.0;
    if (c < width) {  // widths are multiples of 8
#pragma unroll 4
        for (int r = warp; r < rows; r += 8) {
            const T* x = base + r * ld;
            T e[8];
            if constexpr (kVec) {
                constexpr int kW = sizeof(T) * 8 / 16;
#pragma unroll
                for (int w = 0; w < kW; ++w)
                    reinterpret_cast<uint4*>(e)[w] = __ldg(reinterpret_cast<const uint4*>(x) + w);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = x[j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] += to_d(e[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) part[warp][8 * lane + j] = acc[j];
    __syncthreads();
    const int col = c0 + threadIdx.x;
    if (col >= width) return;
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += part[w][threadIdx.x];
    s /= rows;
    if (is_k)
        p.k_mean[(int64_t)col * p.n_kb + b] = s;
    else
        p.q_mean[(int64_t)b * p.qw + col] = s;
}

struct ScoreParams {
    const int2* groups;     // {first query block, blocks}: one sequence's
    const int4* q_blocks;   // {first row, rows | index in the sequence << 8, first key row, key rows}
    const int* first_kb;    // [n_qb] first key block of the block's sequence
    const double* q_mean;
    const double* k_mean;
    int qw, n_kb, d, heads, per_kv, top, keep_local;
    int max_kb;             // row length of the score table
    int32_t* sel;           // [n_qb][heads][top]
};

// f64 -> u64 whose unsigned order is the scores' order; NaN lowest
__device__ __forceinline__ unsigned long long ordered(double v) {
    if (v != v) return 0ull;
    const long long b = __double_as_longlong(v + 0.0);  // -0 and 0 are one score
    return b < 0 ? ~(unsigned long long)b : (unsigned long long)b | 0x8000000000000000ull;
}

__global__ void __launch_bounds__(kScoreThreads) block_score_kernel(ScoreParams p) {
    extern __shared__ double sm[];
    double* qm = sm;                                  // [d][kGroup]
    double* score = sm + (size_t)p.d * kGroup;        // [count][max_kb] as ordered keys
    pdl_wait();
    pdl_trigger();
    const int2 grp = p.groups[blockIdx.x];
    const int h = blockIdx.y;
    const int b0 = grp.x, count = grp.y;
    const int4 qb0 = p.q_blocks[b0];
    const int nkb = (qb0.w + kAttnKRows - 1) / kAttnKRows;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (nkb > p.top) {
        for (int e = threadIdx.x; e < p.d * kGroup; e += kScoreThreads) {
            const int r = e / p.d, j = e - r * p.d;
            qm[j * kGroup + r] = r < count ? p.q_mean[(int64_t)(b0 + r) * p.qw + h * p.d + j] : 0.0;
        }
        __syncthreads();
        const double* km = p.k_mean + (int64_t)(h / p.per_kv) * p.d * p.n_kb + p.first_kb[b0];
        for (int c = threadIdx.x; c < nkb; c += kScoreThreads) {
            double acc[kGroup];
#pragma unroll
            for (int r = 0; r < kGroup; ++r) acc[r] = 0.0;
#pragma unroll 4
            for (int j = 0; j < p.d; ++j) {
                const double kv = km[(int64_t)j * p.n_kb + c];
#pragma unroll
                for (int r = 0; r < kGroup; ++r) acc[r] = fma(qm[j * kGroup + r], kv, acc[r]);
            }
#pragma unroll
            for (int r = 0; r < kGroup; ++r)
                if (r < count) {
                    unsigned long long key = ordered(acc[r]);
                    if (p.keep_local) {
                        // the key blocks of the query block's own rows come first
                        const int own = ((qb0.y >> kAttnRowsBits) + r) * (kAttnQRows / kAttnKRows);
                        if (c >= own && c < own + kAttnQRows / kAttnKRows) key = ~0ull;
                    }
                    reinterpret_cast<unsigned long long*>(score)[(size_t)r * p.max_kb + c] = key;
                }
        }
        __syncthreads();
    }
    for (int r = warp; r < count; r += kScoreThreads / 32) {
        int32_t* out = p.sel + ((int64_t)(b0 + r) * p.heads + h) * p.top;
        if (nkb <= p.top) {  // all of them
            for (int i = lane; i < p.top; i += 32) out[i] = i < nkb ? i : -1;
            continue;
        }
        const unsigned long long* key = reinterpret_cast<unsigned long long*>(score) + (size_t)r * p.max_kb;
        // the largest t with at least `top` keys >= t, bit by bit from the top
        unsigned long long t = 0ull;
        for (int bit = 63; bit >= 0; --bit) {
            const unsigned long long cand = t | (1ull << bit);
            int m = 0;
            for (int c = lane; c < nkb; c += 32) m += key[c] >= cand;
            m = __reduce_add_sync(0xffffffffu, m);
            if (m >= p.top) {
                t = cand;
                if (m == p.top) break;
            }
        }
        int above = 0;
        for (int c = lane; c < nkb; c += 32) above += key[c] > t;
        above = __reduce_add_sync(0xffffffffu, above);
        // every key above t, and the first of those equal to it, in index order;
        // when exactly `top` keys are >= t the equal ones all fit
        int ties = p.top - above, done = 0;
        for (int c0 = 0; c0 < nkb && done < p.top; c0 += 32) {
            const int c = c0 + lane;
            const unsigned long long kc = c < nkb ? key[c] : 0ull;
            const bool gt = c < nkb && kc > t, eq = c < nkb && kc == t;
            const unsigned em = __ballot_sync(0xffffffffu, eq), lt = (1u << lane) - 1u;
            const bool take = gt || (eq && __popc(em & lt) < ties);
            const unsigned tm = __ballot_sync(0xffffffffu, take);
            if (take) out[done + __popc(tm & lt)] = c;
            done += __popc(tm);
            ties -= min(ties, __popc(em));
        }
    }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool check_offsets(const int64_t* off, int64_t n_seq, int64_t* rows, int64_t* blocks, int64_t block_rows) {
    if (off[0] < 0) return false;
    *blocks = 0;
    for (int64_t s = 0; s < n_seq; ++s) {
        if (off[s + 1] < off[s]) return false;
        *blocks += ceil_div(off[s + 1] - off[s], block_rows);
    }
    *rows = off[n_seq];
    return off[n_seq] <= (1ll << 31) - 256;
}

}  // namespace

extern "C" S3DSP_API s3d_status s3dsp_attn_plan_create(s3dsp_context* ctx, const int64_t* h_q_offsets,
                                                       const int64_t* h_k_offsets, int64_t n_seq,
                                                       s3dsp_attn_plan** out, char* error, uint64_t error_capacity) {
    clear_error(error, error_capacity);
    if (!ctx || !h_q_offsets || !out) return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "NULL argument");
    *out = nullptr;
    if (n_seq < 0 || n_seq > (1 << 24)) return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "bad sequence count");
    const bool self = !h_k_offsets;
    const int64_t* ko = self ? h_q_offsets : h_k_offsets;
    int64_t nq, nk, nqb, nkb;
    if (!check_offsets(h_q_offsets, n_seq, &nq, &nqb, kAttnQRows) || !check_offsets(ko, n_seq, &nk, &nkb, kAttnKRows))
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT,
                    "offsets must start at 0 or later, never fall, and end below 2^31 - 255");
    S3DSP_CUDA(cudaSetDevice(ctx->device), "cudaSetDevice");
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    S3DSP_CUDA(cudaStreamIsCapturing(ctx->stream, &cap), "cudaStreamIsCapturing");
    if (cap != cudaStreamCaptureStatusNone)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT,
                    "a plan is made from host memory: make it before the stream capture");
    int64_t max_kb = 0;
    for (int64_t s = 0; s < n_seq; ++s) {
        const int64_t m = ceil_div(ko[s + 1] - ko[s], kAttnKRows);
        if (m > max_kb) max_kb = m;
    }
    // query blocks of a selection group: as many score rows as fit in shared
    // memory beside 16 mean rows of the widest head
    const int64_t fit = max_kb > 0 ? (kSmemOptIn / 8 - 256 * kAttnGroupRows) / max_kb : kAttnGroupRows;
    const int group = fit >= kAttnGroupRows ? kAttnGroupRows : fit >= 8 ? 8 : fit >= 4 ? 4 : fit >= 2 ? 2 : 1;
    auto* plan = new (std::nothrow) s3dsp_attn_plan();
    // one upload: q_blocks int4, k_blocks int2, groups int2, first_kb int
    const size_t bytes = (size_t)nqb * (sizeof(int4) + sizeof(int2) + sizeof(int)) + (size_t)nkb * sizeof(int2) + 16;
    char* host = plan ? static_cast<char*>(::operator new(bytes, std::nothrow)) : nullptr;
    if (!host) {
        delete plan;
        return fail(error, error_capacity, S3D_OUT_OF_MEMORY, "plan allocation");
    }
    int4* qb = reinterpret_cast<int4*>(host);
    int2* kb = reinterpret_cast<int2*>(qb + nqb);
    int2* groups = kb + nkb;
    int* first_kb = reinterpret_cast<int*>(groups + nqb);
    int64_t iq = 0, ik = 0, ig = 0;
    for (int64_t s = 0; s < n_seq; ++s) {
        const int64_t q0 = h_q_offsets[s], ql = h_q_offsets[s + 1] - q0, k0 = ko[s], kl = ko[s + 1] - k0;
        const int64_t nb = ceil_div(ql, kAttnQRows);
        for (int64_t b = 0; b < nb; ++b) {
            const int64_t left = ql - b * kAttnQRows;
            if (b % group == 0) groups[ig++] = make_int2((int)iq, (int)(nb - b < group ? nb - b : group));
            plan->sum_kb += ceil_div(kl, kAttnKRows);
            if (plan->max_q_rows < left) plan->max_q_rows = (int)(left < kAttnQRows ? left : kAttnQRows);
            first_kb[iq] = (int)ik;
            qb[iq++] = make_int4((int)(q0 + b * kAttnQRows),
                                 (int)((left < kAttnQRows ? left : kAttnQRows) | (b << kAttnRowsBits)), (int)k0, (int)kl);
        }
        for (int64_t b = 0; b < ceil_div(kl, kAttnKRows); ++b) {
            const int64_t left = kl - b * kAttnKRows;
            kb[ik++] = make_int2((int)(k0 + b * kAttnKRows), (int)(left < kAttnKRows ? left : kAttnKRows));
        }
    }
    plan->device = ctx->device;
    plan->self = self;
    plan->n_q = nq, plan->n_k = nk;
    plan->first_q = h_q_offsets[0];
    plan->n_qb = (int)nqb, plan->n_kb = (int)nkb, plan->n_groups = (int)ig;
    plan->max_kb = (int)max_kb;
    plan->group = group;
    cudaError_t e = malloc_async(&plan->mem, bytes, ctx->stream);
    if (e == cudaSuccess) {
        // pageable memory: staged before the call returns
        e = cudaMemcpyAsync(plan->mem, host, bytes, cudaMemcpyHostToDevice, ctx->stream);
        if (e != cudaSuccess) cudaFreeAsync(plan->mem, ctx->stream);
    }
    ::operator delete(host);
    if (e != cudaSuccess) {
        delete plan;
        return cuda_fail(error, error_capacity, e, "plan upload");
    }
    plan->q_blocks = static_cast<int4*>(plan->mem);
    plan->k_blocks = reinterpret_cast<int2*>(plan->q_blocks + nqb);
    plan->groups = plan->k_blocks + nkb;
    plan->first_kb = reinterpret_cast<int*>(plan->groups + nqb);
    *out = plan;
    return S3D_OK;
}

extern "C" S3DSP_API void s3dsp_attn_plan_free(s3dsp_context* ctx, s3dsp_attn_plan* plan) {
    if (!plan) return;
    if (ctx) {
        cudaSetDevice(ctx->device);
        cudaFreeAsync(plan->mem, ctx->stream);
    }
    delete plan;
}

extern "C" S3DSP_API s3d_status s3dsp_attn_plan_info(const s3dsp_attn_plan* plan, int64_t* n_q, int64_t* n_k,
                                                     int64_t* q_blocks, int64_t* k_blocks, int64_t* max_k_blocks) {
    if (!plan) return S3D_INVALID_ARGUMENT;
    if (n_q) *n_q = plan->n_q;
    if (n_k) *n_k = plan->n_k;
    if (q_blocks) *q_blocks = plan->n_qb;
    if (k_blocks) *k_blocks = plan->n_kb;
    if (max_k_blocks) *max_k_blocks = plan->max_kb;
    return S3D_OK;
}

extern "C" S3DSP_API s3d_status s3dsp_block_select(s3dsp_context* ctx, const s3dsp_attn_plan* plan, const void* q,
                                                   int64_t q_stride, int32_t heads, const void* k, int64_t k_stride,
                                                   int32_t kv_heads, uint32_t dtype, int32_t d, int32_t top,
                                                   int32_t keep_local, int32_t* d_sel, char* error,
                                                   uint64_t error_capacity) {
    clear_error(error, error_capacity);
    if (!ctx || !plan) return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "NULL argument");
    if (plan->device != ctx->device)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "the plan is on device %d, the context on %d",
                    plan->device, ctx->device);
    if (!dtype_ok(dtype)) return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "bad dtype");
    if (d <= 0 || d % 8 || d > 256)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "head dimension %d (a multiple of 8 up to 256)", d);
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads > 4096)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "%d heads over %d key heads", heads, kv_heads);
    const int64_t qw = (int64_t)heads * d, kw = (int64_t)kv_heads * d;
    if (q_stride < qw || k_stride < kw)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "row stride below heads * d");
    if (top < 1 || top > kAttnMaxTop)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "top %d outside [1, %d]", top, kAttnMaxTop);
    if (keep_local && !plan->self)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "keep_local needs a plan whose keys are the query rows");
    if (plan->n_qb == 0) return S3D_OK;
    if (!q || !d_sel || (plan->n_k > 0 && !k)) return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "NULL argument");
    const size_t es = dtype_size(dtype);
    if (((uintptr_t)q | (uintptr_t)k) & (es - 1))
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "pointer not aligned to its type");
    const size_t smem = sizeof(double) * ((size_t)d * kGroup + (size_t)plan->group * plan->max_kb);
    if (smem > (size_t)kSmemOptIn)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "a sequence has %d key blocks: more than a selection takes",
                    plan->max_kb);
    S3DSP_CUDA(cudaSetDevice(ctx->device), "cudaSetDevice");
    static std::atomic<uint64_t> optin{0};
    S3DSP_CUDA(smem_optin((const void*)block_score_kernel, ctx->device, optin), "block_score_kernel");
    double* means = nullptr;
    const size_t n_qm = (size_t)plan->n_qb * qw, n_km = (size_t)plan->n_kb * kw;
    S3DSP_CUDA(malloc_async(&means, (n_qm + n_km) * sizeof(double), ctx->stream), "block means");
    MeanParams m = {q, k, q_stride, k_stride, (int)qw, (int)kw, plan->n_qb, plan->n_kb, plan->q_blocks, plan->k_blocks,
                    means, means + n_qm};
    const bool vec = !(((uintptr_t)q | (uintptr_t)k | (q_stride * es) | (k_stride * es)) & 15);
    const dim3 mg((unsigned)(plan->n_qb + plan->n_kb), (unsigned)ceil_div(qw, kMeanCols));
    cudaError_t e = cudaSuccess;
    auto mean = [&](auto kernel) { e = launch_pdl(kernel, mg, dim3(kMeanThreads), 0, ctx->stream, m); };
    if (dtype == S3DSP_F32)
        vec ? mean(block_mean_kernel<float, true>) : mean(block_mean_kernel<float, false>);
    else if (dtype == S3DSP_BF16)
        vec ? mean(block_mean_kernel<__nv_bfloat16, true>) : mean(block_mean_kernel<__nv_bfloat16, false>);
    else
        vec ? mean(block_mean_kernel<__half, true>) : mean(block_mean_kernel<__half, false>);
    if (e == cudaSuccess) {
        ScoreParams s = {plan->groups, plan->q_blocks, plan->first_kb, means, means + n_qm, (int)qw, plan->n_kb, d, heads,
                         heads / kv_heads, top, keep_local, plan->max_kb, d_sel};
        e = launch_pdl(block_score_kernel, dim3((unsigned)plan->n_groups, (unsigned)heads), dim3(kScoreThreads), smem,
                       ctx->stream, s);
    }
    const cudaError_t f = cudaFreeAsync(means, ctx->stream);
    if (e == cudaSuccess) e = f;
    if (e != cudaSuccess) return cuda_fail(error, error_capacity, e, "block_select kernels");
    return S3D_OK;
}

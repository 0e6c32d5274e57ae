// Plans of ragged attention batches, and the selection of key blocks by a
// cheap score.
//
//   s3dsp_attn_plan_create  cuts every sequence into query blocks of 128 rows and key blocks of 64
//   s3dsp_block_select      per (query block, head): the key blocks of its sequence with the
//                           largest <mean of the block's q rows, mean of the key block's k rows>
//
// A selection is whole numbers: two scores that differ by less than f32
// rounding would swap blocks between two ways of adding the same rows, so the
// sums, means and scores are f64 (exact sums of 16-bit rows, in practice), each
// added in one fixed order, whatever the grid. The f64 work is 1 / (128 * 64) of the attention it steers.
//
//   block_mean_kernel   one pass over q and k (memory bound): a warp lane owns eight columns, eight
//                       warps share the block's rows, f64 sums joined in warp order
//   block_score_kernel  scores of 32 query blocks x 128 key blocks of one sequence and head, a tile
//                       product in f64 (bound by the f64 pipe, 64 FMAs a cycle and SM), written as
//                       64-bit keys whose unsigned order is the scores'
//   top_warp_kernel     one warp per (query block, head): the top-th largest key by bisection, the
//                       keys' upper halves in registers; the chosen indices in ascending order
//   top_block_kernel    the same with one CTA per row and the keys in shared memory, for a batch with a
//                       sequence of more key blocks than a warp's registers take (1,024): up to 64
//                       counts over the keys, each with two barriers; 65,600 rows (1,025 key blocks) 367 us
//                       against 140 for 65,500
//
// 65,500 rows, 16 heads of 64, bf16, lists of 32 (one B200): 141 us, of which the means 54 (268 MB
// at 5.0 TB/s), the scores 55, the lists 30. Scores in f32 with an error bound, and f64 only where
// the bound leaves a list in doubt: scores 37, lists 40, 135 us in all; at 28,000 and 1,900 rows
// 70 and 27 us where this takes 66 and 25. Means with the 16-bit values taken to f64 by integer
// instructions, or with a row's columns read by neighbouring CTAs: 54 and 61 us.
#include <algorithm>

#include "s3dsp_internal.h"

using namespace s3dsp;

namespace {

constexpr int kMeanThreads = 256;
constexpr int kMeanCols = 256;  // columns per CTA of the mean kernel: 32 lanes x 8
constexpr int kTileQ = kAttnGroupRows, kTileK = 128, kTileD = 16;  // of the score kernel
constexpr int kScoreThreads = 32 * (kTileK / 32);                    // a warp per 32 key blocks
constexpr int kScoreLd = kTileD + 4;                                // shared row: 8 rows x 4 columns hit every bank once
constexpr int kWarpKeys = 32;                                     // key blocks per lane of top_warp_kernel
constexpr size_t kScoreSmem = 2 * sizeof(double) * (kTileQ + kTileK) * kScoreLd;  // four CTAs per SM
constexpr int kMaxKeys = 28000;                                   // key blocks of a sequence: top_block_kernel's memory
constexpr size_t kScoreBytes = (size_t)1 << 29;                   // scratch of scores that a pass may take

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
    double* q_mean;  // [n_qb][qw]
    double* k_mean;  // [n_kb][kw]
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
        constexpr int U = sizeof(T) == 4 ? 4 : 8;  // rows in flight
        for (int r0 = warp; r0 < rows; r0 += 8 * U) {
            T e[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const T* x = base + (int64_t)(r0 + 8 * u) * ld;
                if (r0 + 8 * u >= rows) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) e[u][j] = T(0.f);
                } else if constexpr (kVec) {
#pragma unroll
                    for (int w = 0; w < (int)sizeof(T) / 2; ++w)
                        reinterpret_cast<uint4*>(e[u])[w] = __ldg(reinterpret_cast<const uint4*>(x) + w);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) e[u][j] = x[j];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[j] += to_d(e[u][j]);
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
    (is_k ? p.k_mean + (int64_t)b * p.kw : p.q_mean + (int64_t)b * p.qw)[col] = s;
}

struct ScoreParams {
    const int2* groups;     // {first query block, blocks}: one sequence's; those of this pass
    const int4* q_blocks;   // {first row, rows | index in the sequence << 8, first key row, key rows}
    const int* first_kb;    // [n_qb] first key block of the block's sequence
    const double* q_mean;
    const double* k_mean;
    int qw, kw, d, heads, per_kv, top, keep_local;
    int block0, block_count;  // query blocks of this pass
    int head0, head_count;    // heads of this pass
    int max_kb;               // keys of a row
    unsigned long long* keys;  // [block_count][head_count][max_kb]
    int32_t* sel;              // [n_qb][heads][top]
};

// f64 -> u64 whose unsigned order is the scores' order; NaN lowest
__device__ __forceinline__ unsigned long long ordered(double v) {
    if (v != v) return 0ull;
    const long long b = __double_as_longlong(v + 0.0);  // -0 and 0 are one score
    return b < 0 ? ~(unsigned long long)b : (unsigned long long)b | 0x8000000000000000ull;
}

// d (8 x 8, two values a lane) += a (8 x 4) b^T (8 x 4), f64
__device__ __forceinline__ void mma_f64(double (&d)[2], double a, double b) {
    asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
                 : "+d"(d[0]), "+d"(d[1])
                 : "d"(a), "d"(b));
}

// A warp owns 32 query blocks x 32 key blocks as 4 x 4 f64 MMAs: eight shared
// loads feed sixteen of them. (Scalar FMAs run at the same rate but need a
// shared load each: 90 us with 4 x 4 register blocks where this takes 55, for
// 512 x 1,024 blocks and 16 heads of 64.) Every score is the same sequence of
// MMA steps, so that equal blocks have equal scores.
__global__ void __launch_bounds__(kScoreThreads) block_score_kernel(const ScoreParams p) {
    // two stages of kTileD columns of the query rows and, below them, the key rows
    extern __shared__ __align__(16) double stage[][kTileQ + kTileK][kScoreLd];
    pdl_wait();
    pdl_trigger();
    const int2 grp = p.groups[blockIdx.x];
    const int b0 = grp.x, count = grp.y, c0 = blockIdx.y * kTileK, h = p.head0 + blockIdx.z;
    const int4 qb0 = p.q_blocks[b0];
    const int nkb = (qb0.w + kAttnKRows - 1) / kAttnKRows;
    if (c0 >= nkb || nkb <= p.top) return;  // all blocks are taken: no scores needed
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int lr = lane >> 2, lk = lane & 3;  // the lane's row and column of an operand
    const double* qm = p.q_mean + (int64_t)b0 * p.qw + (int64_t)h * p.d;
    const double* km = p.k_mean + (int64_t)(p.first_kb[b0] + c0) * p.kw + (int64_t)(h / p.per_kv) * p.d;
    double acc[4][4][2];
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y][0] = acc[x][y][1] = 0.0;
    const bool work = c0 + 32 * warp < nkb;
    // rows or columns that are not there: zeros (d is a multiple of 8)
    auto load = [&](int j0, int st) {
        const int j = 2 * (threadIdx.x % (kTileD / 2));
#pragma unroll
        for (int r = threadIdx.x / (kTileD / 2); r < kTileQ + kTileK; r += kScoreThreads / (kTileD / 2)) {
            const bool q = r < kTileQ, in = j0 + j < p.d && (q ? r < count : c0 + r - kTileQ < nkb);
            const double* src = q ? qm + (int64_t)r * p.qw : km + (int64_t)(r - kTileQ) * p.kw;
            const uint32_t dst = (uint32_t)__cvta_generic_to_shared(&stage[st][r][j]);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(in ? src + j0 + j : qm),
                         "r"(in ? 16 : 0)
                         : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    load(0, 0);
    for (int j0 = 0, st = 0; j0 < p.d; j0 += kTileD, st ^= 1) {
        load(j0 + kTileD, st ^ 1);  // past the last column: zeros that nothing reads
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncthreads();
        if (work) {
#pragma unroll
            for (int i = 0; i < kTileD; i += 4) {
                double a[4], b[4];
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    a[x] = stage[st][8 * x + lr][i + lk], b[x] = stage[st][kTileQ + 32 * warp + 8 * x + lr][i + lk];
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int y = 0; y < 4; ++y) mma_f64(acc[x][y], a[x], b[y]);
            }
        }
        __syncthreads();
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (!work) return;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        const int r = 8 * x + lr;
        if (r >= count) continue;
        // the key blocks of the query block's own rows come first
        const int own = p.keep_local ? ((qb0.y >> kAttnRowsBits) + r) * (kAttnQRows / kAttnKRows) : -2;
        unsigned long long* row = p.keys + ((int64_t)(b0 + r - p.block0) * p.head_count + blockIdx.z) * p.max_kb;
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = c0 + 32 * warp + 8 * y + 2 * lk + e;
                if (c < nkb) row[c] = c >= own && c < own + kAttnQRows / kAttnKRows ? ~0ull : ordered(acc[x][y][e]);
            }
    }
}

// Writes the lane's index c to the row's list when it is taken: keys above the
// threshold, and the first `ties` of those equal to it. A warp's step of 32.
__device__ __forceinline__ void emit(int32_t* out, int c, bool above, bool equal, int lane, int& done, int& ties) {
    const unsigned below = (1u << lane) - 1u, em = __ballot_sync(0xffffffffu, equal);
    const bool take = above || (equal && __popc(em & below) < ties);
    const unsigned tm = __ballot_sync(0xffffffffu, take);
    if (take) out[done + __popc(tm & below)] = c;
    done += __popc(tm);
    ties -= min(ties, __popc(em));
}

constexpr int kCandidates = 128;
__global__ void __launch_bounds__(128) top_warp_kernel(const ScoreParams p) {
    __shared__ int candidates[4][kCandidates];
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (item >= (int64_t)p.block_count * p.head_count) return;
    const int b = p.block0 + (int)(item / p.head_count), h = p.head0 + (int)(item % p.head_count);
    const int nkb = (p.q_blocks[b].w + kAttnKRows - 1) / kAttnKRows;
    int32_t* out = p.sel + ((int64_t)b * p.heads + h) * p.top;
    if (nkb <= p.top) {  // all of them
        for (int i = lane; i < p.top; i += 32) out[i] = i < nkb ? i : -1;
        return;
    }
    const uint2* key = reinterpret_cast<const uint2*>(p.keys + item * p.max_kb);  // {lower, upper half}
    const int steps = (nkb + 31) / 32;
    uint32_t hi[kWarpKeys];
    uint32_t lo_bound = 0xffffffffu, hi_bound = 0u;
#pragma unroll
    for (int i = 0; i < kWarpKeys; ++i) {
        const int c = 32 * i + lane;
        hi[i] = 0u;
        if (i < steps && c < nkb) {
            hi[i] = key[c].y;
            lo_bound = min(lo_bound, hi[i]);
            hi_bound = max(hi_bound, hi[i]);
        }
    }
    // lo: at_lo >= top upper halves are >= lo; up: fewer are >= up. For up to 32
    // blocks the top-th largest of the lanes' maxima is such an lo, close to the
    // threshold (each lane holds every 32nd block).
    const uint32_t low = __reduce_min_sync(0xffffffffu, lo_bound);
    uint64_t up = (uint64_t)__reduce_max_sync(0xffffffffu, hi_bound) + 1;
    uint32_t lo = low;
    if (p.top <= 32) {
        int rank = 0;
#pragma unroll
        for (int x = 0; x < 32; ++x) {
            const uint32_t other = __shfl_sync(0xffffffffu, hi_bound, x);
            rank += other > hi_bound || (other == hi_bound && x < lane);
        }
        const unsigned m = __ballot_sync(0xffffffffu, rank == p.top - 1);
        lo = max(low, __shfl_sync(0xffffffffu, hi_bound, __ffs(m) - 1));
    }
    auto count = [&](uint32_t t) {
        int m = 0;
#pragma unroll
        for (int i = 0; i < kWarpKeys; ++i)
            if (i < steps) m += 32 * i + lane < nkb && hi[i] >= t;
        return (int)__reduce_add_sync(0xffffffffu, m);
    };
    int at_lo = count(lo);
    while (up - lo > 1 && at_lo > kCandidates) {
        const uint32_t mid = (uint32_t)(lo + (up - lo) / 2);
        const int m = count(mid);
        if (m >= p.top)
            lo = mid, at_lo = m;
        else
            up = mid;
    }
    if (at_lo <= kCandidates) {
        // the blocks left, in index order, four to a lane; their whole keys decide
        int* cand = candidates[threadIdx.x >> 5];
        int n = 0;
#pragma unroll
        for (int i = 0; i < kWarpKeys; ++i)
            if (i < steps) {
                const bool is = 32 * i + lane < nkb && hi[i] >= lo;
                const unsigned m = __ballot_sync(0xffffffffu, is);
                if (is) cand[n + __popc(m & ((1u << lane) - 1u))] = 32 * i + lane;
                n += __popc(m);
            }
        __syncwarp();
        const unsigned long long* key64 = p.keys + item * p.max_kb;
        unsigned long long k[kCandidates / 32];
        int c[kCandidates / 32];
#pragma unroll
        for (int i = 0; i < kCandidates / 32; ++i) {
            const bool is = 32 * i + lane < n;
            c[i] = is ? cand[32 * i + lane] : -1;
            k[i] = is ? key64[c[i]] : 0ull;
        }
        unsigned long long a = (unsigned long long)lo << 32;
        unsigned long long z = up > 0xffffffffull ? ~0ull : ((unsigned long long)up << 32) - 1;  // fewer than top are above z
        // the largest threshold in [a, z] that `top` keys reach
        int at_a = n;
        while (a < z && at_a != p.top) {
            const unsigned long long mid = a + (z - a) / 2 + 1;
            int m = 0;
#pragma unroll
            for (int i = 0; i < kCandidates / 32; ++i) m += c[i] >= 0 && k[i] >= mid;
            m = __reduce_add_sync(0xffffffffu, m);
            if (m >= p.top)
                a = mid, at_a = m;
            else
                z = mid - 1;
        }
        int over = 0, done = 0;
#pragma unroll
        for (int i = 0; i < kCandidates / 32; ++i) over += c[i] >= 0 && k[i] > a;
        int ties = p.top - (int)__reduce_add_sync(0xffffffffu, over);
        if (at_a == p.top) ties = n;  // all that reach it
#pragma unroll
        for (int i = 0; i < kCandidates / 32; ++i)
            if (32 * i < n) emit(out, c[i], c[i] >= 0 && k[i] > a, c[i] >= 0 && k[i] == a, lane, done, ties);
        return;
    }
    // lists longer than that, or as many keys that share the threshold's upper
    // half (up = lo + 1): bisect on
    while (up - lo > 1 && at_lo != p.top) {
        const uint32_t mid = (uint32_t)(lo + (up - lo) / 2);
        const int m = count(mid);
        if (m >= p.top)
            lo = mid, at_lo = m;
        else
            up = mid;
    }
    int done = 0, ties = 0;
    if (at_lo == p.top) {  // those >= lo are the list
#pragma unroll
        for (int i = 0; i < kWarpKeys; ++i)
            if (i < steps) emit(out, 32 * i + lane, 32 * i + lane < nkb && hi[i] >= lo, false, lane, done, ties);
        return;
    }
    // several keys share the threshold's upper half: bisect their lower halves
    int above = 0;
#pragma unroll
    for (int i = 0; i < kWarpKeys; ++i)
        if (i < steps) above += 32 * i + lane < nkb && hi[i] > lo;
    above = __reduce_add_sync(0xffffffffu, above);
    const int want = p.top - above;
    uint32_t t = 0u;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t cand = t | (1u << bit);
        int m = 0;
        for (int i = 0; i < steps; ++i) {
            const int c = 32 * i + lane;
            if (c < nkb) {
                const uint2 k = key[c];
                m += k.y == lo && k.x >= cand;
            }
        }
        if (__reduce_add_sync(0xffffffffu, m) >= want) t = cand;
    }
    int over = 0;
    for (int i = 0; i < steps; ++i) {
        const int c = 32 * i + lane;
        if (c < nkb) {
            const uint2 k = key[c];
            over += k.y == lo && k.x > t;
        }
    }
    ties = want - __reduce_add_sync(0xffffffffu, over);
    for (int i = 0; i < steps; ++i) {
        const int c = 32 * i + lane;
        const uint2 k = c < nkb ? key[c] : make_uint2(0u, 0u);
        emit(out, c, c < nkb && (k.y > lo || (k.y == lo && k.x > t)), c < nkb && k.y == lo && k.x == t, lane, done, ties);
    }
}

constexpr int kTopThreads = 512;
__global__ void __launch_bounds__(kTopThreads) top_block_kernel(const ScoreParams p) {
    extern __shared__ unsigned long long key[];  // [max_kb], then two counters
    int* total = reinterpret_cast<int*>(key + p.max_kb);
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t item = blockIdx.x;
    const int b = p.block0 + (int)(item / p.head_count), h = p.head0 + (int)(item % p.head_count);
    const int nkb = (p.q_blocks[b].w + kAttnKRows - 1) / kAttnKRows;
    int32_t* out = p.sel + ((int64_t)b * p.heads + h) * p.top;
    if (nkb <= p.top) {
        for (int i = threadIdx.x; i < p.top; i += kTopThreads) out[i] = i < nkb ? i : -1;
        return;
    }
    for (int c = threadIdx.x; c < nkb; c += kTopThreads) key[c] = p.keys[item * p.max_kb + c];
    if (threadIdx.x < 2) total[threadIdx.x] = 0;
    __syncthreads();
    int turn = 0;  // the counter in use; the other one is cleared meanwhile
    auto count = [&](unsigned long long t) {
        int m = 0;
        for (int c = threadIdx.x; c < nkb; c += kTopThreads) m += key[c] >= t;
        m = __reduce_add_sync(0xffffffffu, m);
        if (lane == 0) atomicAdd(&total[turn], m);
        __syncthreads();
        m = total[turn];
        if (threadIdx.x == 0) total[turn ^ 1] = 0;
        turn ^= 1;
        __syncthreads();
        return m;
    };
    unsigned long long t = 0ull;
    for (int bit = 63; bit >= 0; --bit) {
        const unsigned long long cand = t | (1ull << bit);
        const int m = count(cand);
        if (m >= p.top) t = cand;
        if (m == p.top) break;
    }
    int ties = p.top - (t == ~0ull ? 0 : count(t + 1)), done = 0;
    if (threadIdx.x >= 32) return;
    for (int c0 = 0; c0 < nkb && done < p.top; c0 += 32) {
        const int c = c0 + lane;
        const unsigned long long k = c < nkb ? key[c] : 0ull;
        emit(out, c, c < nkb && k > t, c < nkb && k == t, lane, done, ties);
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
    auto* plan = new (std::nothrow) s3dsp_attn_plan();
    // one upload: q_blocks int4, k_blocks int2, groups int2, first_kb int, order int
    const size_t bytes = (size_t)nqb * (sizeof(int4) + sizeof(int2) + 2 * sizeof(int)) + (size_t)nkb * sizeof(int2) + 16;
    char* host = plan ? static_cast<char*>(::operator new(bytes, std::nothrow)) : nullptr;
    if (host) {
        plan->by_length = static_cast<int4*>(::operator new(((size_t)n_seq + 1) * sizeof(int4), std::nothrow));
        plan->group_first = static_cast<int*>(::operator new(((size_t)nqb + 1) * sizeof(int), std::nothrow));
    }
    if (!host || !plan->by_length || !plan->group_first) {
        ::operator delete(host);
        if (plan) ::operator delete(plan->by_length), ::operator delete(plan->group_first);
        delete plan;
        return fail(error, error_capacity, S3D_OUT_OF_MEMORY, "plan allocation");
    }
    int4* qb = reinterpret_cast<int4*>(host);
    int2* kb = reinterpret_cast<int2*>(qb + nqb);
    int2* groups = kb + nkb;
    int* first_kb = reinterpret_cast<int*>(groups + nqb);
    int* order = first_kb + nqb;
    int4* seqs = plan->by_length;  // {key blocks, sequence, first query block, query blocks} until it is sorted
    int64_t iq = 0, ik = 0, ig = 0, is = 0;
    for (int64_t s = 0; s < n_seq; ++s) {
        const int64_t q0 = h_q_offsets[s], ql = h_q_offsets[s + 1] - q0, k0 = ko[s], kl = ko[s + 1] - k0;
        const int64_t nb = ceil_div(ql, kAttnQRows);
        if (nb > 0) {
            const int blocks = (int)ceil_div(kl, kAttnKRows);
            seqs[is++] = make_int4(blocks, (int)s, (int)iq, (int)nb);
            if (blocks > plan->max_list) plan->max_list = blocks;
        }
        for (int64_t b = 0; b < nb; ++b) {
            const int64_t left = ql - b * kAttnQRows;
            if (b % kAttnGroupRows == 0) {
                plan->group_first[ig] = (int)iq;
                groups[ig++] = make_int2((int)iq, (int)(nb - b < kAttnGroupRows ? nb - b : kAttnGroupRows));
            }
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
    std::sort(seqs, seqs + is, [](const int4& a, const int4& b) { return a.x != b.x ? a.x > b.x : a.y < b.y; });
    int64_t io = 0;
    for (int64_t s = 0; s < is; ++s) {
        for (int b = 0; b < seqs[s].w; ++b) order[io++] = seqs[s].z + b;
        seqs[s].y = (int)io;
    }
    plan->n_by_length = (int)is;
    plan->group_first[ig] = (int)nqb;
    plan->device = ctx->device;
    plan->self = self;
    plan->n_q = nq, plan->n_k = nk;
    plan->n_qb = (int)nqb, plan->n_kb = (int)nkb, plan->n_groups = (int)ig;
    plan->max_kb = (int)max_kb;
    cudaError_t e = malloc_async(&plan->mem, bytes, ctx->stream);
    if (e == cudaSuccess) {
        // pageable memory: staged before the call returns
        e = cudaMemcpyAsync(plan->mem, host, bytes, cudaMemcpyHostToDevice, ctx->stream);
        if (e != cudaSuccess) cudaFreeAsync(plan->mem, ctx->stream);
    }
    ::operator delete(host);
    if (e != cudaSuccess) {
        ::operator delete(plan->by_length);
        ::operator delete(plan->group_first);
        delete plan;
        return cuda_fail(error, error_capacity, e, "plan upload");
    }
    plan->q_blocks = static_cast<int4*>(plan->mem);
    plan->k_blocks = reinterpret_cast<int2*>(plan->q_blocks + nqb);
    plan->groups = plan->k_blocks + nkb;
    plan->first_kb = reinterpret_cast<int*>(plan->groups + nqb);
    plan->order = plan->first_kb + nqb;
    *out = plan;
    return S3D_OK;
}

extern "C" S3DSP_API void s3dsp_attn_plan_free(s3dsp_context* ctx, s3dsp_attn_plan* plan) {
    if (!plan) return;
    cudaSetDevice(plan->device);
    cudaFreeAsync(plan->mem, ctx ? ctx->stream : nullptr);
    ::operator delete(plan->by_length);
    ::operator delete(plan->group_first);
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
    if ((int64_t)plan->n_qb * heads > 0x7fffffff)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "too many query blocks times heads");
    const size_t es = dtype_size(dtype);
    if (((uintptr_t)q | (uintptr_t)k) & (es - 1))
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "pointer not aligned to its type");
    const int longest = plan->max_list;  // key blocks of a row's sequence, at most
    if (longest > kMaxKeys)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "a sequence has %d key blocks (at most %d)", longest,
                    kMaxKeys);
    S3DSP_CUDA(cudaSetDevice(ctx->device), "cudaSetDevice");
    static std::atomic<uint64_t> optin{0}, score_optin{0};
    S3DSP_CUDA(smem_optin((const void*)block_score_kernel, ctx->device, score_optin), "block_score_kernel");
    S3DSP_CUDA(smem_optin((const void*)top_block_kernel, ctx->device, optin), "top_block_kernel");
    double* means = nullptr;
    const size_t n_qm = (size_t)plan->n_qb * qw, n_km = (size_t)plan->n_kb * kw;
    // scores of as many heads at a time as kScoreBytes take, or of one head and as many groups of query
    // blocks (one at least: 32 rows of up to 28,000 keys are 7 MB)
    const size_t row_bytes = (size_t)plan->n_qb * longest * sizeof(unsigned long long);
    const bool scored = longest > top;
    int64_t pass = scored && row_bytes * heads > kScoreBytes ? kScoreBytes / row_bytes : heads;
    if (pass < 1) pass = 1;
    int64_t pass_blocks = plan->n_qb;
    if (scored && row_bytes > kScoreBytes) pass_blocks = kScoreBytes / (longest * sizeof(unsigned long long));
    const size_t score_bytes = scored ? row_bytes / plan->n_qb * pass_blocks * pass : 0;
    S3DSP_CUDA(malloc_async(&means, (n_qm + n_km) * sizeof(double) + score_bytes + 16, ctx->stream), "block scores");
    MeanParams m = {q, k, q_stride, k_stride, (int)qw, (int)kw, plan->n_qb, plan->n_kb, plan->q_blocks, plan->k_blocks,
                    means, means + n_qm};
    const bool vec = !(((uintptr_t)q | (uintptr_t)k | (q_stride * es) | (k_stride * es)) & 15);
    const dim3 mg((unsigned)(plan->n_qb + plan->n_kb), (unsigned)ceil_div(qw, kMeanCols));
    cudaError_t e = cudaSuccess;
    auto mean = [&](auto kernel) { e = launch_pdl(kernel, mg, dim3(kMeanThreads), 0, ctx->stream, m); };
    if (!scored)
        ;  // every list holds all blocks
    else if (dtype == S3DSP_F32)
        vec ? mean(block_mean_kernel<float, true>) : mean(block_mean_kernel<float, false>);
    else if (dtype == S3DSP_BF16)
        vec ? mean(block_mean_kernel<__nv_bfloat16, true>) : mean(block_mean_kernel<__nv_bfloat16, false>);
    else
        vec ? mean(block_mean_kernel<__half, true>) : mean(block_mean_kernel<__half, false>);
    ScoreParams s = {plan->groups, plan->q_blocks, plan->first_kb, means, means + n_qm, (int)qw, (int)kw, d,
                     heads, heads / kv_heads, top, keep_local, 0, 0, 0, 0, longest,
                     reinterpret_cast<unsigned long long*>(means + n_qm + n_km), d_sel};
    const int* first = plan->group_first;
    for (int g0 = 0, g1; g0 < plan->n_groups && e == cudaSuccess; g0 = g1) {
        // whole groups, up to pass_blocks query blocks
        g1 = (int)(std::upper_bound(first + g0 + 1, first + plan->n_groups + 1, first[g0] + pass_blocks) - first) - 1;
        s.groups = plan->groups + g0;
        s.block0 = first[g0];
        s.block_count = first[g1] - first[g0];
        for (int h0 = 0; h0 < heads && e == cudaSuccess; h0 += (int)pass) {
            s.head0 = h0;
            s.head_count = (int)(heads - h0 < pass ? heads - h0 : pass);
            if (scored)
                e = launch_pdl(block_score_kernel,
                               dim3((unsigned)(g1 - g0), (unsigned)ceil_div(longest, kTileK), (unsigned)s.head_count),
                               dim3(kScoreThreads), kScoreSmem, ctx->stream, s);
            if (e != cudaSuccess) break;
            const int64_t items = (int64_t)s.block_count * s.head_count;
            if (longest <= 32 * kWarpKeys)
                e = launch_pdl(top_warp_kernel, dim3((unsigned)ceil_div(items, 4)), dim3(128), 0, ctx->stream, s);
            else
                e = launch_pdl(top_block_kernel, dim3((unsigned)items), dim3(kTopThreads),
                               (longest + 1) * sizeof(unsigned long long), ctx->stream, s);
        }
    }
    const cudaError_t f = cudaFreeAsync(means, ctx->stream);
    if (e == cudaSuccess) e = f;
    if (e != cudaSuccess) return cuda_fail(error, error_capacity, e, "block_select kernels");
    return S3D_OK;
}

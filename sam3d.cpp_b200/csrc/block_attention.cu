// Block attention: out = softmax(scale q k^T) v of each query row over the
// rows of its listed key blocks (64 rows each), or over its whole sequence.
//
// One CTA per (query block of 128 rows, head); short blocks of grouped heads
// share a tile; where there are few tiles, or a few long ones, lists are split
// over CTAs and joined by a second kernel. The row maximum and sum run along with
// the blocks (online softmax), so scores never leave the SM:
//
//   key warp        K tiles by TMA into a ring; S = Q K^T (tcgen05, f32 in TMEM)
//   value warp      V tiles by TMA into a ring; O += P V with P read from TMEM
//   softmax warps   one thread per query row: S from TMEM, p = 2^(c s - c m), maximum and sum on the
//                   way, P back into S's first columns
//
// Two score buffers: the scores of the next block are computed while this
// block's softmax runs, and P(j) V(j) while softmax(j + 1) runs, so that the
// softmax warps wait for neither. Q K^T writes a buffer again only after P V,
// its last reader, has completed.
//
// Weights are taken against the maximum of the blocks before. The block's own
// maximum is found along the way, and only where it has grown by more than
// kSlack (in powers of two) is it taken over: O is rescaled, a round trip
// through TMEM, and the block's weights are computed again from the scores in
// registers. The softmax is the same for any reference near the maximum. P is
// rounded to the input type (8 or 11 bits, as v has), which the MMA wants of
// both operands: the relative error of an output goes from 0.0017 to 0.0023 in
// bf16 and from 0.00021 to 0.00029 in f16. Its sum is taken before that, in f32.
//
// Rows past the block's keys: their scores are replaced by -inf (so p is 0)
// and their V rows by zeros in shared memory, whatever they hold.
//
// What bounds it (one B200, dense, 4,096 x 4,096 rows, 128 x 64 tiles):
//   d = 64   148 heads, 827 us, 768 TFLOP/s (0.45 of the measured bf16 peak). The softmax warps: 64
//            exponentials a row and tile at 16 a cycle and SM are 512 cycles, a tile takes about 690
//            (1.7 GHz under this load); MMAs and barriers alone 540 us. A part of the exponentials on
//            the FMA pipe (a polynomial): 851 us with one in eight, 894 with two. Two threads per row, or
//            two groups of softmax warps per CTA: 909, 896. One warp for all MMAs: 868.
//   d = 128  74 heads, 516 us, 1,232 TFLOP/s (0.73): MMAs and barriers alone 456 us; tensor pipe and
//            exponentials busy 62 % of the cycles each
#include <algorithm>
#include <cmath>
#include <limits>

#include "tc_common.cuh"

using namespace s3dsp;
using namespace s3dsp::tc;

namespace {

constexpr int kQ = kAttnQRows, kK = kAttnKRows;
constexpr int kQPanel = kQ * 128, kKPanel = kK * 128;  // bytes of 64 columns of a Q / K / V tile
// How far (in powers of two) a row's maximum may grow past the one in use.
constexpr float kSlack = 8.f;
// All weights carry a factor 2^kShift, which the division by their sum takes out
// again. bf16: a weight is 1 at most, so that their sum with v ends where f32 does
// for weights exp(s - max) (|v| times the rows 2^128), however the maximum grew.
// f16, whose range is short: the largest weight is 2^15 (of 65,504), so that one
// is exact to its 11 bits down to 2^-21 of the row's largest and lost only
// below 2^-32 of it. Without the shift many keys of weight 2^-14 to 2^-25 beside a
// single large one came out wrong by up to their whole sum.
template <bool kF16>
constexpr float kShift = kF16 ? 7.f : -kSlack;
// A score's weight is 2^(slope s + bias), one FMA: slope = c, and bias = kShift - c m
// rounded once for the row, so that a row's reference is its bias, and what it has summed up is
// rescaled by the difference of two. Past this value of c |m|, where neighbouring f32 scores are about
// a power of two apart, the rounding of c m would decide a weight: the slope is c's power of two
// (or less, where slope m ends), with which slope m is exact.
constexpr float kFar = 1 << 23;
template <bool kF16>
__device__ __forceinline__ float weight_shift(float m, float c) {
    return fabsf(m) * c > kFar ? 0.f : kShift<kF16>;
}
constexpr int kMinChunk = 4;    // key blocks of a chunk of a split list, at least
constexpr int kMaxChunks = 128;
constexpr int kMinSaved = 10;   // key blocks that a split has to take off the longest list
constexpr int kJoinRows = 8192;
constexpr int64_t kMaxPartBytes = 1 << 28;  // partial sums of split lists

struct AttnParams {
    const int4* q_blocks;
    const int32_t* sel;  // [n_qb][heads][top], or nullptr
    int top, heads, per_kv;
    int pack;   // heads of a group that share a tile: tile row r is query row r / pack, head r % pack
    int n_qb, per_block;  // query blocks, tiles of each: heads / pack
    // Tiles whose lists are split come first: the n_long first query blocks of `order`, head by head, and
    // `chunks` CTAs each with `chunk` list entries. Then the other tiles: query block by query block of
    // `order`, or without one head by head.
    const int* order;
    int n_long, chunk, chunks, split_ctas;
    float c;    // scale * log2(e)
    const void* q;
    int64_t q_stride;
    void* out;
    int64_t out_stride;
    int tiles, tile_rows;  // split tiles; most rows of a tile
    float* part_o;   // [tiles][chunks][tile_rows][D] unnormalised sums
    float2* part_ml; // [tiles][chunks][tile_rows] their row maximum and sum
    uint32_t* status;
};

// Two CTAs per SM: 256 of its 512 TMEM columns each, kBufs score buffers of 64
// columns and the accumulator; K and V rings as deep as half the shared memory
// takes.
template <int D>
struct Cfg {
    static constexpr int kPanels = D / 64;
    // Q as a TMEM operand where the accumulator leaves the columns: Q K^T then reads only K from shared
    // memory (d = 64: 827 against 850 us); else in shared memory
    static constexpr bool kQTmem = D == 64;
    static constexpr int kBufs = 2;            // blocks whose scores are computed ahead of the softmax
    static constexpr int kKS = D == 64 ? 4 : 2, kVS = kKS;
    static constexpr int kThreads = 128 + 64;
    // d = 128 takes registers as for 8 warps (128 each). With the 168 that six warps allow, two CTAs of
    // six fit on an SM only where they put their pairs of warps on different schedulers, which they do
    // not always after CTAs of different lengths (8 single rows: 64 against 58 us). d = 64 takes the
    // registers all the same: 827 against 843 us dense, 521 against 536 sparse.
    static constexpr int kRegThreads = D == 64 ? kThreads : 256;
    static constexpr int kTmemCols = 256;
    static constexpr int kOCol = 64 * kBufs, kQCol = kOCol + D;  // S buffers | O | Q
    static_assert(kQCol + (kQTmem ? D / 2 : 0) <= kTmemCols, "TMEM");
    // q_full | k_full, k_empty [kKS] | v_full, v_empty [kVS] | s_full, p_full, o_done [kBufs] | drained [2]
    static constexpr int kBars = 1 + 2 * kKS + 2 * kVS + 3 * kBufs + 2;
    static constexpr int kQBytes = kQTmem ? 0 : kPanels * kQPanel;
    static constexpr size_t kTiles = kQBytes + (size_t)(kKS + kVS) * kPanels * kKPanel;
    static constexpr size_t smem(int list) { return 1024 + kTiles + kBars * 8 + 16 + (size_t)list * 4; }
};


// A place in a ring of N: the slot and the parity of its current pass.
template <int N>
struct Cursor {
    int slot = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next() {
        if (++slot == N) slot = 0, parity ^= 1u;
    }
};

// true in one lane of the (converged) warp. The compiler knows that a branch
// on it has one thread, so MMA descriptors stay in uniform registers: behind
// `lane == 0` each tcgen05 instruction cost about 80 cycles to issue, which
// made the issuing warp the bottleneck.
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"((unsigned long long)map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)map) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// D (f32, TMEM) += A (16-bit, TMEM) * B (shared memory)
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// 16-bit operand whose N (or M) index is contiguous: 128-byte rows of 64
// columns, one row per K index, 128-byte swizzle; 8-row groups 1,024 bytes
// apart along K, 64-column panels kKPanel bytes apart along N.
__device__ __forceinline__ uint64_t mn_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(kKPanel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
#define S3DSP_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), \
                       "=r"(v[o + 6]), "=r"(v[o + 7])
#define S3DSP_I8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), \
                       "r"(v[o + 6]), "r"(v[o + 7])
#define S3DSP_RW8(v, o) "+r"(v[o]), "+r"(v[o + 1]), "+r"(v[o + 2]), "+r"(v[o + 3]), "+r"(v[o + 4]), "+r"(v[o + 5]), \
                        "+r"(v[o + 6]), "+r"(v[o + 7])
// 32 columns of this thread's TMEM lane (no wait)
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : S3DSP_R8(v, 0), S3DSP_R8(v, 8), S3DSP_R8(v, 16), S3DSP_R8(v, 24)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::S3DSP_I8(v, 0),
        S3DSP_I8(v, 8), S3DSP_I8(v, 16), S3DSP_I8(v, 24), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::S3DSP_I8(v, 0), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// values loaded by tmem_ld32, usable only from here on: the compiler sees them
// change after the wait, so no use moves before it
__device__ __forceinline__ void tmem_settle(uint32_t (&v)[32]) {
    asm volatile("" : S3DSP_RW8(v, 0), S3DSP_RW8(v, 8), S3DSP_RW8(v, 16), S3DSP_RW8(v, 24)::"memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::S3DSP_I8(
            v, 0),
        S3DSP_I8(v, 8), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : S3DSP_R8(v, 0) : "r"(taddr) : "memory");
    tmem_wait_ld();
    asm volatile("" : S3DSP_RW8(v, 0)::"memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// the larger of three; NaN if one is
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float exp2_hw(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two-lane f32 arithmetic (sm_100: one instruction for both, each rounded as the scalar one)
struct F2 {
    float x, y;
};
__device__ __forceinline__ F2 fma2v(F2 a, F2 b, F2 c) {
    F2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ F2 add2v(F2 a, F2 b) {
    F2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ F2 both(float v) { return F2{v, v}; }
// (lo, hi) as two 16-bit floats of one register
template <bool kF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if constexpr (kF16)
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

template <int D, bool kF16>
__global__ void __launch_bounds__(Cfg<D>::kRegThreads, 2)
    block_attention_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                           const __grid_constant__ CUtensorMap vmap, const AttnParams p) {
    using C = Cfg<D>;
    constexpr int B = C::kBufs;
    extern __shared__ uint8_t raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    uint8_t* sm = raw + (base - smem_u32(raw));
    const uint32_t sQ = base, sK = sQ + C::kQBytes, sV = sK + C::kKS * C::kPanels * kKPanel;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + C::kTiles);
    const uint32_t q_full = smem_u32(bars), k_full = q_full + 8, k_empty = k_full + 8 * C::kKS,
                   v_full = k_empty + 8 * C::kKS, v_empty = v_full + 8 * C::kVS, s_full = v_empty + 8 * C::kVS,
                   p_full = s_full + 8 * B, o_done = p_full + 8 * B, drained = o_done + 8 * B;
    volatile int* abort_flag = reinterpret_cast<int*>(bars + C::kBars);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + C::kBars) + 1;
    volatile int* n_listed = reinterpret_cast<int*>(bars + C::kBars) + 2;
    volatile int* drain_flag = reinterpret_cast<int*>(bars + C::kBars) + 3;
    int* list = reinterpret_cast<int*>(bars + C::kBars) + 4;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kKeyWarp = 4, kValueWarp = 5;
    if (threadIdx.x == 0) {
        mbar_init(q_full, C::kQTmem ? 4 : 1);
        for (int s = 0; s < C::kKS; ++s) mbar_init(k_full + 8 * s, 1), mbar_init(k_empty + 8 * s, 1);
        for (int s = 0; s < C::kVS; ++s) mbar_init(v_full + 8 * s, 1), mbar_init(v_empty + 8 * s, 1);
        for (int s = 0; s < B; ++s)
            mbar_init(s_full + 8 * s, 1), mbar_init(p_full + 8 * s, 4), mbar_init(o_done + 8 * s, 1);
        mbar_init(drained, 1);
        mbar_init(drained + 8, 1);
        *abort_flag = 0;
        *drain_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (lane == 0) {
        if (warp == kKeyWarp) prefetch_map(&kmap);
        if (warp == kValueWarp) prefetch_map(&vmap);
    }
    pdl_wait();
    const bool split = (int)blockIdx.x < p.split_ctas;
    const int tile = split ? (int)blockIdx.x / p.chunks : (int)blockIdx.x - p.split_ctas;
    const int first = split ? (int)blockIdx.x % p.chunks * p.chunk : 0;
    const bool by_block = p.order && !split;
    const int of = by_block ? p.per_block : split ? p.n_long : p.n_qb;
    const int at_qb = by_block ? p.n_long + tile / of : tile % of;
    const int bq = p.order ? __ldg(p.order + at_qb) : at_qb, h = (by_block ? tile % of : tile / of) * p.pack;
    // the list's first entries and the block's table entry are read together
    const int32_t* sel = p.sel ? p.sel + ((int64_t)bq * p.heads + h) * p.top : nullptr;
    int e = -1;
    if (warp == 0 && lane < p.top) e = __ldg(sel + lane);
    const int4 qb = __ldg(p.q_blocks + bq);
    const int q_row0 = qb.x, q_rows = (qb.y & kAttnRowsMask) * p.pack, k_row0 = qb.z, k_rows = qb.w;
    const int nkb = (k_rows + kK - 1) / kK;
    if (split && !sel && first >= nkb) {
        // a chunk past a short list: nothing to add
        if ((int)threadIdx.x < q_rows) p.part_ml[(int64_t)blockIdx.x * p.tile_rows + threadIdx.x] = make_float2(-INFINITY, 0.f);
        return;
    }
    if (warp == kValueWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                     "r"((uint32_t)C::kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // the softmax threads' rows of Q, on their way while the list is made
    const bool has_row = threadIdx.x < q_rows;
    uint4 q_row[C::kQTmem ? D / 8 : 1];
    if (C::kQTmem && warp < 4) {
        const uint4* src = reinterpret_cast<const uint4*>(
            static_cast<const uint16_t*>(p.q) + (q_row0 + (has_row ? (int)threadIdx.x / p.pack : 0)) * p.q_stride +
            (int64_t)(h + (has_row ? (int)threadIdx.x % p.pack : 0)) * D);
#pragma unroll
        for (int x = 0; x < D / 8; ++x) q_row[x] = has_row ? __ldg(src + x) : make_uint4(0, 0, 0, 0);
    }
    if (warp == 0) {
        // the listed blocks that exist, in list order
        int n = nkb;
        if (sel) {
            n = 0;
            for (int i0 = 0; i0 < p.top; i0 += 32) {
                if (i0 > 0) e = i0 + lane < p.top ? __ldg(sel + i0 + lane) : -1;
                if (e >= nkb) atomicOr(p.status, kErrRowRange);
                const unsigned m = __ballot_sync(0xffffffffu, e >= 0 && e < nkb);
                if (e >= 0 && e < nkb) list[n + __popc(m & ((1u << lane) - 1u))] = e;
                n += __popc(m);
            }
        }
        if (lane == 0) *n_listed = n;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();
    const uint32_t tmem = *tmem_holder;
    const int n = split ? max(0, min(p.chunk, *n_listed - first)) : *n_listed;
    auto block_of = [&](int j) { return p.sel ? list[first + j] : first + j; };
    const int last_block = nkb - 1, last_rows = k_rows - last_block * kK;  // the sequence's last block may be short

    // after a wait gave up: the copies and MMAs that this thread has issued land
    // before shared memory and TMEM are given back
    auto drain = [&](uint32_t full, int ring, int loaded, bool q) {
        if (q) mbar_wait(q_full, 0, drain_flag, p.status);
        for (int j = max(0, loaded - ring); j < loaded; ++j)
            mbar_wait(full + 8 * (j % ring), (j / ring) & 1, drain_flag, p.status);
        mma_commit(drained + 8 * (warp & 1));
        mbar_wait(drained + 8 * (warp & 1), 0, drain_flag, p.status);
    };
    constexpr uint32_t kTileBytes = C::kPanels * kKPanel;
    constexpr uint32_t kFmt = kF16 ? 0u : 1u;
    auto wait = [&](uint32_t bar, uint32_t parity) { return mbar_wait(bar, parity, abort_flag, p.status); };
    if (warp == kKeyWarp) {
        // ================= K tiles, and S = Q K^T =================
        if (n > 0 && elect_one()) {
            constexpr uint32_t kIdesc = (1u << 4) | (kFmt << 7) | (kFmt << 10) | ((kK >> 3) << 17) | ((kQ >> 4) << 24);
            const int kc = (h / p.per_kv) * D;
            int loaded = 0;
            Cursor<C::kKS> ls;  // the next tile's place
            auto load = [&]() {
                const int y = k_row0 + block_of(loaded) * kK;
                mbar_arrive_tx(k_full + 8 * ls.slot, kTileBytes);
                for (int i = 0; i < C::kPanels; ++i)
                    tma_load_2d(sK + ls.slot * kTileBytes + i * kKPanel, &kmap, kc + 64 * i, y, k_full + 8 * ls.slot);
                ls.next();
                ++loaded;
            };
            if constexpr (!C::kQTmem) {
                mbar_arrive_tx(q_full, C::kPanels * kQPanel);
                for (int i = 0; i < C::kPanels; ++i) tma_load_3d(sQ + i * kQPanel, &qmap, 64 * i, h, q_row0, q_full);
            }
            while (loaded < min(n, C::kKS)) load();
            bool ok = wait(q_full, 0);
            tc_fence_after();
            const uint64_t dq = sw128_desc(sQ), dk = sw128_desc(sK);
            Cursor<C::kKS> ks, es;  // the tile, and the oldest one whose place may be free
            Cursor<B> sb, ob;        // the score buffer, and the product that last read it
            for (int j = 0; j < n && ok; ++j, ks.next(), sb.next()) {
                if (j > 0 && loaded < n) {
                    // the tile before this one has been read: another takes its place
                    ok = wait(k_empty + 8 * es.slot, es.parity);
                    es.next();
                    if (ok) load();
                }
                if (j >= B) {
                    ok = ok && wait(o_done + 8 * ob.slot, ob.parity);
                    ob.next();
                }
                ok = ok && wait(k_full + 8 * ks.slot, ks.parity);
                if (!ok) break;
                tc_fence_after();
                const uint64_t dkt = dk + ((ks.slot * kTileBytes) >> 4);
#pragma unroll
                for (int x = 0; x < D / 16; ++x) {
                    const uint64_t b = dkt + (((x / 4) * kKPanel + (x % 4) * 32) >> 4);
                    if constexpr (C::kQTmem)
                        mma_ts(tmem + 64 * sb.slot, tmem + C::kQCol + 8 * x, b, kIdesc, x > 0);
                    else
                        mma_bf16(tmem + 64 * sb.slot, dq + (((x / 4) * kQPanel + (x % 4) * 32) >> 4), b, kIdesc, x > 0);
                }
                mma_commit(s_full + 8 * sb.slot);
                mma_commit(k_empty + 8 * ks.slot);
            }
            if (!ok) drain(k_full, C::kKS, loaded, !C::kQTmem);
        }
        __syncwarp();
    } else if (warp == kValueWarp) {
        // ================= V tiles, and O += P V =================
        if (n > 0 && elect_one()) {
            constexpr uint32_t kIdesc = (1u << 4) | (kFmt << 7) | (kFmt << 10) | (1u << 16) | ((D >> 3) << 17) | ((kQ >> 4) << 24);
            const int kc = (h / p.per_kv) * D;
            int loaded = 0;
            Cursor<C::kVS> ls;
            auto load = [&]() {
                const int y = k_row0 + block_of(loaded) * kK;
                mbar_arrive_tx(v_full + 8 * ls.slot, kTileBytes);
                for (int i = 0; i < C::kPanels; ++i)
                    tma_load_2d(sV + ls.slot * kTileBytes + i * kKPanel, &vmap, kc + 64 * i, y, v_full + 8 * ls.slot);
                ls.next();
                ++loaded;
            };
            while (loaded < min(n, C::kVS)) load();
            const uint64_t dv = mn_desc(sV);
            bool ok = true;
            Cursor<C::kVS> vs, es;
            Cursor<B> pb;
            for (int j = 0; j < n && ok; ++j, vs.next(), pb.next()) {
                if (j > 0 && loaded < n) {
                    ok = wait(v_empty + 8 * es.slot, es.parity);
                    es.next();
                    if (ok) load();
                }
                ok = ok && wait(v_full + 8 * vs.slot, vs.parity) && wait(p_full + 8 * pb.slot, pb.parity);
                if (!ok) break;
                tc_fence_after();
                const uint64_t dvt = dv + ((vs.slot * kTileBytes) >> 4);
#pragma unroll
                for (int x = 0; x < kK / 16; ++x)
                    mma_ts(tmem + C::kOCol, tmem + 64 * pb.slot + 8 * x, dvt + ((x * 2048) >> 4), kIdesc,
                           (j > 0 || x > 0) ? 1u : 0u);
                mma_commit(o_done + 8 * pb.slot);
                mma_commit(v_empty + 8 * vs.slot);
            }
            if (!ok) drain(v_full, C::kVS, loaded, false);
        }
        __syncwarp();
    } else {
        // ================= softmax: thread = query row (TMEM lane) =================
        const int row = threadIdx.x;
        const uint32_t t0 = tmem + ((uint32_t)(32 * warp) << 16);
        const bool live = 32 * warp < q_rows;  // a warp without rows only keeps the barriers' counts
        float m = -INFINITY, l = 0.f, slope = p.c, bias = 0.f;
        bool ok = true;
        // m as the row's maximum (a maximum of -inf weighs its scores of -inf by 0, one of inf or NaN makes the row NaN)
        auto refer = [&](float to) {
            m = to;
            slope = p.c;
            bias = m == -INFINITY ? 0.f : fmaf(-m, p.c, m - m + kShift<kF16>);
            if (fabsf(m) * p.c > kFar && fabsf(m) < INFINITY) {  // without kShift
                auto power = [](float v) { return __uint_as_float(__float_as_uint(v) & 0x7f800000u); };
                slope = fminf(power(p.c), power(0x1p126f / fabsf(m)));
                bias = -m * slope;
            }
        };
        auto wait = [&](uint32_t bar, uint32_t parity) {
            return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.status)) != 0;
        };
        Cursor<B> sb, ob;  // the block's buffer, and that of the product before it
        // V rows of block j that are not the sequence's: zeros (p is 0 there, and 0 * NaN is not)
        auto clear_tail = [&](int j) {
            const int t = j % C::kVS;
            if (!wait(v_full + 8 * t, (j / C::kVS) & 1)) return false;
            for (int x = 0; x < C::kPanels; ++x)
                for (int a = last_rows * 128 + row * 16; a < kKPanel; a += kQ * 16)
                    *reinterpret_cast<uint4*>(sm + (sV - base) + (t * C::kPanels + x) * kKPanel + a) = make_uint4(0, 0, 0, 0);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            return true;
        };
        auto hand_over = [&]() {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * sb.slot);
            ob = sb;
            sb.next();
        };
        if constexpr (C::kQTmem) if (n > 0) {
            // this row of Q into TMEM, two values a column (rows that are not there are never looked at)
            if (live) {
                uint32_t w[32];
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    w[4 * x] = q_row[x].x, w[4 * x + 1] = q_row[x].y, w[4 * x + 2] = q_row[x].z, w[4 * x + 3] = q_row[x].w;
                tmem_st32(t0 + C::kQCol, w);
                tmem_wait_st();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        bool short_block = last_rows < kK && n > 0 && block_of(0) == last_block;
        for (int j = 0; live && j < n; ++j) {
            const uint32_t ts = t0 + 64 * sb.slot;
            ok = wait(s_full + 8 * sb.slot, sb.parity);
            if (!ok) break;
            tc_fence_after();
            uint32_t s[2][32];
            tmem_ld32(ts, s[0]);
            tmem_ld32(ts + 32, s[1]);
            tmem_wait_ld();
            tmem_settle(s[0]);
            tmem_settle(s[1]);
            if (short_block) {
#pragma unroll
                for (int x = 0; x < kK; ++x)
                    if (x >= last_rows) s[x / 32][x % 32] = 0xff800000u;  // -inf
                ok = clear_tail(j);
                if (!ok) break;
            }
            short_block = last_rows < kK && j + 1 < n && block_of(j + 1) == last_block;  // of the next step
            // The weights against the maximum so far, into the scores' first columns, and their sum; the
            // block's own maximum is found along the way. Only where that has grown by more than kSlack
            // does the row take it over: O and l are rescaled and the weights computed again (the scores
            // are still in registers).
            if (j == 0) {
                float mx[4] = {m, m, m, m};
#pragma unroll
                for (int x = 0; x < kK; x += 2)
                    mx[(x / 2) & 3] = max3(mx[(x / 2) & 3], __uint_as_float(s[x / 32][x % 32]), __uint_as_float(s[x / 32][x % 32 + 1]));
                refer(max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]));
            }
            F2 sum[2];
            for (int attempt = 0;; ++attempt) {
                float mx[2] = {m, m};
                sum[0] = sum[1] = both(0.f);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t w[16];
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const F2 sc = {__uint_as_float(s[half][2 * x]), __uint_as_float(s[half][2 * x + 1])};
                        mx[x & 1] = max3(mx[x & 1], sc.x, sc.y);
                        F2 v = fma2v(sc, both(slope), both(bias));
                        v = F2{exp2_hw(v.x), exp2_hw(v.y)};
                        sum[x & 1] = add2v(sum[x & 1], v);
                        w[x] = pack2<kF16>(v.x, v.y);
                    }
                    tmem_st16(ts + 16 * half, w);
                }
                const float mt = max3(mx[0], mx[1], mx[1]);
                // a NaN maximum counts as grown, and stays
                const bool grown = !((mt - m) * p.c <= kSlack) && !(mt == -INFINITY);
                if (attempt > 0 || !__any_sync(0xffffffffu, grown)) break;
                float alpha = 1.f;
                if (grown) {
                    const float from = m, before = bias;
                    refer(mt);
                    const float was = weight_shift<kF16>(from, p.c), is = weight_shift<kF16>(m, p.c);
                    alpha = exp2_hw(was != 0.f && is != 0.f ? bias - before : (from - m) * p.c + (is - was));
                }
                if (j > 0) {
                    ok = wait(o_done + 8 * ob.slot, ob.parity);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 8) {
                        uint32_t o[8];
                        tmem_ld8(t0 + C::kOCol + c0, o);
#pragma unroll
                        for (int x = 0; x < 8; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
                        tmem_st8(t0 + C::kOCol + c0, o);
                    }
                }
                l *= alpha;
            }
            if (!ok) break;
            const F2 total = add2v(sum[0], sum[1]);
            l += total.x + total.y;
            tmem_wait_st();
            hand_over();
        }
        for (int j = 0; !live && j < n && ok; ++j) {
            ok = wait(s_full + 8 * sb.slot, sb.parity);
            if (ok && last_rows < kK && block_of(j) == last_block) ok = clear_tail(j);
            if (ok) hand_over();
        }
        // the last product (they complete in order). A wait tells two neighbouring phases of its
        // barrier apart: with one o_done per buffer the phase before is over when s_full is seen
        if (ok && n > 0) ok = wait(o_done + 8 * ((n - 1) % B), ((n - 1) / B) & 1);
        tc_fence_after();
        if (ok && live) {
            const bool none = l == 0.f;  // nothing listed, or every score -inf
            const float inv = none ? 0.f : 1.f / l;
            const int64_t out_row = q_row0 + row / p.pack;
            const int head = h + row % p.pack;
            const int64_t part = (int64_t)blockIdx.x * p.tile_rows + row;
            // a chunk's sums are handed on against the maximum itself, with 2^kShift
            float exact = 1.f;
            if (split && fabsf(m) < INFINITY)
                exact = exp2_hw(kShift<kF16> - (slope == p.c ? fmaf(m, p.c, bias) : 0.f));
            if (split && row < q_rows) p.part_ml[part] = make_float2(m, l * exact);
            uint16_t* dst = static_cast<uint16_t*>(p.out) + out_row * p.out_stride + (int64_t)head * D;
#pragma unroll
            for (int c0 = 0; c0 < D; c0 += 32) {
                uint32_t o[32];
                if (n > 0) {
                    tmem_ld32(t0 + C::kOCol + c0, o);
                    tmem_wait_ld();
                    tmem_settle(o);
                }
                if (row >= q_rows) continue;
                if (split) {
                    if (n == 0) break;  // m = -inf: never read
                    float4* d4 = reinterpret_cast<float4*>(p.part_o + part * D + c0);
#pragma unroll
                    for (int y = 0; y < 8; ++y)
                        d4[y] = make_float4(__uint_as_float(o[4 * y]) * exact, __uint_as_float(o[4 * y + 1]) * exact,
                                            __uint_as_float(o[4 * y + 2]) * exact, __uint_as_float(o[4 * y + 3]) * exact);
                    continue;
                }
                uint4* d4 = reinterpret_cast<uint4*>(dst + c0);
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    uint32_t w[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        w[x] = none ? 0u
                                    : pack2<kF16>(__uint_as_float(o[8 * y + 2 * x]) * inv,
                                                  __uint_as_float(o[8 * y + 2 * x + 1]) * inv);
                    d4[y] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == kValueWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::kTmemCols));
    }
}

// Joins the chunks of a tile's rows: sums weighed by 2^(c (m_z - max m)). kPer
// warps per row: warp w of them adds chunks w, w + kPer, ..., D / 32 columns per
// lane, and the warps' sums are added in order. A chunk without blocks has
// m = -inf and is not read.
constexpr int kJoinWarps = 8;  // of a CTA
template <int D, bool kF16, int kPer>
__global__ void __launch_bounds__(32 * kJoinWarps) join_chunks_kernel(const AttnParams p) {
    static_assert(kPer == 1 || kPer == kJoinWarps, "a row is a warp's or a CTA's");
    __shared__ float sums[kPer == 1 ? 1 : kJoinWarps][D + 1];
    pdl_wait();
    pdl_trigger();
    constexpr int kC = D / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int at_row = kPer == 1 ? blockIdx.x * kJoinWarps + warp : blockIdx.x;
    const int tile = at_row / p.tile_rows, row = at_row % p.tile_rows;
    if (tile >= p.tiles) return;
    const int64_t step = p.tile_rows, at = (int64_t)tile * p.chunks * step + row;
    // every warp has all chunks' (m, l), chunk 32 i + lane in slot i
    float2 ml[kMaxChunks / 32];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kMaxChunks / 32; ++i) {
        const int z = 32 * i + lane;
        ml[i] = z < p.chunks ? p.part_ml[z * step + at] : make_float2(-INFINITY, 0.f);
    }
    const int at_qb = tile % p.n_long;
    const int4 qb = p.q_blocks[p.order ? p.order[at_qb] : at_qb];
    if (row >= (qb.y & kAttnRowsMask) * p.pack) return;
#pragma unroll
    for (int i = 0; i < kMaxChunks / 32; ++i) top = max3(top, ml[i].x, ml[i].x);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) {
        const float m = __shfl_xor_sync(0xffffffffu, top, x);
        top = max3(top, m, m);
    }
    float acc[kC], l = 0.f;
#pragma unroll
    for (int x = 0; x < kC; ++x) acc[x] = 0.f;
    if (!(top == -INFINITY)) {
#pragma unroll
        for (int i = 0; i < kMaxChunks / 32; ++i) {
            if (32 * i >= p.chunks) break;
            const float wl = ml[i].x == -INFINITY ? 0.f : exp2_hw((ml[i].x - top) * p.c);  // the chunk's weight
            const unsigned some = __ballot_sync(0xffffffffu, !(ml[i].x == -INFINITY));
#pragma unroll 4
            for (int src = kPer == 1 ? 0 : warp; src < min(32, p.chunks - 32 * i); src += kPer) {
                const float w = __shfl_sync(0xffffffffu, wl, src), lz = __shfl_sync(0xffffffffu, ml[i].y, src);
                if (!(some >> src & 1u)) continue;
                l = fmaf(w, lz, l);
                const float* o = p.part_o + ((32 * i + src) * step + at) * D + lane * kC;
#pragma unroll
                for (int x = 0; x < kC; ++x) acc[x] = fmaf(w, __ldg(o + x), acc[x]);
            }
        }
    }
    const int64_t out_row = qb.x + row / p.pack;
    const int head = tile / p.n_long * p.pack + row % p.pack;
    uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + out_row * p.out_stride + (int64_t)head * D);
    if constexpr (kPer == 1) {
        const bool none = l == 0.f;
        const float inv = none ? 0.f : 1.f / l;
#pragma unroll
        for (int x = 0; x < kC; x += 2)
            out[(lane * kC + x) / 2] = none ? 0u : pack2<kF16>(acc[x] * inv, acc[x + 1] * inv);
    } else {
#pragma unroll
        for (int x = 0; x < kC; ++x) sums[warp][lane * kC + x] = acc[x];
        if (lane == 0) sums[warp][D] = l;
        __syncthreads();
        if (threadIdx.x >= D / 2) return;
        float a0 = 0.f, a1 = 0.f;
        l = 0.f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) {
            a0 += sums[w][2 * threadIdx.x];
            a1 += sums[w][2 * threadIdx.x + 1];
            l += sums[w][D];
        }
        const bool none = l == 0.f;
        const float inv = none ? 0.f : 1.f / l;
        out[threadIdx.x] = none ? 0u : pack2<kF16>(a0 * inv, a1 * inv);
    }
}

// [rows][cols] 16-bit rows, tiles of box_rows x 64 columns with the 128-byte swizzle
s3d_status encode_rows(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t stride, int box_rows,
                       bool f16, char* error, uint64_t error_capacity) {
    auto encode = get_encode_fn();
    if (!encode) return fail(error, error_capacity, S3D_INTERNAL_ERROR, "cuTensorMapEncodeTiled unavailable");
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)stride * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult cr = encode(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                               const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (cr != CUDA_SUCCESS)
        return fail(error, error_capacity, S3D_INTERNAL_ERROR, "cuTensorMapEncodeTiled failed (%d)", (int)cr);
    return S3D_OK;
}

// q as [rows][heads][d]: tiles of `pack` heads x kQ / pack rows x 64 columns
s3d_status encode_q(CUtensorMap* map, const void* base, int64_t rows, int heads, int d, int64_t stride, int pack,
                    bool f16, char* error, uint64_t error_capacity) {
    auto encode = get_encode_fn();
    if (!encode) return fail(error, error_capacity, S3D_INTERNAL_ERROR, "cuTensorMapEncodeTiled unavailable");
    const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)rows};
    const cuuint64_t strides[2] = {(cuuint64_t)d * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)pack, (cuuint32_t)(kQ / pack)};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult cr = encode(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                               const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (cr != CUDA_SUCCESS)
        return fail(error, error_capacity, S3D_INTERNAL_ERROR, "cuTensorMapEncodeTiled failed (%d)", (int)cr);
    return S3D_OK;
}

template <int D, bool kF16>
cudaError_t launch(s3dsp_context* ctx, dim3 grid, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                   const AttnParams& p) {
    static std::atomic<uint64_t> optin{0};
    cudaError_t e = smem_optin((const void*)block_attention_kernel<D, kF16>, ctx->device, optin);
    if (e != cudaSuccess) return e;
    e = launch_pdl(block_attention_kernel<D, kF16>, grid, dim3(Cfg<D>::kThreads), Cfg<D>::smem(p.sel ? p.top : 0),
                   ctx->stream, q, k, v, p);
    if (e != cudaSuccess || p.chunks == 1) return e;
    // A CTA per row where they all fit the SMs at once, else a warp per row: 64
    // tiles of 128 rows, 18 chunks: 89 us for the call with a warp, 119 with a CTA;
    // 84 tiles, 3 chunks: 26 and 67.
    const int64_t rows = (int64_t)p.tiles * p.tile_rows;
    const dim3 block(32 * kJoinWarps);
    if (rows <= 8 * (int64_t)ctx->sm_count)
        return launch_pdl(join_chunks_kernel<D, kF16, kJoinWarps>, dim3((unsigned)rows), block, 0, ctx->stream, p);
    return launch_pdl(join_chunks_kernel<D, kF16, 1>, dim3((unsigned)((rows + kJoinWarps - 1) / kJoinWarps)), block, 0,
                      ctx->stream, p);
}

}  // namespace

extern "C" S3DSP_API s3d_status s3dsp_block_attention(s3dsp_context* ctx, const s3dsp_attn_plan* plan, const void* q,
                                                      int64_t q_stride, int32_t heads, const void* k, int64_t k_stride,
                                                      const void* v, int64_t v_stride, int32_t kv_heads,
                                                      uint32_t dtype, int32_t d, float scale, const int32_t* d_sel,
                                                      int32_t top, void* out, int64_t out_stride, char* error,
                                                      uint64_t error_capacity) {
    clear_error(error, error_capacity);
    if (!ctx || !plan) return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "NULL argument");
    if (plan->device != ctx->device)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "the plan is on device %d, the context on %d",
                    plan->device, ctx->device);
    if (dtype != S3DSP_BF16 && dtype != S3DSP_F16)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "dtype %u (bf16 or f16 supported)", dtype);
    if (d != 64 && d != 128)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "head dimension %d (64 or 128 supported)", d);
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads > 4096)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "%d heads over %d key heads", heads, kv_heads);
    const int64_t qw = (int64_t)heads * d, kw = (int64_t)kv_heads * d;
    if (q_stride < qw || out_stride < qw || k_stride < kw || v_stride < kw)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "row stride below heads * d");
    // the tensor maps' row stride: a multiple of 16 bytes below 2^40
    constexpr int64_t kMaxStride = 1ll << 38;
    if ((q_stride | k_stride | v_stride | out_stride) & 7 || q_stride > kMaxStride || k_stride > kMaxStride ||
        v_stride > kMaxStride)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "row strides must be multiples of 8 elements");
    if (!(scale > 0.f) || std::isinf(scale))
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "scale must be positive and finite");
    if (d_sel ? (top < 1 || top > kAttnMaxTop) : top != 0)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "top %d (1 to %d with a selection, else 0)", top,
                    kAttnMaxTop);
    if (plan->n_qb == 0) return S3D_OK;
    if (!q || !out || (plan->n_k > 0 && (!k || !v)))
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "NULL argument");
    if (out == q || out == k || out == v)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "out must not overlap q, k or v");
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "pointers need 16-byte alignment");
    S3DSP_CUDA(cudaSetDevice(ctx->device), "cudaSetDevice");
    const bool f16 = dtype == S3DSP_F16;
    // Heads of a group share a tile where every query block is short enough for
    // it (without a selection, whose lists are each head's own): one pass over
    // K and V and one tile instead of `pack`. The largest power of two that
    // divides the group and fits.
    const int group = heads / kv_heads;
    int pack = 1;
    if (!d_sel)
        while (group % (2 * pack) == 0 && 2 * pack * plan->max_q_rows <= kQ) pack *= 2;
    // Several CTAs share a tile's list in chunks of equal length where the tiles
    // leave half or more of the CTA slots (two per SM) empty, or where a few lists
    // are far longer than the rest: chunks by what the lists hold together, so that
    // they fill the slots about once. Lists of a chunk or less stay whole (with a
    // selection all are taken for long). A chunk has at least kMinChunk blocks, and
    // the split has to save the time of kMinSaved blocks, and of one more per
    // kJoinRows rows of partial sums: a block takes a CTA about 0.7 us (d = 64), the
    // joining kernel about 6 and its traffic. Without and with the split: 8 rows
    // over 92k keys, 4 key heads, 527 and 42 us; 2,000 rows over 20,000, 4 heads, 203
    // and 91; 1,024 over 2,048, 8 heads, 29 and 25; 1,024 over 1,024, 18 and 22 (not
    // split); eight sequences of 1,000 rows, one over 20,000 keys, the others over
    // 100, 257 and 97. Sharing only the tiles of a last, half empty wave was measured
    // too, 720 tiles of 119 blocks: 304 us against 290. A CTA alone on an SM runs
    // 1.2x as fast as one of two.
    const int64_t tiles = (int64_t)plan->n_qb * (heads / pack), slots = 2 * (int64_t)ctx->sm_count;
    if (tiles > 0x3fffffff) return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "too many query blocks times heads");
    const int longest = d_sel && top < plan->max_list ? top : plan->max_list;  // list of a query block, at most
    const int64_t per_block = heads / pack;  // tiles of a query block
    const int64_t work = (d_sel ? (int64_t)plan->n_qb * longest : plan->sum_kb) * per_block;  // blocks in all lists
    int64_t chunk, last = longest;
    if (tiles <= slots / 2) {
        // sum over the lists of ceil(length / chunk) <= (their sum) / chunk + their number
        const int64_t lists = slots / per_block - plan->n_qb;
        chunk = (work / per_block + lists - 1) / (lists > 0 ? lists : 1);
    } else {
        // a few long lists among many: they end within a slot's share of the work, and one chunk more
        chunk = (work + slots - 1) / slots;
        last -= chunk;
    }
    if (chunk < kMinChunk) chunk = kMinChunk;
    if (chunk < (longest + kMaxChunks - 1) / kMaxChunks) chunk = (longest + kMaxChunks - 1) / kMaxChunks;
    // Every split tile has `shares` places, as many as the longest list takes. Where many lists are little
    // longer than a chunk most of these stay empty: chunks are made longer until the places fit
    // kMaxPartBytes (one list of 6,213 blocks beside 83 of 50, d = 128: 10,668 places of 66 KB with chunks
    // of 49 and 219 us, 64 with chunks of 98 and 89 us)
    const int64_t tile_rows = plan->max_q_rows * pack, row_bytes = d * sizeof(float) + sizeof(float2);
    int64_t shares, n_long, split_tiles, all;
    for (;; chunk *= 2) {
        shares = longest > chunk ? (longest + chunk - 1) / chunk : 1;
        n_long = plan->n_qb;  // query blocks whose lists are longer than a chunk
        if (!d_sel) {
            const int4* seq = std::partition_point(plan->by_length, plan->by_length + plan->n_by_length,
                                                   [&](const int4& s) { return s.x > chunk; });
            n_long = seq == plan->by_length ? 0 : seq[-1].y;
        }
        split_tiles = n_long * per_block;
        all = split_tiles * shares;
        if (shares == 1 || all * tile_rows * row_bytes <= kMaxPartBytes) break;
    }
    const int64_t filled = all < work / chunk + split_tiles ? all : work / chunk + split_tiles;
    const bool split = last - chunk >= kMinSaved + filled * tile_rows / kJoinRows;
    CUtensorMap qm, km, vm;
    S3DSP_TRY(encode_q(&qm, q, plan->n_q, heads, d, q_stride, pack, f16, error, error_capacity));
    // a plan without key rows lists nothing: its maps are never read through
    const bool keys = plan->n_k > 0;
    S3DSP_TRY(encode_rows(&km, keys ? k : q, keys ? plan->n_k : 1, kw, k_stride, kK, f16, error, error_capacity));
    S3DSP_TRY(encode_rows(&vm, keys ? v : q, keys ? plan->n_k : 1, kw, v_stride, kK, f16, error, error_capacity));
    AttnParams p = {};
    p.q_blocks = plan->q_blocks;
    p.sel = d_sel;
    p.top = top;
    p.heads = heads;
    p.per_kv = group;
    p.pack = pack;
    p.n_qb = plan->n_qb;
    p.tile_rows = (int)tile_rows;
    // Where the lists' lengths differ, the longest start first, with all their heads, so that short ones
    // fill the end: objects of 15,159, 4,211, 8,190 and 2,777 rows, 16 heads, 1,667 us against 1,800 in the
    // sequences' order, head by head, and 1,775 with the longest of each head first. Equal lengths stay in
    // their order, which reads a head's rows close together (forty objects of 300: 63 against 65).
    if (!d_sel && (split || 4 * (int64_t)longest * plan->n_qb > 5 * plan->sum_kb)) p.order = plan->order;
    p.per_block = (int)per_block;
    p.chunks = 1;
    if (split) {
        p.n_long = (int)n_long;
        p.chunk = (int)chunk;
        p.chunks = (int)shares;
        p.tiles = (int)split_tiles;
        p.split_ctas = (int)all;
    }
    p.c = std::min(scale * 1.4426950408889634f, std::numeric_limits<float>::max());
    p.q = q;
    p.q_stride = q_stride;
    p.out = out;
    p.out_stride = out_stride;
    p.status = ctx->d_status;
    char* parts = nullptr;
    if (split) {
        const size_t rows = (size_t)all * tile_rows;
        S3DSP_CUDA(malloc_async(&parts, rows * row_bytes, ctx->stream), "chunk sums");
        p.part_o = reinterpret_cast<float*>(parts);
        p.part_ml = reinterpret_cast<float2*>(parts + rows * d * sizeof(float));
    }
    const dim3 grid((unsigned)(split ? all + tiles - split_tiles : tiles));
    cudaError_t e = d == 64 ? (f16 ? launch<64, true>(ctx, grid, qm, km, vm, p) : launch<64, false>(ctx, grid, qm, km, vm, p))
                            : (f16 ? launch<128, true>(ctx, grid, qm, km, vm, p)
                                   : launch<128, false>(ctx, grid, qm, km, vm, p));
    if (parts) {
        const cudaError_t f = cudaFreeAsync(parts, ctx->stream);
        if (e == cudaSuccess) e = f;
    }
    if (e != cudaSuccess) return cuda_fail(error, error_capacity, e, "block_attention kernels");
    return S3D_OK;
}

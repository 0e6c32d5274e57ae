// Rotary positions with several axes, and the per-head RMS norm of queries and
// keys with the rotation in the same pass:
//
//   s3dsp_rope          y = R(pos) x for every head
//   s3dsp_qk_norm_rope  y = R(pos) (x / sqrt(mean(x^2) + eps) * gamma) for q and for k
//
// A head's d / 2 pairs are dealt out to the axes in order: axis_pairs[0] pairs
// turn with the first position column, the next axis_pairs[1] with the second
// and so on; pairs left over stay as they are. Pair i of an axis with p pairs
// turns by pos * theta^(-i / p).
//
// One read and one write of the rows: memory bound. A thread owns eight pairs
// of one head at a fixed column (two 16-byte accesses of a 16-bit row) and
// walks over the block's rows, so its norm weights stay in registers; a head
// has G = d / 16 lanes (rounded up to a power of two), and its mean square is a
// shuffle tree of G lanes. The sines and cosines of a row are shared by all its
// heads: the block computes them once into shared memory. An angle is
// pos * (freq / 2 pi) turns in f64 minus the nearest whole turn; only the
// remainder is rounded to f32, because a far position times a fast frequency
// has no f32 bits left for the fraction.
#include <cmath>

#include "s3dsp_internal.h"

using namespace s3dsp;

namespace {

constexpr int kMaxThreads = 256;
constexpr int kMaxPairs = 128;  // head dimension up to 256
constexpr int kMaxAxes = 4;

struct RopeTensor {
    const void* x;
    void* y;
    int64_t xs, ys;      // row strides in elements
    const float* gamma;  // nullptr: ones
    int gamma_stride;    // elements from one head's weights to the next (0: shared)
    int heads;
};

struct RopeParams {
    RopeTensor t[2];  // q, k (heads 0: absent)
    int64_t n;
    int d, lanes;  // lanes per head: d / 16 rounded up to a power of two
    int rows;      // rows per block
    int pairs;     // pairs that turn
    int half;      // pair j is (j, j + d/2) instead of (2j, 2j + 1)
    float eps, sign, inv_d;
    const int32_t* pos;
    int64_t pos_stride;
    double turns[kMaxPairs];  // freq / 2 pi
    uint8_t axis[kMaxPairs];
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
    return __float2bfloat16(v);
}
template <>
__device__ __forceinline__ __half from_f<__half>(float v) {
    return __float2half(v);
}

// two-lane f32 arithmetic (sm_100: one instruction, each lane rounded as the scalar one)
struct F2 {
    float x, y;
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// A lane's sixteen values of a head's row, as it is loaded: kChunks contiguous
// chunks of 16 bytes, chunk k at column k d / kChunks + l kLen of lane l, so that
// the lanes of a head read side by side. Its eight pairs (i = 0 .. 7):
// kHalf: value i of the first eight with value i of the other eight; else
// neighbours. kVec false (rows not 16-byte aligned, or d not a multiple of 16):
// pairs 8l .. 8l + 7, value by value.
template <typename T, bool kVec, bool kHalf>
struct Lane {
    static constexpr int kLen = 16 / (int)sizeof(T), kChunks = 16 / kLen;
    // contiguous pairs, and how many such groups make eight
    static constexpr int kRun = !kVec ? 8 : kHalf ? (kChunks == 2 ? 8 : 4) : kLen / 2, kGroups = 8 / kRun;
    uint4 raw[kChunks];

    // pair i of lane l in a head of np pairs, and the other way round
    static __device__ __forceinline__ int pair(int l, int i, int np) { return i / kRun * (np / kGroups) + l * kRun + i % kRun; }
    static __device__ __forceinline__ void place(int j, int np, int& l, int& i) {
        const int g = kGroups == 1 ? 0 : j / (np / kGroups), in = kGroups == 1 ? j : j - g * (np / kGroups);
        l = in / kRun;
        i = g * kRun + in % kRun;
    }
    __device__ __forceinline__ void load(const T* x, int l, int np) {
        T* e = reinterpret_cast<T*>(raw);
        if constexpr (kVec) {
#pragma unroll
            for (int k = 0; k < kChunks; ++k) raw[k] = *reinterpret_cast<const uint4*>(x + k * (2 * np / kChunks) + l * kLen);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = 8 * l + i;
                e[kHalf ? i : 2 * i] = j < np ? x[kHalf ? j : 2 * j] : from_f<T>(0.f);
                e[kHalf ? 8 + i : 2 * i + 1] = j < np ? x[kHalf ? np + j : 2 * j + 1] : from_f<T>(0.f);
            }
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int k = 0; k < kChunks; ++k) raw[k] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void get(float (&a)[8], float (&b)[8]) const {
        const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = to_f(e[kHalf ? i : 2 * i]), b[i] = to_f(e[kHalf ? 8 + i : 2 * i + 1]);
    }
    // the rotated values to the same places of y
    template <typename TOut>
    static __device__ __forceinline__ void store(TOut* y, int l, int np, const float (&a)[8], const float (&b)[8]) {
        if constexpr (kVec) {
            TOut e[16];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[kHalf ? i : 2 * i] = from_f<TOut>(a[i]), e[kHalf ? 8 + i : 2 * i + 1] = from_f<TOut>(b[i]);
#pragma unroll
            for (int k = 0; k < kChunks; ++k) {
                TOut* p = y + k * (2 * np / kChunks) + l * kLen;
                const TOut* c = e + k * kLen;
                if constexpr (kLen * sizeof(TOut) == 8) {
                    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(c);
                } else {
#pragma unroll
                    for (int w = 0; w < (int)(kLen * sizeof(TOut) / 16); ++w)
                        reinterpret_cast<uint4*>(p)[w] = reinterpret_cast<const uint4*>(c)[w];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = 8 * l + i;
                if (j >= np) break;
                y[kHalf ? j : 2 * j] = from_f<TOut>(a[i]);
                y[kHalf ? np + j : 2 * j + 1] = from_f<TOut>(b[i]);
            }
        }
    }
};

template <typename TIn, typename TOut, bool kVec, bool kHalf, bool kNorm>
__global__ void __launch_bounds__(kMaxThreads, 3) qk_rope_kernel(const __grid_constant__ RopeParams p) {
    using L = Lane<TIn, kVec, kHalf>;
    // a row's cosines and sines: a lane reads its eight pairs as four words (cos, cos, sin, sin) of two,
    // word w of all lanes side by side (no bank conflicts)
    extern __shared__ float4 cs[];  // [rows][4][G]
    pdl_wait();
    pdl_trigger();
    const int G = p.lanes, np = p.d / 2, threads = blockDim.x;
    const int64_t row0 = (int64_t)blockIdx.x * p.rows;
    const int rows = (int)min((int64_t)p.rows, p.n - row0);
    const int l = threadIdx.x & (G - 1);  // this thread's place in its head
    const int heads = p.t[0].heads + p.t[1].heads, step = threads / G;

    bool on = false, is_k = false;
    int h = 0;
    const TIn* x = nullptr;
    TOut* y = nullptr;
    L now, next;  // the next row's values are in flight while this one's are worked on
    auto fetch = [&](int r) {
        if (on && r < rows)
            next.load(x, l, np);
        else
            next.clear();
        x += p.t[is_k].xs;
    };
    // the block's first row of head h0 + this thread's
    auto begin = [&](int h0) {
        h = h0 + threadIdx.x / G;
        on = 8 * l < np && h < heads;
        is_k = h >= p.t[0].heads;
        if (is_k) h -= p.t[0].heads;
        x = static_cast<const TIn*>(p.t[is_k].x) + row0 * p.t[is_k].xs + (int64_t)h * p.d;
        y = static_cast<TOut*>(p.t[is_k].y) + row0 * p.t[is_k].ys + (int64_t)h * p.d;
        fetch(0);
    };
    begin(0);
    for (int e = threadIdx.x; e < rows * np; e += threads) {
        const int r = e / np, j = e - r * np;
        float c = 1.f, s = 0.f;
        if (j < p.pairs) {
            double t = (double)p.pos[(row0 + r) * p.pos_stride + p.axis[j]] * p.turns[j];
            t -= rint(t);
            sincospif((float)(2.0 * t), &s, &c);
        }
        int lane, i;
        L::place(j, np, lane, i);
        float* w = reinterpret_cast<float*>(cs + (r * 4 + i / 2) * G + lane) + (i & 1);
        w[0] = c;
        w[2] = s * p.sign;
    }
    __syncthreads();

    // whole warps run every pass: the shuffles need all lanes
    for (int h0 = 0; h0 < heads; h0 += step) {
        float ga[8], gb[8];
        if constexpr (kNorm) {
            const float* g = p.t[is_k].gamma + (int64_t)h * p.t[is_k].gamma_stride;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = L::pair(l, i, np);
                const bool has = on && p.t[is_k].gamma && j < np;
                ga[i] = has ? __ldg(g + (kHalf ? j : 2 * j)) : 1.f;
                gb[i] = has ? __ldg(g + (kHalf ? np + j : 2 * j + 1)) : 1.f;
            }
        }
#pragma unroll 2
        for (int r = 0; r < rows; ++r, y += p.t[is_k].ys) {
            now = next;
            fetch(r + 1);
            float a[8], b[8];
            now.get(a, b);
            float rs = 1.f;
            if constexpr (kNorm) {
                float s0 = 0.f, s1 = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    s0 = fmaf(a[i], a[i], s0);
                    s1 = fmaf(b[i], b[i], s1);
                }
                float ss = s0 + s1;
                for (int m = G / 2; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
                rs = rsqrtf(ss * p.inv_d + p.eps);
            }
            if (!on) continue;
            const float4* w = cs + r * 4 * G + l;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float4 t4 = w[i / 2 * G];
                F2 c = {t4.x, t4.y}, s = {t4.z, t4.w}, u = {a[i], a[i + 1]}, v = {b[i], b[i + 1]};
                if constexpr (kNorm) {
                    c = mul2(c, F2{rs, rs});
                    s = mul2(s, F2{rs, rs});
                    u = mul2(u, F2{ga[i], ga[i + 1]});
                    v = mul2(v, F2{gb[i], gb[i + 1]});
                }
                const F2 vs = mul2(v, s);
                const F2 p0 = fma2(u, c, F2{-vs.x, -vs.y}), p1 = fma2(u, s, mul2(v, c));
                a[i] = p0.x, a[i + 1] = p0.y;
                b[i] = p1.x, b[i + 1] = p1.y;
            }
            L::store(y, l, np, a, b);
        }
        if (h0 + step < heads) begin(h0 + step);
    }
}

template <typename TIn, typename TOut, bool kNorm>
cudaError_t launch_typed(const s3dsp_context* ctx, RopeParams& p, bool vec) {
    // as many threads as the lanes of a row's heads need, in passes of equal size
    const int lanes = (p.t[0].heads + p.t[1].heads) * p.lanes, passes = (lanes + kMaxThreads - 1) / kMaxThreads;
    const unsigned threads = (unsigned)((lanes + passes - 1) / passes + 31) / 32 * 32;
    // rows per block: eight share one column's norm weights; fewer when the blocks would not fill the
    // SMs with the 24 warps that their registers take
    const int64_t fill = p.n * threads / ((int64_t)ctx->sm_count * 768);
    p.rows = fill >= 8 ? 8 : fill >= 4 ? 4 : fill >= 2 ? 2 : 1;
    const dim3 grid((unsigned)((p.n + p.rows - 1) / p.rows));
    const size_t smem = (size_t)p.rows * 4 * p.lanes * sizeof(float4);
    auto go = [&](auto kernel) { return launch_pdl(kernel, grid, dim3(threads), smem, ctx->stream, p); };
    if (vec)
        return p.half ? go(qk_rope_kernel<TIn, TOut, true, true, kNorm>) : go(qk_rope_kernel<TIn, TOut, true, false, kNorm>);
    return p.half ? go(qk_rope_kernel<TIn, TOut, false, true, kNorm>) : go(qk_rope_kernel<TIn, TOut, false, false, kNorm>);
}
template <typename TIn, bool kNorm>
cudaError_t launch_in(const s3dsp_context* ctx, RopeParams& p, uint32_t yd, bool vec) {
    if (yd == S3DSP_F32) return launch_typed<TIn, float, kNorm>(ctx, p, vec);
    if (yd == S3DSP_BF16) return launch_typed<TIn, __nv_bfloat16, kNorm>(ctx, p, vec);
    return launch_typed<TIn, __half, kNorm>(ctx, p, vec);
}
template <bool kNorm>
cudaError_t launch(const s3dsp_context* ctx, RopeParams& p, uint32_t xd, uint32_t yd, bool vec) {
    if (xd == S3DSP_F32) return launch_in<float, kNorm>(ctx, p, yd, vec);
    if (xd == S3DSP_BF16) return launch_in<__nv_bfloat16, kNorm>(ctx, p, yd, vec);
    return launch_in<__half, kNorm>(ctx, p, yd, vec);
}

// shape, positions and frequencies common to both entry points
s3d_status fill_params(RopeParams& p, int64_t n, int32_t d, const int32_t* d_pos,
                       int64_t pos_stride, int32_t axes, const int32_t* axis_pairs, double theta, uint32_t flags,
                       char* error, uint64_t error_capacity) {
    if (n < 0 || n > (1ll << 31) - 1)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "row count %lld out of range", (long long)n);
    if (d <= 0 || d % 8 || d > 2 * kMaxPairs)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "head dimension %d (a multiple of 8 up to %d)", d,
                    2 * kMaxPairs);
    if (axes < 0 || axes > kMaxAxes || (axes > 0 && !axis_pairs))
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "%d axes (0 to %d, with axis_pairs)", axes, kMaxAxes);
    if (axes > 0 && n > 0 && (!d_pos || pos_stride < axes))
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "positions missing, or a row stride below the axes");
    if (axes > 0 && !(theta > 0.0 && std::isfinite(theta)))
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "theta must be positive and finite");
    p.n = n;
    p.d = d;
    p.lanes = 1;
    while (p.lanes * 16 < d) p.lanes *= 2;
    p.inv_d = 1.0f / (float)d;
    p.half = (flags & S3DSP_ROPE_HALF) ? 1 : 0;
    p.sign = (flags & S3DSP_ROPE_INVERSE) ? -1.f : 1.f;
    p.pos = d_pos;
    p.pos_stride = pos_stride;
    p.pairs = 0;
    for (int a = 0; a < axes; ++a) {
        if (axis_pairs[a] < 0 || axis_pairs[a] > d / 2 - p.pairs)
            return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "axis_pairs exceed the head's %d pairs", d / 2);
        for (int i = 0; i < axis_pairs[a]; ++i) {
            p.turns[p.pairs] = pow(theta, -(double)i / axis_pairs[a]) / 6.283185307179586476925;
            p.axis[p.pairs++] = (uint8_t)a;
        }
    }
    return S3D_OK;
}

// one tensor's pointers and strides; clears *vec unless its rows take 16-byte accesses
s3d_status fill_tensor(RopeTensor& t, const void* x, uint32_t xd, int64_t xs, void* y, uint32_t yd, int64_t ys,
                       int32_t heads, int32_t d, const char* name, bool* vec, char* error, uint64_t error_capacity) {
    if (!x || !y) return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "%s: NULL argument", name);
    if (heads <= 0 || heads > 65536) return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "%s: bad head count", name);
    const int64_t w = (int64_t)heads * d;
    if (xs < w || ys < w)
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "%s: row stride below heads * d = %lld", name, (long long)w);
    if (x == y && (xs != ys || xd != yd))
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT,
                    "%s: in place needs the same type and row stride", name);
    const size_t xe = dtype_size(xd), ye = dtype_size(yd);
    if (((uintptr_t)x & (xe - 1)) || ((uintptr_t)y & (ye - 1)))
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "%s: pointer not aligned to its type", name);
    if (((uintptr_t)x | (uintptr_t)y | (xs * xe) | (ys * ye)) & 15 || d % 16) *vec = false;
    t = RopeTensor{x, y, xs, ys, nullptr, 0, heads};
    return S3D_OK;
}

}  // namespace

extern "C" S3DSP_API s3d_status s3dsp_rope(s3dsp_context* ctx, const void* x, uint32_t x_dtype, int64_t n,
                                           int64_t x_stride, int32_t heads, int32_t d, const int32_t* d_pos,
                                           int64_t pos_stride, int32_t axes, const int32_t* axis_pairs, double theta,
                                           uint32_t flags, void* y, uint32_t y_dtype, int64_t y_stride, char* error,
                                           uint64_t error_capacity) {
    clear_error(error, error_capacity);
    if (!ctx) return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "ctx is NULL");
    if (!dtype_ok(x_dtype) || !dtype_ok(y_dtype)) return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "bad dtype");
    if (flags & ~(S3DSP_ROPE_HALF | S3DSP_ROPE_INVERSE))
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "unknown flags 0x%x", flags);
    RopeParams p = {};
    bool vec = true;
    S3DSP_TRY(fill_params(p, n, d, d_pos, pos_stride, axes, axis_pairs, theta, flags, error, error_capacity));
    if (n == 0) return S3D_OK;
    S3DSP_TRY(fill_tensor(p.t[0], x, x_dtype, x_stride, y, y_dtype, y_stride, heads, d, "x", &vec, error, error_capacity));
    S3DSP_CUDA(cudaSetDevice(ctx->device), "cudaSetDevice");
    S3DSP_CUDA(launch<false>(ctx, p, x_dtype, y_dtype, vec), "qk_rope_kernel");
    return S3D_OK;
}

extern "C" S3DSP_API s3d_status s3dsp_qk_norm_rope(
    s3dsp_context* ctx, const void* q, int64_t q_stride, int32_t heads, const float* q_gamma, const void* k,
    int64_t k_stride, int32_t kv_heads, const float* k_gamma, uint32_t x_dtype, int64_t n, int32_t d, float eps,
    const int32_t* d_pos, int64_t pos_stride, int32_t axes, const int32_t* axis_pairs, double theta, uint32_t flags,
    void* q_out, int64_t q_out_stride, void* k_out, int64_t k_out_stride, uint32_t y_dtype, char* error,
    uint64_t error_capacity) {
    clear_error(error, error_capacity);
    if (!ctx) return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "ctx is NULL");
    if (!dtype_ok(x_dtype) || !dtype_ok(y_dtype)) return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "bad dtype");
    if (flags & ~(S3DSP_ROPE_HALF | S3DSP_QK_GAMMA_SHARED))
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "unknown flags 0x%x", flags);
    if (!(eps >= 0.f) || std::isinf(eps)) return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "bad eps");
    if (!k && (kv_heads != 0 || k_out))
        return fail(error, error_capacity, S3D_INVALID_ARGUMENT, "no k: kv_heads must be 0 and k_out NULL");
    RopeParams p = {};
    bool vec = true;
    S3DSP_TRY(fill_params(p, n, d, d_pos, pos_stride, axes, axis_pairs, theta, flags, error, error_capacity));
    if (n == 0) return S3D_OK;
    S3DSP_TRY(fill_tensor(p.t[0], q, x_dtype, q_stride, q_out, y_dtype, q_out_stride, heads, d, "q", &vec, error,
                          error_capacity));
    if (k)
        S3DSP_TRY(fill_tensor(p.t[1], k, x_dtype, k_stride, k_out, y_dtype, k_out_stride, kv_heads, d, "k", &vec, error,
                              error_capacity));
    p.eps = eps;
    p.t[0].gamma = q_gamma;
    p.t[1].gamma = k_gamma;
    p.t[0].gamma_stride = p.t[1].gamma_stride = (flags & S3DSP_QK_GAMMA_SHARED) ? 0 : d;
    S3DSP_CUDA(cudaSetDevice(ctx->device), "cudaSetDevice");
    S3DSP_CUDA(launch<true>(ctx, p, x_dtype, y_dtype, vec), "qk_rope_kernel");
    return S3D_OK;
}

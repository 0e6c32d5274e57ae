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
// One read and one write of the rows: memory bound. A thread owns four pairs
// (eight values, 16 bytes of a 16-bit row) of one head at a fixed column and
// walks over the block's rows, so its eight norm weights stay in registers;
// the 32 lanes of a warp hold 32 / G heads of G = d / 8 (rounded up to a power
// of two) lanes each, and the mean square is a shuffle tree of G lanes. The
// sines and cosines of a row are shared by all its heads: the block computes
// them once into shared memory. An angle is pos * (freq / 2 pi) turns in f64
// minus the nearest whole turn; only the remainder is rounded to f32, because
// a far position times a fast frequency has no f32 bits left for the fraction.
#include <cmath>

#include "s3dsp_internal.h"

using namespace s3dsp;

namespace {

constexpr int kThreads = 256;
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
    int d, lanes;  // lanes per head: d / 8 rounded up to a power of two
    int rows;      // rows per block
    int pairs;     // pairs that turn
    int half;      // pair j is (j, j + d/2) instead of (2j, 2j + 1)
    float eps, sign;
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

// four consecutive values at p; kVec: p is aligned to four values
template <typename T, bool kVec>
__device__ __forceinline__ void load4(const T* p, float (&f)[4]) {
    if constexpr (!kVec) {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = to_f(p[j]);
    } else if constexpr (sizeof(T) == 4) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
    } else {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = to_f(e[j]);
    }
}
template <typename T, bool kVec>
__device__ __forceinline__ void store4(T* p, const float (&f)[4]) {
    if constexpr (!kVec) {
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = from_f<T>(f[j]);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
        uint2 u;
        T* e = reinterpret_cast<T*>(&u);
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = from_f<T>(f[j]);
        *reinterpret_cast<uint2*>(p) = u;
    }
}

template <typename TIn, typename TOut, bool kVec, bool kNorm>
__global__ void __launch_bounds__(kThreads) qk_rope_kernel(const __grid_constant__ RopeParams p) {
    extern __shared__ float2 cs[];  // [rows][d / 2] (cos, sin)
    pdl_wait();
    pdl_trigger();
    const int64_t row0 = (int64_t)blockIdx.x * p.rows;
    const int rows = (int)min((int64_t)p.rows, p.n - row0);
    const int np = p.d / 2;
    for (int e = threadIdx.x; e < rows * np; e += kThreads) {
        const int r = e / np, j = e - r * np;
        float c = 1.f, s = 0.f;
        if (j < p.pairs) {
            double t = (double)p.pos[(row0 + r) * p.pos_stride + p.axis[j]] * p.turns[j];
            t -= rint(t);
            sincospif((float)(2.0 * t), &s, &c);
        }
        cs[e] = make_float2(c, s * p.sign);
    }
    __syncthreads();

    const int G = p.lanes;
    const int l = threadIdx.x & (G - 1);  // this thread's place in its head: pairs 4l .. 4l + 3
    const bool live = 8 * l < p.d;
    // elements of the two halves of this thread's eight values
    const int o0 = p.half ? 4 * l : 8 * l, o1 = p.half ? np + 4 * l : 8 * l + 4;
    const int heads = p.t[0].heads + p.t[1].heads;
    const int step = kThreads / G;
    // whole warps run every pass: the shuffles need all lanes
    for (int h0 = 0; h0 < heads; h0 += step) {
        const int hh = h0 + threadIdx.x / G;
        const bool k = hh >= p.t[0].heads;
        const RopeTensor& t = p.t[k ? 1 : 0];
        const int h = k ? hh - p.t[0].heads : hh;
        const bool on = live && hh < heads;
        const TIn* x = static_cast<const TIn*>(t.x) + row0 * t.xs + (int64_t)h * p.d;
        TOut* y = static_cast<TOut*>(t.y) + row0 * t.ys + (int64_t)h * p.d;
        float g0[4], g1[4];
        if constexpr (kNorm) {
#pragma unroll
            for (int j = 0; j < 4; ++j) g0[j] = g1[j] = 1.f;
            if (on && t.gamma) {
                const float* g = t.gamma + (int64_t)h * t.gamma_stride;
#pragma unroll
                for (int j = 0; j < 4; ++j) g0[j] = __ldg(g + o0 + j), g1[j] = __ldg(g + o1 + j);
            }
        }
        constexpr int U = 4;  // rows in flight
        for (int r0 = 0; r0 < rows; r0 += U) {
            float a[U][4], b[U][4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (on && r0 + u < rows) {
                    load4<TIn, kVec>(x + (r0 + u) * t.xs + o0, a[u]);
                    load4<TIn, kVec>(x + (r0 + u) * t.xs + o1, b[u]);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) a[u][j] = b[u][j] = 0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = r0 + u;
                if constexpr (kNorm) {
                    float ss = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) ss = fmaf(a[u][j], a[u][j], fmaf(b[u][j], b[u][j], ss));
                    for (int m = G / 2; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
                    const float rs = 1.0f / sqrtf(ss / (float)p.d + p.eps);
#pragma unroll
                    for (int j = 0; j < 4; ++j) a[u][j] *= rs * g0[j], b[u][j] *= rs * g1[j];
                }
                if (!on || r >= rows) continue;
                float f0[4], f1[4];
                const float2* w = cs + r * np + 4 * l;
                if (p.half) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        f0[j] = a[u][j] * w[j].x - b[u][j] * w[j].y;
                        f1[j] = a[u][j] * w[j].y + b[u][j] * w[j].x;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        f0[2 * j] = a[u][2 * j] * w[j].x - a[u][2 * j + 1] * w[j].y;
                        f0[2 * j + 1] = a[u][2 * j] * w[j].y + a[u][2 * j + 1] * w[j].x;
                        f1[2 * j] = b[u][2 * j] * w[2 + j].x - b[u][2 * j + 1] * w[2 + j].y;
                        f1[2 * j + 1] = b[u][2 * j] * w[2 + j].y + b[u][2 * j + 1] * w[2 + j].x;
                    }
                }
                store4<TOut, kVec>(y + r * t.ys + o0, f0);
                store4<TOut, kVec>(y + r * t.ys + o1, f1);
            }
        }
    }
}

template <typename TIn, typename TOut, bool kNorm>
cudaError_t launch_typed(const s3dsp_context* ctx, const RopeParams& p, bool vec) {
    const dim3 grid((unsigned)((p.n + p.rows - 1) / p.rows));
    const size_t smem = (size_t)p.rows * (p.d / 2) * sizeof(float2);
    return vec ? launch_pdl(qk_rope_kernel<TIn, TOut, true, kNorm>, grid, dim3(kThreads), smem, ctx->stream, p)
               : launch_pdl(qk_rope_kernel<TIn, TOut, false, kNorm>, grid, dim3(kThreads), smem, ctx->stream, p);
}
template <typename TIn, bool kNorm>
cudaError_t launch_in(const s3dsp_context* ctx, const RopeParams& p, uint32_t yd, bool vec) {
    if (yd == S3DSP_F32) return launch_typed<TIn, float, kNorm>(ctx, p, vec);
    if (yd == S3DSP_BF16) return launch_typed<TIn, __nv_bfloat16, kNorm>(ctx, p, vec);
    return launch_typed<TIn, __half, kNorm>(ctx, p, vec);
}
template <bool kNorm>
cudaError_t launch(const s3dsp_context* ctx, const RopeParams& p, uint32_t xd, uint32_t yd, bool vec) {
    if (xd == S3DSP_F32) return launch_in<float, kNorm>(ctx, p, yd, vec);
    if (xd == S3DSP_BF16) return launch_in<__nv_bfloat16, kNorm>(ctx, p, yd, vec);
    return launch_in<__half, kNorm>(ctx, p, yd, vec);
}

// rows per block: eight share one column's norm weights; fewer when that would leave SMs without a block
int rows_per_block(const s3dsp_context* ctx, int64_t n) {
    const int64_t fill = n / ((int64_t)ctx->sm_count * 4);
    return fill >= 8 ? 8 : fill >= 4 ? 4 : fill >= 2 ? 2 : 1;
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
    while (p.lanes * 8 < d) p.lanes *= 2;
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
    if (((uintptr_t)x | (uintptr_t)y | (xs * xe) | (ys * ye)) & 15) *vec = false;
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
    p.rows = rows_per_block(ctx, n);
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
    p.rows = rows_per_block(ctx, n);
    S3DSP_CUDA(cudaSetDevice(ctx->device), "cudaSetDevice");
    S3DSP_CUDA(launch<true>(ctx, p, x_dtype, y_dtype, vec), "qk_rope_kernel");
    return S3D_OK;
}

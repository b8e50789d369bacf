// radzero_hip — the norms before and after a block, fused with its gate, its residual scale and the residual sum.
//
//   t  = post_norm(y)                       (or y)
//   r' = alpha r + scale[c] gate[row][c] t  (either factor may be absent)
//   x  = pre_norm(r')                       (the next block's operand)
//   norm(a) = (a - mean a) / sqrt(mean (a - mean a)^2 + eps) * w + b       LayerNorm
//           = a / sqrt(mean a^2 + eps) * w + b                             root-mean-square norm
//
// Bound by HBM: y and r are read once, r' and x written once, everything between stays in the registers of the threads that own a row.
// Statistics are taken in fp32 from those registers in two passes (mean first, then the squares of the differences): a sum of squares minus
// a squared mean would lose a row whose mean is large against its spread.
#include "rz_common.h"
#include "rz_kernels.h"

namespace rz {

namespace {

constexpr int kVec = 4;           // columns per chunk: 768 = 3 chunks per lane of a wave, no lane idle

// rows need no alignment beyond their element's: odd widths put every second row off 16 bytes, and the hardware takes such vector accesses
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Loose4 { T v[4]; };

template <typename T> __device__ __forceinline__ void load4(const T* p, int col, int dim, float (&v)[4]) {
    if (col + 4 <= dim) {
        const Loose4<T> x = *reinterpret_cast<const Loose4<T>*>(p + col);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = to_f32(x.v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = col + e < dim ? to_f32(p[col + e]) : 0.f;
    }
}
template <typename T> __device__ __forceinline__ void store4(T* p, int col, int dim, const float (&v)[4]) {
    if (col + 4 <= dim) {
        Loose4<T> x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x.v[e] = from_f32<T>(v[e]);
        *reinterpret_cast<Loose4<T>*>(p + col) = x;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < dim) p[col + e] = from_f32<T>(v[e]);
    }
}

// sum over the threads of a row: one wave, or a whole workgroup of TPR / 64 waves
template <int TPR> __device__ __forceinline__ float row_sum(float v, float* lds) {
    v = wave_sum(v);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        __syncthreads();                                  // the previous sum's readers are done
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += lds[w];
    }
    return v;
}

// one norm of the row in v[NC][4]; columns behind dim hold 0 and are kept at 0 through the statistics
template <int TPR, int NC>
__device__ __forceinline__ void norm_row(float (&v)[NC][4], int kind, const float* w, const float* b, float eps, int lane, int dim, float* lds) {
    const float inv = 1.0f / (float)dim;
    if (kind == RZ_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NC; ++j) s += (v[j][0] + v[j][1]) + (v[j][2] + v[j][3]);
        const float mean = row_sum<TPR>(s, lds) * inv;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int col = (lane + j * TPR) * kVec;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = col + e < dim ? v[j][e] - mean : 0.f;
        }
    }
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) q = fmaf(v[j][e], v[j][e], q);
    const float r = 1.0f / sqrtf(row_sum<TPR>(q, lds) * inv + eps);
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        const int col = (lane + j * TPR) * kVec;
        if (col < dim) {
            float g[4] = {1.f, 1.f, 1.f, 1.f}, h[4] = {0.f, 0.f, 0.f, 0.f};
            if (w) load4(w, col, dim, g);
            if (b) load4(b, col, dim, h);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = fmaf(v[j][e] * r, g[e], h[e]);
        }
    }
}

template <typename T, typename RT, int TPR, int NC>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void residual_norm_kernel(const rz_residual_norm_args a, int64_t total_rows) {
    __shared__ float lds[TPR > 64 ? TPR / 64 : 1];
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1;        // rows per workgroup
    const int lane = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    if (row >= total_rows) return;                        // whole waves, and never a part of a workgroup that shares a row
    const int64_t b = row / a.rows, n = row - b * a.rows;
    const int dim = a.dim;

    float v[NC][4];
    if (a.y_dev) {
        const T* y = (const T*)a.y_dev + b * a.y_batch_stride + n * a.y_row_stride;
#pragma unroll
        for (int j = 0; j < NC; ++j) load4(y, (lane + j * TPR) * kVec, dim, v[j]);
    }
    float h[NC][4];
    {
        const RT* r = (const RT*)a.resid_dev + b * a.resid_batch_stride + n * a.resid_row_stride;
#pragma unroll
        for (int j = 0; j < NC; ++j) load4(r, (lane + j * TPR) * kVec, dim, h[j]);
    }
    if (a.y_dev) {
        if (a.post_kind) norm_row<TPR, NC>(v, a.post_kind, a.post_weight_dev, a.post_bias_dev, a.post_eps, lane, dim, lds);
        const float* gate = a.gate_dev ? a.gate_dev + b * a.gate_batch_stride + n * a.gate_row_stride : nullptr;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int col = (lane + j * TPR) * kVec;
            if (col >= dim) continue;
            float f[4] = {1.f, 1.f, 1.f, 1.f}, g[4] = {1.f, 1.f, 1.f, 1.f};
            if (a.scale_dev) load4(a.scale_dev, col, dim, f);
            if (gate) load4(gate, col, dim, g);
#pragma unroll
            for (int e = 0; e < 4; ++e) h[j][e] = fmaf(a.alpha, h[j][e], f[e] * g[e] * v[j][e]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) h[j][e] *= a.alpha;
    }
    if (a.resid_out_dev) {
        RT* r = (RT*)a.resid_out_dev + b * a.resid_out_batch_stride + n * a.resid_out_row_stride;
#pragma unroll
        for (int j = 0; j < NC; ++j) store4(r, (lane + j * TPR) * kVec, dim, h[j]);
    }
    if (!a.out_dev) return;
    if (a.pre_kind) norm_row<TPR, NC>(h, a.pre_kind, a.pre_weight_dev, a.pre_bias_dev, a.pre_eps, lane, dim, lds);
    T* o = (T*)a.out_dev + b * a.out_batch_stride + n * a.out_row_stride;
#pragma unroll
    for (int j = 0; j < NC; ++j) store4(o, (lane + j * TPR) * kVec, dim, h[j]);
}

template <typename T, typename RT> hipError_t launch(const rz_residual_norm_args& a, hipStream_t s) {
    const int64_t rows = (int64_t)a.batch * a.rows;
    const int chunks = (a.dim + kVec - 1) / kVec;
    // the fewest threads whose registers hold the row: one wave per row needs no LDS and no barrier
#define RZ_ROWS(TPR, NC)                                                                                                        \
    if (chunks <= TPR * NC) {                                                                                                   \
        constexpr int kBlock = TPR < 256 ? 256 : TPR, kRpb = kBlock / TPR;                                                      \
        hipLaunchKernelGGL((residual_norm_kernel<T, RT, TPR, NC>), dim3((unsigned)((rows + kRpb - 1) / kRpb)), dim3(kBlock), 0, s, a, rows); \
        return hipGetLastError();                                                                                               \
    }
    RZ_ROWS(64, 1) RZ_ROWS(64, 2) RZ_ROWS(64, 3) RZ_ROWS(64, 4) RZ_ROWS(256, 2) RZ_ROWS(256, 4) RZ_ROWS(256, 8) RZ_ROWS(1024, 4)
#undef RZ_ROWS
    return hipErrorInvalidValue;                          // api.hip refuses dim > RZ_NORM_MAX_DIM before
}

}  // namespace

hipError_t launch_residual_norm(const rz_residual_norm_args& a, hipStream_t s) {
    const bool rf = a.resid_dtype == DT_F32;
    if (a.dtype == DT_F32) return launch<float, float>(a, s);
    if (a.dtype == DT_BF16) return rf ? launch<bf16_t, float>(a, s) : launch<bf16_t, bf16_t>(a, s);
    return rf ? launch<f16_t, float>(a, s) : launch<f16_t, f16_t>(a, s);
}

}  // namespace rz

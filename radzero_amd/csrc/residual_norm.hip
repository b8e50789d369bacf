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
// a squared mean would lose a row whose mean is large against its spread.  32 x 5330 rows of 768 (bf16 y, fp32 residual): 290 us, 5.4 TB/s;
// 8 x 1370 rows of 1001 (f16): 18.9 us, 4.7 TB/s; a few rows: the launch.  Tried and left: the vectors kept in registers over several rows of
// a wave, the next row prefetched (418 us: 193 registers, two waves a SIMD), loads past the caches (no change; 25 us at the odd width, where
// two rows share a line).
#include <algorithm>

#include "rz_common.h"
#include "rz_kernels.h"

namespace rz {

namespace {

constexpr int kMostBlocks = 1 << 20;   // workgroups of a launch: a launch takes less than 2^32 threads
constexpr int kVec = 4;           // columns per chunk: 768 = 3 chunks per lane of a wave, no lane idle

// rows need no alignment beyond their element's: odd widths put every second row off 16 bytes, and the hardware takes such vector accesses
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Loose4 { T v[4]; };

// Chunks of a row that no width this form takes cuts short: the launcher takes the fewest threads and chunks that hold the row.
template <int TPR, int NC> constexpr int kWhole = TPR <= 64 ? NC - 1 : NC / 2;

// A thread's columns of a row as they lie in memory.  Loads and conversions are apart, so that all of a row's loads are in flight before the first is waited for.
template <typename T, int TPR, int NC> struct Raw {
    Loose4<T> x[NC];
    __device__ __forceinline__ void load(const T* p, int lane, int dim) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int col = (lane + j * TPR) * kVec;
            if (j < kWhole<TPR, NC> || col + kVec <= dim) x[j] = *reinterpret_cast<const Loose4<T>*>(p + col);
            else
#pragma unroll
                for (int e = 0; e < kVec; ++e) x[j].v[e] = col + e < dim ? p[col + e] : from_f32<T>(0.f);
        }
    }
    __device__ __forceinline__ void get(float (&v)[NC][4]) const {
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int e = 0; e < kVec; ++e) v[j][e] = to_f32(x[j].v[e]);
    }
};
template <bool STREAM, typename T> __device__ __forceinline__ void store4(T* p, int col, int dim, const float (&v)[4], bool whole) {
    T x[kVec];
#pragma unroll
    for (int e = 0; e < kVec; ++e) x[e] = from_f32<T>(v[e]);
    if (whole || col + kVec <= dim) {
        typedef T V __attribute__((ext_vector_type(kVec), aligned(sizeof(T))));
        const V w = {x[0], x[1], x[2], x[3]};
        if constexpr (STREAM) __builtin_nontemporal_store(w, reinterpret_cast<V*>(p + col));
        else *reinterpret_cast<V*>(p + col) = w;
    } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e)
            if (col + e < dim) p[col + e] = x[e];
    }
}

// sum over the threads of a row: some neighbours of a wave, all of it, or a whole workgroup of TPR / 64 waves
template <int TPR> __device__ __forceinline__ float row_sum(float v, float* lds) {
#pragma unroll
    for (int o = min(TPR, 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
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

// a thread's columns of a vector that may be absent
template <int TPR, int NC> struct Vector {
    float v[NC][4];
    __device__ __forceinline__ void load(const float* p, float otherwise, int lane, int dim) {
        if (p) {
            Raw<float, TPR, NC> x;
            x.load(p, lane, dim);
            x.get(v);
        } else
#pragma unroll
            for (int j = 0; j < NC; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[j][e] = otherwise;
    }
};

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
    Vector<TPR, NC> g, h;
    g.load(w, 1.f, lane, dim);
    h.load(b, 0.f, lane, dim);
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[j][e] = fmaf(v[j][e] * r, g.v[j][e], h.v[j][e]);
}

template <typename T, typename RT, int TPR, int NC, bool STREAM>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void residual_norm_kernel(const rz_residual_norm_args a, int from_row, int total_rows) {
    __shared__ float lds[TPR > 64 ? TPR / 64 : 1];
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1, WHOLE = kWhole<TPR, NC>;       // rows per workgroup
    const int lane = threadIdx.x % TPR, dim = a.dim;
    const int group = threadIdx.x / TPR;
    const int64_t first = from_row + (int64_t)blockIdx.x * RPB + (TPR >= 64 ? __builtin_amdgcn_readfirstlane(group) : group);
    if (first >= total_rows) return;                      // all threads of a row, and never a part of a workgroup that shares one
    const unsigned row = (unsigned)first, batch = row / (unsigned)a.rows;
    const int64_t b = batch, n = row - batch * (unsigned)a.rows;

    Raw<T, TPR, NC> y;
    if (a.y_dev) y.load((const T*)a.y_dev + b * a.y_batch_stride + n * a.y_row_stride, lane, dim);
    Raw<RT, TPR, NC> r;
    r.load((const RT*)a.resid_dev + b * a.resid_batch_stride + n * a.resid_row_stride, lane, dim);

    float h[NC][4];
    if (a.y_dev) {
        float v[NC][4];
        y.get(v);
        if (a.post_kind) norm_row<TPR, NC>(v, a.post_kind, a.post_weight_dev, a.post_bias_dev, a.post_eps, lane, dim, lds);
        Vector<TPR, NC> f, g;
        f.load(a.scale_dev, 1.f, lane, dim);
        g.load(a.gate_dev ? a.gate_dev + b * a.gate_batch_stride + n * a.gate_row_stride : nullptr, 1.f, lane, dim);
        r.get(h);
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) h[j][e] = fmaf(a.alpha, h[j][e], f.v[j][e] * g.v[j][e] * v[j][e]);
    } else {
        r.get(h);
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) h[j][e] *= a.alpha;
    }
    if (a.resid_out_dev) {
        RT* o = (RT*)a.resid_out_dev + b * a.resid_out_batch_stride + n * a.resid_out_row_stride;
#pragma unroll
        for (int j = 0; j < NC; ++j) store4<STREAM>(o, (lane + j * TPR) * kVec, dim, h[j], j < WHOLE);
    }
    if (!a.out_dev) return;
    if (a.pre_kind) norm_row<TPR, NC>(h, a.pre_kind, a.pre_weight_dev, a.pre_bias_dev, a.pre_eps, lane, dim, lds);
    T* o = (T*)a.out_dev + b * a.out_batch_stride + n * a.out_row_stride;
#pragma unroll
    for (int j = 0; j < NC; ++j) store4<STREAM>(o, (lane + j * TPR) * kVec, dim, h[j], j < WHOLE);
}

template <typename T, typename RT, bool STREAM> hipError_t launch(const rz_residual_norm_args& a, hipStream_t s) {
    const int rows = a.batch * a.rows, chunks = (a.dim + kVec - 1) / kVec;
    // Few threads with up to four chunks each: rows up to 512 columns share a wave, up to 1024 take one, without LDS or a barrier.  98304 rows, bf16, root-mean-square
    // norm alone, us, so / with a wave each: 64 columns 8.4 / 27.5, 128 11.7 / 28.2, 192 13.9 / 28.4, 256 17.9 / 24.6; 49152 rows of 384 13.6 / 17.6, of 512 17.8 / 19.1.
#define RZ_ROWS(TPR, NC)                                                                                                        \
    if (chunks > TPR * kWhole<TPR, NC> && chunks <= TPR * NC) {                                                                                            \
        constexpr int kBlock = TPR < 256 ? 256 : TPR, kRpb = kBlock / TPR;                                                      \
        for (int64_t from = 0; from < rows; from += (int64_t)kMostBlocks * kRpb)                                                \
            hipLaunchKernelGGL((residual_norm_kernel<T, RT, TPR, NC, STREAM>), dim3((unsigned)std::min<int64_t>(kMostBlocks, (rows - from - 1) / kRpb + 1)), \
                               dim3(kBlock), 0, s, a, (int)from, rows);                                                         \
        return hipGetLastError();                                                                                               \
    }
    RZ_ROWS(4, 1) RZ_ROWS(16, 1) RZ_ROWS(16, 2) RZ_ROWS(16, 3) RZ_ROWS(16, 4) RZ_ROWS(32, 3) RZ_ROWS(32, 4) RZ_ROWS(64, 3) RZ_ROWS(64, 4) RZ_ROWS(256, 2) RZ_ROWS(256, 4) RZ_ROWS(256, 8) RZ_ROWS(1024, 4)
#undef RZ_ROWS
    return hipErrorInvalidValue;                          // api.hip refuses dim > RZ_NORM_MAX_DIM before
}

// What is written goes past the caches once it is more than the eight L2s' 32 MB: none of it would still be there for its reader, and the vectors stay.
// 32 x 5330 rows of 768, bf16 beside an fp32 residual: 290 us against 301; 8 x 1370 rows of 1001, f16: 18.5 us against 19.8.
template <typename T, typename RT> hipError_t launch(const rz_residual_norm_args& a, hipStream_t s) {
    const double written = (double)a.batch * a.rows * a.dim * ((a.resid_out_dev ? sizeof(RT) : 0) + (a.out_dev ? sizeof(T) : 0));
    return written > 32.0 * (1 << 20) ? launch<T, RT, true>(a, s) : launch<T, RT, false>(a, s);
}

}  // namespace

hipError_t launch_residual_norm(const rz_residual_norm_args& a, hipStream_t s) {
    const bool rf = a.resid_dtype == DT_F32;
    if (a.dtype == DT_F32) return launch<float, float>(a, s);
    if (a.dtype == DT_BF16) return rf ? launch<bf16_t, float>(a, s) : launch<bf16_t, bf16_t>(a, s);
    return rf ? launch<f16_t, float>(a, s) : launch<f16_t, f16_t>(a, s);
}

}  // namespace rz

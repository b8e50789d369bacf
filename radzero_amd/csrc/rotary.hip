// radzero_hip — rotary positions on the heads of q and k.
//
//   angle(token, p) = position(token, axis of p) * freq[p],   p = 0 .. P - 1,  P = rotary_dim / 2
//   (u, w) -> amplitude * (u cos - w sin, u sin + w cos)
//   half layout: u = x[p], w = x[p + P];  interleaved: u = x[2 p], w = x[2 p + 1];  columns behind rotary_dim pass through
//   several axes (row and column of a patch): pairs are dealt to them in equal runs, p / (P / axes)
//
// Bound by HBM: every head is read and written once.  The angles of a token are the same in all heads of q and k: a workgroup takes a few
// tokens, writes their cosines and sines to LDS once and then streams all heads of both tensors past that table.
// Angles are formed in 64 bits: in fp32 the product of a position near 2^20 and a frequency near 1 is off by 2^-4 radian.  Only the
// fraction of a turn, in fp32, goes through sin and cos (2e-7 radian).  32 x 5330 tokens, 12 + 12 heads of 64, bf16: 203 us, 5.2 TB/s; one token: the launch, 4 us.
#include <algorithm>

#include "rz_common.h"
#include "rz_kernels.h"

namespace rz {

namespace {

constexpr int kThreads = 256;
constexpr int kTable = 2048;                  // (cos, sin) entries of a workgroup's tokens: 16 KB of LDS

template <typename T, int V> struct __attribute__((packed, aligned(V * sizeof(T) > 16 ? 16 : V * sizeof(T)))) Chunk { T v[V]; };

struct Heads {                                // one tensor: strides in elements
    const void* in; void* out;
    int64_t ib, it, ih, ob, ot, oh;
    int heads;
};

template <typename T, int LAYOUT, int V, bool LOOSE>
__device__ __forceinline__ void turn(const T* x, T* o, int c, int P, int tail, float2* const tab) {
    // LOOSE: single elements, any alignment and any P
    typedef Chunk<T, V> C;
    if constexpr (LAYOUT == RZ_ROTARY_HALF) {
        const int runs = P / V;
        if (c < runs) {
            const int p = c * V;
            const C u = *reinterpret_cast<const C*>(x + p), w = *reinterpret_cast<const C*>(x + P + p);
            C a, b;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 t = tab[p + e];
                const float uf = to_f32(u.v[e]), wf = to_f32(w.v[e]);
                a.v[e] = from_f32<T>(fmaf(uf, t.x, -(wf * t.y)));
                b.v[e] = from_f32<T>(fmaf(uf, t.y, wf * t.x));
            }
            *reinterpret_cast<C*>(o + p) = a;
            *reinterpret_cast<C*>(o + P + p) = b;
            return;
        }
        c -= runs;
    } else {
        const int runs = 2 * P / V;
        if (c < runs) {
            if constexpr (LOOSE) {
                const float2 t = tab[c];
                const float uf = to_f32(x[2 * c]), wf = to_f32(x[2 * c + 1]);
                o[2 * c] = from_f32<T>(fmaf(uf, t.x, -(wf * t.y)));
                o[2 * c + 1] = from_f32<T>(fmaf(uf, t.y, wf * t.x));
            } else {
                const C u = *reinterpret_cast<const C*>(x + c * V);
                C a;
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    const float2 t = tab[(c * V + e) / 2];
                    const float uf = to_f32(u.v[e]), wf = to_f32(u.v[e + 1]);
                    a.v[e] = from_f32<T>(fmaf(uf, t.x, -(wf * t.y)));
                    a.v[e + 1] = from_f32<T>(fmaf(uf, t.y, wf * t.x));
                }
                *reinterpret_cast<C*>(o + c * V) = a;
            }
            return;
        }
        c -= runs;
    }
    if constexpr (LOOSE) {                    // pass-through columns, as many per step as a run of the rotated ones
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (c * V + e < tail) o[2 * P + c * V + e] = x[2 * P + c * V + e];
    } else {
        *reinterpret_cast<C*>(o + 2 * P + c * V) = *reinterpret_cast<const C*>(x + 2 * P + c * V);
    }
}

template <typename T, int LAYOUT, int V, bool LOOSE>
__global__ __launch_bounds__(kThreads) void rotary_kernel(Heads q, Heads k, const int64_t* positions, int64_t pos_batch, int64_t pos_token, int axes,
                                                          const double* freqs, float amplitude, int64_t total_tokens, int tokens, int head_dim, int P,
                                                          int per_block) {
    __shared__ float2 tab[kTable];
    const int per_axis = P / axes;
    for (int64_t t0 = (int64_t)blockIdx.x * per_block; t0 < total_tokens; t0 += (int64_t)gridDim.x * per_block) {
        const int here = (int)min((int64_t)per_block, total_tokens - t0);
        for (int i = threadIdx.x; i < here * P; i += kThreads) {
            const int t = i / P, p = i - t * P;
            const int64_t row = t0 + t, b = row / tokens, n = row - b * tokens;
            const double angle = (double)positions[b * pos_batch + n * pos_token + p / per_axis] * freqs[p];
            const double turns = angle * 0.15915494309189533577;                    // 1 / (2 pi)
            float s, c;
            sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
            tab[i] = make_float2(amplitude * c, amplitude * s);
        }
        __syncthreads();
        const int tail = head_dim - 2 * P;
        const int runs = (LAYOUT == RZ_ROTARY_HALF ? P / V : 2 * P / V) + (tail + V - 1) / V;
        const int heads = q.heads + k.heads, units = heads * runs;
        for (int i = threadIdx.x; i < here * units; i += kThreads) {
            const int t = i / units, u = i - t * units, h = u / runs, c = u - h * runs;
            const int64_t row = t0 + t, b = row / tokens, n = row - b * tokens;
            const Heads& x = h < q.heads ? q : k;
            const int hh = h < q.heads ? h : h - q.heads;
            turn<T, LAYOUT, V, LOOSE>((const T*)x.in + b * x.ib + n * x.it + hh * x.ih, (T*)x.out + b * x.ob + n * x.ot + hh * x.oh, c, P, tail, tab + t * P);
        }
        __syncthreads();                                                            // the table's readers are done
    }
}

template <typename T, int LAYOUT> hipError_t launch(const rz_rotary_args& a, hipStream_t s) {
    Heads q{a.q_dev, a.q_out_dev, a.q_batch_stride, a.q_token_stride, a.q_head_stride, a.q_out_batch_stride, a.q_out_token_stride, a.q_out_head_stride, a.q_heads};
    Heads k{a.k_dev, a.k_out_dev, a.k_batch_stride, a.k_token_stride, a.k_head_stride, a.k_out_batch_stride, a.k_out_token_stride, a.k_out_head_stride, a.k_heads};
    const int64_t total = (int64_t)a.batch * a.tokens;
    const int P = a.rotary_dim / 2;
    auto fits = [&](int v) {                  // may every access take v elements at once
        const int64_t m = v;
        auto ok = [&](const Heads& x) {
            return !x.heads || !(((uintptr_t)x.in | (uintptr_t)x.out) % (v * sizeof(T)) || x.ib % m || x.it % m || x.ih % m || x.ob % m || x.ot % m || x.oh % m);
        };
        return (LAYOUT == RZ_ROTARY_HALF ? P : 2 * P) % v == 0 && (a.head_dim - 2 * P) % v == 0 && ok(q) && ok(k);
    };
    // tokens of a workgroup: as many as the table holds up to 8 (the table's cost is spread over them all the same), fewer while the grid
    // would leave CUs without work
    int per = kTable / P < 8 ? kTable / P : 8;
    while (per > 1 && (total + per - 1) / per < 1024) per /= 2;
    const dim3 grid((unsigned)std::min<int64_t>((total + per - 1) / per, 1 << 20));       // a launch takes less than 2^32 threads
#define RZ_TURN(V, LOOSE)                                                                                                                \
    hipLaunchKernelGGL((rotary_kernel<T, LAYOUT, V, LOOSE>), grid, dim3(kThreads), 0, s, q, k, a.positions_dev, a.positions_batch_stride, \
                       a.positions_token_stride, a.n_axes, a.freqs_dev, a.amplitude, total, a.tokens, a.head_dim, P, per)
    constexpr int kWide = 16 / (int)sizeof(T);
    if (fits(kWide)) RZ_TURN(kWide, false);
    else if (sizeof(T) == 2 && fits(4)) RZ_TURN(4, false);
    else if (LAYOUT == RZ_ROTARY_HALF) RZ_TURN(1, true);
    else RZ_TURN(2, true);
#undef RZ_TURN
    return hipGetLastError();
}

template <typename T> hipError_t launch(const rz_rotary_args& a, hipStream_t s) {
    return a.layout == RZ_ROTARY_HALF ? launch<T, RZ_ROTARY_HALF>(a, s) : launch<T, RZ_ROTARY_INTERLEAVED>(a, s);
}

}  // namespace

hipError_t launch_rotary(const rz_rotary_args& a, hipStream_t s) {
    return a.dtype == DT_F32 ? launch<float>(a, s) : a.dtype == DT_BF16 ? launch<bf16_t>(a, s) : launch<f16_t>(a, s);
}

}  // namespace rz

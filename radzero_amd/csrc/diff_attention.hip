// radzero_hip — differential attention: the difference of two softmax maps over the same values.
//
//   s_m[i][j] = scale * q_m[i] . k_m[j],  m = 1, 2 (the halves of a head's row);  hidden keys count for nothing
//   o[i] = sum_j (softmax(s_1[i])[j] - lambda softmax(s_2[i])[j]) v[j]
//   lambda = exp(lq1 . lk1) - exp(lq2 . lk2) + lambda_init
//   out[i] = out_scale * o[i] / sqrt(mean(o[i]^2) + eps) * w      (or out_scale * o[i] without a norm weight)
//
// One pass over the keys: each map keeps its running maximum and sum and its own sum of values; the maps meet when both sums are known.
#include "rz_common.h"
#include "rz_kernels.h"

namespace rz {

namespace {

// one wave per query row and head; a lane owns one key of a tile of 64 for the scores, and every 64th column for the values
template <typename T> __global__ __launch_bounds__(64) void diff_attention_kernel(const rz_diff_attention_args a) {
    const int lane = threadIdx.x, d = a.head_dim, w = 2 * d;
    int64_t id = blockIdx.x;
    const int h = (int)(id % a.heads);
    id /= a.heads;
    const int i = (int)(id % a.n_q), b = (int)(id / a.n_q), hk = h / (a.heads / a.kv_heads);
    const T* q = (const T*)a.q_dev + b * a.q_batch_stride + i * a.q_token_stride + h * a.q_head_stride;
    const T* k = (const T*)a.k_dev + b * a.k_batch_stride + hk * a.k_head_stride;
    const T* v = (const T*)a.v_dev + b * a.v_batch_stride + hk * a.v_head_stride;
    int n = a.n_k;
    if (a.kv_lens_dev) n = min(max(a.kv_lens_dev[b], 0), n);
    int end = n;
    if (a.causal) end = min(n, i + 1 + (a.causal == RZ_CAUSAL_END ? n - a.n_q : 0));
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[2][4] = {};
    const float c = a.scale * 1.44269504088896340736f;
    for (int j0 = 0; j0 < end; j0 += 64) {
        const int j = j0 + lane;
        const bool seen = j < end && (!a.mask_dev || a.mask_dev[b * a.mask_batch_stride + j] != 0);
        if (!__ballot(seen)) continue;
        float p[2];
        for (int x = 0; x < 2; ++x) {
            float s = -INFINITY;
            if (seen) {
                s = 0.f;
                for (int e = 0; e < d; ++e) s = fmaf(to_f32(q[x * d + e]), to_f32(k[j * a.k_token_stride + x * d + e]), s);
            }
            const float mn = fmaxf(m[x], wave_max(s));
            const float f = mn == -INFINITY ? 1.f : exp2f((m[x] - mn) * c);
            p[x] = !seen ? 0.f : mn == -INFINITY ? s * 0.f : exp2f((s - mn) * c);
            l[x] = l[x] * f + wave_sum(p[x]);
            for (int y = 0; y < 4; ++y) o[x][y] *= f;
            m[x] = mn;
        }
        for (int t = 0; t < 64; ++t) {
            if (!__shfl((int)seen, t, 64)) continue;
            const float p1 = __shfl(p[0], t, 64), p2 = __shfl(p[1], t, 64);
            for (int y = 0; y < 4 && lane + 64 * y < w; ++y) {
                const float x = to_f32(v[(j0 + t) * a.v_token_stride + lane + 64 * y]);
                o[0][y] = fmaf(p1, x, o[0][y]);
                o[1][y] = fmaf(p2, x, o[1][y]);
            }
        }
    }
    const float* lam = a.lambda_qk_dev + h * a.lambda_head_stride;
    float x1 = 0.f, x2 = 0.f;
    for (int e = lane; e < d; e += 64) {
        x1 = fmaf(lam[e], lam[d + e], x1);
        x2 = fmaf(lam[2 * d + e], lam[3 * d + e], x2);
    }
    const float lambda = expf(wave_sum(x1)) - expf(wave_sum(x2)) + a.lambda_init;
    const float r1 = l[0] == 0.f ? 0.f : 1.f / l[0], r2 = l[1] == 0.f ? 0.f : lambda / l[1];
    float ss = 0.f;
    for (int y = 0; y < 4; ++y) {
        o[0][y] = o[0][y] * r1 - o[1][y] * r2;
        if (lane + 64 * y < w) ss += o[0][y] * o[0][y];
    }
    float f = a.out_scale;
    if (a.norm_weight_dev) f /= sqrtf(wave_sum(ss) / (float)w + a.norm_eps);
    T* out = (T*)a.out_dev + b * a.out_batch_stride + i * a.out_token_stride + h * a.out_head_stride;
    for (int y = 0; y < 4 && lane + 64 * y < w; ++y) {
        const int col = lane + 64 * y;
        out[col] = from_f32<T>(o[0][y] * f * (a.norm_weight_dev ? a.norm_weight_dev[col] : 1.f));
    }
}

}  // namespace

size_t diff_attention_workspace_bytes(const rz_diff_attention_args&) { return 0; }

hipError_t launch_diff_attention(const rz_diff_attention_args& a, void*, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)a.batch * a.n_q * a.heads));
    if (a.dtype == DT_F32) hipLaunchKernelGGL(diff_attention_kernel<float>, grid, dim3(64), 0, s, a);
    else if (a.dtype == DT_BF16) hipLaunchKernelGGL(diff_attention_kernel<bf16_t>, grid, dim3(64), 0, s, a);
    else hipLaunchKernelGGL(diff_attention_kernel<f16_t>, grid, dim3(64), 0, s, a);
    return hipGetLastError();
}

}  // namespace rz

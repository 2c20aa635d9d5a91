// Attention with capped scores, a distance bias and causal / prefix / document masks over bf16 keys and values, or over the 8-bit cache.
//
//   s = scale q.k;  s = cap tanh(s / cap);  s -= slope |p - kp|;  out = softmax over the visible keys, times v
//
// The query of token t of an episode with n queries and L keys stands at p = q_start + t (L - n + t when none is given), key j at kp = j or k_pos[j].
// Visible: j < L, with `causal` kp <= max(p, prefix - 1), with documents equal ids that are not negative. A query without a visible key gets zeros.
#pragma once

#include "common.cuh"
#include "gemm_tc5.cuh"
#include "quantized_cache.cuh"

namespace fvla {
namespace mattn {

struct Args {
    const void *q, *k, *v;
    const float *k_scale, *v_scale;
    bf16* out;
    float* lse;
    const int *prefix, *q_lens, *k_lens, *q_start, *q_docs, *k_docs, *k_pos;
    const float* slopes;
    float* weights;
    long long qs[3], ks[3], vs[3], os[3];     // strides in elements: episode, token, head
    float scale, cap, decay;
    int episodes, tokens, keys, heads, kv_heads, dim, block, causal;
};

// What an episode's rows have in common.
struct Episode {
    int n, L, start, prefix;
};
__device__ __forceinline__ Episode episode_of(const Args& p, int e) {
    Episode s;
    s.L = p.k_lens ? min(max(p.k_lens[e], 0), p.keys) : p.keys;
    s.n = p.q_lens ? min(max(p.q_lens[e], 0), p.tokens) : p.tokens;
    s.start = p.q_start ? p.q_start[e] : s.L - s.n;
    s.prefix = p.prefix ? p.prefix[e] : 0;
    return s;
}

template <bool Q8>
__device__ __forceinline__ float element(const void* base, const float* scale, const Args& p, const long long (&st)[3], int e, int j, int head, int d) {
    if (d >= p.dim) return 0.f;
    const long long at = e * st[0] + j * st[1] + head * st[2] + d;
    if (!Q8) return __bfloat162float(static_cast<const bf16*>(base)[at]);
    return q8::from_e4m3x2(static_cast<const uint8_t*>(base)[at]).x * scale[((size_t)e * (p.keys / p.block) + j / p.block) * p.kv_heads + head];
}

// One warp per query row: a lane holds dims lane, lane + 32, ...
template <bool Q8>
__global__ void __launch_bounds__(128) attention_rows_kernel(const Args p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= (long long)p.episodes * p.tokens * p.heads) return;
    const int h = (int)(row % p.heads), t = (int)(row / p.heads % p.tokens), e = (int)(row / p.heads / p.tokens);
    const Episode s = episode_of(p, e);
    if (t >= s.n) return;
    const int kv = h / (p.heads / p.kv_heads), pos = s.start + t, limit = max(pos, s.prefix - 1);
    const int doc = p.q_docs ? p.q_docs[(size_t)e * p.tokens + t] : 0;
    float q[8], acc[8], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) { q[i] = element<false>(p.q, nullptr, p, p.qs, e, t, h, lane + 32 * i); acc[i] = 0.f; }
    for (int j = 0; j < s.L; ++j) {
        const int kp = p.k_pos ? p.k_pos[(size_t)e * p.keys + j] : j;
        if (p.causal && kp > limit) continue;
        if (p.k_docs) { const int d = p.k_docs[(size_t)e * p.keys + j]; if (d != doc || d < 0) continue; }
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) x = fmaf(q[i], element<Q8>(p.k, p.k_scale, p, p.ks, e, j, kv, lane + 32 * i), x);
        x = warp_sum(x) * p.scale;
        if (p.cap > 0.f) x = p.cap * tanhf(x / p.cap);
        if (p.slopes) x -= p.slopes[h] * fabsf((float)(pos - kp));
        const float top = fmaxf(m, x), was = m == -INFINITY ? 0.f : expf(m - top), pr = x == -INFINITY ? 0.f : expf(x - (top == -INFINITY ? 0.f : top));      // (a row of NaN has no maximum)
        m = top;
        l = l * was + pr;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = acc[i] * was + pr * element<Q8>(p.v, p.v_scale, p, p.vs, e, j, kv, lane + 32 * i);
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < p.dim) p.out[e * p.os[0] + t * p.os[1] + h * p.os[2] + lane + 32 * i] = __float2bfloat16_rn(acc[i] * inv);
    if (p.lse && lane == 0) p.lse[((size_t)e * p.heads + h) * p.tokens + t] = l > 0.f ? m + logf(l) : (l == 0.f ? -INFINITY : l);
}

// weights[e][j] = decay * weights[e][j] + the probabilities that key j got from all rows, from the rows' log-sum-exp. One warp per key.
template <bool Q8>
__global__ void __launch_bounds__(128) key_weights_kernel(const Args p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const long long key = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (key >= (long long)p.episodes * p.keys) return;
    const int j = (int)(key % p.keys), e = (int)(key / p.keys);
    const Episode s = episode_of(p, e);
    if (j >= s.L) return;
    const int kp = p.k_pos ? p.k_pos[key] : j;
    float sum = 0.f;
    for (int h = 0; h < p.heads; ++h)
        for (int t = 0; t < s.n; ++t) {
            const int pos = s.start + t;
            if (p.causal && kp > max(pos, s.prefix - 1)) continue;
            float x = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x = fmaf(element<false>(p.q, nullptr, p, p.qs, e, t, h, lane + 32 * i), element<Q8>(p.k, p.k_scale, p, p.ks, e, j, h / (p.heads / p.kv_heads), lane + 32 * i), x);
            x = warp_sum(x) * p.scale;
            if (p.cap > 0.f) x = p.cap * tanhf(x / p.cap);
            if (p.slopes) x -= p.slopes[h] * fabsf((float)(pos - kp));
            const float z = p.lse[((size_t)e * p.heads + h) * p.tokens + t];
            if (z != -INFINITY) sum += expf(x - z);
        }
    if (lane == 0) p.weights[key] = (p.decay != 0.f ? p.decay * p.weights[key] : 0.f) + sum;
}

}  // namespace mattn
}  // namespace fvla

// Attention with capped scores, a distance bias and causal / prefix / document masks over bf16 keys and values, or over the 8-bit cache.
//
//   s = scale q.k;  s = cap tanh(s / cap);  s -= slope |p - kp|;  out = softmax over the visible keys, times v
//
// The query of token t of an episode with n queries and L keys stands at p = q_start + t (L - n + t when none is given), key j at kp = j or k_pos[j].
// Visible: j < L, with `causal` kp <= max(p, prefix - 1), with documents equal ids that are not negative. A query without a visible key gets zeros.
//
// Two kernels: tile_attention.cuh (128 rows of tokens x heads against 128 keys at a time; bound by the softmax's instructions, or at head dim 256 by
// how fast keys and values arrive) and few_rows_attention.cuh (up to 32 rows; bound by the bytes of the cache, or where there are few by a chain of
// latencies). Here: what both are given, masks and scores, the join of keys shared out over CTAs, the weights of keys, and the choice between them.
#pragma once

#include "common.cuh"
#include "gemm_tc5.cuh"
#include "quantized_cache.cuh"

namespace fvla {
namespace mattn {

using tc5::mbar_expect_tx;
using tc5::mbar_init;
using tc5::mbar_wait;
using tc5::smem_desc;

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

constexpr int BQ = 128, BKEY = 128, SOFTMAX_WARPS = 8, SOFTMAX0 = 4;
constexpr float RESCALE_THRESHOLD = 8.0f;      // log2 units
// Row sums over the 8-bit cache add up P (a probability times V's scale, at most 2^8, flushed below 2^-126) over that scale: with all scales of V within these
// 60 binades that neither leaves fp32 nor misses what is above 2^-60 of a row.
__device__ __forceinline__ bool odd_scale(float s) { return !(s >= 0x1p-40f && s <= 0x1p20f); }

struct Tile {
    Args a;
    int cluster;                                // few rows: the shares of a row are one cluster
    int group, tile_tokens, tiles, splits;      // query heads per K/V head, tokens per tile
    int q_mul[2], k_mul[2], v_mul[2];           // 0 where an axis (K/V head, episode) is broadcast: its coordinate stays 0
    float* part_o;                              // [split][row][HDP] fp32, row = ((e * tokens + t) * heads + h)
    float2* part_ml;                            // [split][row] maximum (log2) and row sum; of the 8-bit cache, whose row sums have a maximum of their own, the sum's log2
    float* scores;                              // log2 units, or null: what the keys' weights are made of
    long long pitch;                            // few rows: [row][pitch]
    int key_blocks;                             // many: [episode, K/V head, tile][key block][4 keys][128 rows][4]
    const int2* doc_range;                      // [episode][key block] smallest and largest document
    int* status;
};

// Document ids of each block of keys: the smallest and the largest.
__global__ void __launch_bounds__(128) document_ranges_kernel(const int* __restrict__ docs, int2* __restrict__ range, int episodes, int keys, int blocks) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (i >= (long long)episodes * blocks) return;
    const int e = (int)(i / blocks), first = (int)(i % blocks) * BKEY, last = min(first + BKEY, keys);
    int low = 0x7fffffff, high = -0x7fffffff - 1;
    for (int j = first + lane; j < last; j += 32) {
        const int d = docs[(size_t)e * keys + j];
        low = min(low, d);
        high = max(high, d);
    }
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    if (lane == 0) range[i] = make_int2(low, high);
}

__device__ __forceinline__ float fast_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// tanh of scores over their cap. Its Taylor series to y^13 where every |y| of a thread's scores is at most 1/2 (the next term is below 2^-22 of y), which
// is all but always so and costs multiply-adds alone; else 1 - 2 / (1 + e^2y), good to 2^-22 of 1, with two special-function instructions and the series
// to y^7 where that would cancel (|y| < 1/5).
constexpr float kTanh3 = -1.f / 3.f, kTanh5 = 2.f / 15.f, kTanh7 = -17.f / 315.f, kTanh9 = 62.f / 2835.f, kTanh11 = -1382.f / 155925.f, kTanh13 = 21844.f / 6081075.f;
__device__ __forceinline__ float tanh_far(float y) {
    const float far = fmaf(-2.f, fast_rcp(1.f + fast_exp2(2.f * kLog2e * y)), 1.f), y2 = y * y;
    const float near = fmaf(y * y2, fmaf(y2, fmaf(y2, kTanh7, kTanh5), kTanh3), y);
    return y2 < 0.04f ? near : far;
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, int w) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, int w, int v) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v) : "memory");
}
// 32 columns of this thread's TMEM lane, without the wait.
__device__ __forceinline__ void ld32_nowait(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr) : "memory");
}
// What a CTA's rows may see, block by block. Every role evaluates it from the same memory. The last block comes first: where scores fall with distance
// the maximum is found at once, and nothing is rescaled (every block otherwise: 241 us against 178 at head dim 128, 4 096 causal keys, 32 heads).
struct Walk {
    int first, count;                 // key blocks of this CTA (of its split), some of which may hold nothing that is seen
    int q_low, q_high;                // documents of the tile's queries
    const int2* range;                // of the episode's key blocks, or null
    __device__ __forceinline__ int block(int i) const { return first + count - 1 - i; }
    __device__ __forceinline__ bool sees(int i) const {
        if (range == nullptr) return true;
        const int2 r = __ldg(range + block(i));
        return r.y >= q_low && r.x <= q_high;
    }
    __device__ __forceinline__ int next(int i) const {      // the first block from i on that is seen, or count
        while (i < count && !sees(i)) ++i;
        return i;
    }
};

// The shares' sums against the largest of their maxima (the row sums of the 8-bit cache against the largest of theirs). `warps` of a CTA take 32 * PER columns of a row together (grid.y: which): each adds up every
// warps-th share, and the first adds up the warps in their order.
constexpr int JOIN_WARPS = 8;
template <int PER>
__global__ void __launch_bounds__(32 * JOIN_WARPS) attention_join_kernel(const __grid_constant__ Tile p, int hdp, int warps) {
    __shared__ float sums[JOIN_WARPS][32 * PER + 1];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Args& a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % warps, col0 = blockIdx.y * 32 * PER + lane;
    const int row = blockIdx.x * (JOIN_WARPS / warps) + warp / warps, rows = a.episodes * a.tokens * a.heads;      // (below 2^31: checked on the host)
    const int h = row % a.heads, t = row / a.heads % a.tokens, e = min(row / a.heads / a.tokens, a.episodes - 1);
    const bool mine = row < rows && t < episode_of(a, e).n;
    const bool logs = a.k_scale != nullptr;
    const float nothing = logs ? -INFINITY : 0.f;
    // no load waits for another, but for the maxima: shares that held nothing are read as well, and dropped
    float m = -INFINITY, m_sum = -INFINITY;
#pragma unroll 4
    for (int s = lane; s < p.splits; s += 32) {
        const float2 ml = mine ? p.part_ml[(size_t)s * rows + row] : make_float2(0.f, nothing);
        if (ml.y != nothing) { m = fmaxf(m, ml.x); m_sum = fmaxf(m_sum, ml.y); }
    }
    m = warp_max(m);
    const float top = m == -INFINITY ? 0.f : m;
    m_sum = logs ? warp_max(m_sum) : top;
    const float top_sum = m_sum == -INFINITY ? 0.f : m_sum;
    float acc[PER], l = 0.f;                                                         // columns lane, lane + 32, ...
#pragma unroll
    for (int c = 0; c < PER; ++c) acc[c] = 0.f;
    const float* o = p.part_o + (size_t)(mine ? row : 0) * hdp + col0;
    const size_t pitch = (size_t)rows * hdp;
    for (int s0 = part; s0 < p.splits; s0 += 32 * warps) {
        // lane i: the factor of share s0 + i * warps
        const int s = s0 + lane * warps;
        const float2 ml = mine && s < p.splits ? p.part_ml[(size_t)s * rows + row] : make_float2(0.f, nothing);
        const bool held = ml.y != nothing;
        const float w = !held ? 0.f : (ml.x == -INFINITY ? 1.f : fast_exp2(ml.x - top));
        l += warp_sum(!held ? 0.f : (logs ? fast_exp2(ml.y - top_sum) : ml.y * w));
        const int have = min(32, (p.splits - s0 + warps - 1) / warps);
        constexpr int BATCH = PER == 1 ? 16 : 4;                                     // loads in flight before the first is used
        for (int i = 0; i < have; i += BATCH) {
            float x[BATCH][PER];
#pragma unroll
            for (int k = 0; k < BATCH; ++k)
#pragma unroll
                for (int c = 0; c < PER; ++c) x[k][c] = o[(size_t)(s0 + min(i + k, have - 1) * warps) * pitch + 32 * c];
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                const float f = __shfl_sync(0xffffffffu, w, i + k & 31);
                const bool used = __shfl_sync(0xffffffffu, held, i + k & 31);
#pragma unroll
                for (int c = 0; c < PER; ++c) acc[c] = fmaf(i + k < have ? f : 0.f, i + k < have && used ? x[k][c] : 0.f, acc[c]);
            }
        }
    }
    if (warps > 1) {
#pragma unroll
        for (int c = 0; c < PER; ++c) sums[warp][lane + 32 * c] = acc[c];
        if (lane == 0) sums[warp][32 * PER] = l;
        __syncthreads();
        if (part != 0) return;
        for (int w = 1; w < warps; ++w) {
#pragma unroll
            for (int c = 0; c < PER; ++c) acc[c] += sums[warp + w][lane + 32 * c];
            l += sums[warp + w][32 * PER];
        }
    }
    if (!mine) return;
    const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
    const float half = logs ? fast_exp2(0.5f * (top - top_sum)) : 1.f;               // the two maxima may lie beyond fp32's range of one another
    bf16* dst = a.out + e * a.os[0] + t * a.os[1] + h * a.os[2];
#pragma unroll
    for (int c = 0; c < PER; ++c)
        if (col0 + 32 * c < a.dim) dst[col0 + 32 * c] = __float2bfloat16_rn(acc[c] * half * (inv * half));
    if (a.lse && lane == 0 && blockIdx.y == 0) a.lse[((size_t)e * a.heads + h) * a.tokens + t] = l > 0.f ? (top_sum + log2f(l)) * 0.6931471805599453f : (l == 0.f ? -INFINITY : l);
}

// weights[e][j] = decay * weights[e][j] + the probabilities that key j got, from the scores that the attention left and the rows' log-sum-exps. `share`
// warps have 32 keys together; they share out the rows, and their sums are added in the order of the warps.
constexpr int WEIGHT_WARPS = 16;
__global__ void __launch_bounds__(32 * WEIGHT_WARPS) key_weights_kernel(const __grid_constant__ Tile p, int share) {
    __shared__ float part[WEIGHT_WARPS][32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Args& a = p.a;
    const int e = blockIdx.y, lane = threadIdx.x & 31, all = blockDim.x >> 5, warp = (threadIdx.x >> 5) % share, warps = share;
    const int j = (blockIdx.x * (all / share) + (threadIdx.x >> 5) / share) * 32 + lane;
    const Episode s = episode_of(a, e);
    const bool inside = j < s.L, by_number = a.causal && a.k_pos == nullptr;
    const int rows = a.heads * s.n;
    const size_t row0 = (size_t)e * a.heads * a.tokens;
    // tokens before this one do not see key j (by its number), and their scores were not left
    const int from = by_number && j >= s.prefix ? max(0, j - s.start) : 0;
    float sum = 0.f;
    constexpr int BATCH = 8;                                                         // loads in flight before the first is used
    for (int r0 = warp; r0 < rows; r0 += BATCH * warps) {
        float z[BATCH], x[BATCH];
        bool seen[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int r = min(r0 + k * warps, rows - 1), h = r / s.n, t = r - h * s.n;
            const size_t row = row0 + (size_t)h * a.tokens + t;
            z[k] = a.lse[row];
            x[k] = p.scores[row * p.pitch + min((long long)j, p.pitch - 1)];         // what was not left is read as well, and dropped
            seen[k] = r0 + k * warps < rows && inside && t >= from;
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) sum += seen[k] && z[k] != -INFINITY ? fast_exp2(fmaf(z[k], -kLog2e, x[k])) : 0.f;
    }
    if (warps > 1) {
        part[threadIdx.x >> 5][lane] = sum;
        __syncthreads();
        if (warp != 0) return;
        for (int w = 1; w < warps; ++w) sum += part[(threadIdx.x >> 5) + w][lane];
    }
    if (!inside) return;
    float* at = a.weights + (size_t)e * a.keys + j;
    *at = (a.decay != 0.f ? a.decay * *at : 0.f) + sum;
}

// The same from the scores of tiles: a CTA has a block of 128 keys of an episode, a warp four keys at a time, a lane every 32nd row.
__global__ void __launch_bounds__(32 * WEIGHT_WARPS) tile_weights_kernel(const __grid_constant__ Tile p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Args& a = p.a;
    const int e = blockIdx.y, block = blockIdx.x / 2, lane = threadIdx.x & 31, quad = blockIdx.x % 2 * WEIGHT_WARPS + (threadIdx.x >> 5);
    const Episode s = episode_of(a, e);
    const int j = block * BKEY + quad * 4;
    if (j >= s.L) return;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int kt = 0; kt < a.kv_heads * p.tiles; ++kt) {
        const int kv = kt / p.tiles, tile = kt - kv * p.tiles, t0 = tile * p.tile_tokens, tokens = min(p.tile_tokens, s.n - t0);
        // what the tile has walked (as the attention kernel has it)
        if (tokens <= 0 || (a.causal && a.k_pos == nullptr && block * BKEY >= max(s.start + t0 + tokens, s.prefix))) continue;
        const float4* from = reinterpret_cast<const float4*>(p.scores) + ((((size_t)e * a.kv_heads + kv) * p.tiles + tile) * p.key_blocks + block) * (BQ * BKEY / 4) + quad * BQ;
        float4 x[BQ / 32];
        float z[BQ / 32];
#pragma unroll
        for (int k = 0; k < BQ / 32; ++k) {
            const int r = k * 32 + lane, t = r / p.group, h = kv * p.group + r - t * p.group;
            const bool mine = t < tokens;
            x[k] = mine ? from[r] : make_float4(0.f, 0.f, 0.f, 0.f);
            z[k] = mine ? a.lse[((size_t)e * a.heads + h) * a.tokens + t0 + t] : -INFINITY;
        }
#pragma unroll
        for (int k = 0; k < BQ / 32; ++k) {
            const float v[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] += z[k] != -INFINITY ? fast_exp2(fmaf(z[k], -kLog2e, v[c])) : 0.f;
        }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) sum[c] = warp_sum(sum[c]);
    if (lane < 4 && j + lane < s.L) {
        float* at = a.weights + (size_t)e * a.keys + j + lane;
        const float mine = lane == 0 ? sum[0] : (lane == 1 ? sum[1] : (lane == 2 ? sum[2] : sum[3]));
        *at = (a.decay != 0.f ? a.decay * *at : 0.f) + mine;
    }
}

// Tensor map of a strided operand, innermost axis contiguous; an axis of stride 0 is left at one element (its coordinate is 0).
inline int make_map(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const uint64_t* strides, const uint32_t* box, int elem = 2) {
    tc5::EncodeTiledFn fn = tc5::encode_fn();
    if (fn == nullptr) { set_error("cuTensorMapEncodeTiled is not available from the driver"); return FVLA_ERR_LAUNCH; }
    cuuint64_t gdim[5], gstride[4];
    cuuint32_t b[5], step[5];
    for (int i = 0; i < rank; ++i) { gdim[i] = dims[i]; b[i] = box[i]; step[i] = 1; }
    for (int i = 0; i + 1 < rank; ++i) gstride[i] = strides[i] * elem;
    const CUresult r = fn(map, elem == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : (elem == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32), rank, const_cast<void*>(base), gdim, gstride, b, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) { set_error("attention: cuTensorMapEncodeTiled failed with CUresult %d", (int)r); return FVLA_ERR_ARG; }
    return FVLA_OK;
}

}  // namespace mattn
}  // namespace fvla

#include "tile_attention.cuh"
#include "few_rows_attention.cuh"

namespace fvla {
namespace mattn {

// Up to 32 rows per episode and K/V head, and no documents: the kernel for few rows.
inline bool takes_few(const Args& a) { return (long long)a.tokens * (a.heads / a.kv_heads) <= 32 && a.q_docs == nullptr; }
// Head dimension that the kernel is built for.
inline int padded_dim(const Args& a) { return a.dim <= 64 && !takes_few(a) && a.k_scale == nullptr ? 64 : (a.dim <= 128 ? 128 : 256); }

// Shares of the key blocks: as many as bring the CTAs up to the number that are resident, at most one per block. (Below: a token of 8 query heads per K/V head of
// 256 unless said, both sides in us.)
inline int plan_splits(const Args& a) {
    const int group = a.heads / a.kv_heads, tile_tokens = BQ / group, blocks = (a.keys + BKEY - 1) / BKEY, sms = tc5::num_sms();
    const bool few = takes_few(a);
    const long long tiles = (few ? 1ll : (long long)((a.tokens + tile_tokens - 1) / tile_tokens)) * a.kv_heads * a.episodes;
    int per_sm = 1;
    if (few) {
        const int tile_bytes = 128 * padded_dim(a) * (a.k_scale ? 1 : 2);
        per_sm = few_rows(a) == 32 ? (tile_bytes == 16384 ? 2 : 1) : (tile_bytes == 16384 ? 3 : (tile_bytes == 32768 ? 2 : 1));
    }
    // Few rows of more tiles than SMs: twice as many, which evens out the last round. 160 episodes over 2 048 / 8 192 rows 40.6 / 92 us, 44.1 / 125 without. At three CTAs
    // an SM (8 bits, head dim 128, 8 K/V heads) from 64 blocks on: 24 episodes of 8 192 58.4 (60.5), 32 of 16 384 130 (155), but of 4 096 38.3 (35.5).
    const bool twice = few && tiles > sms && (per_sm < 3 || blocks >= 64);
    const long long room = (long long)sms * per_sm * (twice ? 2 : 1) / tiles;
    // A cluster rather than a second launch that joins the shares, up to two blocks for each of its CTAs, and up to four where there are some tiles. 8 bits, 16 blocks: one
    // episode 9.5 (11.1 with a join), 32 of them 11.7 (14.5); 32 blocks: one 12.0 (11.3), four 12.0 (12.2), 32 18.1 (21.8). bf16, 32 blocks: four 12.7 (11.0), twelve
    // 15.0 (16.6). Where a CTA takes a whole SM, clusters of eight leave SMs over: 14 of them 9.6 (12.0), but 16 take a second round, 17.7 (12.2).
    const bool fits = per_sm > 1 || 5 * CLUSTER * tiles <= 4 * sms;
    if (few && fits && room > CLUSTER && blocks <= (tiles * per_sm >= 8 ? 4 : 2) * CLUSTER) return blocks < CLUSTER ? (blocks > 0 ? blocks : 1) : CLUSTER;
    return (int)(room < 1 ? 1 : (room < blocks ? room : (blocks > 0 ? blocks : 1)));
}
inline size_t score_pitch(const Args& a) { return ((size_t)a.keys + BKEY - 1) / BKEY * BKEY; }
// Of the scores: rows one by one, or tiles of 128.
inline size_t score_bytes(const Args& a) {
    const int tile_tokens = BQ / (a.heads / a.kv_heads);
    const size_t rows = takes_few(a) ? (size_t)a.episodes * a.tokens * a.heads : (size_t)a.episodes * a.kv_heads * ((a.tokens + tile_tokens - 1) / tile_tokens) * BQ;
    return rows * score_pitch(a) * sizeof(float);
}
inline size_t align256(size_t v) { return (v + 255) / 256 * 256; }
inline size_t workspace_bytes(const Args& a) {
    const int splits = plan_splits(a);
    const size_t rows = (size_t)a.episodes * a.tokens * a.heads;
    size_t n = a.q_docs ? align256((size_t)a.episodes * ((a.keys + BKEY - 1) / BKEY) * sizeof(int2)) : 0;
    if (a.weights) n += score_bytes(a);
    if (splits > (takes_few(a) ? CLUSTER : 1)) n += align256(splits * rows * sizeof(float2)) + splits * rows * padded_dim(a) * sizeof(float);
    return n;
}

inline int launch_join(const Tile& p, int hdp, cudaStream_t st) {
    const long long rows = (long long)p.a.episodes * p.a.tokens * p.a.heads;
    // From eight shares on several warps for a row; of a few rows also a CTA for 32 columns. Both sides in us, attention and join: 8 rows of 256, 296 shares 25.6 (28.0 with the
    // whole row to a CTA), 24 rows, 98 shares 20.3 (20.9 with columns apart); 408 rows, 32 shares: eight warps 19.3, four 20.7, one 24.8, columns apart 38.6; 800 rows: 26.0,
    // 23.7, 28.6, 61; 2 400 rows, 7 shares: one warp 57, four 62.
    const bool columns = rows <= 12 && p.splits >= 16;
    const int warps = p.splits < 8 ? 1 : (rows < 512 ? 8 : 4), each = JOIN_WARPS / warps, per = columns ? 1 : hdp / 32;
    const auto kern = per == 1 ? attention_join_kernel<1> : (per == 2 ? attention_join_kernel<2> : (per == 4 ? attention_join_kernel<4> : attention_join_kernel<8>));
    const cudaError_t e = launch_pdl(kern, dim3((unsigned)((rows + each - 1) / each), hdp / (32 * per)), dim3(32 * JOIN_WARPS), 0, st, p, hdp, warps);
    if (e != cudaSuccess) { set_error("attention_join_kernel: %s", cudaGetErrorString(e)); return FVLA_ERR_LAUNCH; }
    return check_launch("attention_join_kernel");
}

template <int HDP, bool Q8>
inline int launch_tile(const Tile& p, const CUtensorMap& tmQ, const CUtensorMap& tmK, const CUtensorMap& tmV, const CUtensorMap& tmO, cudaStream_t st) {
    using C = TileCfg<HDP, Q8>;
    auto kern = attention_tile_kernel<HDP, Q8>;
    static PerDeviceFlag configured;
    if (!configured.get()) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) { set_error("cudaFuncSetAttribute: %s", cudaGetErrorString(e)); return FVLA_ERR_LAUNCH; }
        configured.set();
    }
    const Args& a = p.a;
    cudaError_t e = launch_pdl(kern, dim3((unsigned)(p.tiles * p.splits * a.kv_heads * a.episodes)), dim3(C::THREADS), C::SMEM, st, p, tmQ, tmK, tmV, tmO);
    if (e != cudaSuccess) { set_error("attention_tile_kernel: %s", cudaGetErrorString(e)); return FVLA_ERR_LAUNCH; }
    int rc = check_launch("attention_tile_kernel");
    return rc || p.splits == 1 ? rc : launch_join(p, HDP, st);
}

inline int launch_weights(const Tile& p, cudaStream_t st) {
    const Args& a = p.a;
    cudaError_t e;
    if (takes_few(a)) {
        // A warp for up to 16 rows, sixteen for the most: eight rows or more for each; CTAs of four warps at least. Attention and weights, with 1 / 2 / 4 / 8 / 16 warps, us: 8 rows
        // over 131 072 keys 31.6 / 32.0 / 36.0 / 44.4 / 50.0, 32 rows over 4 096 of eight episodes 25.0 / 21.6 / 20.1 / 20.6 / 24.2, over 16 384 of 32 146 / 146 / 150 / 181 / 249,
        // 128 rows over 4 096 of two 40.0 / 30.1 / 25.2 / 22.0 / 20.0.
        const int rows_each = a.tokens * a.heads;
        int share = 1;
        while (share < WEIGHT_WARPS && rows_each > 16 * share) share *= 2;
        const int all = share < 4 ? 4 : share, keys_each = 32 * (all / share);
        e = launch_pdl(key_weights_kernel, dim3((a.keys + keys_each - 1) / keys_each, a.episodes), dim3(32 * all), 0, st, p, share);
    } else {
        e = launch_pdl(tile_weights_kernel, dim3(2 * p.key_blocks, a.episodes), dim3(32 * WEIGHT_WARPS), 0, st, p);
    }
    if (e != cudaSuccess) { set_error("key_weights_kernel: %s", cudaGetErrorString(e)); return FVLA_ERR_LAUNCH; }
    return check_launch("key_weights_kernel");
}

inline int launch_attention(const Args& a, void* ws, int* status, cudaStream_t st) {
    Tile p;
    p.a = a;
    p.group = a.heads / a.kv_heads;
    p.tile_tokens = BQ / p.group;
    p.tiles = (a.tokens + p.tile_tokens - 1) / p.tile_tokens;
    p.splits = plan_splits(a);
    p.cluster = takes_few(a) && p.splits <= CLUSTER;
    p.status = status;
    const int blocks = (a.keys + BKEY - 1) / BKEY, hdp = padded_dim(a);
    const size_t rows = (size_t)a.episodes * a.tokens * a.heads;
    uint8_t* at = static_cast<uint8_t*>(ws);
    p.doc_range = nullptr;
    if (a.q_docs) {
        int2* range = reinterpret_cast<int2*>(at);
        at += align256((size_t)a.episodes * blocks * sizeof(int2));
        p.doc_range = range;
        if (blocks > 0) {
            const cudaError_t e = launch_pdl(document_ranges_kernel, dim3((unsigned)(((long long)a.episodes * blocks + 3) / 4)), dim3(128), 0, st, a.k_docs, range, a.episodes,
                                             a.keys, blocks);
            if (e != cudaSuccess) { set_error("document_ranges_kernel: %s", cudaGetErrorString(e)); return FVLA_ERR_LAUNCH; }
            const int rc = check_launch("document_ranges_kernel");
            if (rc) return rc;
        }
    }
    p.scores = nullptr;
    p.pitch = (long long)score_pitch(a);
    p.key_blocks = blocks;
    if (a.weights) {
        p.scores = reinterpret_cast<float*>(at);
        at += score_bytes(a);
    }
    p.part_ml = reinterpret_cast<float2*>(at);
    p.part_o = reinterpret_cast<float*>(at + align256(p.splits * rows * sizeof(float2)));
    CUtensorMap tmQ = {}, tmK = {}, tmV = {}, tmO = {};
    const bool few = takes_few(a), q8 = a.k_scale != nullptr;
    p.q_mul[0] = 1;
    p.q_mul[1] = a.qs[0] != 0;
    if (!few) {
        const uint64_t dims[5] = {(uint64_t)a.dim, (uint64_t)p.group, (uint64_t)a.tokens, (uint64_t)a.kv_heads, p.q_mul[1] ? (uint64_t)a.episodes : 1};
        const uint64_t strides[4] = {(uint64_t)a.qs[2], (uint64_t)a.qs[1], (uint64_t)a.qs[2] * p.group, p.q_mul[1] ? (uint64_t)a.qs[0] : 256};
        const uint32_t box[5] = {64, (uint32_t)p.group, (uint32_t)p.tile_tokens, 1, 1};
        int rc = make_map(&tmQ, a.q, 5, dims, strides, box);
        if (rc) return rc;
        const uint64_t out_dims[5] = {dims[0], dims[1], dims[2], dims[3], (uint64_t)a.episodes};
        const uint64_t out_strides[4] = {(uint64_t)a.os[2], (uint64_t)a.os[1], (uint64_t)a.os[2] * p.group, (uint64_t)a.os[0]};
        if (p.splits == 1) {
            rc = make_map(&tmO, a.out, 5, out_dims, out_strides, box);
        } else {
            const uint64_t wide = hdp, row = wide * a.heads;
            const uint64_t part_dims[5] = {wide, dims[1], dims[2], dims[3], (uint64_t)a.episodes * p.splits}, part_strides[4] = {wide, row, wide * p.group, row * a.tokens};
            const uint32_t part_box[5] = {32, box[1], box[2], 1, 1};
            rc = make_map(&tmO, p.part_o, 5, part_dims, part_strides, part_box, 4);
        }
        if (rc) return rc;
    }
    p.k_mul[0] = a.ks[2] != 0; p.k_mul[1] = a.ks[0] != 0; p.v_mul[0] = a.vs[2] != 0; p.v_mul[1] = a.vs[0] != 0;
    if (a.keys > 0) {
        for (int i = 0; i < 2; ++i) {
            const long long* s = i == 0 ? a.ks : a.vs;
            const int* mul = i == 0 ? p.k_mul : p.v_mul;
            const uint64_t dims[4] = {(uint64_t)a.dim, (uint64_t)a.keys, mul[0] ? (uint64_t)a.kv_heads : 1, mul[1] ? (uint64_t)a.episodes : 1};
            const uint64_t strides[3] = {(uint64_t)s[1], mul[0] ? (uint64_t)s[2] : 256, mul[1] ? (uint64_t)s[0] : 256};
            const uint32_t box[4] = {q8 ? 128u : 64u, i == 0 || few ? 128u : 16384u / (uint32_t)(hdp * (q8 ? 1 : 2)), 1, 1};      // V of the tile kernel: 16 KB of keys
            const int rc = make_map(i == 0 ? &tmK : &tmV, i == 0 ? a.k : a.v, 4, dims, strides, box, q8 ? 1 : 2);
            if (rc) return rc;
        }
    }
    int rc;
    if (few) {
        if (q8) rc = hdp == 128 ? launch_few<128, true>(p, tmK, tmV, st) : launch_few<256, true>(p, tmK, tmV, st);
        else rc = hdp == 128 ? launch_few<128, false>(p, tmK, tmV, st) : launch_few<256, false>(p, tmK, tmV, st);
        if (!rc && !p.cluster) rc = launch_join(p, hdp, st);
    } else if (q8) {
        rc = hdp == 128 ? launch_tile<128, true>(p, tmQ, tmK, tmV, tmO, st) : launch_tile<256, true>(p, tmQ, tmK, tmV, tmO, st);
    } else {
        rc = hdp == 64 ? launch_tile<64, false>(p, tmQ, tmK, tmV, tmO, st) : (hdp == 128 ? launch_tile<128, false>(p, tmQ, tmK, tmV, tmO, st) : launch_tile<256, false>(p, tmQ, tmK, tmV, tmO, st));
    }
    return rc || a.weights == nullptr || a.keys == 0 ? rc : launch_weights(p, st);
}

// The decay of the weights alone, where there is no query.
inline int launch_weights(const Args& a, cudaStream_t st) {
    Tile p = {};
    p.a = a;
    return a.keys == 0 ? FVLA_OK : launch_weights(p, st);
}

}  // namespace mattn
}  // namespace fvla

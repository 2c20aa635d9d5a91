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

// ------------------------------------------------------------------------------------------------------------------------------------
// One CTA has 128 rows (tokens x the query heads of one K/V head) of an episode and walks the key blocks that any of them sees, or one of `splits`
// equal shares of them:
//   warp 0      TMA: the Q tile; bf16 keys and values, each through a ring of STAGES blocks of 128 keys
//   warp 1      one lane issues S = Q K^T (into one of two TMEM score buffers, a block ahead) and O += P V (TMEM)
//   warps 4-11  softmax: two threads per row, 64 keys each; P goes to shared memory as the A operand of P V. The accumulator is rescaled
//               only where the maximum has grown by more than 2^8.
//   warps 12-19 (8-bit cache) four warps read e4m3 keys, four values, a block ahead in registers, and write them as fp16 operands
// The 8-bit cache: e4m3 is exact in fp16, and the products run in fp16. A row of Q is first brought to [1, 2) by its own power of two, so that
// what fp16's range cuts off is below 2^-24 of the row's largest element. The scale of K multiplies the scores in fp32. The scale of V, a power of two,
// moves into the exponent of P: w = log2 p + log2 V_scale, P = 2^(w - max w), and the row sum takes it back per block.
constexpr int BQ = 128, BKEY = 128, SOFTMAX_WARPS = 8, SOFTMAX0 = 4, CONVERT0 = SOFTMAX0 + SOFTMAX_WARPS;
constexpr float RESCALE_THRESHOLD = 8.0f;      // log2 units

template <int HDP, bool Q8>
struct Cfg {
    static constexpr int ATOMS = HDP / 64;
    static constexpr int STAGES = HDP == 256 ? 1 : 2;
    static constexpr int Q_BYTES = BQ * HDP * 2, KV_BYTES = BKEY * HDP * 2, P_BYTES = BQ * BKEY * 2;
    static constexpr int OFF_Q = 0, OFF_K = OFF_Q + Q_BYTES, OFF_V = OFF_K + STAGES * KV_BYTES, OFF_P = OFF_V + STAGES * KV_BYTES;
    static constexpr int OFF_X = OFF_P + P_BYTES;                    // one float per softmax thread
    static constexpr int OFF_BAR = OFF_X + 2 * BQ * 4;
    static constexpr int SMEM = 1024 + OFF_BAR + 192;
    static constexpr int THREADS = 32 * (Q8 ? CONVERT0 + 8 : CONVERT0);
    static constexpr uint32_t O_COL = 256;
};

struct Tile {
    Args a;
    int cluster;                                // few rows: the shares of a row are one cluster
    int group, tile_tokens, tiles, splits;      // query heads per K/V head, tokens per tile
    int q_mul[2], k_mul[2], v_mul[2];           // 0 where an axis (K/V head, episode) is broadcast: its coordinate stays 0
    float* part_o;                              // [split][row][HDP] fp32, row = ((e * tokens + t) * heads + h)
    float2* part_ml;                            // [split][row] maximum (log2) and sum
    float* scores;                              // [row][pitch] log2 units, or null: what the keys' weights are made of
    long long pitch;
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

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float fast_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// tanh(y) = 1 - 2 / (1 + e^2y), good to 2^-22 of 1; its series up to y^7 where that would cancel (the next term is below 2^-22 of y).
__device__ __forceinline__ float tanh_f(float y) {
    const float far = fmaf(-2.f, fast_rcp(1.f + fast_exp2(2.f * kLog2e * y)), 1.f), y2 = y * y;
    const float near = fmaf(y * y2, fmaf(y2, fmaf(y2, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), y);
    return y2 < 0.04f ? near : far;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t pair) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)pair));
    return h;
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
__device__ __forceinline__ void st32(uint32_t taddr, const float (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]),
          "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]),
          "f"(v[16]), "f"(v[17]), "f"(v[18]), "f"(v[19]), "f"(v[20]), "f"(v[21]), "f"(v[22]), "f"(v[23]),
          "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]), "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31])
        : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// What a CTA's rows may see, block by block. Every role evaluates it from the same memory.
struct Walk {
    int first, count;                 // key blocks of this CTA (of its split), some of which may hold nothing that is seen
    int q_low, q_high;                // documents of the tile's queries
    const int2* range;                // of the episode's key blocks, or null
    __device__ __forceinline__ bool sees(int i) const {
        if (range == nullptr) return true;
        const int2 r = __ldg(range + first + i);
        return r.y >= q_low && r.x <= q_high;
    }
    __device__ __forceinline__ int next(int i) const {      // the first block from i on that is seen, or count
        while (i < count && !sees(i)) ++i;
        return i;
    }
};

template <int HDP, bool Q8>
__global__ void __launch_bounds__(Cfg<HDP, Q8>::THREADS, 1)
attention_tile_kernel(const __grid_constant__ Tile p, const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV) {
    using C = Cfg<HDP, Q8>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t sQ = base + C::OFF_Q, sP = base + C::OFF_P, bars = base + C::OFF_BAR;
    auto sK = [&](int s) { return base + C::OFF_K + s * C::KV_BYTES; };
    auto sV = [&](int s) { return base + C::OFF_V + s * C::KV_BYTES; };
    const uint32_t q_full = bars, q_ready = bars + 8, p_full = bars + 16, p_empty = bars + 24, o_done = bars + 32;
    auto s_full = [&](int b) { return bars + 40 + b * 8; };
    auto s_empty = [&](int b) { return bars + 56 + b * 8; };
    auto k_full = [&](int s) { return bars + 72 + s * 8; };
    auto k_empty = [&](int s) { return bars + 88 + s * 8; };
    auto v_full = [&](int s) { return bars + 104 + s * 8; };
    auto v_empty = [&](int s) { return bars + 120 + s * 8; };
    const uint32_t tmem_slot = bars + 136;
    volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(gen + C::OFF_BAR + 136);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + C::OFF_BAR + 140);
    int* shared_int = reinterpret_cast<int*>(gen + C::OFF_BAR + 144);      // smallest and largest document of the queries, first and last block seen

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Args& a = p.a;
    const int e = blockIdx.z, kv = blockIdx.y, split = blockIdx.x % p.splits, tile = p.tiles - 1 - (int)(blockIdx.x / p.splits);      // the longest causal rows first
    const int t0 = tile * p.tile_tokens;

    if (tid == 0) {
        mbar_init(q_full, 1); mbar_init(q_ready, SOFTMAX_WARPS); mbar_init(p_full, SOFTMAX_WARPS); mbar_init(p_empty, 1); mbar_init(o_done, 1);
        for (int b = 0; b < 2; ++b) { mbar_init(s_full(b), 1); mbar_init(s_empty(b), SOFTMAX_WARPS); }
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(k_full(s), Q8 ? 4 : 1); mbar_init(v_full(s), Q8 ? 4 : 1);
            mbar_init(k_empty(s), 1); mbar_init(v_empty(s), 1);
        }
        *abort_flag = 0;
        shared_int[0] = shared_int[2] = 0x7fffffff;
        shared_int[1] = shared_int[3] = -0x7fffffff - 1;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        tc5::tmem_alloc(tmem_slot, 512);
        tc5::tmem_relinquish();
    }
    tc5::tc_fence_before();
    __syncthreads();
    tc5::tc_fence_after();
    const uint32_t tmem = *tmem_slot_ptr;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const Episode s = episode_of(a, e);
    const int tokens = min(p.tile_tokens, s.n - t0);      // of this tile; none: nothing to write
    Walk walk;
    walk.range = nullptr;
    walk.q_low = walk.q_high = 0;
    int first = 0, last = 0;
    if (tokens > 0) {
        int most = s.L;
        if (a.causal && a.k_pos == nullptr) most = max(0, min(most, max(s.start + t0 + tokens, s.prefix)));
        last = (most + BKEY - 1) / BKEY;
        if (a.q_docs != nullptr) {
            const int blocks = (a.keys + BKEY - 1) / BKEY;
            for (int t = tid; t < tokens; t += C::THREADS) {
                const int d = a.q_docs[(size_t)e * a.tokens + t0 + t];
                if (d >= 0) {                                  // padding sees nothing
                    atomicMin(shared_int, d);
                    atomicMax(shared_int + 1, d);
                }
            }
            __syncthreads();
            walk.q_low = shared_int[0];
            walk.q_high = shared_int[1];
            walk.range = p.doc_range + (size_t)e * blocks;
            walk.first = 0;
            for (int j = tid; j < last; j += C::THREADS)
                if (walk.sees(j)) { atomicMin(shared_int + 2, j); atomicMax(shared_int + 3, j); }
            __syncthreads();
            first = min(shared_int[2], last);
            last = max(first, min(last, shared_int[3] + 1));
        }
    }
    const int share = (last - first + p.splits - 1) / p.splits;
    walk.first = first + split * share;
    walk.count = max(0, min(share, last - walk.first));

    const bool any = walk.next(0) < walk.count;

    // (8-bit cache) 640 threads start with 96 registers each: 40 + 2 x 120 + 2 x 96 = 472 of 480 for a thread of every warpgroup
    if (warp < SOFTMAX0) {
    if (Q8) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0) {
        if (lane == 0 && any) {
            tc5::prefetch_tensormap(&tmQ);
            mbar_expect_tx(q_full, C::ATOMS * 128 * p.group * p.tile_tokens);
#pragma unroll
            for (int c = 0; c < C::ATOMS; ++c) tma_load_5d(sQ + c * 16384, &tmQ, q_full, c * 64, 0, t0, kv * p.q_mul[0], e * p.q_mul[1]);
        }
        if (!Q8 && lane < 2) {
            // lane 0 feeds the key blocks, lane 1 the value blocks
            const CUtensorMap* map = lane == 0 ? &tmK : &tmV;
            tc5::prefetch_tensormap(map);
            const int y = lane == 0 ? kv * p.k_mul[0] : kv * p.v_mul[0], z = lane == 0 ? e * p.k_mul[1] : e * p.v_mul[1];
            int n = 0;
            for (int i = walk.next(0); i < walk.count; i = walk.next(i + 1), ++n) {
                const int st = n % C::STAGES, key = (walk.first + i) * BKEY;
                const uint32_t full = lane == 0 ? k_full(st) : v_full(st), empty = lane == 0 ? k_empty(st) : v_empty(st);
                if (!mbar_wait(empty, (uint32_t)((n / C::STAGES) & 1) ^ 1u, abort_flag)) break;
                mbar_expect_tx(full, C::KV_BYTES);
                if (lane == 0) {
#pragma unroll
                    for (int c = 0; c < C::ATOMS; ++c) tma_load_4d(sK(st) + c * 16384, map, full, c * 64, key, y, z);
                } else {
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                        for (int c = 0; c < C::ATOMS; ++c)
                            tma_load_4d(sV(st) + kb * (C::KV_BYTES / 2) + c * 8192, map, full, c * 64, key + kb * 64, y, z);
                }
            }
        }
    } else if (warp == 1) {
        if (tc5::elect_one()) {
            constexpr uint32_t type = Q8 ? 0u : 1u;      // fp16 or bf16 operands
            constexpr uint32_t id_qk = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)(BKEY >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
            constexpr uint32_t id_pv = (1u << 4) | (type << 7) | (type << 10) | (1u << 16) | ((uint32_t)(HDP >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
            auto issue_qk = [&](int n) -> bool {
                const int b = n & 1, st = n % C::STAGES;
                if (!mbar_wait(k_full(st), (uint32_t)((n / C::STAGES) & 1), abort_flag)) return false;
                if (!mbar_wait(s_empty(b), (uint32_t)((n >> 1) & 1) ^ 1u, abort_flag)) return false;
                tc5::tc_fence_after();
#pragma unroll
                for (int kk = 0; kk < HDP / 16; ++kk) {
                    const uint64_t ad = smem_desc(sQ + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024);
                    const uint64_t bd = smem_desc(sK(st) + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024);
                    tc5::umma_bf16(tmem + b * BKEY, ad, bd, id_qk, kk > 0 ? 1u : 0u);
                }
                tc5::umma_commit(k_empty(st));
                tc5::umma_commit(s_full(b));
                return true;
            };
            int i = walk.next(0), n = 0;
            bool ok = i < walk.count && mbar_wait(Q8 ? q_ready : q_full, 0, abort_flag);
            tc5::tc_fence_after();
            if (ok) ok = issue_qk(0);
            for (; i < walk.count && ok; ++n) {
                i = walk.next(i + 1);
                if (i < walk.count) { ok = issue_qk(n + 1); if (!ok) break; }
                const int st = n % C::STAGES;
                if (!mbar_wait(p_full, (uint32_t)(n & 1), abort_flag)) break;
                if (!mbar_wait(v_full(st), (uint32_t)((n / C::STAGES) & 1), abort_flag)) break;
                tc5::tc_fence_after();
#pragma unroll
                for (int k16 = 0; k16 < BKEY / 16; ++k16) {
                    const uint64_t ad = smem_desc(sP + (k16 >> 2) * 16384 + (k16 & 3) * 32, 16, 1024);
                    const uint64_t bd = smem_desc(sV(st) + (k16 >> 2) * (C::KV_BYTES / 2) + (k16 & 3) * 2048, 8192, 1024);
                    tc5::umma_bf16(tmem + C::O_COL, ad, bd, id_pv, (n > 0 || k16 > 0) ? 1u : 0u);
                }
                tc5::umma_commit(v_empty(st));
                tc5::umma_commit(p_empty);
                tc5::umma_commit(o_done);
            }
        }
    }
    } else if (warp < CONVERT0) {
        if (Q8) asm volatile("setmaxnreg.inc.sync.aligned.u32 120;");
        // Softmax. Every thread runs every iteration and every named barrier even after a wait has given up (`ok` false), so nobody is left behind.
        const int quad = warp & 3, half = (warp - SOFTMAX0) >> 2;      // TMEM lane group this warp may access; which 64 keys of a block
        const int row = quad * 32 + lane;
        const uint32_t t_lane = (uint32_t)(quad * 32) << 16;
        float* xch = reinterpret_cast<float*>(gen + C::OFF_X);
        const bool busy = quad * 32 < tokens * p.group;                // a warp without rows only signals
        const int t = row / p.group, h = kv * p.group + row - t * p.group;
        const bool mine = t < tokens;
        const int pos = s.start + t0 + t;
        const int limit = a.causal ? max(pos, s.prefix - 1) : 0x7fffffff;
        const int key_limit = a.k_pos || !a.causal ? s.L : min(s.L, limit < 0x7fffffff ? limit + 1 : limit);
        const int doc = a.q_docs && mine ? a.q_docs[(size_t)e * a.tokens + t0 + t] : -1;
        const float slope = a.slopes && mine ? a.slopes[h] * kLog2e : 0.f;
        const bool capped = a.cap > 0.f;
        float factor = capped ? a.scale / a.cap : a.scale * kLog2e;    // to the cap's argument, or straight to log2 units
        const float cap2 = a.cap * kLog2e;
        bool ok = true;
        auto pair_barrier = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory"); };

        if (Q8 && any) {
            // Q from bf16 to fp16, each row by its own power of two
            ok = mbar_wait(q_full, 0, abort_flag);
            __syncwarp();
            if (busy) {
                uint32_t amax = 0;
                for (int c = 0; c < C::ATOMS; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4 u = *reinterpret_cast<const uint4*>(gen + C::OFF_Q + c * 16384 + row * 128 + (((half * 4 + i) ^ (row & 7)) << 4));
                        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) amax = max(amax, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
                    }
                xch[half * BQ + row] = __uint_as_float(amax);
                pair_barrier();
                amax = max(amax, __float_as_uint(xch[(half ^ 1) * BQ + row]));
                const int ex = min(max((int)(amax >> 7) - 127, -126), 126);
                const float down = __int_as_float((127 - ex) << 23);
                factor *= __int_as_float((127 + ex) << 23);
                for (int c = 0; c < C::ATOMS; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint4* at = reinterpret_cast<uint4*>(gen + C::OFF_Q + c * 16384 + row * 128 + (((half * 4 + i) ^ (row & 7)) << 4));
                        const uint4 u = *at;
                        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
                        uint32_t o[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) { const float2 f = unpack_bf16x2(w[k]); o[k] = pack_f16x2(f.x * down, f.y * down); }
                        *at = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                pair_barrier();                                        // xch is free again
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) tc5::mbar_arrive(q_ready);
        }

        float m_used = -INFINITY, l = 0.f;
        int n = 0;
        for (int i = walk.next(0); i < walk.count; i = walk.next(i + 1), ++n) {
            const int b = n & 1, key0 = (walk.first + i) * BKEY + half * 64;
            float kf[4], lv[4];                                        // (8-bit cache) per 16 keys: factor of the scores, log2 of V's scale
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                kf[g] = factor; lv[g] = 0.f;
                if (Q8) {
                    const size_t at = ((size_t)e * (a.keys / a.block) + min(key0 + g * 16, a.keys - 1) / a.block) * a.kv_heads + kv;
                    kf[g] = factor * __ldg(a.k_scale + at);
                    lv[g] = (float)((int)(__float_as_uint(__ldg(a.v_scale + at)) >> 23) - 127);
                }
            }
            ok = ok && mbar_wait(s_full(b), (uint32_t)((n >> 1) & 1), abort_flag);
            __syncwarp();                                              // the TMEM accesses below are warp-collective
            tc5::tc_fence_after();
            uint32_t r[64];
            if (busy) {
                ld32_nowait(tmem + t_lane + b * BKEY + half * 64, r);
                ld32_nowait(tmem + t_lane + b * BKEY + half * 64 + 32, r + 32);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            }
            tc5::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc5::mbar_arrive(s_empty(b));
            // keys whose values may be anything: behind the last one, or under a negative document
            bool tail = !Q8 && (walk.first + i + 1) * BKEY > s.L;
            if (walk.range != nullptr) tail = tail || __ldg(walk.range + walk.first + i).x < 0;
            if (busy) {
                float (&v)[64] = reinterpret_cast<float (&)[64]>(r);
                if (capped) {
#pragma unroll
                    for (int c = 0; c < 64; ++c) v[c] = cap2 * tanh_f(v[c] * kf[c >> 4]);
                } else {
#pragma unroll
                    for (int c = 0; c < 64; ++c) v[c] *= kf[c >> 4];
                }
                if (a.slopes) {
                    const float d0 = (float)(pos - key0);
                    if (a.k_pos) {
#pragma unroll
                        for (int c = 0; c < 64; ++c) v[c] = fmaf(-slope, fabsf((float)(pos - __ldg(a.k_pos + (size_t)e * a.keys + min(key0 + c, a.keys - 1)))), v[c]);
                    } else {
#pragma unroll
                        for (int c = 0; c < 64; ++c) v[c] = fmaf(-slope, fabsf(d0 - (float)c), v[c]);
                    }
                }
                // visible keys, as bits
                uint32_t see[2] = {0xffffffffu, 0xffffffffu};
                if (key0 + 64 > key_limit) {
                    const int have = max(0, key_limit - key0);
                    see[0] = have >= 32 ? 0xffffffffu : (1u << have) - 1u;
                    see[1] = have >= 64 ? 0xffffffffu : (have > 32 ? (1u << (have - 32)) - 1u : 0u);
                }
                if (walk.range != nullptr) {
                    // a lane looks at two keys; one vote for each document among the warp's rows (one or two, as a rule)
                    const int* tag = a.k_docs + (size_t)e * a.keys;
                    const int low = __ldg(tag + min(key0 + lane, a.keys - 1)), high = __ldg(tag + min(key0 + 32 + lane, a.keys - 1));
                    uint32_t left = __ballot_sync(0xffffffffu, doc >= 0);
                    if (doc < 0) see[0] = see[1] = 0u;
                    while (left) {
                        const int d = __shfl_sync(0xffffffffu, doc, __ffs(left) - 1);
                        const uint32_t b0 = __ballot_sync(0xffffffffu, low == d), b1 = __ballot_sync(0xffffffffu, high == d);
                        if (doc == d) { see[0] &= b0; see[1] &= b1; }
                        left &= ~__ballot_sync(0xffffffffu, doc == d);
                    }
                }
                if (a.k_pos && a.causal) {
                    const int* at = a.k_pos + (size_t)e * a.keys;
                    uint32_t seen[2] = {0u, 0u};
#pragma unroll
                    for (int c = 0; c < 64; ++c)
                        if (__ldg(at + min(key0 + c, a.keys - 1)) <= limit) seen[c >> 5] |= 1u << (c & 31);
                    see[0] &= seen[0];
                    see[1] &= seen[1];
                }
                // what is hidden becomes -infinity, and 2^-infinity is 0
                if (!__all_sync(0xffffffffu, (see[0] & see[1]) == 0xffffffffu)) {
#pragma unroll
                    for (int c = 0; c < 64; ++c) v[c] = see[c >> 5] & (1u << (c & 31)) ? v[c] : -INFINITY;
                }
                if (Q8 && p.scores != nullptr && mine) {
                    float4* dst = reinterpret_cast<float4*>(p.scores + (((size_t)e * a.heads + h) * a.tokens + t0 + t) * p.pitch + key0);
#pragma unroll
                    for (int c = 0; c < 64; c += 4) dst[c / 4] = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 64; ++c) top[c >> 4] = fmaxf(top[c >> 4], v[c]);
                float mx = fmaxf(fmaxf(top[0] + lv[0], top[1] + lv[1]), fmaxf(top[2] + lv[2], top[3] + lv[3]));
                if (n > 0) pair_barrier();                             // the maxima of the block before have been read
                xch[half * BQ + row] = mx;
                pair_barrier();
                mx = fmaxf(mx, xch[(half ^ 1) * BQ + row]);
                const bool grow = m_used != -INFINITY && mx > m_used + RESCALE_THRESHOLD;
                if (__any_sync(0xffffffffu, grow)) {
                    // the accumulator must be quiet while it is rescaled: the products of the block before have to be complete
                    ok = ok && (n == 0 || mbar_wait(o_done, (uint32_t)((n - 1) & 1), abort_flag));
                    __syncwarp();
                    tc5::tc_fence_after();
                    const float alpha = grow ? fast_exp2(m_used - mx) : 1.0f;
#pragma unroll 1
                    for (int c = 0; c < HDP / 64; ++c) {
                        float o[32];
                        const uint32_t at = tmem + t_lane + C::O_COL + half * (HDP / 2) + c * 32;
                        tc5::tmem_ld32(at, o);
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] *= alpha;
                        st32(at, o);
                    }
                    l *= alpha;
                    tc5::tc_fence_before();
                }
                if (grow || m_used == -INFINITY) m_used = mx;
                const float m = m_used == -INFINITY ? 0.f : m_used;    // (nothing but NaN, or nothing at all, so far)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float sum = 0.f;
                    const float off = lv[g] - m;
#pragma unroll
                    for (int c = g * 16; c < g * 16 + 16; ++c) {
                        v[c] = fast_exp2(v[c] + off);
                        sum += v[c];
                    }
                    l += Q8 ? sum * fast_exp2(-lv[g]) : sum;
                }
            }
            ok = ok && mbar_wait(p_empty, (uint32_t)(n & 1) ^ 1u, abort_flag);      // the products of the block before have read P
            __syncwarp();
            if (busy) {
                const float (&v)[64] = reinterpret_cast<const float (&)[64]>(r);
                // 8 keys = 16 bytes = one piece of this row's 128 bytes in atom `half`, 128-byte swizzle
#pragma unroll
                for (int piece = 0; piece < 8; ++piece) {
                    uint32_t o[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float lo = v[piece * 8 + 2 * k], hi = v[piece * 8 + 2 * k + 1];
                        o[k] = Q8 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
                    }
                    *reinterpret_cast<uint4*>(gen + C::OFF_P + half * 16384 + row * 128 + ((piece ^ (row & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
                }
            }
            if (tail) {
                // zeros in the place of those values: 0 * NaN would reach every row
                const int st = n % C::STAGES, key = (tid - 32 * SOFTMAX0) >> 1, at = (walk.first + i) * BKEY + key;
                const bool bad = at >= s.L || (walk.range != nullptr && __ldg(a.k_docs + (size_t)e * a.keys + at) < 0);
                if (!Q8) {
                    ok = ok && mbar_wait(v_full(st), (uint32_t)((n / C::STAGES) & 1), abort_flag);
                    if (bad)
                        for (int c = 0; c < C::ATOMS; ++c)
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                *reinterpret_cast<uint4*>(gen + C::OFF_V + st * C::KV_BYTES + (key >> 6) * (C::KV_BYTES / 2) + c * 8192 + (key & 63) * 128 + (tid & 1) * 64 + k * 16) =
                                    make_uint4(0, 0, 0, 0);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");            // P -> visible to the MMA
            tc5::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc5::mbar_arrive(p_full);
        }
        if (n > 0) ok = ok && mbar_wait(o_done, (uint32_t)((n - 1) & 1), abort_flag);
        __syncwarp();
        tc5::tc_fence_after();
        if (busy) {
            // the row's sum from its two threads, then half of the columns each
            pair_barrier();                                                          // the last maxima have been read
            xch[half * BQ + row] = l;
            pair_barrier();
            l += xch[(half ^ 1) * BQ + row];
            const size_t flat = ((size_t)e * a.tokens + t0 + (mine ? t : 0)) * a.heads + h;
            const bool store = ok && mine;
            if (p.splits > 1) {
                const size_t at = (size_t)split * a.episodes * a.tokens * a.heads + flat;
                if (store && half == 0) p.part_ml[at] = make_float2(m_used, l);
#pragma unroll 1
                for (int c = 0; c < (n > 0 ? HDP / 64 : 0); ++c) {
                    float o[32];
                    tc5::tmem_ld32(tmem + t_lane + C::O_COL + half * (HDP / 2) + c * 32, o);
                    if (store) {
                        float4* dst = reinterpret_cast<float4*>(p.part_o + at * HDP + half * (HDP / 2) + c * 32);
#pragma unroll
                        for (int k = 0; k < 8; ++k) dst[k] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                    }
                    __syncwarp();
                }
            } else {
                const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);         // NaN stays
                if (store && half == 0 && a.lse)
                    a.lse[((size_t)e * a.heads + h) * a.tokens + t0 + t] = l > 0.f ? ((m_used == -INFINITY ? 0.f : m_used) + log2f(l)) * 0.6931471805599453f : (l == 0.f ? -INFINITY : l);
                bf16* dst = a.out + e * a.os[0] + (t0 + (mine ? t : 0)) * a.os[1] + h * a.os[2];
#pragma unroll 1
                for (int c = 0; c < HDP / 64; ++c) {
                    float o[32];
                    const int col = half * (HDP / 2) + c * 32;
                    if (n > 0) tc5::tmem_ld32(tmem + t_lane + C::O_COL + col, o);
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = n > 0 ? o[k] * inv : 0.f;
                    if (store) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (col + k * 8 < a.dim)
                                *reinterpret_cast<uint4*>(dst + col + k * 8) = make_uint4(pack_bf16x2(o[8 * k], o[8 * k + 1]), pack_bf16x2(o[8 * k + 2], o[8 * k + 3]),
                                                                                        pack_bf16x2(o[8 * k + 4], o[8 * k + 5]), pack_bf16x2(o[8 * k + 6], o[8 * k + 7]));
                    }
                    __syncwarp();
                }
            }
        }
    } else if (Q8) {
        // e4m3 -> fp16 operands: warps 12-15 the keys, 16-19 the values
        const bool values = warp >= CONVERT0 + 4;
        const int ct = tid - 32 * (values ? CONVERT0 + 4 : CONVERT0);
        const uint8_t* src = values ? static_cast<const uint8_t*>(a.v) + e * a.vs[0] + kv * a.vs[2] : static_cast<const uint8_t*>(a.k) + e * a.ks[0] + kv * a.ks[2];
        const long long pitch = values ? a.vs[1] : a.ks[1];
        constexpr int CHUNKS = HDP / 16, PER = BKEY * CHUNKS / 128;      // 16-byte chunks of a row; of a block, per thread
        uint4 held[PER];
        auto fetch = [&](int i) {
#pragma unroll
            for (int c = 0; c < PER; ++c) {
                const int at = c * 128 + ct, key = (walk.first + i) * BKEY + at / CHUNKS, col = at % CHUNKS * 16;
                held[c] = key < s.L && col < a.dim ? __ldg(reinterpret_cast<const uint4*>(src + key * pitch + col)) : make_uint4(0, 0, 0, 0);
            }
        };
        int i = walk.next(0), n = 0;
        if (i < walk.count) fetch(i);
        bool ok = true;
        for (; i < walk.count && ok; ++n) {
            const int st = n % C::STAGES;
            const uint32_t full = values ? v_full(st) : k_full(st), empty = values ? v_empty(st) : k_empty(st);
            ok = mbar_wait(empty, (uint32_t)((n / C::STAGES) & 1) ^ 1u, abort_flag);
            __syncwarp();
            uint8_t* dst = gen + (values ? C::OFF_V : C::OFF_K) + st * C::KV_BYTES;
#pragma unroll
            for (int c = 0; c < PER; ++c) {
                const int at = c * 128 + ct, key = at / CHUNKS, atom = at % CHUNKS >> 2, piece = (at & 3) * 2;
                const uint4 u = held[c];
                const uint4 low = make_uint4(e4m3x2_to_f16x2(u.x & 0xffffu), e4m3x2_to_f16x2(u.x >> 16), e4m3x2_to_f16x2(u.y & 0xffffu), e4m3x2_to_f16x2(u.y >> 16));
                const uint4 high = make_uint4(e4m3x2_to_f16x2(u.z & 0xffffu), e4m3x2_to_f16x2(u.z >> 16), e4m3x2_to_f16x2(u.w & 0xffffu), e4m3x2_to_f16x2(u.w >> 16));
                uint8_t* line = dst + (values ? (key >> 6) * (C::KV_BYTES / 2) + atom * 8192 + (key & 63) * 128 : atom * 16384 + key * 128);
                // lanes 4-7 of eight begin with the other half, so that the eight stores of a phase fall on eight bank groups
                const bool swap = (lane & 4) != 0;
                *reinterpret_cast<uint4*>(line + (((piece + (swap ? 1 : 0)) ^ (key & 7)) << 4)) = swap ? high : low;
                *reinterpret_cast<uint4*>(line + (((piece + (swap ? 0 : 1)) ^ (key & 7)) << 4)) = swap ? low : high;
            }
            i = walk.next(i + 1);
            if (i < walk.count) fetch(i);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) tc5::mbar_arrive(full);
        }
    }

    tc5::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc5::tc_fence_after();
        tc5::tmem_dealloc(tmem, 512);
    }
    if (tid == 0 && *abort_flag && p.status) atomicExch(p.status, 9);
}

// The shares' sums against the largest of their maxima. `warps` of a CTA take 32 * PER columns of a row together (grid.y: which): each adds up every
// warps-th share, and the first adds up the warps in their order.
constexpr int JOIN_WARPS = 8;
template <int PER>
__global__ void __launch_bounds__(32 * JOIN_WARPS) attention_join_kernel(const __grid_constant__ Tile p, int hdp, int warps) {
    __shared__ float sums[JOIN_WARPS][32 * PER + 1];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Args& a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % warps, col0 = blockIdx.y * 32 * PER + lane;
    const long long row = (long long)blockIdx.x * (JOIN_WARPS / warps) + warp / warps, rows = (long long)a.episodes * a.tokens * a.heads;
    const int h = (int)(row % a.heads), t = (int)(row / a.heads % a.tokens), e = (int)min(row / a.heads / a.tokens, (long long)a.episodes - 1);
    const bool mine = row < rows && t < episode_of(a, e).n;
    // no load waits for another, but for the maxima: shares that held nothing are read as well, and dropped
    float m = -INFINITY;
#pragma unroll 4
    for (int s = lane; s < p.splits; s += 32) {
        const float2 ml = mine ? p.part_ml[s * rows + row] : make_float2(0.f, 0.f);
        if (ml.y != 0.f) m = fmaxf(m, ml.x);
    }
    m = warp_max(m);
    const float top = m == -INFINITY ? 0.f : m;
    float acc[PER], l = 0.f;                                                         // columns lane, lane + 32, ...
#pragma unroll
    for (int c = 0; c < PER; ++c) acc[c] = 0.f;
    const float* o = p.part_o + (mine ? row : 0) * hdp + col0;
    const size_t pitch = (size_t)rows * hdp;
    for (int s0 = part; s0 < p.splits; s0 += 32 * warps) {
        // lane i: the factor of share s0 + i * warps
        const int s = s0 + lane * warps;
        const float2 ml = mine && s < p.splits ? p.part_ml[s * rows + row] : make_float2(0.f, 0.f);
        const float w = ml.y == 0.f ? 0.f : (ml.x == -INFINITY ? 1.f : fast_exp2(ml.x - top));
        l += warp_sum(ml.y == 0.f ? 0.f : ml.y * w);
        const int have = min(32, (p.splits - s0 + warps - 1) / warps);
#pragma unroll (PER == 1 ? 16 : 4)
        for (int i = 0; i < have; ++i) {
            const float f = __shfl_sync(0xffffffffu, w, i), used = __shfl_sync(0xffffffffu, ml.y, i);
#pragma unroll
            for (int c = 0; c < PER; ++c) {
                const float x = o[(size_t)(s0 + i * warps) * pitch + 32 * c];
                acc[c] = fmaf(f, used != 0.f ? x : 0.f, acc[c]);
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
    bf16* dst = a.out + e * a.os[0] + t * a.os[1] + h * a.os[2];
#pragma unroll
    for (int c = 0; c < PER; ++c)
        if (col0 + 32 * c < a.dim) dst[col0 + 32 * c] = __float2bfloat16_rn(acc[c] * inv);
    if (a.lse && lane == 0 && blockIdx.y == 0) a.lse[((size_t)e * a.heads + h) * a.tokens + t] = l > 0.f ? (top + log2f(l)) * 0.6931471805599453f : (l == 0.f ? -INFINITY : l);
}

// weights[e][j] = decay * weights[e][j] + the probabilities that key j got, from the scores that the attention left and the rows' log-sum-exps. A CTA
// has 32 keys; its warps share out the rows, and their sums are added in the order of the warps.
constexpr int WEIGHT_WARPS = 16;
__global__ void __launch_bounds__(32 * WEIGHT_WARPS) key_weights_kernel(const __grid_constant__ Tile p) {
    __shared__ float part[WEIGHT_WARPS][32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Args& a = p.a;
    const int e = blockIdx.y, j = blockIdx.x * 32 + (threadIdx.x & 31), warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const Episode s = episode_of(a, e);
    const bool inside = j < s.L, by_number = a.causal && a.k_pos == nullptr;
    const int rows = a.heads * s.n;
    const size_t row0 = (size_t)e * a.heads * a.tokens;
    // tokens before this one do not see key j (by its number), and their scores were not left
    const int from = by_number && j >= s.prefix ? max(0, j - s.start) : 0;
    float sum = 0.f;
#pragma unroll 8
    for (int r = warp; r < rows; r += warps) {
        const int h = r / s.n, t = r - h * s.n;
        const size_t row = row0 + (size_t)h * a.tokens + t;
        const float z = a.lse[row], x = p.scores[row * p.pitch + j];      // what was not left is read as well (j < pitch), and dropped
        if (inside && t >= from && z != -INFINITY) sum += fast_exp2(fmaf(z, -kLog2e, x));
    }
    part[warp][threadIdx.x & 31] = sum;
    __syncthreads();
    if (warp != 0 || !inside) return;
    for (int w = 1; w < warps; ++w) sum += part[w][threadIdx.x];
    float* at = a.weights + (size_t)e * a.keys + j;
    *at = (a.decay != 0.f ? a.decay * *at : 0.f) + sum;
}

// Tensor map of a strided operand, innermost axis contiguous; an axis of stride 0 is left at one element (its coordinate is 0).
inline int make_map(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const uint64_t* strides, const uint32_t* box, int elem = 2) {
    tc5::EncodeTiledFn fn = tc5::encode_fn();
    if (fn == nullptr) { set_error("cuTensorMapEncodeTiled is not available from the driver"); return FVLA_ERR_LAUNCH; }
    cuuint64_t gdim[5], gstride[4];
    cuuint32_t b[5], step[5];
    for (int i = 0; i < rank; ++i) { gdim[i] = dims[i]; b[i] = box[i]; step[i] = 1; }
    for (int i = 0; i + 1 < rank; ++i) gstride[i] = strides[i] * elem;
    const CUresult r = fn(map, elem == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), gdim, gstride, b, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) { set_error("attention: cuTensorMapEncodeTiled failed with CUresult %d", (int)r); return FVLA_ERR_ARG; }
    return FVLA_OK;
}

}  // namespace mattn
}  // namespace fvla

#include "few_rows_attention.cuh"

namespace fvla {
namespace mattn {

// Up to 32 rows per episode and K/V head, and no documents: the kernel for few rows.
inline bool takes_few(const Args& a) { return (long long)a.tokens * (a.heads / a.kv_heads) <= 32 && a.q_docs == nullptr; }
// Head dimension that the kernel is built for.
inline int padded_dim(const Args& a) { return a.dim <= 64 && !takes_few(a) ? 64 : (a.dim <= 128 ? 128 : 256); }

constexpr int CLUSTER = 8;      // shares that a cluster puts together
// Shares of the key blocks: as many as bring the CTAs up to the number that are resident, at most one per block.
inline int plan_splits(const Args& a) {
    const int group = a.heads / a.kv_heads, tile_tokens = BQ / group, blocks = (a.keys + BKEY - 1) / BKEY;
    const bool few = takes_few(a);
    const long long tiles = (few ? 1ll : (long long)((a.tokens + tile_tokens - 1) / tile_tokens)) * a.kv_heads * a.episodes;
    int per_sm = 1;
    if (few) {
        const int tile_bytes = 128 * padded_dim(a) * (a.k_scale ? 1 : 2);
        per_sm = few_rows(a) == 32 ? (tile_bytes == 16384 ? 2 : 1) : (tile_bytes == 16384 ? 3 : (tile_bytes == 32768 ? 2 : 1));
    }
    const long long room = (long long)tc5::num_sms() * per_sm * (few && tiles > tc5::num_sms() ? 2 : 1) / tiles;
    if (few && room > CLUSTER && blocks <= 2 * CLUSTER) return blocks < CLUSTER ? (blocks > 0 ? blocks : 1) : CLUSTER;      // no second launch for two blocks each
    return (int)(room < 1 ? 1 : (room < blocks ? room : (blocks > 0 ? blocks : 1)));
}
inline size_t score_pitch(const Args& a) { return ((size_t)a.keys + BKEY - 1) / BKEY * BKEY; }
inline size_t align256(size_t v) { return (v + 255) / 256 * 256; }
inline size_t workspace_bytes(const Args& a) {
    const int splits = plan_splits(a);
    const size_t rows = (size_t)a.episodes * a.tokens * a.heads;
    size_t n = a.q_docs ? align256((size_t)a.episodes * ((a.keys + BKEY - 1) / BKEY) * sizeof(int2)) : 0;
    if (a.weights) n += rows * score_pitch(a) * sizeof(float);
    if (splits > (takes_few(a) ? CLUSTER : 1)) n += align256(splits * rows * sizeof(float2)) + splits * rows * padded_dim(a) * sizeof(float);
    return n;
}

inline int launch_join(const Tile& p, int hdp, cudaStream_t st) {
    const long long rows = (long long)p.a.episodes * p.a.tokens * p.a.heads;
    // many shares: eight warps for 32 columns of a row; few: a warp or some for the whole row
    const int warps = p.splits >= 16 ? 8 : (p.splits >= 8 ? 4 : (p.splits >= 4 ? 2 : 1)), each = JOIN_WARPS / warps, per = p.splits >= 16 ? 1 : hdp / 32;
    const auto kern = per == 1 ? attention_join_kernel<1> : (per == 2 ? attention_join_kernel<2> : (per == 4 ? attention_join_kernel<4> : attention_join_kernel<8>));
    const cudaError_t e = launch_pdl(kern, dim3((unsigned)((rows + each - 1) / each), hdp / (32 * per)), dim3(32 * JOIN_WARPS), 0, st, p, hdp, warps);
    if (e != cudaSuccess) { set_error("attention_join_kernel: %s", cudaGetErrorString(e)); return FVLA_ERR_LAUNCH; }
    return check_launch("attention_join_kernel");
}

template <int HDP, bool Q8>
inline int launch_tile(const Tile& p, const CUtensorMap& tmQ, const CUtensorMap& tmK, const CUtensorMap& tmV, cudaStream_t st) {
    using C = Cfg<HDP, Q8>;
    auto kern = attention_tile_kernel<HDP, Q8>;
    static PerDeviceFlag configured;
    if (!configured.get()) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) { set_error("cudaFuncSetAttribute: %s", cudaGetErrorString(e)); return FVLA_ERR_LAUNCH; }
        configured.set();
    }
    const Args& a = p.a;
    cudaError_t e = launch_pdl(kern, dim3(p.tiles * p.splits, a.kv_heads, a.episodes), dim3(C::THREADS), C::SMEM, st, p, tmQ, tmK, tmV);
    if (e != cudaSuccess) { set_error("attention_tile_kernel: %s", cudaGetErrorString(e)); return FVLA_ERR_LAUNCH; }
    int rc = check_launch("attention_tile_kernel");
    return rc || p.splits == 1 ? rc : launch_join(p, HDP, st);
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
    if (a.weights) {
        p.scores = reinterpret_cast<float*>(at);
        at += rows * p.pitch * sizeof(float);
    }
    p.part_ml = reinterpret_cast<float2*>(at);
    p.part_o = reinterpret_cast<float*>(at + align256(p.splits * rows * sizeof(float2)));
    CUtensorMap tmQ = {}, tmK = {}, tmV = {};
    const bool few = takes_few(a), q8 = a.k_scale != nullptr;
    p.q_mul[0] = 1;
    p.q_mul[1] = a.qs[0] != 0;
    if (!few) {
        const uint64_t dims[5] = {(uint64_t)a.dim, (uint64_t)p.group, (uint64_t)a.tokens, (uint64_t)a.kv_heads, p.q_mul[1] ? (uint64_t)a.episodes : 1};
        const uint64_t strides[4] = {(uint64_t)a.qs[2], (uint64_t)a.qs[1], (uint64_t)a.qs[2] * p.group, p.q_mul[1] ? (uint64_t)a.qs[0] : 256};
        const uint32_t box[5] = {64, (uint32_t)p.group, (uint32_t)p.tile_tokens, 1, 1};
        const int rc = make_map(&tmQ, a.q, 5, dims, strides, box);
        if (rc) return rc;
    }
    p.k_mul[0] = a.ks[2] != 0; p.k_mul[1] = a.ks[0] != 0; p.v_mul[0] = a.vs[2] != 0; p.v_mul[1] = a.vs[0] != 0;
    if ((few || !q8) && a.keys > 0) {
        for (int i = 0; i < 2; ++i) {
            const long long* s = i == 0 ? a.ks : a.vs;
            const int* mul = i == 0 ? p.k_mul : p.v_mul;
            const uint64_t dims[4] = {(uint64_t)a.dim, (uint64_t)a.keys, mul[0] ? (uint64_t)a.kv_heads : 1, mul[1] ? (uint64_t)a.episodes : 1};
            const uint64_t strides[3] = {(uint64_t)s[1], mul[0] ? (uint64_t)s[2] : 256, mul[1] ? (uint64_t)s[0] : 256};
            const uint32_t box[4] = {q8 ? 128u : 64u, i == 0 || few ? 128u : 64u, 1, 1};
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
        rc = hdp == 64 ? launch_tile<64, true>(p, tmQ, tmK, tmV, st) : (hdp == 128 ? launch_tile<128, true>(p, tmQ, tmK, tmV, st) : launch_tile<256, true>(p, tmQ, tmK, tmV, st));
    } else {
        rc = hdp == 64 ? launch_tile<64, false>(p, tmQ, tmK, tmV, st) : (hdp == 128 ? launch_tile<128, false>(p, tmQ, tmK, tmV, st) : launch_tile<256, false>(p, tmQ, tmK, tmV, st));
    }
    if (rc || a.weights == nullptr || a.keys == 0) return rc;
    const int rows_each = a.tokens * a.heads, warps = rows_each < 4 * WEIGHT_WARPS ? (rows_each + 3) / 4 : WEIGHT_WARPS;      // four rows or more for a warp
    const cudaError_t e = launch_pdl(key_weights_kernel, dim3((a.keys + 31) / 32, a.episodes), dim3(32 * warps), 0, st, p);
    if (e != cudaSuccess) { set_error("key_weights_kernel: %s", cudaGetErrorString(e)); return FVLA_ERR_LAUNCH; }
    return check_launch("key_weights_kernel");
}

}  // namespace mattn
}  // namespace fvla

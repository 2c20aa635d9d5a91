// Attention of few rows: a decoding step of at most 32 rows (tokens x the query heads of a K/V head), bound by the bytes of the cache: 32 episodes of
// up to 16 384 rows of 8 heads of 128, 805 MB, in 130 us, 0.95 of the measured copy rate (144 us at the clocks of a long run); with the cache converted
// to fp16 operands by warps of their own 730 us. One token over 819 rows is a chain of latencies, 8 us: lengths, Q, the tiles' first bytes, two products,
// the cluster's exchange.
//
// The keys are the 128-row operand of both products, so that every thread of the softmax has one key and all rows of it:
//   S^T (128 keys x rows) = K Q^T,      O^T (128 dims x rows, one or two halves) += V^T P^T
// K and V tiles go from TMA straight to the tensor cores, also the 8-bit ones (kind::f8f6f4): nothing is converted. Instead the few rows are split
// into e4m3 terms, each a row of the other operand. A bf16 q brought to 2^7..2^8 by its row's power of two is the sum of two terms of 4 bits, the second
// times 2^5 (exactly, but for elements below e4m3's smallest normal number, 2^-13 of the largest: 2^-4 of half its smallest step, 2^-21 of the largest). A
// probability is the sum of three (times 2^4 and 2^8): with the maximum at 2^4 it is off by at most 2^-12 of itself or 2^-22 of the row's largest.
// The scale of V moves into their exponent, and the row sum takes it back; where a share has very small or large scales (a block of zeros has 2^-120, and
// its inverse would end fp32's range), the row sum is taken from the scores themselves against a maximum of its own. What a share leaves is its maximum, its
// sums and the log2 of its row sum.
//   warp 0      TMA: K and V tiles of 128 keys in turn through a ring of SLOTS
//   warp 1      one lane issues the MMAs, S^T a block ahead
//   warps 2-5   softmax: thread = key. The rows' maxima by redux and through shared memory, sums kept per thread until the end.
// Each CTA has a share of an episode's blocks of one K/V head. Up to eight shares are a cluster: its CTAs leave their unnormalised sums in shared
// memory and each puts together a part of the result. More than eight leave them in scratch, and attention_join_kernel adds them up.
#pragma once

namespace fvla {
namespace mattn {

__device__ __forceinline__ float redux_max(float x) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}
// N consecutive columns (a multiple of 16) of this thread's TMEM lane.
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[N]) {
    uint32_t r[N];
    int c = 0;
#pragma unroll
    for (; c + 32 <= N; c += 32) ld32_nowait(taddr + c, r + c);
    if (c < N)
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
            : "=r"(r[N - 16]), "=r"(r[N - 15]), "=r"(r[N - 14]), "=r"(r[N - 13]), "=r"(r[N - 12]), "=r"(r[N - 11]), "=r"(r[N - 10]), "=r"(r[N - 9]),
              "=r"(r[N - 8]), "=r"(r[N - 7]), "=r"(r[N - 6]), "=r"(r[N - 5]), "=r"(r[N - 4]), "=r"(r[N - 3]), "=r"(r[N - 2]), "=r"(r[N - 1])
            : "r"(taddr + N - 16) : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void st16(uint32_t taddr, const float* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]),
          "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]) : "memory");
}

constexpr int FEW_THREADS = 192, CLUSTER = 8;      // shares that a cluster puts together

template <int HDP, bool Q8, int NR>
struct FewCfg {
    static constexpr int round16(int n) { return (n + 15) / 16 * 16; }
    static constexpr int QT = Q8 ? 2 : 1, PT = Q8 ? 3 : 1;               // terms of Q and of P
    static constexpr int NS = round16(NR * QT), NO = round16(NR * PT);   // columns of S^T and of a half of O^T
    static constexpr int HALVES = HDP / 128, ELEM = Q8 ? 1 : 2;
    static constexpr int ATOMS = HDP * ELEM / 128;                       // 128-byte columns of a tile
    static constexpr int TILE = ATOMS * 16384;
    static constexpr int KEY_ATOMS = 128 * ELEM / 128;                   // of P
    static constexpr int Q_BYTES = ATOMS * NS * 128, P_BYTES = KEY_ATOMS * NO * 128;
    // tiles in flight: three CTAs per SM with four tiles of 16 KB, two with three of 32 KB, one with three of 64 KB (32 rows: two, one, one)
    static constexpr int SLOTS = TILE == 16384 ? 4 : 3;
    static constexpr int PER_SM = NR == 32 ? (TILE == 16384 ? 2 : 1) : (TILE == 16384 ? 3 : (TILE == 32768 ? 2 : 1));
    static constexpr int OFF_Q = 0, OFF_P = OFF_Q + Q_BYTES, OFF_T = OFF_P + P_BYTES;
    static constexpr int OFF_F = OFF_T + SLOTS * TILE;                   // per row: factor, slope (floats), position, limit, number (ints)
    static constexpr int OFF_M = OFF_F + 5 * NR * 4;                     // maxima of the four warps, twice
    static constexpr int OFF_W = OFF_M + 2 * 4 * NR * 4;                 // of each warp, per row: the maximum in use, the factor of what is accumulated
    static constexpr int OFF_BAR = OFF_W + 4 * 2 * NR * 4;
    static constexpr int SMEM = 1024 + OFF_BAR + 160;
    static constexpr int S_COL = 0, O_COL = 2 * NS;
    static constexpr int USED = 2 * NS + HALVES * NO;
    static constexpr uint32_t COLS = USED <= 64 ? 64 : (USED <= 128 ? 128 : (USED <= 256 ? 256 : 512));
    static constexpr float SHIFT = Q8 ? 4.f : 0.f, THRESHOLD = Q8 ? 4.f : RESCALE_THRESHOLD;
};

template <int HDP, bool Q8, int NR>
__global__ void __launch_bounds__(FEW_THREADS, (FewCfg<HDP, Q8, NR>::PER_SM))
attention_few_rows_kernel(const __grid_constant__ Tile p, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV) {
    using C = FewCfg<HDP, Q8, NR>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t bars = base + C::OFF_BAR;
    const uint32_t q_ready = bars, p_full = bars + 8, o_done = bars + 16;
    auto s_full = [&](int b) { return bars + 24 + b * 8; };
    auto s_empty = [&](int b) { return bars + 40 + b * 8; };
    auto full = [&](int s) { return bars + 56 + s * 8; };
    auto empty = [&](int s) { return bars + 88 + s * 8; };
    volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(gen + C::OFF_BAR + 120);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + C::OFF_BAR + 124);
    volatile int* odd_scales = reinterpret_cast<volatile int*>(gen + C::OFF_BAR + 128);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Args& a = p.a;
    const int e = blockIdx.z, kv = blockIdx.y, split = blockIdx.x;

    if (tid == 0) {
        mbar_init(q_ready, 4); mbar_init(p_full, 4); mbar_init(o_done, 1);
        for (int b = 0; b < 2; ++b) { mbar_init(s_full(b), 1); mbar_init(s_empty(b), 4); }
        for (int s = 0; s < C::SLOTS; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        *abort_flag = 0;
        *odd_scales = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        tc5::tmem_alloc(bars + 120, C::COLS);
        tc5::tmem_relinquish();
    }
    tc5::tc_fence_before();
    __syncthreads();
    tc5::tc_fence_after();
    const uint32_t tmem = *tmem_slot_ptr;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // Q's rows are asked for before the lengths are known: a warp of the softmax has every fourth
    constexpr int PER = HDP / 32, Q_ROWS = NR / 4;                             // elements of a lane: 4 or 8; rows of a warp
    uint2 q_raw[Q_ROWS][PER / 4];
    if (warp >= 2) {
#pragma unroll
        for (int i = 0; i < Q_ROWS; ++i) {
            const int r = i * 4 + (warp & 3), t = r / p.group, h = kv * p.group + r - t * p.group, d = lane * PER;
#pragma unroll
            for (int k = 0; k < PER / 4; ++k) {
                q_raw[i][k] = make_uint2(0, 0);
                if (t < a.tokens && d + 4 * k < a.dim) q_raw[i][k] = __ldg(reinterpret_cast<const uint2*>(static_cast<const bf16*>(a.q) + e * a.qs[0] + t * a.qs[1] + h * a.qs[2] + d + 4 * k));
            }
        }
    }
    const Episode s = episode_of(a, e);
    int most = s.n > 0 ? s.L : 0;
    if (a.causal && a.k_pos == nullptr) most = max(0, min(most, max(s.start + s.n, s.prefix)));
    const int blocks = (most + BKEY - 1) / BKEY;
    const int first = (int)((long long)blocks * split / p.splits), count = (int)((long long)blocks * (split + 1) / p.splits) - first;

    if (warp == 0) {
        if (lane == 0 && count > 0) {
            tc5::prefetch_tensormap(&tmK);
            tc5::prefetch_tensormap(&tmV);
            for (int i = 0; i < 2 * count; ++i) {
                const int st = i % C::SLOTS;
                const CUtensorMap* map = i & 1 ? &tmV : &tmK;
                const int* mul = i & 1 ? p.v_mul : p.k_mul;
                if (!mbar_wait(empty(st), (uint32_t)((i / C::SLOTS) & 1) ^ 1u, abort_flag)) break;
                mbar_expect_tx(full(st), C::TILE);
#pragma unroll
                for (int c = 0; c < C::ATOMS; ++c)
                    tma_load_4d(base + C::OFF_T + st * C::TILE + c * 16384, map, full(st), c * (128 / C::ELEM), (first + (i >> 1)) * BKEY, kv * mul[0], e * mul[1]);
            }
        }
    } else if (warp == 1) {
        if (tc5::elect_one() && count > 0) {
            constexpr uint32_t type = Q8 ? 0u : 1u;                      // e4m3 or bf16
            constexpr uint32_t id_qk = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)(C::NS >> 3) << 17) | (8u << 24);
            constexpr uint32_t id_pv = (1u << 4) | (type << 7) | (type << 10) | (1u << 15) | ((uint32_t)(C::NO >> 3) << 17) | (8u << 24);
            auto mma = [&](uint32_t d, uint64_t ad, uint64_t bd, uint32_t id, bool acc) {
                if (Q8) umma_f8(d, ad, bd, id, acc);
                else tc5::umma_bf16(d, ad, bd, id, acc);
            };
            auto issue_qk = [&](int n) -> bool {
                const int st = 2 * n % C::SLOTS, b = n & 1;
                if (!mbar_wait(full(st), (uint32_t)((2 * n / C::SLOTS) & 1), abort_flag)) return false;
                if (!mbar_wait(s_empty(b), (uint32_t)((n >> 1) & 1) ^ 1u, abort_flag)) return false;
                tc5::tc_fence_after();
#pragma unroll
                for (int k = 0; k < 4 * C::ATOMS; ++k)                   // 32 bytes of the head dimension at a time
                    mma(tmem + C::S_COL + b * C::NS, smem_desc(base + C::OFF_T + st * C::TILE + (k >> 2) * 16384 + (k & 3) * 32, 16, 1024),
                        smem_desc(base + C::OFF_Q + (k >> 2) * (C::NS * 128) + (k & 3) * 32, 16, 1024), id_qk, k > 0);
                tc5::umma_commit(empty(st));
                tc5::umma_commit(s_full(b));
                return true;
            };
            bool ok = mbar_wait(q_ready, 0, abort_flag);
            tc5::tc_fence_after();
            ok = ok && issue_qk(0);
            for (int n = 0; n < count && ok; ++n) {
                if (n + 1 < count) { ok = issue_qk(n + 1); if (!ok) break; }
                const int st = (2 * n + 1) % C::SLOTS;
                if (!mbar_wait(p_full, (uint32_t)(n & 1), abort_flag)) break;
                if (!mbar_wait(full(st), (uint32_t)(((2 * n + 1) / C::SLOTS) & 1), abort_flag)) break;
                tc5::tc_fence_after();
                constexpr int KEYS = 32 / C::ELEM;                       // keys per MMA
#pragma unroll
                for (int h = 0; h < C::HALVES; ++h)
#pragma unroll
                    for (int k = 0; k < BKEY / KEYS; ++k)
                        mma(tmem + C::O_COL + h * C::NO, smem_desc(base + C::OFF_T + st * C::TILE + h * C::ELEM * 16384 + k * KEYS * 128, 16384, 1024),
                            smem_desc(base + C::OFF_P + (k >> 2) * (C::NO * 128) + (k & 3) * 32, 16, 1024), id_pv, n > 0 || k > 0);
                tc5::umma_commit(empty(st));
                tc5::umma_commit(o_done);
            }
        }
    } else {
        const int quad = warp & 3, key = quad * 32 + lane;                     // key of a block = TMEM lane
        const uint32_t t_lane = (uint32_t)(quad * 32) << 16;
        const int group = p.group, rows = s.n * group;                         // row = token * group + head
        float* row_f = reinterpret_cast<float*>(gen + C::OFF_F);
        float* row_slope = row_f + NR;
        int* row_pos = reinterpret_cast<int*>(row_f + 2 * NR);
        int* row_limit = row_pos + NR;
        int* row_number = row_limit + NR;                                      // in the log-sum-exps and scores of the episode
        float* maxima = reinterpret_cast<float*>(gen + C::OFF_M);
        float* in_use = reinterpret_cast<float*>(gen + C::OFF_W) + quad * 2 * NR;
        float* rescale = in_use + NR;
        const bool capped = a.cap > 0.f;
        auto barrier = []() { asm volatile("bar.sync 1, 128;" ::: "memory"); };
        bool ok = true;

        const float* ks = a.k_scale + (size_t)e * (Q8 ? a.keys / a.block : 0) * a.kv_heads + kv;
        const float* vs = a.v_scale + (size_t)e * (Q8 ? a.keys / a.block : 0) * a.kv_heads + kv;
        const int shift = Q8 ? 31 - __clz(a.block) : 0;                        // blocks are powers of two
        // a key's scales and position, fetched a block ahead
        float next_k = 1.f, next_v = 1.f;
        int next_pos = 0;
        auto fetch = [&](int n) {
            const int j = min((first + n) * BKEY + key, s.L - 1);             // (what lies behind the last row may be anything, scales too)
            if (Q8) {
                next_k = __ldg(ks + (size_t)(j >> shift) * a.kv_heads);
                next_v = __ldg(vs + (size_t)(j >> shift) * a.kv_heads);
            }
            if (a.k_pos) next_pos = __ldg(a.k_pos + (size_t)e * a.keys + j);
        };
        if (count > 0) {
            fetch(0);
            const int scale_end = Q8 ? (min((first + count) * BKEY, s.L) + a.block - 1) >> shift : 0, scale0 = (first * BKEY >> shift) + key;
            const float scale = scale0 < scale_end ? __ldg(vs + (size_t)scale0 * a.kv_heads) : 1.f;
            // Q as the K-major operand, and what the rows have of their own (rows of the operand behind NR, and their columns of S^T, are never looked at)
#pragma unroll
            for (int i = 0; i < Q_ROWS; ++i) {
                const int r = i * 4 + quad, t = r / group, h = kv * group + r - t * group;
                float q[PER];
                uint32_t amax = 0;
#pragma unroll
                for (int k = 0; k < PER / 4; ++k) {
                    const uint2 u = r < rows ? q_raw[i][k] : make_uint2(0, 0);
                    const float2 x = unpack_bf16x2(u.x), y = unpack_bf16x2(u.y);
                    q[4 * k] = x.x; q[4 * k + 1] = x.y; q[4 * k + 2] = y.x; q[4 * k + 3] = y.y;
                    amax = max(max(amax, max(u.x & 0x7fffu, (u.x >> 16) & 0x7fffu)), max(u.y & 0x7fffu, (u.y >> 16) & 0x7fffu));
                }
                float f = capped ? a.scale / a.cap : a.scale * kLog2e;
                const int at = lane * PER * C::ELEM;                            // byte within the row
                uint8_t* line = gen + C::OFF_Q + (at >> 7) * (C::NS * 128);
                const int piece = (at & 127) >> 4, in = at & 15;
                if (Q8) {
                    amax = __reduce_max_sync(0xffffffffu, amax);
                    const int ex = min(max((int)(amax >> 7) - 127, -119), 127);      // the largest element to 2^7..2^8
                    const float up = __int_as_float((134 - ex) << 23);
                    f *= __int_as_float((120 + ex) << 23);
                    if (amax >= 0x7f80u) f = __int_as_float(0x7fffffff);        // an infinity or NaN: the row is NaN
#pragma unroll
                    for (int k = 0; k < PER / 4; ++k) {
                        const float x[4] = {q[4 * k] * up, q[4 * k + 1] * up, q[4 * k + 2] * up, q[4 * k + 3] * up};
                        const uint32_t lo = q8::to_e4m3x2(x[0], x[1]), hi = q8::to_e4m3x2(x[2], x[3]);
                        const float2 a0 = q8::from_e4m3x2(lo), a1 = q8::from_e4m3x2(hi);
                        *reinterpret_cast<uint32_t*>(line + r * 128 + ((piece ^ (r & 7)) << 4) + in + 4 * k) = lo | hi << 16;
                        *reinterpret_cast<uint32_t*>(line + (NR + r) * 128 + ((piece ^ ((NR + r) & 7)) << 4) + in + 4 * k) =
                            q8::to_e4m3x2((x[0] - a0.x) * 32.f, (x[1] - a0.y) * 32.f) | q8::to_e4m3x2((x[2] - a1.x) * 32.f, (x[3] - a1.y) * 32.f) << 16;
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < PER / 4; ++k) *reinterpret_cast<uint2*>(line + r * 128 + ((piece ^ (r & 7)) << 4) + in + 8 * k) = r < rows ? q_raw[i][k] : make_uint2(0, 0);
                }
                if (lane == 0) {
                    const int pos = s.start + t;
                    row_f[r] = f;
                    row_slope[r] = a.slopes && r < rows ? a.slopes[h] * kLog2e : 0.f;
                    row_pos[r] = pos;
                    row_limit[r] = a.causal ? max(pos, s.prefix - 1) : 0x7fffffff;
                    row_number[r] = h * a.tokens + t;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            barrier();
            if (lane == 0) tc5::mbar_arrive(q_ready);
            if (Q8) {
                // while the scores are made: whether a scale of V in this share is very small or large
                bool odd = odd_scale(scale);
                for (int i = scale0 + BKEY; i < scale_end; i += BKEY) odd |= odd_scale(__ldg(vs + (size_t)i * a.kv_heads));
                if (odd) *odd_scales = 1;
                barrier();
            }
        }

        float m_lane = -INFINITY;                                              // lane r: the maximum that row r's sums stand against
        float l[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) l[r] = 0.f;
        const float cap2 = a.cap * kLog2e;
        // the sums l stand against `in_use`, or, where a scale is very small or large, against (lane r: row r) m_score
        float m_score = -INFINITY;
        float* scores = p.scores + (size_t)e * a.heads * a.tokens * p.pitch;
        // The walk twice, each form in a loop of its own (32 episodes of 16 K rows: 149 us where one loop has a branch, 144 without).
        const bool odd = Q8 && count > 0 && *odd_scales;
#pragma unroll
        for (int form = 0; form < (Q8 ? 2 : 1); ++form)
        for (int n = 0; n < count && (form == 1) == odd; ++n) {
            const int b = n & 1, j = (first + n) * BKEY + key;
            const bool inside = j < s.L;
            const float kf = next_k, lv = Q8 ? q8::log2_of_scale(next_v) : 0.f;      // K's scale; log2 of V's
            const int kp = a.k_pos ? next_pos : j;
            const float iv = Q8 ? (form == 0 ? __frcp_rn(next_v) : 0.f) : 1.f;      // what a probability counts in the row sum
            if (n + 1 < count) fetch(n + 1);
            ok = ok && mbar_wait(s_full(b), (uint32_t)((n >> 1) & 1), abort_flag);
            __syncwarp();
            tc5::tc_fence_after();
            float c[C::NS];
            tmem_ld(tmem + t_lane + C::S_COL + b * C::NS, c);
            tc5::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc5::mbar_arrive(s_empty(b));
            float v[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) v[r] = (Q8 ? fmaf(c[(NR + r) % C::NS], 1.f / 32.f, c[r]) : c[r]) * (row_f[r] * kf);
            if (capped) {
#pragma unroll
                for (int r = 0; r < NR; ++r) v[r] = cap2 * tanh_far(v[r]);
            }
            if (a.slopes) {
#pragma unroll
                for (int r = 0; r < NR; ++r) v[r] = fmaf(-row_slope[r], fabsf((float)(row_pos[r] - kp)), v[r]);
            }
            if (a.causal) {
#pragma unroll
                for (int r = 0; r < NR; ++r) v[r] = inside && kp <= row_limit[r] ? v[r] : -INFINITY;
            } else if (!inside) {
#pragma unroll
                for (int r = 0; r < NR; ++r) v[r] = -INFINITY;
            }
            if (Q8 && p.scores != nullptr) {
#pragma unroll
                for (int r = 0; r < NR; ++r)
                    if (r < rows) scores[(size_t)row_number[r] * p.pitch + j] = v[r];
            }
            float* board = maxima + b * 4 * NR;
            if (form == 1) {
                // the row sums by exponentials of their own, with the arrays that the probabilities take below
                float most = -INFINITY;
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const float x = redux_max(v[r]);
                    if (lane == r) most = x;
                }
                if (lane < NR) board[quad * NR + lane] = most;
                barrier();
                if (lane < NR) {
                    const float was = m_score;
                    m_score = fmaxf(m_score, fmaxf(fmaxf(board[lane], board[NR + lane]), fmaxf(board[2 * NR + lane], board[3 * NR + lane])));
                    rescale[lane] = was == m_score || was == -INFINITY ? 1.f : fast_exp2(was - m_score);
                    in_use[lane] = m_score == -INFINITY ? 0.f : m_score;
                }
                __syncwarp();
#pragma unroll
                for (int r = 0; r < NR; ++r) l[r] = fmaf(l[r], rescale[r], fast_exp2(v[r] - in_use[r]));
                barrier();                                                     // the maxima have been read
            }
            float mine = -INFINITY;
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                v[r] += lv;
                const float x = redux_max(v[r]);
                if (lane == r) mine = x;
            }
            if (lane < NR) board[quad * NR + lane] = mine;
            barrier();
            bool grow = false;
            if (lane < NR) {
                const float mx = fmaxf(fmaxf(board[lane], board[NR + lane]), fmaxf(board[2 * NR + lane], board[3 * NR + lane]));
                grow = m_lane != -INFINITY && mx > m_lane + C::THRESHOLD;
                rescale[lane] = grow ? fast_exp2(m_lane - mx) : 1.f;
                if (grow || m_lane == -INFINITY) m_lane = mx;
                in_use[lane] = (m_lane == -INFINITY ? 0.f : m_lane) - C::SHIFT;      // (nothing but NaN, or nothing at all, so far)
            }
            const bool any = __any_sync(0xffffffffu, grow);
            __syncwarp();
            // P of the block before, and its products, are done with; the same for every warp, since all of them see the same maxima
            ok = ok && (n == 0 || mbar_wait(o_done, (uint32_t)((n - 1) & 1), abort_flag));
            __syncwarp();
            if (any) {
                tc5::tc_fence_after();
#pragma unroll
                for (int h = 0; h < C::HALVES; ++h)
#pragma unroll
                    for (int c0 = 0; c0 < C::NO; c0 += 16) {
                        float o[16];
                        const uint32_t at = tmem + t_lane + C::O_COL + h * C::NO + c0;
                        tc5::tmem_ld16(at, o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] *= c0 + i < NR * C::PT ? rescale[(c0 + i) % NR] : 1.f;
                        st16(at, o);
                    }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc5::tc_fence_before();
                if (form == 0) {
#pragma unroll
                    for (int r = 0; r < NR; ++r) l[r] *= rescale[r];
                }
            }
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                v[r] = fast_exp2(v[r] - in_use[r]);
                l[r] = fmaf(v[r], iv, l[r]);
            }
            // P^T: a row of 128 keys per row and term
            if (Q8) {
                auto at = [&](int row) { return gen + C::OFF_P + row * 128 + (((key >> 4) ^ (row & 7)) << 4) + (key & 15); };
#pragma unroll
                for (int r = 0; r < NR; r += 2) {
                    float x = v[r], y = v[r + 1];
                    float up = 1.f;
#pragma unroll
                    for (int term = 0; term < 3; ++term) {
                        const uint32_t w = q8::to_e4m3x2(x * up, y * up);
                        *at(term * NR + r) = (uint8_t)w;
                        *at(term * NR + r + 1) = (uint8_t)(w >> 8);
                        const float2 back = q8::from_e4m3x2(w);
                        x = fmaf(-back.x, 1.f / up, x);
                        y = fmaf(-back.y, 1.f / up, y);
                        up *= 16.f;
                    }
                }
            } else {
                // (the operand of the second product is bf16, as K and V are: half a step, 2^-8 of a probability; the row sum has all 24 bits)
#pragma unroll
                for (int r = 0; r < NR; ++r)
                    *reinterpret_cast<bf16*>(gen + C::OFF_P + (key >> 6) * (C::NO * 128) + r * 128 + ((((key & 63) >> 3) ^ (r & 7)) << 4) + (key & 7) * 2) = __float2bfloat16_rn(v[r]);
            }
            if ((first + n + 1) * BKEY > s.L) {
                // values behind the last key may be anything, and 0 * NaN would reach every row: zeros in their place
                const int vs_slot = (2 * n + 1) % C::SLOTS;
                ok = ok && mbar_wait(full(vs_slot), (uint32_t)(((2 * n + 1) / C::SLOTS) & 1), abort_flag);
                if (!inside)
                    for (int i = 0; i < C::ATOMS * 8; ++i)
                        *reinterpret_cast<uint4*>(gen + C::OFF_T + vs_slot * C::TILE + (i >> 3) * 16384 + key * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tc5::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc5::mbar_arrive(p_full);
        }
        if (count > 0) ok = ok && mbar_wait(o_done, (uint32_t)((count - 1) & 1), abort_flag);
        __syncwarp();
        tc5::tc_fence_after();

        // the rows' sums over the 128 threads, then O^T: thread = dim, so that a row's dims are stored side by side
        float total = 0.f;
        if (count > 0) {
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const float x = warp_sum(l[r]);
                if (lane == r) total = x;
            }
            barrier();                                                          // the last maxima have been read
            if (lane < NR) maxima[quad * NR + lane] = total;
            barrier();
        }
        const size_t all = (size_t)a.episodes * a.tokens * a.heads;
        auto flat = [&](int r) {
            const int t = r / group;
            return (size_t)split * all + ((size_t)e * a.tokens + t) * a.heads + kv * group + r - t * group;
        };
        if (quad == 0 && lane < NR) {
            const float sum = count > 0 ? maxima[lane] + maxima[NR + lane] + maxima[2 * NR + lane] + maxima[3 * NR + lane] : 0.f;
            float2 ml = make_float2(count > 0 ? in_use[lane] : -INFINITY, sum);
            if (Q8) ml.y = sum == 0.f ? -INFINITY : log2f(sum) + (odd ? (m_score == -INFINITY ? 0.f : m_score) : ml.x);
            if (p.cluster) reinterpret_cast<float2*>(gen + C::OFF_F)[lane] = ml;      // (the rows' factors are no longer needed)
            else if (lane < rows) p.part_ml[flat(lane)] = ml;
        }
        if (count > 0) {
            float* sums = reinterpret_cast<float*>(gen + C::OFF_T);                     // (all tiles have been read)
#pragma unroll
            for (int h = 0; h < C::HALVES; ++h) {
                float o[C::NO];
                tmem_ld(tmem + t_lane + C::O_COL + h * C::NO, o);
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const float x = Q8 ? fmaf(fmaf(o[(2 * NR + r) % C::NO], 1.f / 16.f, o[(NR + r) % C::NO]), 1.f / 16.f, o[r]) : o[r];
                    if (p.cluster) sums[r * HDP + h * 128 + key] = x;
                    else if (r < rows && ok) p.part_o[flat(r) * HDP + h * 128 + key] = x;
                }
            }
        }
    }
    // Tensor memory goes back before the cluster meets: a CTA that held some while it waits for another could wait for ever, where that one waits for tensor memory
    // that a cluster of another kernel (on another stream) holds in the same way.
    __syncwarp();
    tc5::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc5::tc_fence_after();
        tc5::tmem_dealloc(tmem, C::COLS);
    }
    if (p.cluster) {
        auto cluster_barrier = []() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); };
        __syncwarp();
        cluster_barrier();
        if (warp >= 2 && s.n > 0) {
            // row r of this CTA's part: its shares against the largest of their maxima
            const int group = p.group, rows = s.n * group, me = tid - 64;
            for (int i = split * 128 + me; i < rows * HDP; i += p.splits * 128) {
                const int r = i / HDP, d = i % HDP;
                // all that the CTAs have of it at once; what a share that held nothing has left is dropped
                constexpr float NOTHING = Q8 ? -INFINITY : 0.f;
                float2 ml[CLUSTER];
                float y[CLUSTER], top = -INFINITY, top_sum = -INFINITY, sum = 0.f, x = 0.f;
#pragma unroll
                for (int c = 0; c < CLUSTER; ++c) {
                    ml[c] = make_float2(-INFINITY, NOTHING);
                    if (c < p.splits) {
                        uint32_t at;
                        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(base + C::OFF_F + r * 8), "r"(c));
                        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(ml[c].x), "=f"(ml[c].y) : "r"(at) : "memory");
                        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(base + C::OFF_T + i * 4), "r"(c));
                        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(y[c]) : "r"(at) : "memory");
                    }
                }
#pragma unroll
                for (int c = 0; c < CLUSTER; ++c)
                    if (ml[c].y != NOTHING) { top = fmaxf(top, ml[c].x); top_sum = fmaxf(top_sum, ml[c].y); }
                if (!Q8) top_sum = top;
#pragma unroll
                for (int c = 0; c < CLUSTER; ++c) {
                    const float w = ml[c].y == NOTHING ? 0.f : fast_exp2(ml[c].x - top);
                    sum = Q8 ? sum + (ml[c].y == NOTHING ? 0.f : fast_exp2(ml[c].y - top_sum)) : fmaf(ml[c].y, w, sum);
                    x = ml[c].y == NOTHING ? x : fmaf(y[c], w, x);
                }
                const float inv = sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);
                const float half = Q8 && sum > 0.f ? fast_exp2(0.5f * (top - top_sum)) : 1.f;      // the two maxima may lie beyond fp32's range of one another
                const int t = r / group, h = kv * group + r - t * group;
                if (d < a.dim) a.out[e * a.os[0] + t * a.os[1] + h * a.os[2] + d] = __float2bfloat16_rn(x * half * (inv * half));
                if (a.lse && d == 0) a.lse[((size_t)e * a.heads + h) * a.tokens + t] = sum > 0.f ? (top_sum + log2f(sum)) * 0.6931471805599453f : (sum == 0.f ? -INFINITY : sum);
            }
        }
        __syncwarp();
        cluster_barrier();                                                              // nobody leaves while its sums may be read
    }
    if (tid == 0 && *abort_flag && p.status) atomicExch(p.status, 9);
}

// Rows that the kernel is built for.
inline int few_rows(const Args& a) {
    const int rows = a.tokens * (a.heads / a.kv_heads);
    return rows <= 8 ? 8 : (rows <= 16 ? 16 : 32);
}

template <int HDP, bool Q8, int NR>
inline int launch_few(const Tile& p, const CUtensorMap& tmK, const CUtensorMap& tmV, cudaStream_t st) {
    using C = FewCfg<HDP, Q8, NR>;
    auto kern = attention_few_rows_kernel<HDP, Q8, NR>;
    static PerDeviceFlag configured;
    if (!configured.get()) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) { set_error("cudaFuncSetAttribute: %s", cudaGetErrorString(e)); return FVLA_ERR_LAUNCH; }
        configured.set();
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.splits, p.a.kv_heads, p.a.episodes); cfg.blockDim = dim3(FEW_THREADS); cfg.dynamicSmemBytes = C::SMEM; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.cluster ? p.splits : 1; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p, tmK, tmV);
    if (e != cudaSuccess) { set_error("attention_few_rows_kernel: %s", cudaGetErrorString(e)); return FVLA_ERR_LAUNCH; }
    return check_launch("attention_few_rows_kernel");
}
template <int HDP, bool Q8>
inline int launch_few(const Tile& p, const CUtensorMap& tmK, const CUtensorMap& tmV, cudaStream_t st) {
    const int nr = few_rows(p.a);
    return nr == 8 ? launch_few<HDP, Q8, 8>(p, tmK, tmV, st) : (nr == 16 ? launch_few<HDP, Q8, 16>(p, tmK, tmV, st) : launch_few<HDP, Q8, 32>(p, tmK, tmV, st));
}

}  // namespace mattn
}  // namespace fvla

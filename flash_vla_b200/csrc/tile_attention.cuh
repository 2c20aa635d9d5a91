// Attention of many rows. One CTA has 128 rows (tokens x the query heads of one K/V head) of an episode and walks the key blocks that any of them
// sees, or one of `splits` equal shares of them:
//   warps 0, 3  TMA: the Q tile and K, and V, each in granules of 16 KB through a ring (K: 128 bytes of the head dimension of 128 keys; V: some
//               keys, whole): what is in flight is then limited by shared memory alone, not by tile sizes
//   warps 1, 2  one lane of each issues S = Q K^T into one of BUFFERS TMEM score buffers, and O += P V (TMEM). (An issue takes 50 to 100 clocks with
//               its waits; one lane for both was the bottleneck at head dim 128: 301 us against 281.)
//   warps 4-11  softmax: two groups of 128 threads, thread = row, which take the blocks in turn. P goes back to TMEM over the scores, as the A operand
//               of P V; with bf16 keys of head dim 256, whose two score buffers have to be free early, through shared memory (113 us against 127). All
//               that one block needs from the one before is the running maximum: the other group hands it on (per warp, 32 rows) before it begins
//               its exponentials, and those of one block run beside the other's loads and maxima. The accumulator is rescaled only
//               where the maximum has grown by more than a threshold.
// 4 096 keys, 32 query heads of 128, or 8 of 256 over 4 K/V heads, without a mask: 266 us (1 033 TFLOP/s) and 111 us (1 243 TFLOP/s). A block of 128 keys
// takes 2 200 to 2 500 clocks: at head dim 128 the softmax's instructions (128 exponentials of a row at 16 clocks a warp among them), at 256 the arrival of
// 128 KB of keys and values through 128 KB of rings. A CTA's two ends, 7 000 and 5 000 clocks, are the rest of short walks.
// The 8-bit cache runs in 8 bits (kind::f8f6f4; 256 tokens of eight episodes over 4 096 rows of 256: 137 us, 375 TFLOP/s), its values straight from TMA. A
// bf16 row of Q, brought to 2^7..2^8 by its own power of two, is the sum of an e4m3 term and an e5m2 term: what rounding to 4 bits leaves of 8 has at most 3.
// (Elements below e4m3's smallest normal number, 2^-13 of the largest, are off by 2^-3 of half its smallest step, 2^-20 of the largest.) A probability is the
// sum of two e4m3 terms and an e5m2 term. Probabilities stand against the running maximum at 2^6 and are rescaled when it has grown by 2^2: the first two
// terms leave 2^-8 of a value, or half of e4m3's smallest step, 2^-10, and the third 2^-3 of that. So a probability is off by at most 2^-11 of itself or 2^-19
// of the row's largest. The scale of K multiplies the scores in fp32; the scale of V moves into the exponent of P (w = log2 p + log2 V_scale, P =
// 2^(w - max w)), and the row sum takes it back, or, where a share has very small or large scales (a block of zeros has 2^-120, and its inverse would end
// fp32's range), is taken from the scores themselves against a maximum of their own.
#pragma once

namespace fvla {
namespace mattn {

__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]
template <bool F8>
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    if (F8)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t}"
            ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
            ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void st32_nowait(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
          "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
          "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
// Two fp32 operations at a time: (a0, a1) * b + c;  (a0, a1) + (x0, x1) * b;  (a0, a1) + (b0, b1);  (a0, a1) * b
__device__ __forceinline__ unsigned long long pair(float x, float y) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpair(unsigned long long v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ void fma2(float& a0, float& a1, float b, float c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pair(a0, a1)), "l"(pair(b, b)), "l"(pair(c, c)));
    unpair(r, a0, a1);
}
__device__ __forceinline__ void axpy2(float& a0, float& a1, float x0, float x1, float b) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pair(x0, x1)), "l"(pair(b, b)), "l"(pair(a0, a1)));
    unpair(r, a0, a1);
}
__device__ __forceinline__ void add2(float& a0, float& a1, float b0, float b1) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair(a0, a1)), "l"(pair(b0, b1)));
    unpair(r, a0, a1);
}
__device__ __forceinline__ void mul2(float& a0, float& a1, float b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair(a0, a1)), "l"(pair(b, b)));
    unpair(r, a0, a1);
}
// scale tanh of two values of at most 1/2, by the series
__device__ __forceinline__ void tanh2(float& a0, float& a1, float scale) {
    unsigned long long y = pair(a0, a1), q, t;
    asm("mul.rn.f32x2 %0, %1, %1;" : "=l"(q) : "l"(y));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(t) : "l"(q), "l"(pair(kTanh13, kTanh13)), "l"(pair(kTanh11, kTanh11)));
    asm("fma.rn.f32x2 %0, %1, %0, %2;" : "+l"(t) : "l"(q), "l"(pair(kTanh9, kTanh9)));
    asm("fma.rn.f32x2 %0, %1, %0, %2;" : "+l"(t) : "l"(q), "l"(pair(kTanh7, kTanh7)));
    asm("fma.rn.f32x2 %0, %1, %0, %2;" : "+l"(t) : "l"(q), "l"(pair(kTanh5, kTanh5)));
    asm("fma.rn.f32x2 %0, %1, %0, %2;" : "+l"(t) : "l"(q), "l"(pair(kTanh3, kTanh3)));
    asm("fma.rn.f32x2 %0, %1, %0, %2;" : "+l"(t) : "l"(q), "l"(pair(1.f, 1.f)));
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(y) : "l"(pair(scale, scale)));
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(y) : "l"(t));
    unpair(y, a0, a1);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

template <int HDP, bool Q8>
struct TileCfg {
    static constexpr int ELEM = Q8 ? 1 : 2, QT = Q8 ? 2 : 1, PT = Q8 ? 3 : 1;      // bytes of a cached value; terms of Q and of P
    static constexpr int GRANULE = 16384, GRANULES = HDP * ELEM / 128;             // of a K or V block
    static constexpr int V_KEYS = BKEY / GRANULES;                                 // keys of a V granule
    static constexpr int Q_ATOMS = HDP / 64, Q_BYTES = Q_ATOMS * 16384;            // as bf16, and as two terms of e4m3
    static constexpr int BUFFERS = HDP == 256 ? 2 : 3;                             // 128 columns each, beside HDP columns of the accumulator
    // P as an operand in shared memory: where tensor memory has only two score buffers, these are then free again as soon as the scores have been read
    static constexpr bool P_SHARED = HDP == 256 && !Q8;
    static constexpr int SLOTS = P_SHARED ? 4 : (HDP == 256 ? 5 : 6);              // of each ring
    static constexpr int OFF_Q = 0, OFF_P = OFF_Q + Q_BYTES, OFF_R = OFF_P + (P_SHARED ? BQ * BKEY * 2 : 0), OFF_X = OFF_R + 2 * SLOTS * GRANULE;      // rings; a maximum per row, a float per row and group
    static constexpr int OFF_BAR = OFF_X + 3 * BQ * 4;
    static constexpr int SMEM = 1024 + OFF_BAR + 344;
    static constexpr int THREADS = 32 * (SOFTMAX0 + SOFTMAX_WARPS);
    static constexpr uint32_t O_COL = BUFFERS * BKEY;
    static constexpr float SHIFT = Q8 ? 6.f : 0.f, THRESHOLD = Q8 ? 2.f : RESCALE_THRESHOLD;
};

template <int HDP, bool Q8>
__global__ void __launch_bounds__(TileCfg<HDP, Q8>::THREADS, 1)
attention_tile_kernel(const __grid_constant__ Tile p, const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO) {
    using C = TileCfg<HDP, Q8>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t sQ = base + C::OFF_Q, ring = base + C::OFF_R, bars = base + C::OFF_BAR;
    const uint32_t q_full = bars, q_ready = bars + 8;
    auto s_full = [&](int b) { return bars + 16 + b * 8; };
    auto p_full = [&](int b) { return bars + 40 + b * 8; };
    auto o_done = [&](int b) { return bars + 64 + b * 8; };                // of even and odd blocks
    const uint32_t finished = bars + 80;                                   // all products (a wait for a block's own phase could come too late for its parity)
    auto p_read = [&](int b) { return bars + 96 + b * 8; };                // the buffer may take scores: the product has read P, or (P_SHARED) the softmax its scores
    // rings: K slots, then V slots
    auto full = [&](int s) { return bars + 120 + s * 8; };
    auto empty = [&](int s) { return bars + 120 + C::SLOTS * 16 + s * 8; };
    const uint32_t tmem_slot = bars + 120 + C::SLOTS * 32;
    uint8_t* after = gen + C::OFF_BAR + 120 + C::SLOTS * 32;
    volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(after);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(after + 4);
    volatile int* odd_scales = reinterpret_cast<volatile int*>(after + 24);
    int* shared_int = reinterpret_cast<int*>(after + 8);      // smallest and largest document of the queries, first and last block seen

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Args& a = p.a;
    // the tiles of all heads and episodes from the last (under a causal mask the longest) to the first, the shares of a tile side by side
    const int per_tile = p.splits * a.kv_heads * a.episodes, in_tile = blockIdx.x % per_tile;
    const int tile = p.tiles - 1 - (int)(blockIdx.x / per_tile), split = in_tile % p.splits, kv = in_tile / p.splits % a.kv_heads, e = in_tile / p.splits / a.kv_heads;
    const int t0 = tile * p.tile_tokens;

    if (tid == 0) {
        mbar_init(q_full, 1); mbar_init(q_ready, SOFTMAX_WARPS);
        for (int b = 0; b < C::BUFFERS; ++b) { mbar_init(s_full(b), 1); mbar_init(p_full(b), SOFTMAX_WARPS / 2); mbar_init(p_read(b), C::P_SHARED ? 4 : 1); }
        for (int b = 0; b < 2; ++b) mbar_init(o_done(b), 1);
        mbar_init(finished, 1);
        for (int s = 0; s < 2 * C::SLOTS; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        *abort_flag = 0;
        *odd_scales = 0;
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

    // Q is asked for before the lengths are known
    if (tid == 0) {
        tc5::prefetch_tensormap(&tmQ);
        mbar_expect_tx(q_full, C::Q_ATOMS * 128 * p.group * p.tile_tokens);
#pragma unroll
        for (int c = 0; c < C::Q_ATOMS; ++c) tma_load_5d(sQ + c * 16384, &tmQ, q_full, c * 64, 0, t0, kv * p.q_mul[0], e * p.q_mul[1]);
    }
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
            walk.count = last;
            for (int j = tid; j < last; j += C::THREADS)
                if (walk.sees(j)) { atomicMin(shared_int + 2, walk.block(j)); atomicMax(shared_int + 3, walk.block(j)); }
            __syncthreads();
            first = min(shared_int[2], last);
            last = max(first, min(last, shared_int[3] + 1));
        }
    }
    walk.first = first + (int)((long long)(last - first) * split / p.splits);
    walk.count = first + (int)((long long)(last - first) * (split + 1) / p.splits) - walk.first;
    const bool any = walk.next(0) < walk.count;
    if (!any) mbar_wait(q_full, 0, abort_flag);           // nobody else waits for it: neither Q's buffer nor this CTA may go before it has come

    // 384 threads start with 168 registers each: 56 + 2 x 224 = 504 = 3 x 168
    if (warp < SOFTMAX0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        constexpr uint32_t type = Q8 ? 0u : 1u, E5M2 = 1u << 7;      // e4m3 or bf16 operands; A in e5m2
        int at = 0;                                                  // slot of this warp's ring, and the parity of its round
        uint32_t phase = 0;
        auto advance = [&]() { if (++at == C::SLOTS) { at = 0; phase ^= 1u; } };
        if (warp == 0) {
            if (lane == 0 && any) {
                tc5::prefetch_tensormap(&tmK);
                bool ok = true;
                for (int i = walk.next(0); i < walk.count && ok; i = walk.next(i + 1)) {
#pragma unroll 1
                    for (int c = 0; c < C::GRANULES; ++c) {
                        ok = mbar_wait(empty(at), phase ^ 1u, abort_flag);
                        if (!ok) break;
                        mbar_expect_tx(full(at), C::GRANULE);
                        tma_load_4d(ring + at * C::GRANULE, &tmK, full(at), c * (128 / C::ELEM), walk.block(i) * BKEY, kv * p.k_mul[0], e * p.k_mul[1]);
                        advance();
                    }
                }
            }
        } else if (warp == 3) {
            if (lane == 0 && any) {
                tc5::prefetch_tensormap(&tmV);
                bool ok = true;
                for (int i = walk.next(0); i < walk.count && ok; i = walk.next(i + 1)) {
#pragma unroll 1
                    for (int c = 0; c < C::GRANULES; ++c) {
                        const int slot = C::SLOTS + at;
                        ok = mbar_wait(empty(slot), phase ^ 1u, abort_flag);
                        if (!ok) break;
                        mbar_expect_tx(full(slot), C::GRANULE);
#pragma unroll
                        for (int d = 0; d < C::GRANULES; ++d)
                            tma_load_4d(ring + slot * C::GRANULE + d * C::V_KEYS * 128, &tmV, full(slot), d * (128 / C::ELEM), walk.block(i) * BKEY + c * C::V_KEYS,
                                        kv * p.v_mul[0], e * p.v_mul[1]);
                        advance();
                    }
                }
            }
        } else if (warp == 1) {
            if (any && tc5::elect_one()) {
                constexpr uint32_t id_qk = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)(BKEY >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
                bool ok = mbar_wait(Q8 ? q_ready : q_full, 0, abort_flag);
                int buffer = 0, round = 0;
                for (int i = walk.next(0); i < walk.count && ok; i = walk.next(i + 1)) {
                    if (round > 0) { ok = mbar_wait(p_read(buffer), (uint32_t)(round - 1) & 1u, abort_flag); if (!ok) break; }
#pragma unroll 1
                    for (int c = 0; c < C::GRANULES; ++c) {
                        ok = mbar_wait(full(at), phase, abort_flag);
                        if (!ok) break;
                        tc5::tc_fence_after();
                        const uint64_t ad = smem_desc(sQ + c * 16384, 16, 1024), bd = smem_desc(ring + at * C::GRANULE, 16, 1024);
#pragma unroll
                        for (int term = 0; term < C::QT; ++term)
#pragma unroll
                            for (int k = 0; k < 4; ++k) {             // 32 bytes further on: 2 in a descriptor
                                if (Q8) umma_f8(tmem + buffer * BKEY, ad + term * C::GRANULES * 1024 + 2 * k, bd + 2 * k, id_qk | (term == 1 ? E5M2 : 0u), c > 0 || term > 0 || k > 0);
                                else tc5::umma_bf16(tmem + buffer * BKEY, ad + 2 * k, bd + 2 * k, id_qk, c > 0 || k > 0);
                            }
                        tc5::umma_commit(empty(at));
                        advance();
                    }
                    if (!ok) break;
                    tc5::umma_commit(s_full(buffer));
                    if (++buffer == C::BUFFERS) { buffer = 0; ++round; }
                }
            }
        } else if (warp == 2) {
            if (any && tc5::elect_one()) {
                constexpr uint32_t id_pv = (1u << 4) | (type << 7) | (type << 10) | (1u << 16) | ((uint32_t)(HDP >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
                constexpr int KEYS = 32 / C::ELEM;                     // keys per MMA, 8 columns of P
                bool ok = true;
                int buffer = 0, n = 0;
                uint32_t round = 0;
                for (int i = walk.next(0); i < walk.count && ok; i = walk.next(i + 1), ++n) {
                    ok = mbar_wait(p_full(buffer), round, abort_flag);
                    if (!ok) break;
#pragma unroll 1
                    for (int c = 0; c < C::GRANULES; ++c) {
                        const int slot = C::SLOTS + at;
                        ok = mbar_wait(full(slot), phase, abort_flag);
                        if (!ok) break;
                        tc5::tc_fence_after();
                        const uint64_t bd = smem_desc(ring + slot * C::GRANULE, C::V_KEYS * 128, 1024);
                        const uint32_t pa = tmem + buffer * BKEY + c * (C::V_KEYS / KEYS) * 8;
#pragma unroll
                        for (int k = 0; k < C::V_KEYS / KEYS; ++k)
#pragma unroll
                            for (int term = 0; term < C::PT; ++term)
                                if (C::P_SHARED) tc5::umma_bf16(tmem + C::O_COL, smem_desc(base + C::OFF_P + (c >> 1) * 16384 + ((c & 1) * 2 + k) * 32, 16, 1024), bd + k * KEYS * 8, id_pv, n > 0 || c > 0 || k > 0);
                                else umma_ts<Q8>(tmem + C::O_COL, pa + term * 32 + k * 8, bd + k * KEYS * 8, id_pv | (term == 2 ? E5M2 : 0u), n > 0 || c > 0 || k > 0 || term > 0);
                        tc5::umma_commit(empty(slot));
                        advance();
                    }
                    if (!ok) break;
                    if (!C::P_SHARED) tc5::umma_commit(p_read(buffer));
                    tc5::umma_commit(o_done(n & 1));
                    if (++buffer == C::BUFFERS) { buffer = 0; round ^= 1u; }
                }
                if (ok) tc5::umma_commit(finished);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // Every thread runs every iteration and every named barrier even after a wait has given up (`ok` false), so nobody is left behind.
        const int quad = warp & 3, g = (warp - SOFTMAX0) >> 2;         // TMEM lanes that this warp may access; which blocks it takes
        const int row = quad * 32 + lane;
        const uint32_t t_lane = (uint32_t)(quad * 32) << 16;
        float* m_shared = reinterpret_cast<float*>(gen + C::OFF_X);    // the maximum that each row's accumulator stands against
        float* xch = m_shared + BQ;                                    // [group][row]
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

        if (Q8 && any) {
            // Q from bf16 to its two terms, in place: a thread has half of a row, and a row stays on its own lines
            ok = mbar_wait(q_full, 0, abort_flag);
            __syncwarp();
            constexpr int PIECES = HDP / 16;                           // of 16 bytes, 8 values, of half a row
            uint4 u[PIECES];
            uint32_t amax = 0;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int at = g * PIECES + i;
                u[i] = *reinterpret_cast<const uint4*>(gen + C::OFF_Q + (at >> 3) * 16384 + row * 128 + (((at & 7) ^ (row & 7)) << 4));
                const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) amax = max(amax, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
            }
            xch[g * BQ + row] = __uint_as_float(amax);
            asm volatile("bar.sync 9, 256;" ::: "memory");
            amax = max(amax, __float_as_uint(xch[(g ^ 1) * BQ + row]));
            const int ex = min(max((int)(amax >> 7) - 127, -119), 127);      // the largest element to 2^7..2^8
            const float up = __int_as_float((134 - ex) << 23);
            factor *= __int_as_float((120 + ex) << 23);
            if (amax >= 0x7f80u) factor = __int_as_float(0x7fffffff);        // an infinity or NaN: the row is NaN
#pragma unroll
            for (int i = 0; i < PIECES; i += 2) {
                uint32_t one[4], two[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint4& v = u[i + (k >> 1)];
                    const float2 x = unpack_bf16x2(k & 1 ? v.z : v.x), y = unpack_bf16x2(k & 1 ? v.w : v.y);
                    const float f[4] = {x.x * up, x.y * up, y.x * up, y.y * up};
                    const uint32_t lo = q8::to_e4m3x2(f[0], f[1]), hi = q8::to_e4m3x2(f[2], f[3]);
                    const float2 a0 = q8::from_e4m3x2(lo), a1 = q8::from_e4m3x2(hi);
                    one[k] = lo | hi << 16;
                    two[k] = q8::to_e5m2x2(f[0] - a0.x, f[1] - a0.y) | q8::to_e5m2x2(f[2] - a1.x, f[3] - a1.y) << 16;
                }
                const int at = (g * PIECES + i) / 2;                             // piece of 16 values in the row
                uint8_t* line = gen + C::OFF_Q + (at >> 3) * 16384 + row * 128 + (((at & 7) ^ (row & 7)) << 4);
                *reinterpret_cast<uint4*>(line) = make_uint4(one[0], one[1], one[2], one[3]);
                *reinterpret_cast<uint4*>(line + C::GRANULES * 16384) = make_uint4(two[0], two[1], two[2], two[3]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            asm volatile("bar.sync 9, 256;" ::: "memory");                       // xch is free again
            if (lane == 0) tc5::mbar_arrive(q_ready);
            // while the scores are made: whether a scale of V in this share is very small or large
            const int shift = 31 - __clz(a.block), end = (min((walk.first + walk.count) * BKEY, s.L) + a.block - 1) >> shift;
            bool odd = false;
            for (int i = (walk.first * BKEY >> shift) + tid - 32 * SOFTMAX0; i < end; i += 32 * SOFTMAX_WARPS)
                odd |= odd_scale(__ldg(a.v_scale + ((size_t)e * (a.keys >> shift) + i) * a.kv_heads + kv));
            if (odd) *odd_scales = 1;
            asm volatile("bar.sync 9, 256;" ::: "memory");
        }

        float m_used = -INFINITY, l = 0.f;                             // what this group's sum stands against
        const int shift = Q8 ? 31 - __clz(a.block) : 0;                // blocks are powers of two
        const bool plain = !capped && a.slopes == nullptr && (factor > 1e-30f || !mine);
        const bool fast = !Q8 && __all_sync(0xffffffffu, plain);       // the factor goes into the exponential's argument
        const bool tagged = walk.range != nullptr || (a.k_pos != nullptr && a.causal);
        const int clear = tagged ? 0 : __reduce_min_sync(0xffffffffu, mine ? key_limit : s.L);      // below, every row of the warp sees every key
        const int nearest = __reduce_min_sync(0xffffffffu, mine ? pos : 0x7fffffff);                // and no row's position lies before a key
        int n = 0, buffer = g, parity = 0, i = walk.next(0);
        if (g == 1 && i < walk.count) { i = walk.next(i + 1); n = 1; }
        // each form of the row sum has a loop of its own, and which it is is read again where it matters: a register for it costs the loop 120 bytes of spills
#pragma unroll
        for (int form = 0; form < (Q8 ? 2 : 1); ++form)
        if (!Q8 || (*odd_scales != 0) == (form == 1)) while (i < walk.count) {
            const int after_i = walk.next(i + 1), key0 = walk.block(i) * BKEY;
            float kf[8], lv[8];                                        // (8-bit cache) per 16 keys: factor of the scores; log2 of V's scale
            if (Q8 && busy) {
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const size_t at = ((size_t)e * (a.keys >> shift) + (min(key0 + c * 16, s.L - 1) >> shift)) * a.kv_heads + kv;
                    kf[c] = factor * __ldg(a.k_scale + at);
                    lv[c] = q8::log2_of_scale(__ldg(a.v_scale + at));
                }
            }
            const uint32_t t_s = tmem + t_lane + buffer * BKEY;
            ok = ok && mbar_wait(s_full(buffer), (uint32_t)parity, abort_flag);
            __syncwarp();                                              // the TMEM accesses below are warp-collective
            tc5::tc_fence_after();
            if (busy) {
                uint32_t r[BKEY];
#pragma unroll
                for (int c = 0; c < 4; ++c) ld32_nowait(t_s + 32 * c, r + 32 * c);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (C::P_SHARED) {
                    tc5::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) tc5::mbar_arrive(p_read(buffer));
                }
                float (&v)[BKEY] = reinterpret_cast<float (&)[BKEY]>(r);
                if (!fast) {
                    if (Q8 || capped || a.k_pos) {
#pragma unroll
                        for (int c = 0; c < BKEY; c += 2) mul2(v[c], v[c + 1], Q8 ? kf[c >> 4] : factor);
                        if (capped) {
                            float size = 0.f;
#pragma unroll
                            for (int c = 0; c < BKEY; c += 2) size = max3(size, fabsf(v[c]), fabsf(v[c + 1]));
                            if (__all_sync(0xffffffffu, size <= 0.5f || !mine)) {
#pragma unroll
                                for (int c = 0; c < BKEY; c += 2) tanh2(v[c], v[c + 1], cap2);
                            } else {
#pragma unroll
                                for (int c = 0; c < BKEY; ++c) v[c] = cap2 * tanh_far(v[c]);
                            }
                        }
                        if (a.slopes) {
                            if (a.k_pos) {
                                const int* at = a.k_pos + (size_t)e * a.keys;
#pragma unroll
                                for (int c = 0; c < BKEY; ++c) v[c] = fmaf(-slope, fabsf((float)(pos - __ldg(at + min(key0 + c, a.keys - 1)))), v[c]);
                            } else {
                                const float d0 = (float)(pos - key0);
#pragma unroll
                                for (int c = 0; c < BKEY; ++c) v[c] = fmaf(-slope, fabsf(d0 - (float)c), v[c]);
                            }
                        }
                    } else {
                        const float d0 = (float)(pos - key0);
                        if (key0 + BKEY - 1 <= nearest) {
                            // keys before every row of the warp: score + slope c - slope d0
                            const float off = -slope * d0;
                            float c0 = 0.f, c1 = 1.f;
#pragma unroll
                            for (int c = 0; c < BKEY; c += 2) {
                                fma2(v[c], v[c + 1], factor, off);
                                axpy2(v[c], v[c + 1], c0, c1, slope);
                                add2(c0, c1, 2.f, 2.f);
                            }
                        } else {
#pragma unroll
                            for (int c = 0; c < BKEY; ++c) v[c] = fmaf(-slope, fabsf(d0 - (float)c), v[c] * factor);
                        }
                    }
                }
                if (key0 + BKEY > clear) {
                    // visible keys, as bits; what is hidden becomes -infinity, and 2^-infinity is 0
                    uint32_t see[4];
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int have = key_limit - key0 - 32 * w;
                        see[w] = have >= 32 ? 0xffffffffu : (have > 0 ? (1u << have) - 1u : 0u);
                    }
                    if (walk.range != nullptr) {
                        // a lane looks at four keys; one vote for each document among the warp's rows (one or two, as a rule)
                        const int* tag = a.k_docs + (size_t)e * a.keys;
                        int ids[4];
#pragma unroll
                        for (int w = 0; w < 4; ++w) ids[w] = __ldg(tag + min(key0 + 32 * w + lane, a.keys - 1));
                        uint32_t left = __ballot_sync(0xffffffffu, doc >= 0);
                        if (doc < 0) see[0] = see[1] = see[2] = see[3] = 0u;
                        while (left) {
                            const int d = __shfl_sync(0xffffffffu, doc, __ffs(left) - 1);
#pragma unroll
                            for (int w = 0; w < 4; ++w) {
                                const uint32_t votes = __ballot_sync(0xffffffffu, ids[w] == d);
                                if (doc == d) see[w] &= votes;
                            }
                            left &= ~__ballot_sync(0xffffffffu, doc == d);
                        }
                    }
                    if (a.k_pos && a.causal) {
                        const int* at = a.k_pos + (size_t)e * a.keys;
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            uint32_t seen = 0u;
#pragma unroll
                            for (int c = 0; c < 32; ++c)
                                if (__ldg(at + min(key0 + 32 * w + c, a.keys - 1)) <= limit) seen |= 1u << c;
                            see[w] &= seen;
                        }
                    }
                    if (!__all_sync(0xffffffffu, (see[0] & see[1] & see[2] & see[3]) == 0xffffffffu)) {
#pragma unroll
                        for (int c = 0; c < BKEY; ++c) v[c] = see[c >> 5] & (1u << (c & 31)) ? v[c] : -INFINITY;
                    }
                }
                if (Q8 && p.scores != nullptr) {
                    // [episode, K/V head, tile][key block][4 keys][row]: the rows of a warp side by side
                    float4* dst = reinterpret_cast<float4*>(p.scores) + ((((size_t)e * a.kv_heads + kv) * p.tiles + tile) * p.key_blocks + key0 / BKEY) * (BQ * BKEY / 4) + row;
#pragma unroll
                    for (int c = 0; c < BKEY; c += 4) dst[c / 4 * BQ] = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
                }
                float top[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    float x = fmaxf(v[16 * q], v[16 * q + 1]);
#pragma unroll
                    for (int c = 2; c < 16; c += 2) x = max3(x, v[16 * q + c], v[16 * q + c + 1]);
                    top[q] = Q8 ? x + lv[q] : x;
                }
                float mx = max3(max3(top[0], top[1], top[2]), max3(top[3], top[4], top[5]), fmaxf(top[6], top[7]));
                if (fast) mx *= factor;
                // the maximum that the blocks before have left, and what becomes of it
                if (n > 0) asm volatile("bar.sync %0, 64;" ::"r"(1 + g * 4 + quad) : "memory");
                const float m_old = n > 0 ? m_shared[row] : -INFINITY;
                const bool grow = m_old != -INFINITY && mx > m_old + C::THRESHOLD;
                const float m_new = grow || m_old == -INFINITY ? mx : m_old;
                if (__any_sync(0xffffffffu, grow)) {
                    // the accumulator must be quiet while it is rescaled: the products of the block before have to be complete
                    ok = ok && mbar_wait(o_done(g ^ 1), (uint32_t)(((n - 1) >> 1) & 1), abort_flag);
                    __syncwarp();
                    tc5::tc_fence_after();
                    const float alpha = grow ? fast_exp2(m_old - m_new) : 1.0f;
#pragma unroll 1
                    for (int c = 0; c < HDP / 32; ++c) {
                        uint32_t o[32];
                        ld32_nowait(tmem + t_lane + C::O_COL + c * 32, o);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                        st32_nowait(tmem + t_lane + C::O_COL + c * 32, o);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc5::tc_fence_before();
                }
                m_shared[row] = m_new;
                if (after_i < walk.count) asm volatile("bar.arrive %0, 64;" ::"r"(1 + (g ^ 1) * 4 + quad) : "memory");
                if (form == 0 && m_new != m_used) {
                    l *= m_used == -INFINITY ? 1.f : fast_exp2(m_used - m_new);
                    m_used = m_new;
                }
                const float m = (m_new == -INFINITY ? 0.f : m_new) - C::SHIFT;      // (nothing but NaN, or nothing at all, so far)
                if (!Q8) {
                    // the operand of the second product is bf16, as K and V are: half a step, 2^-8 of a probability; the row sum takes all 24 bits
                    const float f = fast ? factor : 1.f;
                    float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
                    for (int c = 0; c < BKEY; c += 4) {
                        fma2(v[c], v[c + 1], f, -m);
                        fma2(v[c + 2], v[c + 3], f, -m);
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[c + k] = fast_exp2(v[c + k]);
                        add2(s0, s1, v[c], v[c + 1]);
                        add2(s2, s3, v[c + 2], v[c + 3]);
                        r[c / 2] = pack_bf16x2(v[c], v[c + 1]);
                        r[c / 2 + 1] = pack_bf16x2(v[c + 2], v[c + 3]);
                        if (!C::P_SHARED && c == 60) st32_nowait(t_s, r);
                    }
                    l += (s0 + s1) + (s2 + s3);
                    if (C::P_SHARED) {
                        // the products of the block before have read P (128-byte swizzle: 8 keys are a piece of a row's 128 bytes in an atom of 64)
                        ok = ok && (n == 0 || mbar_wait(o_done(g ^ 1), (uint32_t)(((n - 1) >> 1) & 1), abort_flag));
                        __syncwarp();
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            *reinterpret_cast<uint4*>(gen + C::OFF_P + (k >> 3) * 16384 + row * 128 + (((k & 7) ^ (row & 7)) << 4)) =
                                make_uint4(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]);
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    } else {
                        st32_nowait(t_s + 32, r + 32);
                    }
                } else {
                    // Three terms of four values to a word, 32 columns each. What a term leaves is found by converting it back (4 300 clocks a block; 7 300 with splitting by
                    // additions instead).
                    uint32_t w[3][32];
                    if (form == 1) {
                        // the row sum from the scores, against a maximum of theirs
                        float most = m_used;
#pragma unroll
                        for (int c = 0; c < BKEY; c += 2) most = max3(most, v[c], v[c + 1]);
                        const float m_sum = most == -INFINITY ? 0.f : most;
                        l *= m_used == -INFINITY ? 1.f : fast_exp2(m_used - m_sum);
                        m_used = most;
#pragma unroll
                        for (int c = 0; c < BKEY; ++c) l += fast_exp2(v[c] - m_sum);
                    }
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        float sum = 0.f;
                        const float off = lv[q] - m;
#pragma unroll
                        for (int c = q * 16; c < q * 16 + 16; c += 4) {
                            float x[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) { x[k] = fast_exp2(v[c + k] + off); sum += x[k]; }
#pragma unroll
                            for (int term = 0; term < 3; ++term) {
                                const uint32_t lo = term < 2 ? q8::to_e4m3x2(x[0], x[1]) : q8::to_e5m2x2(x[0], x[1]);
                                const uint32_t hi = term < 2 ? q8::to_e4m3x2(x[2], x[3]) : q8::to_e5m2x2(x[2], x[3]);
                                w[term][c / 4] = lo | hi << 16;
                                if (term < 2) {
                                    const float2 b0 = q8::from_e4m3x2(lo), b1 = q8::from_e4m3x2(hi);
                                    x[0] -= b0.x; x[1] -= b0.y; x[2] -= b1.x; x[3] -= b1.y;
                                }
                            }
                        }
                        if (form == 0) l = fmaf(sum, fast_exp2(-lv[q]), l);
                    }
#pragma unroll
                    for (int term = 0; term < 3; ++term) st32_nowait(t_s + 32 * term, w[term]);
                }
                if (!C::P_SHARED) asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            } else if (C::P_SHARED) {
                // (waits like the others: two blocks on, it would otherwise signal the same barrier before they have signalled it for this one)
                if (lane == 0) tc5::mbar_arrive(p_read(buffer));
                ok = ok && (n == 0 || mbar_wait(o_done(g ^ 1), (uint32_t)(((n - 1) >> 1) & 1), abort_flag));
                __syncwarp();
            }
            // keys whose values may be anything, behind the last one or under a negative document: zeros, for 0 * NaN would reach every row
            bool tail = key0 + BKEY > s.L;
            if (walk.range != nullptr) tail = tail || __ldg(walk.range + walk.block(i)).x < 0;
            if (tail) {
                const int key = row, at = key0 + key;
                const bool bad = at >= s.L || (walk.range != nullptr && __ldg(a.k_docs + (size_t)e * a.keys + at) < 0);
#pragma unroll 1
                for (int c = 0; c < C::GRANULES; ++c) {
                    const int granule = n * C::GRANULES + c, slot = C::SLOTS + granule % C::SLOTS;
                    ok = ok && mbar_wait(full(slot), (uint32_t)(granule / C::SLOTS & 1), abort_flag);
                    if (bad && key / C::V_KEYS == c)
                        for (int k = 0; k < C::GRANULES * 8; ++k)
                            *reinterpret_cast<uint4*>(gen + C::OFF_R + slot * C::GRANULE + (k >> 3) * (C::V_KEYS * 128) + key % C::V_KEYS * 128 + (k & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            tc5::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc5::mbar_arrive(p_full(buffer));
            // this group's next block is the one after the other group's
            buffer += 2;
            if (buffer >= C::BUFFERS) { buffer -= C::BUFFERS; parity ^= 1; }
            n += 2;
            i = after_i < walk.count ? walk.next(after_i + 1) : walk.count;
        }
        if (any) ok = ok && mbar_wait(finished, 0, abort_flag);
        __syncwarp();
        asm volatile("bar.sync 9, 256;" ::: "memory");                               // and every row's last maximum is there
        tc5::tc_fence_after();
        // the row's sum from its two threads, then half of the columns each
        const float m_all = any && busy ? m_shared[row] : -INFINITY;
        const float m_end = (m_all == -INFINITY ? 0.f : m_all) - C::SHIFT;
        float m_sum = m_end, half = 1.f;                               // what l stands against; root of what lies between the accumulator's maximum and that
        if (!Q8) {
            if (m_used != -INFINITY) l *= fast_exp2(m_used - m_all);
            xch[g * BQ + row] = l;
            asm volatile("bar.sync 9, 256;" ::: "memory");
            l = xch[row] + xch[BQ + row];
        } else {
            float* maxima = reinterpret_cast<float*>(gen + C::OFF_R + (2 * C::SLOTS - 1) * C::GRANULE);      // (the rings are idle; results take their first slots at most)
            xch[g * BQ + row] = l;
            maxima[g * BQ + row] = *odd_scales ? m_used : m_used - C::SHIFT;
            asm volatile("bar.sync 9, 256;" ::: "memory");
            const float m0 = maxima[row], m1 = maxima[BQ + row], m_both = fmaxf(m0, m1);
            m_sum = m_both == -INFINITY ? 0.f : m_both;
            l = xch[row] * fast_exp2(m0 - m_sum) + xch[BQ + row] * fast_exp2(m1 - m_sum);
            half = fast_exp2(0.5f * (m_end - m_sum));
        }
        const bool store = ok && mine;
        constexpr int SPAN = HDP / 2;                                  // columns of a thread
        if (p.splits == 1) {
            const float inv = (l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l)) * half;    // NaN stays
            if (store && g == 0 && a.lse)
                a.lse[((size_t)e * a.heads + h) * a.tokens + t0 + t] = l > 0.f ? (m_sum + log2f(l)) * 0.6931471805599453f : (l == 0.f ? -INFINITY : l);
            // Q's buffer takes the results in Q's layout, and the TMA stores them: all rows of the box, or all that the tensor has. A tile that ends at its
            // episode's last query is stored by its threads (for four prefixes of 8 x 256, 37.1 us if all are).
            const bool whole = tokens == p.tile_tokens || t0 + tokens == a.tokens;
            bf16* dst = a.out + e * a.os[0] + (t0 + (mine ? t : 0)) * a.os[1] + h * a.os[2];
#pragma unroll 1
            for (int c = 0; c < (busy ? SPAN : 0); c += 32) {
                float o[32];
                const int col = g * SPAN + c;
                if (any) tc5::tmem_ld32(tmem + t_lane + C::O_COL + col, o);
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = any ? (Q8 ? o[k] * half : o[k]) * inv : 0.f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint4 u = make_uint4(pack_bf16x2(o[8 * k], o[8 * k + 1]), pack_bf16x2(o[8 * k + 2], o[8 * k + 3]), pack_bf16x2(o[8 * k + 4], o[8 * k + 5]),
                                               pack_bf16x2(o[8 * k + 6], o[8 * k + 7]));
                    const int piece = (col >> 3) + k;
                    if (whole) *reinterpret_cast<uint4*>(gen + C::OFF_Q + (piece >> 3) * 16384 + row * 128 + (((piece & 7) ^ (row & 7)) << 4)) = u;
                    else if (store && piece * 8 < a.dim) *reinterpret_cast<uint4*>(dst + piece * 8) = u;
                }
                __syncwarp();
            }
            if (whole && tokens > 0) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                asm volatile("bar.sync 9, 256;" ::: "memory");
                if (tid == 32 * SOFTMAX0 && ok) {
#pragma unroll 1
                    for (int c = 0; c * 64 < a.dim; ++c)
                        asm volatile("cp.async.bulk.tensor.5d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5, %6}], [%1];"
                                     ::"l"(reinterpret_cast<uint64_t>(&tmO)), "r"(sQ + c * 16384), "r"(c * 64), "r"(0), "r"(t0), "r"(kv), "r"(e) : "memory");
                    asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group 0;" ::: "memory");
                }
            }
        } else {
            // Sums of a share, 32 bits wide, by way of the rings, which are idle now, and the TMA, 32 columns at a time. (Rows behind the episode's last query
            // are written as well: nobody reads them.)
            if (store && g == 0)
                p.part_ml[((size_t)split * a.episodes + e) * a.tokens * a.heads + (size_t)(t0 + t) * a.heads + h] = make_float2(l == 0.f ? -INFINITY : m_end, !Q8 ? l : (l == 0.f ? -INFINITY : m_sum + log2f(l)));
#pragma unroll 1
            for (int c = 0; c < (busy && any ? SPAN : 0); c += 32) {
                float o[32];
                const int col = g * SPAN + c;
                tc5::tmem_ld32(tmem + t_lane + C::O_COL + col, o);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    *reinterpret_cast<float4*>(gen + C::OFF_R + (col >> 5) * 16384 + row * 128 + ((k ^ (row & 7)) << 4)) = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
            }
            if (any) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                asm volatile("bar.sync 9, 256;" ::: "memory");
                if (tid == 32 * SOFTMAX0 && ok) {
#pragma unroll 1
                    for (int c = 0; c < HDP / 32; ++c)
                        asm volatile("cp.async.bulk.tensor.5d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5, %6}], [%1];"
                                     ::"l"(reinterpret_cast<uint64_t>(&tmO)), "r"(ring + c * 16384), "r"(c * 32), "r"(0), "r"(t0), "r"(kv), "r"(split * a.episodes + e) : "memory");
                    asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group 0;" ::: "memory");
                }
            }
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

}  // namespace mattn
}  // namespace fvla

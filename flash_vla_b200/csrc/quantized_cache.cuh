// The 8-bit KV cache: e4m3 values with one power-of-two scale per block of rows and K/V head.
//
//   value = e4m3 * scale,   scale = the smallest power of two s with amax(block) <= 448 s   (at least 2^-120)
//
// e4m3 is a floating format: a power-of-two scale loses none of its precision (it only moves the exponents), and division by it is exact, so a value
// is rounded once, to e4m3, and a block whose scale has to grow later moves its old values by a power of two, exact down to the subnormals.
// Values that are not finite are held as NaN and do not take part in amax. (Reciprocals below are exact for powers of two.)
#pragma once

#include "common.cuh"

namespace fvla {
namespace q8 {

constexpr int kMinExponent = -120;

// Bits of the scale for a block whose largest finite |bf16 value| has the bits `amax` (bf16, sign cleared).
// 448 = 1.75 * 2^8: an amax of m * 2^x (1 <= m < 2) needs 2^(x-8) up to m = 1.75 and 2^(x-7) above it.
__device__ __forceinline__ float scale_of(uint32_t amax) {
    const int x = (int)(amax >> 7) - 127;                       // a subnormal amax lands far below the smallest scale
    const int e = x - ((amax & 0x7fu) <= 0x60u ? 8 : 7);
    return __int_as_float((max(e, kMinExponent) + 127) << 23);
}
// log2 of a positive scale, exact for a power of two. (Scales that this file makes are powers of two; a program may bring others.)
__device__ __forceinline__ float log2_of_scale(float s) {
    const uint32_t u = __float_as_uint(s), m = u & 0x7fffffu;
    const float whole = (float)((int)(u >> 23) - 127);
    return m == 0 ? whole : whole + __log2f(__uint_as_float(m | 0x3f800000u));
}

__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t pair) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)pair));
    float2 f;
    asm("{.reg .f16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;}" : "=f"(f.x), "=f"(f.y) : "r"(h));
    return f;
}
__device__ __forceinline__ uint32_t to_e5m2x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// Two bf16 values over a power of two -> e4m3 pair; what is not finite becomes NaN (0x7f).
__device__ __forceinline__ uint32_t quantize_pair(uint32_t bf, float inv) {
    const float2 f = unpack_bf16x2(bf);
    uint32_t r = to_e4m3x2(f.x * inv, f.y * inv);
    if ((bf & 0x7f80u) == 0x7f80u) r = (r & 0xff00u) | 0x7fu;
    if ((bf & 0x7f800000u) == 0x7f800000u) r = (r & 0x00ffu) | 0x7f00u;
    return r;
}
// Four e4m3 values times a power of two, rounded again.
__device__ __forceinline__ uint32_t rescale4(uint32_t v, float ratio) {
    const float2 a = from_e4m3x2(v & 0xffffu), b = from_e4m3x2(v >> 16);
    return to_e4m3x2(a.x * ratio, a.y * ratio) | (to_e4m3x2(b.x * ratio, b.y * ratio) << 16);
}
__device__ __forceinline__ uint32_t amax_pair(uint32_t amax, uint32_t bf) {
    const uint32_t lo = bf & 0x7fffu, hi = (bf >> 16) & 0x7fffu;
    if (lo < 0x7f80u) amax = max(amax, lo);
    if (hi < 0x7f80u) amax = max(amax, hi);
    return amax;
}

struct AppendArgs {
    const bf16* x[2];                 // new K, V rows (episodes, tokens, kv_heads, dim)
    uint8_t* held[2];                 // cache
    float* scale[2];                  // (episodes, blocks, kv_heads)
    long long xs[2][3], hs[2][3];     // strides in elements: episode, row, head
    const int *starts, *counts;
    int* status;
    int tokens, rows, blocks, block, kv_heads, dim;
};

constexpr int APPEND_THREADS = 256;

// One CTA per (block that a run of new rows can touch and head, K or V, episode): its new rows' amax, the scale, then old rows moved to that scale
// and new rows rounded. A thread takes 16 values at a time (32 bytes in, 16 out) and keeps all of its PER pieces in registers between the two, so that
// every byte is read once and all reads are in flight together; bound by the bytes (1 073 rows of 8 heads of 256 for eight episodes, 105 MB, 22 us:
// 4.8 TB/s, and 34 us when every value was looked at for infinities on its own).
template <int PER>
__global__ void __launch_bounds__(APPEND_THREADS) cache_append_kernel(const __grid_constant__ AppendArgs p) {
    __shared__ uint32_t warp_max[APPEND_THREADS / 32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int e = blockIdx.z, kv = blockIdx.y, head = blockIdx.x % p.kv_heads, w = blockIdx.x / p.kv_heads, threads = blockDim.x;
    const long long start = p.starts[e];
    const int count = p.counts ? min(max(p.counts[e], 0), p.tokens) : p.tokens;
    if (count > 0 && (start < 0 || start + count > p.rows) && threadIdx.x == 0 && blockIdx.x == 0 && kv == 0 && p.status) atomicExch(p.status, 8);
    const long long from = max(start, 0ll), to = min(start + count, (long long)p.rows);      // rows outside the cache are left out
    if (from >= to) return;
    const long long b = from / p.block + w, row0 = b * p.block;
    if (row0 >= to) return;
    const int first = (int)(max(from, row0) - row0), last = (int)(min(to, row0 + p.block) - row0);     // new rows of this block
    const int old = from > row0 ? first : 0;                                                           // rows that were there before
    const int chunks = p.dim / 16;
    const bf16* x = p.x[kv] + e * p.xs[kv][0] + (row0 - start) * p.xs[kv][1] + head * p.xs[kv][2];
    uint8_t* held = p.held[kv] + e * p.hs[kv][0] + row0 * p.hs[kv][1] + head * p.hs[kv][2];
    float* scale = p.scale[kv] + ((size_t)e * p.blocks + b) * p.kv_heads + head;
    const float was = old > 0 ? *scale : 0.f;

    uint4 u[PER][2];
    uint32_t amax = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = first * chunks + k * threads + threadIdx.x;
        const bool mine = i < last * chunks;
        const uint4* src = reinterpret_cast<const uint4*>(x + (long long)(i / chunks) * p.xs[kv][1] + (i % chunks) * 16);
#pragma unroll
        for (int h = 0; h < 2; ++h) u[k][h] = mine ? __ldg(src + h) : make_uint4(0, 0, 0, 0);
    }
    // two magnitudes at a time; a block with a value that is not finite (all but none) is looked through again, and rounded with care below
    uint32_t both = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h)
            both = __vmaxu2(__vmaxu2(both, __vmaxu2(u[k][h].x & 0x7fff7fffu, u[k][h].y & 0x7fff7fffu)), __vmaxu2(u[k][h].z & 0x7fff7fffu, u[k][h].w & 0x7fff7fffu));
    amax = max(both & 0xffffu, both >> 16);
    const bool odd = __syncthreads_or(amax >= 0x7f80u);          // and every thread has read the old scale
    if (odd) {
        amax = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) amax = amax_pair(amax_pair(amax_pair(amax_pair(amax, u[k][h].x), u[k][h].y), u[k][h].z), u[k][h].w);
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = amax;
    __syncthreads();
    for (int i = 0; i < threads / 32; ++i) amax = max(amax, warp_max[i]);
    const float now = fmaxf(was, scale_of(amax));
    if (threadIdx.x == 0) *scale = now;
    if (now != was) {
        const float ratio = was * __frcp_rn(now);
        for (int i = threadIdx.x; i < old * chunks; i += threads) {
            uint4* at = reinterpret_cast<uint4*>(held + (long long)(i / chunks) * p.hs[kv][1] + (i % chunks) * 16);
            const uint4 v = *at;
            *at = make_uint4(rescale4(v.x, ratio), rescale4(v.y, ratio), rescale4(v.z, ratio), rescale4(v.w, ratio));
        }
    }
    const float inv = __frcp_rn(now);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = first * chunks + k * threads + threadIdx.x;
        if (i >= last * chunks) break;
        uint32_t o[4];
        if (odd) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                o[2 * h] = quantize_pair(u[k][h].x, inv) | (quantize_pair(u[k][h].y, inv) << 16);
                o[2 * h + 1] = quantize_pair(u[k][h].z, inv) | (quantize_pair(u[k][h].w, inv) << 16);
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float2 a = unpack_bf16x2(u[k][h].x), b2 = unpack_bf16x2(u[k][h].y), c = unpack_bf16x2(u[k][h].z), d = unpack_bf16x2(u[k][h].w);
                o[2 * h] = to_e4m3x2(a.x * inv, a.y * inv) | (to_e4m3x2(b2.x * inv, b2.y * inv) << 16);
                o[2 * h + 1] = to_e4m3x2(c.x * inv, c.y * inv) | (to_e4m3x2(d.x * inv, d.y * inv) << 16);
            }
        }
        *reinterpret_cast<uint4*>(held + (long long)(i / chunks) * p.hs[kv][1] + (i % chunks) * 16) = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

// ------------------------------------------------------------------------------------------------ eviction
struct EvictArgs {
    const uint8_t* held[2];
    const float* scale[2];
    uint8_t* out[2];
    float* out_scale[2];
    long long hs[2][3], os[2][3];     // strides in elements: episode, row, head
    const float* weights;             // (episodes, rows)
    float* out_weights;               // (episodes, out_rows), may be null
    const int *lengths, *positions;   // positions (episodes, rows), may be null: row numbers
    int *out_lengths, *out_positions; // (episodes), (episodes, out_rows; may be null)
    int* source;                      // scratch (episodes, keep): the rows that stay, in order
    int rows, blocks, out_rows, out_blocks, block, out_block, kv_heads, dim, keep, sinks, recent;
};

constexpr int SELECT_THREADS = 1024;

// Order of weights as unsigned integers: larger is kept first. NaN counts as -infinity, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float w) {
    if (w != w) w = -INFINITY;
    const uint32_t u = __float_as_uint(w + 0.f);                // -0 + 0 = +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A cluster of `ctas` CTAs per episode: the threshold by a radix select of 8 bits at a time, then the rows that stay, in order. For both each warp has
// a run of rows of its own; lanes with equal digits add to the histogram together (weights are alike in their leading bits). The CTAs read
// one another's histograms (two in turn, so that one barrier per digit is enough) and, at last, counts. Bound by latencies: a digit takes a load,
// the votes, the barrier and a scan of 256 sums (eight episodes of 16 384 rows 16 us; one CTA each 41).
__device__ __forceinline__ uint32_t remote(const void* shared, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(shared)), "r"(rank));
    return r;
}
__device__ __forceinline__ uint32_t load_remote(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__global__ void __launch_bounds__(SELECT_THREADS) evict_select_kernel(const __grid_constant__ EvictArgs p, int ctas) {
    constexpr int WARPS = SELECT_THREADS / 32;
    __shared__ uint32_t hists[2][256];
    __shared__ uint32_t hist[256];
    __shared__ int cta_ties, cta_kept;
    __shared__ uint32_t s_prefix, s_left;
    __shared__ int warp_ties[WARPS], warp_kept[WARPS];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int e = blockIdx.x / ctas, rank = blockIdx.x % ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;      // (clusters are consecutive CTAs)
    auto cluster_barrier = [ctas]() {
        if (ctas == 1) { __syncthreads(); return; }
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    };
    const int L = min(max(p.lengths[e], 0), p.rows);
    const int n = min(L, p.keep);
    const float* w = p.weights + (size_t)e * p.rows;
    const int low = min(p.sinks, L), high = max(low, L - p.recent);       // rows [low, high) compete
    const int wanted = n - low - (L - high);                              // and so many of them stay (sinks + recent <= keep)
    const int run = ((L + ctas * WARPS - 1) / (ctas * WARPS) + 31) / 32 * 32, begin = (int)min((long long)(rank * WARPS + warp) * run, (long long)L), end = min(begin + run, L);
    const bool choose = L > p.keep;
    // a run of at most 64 rows stays in registers: two rows a lane
    const float held0 = begin + lane < end ? w[begin + lane] : 0.f, held1 = begin + 32 + lane < end ? w[begin + 32 + lane] : 0.f;
    auto weight = [&](int j0) { return j0 == begin ? held0 : (j0 == begin + 32 ? held1 : (j0 + lane < end ? w[j0 + lane] : 0.f)); };
    uint32_t threshold = 0xffffffffu, ties = 0;                           // nothing lies above the largest order
    if (choose && wanted > 0) {
        uint32_t prefix = 0, left = wanted;
        for (int shift = 24; shift >= 0; shift -= 8) {
            uint32_t* part = hists[shift >> 3 & 1];
            if (tid < 256) part[tid] = 0;
            __syncthreads();
#pragma unroll 4
            for (int j0 = begin; j0 < end; j0 += 32) {
                const int j = j0 + lane;
                const bool free = j < end && j >= low && j < high;
                const float x = weight(j0);
                const uint32_t u = free ? order_of(x) : 0;
                const bool counts = free && (shift == 24 || (u >> (shift + 8)) == prefix);
                const uint32_t digit = counts ? (u >> shift) & 255u : 256u;
                const uint32_t same = __match_any_sync(0xffffffffu, digit);
                if (counts && lane == __ffs(same) - 1) atomicAdd(&part[digit], (uint32_t)__popc(same));
            }
            cluster_barrier();
            if (tid < 256) {
                uint32_t sum = 0;
                if (ctas == 1) sum = part[tid];
                else
                    for (int c = 0; c < ctas; ++c) sum += load_remote(remote(part + tid, c));
                hist[tid] = sum;
            }
            __syncthreads();
            if (warp == 0) {
                // lane i has the digits 255 - 8 i .. 248 - 8 i: the digit at which the rows from above reach `left`
                uint32_t mine[8], sum = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) { mine[i] = hist[255 - 8 * lane - i]; sum += mine[i]; }
                uint32_t upto = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) { const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += x; }
                uint32_t above = upto - sum;
                if (above < left && upto >= left) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (above + mine[i] >= left) { s_prefix = (prefix << 8) | (uint32_t)(255 - 8 * lane - i); s_left = left - above; break; }
                        above += mine[i];
                    }
                }
            }
            __syncthreads();
            prefix = s_prefix;
            left = s_left;
        }
        threshold = prefix;
        ties = left;                                                      // so many rows of exactly this weight stay, the first ones
    }
    // what each warp's run has, then where its rows go
    int tied = 0, kept = 0;
#pragma unroll 4
    for (int j0 = begin; j0 < end; j0 += 32) {
        const int j = j0 + lane;
        const bool inside = j < end, free = inside && choose && j >= low && j < high;
        const float x = weight(j0);
        const uint32_t u = free ? order_of(x) : 0;
        tied += __popc(__ballot_sync(0xffffffffu, free && u == threshold));
        kept += __popc(__ballot_sync(0xffffffffu, inside && (!free || u > threshold)));
    }
    if (lane == 0) { warp_ties[warp] = tied; warp_kept[warp] = kept; }
    __syncthreads();
    if (warp == 0) {
        const int x = __reduce_add_sync(0xffffffffu, warp_ties[lane]), y = __reduce_add_sync(0xffffffffu, warp_kept[lane]);      // (32 warps)
        if (lane == 0) { cta_ties = x; cta_kept = y; }
    }
    cluster_barrier();
    int ties_before = 0, kept_before = 0;
    {
        int ties_cta = 0, kept_cta = 0;                                   // of the CTAs before this one
        for (int c = 0; c < rank; ++c) { ties_cta += (int)load_remote(remote(&cta_ties, c)); kept_cta += (int)load_remote(remote(&cta_kept, c)); }
        int x = warp_ties[lane], y = warp_kept[lane];
        const int own = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int z = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += z; }
        x += ties_cta;
        y += min(x, (int)ties) - min(x - own, (int)ties);                 // with the ties of the run that stay
        if (lane == 0) y += kept_cta + min(ties_cta, (int)ties);
        const int all = y - (lane == 0 ? kept_cta + min(ties_cta, (int)ties) : 0);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int z = __shfl_up_sync(0xffffffffu, y, o); if (lane >= o) y += z; }
        ties_before = __shfl_sync(0xffffffffu, x - own, warp);
        kept_before = __shfl_sync(0xffffffffu, y - all, warp);
    }
    for (int j0 = begin; j0 < end; j0 += 32) {
        const int j = j0 + lane;
        const bool inside = j < end, free = inside && choose && j >= low && j < high;
        const float x = weight(j0);
        const uint32_t u = free ? order_of(x) : 0, below = (1u << lane) - 1u;
        const bool tie = free && u == threshold;
        const uint32_t tie_mask = __ballot_sync(0xffffffffu, tie);
        const bool stays = inside && (!free || u > threshold || (tie && ties_before + __popc(tie_mask & below) < (int)ties));
        const uint32_t mask = __ballot_sync(0xffffffffu, stays);
        if (stays) {
            const int rank = kept_before + __popc(mask & below);
            p.source[(size_t)e * p.keep + rank] = j;
            if (p.out_weights) p.out_weights[(size_t)e * p.out_rows + rank] = x;
            if (p.out_positions) p.out_positions[(size_t)e * p.out_rows + rank] = p.positions ? p.positions[(size_t)e * p.rows + j] : j;
        }
        ties_before += __popc(tie_mask);
        kept_before += __popc(mask);
    }
    if (tid == 0 && rank == 0) p.out_lengths[e] = n;
    cluster_barrier();                                                    // nobody leaves while its counts may be read
}

constexpr int MOVE_THREADS = 128;

// One CTA per (block of the result and head, K or V, episode): its scale is the largest of its rows' source scales; rows of another scale
// are moved to it by a power of two. Rows are fetched, PER pieces of 16 bytes a thread in flight, while the scales are looked up.
// Bound by the bytes: 4 096 rows of 8 heads of 128 for eight episodes, 134 MB, 23 us.
template <int PER>
__global__ void __launch_bounds__(MOVE_THREADS) evict_move_kernel(const __grid_constant__ EvictArgs p) {
    __shared__ int row_of[128];
    __shared__ float scale_of_row[128];
    __shared__ float warp_top[MOVE_THREADS / 32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int e = blockIdx.z, kv = blockIdx.y, head = blockIdx.x % p.kv_heads, b = blockIdx.x / p.kv_heads, tid = threadIdx.x;
    const int n = min(min(max(p.lengths[e], 0), p.rows), p.keep);
    const int row0 = b * p.out_block, have = min(p.out_block, n - row0);
    if (have <= 0) return;
    const int j = tid < have ? p.source[(size_t)e * p.keep + row0 + tid] : 0;
    row_of[tid] = j;
    __syncthreads();
    const int chunks = p.dim / 16;
    const uint8_t* held = p.held[kv] + e * p.hs[kv][0] + head * p.hs[kv][2];
    uint8_t* out = p.out[kv] + e * p.os[kv][0] + (long long)row0 * p.os[kv][1] + head * p.os[kv][2];
    float top = tid < have ? p.scale[kv][((size_t)e * p.blocks + j / p.block) * p.kv_heads + head] : 0.f;
    uint4 u[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = k * MOVE_THREADS + tid;
        u[k] = i < have * chunks ? __ldg(reinterpret_cast<const uint4*>(held + row_of[i / chunks] * p.hs[kv][1] + i % chunks * 16)) : make_uint4(0, 0, 0, 0);
    }
    scale_of_row[tid] = top;
    top = warp_max(top);
    if ((tid & 31) == 0) warp_top[tid >> 5] = top;
    __syncthreads();
    const float now = fmaxf(fmaxf(warp_top[0], warp_top[1]), fmaxf(warp_top[2], warp_top[3]));
    if (tid == 0) p.out_scale[kv][((size_t)e * p.out_blocks + b) * p.kv_heads + head] = now;
    const float inv = __frcp_rn(now);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = k * MOVE_THREADS + tid, r = i / chunks;
        if (i >= have * chunks) break;
        const float ratio = scale_of_row[r] * inv;
        if (ratio != 1.f) u[k] = make_uint4(rescale4(u[k].x, ratio), rescale4(u[k].y, ratio), rescale4(u[k].z, ratio), rescale4(u[k].w, ratio));
        *reinterpret_cast<uint4*>(out + r * p.os[kv][1] + i % chunks * 16) = u[k];
    }
}

}  // namespace q8
}  // namespace fvla

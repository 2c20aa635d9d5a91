// extern "C" entries of masked attention and of the 8-bit KV cache: argument validation and launches. Nothing here allocates, frees or synchronises.
#include "common.cuh"
#include "masked_attention.cuh"
#include "quantized_cache.cuh"

namespace fvla {

static inline cudaStream_t S(void* s) { return reinterpret_cast<cudaStream_t>(s); }

template <typename... KArgs, typename... Args>
static int launch(const char* what, void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args) {
    const cudaError_t e = launch_pdl(kern, grid, block, smem, st, args...);
    if (e != cudaSuccess) { set_error("%s: %s", what, cudaGetErrorString(e)); return FVLA_ERR_LAUNCH; }
    return check_launch(what);
}

static bool block_ok(int block) { return block == 16 || block == 32 || block == 64 || block == 128; }
// Element strides such that every row starts on 16 bytes.
static bool strides_ok(const long long (&s)[3], int multiple) { return s[0] % multiple == 0 && s[1] % multiple == 0 && s[2] % multiple == 0; }

static int check_attention(const struct fvla_attention* a) {
    FVLA_REQUIRE(a != nullptr, "attention: null arguments");
    const bool decay = a->tokens == 0 && a->weights != nullptr;            // no query: the weights decay, and nothing else is written
    FVLA_REQUIRE(a->episodes > 0 && (a->tokens > 0 || decay) && a->keys >= 0 && a->heads > 0 && a->kv_heads > 0, "attention: empty shape");
    FVLA_REQUIRE(a->heads % a->kv_heads == 0 && a->heads / a->kv_heads <= 128, "attention: %d heads over %d K/V heads", a->heads, a->kv_heads);
    const bool q8 = a->k_scale != nullptr;
    const int multiple = q8 ? 16 : 8;
    FVLA_REQUIRE(a->head_dim > 0 && a->head_dim <= 256 && a->head_dim % multiple == 0, "attention: head_dim %d (a multiple of %d up to 256)", a->head_dim, multiple);
    FVLA_REQUIRE((decay || (a->q != nullptr && a->out != nullptr)) && (a->keys == 0 || (a->k != nullptr && a->v != nullptr)), "attention: null pointer");
    FVLA_REQUIRE((a->v_scale != nullptr) == q8, "attention: scales of both K and V, or of neither");
    FVLA_REQUIRE(aligned16(a->q) && aligned16(a->k) && aligned16(a->v) && aligned16(a->out), "attention: every tensor must be 16-byte aligned");
    FVLA_REQUIRE(strides_ok(a->q_stride, 8) && strides_ok(a->out_stride, 8) && strides_ok(a->k_stride, multiple) && strides_ok(a->v_stride, multiple),
                 "attention: every row must start on 16 bytes");
    FVLA_REQUIRE((a->tokens <= 1 || a->q_stride[1] > 0) && (a->heads == 1 || a->q_stride[2] > 0) && (a->keys <= 1 || (a->k_stride[1] > 0 && a->v_stride[1] > 0)),
                 "attention: tokens or query heads that share their memory");
    FVLA_REQUIRE((a->episodes == 1 || a->out_stride[0] > 0) && (a->tokens <= 1 || a->out_stride[1] > 0) && (a->heads == 1 || a->out_stride[2] > 0),
                 "attention: rows of the result that share their memory");
    for (int i = 0; i < 3; ++i) FVLA_REQUIRE(a->q_stride[i] >= 0 && a->k_stride[i] >= 0 && a->v_stride[i] >= 0 && a->out_stride[i] >= 0, "attention: negative strides");
    FVLA_REQUIRE(!q8 || (block_ok(a->block) && a->keys % a->block == 0), "attention: blocks of %d rows in %d", a->block, a->keys);
    FVLA_REQUIRE((a->q_docs != nullptr) == (a->k_docs != nullptr), "attention: documents of queries and keys, or of neither");
    FVLA_REQUIRE(a->prefix == nullptr || a->causal, "attention: a prefix without the causal mask");
    FVLA_REQUIRE(a->weights == nullptr || ((a->lse != nullptr || decay) && q8), "attention: weights need the 8-bit cache and the log-sum-exp");
    const auto finite = [](float x) { return x - x == 0.f; };
    FVLA_REQUIRE(a->cap >= 0.f && finite(a->cap * kLog2e) && finite(a->scale * kLog2e) && finite(a->decay) && (a->cap == 0.f || finite(a->scale / a->cap)),
                 "attention: scale, cap and decay must be finite, scale over cap as well, the cap not negative");
    FVLA_REQUIRE((long long)a->tokens * a->heads < (1ll << 31) && (long long)a->episodes * a->tokens * a->heads < (1ll << 31) && (long long)a->episodes * a->kv_heads < 65536, "attention: too many rows");
    FVLA_REQUIRE(((long long)a->tokens / (128 / (a->heads / a->kv_heads)) + 1) * a->kv_heads * a->episodes < (1ll << 30), "attention: too many rows");
    return FVLA_OK;
}

static mattn::Args attention_args(const struct fvla_attention* a) {
    mattn::Args p;
    p.q = a->q; p.k = a->k; p.v = a->v; p.k_scale = static_cast<const float*>(a->k_scale); p.v_scale = static_cast<const float*>(a->v_scale);
    p.out = static_cast<bf16*>(a->out); p.lse = static_cast<float*>(a->lse);
    p.prefix = a->prefix; p.q_lens = a->q_lens; p.k_lens = a->k_lens; p.q_start = a->q_start; p.q_docs = a->q_docs; p.k_docs = a->k_docs; p.k_pos = a->k_pos;
    p.slopes = a->slopes; p.weights = static_cast<float*>(a->weights);
    for (int i = 0; i < 3; ++i) { p.qs[i] = a->q_stride[i]; p.ks[i] = a->k_stride[i]; p.vs[i] = a->v_stride[i]; p.os[i] = a->out_stride[i]; }
    p.scale = a->scale; p.cap = a->cap; p.decay = a->decay;
    p.episodes = a->episodes; p.tokens = a->tokens; p.keys = a->keys; p.heads = a->heads; p.kv_heads = a->kv_heads; p.dim = a->head_dim;
    p.block = a->block; p.causal = a->causal;
    return p;
}

}  // namespace fvla

using namespace fvla;

extern "C" {

size_t fvla_attention_workspace_bytes(const struct fvla_attention* a) {
    return check_attention(a) ? 0 : mattn::workspace_bytes(attention_args(a));
}

int fvla_attention_run(const struct fvla_attention* a, void* stream) {
    int rc = check_attention(a);
    if (rc) return rc;
    const mattn::Args p = attention_args(a);
    if (a->tokens == 0) return mattn::launch_weights(p, S(stream));
    const size_t need = mattn::workspace_bytes(p);
    if (need > 0 && (a->ws == nullptr || a->ws_bytes < need)) { set_error("attention: workspace of %zu bytes needed", need); return FVLA_ERR_WORKSPACE; }
    FVLA_REQUIRE(aligned16(a->ws), "attention: the workspace must be 16-byte aligned");
    return mattn::launch_attention(p, a->ws, device_status_ptr(), S(stream));
}

int fvla_cache_append(const struct fvla_cache_append_args* a, void* stream) {
    FVLA_REQUIRE(a != nullptr, "cache_append: null arguments");
    FVLA_REQUIRE(a->episodes > 0 && a->episodes < 65536 && a->tokens > 0 && a->rows > 0 && a->kv_heads > 0, "cache_append: empty shape");
    FVLA_REQUIRE(a->head_dim > 0 && a->head_dim <= 256 && a->head_dim % 16 == 0, "cache_append: head_dim %d (a multiple of 16 up to 256)", a->head_dim);
    FVLA_REQUIRE(block_ok(a->block) && a->rows % a->block == 0, "cache_append: blocks of %d rows in %d", a->block, a->rows);
    FVLA_REQUIRE(a->tokens <= a->rows, "cache_append: %d rows into a cache of %d", a->tokens, a->rows);
    FVLA_REQUIRE(a->k && a->v && a->k_held && a->v_held && a->k_scale && a->v_scale && a->starts, "cache_append: null pointer");
    FVLA_REQUIRE(aligned16(a->k) && aligned16(a->v) && aligned16(a->k_held) && aligned16(a->v_held), "cache_append: every tensor must be 16-byte aligned");
    FVLA_REQUIRE(strides_ok(a->k_stride, 8) && strides_ok(a->v_stride, 8) && strides_ok(a->k_held_stride, 16) && strides_ok(a->v_held_stride, 16),
                 "cache_append: every row must start on 16 bytes");
    q8::AppendArgs p;
    p.x[0] = static_cast<const bf16*>(a->k); p.x[1] = static_cast<const bf16*>(a->v);
    p.held[0] = static_cast<uint8_t*>(a->k_held); p.held[1] = static_cast<uint8_t*>(a->v_held);
    p.scale[0] = static_cast<float*>(a->k_scale); p.scale[1] = static_cast<float*>(a->v_scale);
    for (int i = 0; i < 3; ++i) { p.xs[0][i] = a->k_stride[i]; p.xs[1][i] = a->v_stride[i]; p.hs[0][i] = a->k_held_stride[i]; p.hs[1][i] = a->v_held_stride[i]; }
    p.starts = a->starts; p.counts = a->counts; p.status = device_status_ptr();
    p.tokens = a->tokens; p.rows = a->rows; p.blocks = a->rows / a->block; p.block = a->block; p.kv_heads = a->kv_heads; p.dim = a->head_dim;
    const int windows = (a->tokens + a->block - 2) / a->block + 1;           // blocks that a run of so many rows can touch
    const int chunks = a->block * a->head_dim / 16, threads = chunks < q8::APPEND_THREADS ? (chunks + 31) / 32 * 32 : q8::APPEND_THREADS;      // pieces of 16 values of a block
    const dim3 grid(windows * a->kv_heads, 2, a->episodes);
    const auto kern = chunks <= q8::APPEND_THREADS ? q8::cache_append_kernel<1> : (chunks <= 2 * q8::APPEND_THREADS ? q8::cache_append_kernel<2> :
                      (chunks <= 4 * q8::APPEND_THREADS ? q8::cache_append_kernel<4> : q8::cache_append_kernel<8>));
    return launch("cache_append_kernel", kern, grid, dim3(threads), 0, S(stream), p);
}

size_t fvla_cache_evict_workspace_bytes(int episodes, int keep) { return episodes > 0 && keep > 0 ? (size_t)episodes * keep * sizeof(int) : 0; }

int fvla_cache_evict(const struct fvla_cache_evict_args* a, void* stream) {
    FVLA_REQUIRE(a != nullptr, "cache_evict: null arguments");
    FVLA_REQUIRE(a->episodes > 0 && a->episodes < 65536 && a->rows > 0 && a->out_rows > 0 && a->kv_heads > 0 && a->keep > 0, "cache_evict: empty shape");
    FVLA_REQUIRE(a->keep <= a->out_rows, "cache_evict: %d rows to keep in a cache of %d", a->keep, a->out_rows);
    FVLA_REQUIRE(a->sinks >= 0 && a->recent >= 0 && (long long)a->sinks + a->recent <= a->keep, "cache_evict: %d first and %d last rows in %d", a->sinks, a->recent, a->keep);
    FVLA_REQUIRE(a->head_dim > 0 && a->head_dim <= 256 && a->head_dim % 16 == 0, "cache_evict: head_dim %d (a multiple of 16 up to 256)", a->head_dim);
    FVLA_REQUIRE(block_ok(a->block) && a->rows % a->block == 0 && block_ok(a->out_block) && a->out_rows % a->out_block == 0, "cache_evict: blocks of %d rows in %d, %d in %d",
                 a->block, a->rows, a->out_block, a->out_rows);
    FVLA_REQUIRE(a->k && a->v && a->k_scale && a->v_scale && a->out_k && a->out_v && a->out_k_scale && a->out_v_scale && a->weights && a->lengths && a->out_lengths,
                 "cache_evict: null pointer");
    FVLA_REQUIRE(aligned16(a->k) && aligned16(a->v) && aligned16(a->out_k) && aligned16(a->out_v), "cache_evict: every tensor must be 16-byte aligned");
    FVLA_REQUIRE(strides_ok(a->k_stride, 16) && strides_ok(a->v_stride, 16) && strides_ok(a->out_k_stride, 16) && strides_ok(a->out_v_stride, 16),
                 "cache_evict: every row must start on 16 bytes");
    if (a->ws == nullptr || a->ws_bytes < fvla_cache_evict_workspace_bytes(a->episodes, a->keep)) {
        set_error("cache_evict: workspace of %zu bytes needed", fvla_cache_evict_workspace_bytes(a->episodes, a->keep));
        return FVLA_ERR_WORKSPACE;
    }
    q8::EvictArgs p;
    p.held[0] = static_cast<const uint8_t*>(a->k); p.held[1] = static_cast<const uint8_t*>(a->v);
    p.scale[0] = static_cast<const float*>(a->k_scale); p.scale[1] = static_cast<const float*>(a->v_scale);
    p.out[0] = static_cast<uint8_t*>(a->out_k); p.out[1] = static_cast<uint8_t*>(a->out_v);
    p.out_scale[0] = static_cast<float*>(a->out_k_scale); p.out_scale[1] = static_cast<float*>(a->out_v_scale);
    for (int i = 0; i < 3; ++i) { p.hs[0][i] = a->k_stride[i]; p.hs[1][i] = a->v_stride[i]; p.os[0][i] = a->out_k_stride[i]; p.os[1][i] = a->out_v_stride[i]; }
    p.weights = static_cast<const float*>(a->weights); p.out_weights = static_cast<float*>(a->out_weights);
    p.lengths = a->lengths; p.positions = a->positions; p.out_lengths = a->out_lengths; p.out_positions = a->out_positions;
    p.source = static_cast<int*>(a->ws);
    p.rows = a->rows; p.blocks = a->rows / a->block; p.out_rows = a->out_rows; p.out_blocks = a->out_rows / a->out_block; p.block = a->block; p.out_block = a->out_block;
    p.kv_heads = a->kv_heads; p.dim = a->head_dim; p.keep = a->keep; p.sinks = a->sinks; p.recent = a->recent;
    // up to 2 048 rows one CTA (two rows a thread), beyond them eight
    const int ctas = a->rows <= 2 * q8::SELECT_THREADS ? 1 : 8;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a->episodes * ctas); cfg.blockDim = dim3(q8::SELECT_THREADS); cfg.stream = S(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    const cudaError_t launched = cudaLaunchKernelEx(&cfg, q8::evict_select_kernel, p, ctas);
    if (launched != cudaSuccess) { set_error("evict_select_kernel: %s", cudaGetErrorString(launched)); return FVLA_ERR_LAUNCH; }
    const int rc = check_launch("evict_select_kernel");
    if (rc) return rc;
    const int chunks = a->out_block * a->head_dim / 16;
    const auto move = chunks <= 2 * q8::MOVE_THREADS ? q8::evict_move_kernel<2> : (chunks <= 4 * q8::MOVE_THREADS ? q8::evict_move_kernel<4> :
                      (chunks <= 8 * q8::MOVE_THREADS ? q8::evict_move_kernel<8> : q8::evict_move_kernel<16>));
    return launch("evict_move_kernel", move, dim3((a->keep + a->out_block - 1) / a->out_block * a->kv_heads, 2, a->episodes), dim3(q8::MOVE_THREADS), 0, S(stream), p);
}

}  // extern "C"

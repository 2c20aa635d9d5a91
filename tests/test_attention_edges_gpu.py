"""Masked attention and the 8-bit cache on the GPU where their arithmetic, their plans and their operands have edges, against plain 64-bit forms."""
from __future__ import annotations

import math

import pytest
import torch

import attention_cases as A
from flash_vla_b200 import op_table
from flash_vla_b200.hardware.nvidia.b200.pi0.backends.cuda import _lib
from flash_vla_b200.hardware.nvidia.b200.pi0.buffers import QuantizedCache, allocate_quantized_cache

pytestmark = pytest.mark.gpu
bf16, f32, i32, e4m3 = torch.bfloat16, torch.float32, torch.int32, torch.float8_e4m3fn
NAN, INF = math.nan, math.inf
P_8BIT = 2.0 ** -11      # half a step of the probabilities over the 8-bit cache


@pytest.fixture(autouse=True)
def no_wait_has_run_out():
    """A kernel that gives up on a wait leaves a code in the device's health word."""
    yield
    torch.cuda.synchronize()
    assert _lib.load().fvla_device_status(None) == 0


def randn(seed, *shape, dtype=bf16):
    return torch.randn(shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(dtype)


def cache_of(K, V, block=64):
    E, rows, HK, D = K.shape
    cache = allocate_quantized_cache(E, rows, HK, D, "cuda", block)
    op_table().cache_append(K, V, cache, A.ints([0] * E))
    return cache


def check_cached(Q, cache, lengths, scale, **kw):
    """Result, log-sum-exp and weights against the 64-bit form, and the result without the two.

    P, a probability times V's scale, is held in three 8-bit terms against the largest P of the row, which stands at 2^6 or more (few rows: 2^4). Two terms of
    e4m3 leave P 2^-8 or, among its subnormals (steps of 2^-9), 2^-10; a third of e5m2 at most 2^-3 of that: P 2^-11, or 2^-13, which is 2^-19 of the largest.
    (Few rows, where the terms are e4m3 times 1, 2^-4 and 2^-8: 2^-10, then 2^-14, then 2^-18 are left, 2^-22 of the largest.) So the probabilities' half
    step is on top of one term for each key: 2^-19 (2^-22) of the largest P, times the value that the cache holds."""
    D, rows = Q.shape[3], cache.K.shape[1]
    want = A.attention(Q, A.widened(cache.K, cache.K_scale), A.widened(cache.V, cache.V_scale), scale, k_lens=lengths, **kw)
    HK = cache.K.shape[2]
    group = Q.shape[2] // HK
    lowest = 2.0 ** (-22 if Q.shape[1] * group <= 32 else -19)
    per_row = cache.V_scale.double().repeat_interleave(rows // cache.V_scale.shape[1], 1).transpose(1, 2).repeat_interleave(group, 1)        # (E, H, rows)
    top = (want["p"] * per_row[:, :, None]).amax(-1)                                                                                    # (E, H, T)
    held = cache.V.double().abs().permute(0, 2, 1, 3).repeat_interleave(group, 1)
    want["spread"] = want["spread"] + (top[..., None] * ((want["p"] > 0).double() @ held)).permute(0, 2, 1, 3) * (lowest / P_8BIT)
    out, lse, bare = torch.full_like(Q, 7.0), torch.full((Q.shape[0], Q.shape[2], Q.shape[1]), 7.0, device="cuda"), torch.full_like(Q, 7.0)
    before = randn(9, Q.shape[0], rows, dtype=f32).abs()
    w = before.clone()
    op_table().cache_attention(Q, cache, lengths, scale, out, lse=lse, weights=w, decay=0.5, **kw)
    A.check_out(out, want, D, P_8BIT)
    A.check_lse(lse, want, D)
    A.check_weights(w, want, D, lengths, before, 0.5)
    op_table().cache_attention(Q, cache, lengths, scale, bare, **kw)
    assert torch.equal(bare, out)
    return out, want


# Both kernels, with the shares of a row in one CTA, in a cluster and in scratch (the comments: shares of a row at 148 SMs)
SHARED_OUT = [  # episodes, tokens, rows, heads, kv heads, dim, block
    (1, 1, 128, 8, 1, 64, 16),      # few rows: 1
    (2, 1, 1024, 8, 1, 256, 64),    # 8, a cluster
    (1, 2, 4096, 16, 2, 128, 32),   # 8 of four blocks
    (1, 4, 1024, 8, 1, 256, 128),   # 32 rows, 8
    (32, 1, 640, 8, 8, 128, 64),    # 3
    (1, 1, 12800, 8, 1, 256, 64),   # 100, in scratch
    (2, 51, 832, 8, 1, 256, 64),    # 128-row tiles: 7
    (1, 40, 640, 8, 2, 64, 16),     # 5
    (8, 160, 512, 8, 1, 128, 64),   # 80 tiles: 1
    (8, 160, 512, 8, 1, 256, 16)]   # 1


@pytest.mark.parametrize("where", ["first", "middle", "last", "all", "all but one", "every other"])
@pytest.mark.parametrize("shape", SHARED_OUT)
def test_values_that_are_zero(shape, where):
    """Blocks of V that are all zero get the smallest scale there is. Their keys count in the row sums like any others."""
    E, T, rows, H, HK, D, block = shape
    K, V = randn(31, E, rows, HK, D), randn(32, E, rows, HK, D)
    middle = rows // 256 * 128
    at = {"first": slice(0, 128), "middle": slice(middle, middle + 128), "last": slice(rows - 128, rows), "all": slice(0, rows), "all but one": slice(0, rows - block),
          "every other": None}[where]
    if at is None:
        V.view(E, rows // block, block, HK, D)[:, ::2] = 0.0
    else:
        V[:, at] = 0.0
    cache = cache_of(K, V, block)
    assert (cache.V_scale == 2.0 ** -120).any()
    lengths = A.ints([rows - 3 * (e % 3) for e in range(E)])
    check_cached(randn(33, E, T, H, D), cache, lengths, D ** -0.5, causal=True)


@pytest.mark.parametrize("T", [1, 4, 40])
@pytest.mark.parametrize("size", [1e-36, 1e-20, 1e30])
def test_values_of_every_size(T, size):
    """V of one small or large size throughout, beside zeros, and beside values of another size that the scores tell apart."""
    E, rows, H, HK, D = 2, 512, 8, 1, 128
    Q, K, V = randn(41, E, T, H, D), randn(42, E, rows, HK, D), randn(43, E, rows, HK, D)
    lengths = A.ints([512, 301])
    V = (V.float() * size).to(bf16)
    check_cached(Q, cache_of(K, V), lengths, D ** -0.5)
    V[:, 128:256] = 0.0
    check_cached(Q, cache_of(K, V), lengths, D ** -0.5)
    V[:, 384:] = randn(44, E, 128, HK, D)
    V[:, 64:128] = randn(45, E, 64, HK, D)
    for scale in (D ** -0.5, 4.0):
        check_cached(Q, cache_of(K, V), lengths, scale)


@pytest.mark.parametrize("T", [1, 4, 40])
@pytest.mark.parametrize("gap", [8.0, 20.0, 70.0, 140.0])
def test_many_small_probabilities_of_zero_values(T, gap):
    """4 032 keys whose V is zero, each `gap` log2 units below (and above) the 64 that have values: together they count in every row sum."""
    rows, H, D = 4096, 8, 128
    Q, K, V = torch.zeros(1, T, H, D, dtype=bf16, device="cuda"), torch.zeros(1, rows, 1, D, dtype=bf16, device="cuda"), torch.zeros(1, rows, 1, D, dtype=bf16, device="cuda")
    Q[..., 0] = 1.0
    V[:, 2048:2112] = randn(51, 1, 64, 1, D)
    for sign in (1.0, -1.0):
        K[..., 0] = 0.0
        K[:, 2048:2112, :, 0] = sign
        check_cached(Q, cache_of(K, V), A.ints([rows]), gap * math.log(2.0))


@pytest.mark.parametrize("T", [1, 4, 40])
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("unused", [0.0, NAN, INF, 1e-40, -1.0])
def test_scales_behind_the_lengths_may_be_anything(T, block, unused):
    """Blocks that no row has reached (a cache whose scales were never initialised) have no part in either kernel."""
    E, rows, H, HK, D = 3, 512, 8, 1, 128
    cache = cache_of(randn(61, E, rows, HK, D), randn(62, E, rows, HK, D), block)
    Q, lengths = randn(63, E, T, H, D), A.ints([512 - 3 * block, 129, 40])
    kw = {"causal": True, "slopes": torch.full((H,), 0.01, device="cuda")}
    want, w = torch.zeros_like(Q), torch.zeros(E, rows, device="cuda")
    op_table().cache_attention(Q, cache, lengths, 0.1, want, weights=w, **kw)
    for e, L in enumerate(lengths.tolist()):
        for scale in cache[2:]:
            scale[e, (L + block - 1) // block:] = unused
    out, again = torch.zeros_like(Q), torch.zeros_like(w)
    op_table().cache_attention(Q, cache, lengths, 0.1, out, weights=again, **kw)
    assert torch.isfinite(out).all() and torch.equal(out, want) and torch.equal(again, w)


def test_clusters_of_two_streams_share_the_tensor_memory():
    """Two kernels whose CTAs fit an SM together by their shared memory, but not by their tensor memory (512 and 64 of 512 columns), each of clusters that meet."""
    rows = 4096
    sets = []
    for i, (E, T, H, HK, D) in enumerate([(16, 4, 8, 1, 256), (16, 1, 8, 2, 128)]):
        cache = cache_of(randn(71 + i, E, rows, HK, D), randn(73 + i, E, rows, HK, D))
        Q, lengths = randn(75 + i, E, T, H, D), A.ints([rows - 7 * e for e in range(E)])
        want = torch.zeros_like(Q)
        op_table().cache_attention(Q, cache, lengths, 0.1, want)
        sets.append((torch.cuda.Stream(), cache, Q, lengths, torch.zeros_like(Q), want))
    torch.cuda.synchronize()
    for _ in range(100):
        for stream, cache, Q, lengths, out, _ in sets:
            with torch.cuda.stream(stream):
                op_table().cache_attention(Q, cache, lengths, 0.1, out)
    torch.cuda.synchronize()
    for *_, out, want in sets:
        assert torch.equal(out, want)


@pytest.mark.parametrize("T,rows", [(1, 4096), (1, 12800), (51, 832)])
def test_weights_where_the_result_replaces_the_queries(T, rows):
    cache = cache_of(randn(81, 2, rows, 1, 256), randn(82, 2, rows, 1, 256))
    Q, lengths = randn(83, 2, T, 8, 256), A.ints([rows, rows - 100])
    out, w = torch.zeros_like(Q), torch.zeros(2, rows, device="cuda")
    op_table().cache_attention(Q, cache, lengths, 0.06, out, weights=w)
    again = torch.zeros_like(w)
    op_table().cache_attention(Q, cache, lengths, 0.06, Q, weights=again)
    assert torch.equal(Q, out) and torch.equal(w, again)


def test_weights_decay_without_a_query():
    """No token at all, as for a batch whose episodes all wait: the weights decay as with no query of an episode's own."""
    cache, w = cache_of(randn(91, 2, 256, 1, 64), randn(92, 2, 256, 1, 64)), torch.full((2, 256), 2.0, device="cuda")
    none = torch.empty(2, 0, 8, 64, dtype=bf16, device="cuda")
    op_table().cache_attention(none, cache, A.ints([256, 100]), 0.1, none.clone(), weights=w, decay=0.25)
    assert (w[0] == 0.5).all() and (w[1, :100] == 0.5).all() and (w[1, 100:] == 2).all()
    w[1, 40] = NAN
    op_table().cache_attention(none, cache, A.ints([0, 50]), 0.1, none.clone(), weights=w, decay=0.0, lse=torch.empty(2, 8, 0, device="cuda"))
    assert (w[0] == 0.5).all() and (w[1, :50] == 0).all() and (w[1, 50:100] == 0.5).all()
    op_table().cache_attention(none, cache, A.ints([256, 256]), 0.1, none.clone())
    op_table().masked_attention(none, randn(93, 2, 5, 1, 64), randn(94, 2, 5, 1, 64), 0.1, none.clone())


@pytest.mark.parametrize("layout", ["rows of K and V", "heads of K and V", "layers"])
def test_evict_between_interleaved_tensors(layout):
    """K and V of a cache as views of one tensor, and the source and the destination as two layers of one stack: what goes where is the same as between whole tensors."""
    E, rows, HK, D, keep = 2, 256, 2, 64, 100

    def views(n):
        if layout == "rows of K and V":
            t = torch.zeros(E, n, 2, HK, D, dtype=torch.uint8, device="cuda").view(e4m3)
            return t[:, :, 0], t[:, :, 1], t
        if layout == "heads of K and V":
            t = torch.zeros(E, n, HK, 2, D, dtype=torch.uint8, device="cuda").view(e4m3)
            return t[:, :, :, 0], t[:, :, :, 1], t
        t = torch.zeros(2, E, 3, n, HK, D, dtype=torch.uint8, device="cuda").view(e4m3)
        return t[0, :, 1], t[1, :, 1], t

    K, V = randn(95, E, rows, HK, D), randn(96, E, rows, HK, D)
    whole = cache_of(K, V)
    k, v, _ = views(rows)
    cache = QuantizedCache(k, v, *(torch.ones(E, rows // 64, HK, device="cuda") for _ in range(2)))
    op_table().cache_append(K, V, cache, A.ints([0] * E))
    w = randn(97, E, rows, dtype=f32)
    k, v, _ = views(128)
    out = QuantizedCache(k, v, *(torch.ones(E, 2, HK, device="cuda") for _ in range(2)))
    want, n, m = allocate_quantized_cache(E, 128, HK, D, "cuda"), A.ints([0, 0]), A.ints([0, 0])
    op_table().cache_evict(whole, A.ints([256, 90]), w, keep, want, n)
    op_table().cache_evict(cache, A.ints([256, 90]), w, keep, out, m)
    assert torch.equal(n, m)
    for a, b in zip(out, want):
        assert A.same_bits(a.contiguous(), b)
    if layout == "layers":                                                     # from one layer to the next
        store = [torch.zeros(E, 3, rows, HK, D, dtype=torch.uint8, device="cuda").view(e4m3) for _ in range(2)]
        src = QuantizedCache(store[0][:, 0], store[1][:, 0], *(s.clone() for s in whole[2:]))
        dst = QuantizedCache(store[0][:, 1], store[1][:, 1], *(torch.ones(E, 4, HK, device="cuda") for _ in range(2)))
        for held, full in zip(src[:2], whole[:2]):
            held.view(torch.uint8).copy_(full.view(torch.uint8))
        op_table().cache_evict(src, A.ints([256, 90]), w, keep, dst, m)
        for a, b in zip(dst[:2], want[:2]):
            assert A.same_bits(a[:, :keep].contiguous()[0], b[0, :keep]) and A.same_bits(a[1, :90].contiguous(), b[1, :90])
    with pytest.raises(ValueError, match="lies over"):                         # one row on: the source's rows in the destination
        t = torch.zeros(E, rows + 128, HK, D, dtype=torch.uint8, device="cuda").view(e4m3)
        op_table().cache_evict(whole._replace(K=t[:, :rows]), A.ints([256, 90]), w, keep, want._replace(K=t[:, rows - 1:rows + 127]), m)


PROMPTS = [  # episodes, tokens, rows, heads, kv heads, dim, block: 128-row tiles over the 8-bit cache whose keys one CTA walks (75 tiles and more, or one block of keys)
    (8, 160, 512, 8, 1, 256, 64), (10, 64, 384, 32, 8, 128, 32), (6, 300, 304, 12, 4, 80, 16), (1, 51, 128, 8, 1, 256, 128), (2, 70, 96, 4, 4, 64, 32), (5, 257, 640, 3, 1, 16, 64)]


@pytest.mark.parametrize("shape", PROMPTS)
@pytest.mark.parametrize("kind", ["plain", "all", "positions"])
def test_prompts_over_the_cache(shape, kind):
    E, T, rows, H, HK, D, block = shape
    size = torch.exp2(torch.arange(rows, device="cuda").div(16, rounding_mode="floor").remainder(7).float() - 3)[None, :, None, None]      # blocks of unlike scales
    cache = cache_of((randn(101, E, rows, HK, D).float() * size).to(bf16), (randn(102, E, rows, HK, D).float() * size.flip(1)).to(bf16), block)
    Q = (randn(103, E, T, H, D).float() * 0.25).to(bf16)
    lengths, q_lens = A.ints([max(1, rows - 37 * e) for e in range(E)]), A.ints([max(0, min(T, T + 10 - 29 * e)) for e in range(E)])
    slopes = torch.tensor([2.0 ** (-4.0 * (h + 1) / H) for h in range(H)], device="cuda")
    kw = {"plain": {}, "all": {"causal": True, "cap": 15.0, "slopes": slopes, "prefix": A.ints([rows // 3] * E), "q_lens": q_lens},
          "positions": {"causal": True, "q_lens": q_lens, "q_start": A.ints([900 + e for e in range(E)]), "slopes": slopes * 0.01,
                        "k_pos": torch.stack([torch.randperm(2 * rows, device="cuda", generator=torch.Generator("cuda").manual_seed(e))[:rows] + 500 for e in range(E)]).to(i32)}}[kind]
    out, want = check_cached(Q, cache, lengths, D ** -0.5, **kw)
    assert (out[~want["rows"]] == 7).all()


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("D", [16, 48, 176])
def test_small_and_odd_head_dims_over_the_cache(T, D):
    cache = cache_of(randn(111, 2, 272, 2, D), randn(112, 2, 272, 2, D), 16)
    check_cached(randn(113, 2, T, 6, D), cache, A.ints([272, 131]), D ** -0.5, causal=True)


@pytest.mark.parametrize("T", [1, 40])
def test_broadcast_queries_and_caches(T):
    """One Q, and one K and V, for all episodes; heads that share theirs. Scales are whole, as the cache has them."""
    E, rows, H, HK, D = 3, 192, 8, 2, 64
    Q, one = randn(121, 1, T, H, D).expand(E, T, H, D), cache_of(randn(122, 1, rows, 1, D), randn(123, 1, rows, 1, D))
    shared = QuantizedCache(*(t.expand(E, rows, HK, D) for t in one[:2]), *(t.expand(E, rows // 64, HK).contiguous() for t in one[2:]))
    lengths = A.ints([192, 65, 1])
    want = A.attention(Q, A.widened(shared.K, shared.K_scale), A.widened(shared.V, shared.V_scale), 0.1, k_lens=lengths, causal=True)
    out = torch.zeros(E, T, H, D, dtype=bf16, device="cuda")
    op_table().cache_attention(Q, shared, lengths, 0.1, out, causal=True)
    A.check_out(out, want, D, P_8BIT)
    K, V = randn(124, E, rows, HK, D), randn(125, E, rows, HK, D)
    op_table().masked_attention(Q, K, V, 0.1, out, k_lens=lengths, causal=True)
    A.check_out(out, A.attention(Q, K, V, 0.1, k_lens=lengths, causal=True), D, 2.0 ** -8)


@pytest.mark.parametrize("T", [1, 24])
def test_many_episodes(T):
    """More episodes than SMs: a CTA has all keys of a tile."""
    E, rows, H, D = 700, 144, 8, 64
    cache = cache_of(randn(131, E, rows, 1, D), randn(132, E, rows, 1, D), 16)
    check_cached(randn(133, E, T, H, D), cache, A.ints([1 + (e * 7) % rows for e in range(E)]), 0.1, causal=True)


def test_evicted_rows_of_a_far_cache():
    """Rows 32 KB apart, byte offsets past 31 bits: K and V of the rows that stay, bit for bit."""
    rows, keep, D = 70016, 64, 64
    store = torch.zeros(2, rows, 1, 32768, dtype=torch.uint8, device="cuda").view(e4m3)
    cache = QuantizedCache(store[:1, :, :, :D], store[1:, :, :, -D:], *(torch.ones(1, rows // 64, 1, device="cuda") for _ in range(2)))
    size = torch.exp2(torch.arange(rows, device="cuda").div(64, rounding_mode="floor").remainder(5).float() - 2)[None, :, None, None]
    op_table().cache_append((randn(141, 1, rows, 1, D).float() * size).to(bf16), (randn(142, 1, rows, 1, D).float() * size).to(bf16), cache, A.ints([0]))
    first = rows - 200
    w = torch.zeros(1, rows, device="cuda")
    w[0, first:] = 1.0                                                          # ties: the first 64 of them stay
    small, n = allocate_quantized_cache(1, keep, 1, D, "cuda"), A.ints([0])
    op_table().cache_evict(cache, A.ints([rows]), w, keep, small, n)
    kept = torch.arange(first, first + keep, device="cuda")
    assert n.tolist() == [keep]
    for got, got_scale, held, scale in ((small.K, small.K_scale, cache.K, cache.K_scale), (small.V, small.V_scale, cache.V, cache.V_scale)):
        source = scale[0, kept // 64, 0]
        assert (source != source[0]).any() and got_scale[0, 0, 0] == source.max()
        moved = A.to_e4m3(held[0, first:first + keep, 0].float() * (source / source.max())[:, None])
        assert A.same_bits(got[0, :, 0].contiguous(), moved)

"""Masked attention and the 8-bit cache on the GPU against plain 64-bit forms."""
from __future__ import annotations

import itertools
import math

import pytest
import torch

import attention_cases as A
from flash_vla_b200 import op_table
from flash_vla_b200.hardware.nvidia.b200.pi0.backends.cuda import _lib, wrappers
from flash_vla_b200.hardware.nvidia.b200.pi0.buffers import QuantizedCache, allocate_quantized_cache
from flash_vla_b200.runtime.cuda import ScratchPool

pytestmark = pytest.mark.gpu
bf16, f32, i32, e4m3 = torch.bfloat16, torch.float32, torch.int32, torch.float8_e4m3fn
NAN, INF = math.nan, math.inf
P_BF16, P_FP16 = 2.0 ** -8, 2.0 ** -11      # half a step of the probabilities' type


@pytest.fixture(autouse=True)
def no_wait_has_run_out():
    """A kernel that gives up on a wait leaves a code in the device's health word."""
    yield
    torch.cuda.synchronize()
    assert _lib.load().fvla_device_status(None) == 0


def randn(seed, *shape, dtype=bf16):
    return torch.randn(shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(dtype)


def slopes_of(H):
    return torch.tensor([2.0 ** (-4.0 * (h + 1) / H) for h in range(H)], device="cuda")


def attend(Q, K, V, scale, out=None, **kw):
    """The op, with destinations that show what it leaves alone."""
    E, T, H, D = Q.shape
    out = torch.full((E, T, H, D), 7.0, dtype=bf16, device="cuda") if out is None else out
    lse = torch.full((E, H, T), 7.0, device="cuda")
    op_table().masked_attention(Q, K, V, scale, out, lse=lse, **kw)
    return out, lse


def check(Q, K, V, scale, p_step=P_BF16, **kw):
    out, lse = attend(Q, K, V, scale, **kw)
    want = A.attention(Q, K, V, scale, **kw)
    A.check_out(out, want, Q.shape[3], p_step)
    A.check_lse(lse, want, Q.shape[3])
    assert (out[~want["rows"]] == 7).all() and (lse.permute(0, 2, 1)[~want["rows"]] == 7).all()
    return out, want


SHAPES = [  # episodes, tokens, keys, heads, kv heads, dim
    (1, 1, 1, 1, 1, 64), (2, 1, 300, 8, 1, 256), (1, 5, 0, 4, 2, 64), (1, 128, 128, 1, 1, 128), (2, 129, 257, 6, 2, 128), (1, 33, 1000, 7, 1, 64),
    (2, 51, 819, 8, 1, 256), (1, 200, 200, 16, 16, 72), (1, 65, 127, 5, 5, 8), (1, 17, 383, 24, 1, 128), (1, 9, 140, 128, 1, 64), (3, 2, 2500, 4, 4, 200),
    (1, 300, 300, 8, 8, 248), (1, 1, 5000, 56, 8, 128)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", ["plain", "causal", "cap", "distance", "all"])
def test_masked_attention(shape, kind):
    E, T, S, H, HK, D = shape
    Q, K, V = randn(1, E, T, H, D), randn(2, E, S, HK, D), randn(3, E, S, HK, D)
    kw = {"plain": {}, "causal": {"causal": True}, "cap": {"cap": 5.0}, "distance": {"slopes": slopes_of(H)},
          "all": {"causal": True, "cap": 20.0, "slopes": slopes_of(H), "prefix": A.ints([S // 3] * E)}}[kind]
    check(Q, K, V, D ** -0.5, **kw)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D,H,HK", [(256, 8, 1), (128, 4, 4), (64, 14, 2)])
def test_lengths_of_every_kind(D, H, HK, causal):
    """Zero, one, all; a whole number of tiles, one row more; more queries than keys; lengths beyond the tensor, which are clamped."""
    k_lens, q_lens = [0, 1, 128, 129, 300, 77, 10, 400], [3, 1, 128, 0, 130, 140, 140, 60]
    Q, K, V = randn(4, 8, 140, H, D), randn(5, 8, 300, HK, D), randn(6, 8, 300, HK, D)
    for e, L in enumerate(k_lens):
        K[e, L:] = NAN
        V[e, L:] = INF if e % 2 else NAN
    for e, n in enumerate(q_lens):
        Q[e, n:] = NAN
    out, lse = attend(Q, K, V, D ** -0.5, causal=causal, k_lens=A.ints(k_lens), q_lens=A.ints(q_lens))
    want = A.attention(Q, K, V, D ** -0.5, causal=causal, k_lens=A.ints([min(L, 300) for L in k_lens]), q_lens=A.ints(q_lens))
    A.check_out(out, want, D, P_BF16)
    A.check_lse(lse, want, D)
    assert (out[~want["rows"]] == 7).all() and (lse.permute(0, 2, 1)[~want["rows"]] == 7).all()
    assert (out[0, :3] == 0).all() and (lse[0, :, :3] == -INF).all()      # no key at all


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D,H,HK", [(256, 8, 1), (64, 3, 3)])
def test_documents_in_any_order(D, H, HK, causal):
    """Ids packed, interleaved and missing; padding (negative ids) holds NaN and infinities."""
    T = S = 513
    for pattern in ("packed", "interleaved", "padded"):
        ids = torch.zeros(1, S, dtype=i32, device="cuda")
        j = torch.arange(S, device="cuda")
        if pattern == "packed":
            ids[0] = ((j > 0).int() + (j > 130).int() + (j > 131).int() + (j > 400).int())
        elif pattern == "interleaved":
            ids[0] = (j * 7 % 5).int()
        else:
            ids[0] = torch.where((j > 200) & (j < 460), -1, (j > 100).int())
        Q, K, V = randn(7, 1, T, H, D), randn(8, 1, S, HK, D), randn(9, 1, S, HK, D)
        K[:, ids[0] < 0], V[:, ids[0] < 0] = INF, NAN
        out, want = check(Q, K, V, D ** -0.5, causal=causal, q_docs=ids, k_docs=ids)
        assert (out[:, ids[0] < 0] == 0).all()
    for T in (1, 3):                                                        # few rows
        q_docs = ids[:, 460:460 + T].contiguous()
        check(randn(7, 1, T, H, D), K, V, D ** -0.5, q_docs=q_docs, k_docs=ids)
    other = torch.full_like(ids, 9)
    out, lse = attend(Q, K, V, 1.0, q_docs=other, k_docs=ids)            # a document that no key has
    assert (out == 0).all() and (lse == -INF).all()


def test_no_keys_and_documents():
    Q, K = randn(7, 2, 3, 4, 64), randn(8, 2, 0, 2, 64)
    ids = torch.zeros(2, 3, dtype=i32, device="cuda")
    out, lse = attend(Q, K, K, 0.1, q_docs=ids, k_docs=ids[:, :0].contiguous())
    assert (out == 0).all() and (lse == -INF).all()


def test_prefix_mask():
    E, T, S, H, D = 4, 200, 300, 8, 256
    Q, K, V = randn(10, E, T, H, D), randn(11, E, S, 1, D), randn(12, E, S, 1, D)
    check(Q, K, V, D ** -0.5, causal=True, prefix=A.ints([0, 1, 250, 999]), k_lens=A.ints([300, 128, 260, 200]), q_lens=A.ints([200, 100, 200, 150]))


def test_strides_and_broadcasts():
    """Heads before tokens, an interleaved K/V tensor, one K/V for all episodes, every second token, a destination between other data."""
    E, T, S, H, HK, D = 3, 70, 150, 4, 2, 64
    Q = randn(13, E, H, T, D).transpose(1, 2)
    KV = randn(14, E, S, 2, HK, D)
    check(Q, KV[:, :, 0], KV[:, :, 1], 0.1, causal=True)
    one = randn(15, 1, S, HK, D)
    check(Q, one.expand(E, S, HK, D), one.expand(E, S, HK, D), 0.1)
    check(randn(16, E, 2 * T, H, D)[:, ::2], KV[:, ::3, 0], KV[:, ::3, 1], 0.1, causal=True)
    shared = randn(17, E, S, 1, D).expand(E, S, HK, D)
    check(Q, shared, KV[:, :, 1], 0.1)
    wide = torch.full((E, T, H, 3 * D), 7.0, dtype=bf16, device="cuda")
    out, _ = attend(Q, KV[:, :, 0], KV[:, :, 1], 0.1, out=wide[..., D:2 * D])
    A.check_out(out, A.attention(Q, KV[:, :, 0], KV[:, :, 1], 0.1), D, P_BF16)
    assert (wide[..., :D] == 7).all() and (wide[..., 2 * D:] == 7).all()
    out = Q.clone()
    attend(out, KV[:, :, 0], KV[:, :, 1], 0.1, out=out)                     # the destination may be Q
    A.check_out(out, A.attention(Q, KV[:, :, 0], KV[:, :, 1], 0.1), D, P_BF16)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_large_and_growing_scores(D):
    """Scores whose maximum grows from block to block, very large ones, and ties."""
    T, S, H = 150, 700, 2
    Q, K, V = randn(18, 1, T, H, D), randn(19, 1, S, H, D), randn(20, 1, S, H, D)
    K = (K.float() * torch.linspace(0.1, 12.0, S, device="cuda")[None, :, None, None]).to(bf16)
    check(Q, K, V, D ** -0.5)
    check(Q, K, V, D ** -0.5, causal=True, cap=30.0)
    check(Q, K, V, -D ** -0.5, causal=True)
    check(Q, torch.zeros_like(K), V, 1.0)
    check(Q, K, V, 0.0)


@pytest.mark.parametrize("cap", [0.01, 1.0, 50.0, 1e4])
def test_caps(cap):
    Q, K, V = randn(21, 1, 130, 4, 128) * 3, randn(22, 1, 260, 2, 128) * 3, randn(23, 1, 260, 2, 128)
    check(Q, K, V, 0.5, cap=cap)


@pytest.mark.parametrize("H,HK,D", [(8, 4, 256), (4, 4, 128), (4, 2, 64)])
def test_long_walks(H, HK, D):
    """Thirty blocks and more to a tile, the last tile almost empty, with every score function; results repeat to the bit."""
    T = S = 4099
    Q, K, V = randn(63, 1, T, H, D), randn(64, 1, S, HK, D), randn(65, 1, S, HK, D)
    for kw in ({}, {"causal": True}, {"causal": True, "cap": 20.0}, {"causal": True, "slopes": slopes_of(H)}):
        outs = [attend(Q, K, V, D ** -0.5, **kw)[0] for _ in range(4)]
        assert all(torch.equal(o, outs[0]) for o in outs[1:])
        want = A.attention(Q, K, V, D ** -0.5, **kw)
        A.check_out(outs[0], want, D, P_BF16)


def test_a_row_of_nan_stays_in_its_row():
    Q, K, V = randn(24, 1, 130, 4, 64), randn(25, 1, 260, 2, 64), randn(26, 1, 260, 2, 64)
    want, _ = attend(Q, K, V, 0.1)
    Q[0, 5, 1] = NAN
    out, _ = attend(Q, K, V, 0.1)
    assert out[0, 5, 1].isnan().all()
    out[0, 5, 1] = want[0, 5, 1]
    assert torch.equal(out, want)


def test_long_keys_and_far_offsets():
    """One token over 70 001 keys of a cache whose rows lie far apart: element offsets pass 32 bits."""
    S, H, D = 70001, 8, 64
    store = torch.empty(S, 1, 64 * 512, dtype=bf16, device="cuda")         # 4.6 GB, 2.3e9 elements
    K, V = store[None, :, :, :D], store[None, :, :, -D:]
    K.copy_(randn(27, 1, S, 1, D))
    V.copy_(randn(28, 1, S, 1, D))
    Q = randn(29, 1, 1, H, D)
    check(Q, K, V, D ** -0.5)
    check(Q, K, V, D ** -0.5, k_lens=A.ints([69_900]), slopes=slopes_of(H) * 1e-3)


def test_repeats_are_bit_equal_and_streams_do_not_mix():
    E, T, S, H, HK, D = 2, 3, 4000, 8, 1, 256
    sets = [(randn(30 + i, E, T, H, D), randn(40 + i, E, S, HK, D), randn(50 + i, E, S, HK, D)) for i in range(3)]
    want = [attend(*s, 0.06)[0] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(5):
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(attend(*s, 0.06)[0])
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 3])


def test_captured_graphs_replayed_on_two_streams():
    """Two graphs, replayed at the same time: each has its scratch; inputs rewritten between replays are read anew."""
    E, T, S, H, HK, D = 1, 1, 6000, 8, 1, 256
    items = []
    for i in range(2):
        Q, K, V = randn(60 + i, E, T, H, D), randn(70 + i, E, S, HK, D), randn(80 + i, E, S, HK, D)
        out = torch.zeros_like(Q)
        lens = A.ints([S])
        g = torch.cuda.CUDAGraph()
        op_table().masked_attention(Q, K, V, 0.06, out, k_lens=lens)
        with torch.cuda.graph(g):
            op_table().masked_attention(Q, K, V, 0.06, out, k_lens=lens)
        items.append((g, Q, K, V, out, lens, torch.cuda.Stream()))
    for L in (S, 100, 4097):
        for g, Q, K, V, out, lens, _ in items:
            lens.fill_(L)
            out.zero_()
        torch.cuda.synchronize()
        for _ in range(20):
            for g, *_, st in items:
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for g, Q, K, V, out, lens, _ in items:
            A.check_out(out, A.attention(Q, K, V, 0.06, k_lens=lens), D, P_BF16)


def test_a_frozen_pool_serves_what_it_warmed_up():
    Q, K, V = randn(1, 1, 1, 8, 256), randn(2, 1, 6000, 1, 256), randn(3, 1, 6000, 1, 256)
    pool = ScratchPool()
    with wrappers.use_pool(pool):
        want, _ = attend(Q, K, V, 0.06)
        pool.freeze()
        held = len(pool)
        got, _ = attend(Q, K, V, 0.06)
        assert torch.equal(want, got) and len(pool) == held


# ------------------------------------------------------------------------------------------------ the 8-bit cache
def filled(seed, E, rows, HK, D, block=64, spread=1.0):
    """A cache of random rows whose blocks have unlike scales."""
    c = allocate_quantized_cache(E, rows, HK, D, "cuda", block)
    size = torch.exp2(torch.randint(-4, 5, (2, E, (c.K.shape[1] + 15) // 16, HK, 1), device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).float() * spread)
    size = size.repeat_interleave(16, 2)[:, :, :c.K.shape[1]]
    K, V = ((randn(seed + i, E, c.K.shape[1], HK, D).float() * size[i]).to(bf16) for i in (0, 1))
    op_table().cache_append(K, V, c, A.ints([0] * E))
    return c, K, V


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("HK,D", [(1, 256), (8, 128), (3, 64), (2, 16)])
def test_append_bit_for_bit(block, HK, D):
    E, rows = 4, 256
    cache = allocate_quantized_cache(E, rows, HK, D, "cuda", block)
    shadow = [t.cpu() for t in cache]
    gen = torch.Generator().manual_seed(5)
    lengths = [0, 0, 0, 0]
    for step, (T, grow) in enumerate([(1, 1.0), (37, 4.0), (1, 600.0), (130, 0.01), (5, 1e-30), (2, 1e30)]):
        K, V = randn(100 + step, E, T, HK, D, dtype=f32).mul(grow).to(bf16), randn(200 + step, E, T, HK, D, dtype=f32).mul(grow).to(bf16)
        counts = [T, T - 1, T // 2, max(0, T - 3)]
        if step == 1:
            K[0, 3, 0, :4] = torch.tensor([NAN, INF, -INF, 0.0], dtype=bf16)
            V[1, :, 0] = 0.0
        starts = A.ints(lengths)
        op_table().cache_append(K, V, cache, starts, A.ints(counts) if step else None)
        shadow = A.append(shadow, K, V, lengths, counts if step else None)
        lengths = [a + (b if step else T) for a, b in zip(lengths, counts)]
        for got, want in zip(cache[:2], shadow[:2]):
            got, want = got.cpu().float(), want.float()
            assert torch.equal(got.nan_to_num(1e9), want.nan_to_num(1e9)), step
        assert torch.equal(cache[2].cpu(), shadow[2]) and torch.equal(cache[3].cpu(), shadow[3]), step
    del gen


def test_append_outside_the_cache_is_left_out_and_reported():
    lib = _lib.load()
    cache = allocate_quantized_cache(3, 128, 1, 64, "cuda", 64)
    K = randn(1, 3, 20, 1, 64)
    assert lib.fvla_device_status(None) == 0
    op_table().cache_append(K, K, cache, A.ints([-5, 120, 1 << 30]))
    torch.cuda.synchronize()
    assert lib.fvla_device_status(None) == 8 and lib.fvla_device_status(None) == 0
    want = A.append([torch.zeros(3, 128, 1, 64, dtype=e4m3), torch.zeros(3, 128, 1, 64, dtype=e4m3), torch.ones(3, 2, 1), torch.ones(3, 2, 1)], K, K, [-5, 120, 1 << 30])
    for got, ref in zip(cache[:2], want[:2]):
        assert A.same_bits(got, ref)
    assert (cache.K[2].float() == 0).all() and (cache.K_scale[2] == 1).all()
    cache2 = allocate_quantized_cache(1, 128, 1, 64, "cuda", 64)
    op_table().cache_append(K[:1], K[:1], cache2, A.ints([128]), A.ints([0]))      # nothing, at the very end
    assert lib.fvla_device_status(None) == 0


def test_append_through_strides():
    """K/V rows as slices of one projection, the cache as a layer of a stack."""
    E, T, HK, D = 2, 70, 2, 64
    qkv = randn(3, E, T, 3, HK, D)
    stack = allocate_quantized_cache(E, 2 * 192, HK, D, "cuda", 64)
    held = [t.view(E, 2, 192, HK, D)[:, 1] for t in stack[:2]]
    scales = [torch.ones(E, 3, HK, device="cuda") for _ in range(2)]
    cache = QuantizedCache(*held, *scales)
    op_table().cache_append(qkv[:, :, 1], qkv[:, :, 2], cache, A.ints([5, 100]))
    want = A.append([torch.zeros(E, 192, HK, D, dtype=e4m3), torch.zeros(E, 192, HK, D, dtype=e4m3), torch.ones(E, 3, HK), torch.ones(E, 3, HK)], qkv[:, :, 1],
                    qkv[:, :, 2], [5, 100])
    for got, ref in zip(cache[:2], want[:2]):
        assert A.same_bits(got.contiguous(), ref)
    assert torch.equal(cache.K_scale.cpu(), want[2]) and (stack.K.view(E, 2, 192, HK, D)[:, 0].float() == 0).all()


CACHED = [  # episodes, tokens, rows, heads, kv heads, dim, block
    (2, 1, 64, 8, 1, 256, 64), (1, 1, 16, 1, 1, 64, 16), (3, 1, 1024, 32, 8, 128, 32), (2, 51, 832, 8, 1, 256, 64), (1, 7, 4096, 14, 2, 64, 128), (2, 3, 640, 4, 4, 80, 16),
    (1, 40, 384, 20, 4, 240, 128), (1, 1, 20480, 8, 1, 256, 128)]


@pytest.mark.parametrize("shape", CACHED)
@pytest.mark.parametrize("kind", ["plain", "causal", "all"])
def test_cache_attention(shape, kind):
    E, T, rows, H, HK, D, block = shape
    cache, _, _ = filled(7, E, rows, HK, D, block, 0.3)
    lengths = A.ints([max(T, rows - 13 * e - (rows // 3) * (e % 2)) for e in range(E)])
    for e, L in enumerate(lengths.tolist()):                                 # behind the last row: NaN
        cache.K.view(torch.uint8)[e, L:] = 0x7f
        cache.V.view(torch.uint8)[e, L:] = 0xff
    Q = randn(8, E, T, H, D)
    kw = {"plain": {}, "causal": {"causal": True}, "all": {"causal": True, "cap": 15.0, "slopes": slopes_of(H), "prefix": A.ints([rows // 4] * E)}}[kind]
    before = randn(9, E, cache.K.shape[1], dtype=f32).abs()
    K, V = A.widened(cache.K, cache.K_scale), A.widened(cache.V, cache.V_scale)
    want = A.attention(Q, K, V, D ** -0.5, k_lens=lengths, **kw)
    for decay in (0.0, 1.0, 0.5):
        out, lse, weights = torch.full_like(Q, 7.0), torch.full((E, H, T), 7.0, device="cuda"), before.clone()
        op_table().cache_attention(Q, cache, lengths, D ** -0.5, out, lse=lse, weights=weights, decay=decay, **kw)
        A.check_out(out, want, D, P_FP16)
        A.check_lse(lse, want, D)
        A.check_weights(weights, want, D, lengths, before, decay)
    bare = torch.full_like(Q, 7.0)
    op_table().cache_attention(Q, cache, lengths, D ** -0.5, bare, **kw)
    assert torch.equal(bare, out)
    held = torch.full_like(weights, NAN)
    op_table().cache_attention(Q, cache, lengths, D ** -0.5, bare, weights=held, decay=0.0, **kw)      # overwritten, without a log-sum-exp of the caller's
    A.check_weights(held.nan_to_num(0.0), want, D, torch.clamp(lengths, max=held.shape[1]), torch.zeros_like(held), 0.0)


def test_cache_attention_with_uneven_scales():
    """Blocks whose scales lie 2^40 apart: the probabilities of small values and the values of large ones both count."""
    cache, _, _ = filled(17, 2, 512, 2, 128, 16, 5.0)
    cache.K_scale.fill_(2.0 ** -7)
    Q, lengths = randn(18, 2, 9, 8, 128), A.ints([512, 300])
    out = torch.zeros_like(Q)
    op_table().cache_attention(Q, cache, lengths, 0.02, out)
    A.check_out(out, A.attention(Q, A.widened(cache.K, cache.K_scale), A.widened(cache.V, cache.V_scale), 0.02, k_lens=lengths), 128, P_FP16)
    for size in (1e-30, 1e30):                                                # queries beyond fp16's range
        big, small = (Q.float() * size).to(bf16), 0.02 / size
        op_table().cache_attention(big, cache, lengths, small, out)
        A.check_out(out, A.attention(big, A.widened(cache.K, cache.K_scale), A.widened(cache.V, cache.V_scale), small, k_lens=lengths), 128, P_FP16)


@pytest.mark.parametrize("T", [1, 30])
def test_cache_attention_with_scales_of_any_size(T):
    """Scales that a program brings need not be powers of two."""
    cache, _, _ = filled(19, 2, 512, 2, 128, 32, 0.3)
    for scale in cache[2:]:
        scale.mul_(torch.rand(scale.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(5)) + 0.7)
    Q, lengths = randn(20, 2, T, 8, 128), A.ints([512, 300])
    out, w = torch.zeros_like(Q), torch.zeros(2, 512, device="cuda")
    op_table().cache_attention(Q, cache, lengths, 0.08, out, weights=w, decay=0.0)
    want = A.attention(Q, A.widened(cache.K, cache.K_scale), A.widened(cache.V, cache.V_scale), 0.08, k_lens=lengths)
    A.check_out(out, want, 128, P_FP16)
    A.check_weights(w, want, 128, lengths, torch.zeros_like(w), 0.0)


def test_cache_rows_far_apart():
    """Rows 32 KB apart, 2.3 GB of them: byte offsets pass 31 bits in all four operators."""
    rows, HK, D, keep = 70016, 1, 64, 64
    store = torch.zeros(2, rows, 1, 32768, dtype=torch.uint8, device="cuda").view(e4m3)
    scales = [torch.ones(1, rows // 64, HK, device="cuda") for _ in range(2)]
    cache = QuantizedCache(store[:1, :, :, :D], store[1:, :, :, -D:], *scales)
    K, V = randn(58, 1, rows, HK, D), randn(59, 1, rows, HK, D)
    op_table().cache_append(K, V, cache, A.ints([0]))
    dense = allocate_quantized_cache(1, rows, HK, D, "cuda")
    op_table().cache_append(K, V, dense, A.ints([0]))
    for a, b in zip(cache, dense):
        assert A.same_bits(a.contiguous(), b)
    for T in (1, 40):
        Q = randn(60, 1, T, 2, D)
        outs = [torch.zeros_like(Q) for _ in range(2)]
        for c, o in zip((cache, dense), outs):
            op_table().cache_attention(Q, c, A.ints([rows - 5]), 0.1, o)
        assert torch.equal(*outs)
    w = torch.zeros(1, rows, device="cuda")
    w[0, rows - 200:] = 1.0
    small = allocate_quantized_cache(1, keep, HK, D, "cuda")
    op_table().cache_evict(cache, A.ints([rows]), w, keep, small, A.ints([0]))
    assert A.same_bits(small.K, cache.K[:, rows - 200:rows - 200 + keep].contiguous()) or not torch.equal(small.K_scale, cache.K_scale[:, :1])
    assert torch.equal(A.widened(small.V, small.V_scale), A.widened(cache.V.contiguous(), cache.V_scale)[:, rows - 200:rows - 200 + keep])


@pytest.mark.parametrize("T", [5, 20])
@pytest.mark.parametrize("positions", ["evicted", "shuffled"])
def test_cache_attention_with_positions(positions, T):
    E, rows, H, HK, D = 2, 384, 8, 2, 64
    cache, _, _ = filled(27, E, rows, HK, D)
    gen = torch.Generator("cuda").manual_seed(3)
    k_pos = torch.stack([torch.randperm(2000, device="cuda", generator=gen)[:rows] for _ in range(E)]).to(i32)
    if positions == "evicted":
        k_pos = k_pos.sort(1)[0]
    Q, lengths, start = randn(28, E, T, H, D), A.ints([384, 200]), A.ints([1990, 900])
    kw = {"causal": True, "prefix": A.ints([100, 950]), "q_start": start, "k_pos": k_pos.contiguous(), "slopes": slopes_of(H) * 0.01}
    out, w = torch.zeros_like(Q), torch.zeros(E, rows, device="cuda")
    op_table().cache_attention(Q, cache, lengths, 0.1, out, weights=w, decay=0.0, **kw)
    want = A.attention(Q, A.widened(cache.K, cache.K_scale), A.widened(cache.V, cache.V_scale), 0.1, k_lens=lengths, **kw)
    A.check_out(out, want, D, P_FP16)
    A.check_weights(w, want, D, lengths, torch.zeros_like(w), 0.0)


def test_cache_lengths_of_zero_and_queries_of_none():
    cache, _, _ = filled(37, 3, 128, 1, 64)
    Q, w = randn(38, 3, 4, 8, 64), torch.full((3, 128), 2.0, device="cuda")
    out = torch.full_like(Q, 7.0)
    op_table().cache_attention(Q, cache, A.ints([0, -4, 128]), 0.1, out, q_lens=A.ints([4, 4, 0]), weights=w, decay=0.5)
    assert (out[:2] == 0).all() and (out[2] == 7).all()
    assert (w[:2] == 2).all() and (w[2] == 1).all()


# ------------------------------------------------------------------------------------------------ eviction
EVICT = [  # rows, keep, lengths, sinks, recent, block, out block, weights
    (256, 64, [256, 200, 64, 0], 4, 16, 64, 64, "random"), (1024, 300, [1024, 301, 300, 299], 0, 0, 16, 128, "ties"), (384, 1, [384, 1, 2, 50], 0, 1, 128, 16, "random"),
    (512, 512, [512, 600, -3, 7], 10, 10, 32, 32, "zeros"), (2048, 777, [2048, 1500, 1025, 1024], 3, 700, 64, 64, "odd"), (4096, 128, [4096, 129, 4095, 2000], 64, 64, 64, 64, "random"),
    (33024, 1000, [33024, 32769, 20000, 1001], 1, 2, 128, 128, "ties")]


@pytest.mark.parametrize("case", EVICT)
@pytest.mark.parametrize("HK,D", [(1, 256), (3, 64)])
def test_evict_bit_for_bit(case, HK, D):
    rows, keep, lengths, sinks, recent, block, out_block, kind = case
    E = len(lengths)
    cache, _, _ = filled(47, E, rows, HK, D, block)
    w = randn(48, E, rows, dtype=f32)
    if kind == "ties":
        w = (w * 2).round()
        w[w == 0] = -0.0
        w[:, ::3] = w[:, ::3].abs()
    elif kind == "zeros":
        w = torch.zeros_like(w)
    elif kind == "odd":
        w[:, ::5], w[:, 1::7], w[:, 2::9] = NAN, INF, -INF
    out_rows = (keep + out_block - 1) // out_block * out_block + out_block
    out = allocate_quantized_cache(E, out_rows, HK, D, "cuda", out_block)
    out_lengths = torch.full((E,), -1, dtype=i32, device="cuda")
    out_w, out_pos = torch.full((E, out_rows), 5.0, device="cuda"), torch.full((E, out_rows), -5, dtype=i32, device="cuda")
    positions = torch.arange(rows, dtype=i32, device="cuda").mul(3).repeat(E, 1)
    op_table().cache_evict(cache, A.ints(lengths), w, keep, out, out_lengths, out_w, positions, out_pos, sinks=sinks, recent=recent)
    kept = A.evict(cache, torch.tensor(lengths), w.cpu(), keep, sinks, recent)
    assert out_lengths.tolist() == [len(k) for k in kept]
    for e, k in enumerate(kept):
        n = len(k)
        assert out_pos[e, :n].tolist() == [3 * j for j in k], e
        assert torch.equal(out_w[e, :n].nan_to_num(9.0), w[e, k].nan_to_num(9.0)) and (out_w[e, n:] == 5).all() and (out_pos[e, n:] == -5).all()
        for got, got_scale, held, scale in ((out.K, out.K_scale, cache.K, cache.K_scale), (out.V, out.V_scale, cache.V, cache.V_scale)):
            idx = torch.tensor(k, device="cuda", dtype=torch.long)
            source = scale[e, idx // block]                                                        # (n, HK)
            now = torch.ones(out_rows // out_block, HK, device="cuda")
            for b in range((n + out_block - 1) // out_block):
                now[b] = source[b * out_block:(b + 1) * out_block].amax(0)
            assert torch.equal(got_scale[e], now)
            moved = A.to_e4m3(held[e].view(torch.uint8)[idx].view(e4m3).float() * (source / now.repeat_interleave(out_block, 0)[:n])[..., None])
            assert A.same_bits(got[e, :n].contiguous(), moved)
            assert (got[e, n:].float() == 0).all()


def test_evict_refuses_its_own_memory():
    cache, _, _ = filled(57, 1, 128, 1, 64)
    w, n = torch.zeros(1, 128, device="cuda"), A.ints([128])
    with pytest.raises(ValueError, match="lies over"):
        op_table().cache_evict(cache, n, w, 64, cache, A.ints([0]))
    with pytest.raises(ValueError, match="lies over"):
        op_table().cache_evict(cache, n, w, 64, allocate_quantized_cache(1, 128, 1, 64, "cuda"), n)


def test_a_captured_step_of_all_of_them():
    """Append, attention with weights and eviction in one graph: replays on rewritten inputs give what the calls themselves give."""
    E, rows, H, HK, D, keep = 2, 256, 8, 2, 128, 64
    ops = op_table()

    def state(seed):
        cache, _, _ = filled(seed, E, rows, HK, D)
        return {"cache": cache, "q": randn(seed, E, 2, H, D), "k": randn(seed + 1, E, 2, HK, D), "v": randn(seed + 2, E, 2, HK, D), "n": A.ints([200, 111]),
                "out": torch.zeros(E, 2, H, D, dtype=bf16, device="cuda"), "w": torch.rand(E, rows, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)),
                "small": allocate_quantized_cache(E, keep, HK, D, "cuda"), "m": A.ints([0, 0]), "pos": torch.zeros(E, keep, dtype=i32, device="cuda")}

    def step(s):
        ops.cache_append(s["k"], s["v"], s["cache"], s["n"])
        ops.cache_attention(s["q"], s["cache"], s["n"] + 2, 0.08, s["out"], causal=True, weights=s["w"], decay=0.5)
        ops.cache_evict(s["cache"], s["n"] + 2, s["w"], keep, s["small"], s["m"], out_positions=s["pos"], sinks=1, recent=4)

    held = state(200)
    step(held)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(held)
    for seed in (300, 400):
        fresh, same = state(seed), state(seed)
        for name in ("q", "k", "v", "n", "w", "out", "m", "pos"):
            held[name].copy_(same[name])
        for name in ("cache", "small"):
            for a, b in zip(held[name], same[name]):
                a.view(torch.uint8).copy_(b.view(torch.uint8))
        g.replay()
        step(fresh)
        for name in ("out", "w", "m", "pos"):
            assert torch.equal(held[name], fresh[name]), name
        for a, b in zip((*held["cache"], *held["small"]), (*fresh["cache"], *fresh["small"])):
            assert A.same_bits(a, b)


def test_a_server_uses_them_together():
    """Prefill of a ragged batch through the masked attention, its K/V into the cache, decoding steps that weigh the rows, an eviction, and decoding on
    the thinned cache with the rows' positions. Every attention is held to the 64-bit form on what the cache holds then; and the whole is captured."""
    E, S, H, HK, D, keep = 3, 300, 8, 2, 128, 96
    ops, lens = op_table(), A.ints([300, 170, 64])
    Q, K, V = randn(71, E, S, H, D), randn(72, E, S, HK, D), randn(73, E, S, HK, D)
    kw = {"cap": 30.0, "slopes": slopes_of(H) * 0.05}
    check(Q, K, V, D ** -0.5, causal=True, prefix=A.ints([128, 128, 64]), q_lens=lens, k_lens=lens, **kw)
    cache, small = allocate_quantized_cache(E, 384, HK, D, "cuda"), allocate_quantized_cache(E, keep + 32, HK, D, "cuda")
    ops.cache_append(K, V, cache, A.ints([0] * E), lens)
    weights, mass = torch.zeros(E, 384, device="cuda"), torch.zeros(E, 384, dtype=torch.float64, device="cuda")
    now, step = lens.clone(), torch.ones(E, dtype=i32, device="cuda")
    for i in range(4):
        q, k, v = randn(80 + i, E, 1, H, D), randn(90 + i, E, 1, HK, D), randn(95 + i, E, 1, HK, D)
        ops.cache_append(k, v, cache, now)
        now = now + step
        out = torch.zeros_like(q)
        ops.cache_attention(q, cache, now, D ** -0.5, out, causal=True, weights=weights, **kw)
        want = A.attention(q, A.widened(cache.K, cache.K_scale), A.widened(cache.V, cache.V_scale), D ** -0.5, causal=True, k_lens=now, **kw)
        A.check_out(out, want, D, P_FP16)
        mass += want["weights"]
    assert ((weights.double() - mass).abs() <= 1e-4 * mass + 1e-12).all()
    n, pos = torch.zeros(E, dtype=i32, device="cuda"), torch.zeros(E, small.K.shape[1], dtype=i32, device="cuda")
    left = torch.zeros(E, small.K.shape[1], device="cuda")
    ops.cache_evict(cache, now, weights, keep, small, n, left, out_positions=pos, sinks=2, recent=8)
    assert n.tolist() == [min(keep, L) for L in now.tolist()]
    q, k, v = randn(103, E, 1, H, D), randn(104, E, 1, HK, D), randn(105, E, 1, HK, D)
    ops.cache_append(k, v, small, n)
    pos.scatter_(1, n.long()[:, None], now[:, None])
    out = torch.zeros_like(q)
    call = lambda: ops.cache_attention(q, small, n + step, D ** -0.5, out, causal=True, q_start=now, k_pos=pos, **kw)      # noqa: E731
    call()
    want = A.attention(q, A.widened(small.K, small.K_scale), A.widened(small.V, small.V_scale), D ** -0.5, causal=True, k_lens=n + step, q_start=now, k_pos=pos, **kw)
    A.check_out(out, want, D, P_FP16)
    eager = out.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    out.zero_()
    g.replay()
    assert torch.equal(out, eager)

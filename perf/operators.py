"""Attention with masks, caps and biases, and the 8-bit KV cache beside it, as cases that can be timed and compared.

  attention  `masked_attention`: scores capped by a tanh or biased by distance, causal / prefix / document masks, lengths
             per episode, over bf16 keys and values. Prompts padded to different lengths, packed documents, single tokens.
  append     `cache_append`: new K / V rows into a cache of e4m3 values with one power-of-two scale for each block of rows
             and K/V head.
  cached     `cache_attention`: the same attention over that cache, and the attention weight that each key received.
  evict      `cache_evict`: the rows with the largest accumulated weight move, in order, to another cache.

A case is a dict of plain values. `run` is one pass: the plain form in elementary torch operations, or (where `own` is set)
the calls that a user makes. Lengths and document borders follow from the case, all other values from the seed.
"""
from __future__ import annotations

import math

import torch

own = False

bf16, f32, f64, i32, e4m3 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.float8_e4m3fn
E4M3_MAX = 448.0


def _attention(name, episodes, tokens, keys, heads, kv_heads, dim, causal=True, prefix=0, docs=0, cap=0.0, distance=False, ragged=False):
    case = {"kind": "attention", "episodes": episodes, "tokens": tokens, "keys": keys, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "causal": causal, "prefix": prefix, "docs": docs, "cap": cap, "distance": distance, "ragged": ragged}
    return dict(case, name=name) if name else case


def _cached(name, episodes, tokens, keys, heads, kv_heads, dim, block=64, causal=True, prefix=0, cap=0.0, distance=False, ragged=True, weights=False):
    case = {"kind": "cached", "episodes": episodes, "tokens": tokens, "keys": keys, "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block,
            "causal": causal, "prefix": prefix, "docs": 0, "cap": cap, "distance": distance, "ragged": ragged, "weights": weights}
    return dict(case, name=name) if name else case


def _append(name, episodes, tokens, rows, kv_heads, dim, block=64):
    case = {"kind": "append", "episodes": episodes, "tokens": tokens, "rows": rows, "kv_heads": kv_heads, "dim": dim, "block": block}
    return dict(case, name=name) if name else case


def _evict(name, episodes, rows, keep, kv_heads, dim, block=64, sinks=4, recent=64):
    case = {"kind": "evict", "episodes": episodes, "rows": rows, "keep": keep, "kv_heads": kv_heads, "dim": dim, "block": block, "sinks": sinks,
            "recent": recent}
    return dict(case, name=name) if name else case


def listed():
    return [
        # the smallest call: one new token of each of two episodes over a bf16 prefix cache of a three-camera prompt
        _attention("attention_token", 2, 1, 817, 8, 1, 256, ragged=True),
        # prefix encoder of four episodes whose prompts differ in length: images and prompt see each other, the tail is causal
        _attention("attention_prefix", 4, 1024, 1024, 8, 1, 256, prefix=768, ragged=True),
        # eight texts packed end to end into one odd sequence, scores capped, two query heads to a K/V head
        _attention("attention_documents", 1, 4099, 4099, 8, 4, 256, docs=8, cap=50.0),
        # a long causal text whose scores fall with distance, a K/V head for every query head
        _attention("attention_distance", 2, 4096, 4096, 16, 16, 128, distance=True),
        # one step of a server that decodes 32 episodes: one row each, inside a block
        _append("append_token", 32, 1, 2048, 8, 128),
        # the prefix rows of eight episodes of four cameras and a prompt, written in one go
        _append("append_prefix", 8, 1073, 2048, 8, 256, block=128),
        # single-token decoding of four episodes over short prefix caches
        _cached("cached_token", 4, 1, 1024, 8, 1, 256),
        # the action chunk of eight episodes over their prefix rows and itself, and what weight each row got
        _cached("cached_chunk", 8, 51, 832, 8, 1, 256, causal=False, weights=True),
        # a server's decoding step: 32 episodes of up to 16 K rows, grouped heads, capped scores
        _cached("cached_server", 32, 1, 16384, 32, 8, 128, cap=30.0),
        # one episode with a very long history, weights for the eviction
        _cached("cached_long", 1, 1, 131072, 8, 1, 256, block=128, ragged=False, weights=True),
        # one layer's cache of four episodes, halved
        _evict("evict_prefix", 4, 1024, 512, 1, 256),
        # long histories of eight episodes cut to a quarter
        _evict("evict_long", 8, 16384, 4096, 8, 128, recent=256),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["attention"] * 3 + ["cached"] * 3 + ["append", "evict"])
    kv_heads = rng.choice((1, 1, 2, 4, 8))
    if kind == "append":
        block = rng.choice((16, 32, 64, 128))
        rows = block * max(1, 4096 // block)
        tokens = rng.choice((1, _log_int(rng, 2, 2000)))
        return _append(None, _log_int(rng, 1, 8 if tokens > 1 else 64), tokens, rows, kv_heads, rng.choice((64, 128, 256)), block)
    if kind == "evict":
        rows = 128 * _log_int(rng, 4, 128)
        keep = rows // rng.choice((2, 4)) - rng.randint(0, 63)
        return _evict(None, _log_int(rng, 1, 8), rows, keep, kv_heads, rng.choice((64, 128)), rng.choice((16, 32, 64, 128)), rng.choice((0, 4)),
                      rng.choice((0, 32, 60)))
    group = rng.choice((1, 4, 8, 8, 7))
    cap = rng.choice((0.0, 0.0, 30.0))
    distance = rng.random() < 0.3
    if kind == "cached":
        dim = rng.choice((64, 128, 256))
        tokens = rng.choice((1, 1, _log_int(rng, 2, 64)))
        keys = 128 * _log_int(rng, 1, 256 if tokens == 1 else 32)
        episodes = _log_int(rng, 1, max(1, min(32, (1 << 18) // (keys * kv_heads))))
        return _cached(None, episodes, tokens, keys, kv_heads * group, kv_heads, dim, rng.choice((16, 32, 64, 128)), rng.random() < 0.6, 0, cap, distance, True,
                       rng.random() < 0.4)
    dim = rng.choice((64, 72, 128, 256))
    keys = _log_int(rng, 64, 2048)
    tokens = rng.choice((1, keys, keys, keys, max(1, keys // 3)))
    if kv_heads * group * dim * keys * tokens > 1 << 33:      # no dearer than the listed ones
        kv_heads = 1
    episodes = rng.randint(1, 4)
    if tokens == keys and rng.random() < 0.4:
        return _attention(None, 1, tokens, keys, kv_heads * group, kv_heads, dim, rng.random() < 0.7, 0, rng.randint(2, 9), cap, distance)
    prefix = rng.choice((0, keys // 2))
    return _attention(None, episodes, tokens, keys, kv_heads * group, kv_heads, dim, prefix > 0 or rng.random() < 0.7, prefix, 0, cap, distance, rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """(query tokens, keys) of every episode."""
    n, T, S = case["episodes"], case["tokens"], case["keys"]
    if not case["ragged"]:
        return [T] * n, [S] * n
    keys = [max(1, S - (e * S) // (2 * n) - (e * 5) % 3) for e in range(n)]
    return [min(T, k) for k in keys], keys


def _documents(case):
    """First row of every document, and the row behind the last one: texts of unlike lengths, a padded tail."""
    S, d = case["keys"], case["docs"]
    shares = [1.0 + (3 * i) % 4 for i in range(d)]
    ends, total = [0], 0.0
    for s in shares:
        total += s
        ends.append(int((S - S // 50) * total / sum(shares)))
    return ends


def _randn(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen)


def _values(gen, episodes, rows, kv_heads, dim):
    """K and V rows: channels of K have offsets of their own."""
    k = _randn(gen, episodes, rows, kv_heads, dim) + _randn(gen, 1, 1, kv_heads, dim)
    return k, _randn(gen, episodes, rows, kv_heads, dim) * 0.5 + 0.1


def _ints(values):
    return torch.tensor(values, dtype=i32, device="cuda")


def _power_of_two(amax):
    """The smallest power of two s with amax / s <= 448, at least 2^-120; amax is an fp32 tensor."""
    mantissa, exponent = torch.frexp(amax)                      # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = exponent - 9 + (mantissa > 0.875).to(exponent.dtype)    # 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e, torch.full_like(e, -120)).clamp(min=-120)
    return torch.ldexp(torch.ones_like(amax), e)


def _quantized(gen, episodes, rows, kv_heads, dim, block):
    """A cache with rows in it: (K, V, K_scale, V_scale)."""
    held, scales = [], []
    for x in _values(gen, episodes, rows, kv_heads, dim):
        b = x.view(episodes, rows // block, block, kv_heads, dim)
        s = _power_of_two(b.abs().amax((2, 4)))
        held.append((b / s[:, :, None, :, None]).to(e4m3).view(episodes, rows, kv_heads, dim))
        scales.append(s)
    return held + scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, n, HK, D = case["kind"], case["episodes"], case["kv_heads"], case["dim"]
    s = {"case": case, "kind": kind}
    if kind in ("attention", "cached"):
        T, S, H = case["tokens"], case["keys"], case["heads"]
        q_lens, k_lens = _lengths(case)
        s |= {"Q": _randn(gen, n, T, H, D).to(bf16), "scale": D ** -0.5, "causal": case["causal"], "cap": case["cap"],
              "q_lens": _ints(q_lens) if case["ragged"] else None, "k_lens": _ints(k_lens) if case["ragged"] or kind == "cached" else None,
              "prefix": _ints([case["prefix"]] * n) if case["prefix"] else None, "docs": None,
              "slopes": torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device="cuda") if case["distance"] else None,
              "out": torch.zeros(n, T, H, D, dtype=bf16, device="cuda"),
              "lse": torch.zeros(n, H, T, device="cuda")}
        if kind == "attention":
            s["K"], s["V"] = (x.to(bf16) for x in _values(gen, n, S, HK, D))
            if case["docs"]:
                ids = torch.full((n, S), -1, dtype=i32)
                ends = _documents(case)
                for d in range(case["docs"]):
                    ids[:, ends[d]:ends[d + 1]] = d
                s["docs"] = ids.cuda()
        else:
            s["cache"] = _quantized(gen, n, S, HK, D, case["block"])
            s["weights"] = torch.zeros(n, S, device="cuda") if case["weights"] else None
    elif kind == "append":
        rows, T, block = case["rows"], case["tokens"], case["block"]
        s["cache"] = _quantized(gen, n, rows, HK, D, block)
        s["K"], s["V"] = (x.to(bf16) for x in _values(gen, n, T, HK, D))
        s["starts"] = torch.randint(0, rows - T + 1, (n,), device="cuda", generator=gen).to(i32)
    else:
        rows, keep, block = case["rows"], case["keep"], case["block"]
        out_rows = (keep + block - 1) // block * block
        s["cache"] = _quantized(gen, n, rows, HK, D, block)
        s["lengths"] = _ints([rows - (e * rows) // (3 * n) - e % 2 for e in range(n)])
        s["weights"] = torch.rand(n, rows, device="cuda", generator=gen).pow(4)
        s["weights"] = torch.where(s["weights"] < 0.01, torch.zeros_like(s["weights"]), s["weights"])      # keys that no query looked at
        s["out_cache"] = [torch.zeros(n, out_rows, HK, D, device="cuda").to(e4m3) for _ in range(2)] + \
                         [torch.ones(n, out_rows // block, HK, device="cuda") for _ in range(2)]
        s["out_lengths"] = torch.zeros(n, dtype=i32, device="cuda")
        s["out_weights"] = torch.zeros(n, out_rows, device="cuda")
        s["out_positions"] = torch.zeros(n, out_rows, dtype=i32, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------ the plain form
def _visible(s, T, S):
    """(n, T, S) truth values: which keys a query sees; and the positions of queries (n, T) and keys (S)."""
    n = s["Q"].shape[0]
    whole = lambda v, most: torch.full((n,), most, dtype=i32, device="cuda") if v is None else v  # noqa: E731
    q_lens, k_lens = whole(s["q_lens"], T), whole(s["k_lens"], S)
    t, j = torch.arange(T, device="cuda", dtype=i32), torch.arange(S, device="cuda", dtype=i32)
    pos = k_lens[:, None] - q_lens[:, None] + t
    see = ((j < k_lens[:, None])[:, None, :] & (t < q_lens[:, None])[:, :, None])
    if s["causal"]:
        most = pos if s["prefix"] is None else torch.maximum(pos, s["prefix"][:, None] - 1)
        see = see & (j <= most[:, :, None])
    if s["docs"] is not None:
        see = see & (s["docs"][:, :, None] == s["docs"][:, None, :]) & (s["docs"] >= 0)[:, None, :]
    return see, pos, j


def _plain_attention(s, K, V):
    """K, V (n, S, kv heads, dim) in 32 bits. -> out (n, T, heads, dim) and lse (n, heads, T), both in 32 bits, and the probabilities."""
    Q = s["Q"].float()
    n, T, H, D = Q.shape
    S, HK = K.shape[1], K.shape[2]
    q = Q.view(n, T, HK, H // HK, D).permute(0, 2, 3, 1, 4).reshape(n, HK, -1, D)
    x = torch.matmul(q, K.permute(0, 2, 3, 1)).view(n, H, T, S) * s["scale"]
    if s["cap"] > 0:
        x = torch.tanh(x / s["cap"]) * s["cap"]
    see, pos, j = _visible(s, T, S)
    if s["slopes"] is not None:
        x = x - s["slopes"][None, :, None, None] * (pos[:, :, None] - j).abs().float()[:, None]
    x = x.masked_fill(~see[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = x.sum(-1, keepdim=True)
    lse = torch.where(total > 0, top + torch.log(total), top)[..., 0]
    x = x / torch.where(total > 0, total, torch.ones_like(total))
    out = torch.matmul(x.view(n, HK, -1, S), V.permute(0, 2, 1, 3))
    out = out.view(n, HK, H // HK, T, D).permute(0, 3, 1, 2, 4).reshape(n, T, H, D)
    if s["q_lens"] is not None:      # rows behind an episode's last query stay as they were: zero
        lse = torch.where((torch.arange(T, device="cuda") < s["q_lens"][:, None])[:, None], lse, torch.zeros_like(lse))
    return out, lse, x


def _widened(held, scale):
    n, rows, HK, D = held.shape
    return (held.float().view(n, scale.shape[1], -1, HK, D) * scale[:, :, None, :, None]).view(n, rows, HK, D)


def _plain_append(s):
    """The blocks that get rows: old rows under the new scale, new rows behind them."""
    block, T, n = s["case"]["block"], s["case"]["tokens"], s["case"]["episodes"]
    starts = s["starts"].long()
    blocks = s["cache"][2].shape[1]
    wide = min((T + block - 2) // block + 1, blocks)                # blocks that T rows can touch
    first = torch.clamp(starts // block, max=blocks - wide)
    at = first[:, None] + torch.arange(wide, device="cuda")          # (n, wide)
    row = (at[:, :, None] * block + torch.arange(block, device="cuda"))
    new = (row >= starts[:, None, None]) & (row < starts[:, None, None] + T)
    token = (row - starts[:, None, None]).clamp(0, T - 1)
    old = (row < starts[:, None, None])
    e = torch.arange(n, device="cuda")[:, None]
    outs = []
    for held, scale, x in zip(s["cache"][:2], s["cache"][2:], (s["K"], s["V"])):
        x = x.float()[e[:, :, None], token]                          # (n, wide, block, kv heads, dim)
        fine = new[..., None, None] & torch.isfinite(x)
        s_new = _power_of_two(torch.where(fine, x.abs(), torch.zeros_like(x)).amax((2, 4)))
        s_old = scale[e, at]
        s_all = torch.where(old.any(2)[..., None], torch.maximum(s_old, s_new), s_new)
        s_all = torch.where(new.any(2)[..., None], s_all, s_old)
        wide_scale, wide_old = s_all[:, :, None, :, None], s_old[:, :, None, :, None]
        h = held.view(n, blocks, block, *held.shape[2:])
        before = h.view(torch.uint8)[e, at].view(e4m3)
        moved = torch.where(new[..., None, None], x / wide_scale, before.float() * (wide_old / wide_scale)).to(e4m3)
        keeps = ~(new | old)[..., None, None]                        # rows behind the new ones stay as they were
        h.view(torch.uint8)[e, at] = torch.where(keeps, before.view(torch.uint8), moved.view(torch.uint8))
        scale[e, at] = s_all
        outs += [held, scale]
    return {"K": outs[0], "K_scale": outs[1], "V": outs[2], "V_scale": outs[3]}


def _kept_rows(s):
    """(n, keep) source rows in order, and (n, keep) which of them exist."""
    case, L = s["case"], s["lengths"].long()
    rows, keep = case["rows"], case["keep"]
    j = torch.arange(rows, device="cuda")
    inside = j < L[:, None]
    forced = inside & ((j < case["sinks"]) | (j >= L[:, None] - case["recent"]))
    w = torch.where(torch.isnan(s["weights"]), torch.full_like(s["weights"], -math.inf), s["weights"])
    order = torch.sort(w, dim=1, descending=True, stable=True)[1]
    rank = forced.long() * 2 + inside.long()                         # always kept, others, rows behind the last
    order = order.gather(1, torch.sort(rank.gather(1, order), dim=1, descending=True, stable=True)[1])
    count = torch.clamp(L, max=keep)
    picked = torch.zeros(case["episodes"], rows, dtype=torch.bool, device="cuda")
    picked.scatter_(1, order[:, :keep], torch.arange(keep, device="cuda") < count[:, None])
    source = torch.sort(torch.where(picked, j, rows), dim=1)[0][:, :keep]
    return source.clamp(max=rows - 1), torch.arange(keep, device="cuda") < count[:, None], count


def _plain_evict(s):
    case = s["case"]
    n, keep, block = case["episodes"], case["keep"], case["block"]
    source, there, count = _kept_rows(s)
    e = torch.arange(n, device="cuda")[:, None]
    out = {}
    pad = s["out_weights"].shape[1] - keep
    padded = lambda v: torch.nn.functional.pad(v, (0,) * (2 * (v.ndim - 2)) + (0, pad))  # noqa: E731
    for name, held, scale, to, to_scale in zip("KV", s["cache"][:2], s["cache"][2:], s["out_cache"][:2], s["out_cache"][2:]):
        s_row = torch.where(there[..., None], scale[e, source // block], torch.zeros((), device="cuda"))
        blocks = padded(s_row).view(n, -1, block, scale.shape[2])
        s_new = blocks.amax(2)
        used = padded(there).view(n, -1, block).any(2)[..., None]
        to_scale.copy_(torch.where(used, s_new, to_scale))
        ratio = blocks / torch.where(used, s_new, torch.ones_like(s_new))[:, :, None]
        values = (held.view(torch.uint8)[e, source].view(e4m3).float() * ratio.view(n, -1, scale.shape[2])[:, :keep, :, None]).to(e4m3)
        to.view(torch.uint8)[:, :keep] = torch.where(there[..., None, None], values.view(torch.uint8), to.view(torch.uint8)[:, :keep])
        out[name], out[name + "_scale"] = to, to_scale
    s["out_lengths"].copy_(count)
    s["out_weights"][:, :keep] = torch.where(there, s["weights"].gather(1, source), s["out_weights"][:, :keep])
    s["out_positions"][:, :keep] = torch.where(there, source.to(i32), s["out_positions"][:, :keep])
    return dict(out, lengths=s["out_lengths"], weights=s["out_weights"], positions=s["out_positions"])


def _plain(s):
    if s["kind"] == "attention":
        out, lse, _ = _plain_attention(s, s["K"].float(), s["V"].float())
        return {"out": out.to(bf16), "lse": lse}
    if s["kind"] == "cached":
        held = s["cache"]
        out, lse, p = _plain_attention(s, _widened(held[0], held[2]), _widened(held[1], held[3]))
        return {"out": out.to(bf16), "lse": lse, "weights": p.sum((1, 2)) if s["weights"] is not None else None}
    return _plain_append(s) if s["kind"] == "append" else _plain_evict(s)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    ops = s.get("ops")
    if ops is None:                      # a program imports the package and builds its table once
        from flash_vla_b200 import op_table
        from flash_vla_b200.hardware.nvidia.b200.pi0.buffers import QuantizedCache
        ops = s["ops"] = op_table()
        for name in ("cache", "out_cache"):
            if name in s:
                s[name] = QuantizedCache(*s[name])
    if s["kind"] == "attention":
        ops.masked_attention(s["Q"], s["K"], s["V"], s["scale"], s["out"], causal=s["causal"], prefix=s["prefix"], q_lens=s["q_lens"], k_lens=s["k_lens"],
                             q_docs=s["docs"], k_docs=s["docs"], cap=s["cap"], slopes=s["slopes"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    if s["kind"] == "cached":
        ops.cache_attention(s["Q"], s["cache"], s["k_lens"], s["scale"], s["out"], causal=s["causal"], prefix=s["prefix"], q_lens=s["q_lens"], cap=s["cap"],
                            slopes=s["slopes"], lse=s["lse"], weights=s["weights"], decay=0.0)
        return {"out": s["out"], "lse": s["lse"], "weights": s["weights"]}
    if s["kind"] == "append":
        ops.cache_append(s["K"], s["V"], s["cache"], s["starts"])
        c = s["cache"]
        return {"K": c.K, "K_scale": c.K_scale, "V": c.V, "V_scale": c.V_scale}
    case = s["case"]
    ops.cache_evict(s["cache"], s["lengths"], s["weights"], case["keep"], s["out_cache"], s["out_lengths"], out_weights=s["out_weights"],
                    out_positions=s["out_positions"], sinks=case["sinks"], recent=case["recent"])
    c = s["out_cache"]
    return {"K": c.K, "K_scale": c.K_scale, "V": c.V, "V_scale": c.V_scale, "lengths": s["out_lengths"], "weights": s["out_weights"],
            "positions": s["out_positions"]}


def run(s):
    return _own(s) if own else _plain(s)


# ------------------------------------------------------------------------------------------------ what a pass has to do
def _pairs(case):
    """(visible query-key pairs of a head, query rows, key rows that some query may see), over all episodes."""
    q_lens, k_lens = _lengths(case)
    if case["docs"]:
        ends, pairs = _documents(case), 0
        for a, b in zip(ends, ends[1:]):
            pairs += (b - a) * (b - a + 1) // 2 if case["causal"] else (b - a) ** 2
        return pairs, case["tokens"], ends[-1]
    pairs = 0
    for n, L in zip(q_lens, k_lens):
        if not case["causal"]:
            pairs += n * L
        else:
            p = case["prefix"]
            pairs += sum(min(L, max(L - n + t + 1, p)) for t in range(n))
    return pairs, sum(q_lens), sum(k_lens)


def work(case):
    n, HK, D = case["episodes"], case["kv_heads"], case["dim"]
    if case["kind"] in ("attention", "cached"):
        pairs, queries, keys = _pairs(case)
        H = case["heads"]
        row = 2 * HK * D * (2 if case["kind"] == "attention" else 1)
        moved = 4 * queries * H * D + 4 * queries * H + keys * row
        if case["kind"] == "cached":
            moved += 8 * keys * HK / case["block"] + (4 * keys if case["weights"] else 0)
        return {"bytes": float(moved), "flops": 4.0 * D * H * pairs}
    if case["kind"] == "append":
        values = 2 * n * case["tokens"] * HK * D
        return {"bytes": float(3 * values + 8 * n * HK * (case["tokens"] / case["block"] + 1)), "flops": 2.0 * values}
    lengths = [case["rows"] - (e * case["rows"]) // (3 * n) - e % 2 for e in range(n)]
    kept = sum(min(L, case["keep"]) for L in lengths)
    return {"bytes": float(4 * sum(lengths) + kept * (4 * HK * D + 8) + 16 * kept * HK / case["block"]), "flops": float(2 * kept * HK * D)}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_attention(s, K, V):
    """One query head of one episode at a time."""
    case = s["case"]
    n, T, H, D = s["Q"].shape
    S, HK = K.shape[1], K.shape[2]
    q_lens, k_lens = _lengths(case)
    out = torch.zeros(n, T, H, D, dtype=f64, device="cuda")
    lse = torch.zeros(n, H, T, dtype=f64, device="cuda")
    weights = torch.zeros(n, S, dtype=f64, device="cuda")
    for e in range(n):
        m, L = q_lens[e], k_lens[e]
        gap = (torch.arange(m, device="cuda", dtype=f64)[:, None] + (L - m)) - torch.arange(L, device="cuda", dtype=f64)[None, :]
        hidden = torch.zeros(m, L, dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden = gap < 0
            hidden[:, :case["prefix"]] = False
        if case["docs"]:
            ids = s["docs"][e]
            hidden = hidden | (ids[:m, None] != ids[None, :L]) | (ids[None, :L] < 0)
        nothing = hidden.all(1)
        for h in range(H):
            x = (s["Q"][e, :m, h].to(f64) @ K[e, :L, h // (H // HK)].T) * s["scale"]
            if case["cap"] > 0:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if s["slopes"] is not None:
                x = x - s["slopes"][h].to(f64) * gap.abs()
            x = x.masked_fill(hidden, -math.inf)
            z = torch.logsumexp(x, 1)
            lse[e, h, :m] = z
            p = torch.exp(x - torch.where(nothing, torch.zeros_like(z), z)[:, None])
            out[e, :m, h] = p @ V[e, :L, h // (H // HK)]
            weights[e, :L] += p.sum(0)
    return out, lse, weights


def _exact_append(s):
    case, found = s["case"], {}
    block = case["block"]
    for name, held, scale, x in zip("KV", s["cache"][:2], s["cache"][2:], (s["K"], s["V"])):
        values, scales = held.to(f64), scale.to(f64)
        for e, start in enumerate(s["starts"].tolist()):
            stop = start + case["tokens"]
            for b in range(start // block, (stop - 1) // block + 1):
                low, high = max(start, b * block), min(stop, (b + 1) * block)
                rows = x[e, low - start:high - start].to(f64)
                most = rows.abs().amax((0, 2))
                need = torch.ldexp(torch.ones_like(most), torch.log2(most / E4M3_MAX).clamp(min=-119.0).sub(0.5).floor().to(i32))      # at most two doublings short
                for _ in range(2):
                    need = torch.where(need * E4M3_MAX < most, 2 * need, need)
                was = scales[e, b].clone()
                now = torch.maximum(was, need) if low > b * block else need
                values[e, b * block:low] *= (was / now)[None, :, None]
                values[e, low:high] = rows / now[None, :, None]
                scales[e, b] = now
        found[name], found[name + "_scale"] = values, scales
    return found


def _exact_evict(s):
    case, found = s["case"], {}
    n, keep, block = case["episodes"], case["keep"], case["block"]
    out_rows = s["out_weights"].shape[1]
    lengths = s["lengths"].tolist()
    picked = []
    for e, L in enumerate(lengths):
        if L <= keep:
            picked.append(list(range(L)))
            continue
        w = s["weights"][e, :L].tolist()
        always = set(range(min(case["sinks"], L))) | set(range(max(0, L - case["recent"]), L))
        rest = sorted((j for j in range(L) if j not in always), key=lambda j: (-w[j], j))
        picked.append(sorted(list(always) + rest[:keep - len(always)]))
    weights = torch.zeros(n, out_rows, dtype=f64, device="cuda")
    for e, rows in enumerate(picked):
        weights[e, :len(rows)] = s["weights"][e, rows].to(f64)
    for name, held, scale in zip("KV", s["cache"][:2], s["cache"][2:]):
        values = torch.zeros(n, out_rows, *held.shape[2:], dtype=f64, device="cuda")
        scales = torch.ones(n, out_rows // block, scale.shape[2], dtype=f64, device="cuda")
        for e, rows in enumerate(picked):
            r = torch.tensor(rows, device="cuda")
            of_row = scale[e].to(f64)[r // block]
            real = held.view(torch.uint8)[e][r].view(e4m3).to(f64) * of_row[..., None]
            for b in range((len(rows) + block - 1) // block):
                part = slice(b * block, min((b + 1) * block, len(rows)))
                scales[e, b] = of_row[part].amax(0)
                values[e, part] = real[part] / scales[e, b][None, :, None]
        found[name], found[name + "_scale"] = values, scales
    return dict(found, lengths=None, weights=weights, positions=None)


def exact(case, seed):
    if case["kind"] in ("attention", "cached") and _pairs(case)[0] * case["heads"] * case["dim"] > 6e10:
        return None
    s = prepare(case, seed)
    if case["kind"] == "attention":
        out, lse, _ = _exact_attention(s, s["K"].to(f64), s["V"].to(f64))
        return {"out": out, "lse": lse}
    if case["kind"] == "cached":
        K, V = (h.to(f64) * sc.to(f64).repeat_interleave(case["block"], 1)[..., None] for h, sc in zip(s["cache"][:2], s["cache"][2:]))
        out, lse, weights = _exact_attention(s, K, V)
        return {"out": out, "lse": lse, "weights": weights if case["weights"] else None}
    return _exact_append(s) if case["kind"] == "append" else _exact_evict(s)

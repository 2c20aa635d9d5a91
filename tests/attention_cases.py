"""Plain 64-bit forms of masked attention and of the 8-bit cache, and the error that the kernels' roundings allow."""
from __future__ import annotations

import math

import torch

f64, bf16, e4m3, i32 = torch.float64, torch.bfloat16, torch.float8_e4m3fn, torch.int32


def ints(values, device="cuda"):
    return torch.tensor(values, dtype=i32, device=device)


def attention(Q, K, V, scale, causal=False, prefix=None, q_lens=None, k_lens=None, q_start=None, q_docs=None, k_docs=None, k_pos=None, cap=0.0,
              slopes=None):
    """-> dict of out, lse, p (E, H, T, S), the sums of p |v| and the largest sum of scale |q k| of a row; hidden keys have no part, whatever they hold."""
    E, T, H, D = Q.shape
    S, HK = K.shape[1], K.shape[2]
    dev = Q.device
    n = torch.full((E,), T, device=dev) if q_lens is None else q_lens.long()
    L = torch.full((E,), S, device=dev) if k_lens is None else k_lens.long()
    start = L - n if q_start is None else q_start.long()
    pos = start[:, None] + torch.arange(T, device=dev)                                       # (E, T)
    kp = torch.arange(S, device=dev).expand(E, S) if k_pos is None else k_pos.long()
    see = (torch.arange(S, device=dev) < L[:, None])[:, None, :].expand(E, T, S)
    if causal:
        limit = pos if prefix is None else torch.maximum(pos, prefix.long()[:, None] - 1)
        see = see & (kp[:, None, :] <= limit[:, :, None])
    if q_docs is not None:
        see = see & (q_docs[:, :, None] == k_docs[:, None, :]) & (k_docs >= 0)[:, None, :]
    rep = lambda x: x.double().permute(0, 2, 1, 3).repeat_interleave(H // HK, 1)             # noqa: E731  (E, H, S, D)
    k, v = rep(K), rep(V)
    seen = see.any(1)[:, None, :, None]
    k, v = torch.where(seen, k, 0.0), torch.where(seen, v, 0.0)                               # what nobody sees may hold anything
    q = Q.double().permute(0, 2, 1, 3)
    x = q @ k.mT * scale
    size = (q.abs() @ k.abs().mT * abs(scale)).masked_fill(~see[:, None], 0.0).amax(-1) if S else x.new_zeros(E, H, T)
    if cap:
        x = cap * torch.tanh(x / cap)
    bias = 0.0
    if slopes is not None:
        far = (pos[:, :, None] - kp[:, None, :]).abs().masked_fill(~see, 0).amax(-1) if S else pos * 0       # (E, T)
        bias = slopes.double().abs()[None, :, None] * far[:, None, :]
        x = x - slopes.double()[None, :, None, None] * (pos[:, :, None] - kp[:, None, :]).abs()[:, None]
    x = x.masked_fill(~see[:, None], -math.inf)
    lse = torch.logsumexp(x, -1) if S else x.new_full((E, H, T), -math.inf)
    p = torch.where(see[:, None], torch.exp(x - torch.where(lse == -math.inf, 0.0, lse)[..., None]), 0.0)
    p = p * (torch.arange(T, device=dev) < n[:, None])[:, None, :, None]
    back = lambda y: y.permute(0, 2, 1, 3)                                                    # noqa: E731
    return {"out": back(p @ v), "lse": lse, "p": p, "spread": back(p @ v.abs()), "size": size, "bias": bias, "rows": torch.arange(T, device=dev) < n[:, None],
            "weights": p.sum((1, 2))}


def score_error(want, D):
    """Bound on a score's error in 32 bits: D products and sums of half a step each (2^-24), cap and exponential on top (2^-19), and of the bias four half
    steps: the slope in units of log2, its product with the distance, that product's sum with the score, and the maximum's subtraction."""
    return want["size"] * D * 2.0 ** -24 + 2.0 ** -19 + want["bias"] * 2.0 ** -22


def check_out(got, want, D, p_step):
    """|error| <= half a bf16 step of the result (2^-8), half a step of the probabilities (2^-8 where the products are in bf16, 2^-11 in fp16) and the
    scores' error times the sum of p |v|: a probability is off by e^(2 error) - 1, its own score's and that of the sum."""
    rows = want["rows"]
    err = (got.double() - want["out"]).abs()
    slack = 2 * score_error(want, D).permute(0, 2, 1)[..., None]
    bound = 2.0 ** -8 * want["out"].abs() + (p_step + slack) * want["spread"] * (1 + 2.0 ** -8) + 1e-30
    bad = (err > bound) & rows[..., None, None]
    bad = bad | (~torch.isfinite(got) & torch.isfinite(want["out"]) & rows[..., None, None])
    assert not bad.any(), (int(bad.sum()), float((err / bound)[rows].max()), bad.nonzero()[:3].tolist())


def check_lse(got, want, D):
    rows = want["rows"][:, None, :].expand_as(want["lse"])
    empty = want["lse"] == -math.inf
    assert torch.equal((got == -math.inf)[rows], empty[rows])
    fine = rows & ~empty
    assert ((got.double() - want["lse"]).abs() <= score_error(want, D) + want["lse"].abs() * 2.0 ** -23)[fine].all()


def check_weights(got, want, D, k_lens, before, decay):
    """A probability's relative error is that of two scores (its own and the log-sum-exp's); sums of positive numbers keep it, plus their roundings."""
    slack = 2 * score_error(want, D)[..., None] + 2.0 ** -18
    bound = (want["p"] * slack).sum((1, 2)) + (before.double() * decay).abs() * 2.0 ** -22 + 1e-30
    full = before.double() * decay + want["weights"]
    inside = torch.arange(got.shape[1], device=got.device) < k_lens[:, None]
    assert ((got.double() - full).abs() <= bound)[inside].all()
    assert torch.equal(got[~inside], before[~inside])


# ------------------------------------------------------------------------------------------------ the 8-bit cache
def needed_scale(x):
    """Smallest power of two s >= 2^-120 with |finite values| <= 448 s."""
    x = x.double()
    most = float(torch.where(torch.isfinite(x), x.abs(), 0.0).max()) if x.numel() else 0.0
    s = 2.0 ** -120
    while 448.0 * s < most:
        s *= 2
    return s


def to_e4m3(x):
    """Round to nearest even; beyond the largest finite value (which only an infinity is), NaN."""
    return x.float().to(e4m3)


def append(cache, K, V, starts, counts=None):
    """The cache after `cache_append`, on the CPU: block by block, head by head. -> list of the four tensors."""
    K_held, V_held, K_scale, V_scale = (t.cpu().clone() for t in cache)
    block = K_held.shape[1] // K_scale.shape[1]
    for held, scale, x in ((K_held, K_scale, K.cpu()), (V_held, V_scale, V.cpu())):
        E, T, HK, _ = x.shape
        for e in range(E):
            start = int(starts[e])
            count = T if counts is None else max(0, min(T, int(counts[e])))
            low, high = max(start, 0), min(start + count, held.shape[1])
            for b in range(low // block, (high + block - 1) // block if high > low else 0):
                first, last = max(low, b * block), min(high, (b + 1) * block)
                for h in range(HK):
                    new = x[e, first - start:last - start, h].float()
                    s = needed_scale(new)
                    if first > b * block:
                        was = float(scale[e, b, h])
                        s = max(s, was)
                        if s != was:
                            held[e, b * block:first, h] = to_e4m3(held[e, b * block:first, h].float() * (was / s))
                    held[e, first:last, h] = to_e4m3(new / s)
                    scale[e, b, h] = s
    return [K_held, V_held, K_scale, V_scale]


def evict(cache, lengths, weights, keep, sinks=0, recent=0):
    """Rows that stay, per episode."""
    kept = []
    for e, L in enumerate(lengths.tolist()):
        L = max(0, min(L, weights.shape[1]))
        if L <= keep:
            kept.append(list(range(L)))
            continue
        always = sorted(set(range(min(sinks, L))) | set(range(max(0, L - recent), L)))
        w = [-math.inf if math.isnan(x) else x for x in weights[e].tolist()]
        rest = sorted((j for j in range(L) if j not in set(always)), key=lambda j: (-w[j], j))
        kept.append(sorted(always + rest[:keep - len(always)]))
    return kept


def same_bits(a, b):
    return torch.equal(a.cpu().view(torch.uint8), b.cpu().view(torch.uint8))


def widened(held, scale):
    """The values that an 8-bit cache stands for, in 64 bits."""
    return held.double() * scale.double().repeat_interleave(held.shape[1] // scale.shape[1], 1)[..., None]

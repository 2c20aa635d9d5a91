"""Attention with masks, caps and biases, and the 8-bit KV cache: call sites without a counterpart in the reference.

The reference's attentions (`kernels/attention.py:20-34`, `fused_wrappers.py:88-115`) have one shape and one mask each. These take batches of
episodes of different lengths, grouped heads and the masks and score functions of other language backbones, and read the cache
either in bf16 or as e4m3 values with a power-of-two scale for each block of rows and K/V head (`QuantizedCache`). A server's step is
`cache_append`, then `cache_attention`; `cache_attention(..., weights=w)` adds up what weight each key received, by which
`cache_evict` later picks the rows that stay.

Conventions of `wrappers.py`: torch tensors in, destinations passed in and written in place, checks on the host, one call into
libfvla_b200 on torch's current stream. Tensors are (episodes, tokens, heads, head_dim) with a contiguous last axis and otherwise any strides that
start every row on 16 bytes; lengths, starts, positions and document ids are int32 on the device, contiguous. They are not read on the host: lengths
outside a tensor are clamped on the device. Scratch comes from the active `ScratchPool` of a program that installed one (`use_pool`, `set_pool`),
whose captured graph then owns it; without one it is allocated for the call, from a graph's own memory during a capture.
"""
from __future__ import annotations

import ctypes
import functools
import operator
import struct

import torch

from . import _lib
from . import wrappers as _w

BLOCKS = (16, 32, 64, 128)      # rows per scale of an 8-bit cache
_INT32, _F32 = torch.int32, torch.float32


def _rows(name, shape, stride, dtype, want, multiple, shared=()):
    """Element strides (episode, token, head) of a 4-D operand; an axis of one element gets a stride that any layout may have. `shared`: axes whose
    elements may share their memory (stride 0); where there is none the operand is written, and no two of its rows may overlap."""
    if dtype != want:
        raise ValueError(f"{name}: expected {want}, got {dtype}")
    if len(shape) != 4:
        raise ValueError(f"{name}: expected (episodes, tokens, heads, head_dim), got shape {tuple(shape)}")
    if shape[3] > 1 and stride[3] != 1:
        raise ValueError(f"{name}: the head dimension must be contiguous, got strides {tuple(stride)}")
    out = []
    for axis, (size, s) in enumerate(zip(shape[:3], stride[:3])):
        if size <= 1:
            s = 256
        if s % multiple:
            raise ValueError(f"{name}: rows must start on 16 bytes, got strides {tuple(stride)}")
        if s == 0 and axis not in shared:
            raise ValueError(f"{name}: rows that share memory, strides {tuple(stride)}")
        out.append(s)
    reach = shape[3]
    for s, n in () if shared else sorted((s, n) for s, n in zip(stride[:3], shape[:3]) if n > 1):
        if s < reach:
            raise ValueError(f"{name}: rows that share memory, shape {tuple(shape)}, strides {tuple(stride)}")
        reach += s * (n - 1)
    return out


def _cache_shapes(name, shapes, strides, dtypes):
    """Block size of a QuantizedCache whose four tensors have these shapes, strides and types."""
    k, v, ks, vs = shapes
    if tuple(k) != tuple(v) or tuple(ks) != tuple(vs):
        raise ValueError(f"{name}: K and V must have one shape, got {tuple(k)} {tuple(v)}, scales {tuple(ks)} {tuple(vs)}")
    if len(k) != 4 or len(ks) != 3 or ks[0] != k[0] or ks[2] != k[2]:
        raise ValueError(f"{name}: expected K (episodes, rows, kv_heads, head_dim) and scales (episodes, blocks, kv_heads), got {tuple(k)} and {tuple(ks)}")
    if ks[1] == 0 or k[1] % ks[1] or k[1] // ks[1] not in BLOCKS:
        raise ValueError(f"{name}: {k[1]} rows in {ks[1]} blocks (blocks of {BLOCKS} rows)")
    for t, dt in zip(("K_scale", "V_scale"), dtypes[2:]):
        if dt != _F32:
            raise ValueError(f"{name}.{t}: expected {_F32}, got {dt}")
    for t, s in zip(("K_scale", "V_scale"), strides[2:]):
        if any(n > 1 and a != b for n, a, b in zip(ks, s, (ks[1] * ks[2], ks[2], 1))):
            raise ValueError(f"{name}.{t}: expected a contiguous tensor, got strides {tuple(s)}")
    if k[3] % 16 or not 0 < k[3] <= 256:
        raise ValueError(f"{name}: head_dim {k[3]} (a multiple of 16 up to 256)")
    return k[1] // ks[1]


def _footprint(shape, stride, size):
    """(bytes from an operand's first to behind its last, bytes of a row, (elements, bytes apart) of the axes before the last)"""
    if 0 in shape:
        return 0, 0, ()
    axes = tuple((n, s * size) for n, s in zip(shape[:-1], stride[:-1]) if n > 1 and s)
    return sum((n - 1) * s for n, s in axes) + shape[-1] * size, shape[-1] * size, axes


def _apart(p, a, q, b):
    """Whether operands of the footprints a and b at p and q share no byte. Ones that interleave (K and V of one tensor, layers of a stack) do so with some
    axis' stride as their period: each then has a part of it of its own."""
    if p + a[0] <= q or q + b[0] <= p:
        return True
    for period in {s for f in (a, b) for _, s in f[2]}:
        inner_a, inner_b = (f[1] + sum((n - 1) * s for n, s in f[2] if s % period) for f in (a, b))
        ahead = (q - p) % period
        if inner_a <= ahead and ahead + inner_b <= period:
            return True
    return False


def _layout(t):
    return t.shape, t.stride(), t.dtype


def _cache_layout(c):
    K, V, K_scale, V_scale = c
    return ((K.shape, V.shape, K_scale.shape, V_scale.shape), (K.stride(), V.stride(), K_scale.stride(), V_scale.stride()),
            (K.dtype, V.dtype, K_scale.dtype, V_scale.dtype))


# The argument blocks of the C entries (`_lib.Attention` and so on) are put together as bytes, addresses first, then what a layout determines and a plan
# remembers: setting some forty ctypes fields costs more than the launch.
_ATTENTION_HEAD, _FLOATS, _CAUSAL = struct.Struct("17PQ"), struct.Struct("3f"), struct.Struct("ii")
_APPEND_HEAD, _EVICT_HEAD = struct.Struct("8P"), struct.Struct("15PQ")


def _between(block, first, last):
    """The bytes of a ctypes structure from field `first` up to field `last` (the end, where there is none)."""
    end = getattr(type(block), last).offset if last else ctypes.sizeof(block)
    return bytes(block)[getattr(type(block), first).offset:end]


@functools.lru_cache(maxsize=1024)
def _attention_plan(q, k, v, out, cache):
    """What operands of these layouts determine of an attention's argument block: (strides, dimensions, scratch bytes without and with documents or
    weights, episodes, tokens, keys, heads, footprints of Q, K, V and out, whether out in Q's place has its rows). `cache`: layout of a QuantizedCache, or None."""
    a = _lib.Attention()
    if cache is None:
        multiple, want, dim_multiple = 8, torch.bfloat16, 8
    else:
        a.block = _cache_shapes("cache", *cache)
        multiple, want, dim_multiple = 16, torch.float8_e4m3fn, 16
        k, v = ((cache[0][i], cache[1][i], cache[2][i]) for i in (0, 1))
    a.q_stride[:] = _rows("Q", *q, torch.bfloat16, 8, shared=(0,))
    a.k_stride[:] = _rows("K", *k, want, multiple, shared=(0, 2))
    a.v_stride[:] = _rows("V", *v, want, multiple, shared=(0, 2))
    a.out_stride[:] = _rows("out", *out, torch.bfloat16, 8)
    (E, T, H, D), (_, S, HK, _) = q[0], k[0]
    if tuple(k[0]) != (E, S, HK, D) or tuple(v[0]) != (E, S, HK, D) or tuple(out[0]) != (E, T, H, D):
        raise ValueError(f"attention: shapes do not fit: Q {tuple(q[0])}, K {tuple(k[0])}, V {tuple(v[0])}, out {tuple(out[0])}")
    if D % dim_multiple or not 0 < D <= 256:
        raise ValueError(f"attention: head_dim {D} (a multiple of {dim_multiple} up to 256)")
    if HK == 0 or H % HK or not 0 < H // HK <= 128:
        raise ValueError(f"attention: {H} query heads over {HK} K/V heads")
    if E * T * H >= 1 << 31 or E * HK >= 1 << 16 or S >= 1 << 31 or E >= 1 << 16:
        raise ValueError(f"attention: {E} episodes of {T} queries of {H} heads over {S} keys: too many")
    a.episodes, a.tokens, a.keys, a.heads, a.kv_heads, a.head_dim = E, T, S, H, HK, D
    nbytes = [0, 0]
    for i, extra in enumerate(((), ("q_docs", "k_docs") if cache is None else ("weights", "lse"))):
        b = type(a).from_buffer_copy(a)
        for name in ("q", "out", "k", "v", *(("k_scale", "v_scale") if cache is not None else ()), *extra):
            setattr(b, name, 16)                # an address that only says that there is a tensor
        if E and T:
            nbytes[i] = _lib.load().fvla_attention_workspace_bytes(ctypes.byref(b))
    held = 2 if cache is None else 1
    footprints = _footprint(q[0], q[1], 2), _footprint(k[0], k[1], held), _footprint(v[0], v[1], held), _footprint(out[0], out[1], 2)
    same = all(n <= 1 or s == o for n, s, o in zip(q[0], q[1], out[1]))
    return _between(a, "q_stride", "scale"), _between(a, "episodes", "causal"), nbytes, E, T, S, H, footprints, same


def _vector(name, t, shape, dtype, device):
    """Address of a small operand. (Without a GPU the large operands, which come last, are the ones refused for their device.)"""
    if t.dtype is dtype and t.shape == shape and t.is_contiguous() and (t.get_device() == device or device < 0):
        return t.data_ptr()
    if t.dtype != dtype:
        raise ValueError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous tensor, got strides {t.stride()}")
    raise ValueError(f"{name}: expected a tensor on the current CUDA device, got {t.device}")


def _misplaced(device, **operands):
    """Says which of four operands, whose layouts have been checked, is not on this device or not aligned."""
    for name, t in operands.items():
        name = name.replace("cache_", "cache.")
        if t.get_device() != device:
            raise ValueError(f"{name}: expected a CUDA tensor on the current device, got {t.device}")
        if t.data_ptr() & 15:
            raise ValueError(f"{name}: expected 16-byte alignment")


def _address(name, t, device):
    """Address of an operand whose layout has been checked."""
    p = t.data_ptr()
    if p & 15 or t.get_device() != device:
        _misplaced(device, **{name: t})
    return p


def _device():
    try:
        return torch._C._cuda_getDevice()
    except Exception:
        return -2                               # no GPU (-1 is the number of the CPU)


def _scratch(role, nbytes, device):
    if _w.default_pool():
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    return _w.scratch(role, (nbytes,), torch.uint8, device)


def _attend(Q, K, V, cache, scale, out, causal, prefix, q_lens, k_lens, q_start, q_docs, k_docs, k_pos, cap, slopes, lse, weights, decay):
    if cache is None:
        K_scale = V_scale = None
        plan = _attention_plan(_layout(Q), _layout(K), _layout(V), _layout(out), None)
    else:
        K, V, K_scale, V_scale = cache
        plan = _attention_plan(_layout(Q), None, None, _layout(out), _cache_layout(cache))
    strides, dims, nbytes, E, T, S, H, (fq, fk, fv, fo), same = plan
    scale, cap, decay = float(scale), float(cap or 0.0), float(decay)
    if not (abs(scale) < 2e38 and abs(decay) < 3.4e38 and (cap == 0.0 or (1.2e-38 < cap < 2e38 and abs(scale) < 3.4e38 * cap))):
        raise ValueError(f"attention: scale {scale}, cap {cap}, decay {decay}: finite numbers within fp32, scale over cap as well, the cap not negative")
    if prefix is not None and not causal:
        raise ValueError("attention: a prefix without the causal mask")
    if (q_docs is None) != (k_docs is None):
        raise ValueError("attention: documents of queries and keys, or of neither")
    q, k, v, o = Q.data_ptr(), K.data_ptr(), V.data_ptr(), out.data_ptr()
    last = o + fo[0]
    if (o < q + fq[0] and q < last and not (o == q and same) and not _apart(o, fo, q, fq)) or (o < k + fk[0] and k < last and not _apart(o, fo, k, fk)) or \
            (o < v + fv[0] and v < last and not _apart(o, fo, v, fv)):
        raise ValueError("attention: out lies over Q, K or V")
    device = _device()
    prefix = 0 if prefix is None else _vector("prefix", prefix, (E,), _INT32, device)
    q_lens = 0 if q_lens is None else _vector("q_lens", q_lens, (E,), _INT32, device)
    k_lens = 0 if k_lens is None else _vector("k_lens", k_lens, (E,), _INT32, device)
    q_start = 0 if q_start is None else _vector("q_start", q_start, (E,), _INT32, device)
    q_docs = 0 if q_docs is None else _vector("q_docs", q_docs, (E, T), _INT32, device)
    k_docs = 0 if k_docs is None else _vector("k_docs", k_docs, (E, S), _INT32, device)
    k_pos = 0 if k_pos is None else _vector("k_pos", k_pos, (E, S), _INT32, device)
    slopes = 0 if slopes is None else _vector("slopes", slopes, (H,), _F32, device)
    lse = 0 if lse is None else _vector("lse", lse, (E, H, T), _F32, device)
    weights = 0 if weights is None else _vector("weights", weights, (E, S), _F32, device)
    if cache is not None:
        K_scale, V_scale = _vector("cache.K_scale", K_scale, K_scale.shape, _F32, device), _vector("cache.V_scale", V_scale, V_scale.shape, _F32, device)
    if (q | k | v | o) & 15 or not Q.get_device() == K.get_device() == V.get_device() == out.get_device() == device:
        _misplaced(device, Q=Q, K=K, V=V, out=out)
    if E == 0 or (T == 0 and not weights):      # (without queries the weights still decay)
        return out
    if S == 0:                                  # no key: documents of none have no address
        q_docs = k_docs = 0
    if weights and not lse and T:
        held = _scratch("attention_lse", 4 * E * H * T, Q.device)
        lse = held.data_ptr()
    need = nbytes[1 if q_docs or weights else 0]
    ws = _scratch("attention_ws", need, Q.device) if need else None
    block = _ATTENTION_HEAD.pack(q, k, v, K_scale or 0, V_scale or 0, o, lse, weights, ws.data_ptr() if need else 0, prefix, q_lens, k_lens, q_start, q_docs, k_docs,
                                 k_pos, slopes, need) + strides + _FLOATS.pack(scale, cap, decay) + dims + _CAUSAL.pack(1 if causal else 0, 0)
    _lib.call("fvla_attention_run", block, torch._C._cuda_getCurrentRawStream(device))
    return out


def masked_attention(Q, K, V, scale, out, causal=False, prefix=None, q_lens=None, k_lens=None, q_docs=None, k_docs=None, cap=0.0, slopes=None,
                     lse=None):
    """out = softmax(bias(cap(scale * Q K^T))) V over the keys that each query sees.

    Q, out (E, T, H, D); K, V (E, S, HK, D), H a multiple of HK; bf16, D a multiple of 8 up to 256. `out` may be Q, row by
    row, and otherwise overlaps neither Q nor K nor V.
    cap > 0: scores become cap * tanh(score / cap). slopes (H,) fp32: slope * |distance| is taken off them.
    k_lens, q_lens (E,): keys and queries of each episode, all by default; rows of `out` (and of `lse`) behind q_lens stay as they were. The queries are the
    last tokens of their episode: token t stands at k_lens - q_lens + t.
    causal: a query sees keys up to its own position; prefix (E,): and all of the first `prefix` keys.
    q_docs (E, T), k_docs (E, S): a query sees the keys of its own document; negative ids are padding.
    A query that sees no key gets zeros. lse (E, H, T) fp32 receives the natural log-sum-exp of the scores, -inf for such a query.
    One new token per episode (T = 1) is the same call. K and V behind k_lens, or under a negative document id, may hold anything; a value
    of V elsewhere that is not finite can reach queries that do not see it."""
    return _attend(Q, K, V, None, scale, out, causal, prefix, q_lens, k_lens, None, q_docs, k_docs, None, cap, slopes, lse, None, 1.0)


def cache_attention(Q, cache, lengths, scale, out, causal=False, prefix=None, q_lens=None, q_start=None, k_pos=None, cap=0.0, slopes=None, lse=None,
                    weights=None, decay=1.0):
    """`masked_attention` over a `QuantizedCache` of which each episode has `lengths` (E,) rows, the queries' own among them.

    q_start (E,): position of each episode's first query, by default lengths - q_lens. k_pos (E, rows): position of each cached row, by default its
    number; a cache that `cache_evict` has thinned out needs both for `causal`, `prefix` (then positions below `prefix`) and `slopes`.
    weights (E, rows) fp32: weights = decay * weights + the probability mass that each row received from all queries and heads; rows
    behind `lengths` stay as they were. decay = 0 overwrites. `out` may be Q."""
    return _attend(Q, None, None, cache, scale, out, causal, prefix, q_lens, lengths, q_start, None, None, k_pos, cap, slopes, lse, weights, decay)


@functools.lru_cache(maxsize=1024)
def _append_plan(k, v, cache):
    a = _lib.CacheAppend()
    a.block = _cache_shapes("cache", *cache)
    a.k_stride[:] = _rows("K", *k, torch.bfloat16, 8, shared=(0, 1, 2))
    a.v_stride[:] = _rows("V", *v, torch.bfloat16, 8, shared=(0, 1, 2))
    for field, i in (("k_held_stride", 0), ("v_held_stride", 1)):
        getattr(a, field)[:] = _rows("cache", cache[0][i], cache[1][i], cache[2][i], torch.float8_e4m3fn, 16)
    E, rows, HK, D = cache[0][0]
    T = k[0][1]
    if tuple(k[0]) != (E, T, HK, D) or tuple(v[0]) != (E, T, HK, D):
        raise ValueError(f"cache_append: K {tuple(k[0])} and V {tuple(v[0])} do not fit a cache of {tuple(cache[0][0])}")
    if T > rows:
        raise ValueError(f"cache_append: {T} rows into a cache of {rows}")
    if E >= 1 << 16 or rows >= 1 << 31 or HK == 0:
        raise ValueError(f"cache_append: a cache of {tuple(cache[0][0])}")
    a.episodes, a.tokens, a.rows, a.kv_heads, a.head_dim = E, T, rows, HK, D
    return _between(a, "k_stride", None), E, T, _footprint(cache[0][0], cache[1][0], 1), _footprint(cache[0][1], cache[1][1], 1)


def cache_append(K, V, cache, starts, counts=None):
    """New rows K, V (E, T, kv_heads, head_dim) bf16 into rows starts[e] .. starts[e] + T - 1 of each episode's cache (counts[e] <= T of them).

    The scale of a block is the smallest power of two that brings its new values into e4m3's range, or the block's own where that is larger and the
    block holds rows before starts[e]; where it has grown, those rows are moved to it. Rows behind the new ones are taken to be unused. Values
    that are not finite become NaN and leave the scale alone. Rows that would lie outside the cache are left out (device status 8)."""
    held_k, held_v, k_scale, v_scale = cache
    rest, E, T, fk, fv = _append_plan(_layout(K), _layout(V), _cache_layout(cache))
    to_k, to_v = held_k.data_ptr(), held_v.data_ptr()
    if (to_k < to_v + fv[0] and to_v < to_k + fk[0] and not _apart(to_k, fk, to_v, fv)) or abs(k_scale.data_ptr() - v_scale.data_ptr()) < 4 * k_scale.numel():
        raise ValueError("cache_append: K and V of the cache share memory")
    device = _device()
    starts = _vector("starts", starts, (E,), _INT32, device)
    counts = 0 if counts is None else _vector("counts", counts, (E,), _INT32, device)
    k_scale, v_scale = _vector("cache.K_scale", k_scale, k_scale.shape, _F32, device), _vector("cache.V_scale", v_scale, v_scale.shape, _F32, device)
    k, v = K.data_ptr(), V.data_ptr()
    if (k | v | to_k | to_v) & 15 or not K.get_device() == V.get_device() == held_k.get_device() == held_v.get_device() == device:
        _misplaced(device, K=K, V=V, cache_K=held_k, cache_V=held_v)
    block = _APPEND_HEAD.pack(k, v, to_k, to_v, k_scale, v_scale, starts, counts) + rest
    if E and T:
        _lib.call("fvla_cache_append", block, torch._C._cuda_getCurrentRawStream(device))


@functools.lru_cache(maxsize=1024)
def _evict_plan(cache, out, keep, sinks, recent):
    a = _lib.CacheEvict()
    a.block, a.out_block = _cache_shapes("cache", *cache), _cache_shapes("out_cache", *out)
    for name, layout, fields in (("cache", cache, ("k_stride", "v_stride")), ("out_cache", out, ("out_k_stride", "out_v_stride"))):
        for i, field in enumerate(fields):
            getattr(a, field)[:] = _rows(name, layout[0][i], layout[1][i], layout[2][i], torch.float8_e4m3fn, 16, shared=(0, 1, 2) if name == "cache" else ())
    E, rows, HK, D = cache[0][0]
    out_rows = out[0][0][1]
    if tuple(out[0][0]) != (E, out_rows, HK, D):
        raise ValueError(f"cache_evict: rows of {tuple(cache[0][0])} into {tuple(out[0][0])}")
    if not 0 < keep <= out_rows:
        raise ValueError(f"cache_evict: {keep} rows to keep in a cache of {out_rows}")
    if sinks < 0 or recent < 0 or sinks + recent > keep:
        raise ValueError(f"cache_evict: the first {sinks} and the last {recent} rows in {keep}")
    if E >= 1 << 16 or rows >= 1 << 31 or HK == 0:
        raise ValueError(f"cache_evict: a cache of {tuple(cache[0][0])}")
    a.episodes, a.rows, a.out_rows, a.kv_heads, a.head_dim, a.keep, a.sinks, a.recent = E, rows, out_rows, HK, D, keep, sinks, recent
    return (_between(a, "k_stride", None), _lib.load().fvla_cache_evict_workspace_bytes(E, keep), E, rows, out_rows,
            tuple(_footprint(layout[0][i], layout[1][i], 1) for layout in (cache, out) for i in (0, 1)))


_first = operator.itemgetter(0)


def _all_apart(spans):
    """Whether no destination among these spans shares a byte with another one of them."""
    spans = [(p, whole or (last - p, last - p, ()), out) for p, last, out, whole in spans if last > p]
    return all(_apart(p, a, q, b) for i, (p, a, out) in enumerate(spans) for q, b, other in spans[:i] if out or other)


def cache_evict(cache, lengths, weights, keep, out_cache, out_lengths, out_weights=None, positions=None, out_positions=None, sinks=0, recent=0):
    """The rows of each episode that stay, in their order, into `out_cache` (another cache of at least `keep` rows).

    min(lengths[e], keep) rows stay: the first `sinks`, the last `recent` and of the others those of the largest weight (weights (E, rows) fp32 as
    `cache_attention` adds them up; equal weights: the first rows; NaN: as -inf). out_lengths (E,) receives their number; out_weights
    (E, out rows) fp32 and out_positions (E, out rows) int32 what weight and position each had (positions (E, rows), or the row numbers). A block's
    scale is the largest among its rows', and values are rounded again where theirs was smaller. What lies behind the last row stays as it was."""
    held_k, held_v, k_scale, v_scale = cache
    to_k, to_v, to_k_scale, to_v_scale = out_cache
    rest, nbytes, E, rows, out_rows, footprints = _evict_plan(_cache_layout(cache), _cache_layout(out_cache), int(keep), int(sinks), int(recent))
    device = _device()
    n, out_n = _vector("lengths", lengths, (E,), _INT32, device), _vector("out_lengths", out_lengths, (E,), _INT32, device)
    w = _vector("weights", weights, (E, rows), _F32, device)
    out_w = 0 if out_weights is None else _vector("out_weights", out_weights, (E, out_rows), _F32, device)
    pos = 0 if positions is None else _vector("positions", positions, (E, rows), _INT32, device)
    out_pos = 0 if out_positions is None else _vector("out_positions", out_positions, (E, out_rows), _INT32, device)
    ks, vs = _vector("cache.K_scale", k_scale, k_scale.shape, _F32, device), _vector("cache.V_scale", v_scale, v_scale.shape, _F32, device)
    to_ks = _vector("out_cache.K_scale", to_k_scale, to_k_scale.shape, _F32, device)
    to_vs = _vector("out_cache.V_scale", to_v_scale, to_v_scale.shape, _F32, device)
    k, v = _address("cache.K", held_k, device), _address("cache.V", held_v, device)
    to_k, to_v = _address("out_cache.K", to_k, device), _address("out_cache.V", to_v, device)
    if E == 0:
        return
    # (first byte, byte behind the last, a destination, footprint where it is not whole)
    small, large, (fk, fv, to_fk, to_fv) = 4 * k_scale.numel(), 4 * to_k_scale.numel(), footprints
    spans = [(n, n + 4 * E, 0, None), (w, w + 4 * E * rows, 0, None), (pos, pos + 4 * E * rows if pos else 0, 0, None), (ks, ks + small, 0, None), (vs, vs + small, 0, None),
             (k, k + fk[0], 0, fk), (v, v + fv[0], 0, fv), (out_n, out_n + 4 * E, 1, None), (out_w, out_w + 4 * E * out_rows if out_w else 0, 1, None),
             (out_pos, out_pos + 4 * E * out_rows if out_pos else 0, 1, None), (to_ks, to_ks + large, 1, None), (to_vs, to_vs + large, 1, None), (to_k, to_k + to_fk[0], 1, to_fk),
             (to_v, to_v + to_fv[0], 1, to_fv)]
    spans.sort(key=_first)
    read = written = 0                          # how far the operands so far reach
    for first, last, out, _ in spans:
        if (first < written or (out and first < read)) and not _all_apart(spans):
            raise ValueError("cache_evict: a destination lies over another operand")
        if out:
            written = last if last > written else written
        else:
            read = last if last > read else read
    ws = _scratch("evict_ws", nbytes, weights.device)
    block = _EVICT_HEAD.pack(k, v, ks, vs, w, to_k, to_v, to_ks, to_vs, out_w, ws.data_ptr(), n, pos, out_n, out_pos, nbytes) + rest
    _lib.call("fvla_cache_evict", block, torch._C._cuda_getCurrentRawStream(device))


OPERATORS = {f.__name__: f for f in (masked_attention, cache_append, cache_attention, cache_evict)}

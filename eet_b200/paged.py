"""Serving from a paged cache: rotary positions, the append of new keys and values to pages, and the attention of new tokens -
one a sequence, or a chunk of a prompt behind its history - over the pages.

A cache is two tensors k_cache, v_cache [pages, kv_heads, page_size, head_dim], fp16 or bf16, allocated by the caller (views
with other strides will do as long as rows of head_dim are contiguous).  Sequence b holds ``lens[b]`` positions; position p
of it is slot ``p % page_size`` of page ``pages[b, p // page_size]``.  The new tokens of all sequences are rows behind one
another: those of sequence b are rows ``starts[b]`` to ``starts[b + 1]``, and they are the last positions of their sequence.
A step of a model with chunks and single tokens side by side is therefore, in each layer,

    q = paged_store(k, v, k_cache, v_cache, pages, starts, lens, q=q, freqs=freqs)
    ctx = paged_mha(q, k_cache, v_cache, pages, starts, lens)

with ``pages`` int32 [sequences, columns], ``starts`` int32 [sequences + 1] and ``lens`` int32 [sequences] on the GPU.  They
are read there, so a captured CUDA graph of these calls serves whatever they hold when it is replayed.  Entries of ``pages``
behind a sequence's last position are not read.  A page number outside the cache is not followed: the call completes and
``EET.check_device_status()`` reports it.

A cache may also hold 8-bit codes: k_cache and v_cache int8 or float8_e4m3fn, beside k_scale and v_scale float32 [pages, kv_heads,
page_size] - half the memory, and half of what a decode step reads.  A row of head_dim values is kept as code * scale with scale = max |y| /
127 or / 448; paged_store writes both, paged_mha and paged_load take both, as k_scale= and v_scale=.  `paged_load` reads rows back.

`PagedMmha` is the attention block around them, beside `EET.LlamaMmha` and `EET.BaichuanMmha`.

The reference serves one contiguous cache an op, all sequences at the same step (csrc/op/llama_mmha.cpp:94-112).
"""
import math
import struct

import torch

from ._lib import check, lib
from .EET import _current_device, _forget, _linear, _norm_head, _on, _pool, _raw_stream

__all__ = ["rotary_frequencies", "apply_rotary", "paged_store", "paged_load", "paged_mha", "PagedMmha"]

_DTYPES = (torch.float16, torch.bfloat16)
_PAGE_SIZES = (16, 32, 64, 128, 256)
_pack_rotary = struct.Struct("6P15qd").pack
_pack_store = struct.Struct("11P26qd").pack
_pack_mha = struct.Struct("9P23qd").pack
_pack_scratch = struct.Struct("Pq").pack
_NO_SCRATCH = _pack_scratch(0, 0)
_CODES = {torch.int8: 1, torch.float8_e4m3fn: 2}
_pack_codes = struct.Struct("2P5q").pack
_pack_load = struct.Struct("9P20q").pack


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, device="cuda:0"):
    """(freqs, magnitude): radians a position of each pair of a head's rotated part, float64 [rotary_dim / 2], and the factor
    on the rotated values (1.0 but for "yarn").

    Pair i turns by base ** (-2 i / rotary_dim) a position.  ``scaling`` stretches that for contexts longer than a model was
    trained on, a dict with "type", "factor" and
      "linear"  every frequency / factor
      "ntk"     base * factor ** (rotary_dim / (rotary_dim - 2)) instead of base
      "bands"   "original" (the trained length L), "low" and "high": pairs that turn more than `high` times in L stay, those that turn
                less than `low` times are divided by factor, between them a blend that is linear in the number of turns
      "yarn"    "original", optional "fast" (32) and "slow" (1): the same idea with a blend that is linear in the pair's index,
                from the index that turns `fast` times in L (rounded down) to the one that turns `slow` times (rounded up), and a
                magnitude of 0.1 ln(factor) + 1, or "magnitude" (Peng et al., 2023)"""
    if rotary_dim <= 0 or rotary_dim % 16:
        raise RuntimeError(f"rotary_frequencies: rotary_dim {rotary_dim} must be a multiple of 16")
    half, magnitude = rotary_dim // 2, 1.0
    scaling = dict(scaling) if scaling else {"type": "none", "factor": 1.0}
    kind, factor = scaling.pop("type"), float(scaling.pop("factor"))
    if not base > 1.0 or not factor > 0.0:
        raise RuntimeError("rotary_frequencies: base must be above 1 and factor above 0")
    if kind == "ntk":
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freqs = [base ** (-2.0 * i / rotary_dim) for i in range(half)]
    if kind == "linear":
        freqs = [f / factor for f in freqs]
    elif kind == "bands":
        length, low, high = (float(scaling.pop(k)) for k in ("original", "low", "high"))
        if not high > low:
            raise RuntimeError("rotary_frequencies: high must be above low")
        stay = [min(1.0, max(0.0, (f * length / (2 * math.pi) - low) / (high - low))) for f in freqs]
        freqs = [s * f + (1.0 - s) * f / factor for s, f in zip(stay, freqs)]
    elif kind == "yarn":
        length = float(scaling.pop("original"))
        fast, slow = float(scaling.pop("fast", 32.0)), float(scaling.pop("slow", 1.0))
        magnitude = float(scaling.pop("magnitude", 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0))
        index = [rotary_dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (fast, slow)]
        low, high = max(0, math.floor(index[0])), min(rotary_dim - 1, math.ceil(index[1]))
        part = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(half)]
        freqs = [s * f / factor + (1.0 - s) * f for s, f in zip(part, freqs)]
    elif kind not in ("none", "ntk"):
        raise RuntimeError(f"rotary_frequencies: unknown scaling type {kind!r}")
    if scaling:
        raise RuntimeError(f"rotary_frequencies: {sorted(scaling)} mean nothing to scaling type {kind!r}")
    return torch.tensor(freqs, dtype=torch.float64, device=device), magnitude


# The checks below run once per tensor and call; a decode step's calls last about as long on the host as on the GPU, so each
# reads as few attributes as it can (a device is compared as its index, -1 for the CPU's).
def _first(who, name, t):
    """Shape, dtype, device index, token and head strides of the tensor that the others are held against."""
    shape, dtype, index = t.shape, t.dtype, t.get_device()
    if len(shape) != 3 or dtype not in _DTYPES or index < 0:
        raise RuntimeError(f"{who}: {name} must be a CUDA fp16 or bf16 tensor [tokens, heads, head_dim], got {tuple(shape)} {t.dtype} "
                           f"on {t.device}")
    strides = t.stride()
    if strides[2] != 1:
        return shape, dtype, index, _heads(who, name, t, shape, dtype, index)   # (refuses it)
    return shape, dtype, index, strides[:2]


def _heads(who, name, t, shape, dtype, index):
    """Token and head strides of a tensor that must have this shape."""
    strides = t.stride()
    if t.shape != shape or t.dtype != dtype or t.get_device() != index or strides[2] != 1:
        raise RuntimeError(f"{who}: {name} must be a {dtype} tensor of shape {tuple(shape)} with a contiguous last dimension on "
                           f"cuda:{index}, got {tuple(t.shape)} {t.dtype} with strides {strides} on {t.device}")
    return strides[:2]


def _output(who, name, t, like, shape, strides, dtype, index):
    """The tensor for a result of the shape of `like`, and its token and head strides."""
    if t is not None:
        return t, _heads(who, name, t, shape, dtype, index)
    _, heads, head_dim = shape
    # (where the rows stand in their order empty_like makes them contiguous by itself: 1.4 us, told to 1.5, torch.empty 1.65)
    if strides[1] >= head_dim and strides[0] >= heads * strides[1]:
        return torch.empty_like(like), (heads * head_dim, head_dim)
    return torch.empty_like(like, memory_format=torch.contiguous_format), (heads * head_dim, head_dim)


def _call(function, args, index):
    """One entry point on the current stream of the tensors' device."""
    if index == _current_device():
        check(function(args, _raw_stream(index)))
    else:
        with torch.cuda.device(index):
            check(function(args, _raw_stream(index)))


def _workspace_bytes(function, args, index):
    if index == _current_device():
        return function(args)
    with torch.cuda.device(index):
        return function(args)


def _array(who, name, t, dtype, numel, index):
    """The address of a contiguous vector on the device."""
    if t.dtype != dtype or t.get_device() != index or t.shape != (numel,) or not t.is_contiguous():
        raise RuntimeError(f"{who}: {name} must be a contiguous {dtype} tensor [{numel}] on cuda:{index}, got {tuple(t.shape)} {t.dtype} on "
                           f"{t.device}")
    return t.data_ptr()


def _cache(who, k_cache, v_cache, dtype, index):
    """(pages, kv_heads, page_size, head_dim) and the strides of a cache of this type, a 16-bit one or that of codes."""
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise RuntimeError(f"{who}: k_cache and v_cache must both be [pages, kv_heads, page_size, head_dim], got {tuple(shape)} and "
                           f"{tuple(v_cache.shape)}")
    if k_cache.dtype != dtype or v_cache.dtype != dtype or k_cache.get_device() != index or v_cache.get_device() != index:
        raise RuntimeError(f"{who}: the caches must be {dtype} on cuda:{index}, as the other tensors are")
    ks, vs = k_cache.stride(), v_cache.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise RuntimeError(f"{who}: the last dimension of the caches must be contiguous")
    if shape[2] not in _PAGE_SIZES:
        raise RuntimeError(f"{who}: page size {shape[2]}, only 16, 32, 64, 128 and 256 are supported")
    return shape, ks[:3] + vs[:3]


def _scales(who, k_cache, k_scale, v_scale, shape, index):
    """What the entry points for codes take behind the arguments of the others."""
    if k_scale is None or v_scale is None:
        raise RuntimeError(f"{who}: a cache of codes has both k_scale and v_scale")
    rows = shape[:3]
    ks, vs = k_scale.stride(), v_scale.stride()
    for name, t, strides in (("k_scale", k_scale, ks), ("v_scale", v_scale, vs)):
        if t.shape != rows or t.dtype != torch.float32 or t.get_device() != index or strides[2] != 1:
            raise RuntimeError(f"{who}: {name} must be a float32 tensor {tuple(rows)} with contiguous slots on cuda:{index}, got "
                               f"{tuple(t.shape)} {t.dtype} with strides {strides} on {t.device}")
    return _pack_codes(k_scale.data_ptr(), v_scale.data_ptr(), _CODES[k_cache.dtype], ks[0], ks[1], vs[0], vs[1])


def _kept_type(who, k_cache, dtype, k_scale, v_scale):
    """The type that both caches must have: q's, or with scales that of codes."""
    if k_scale is None and v_scale is None:
        return dtype
    if k_cache.dtype not in _CODES:
        raise RuntimeError(f"{who}: scales belong to a cache of codes, int8 or float8_e4m3fn, not to {k_cache.dtype}")
    return k_cache.dtype


def _table(who, pages, starts, lens, index):
    """(sequences, columns, row stride) of the page table, the addresses of it, starts and lens."""
    shape = pages.shape
    if len(shape) != 2 or pages.dtype != torch.int32 or pages.get_device() != index or (shape[1] > 1 and pages.stride(1) != 1):
        raise RuntimeError(f"{who}: pages must be an int32 tensor [sequences, columns] with contiguous rows on cuda:{index}, got "
                           f"{tuple(shape)} {pages.dtype} on {pages.device}")
    seqs, columns = shape
    addresses = (pages.data_ptr(), _array(who, "starts", starts, torch.int32, seqs + 1, index),
                 _array(who, "lens", lens, torch.int32, seqs, index))
    return seqs, columns, pages.stride(0) if seqs > 1 else columns, addresses


def apply_rotary(q, k, positions, freqs, interleaved=False, magnitude=1.0, q_out=None, k_out=None):
    """Rotary positions of q [tokens, heads, head_dim] and k [tokens, kv_heads, head_dim] (either may be None): returns
    (q_out, k_out), new tensors unless given; q_out=q works in place.

    positions int64 [tokens]; freqs from rotary_frequencies, float64 [rotary_dim / 2], any rotary_dim up to head_dim that is a
    multiple of 16 - the rest of a head is copied.  Pair i is dims (i, i + rotary_dim / 2), with `interleaved` (2 i, 2 i + 1).
    Token and head strides are free (a view of a fused projection will do) but multiples of 8."""
    who = "apply_rotary"
    like = k if q is None else q
    if like is None:
        raise RuntimeError("apply_rotary: neither q nor k is given")
    shape, dtype, index, strides = _first(who, "k" if q is None else "q", like)
    tokens, heads, head_dim = shape
    kv_heads = 0
    q_str = qo_str = k_str = ko_str = (0, 0)
    q_at = qo_at = k_at = ko_at = 0
    if q is None:
        heads = 0
    else:
        q_str = strides
        q_out, qo_str = _output(who, "q_out", q_out, q, shape, strides, dtype, index)
        q_at, qo_at = q.data_ptr(), q_out.data_ptr()
    if k is not None:
        shape = k.shape
        kv_heads = shape[1] if len(shape) == 3 else 0
        shape = (tokens, kv_heads, head_dim)
        k_str = _heads(who, "k", k, shape, dtype, index)
        k_out, ko_str = _output(who, "k_out", k_out, k, shape, k_str, dtype, index)
        k_at, ko_at = k.data_ptr(), k_out.data_ptr()
    half = freqs.numel()
    args = _pack_rotary(q_at, k_at, qo_at, ko_at, _array(who, "positions", positions, torch.int64, tokens, index),
                        _array(who, "freqs", freqs, torch.float64, half, index), tokens, heads, kv_heads, head_dim, 2 * half,
                        bool(interleaved), dtype == torch.bfloat16, *q_str, *k_str, *qo_str, *ko_str, magnitude)
    _call(lib.eet_rotary, args, index)
    return q_out, k_out


def paged_store(k, v, k_cache, v_cache, pages, starts, lens, q=None, freqs=None, interleaved=False, magnitude=1.0, positions=None,
                q_out=None, k_scale=None, v_scale=None):
    """Appends k and v [tokens, kv_heads, head_dim] of new tokens to their pages, k rotated when freqs is given, and returns q
    [tokens, heads, head_dim] rotated the same way (in q_out; a new tensor unless given, q_out=q works in place; None without q).

    With caches of codes k_scale and v_scale are written beside them: k behind its rotation, in fp32, and v are divided by their scale and
    rounded once, to nearest; a row of zeros has the scale 1, one with a NaN or an infinity NaN.

    The positions of the rotation are those in the sequence, or positions int64 [tokens].  Rows of k, v and q that belong to no
    sequence are not touched; of rows in front of a sequence's first position only q is.  Two sequences must not append to the same
    slot (one that they share must lie before both's new tokens)."""
    who = "paged_store"
    shape, dtype, index, k_str = _first(who, "k", k)
    tokens, kv_heads, head_dim = shape
    v_str = _heads(who, "v", v, shape, dtype, index)
    cache_shape, cache_strides = _cache(who, k_cache, v_cache, _kept_type(who, k_cache, dtype, k_scale, v_scale), index)
    if cache_shape[1] != kv_heads or cache_shape[3] != head_dim:
        raise RuntimeError(f"paged_store: caches of {cache_shape[1]} heads of {cache_shape[3]} beside {kv_heads} heads of {head_dim}")
    seqs, columns, pages_stride, table = _table(who, pages, starts, lens, index)
    heads, q_str, qo_str, q_at, qo_at = 0, (0, 0), (0, 0), 0, 0
    if q is not None:
        q_shape = q.shape
        heads = q_shape[1] if len(q_shape) == 3 else 0
        q_shape = (tokens, heads, head_dim)
        q_str = _heads(who, "q", q, q_shape, dtype, index)
        q_out, qo_str = _output(who, "q_out", q_out, q, q_shape, q_str, dtype, index)
        q_at, qo_at = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise RuntimeError("paged_store: q_out without q")
    half = turns = where = 0
    if freqs is not None:
        half = freqs.numel()
        turns = _array(who, "freqs", freqs, torch.float64, half, index)
    if positions is not None:
        where = _array(who, "positions", positions, torch.int64, tokens, index)
    args = _pack_store(q_at, k.data_ptr(), v.data_ptr(), qo_at, k_cache.data_ptr(), v_cache.data_ptr(), *table, where, turns, tokens, seqs,
                       heads, kv_heads, head_dim, 2 * half, bool(interleaved), dtype == torch.bfloat16, cache_shape[0], cache_shape[2],
                       columns, pages_stride, *q_str, *k_str, *v_str, *qo_str, *cache_strides, magnitude)
    if k_scale is None and v_scale is None:
        _call(lib.eet_paged_store, args, index)
    else:
        _call(lib.eet_paged_store_codes, args + _scales(who, k_cache, k_scale, v_scale, cache_shape, index), index)
    return q_out


def paged_load(k_cache, v_cache, pages, starts, lens, tokens=None, dtype=None, k_scale=None, v_scale=None, k_out=None, v_out=None):
    """Reads rows back from their pages, the mirror of paged_store: returns (k, v) [tokens, kv_heads, head_dim], rows starts[b] to
    starts[b + 1] being the last positions of sequence b (whole histories: starts = 0, lens[0], lens[0] + lens[1], ...).

      tokens         the number of rows, that of k_out by default
      dtype          fp16 or bf16 for a cache of codes, whose values code * scale are rounded to it; a 16-bit cache comes back as it is
      k_out, v_out   new tensors unless given
    Rows that belong to no sequence, or lie in front of its first position, are left as they are, uninitialised in new tensors."""
    who = "paged_load"
    index, kept = k_cache.get_device(), k_cache.dtype
    if index < 0 or (kept not in _DTYPES and kept not in _CODES):
        raise RuntimeError(f"{who}: k_cache must be a CUDA tensor of fp16, bf16, int8 or float8_e4m3fn, got {kept} on {k_cache.device}")
    shape, strides = _cache(who, k_cache, v_cache, kept, index)
    codes = _CODES.get(kept, 0)
    if codes:
        scales = _scales(who, k_cache, k_scale, v_scale, shape, index)
    elif k_scale is not None or v_scale is not None:
        raise RuntimeError(f"{who}: scales belong to a cache of codes, int8 or float8_e4m3fn, not to {kept}")
    else:
        scales = _pack_codes(0, 0, 0, 0, 0, 0, 0)
    given = v_out if k_out is None else k_out
    if dtype is None:
        dtype = given.dtype if given is not None else torch.float16 if codes else kept
    if dtype not in _DTYPES or (not codes and dtype != kept):
        raise RuntimeError(f"{who}: a cache of {kept} is not read back as {dtype}")
    if tokens is None:
        if given is None:
            raise RuntimeError(f"{who}: neither tokens nor k_out is given")
        tokens = given.shape[0]
    kv_heads, head_dim = shape[1], shape[3]
    dense = (kv_heads * head_dim, head_dim)
    rows = None if given is None else torch.Size((tokens, kv_heads, head_dim))
    if k_out is None:
        k_out, k_str = torch.empty((tokens, kv_heads, head_dim), dtype=dtype, device=k_cache.device), dense
    else:
        k_str = _heads(who, "k_out", k_out, rows, dtype, index)
    if v_out is None:
        v_out, v_str = torch.empty_like(k_out) if k_str == dense else torch.empty((tokens, kv_heads, head_dim), dtype=dtype, device=k_cache.device), dense
    else:
        v_str = _heads(who, "v_out", v_out, rows, dtype, index)
    seqs, columns, pages_stride, table = _table(who, pages, starts, lens, index)
    args = _pack_load(k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr() if codes else 0, v_scale.data_ptr() if codes else 0,
                      k_out.data_ptr(), v_out.data_ptr(), *table, tokens, seqs, kv_heads, head_dim, codes, dtype == torch.bfloat16, shape[0],
                      shape[2], columns, pages_stride, *k_str, *v_str, *strides) + scales[24:]
    _call(lib.eet_paged_load, args, index)
    return k_out, v_out


def paged_mha(q, k_cache, v_cache, pages, starts, lens, max_tokens=None, max_len=None, scale=None, window=0, first_key=None,
              alibi_slopes=None, out=None, k_scale=None, v_scale=None):
    """Attention of new tokens q [tokens, heads, head_dim] over the pages, which hold the new tokens' own keys and values already
    (paged_store).  Returns out, the shape of q.

    A token at position p of sequence b sees positions max(0, first_key[b], p - window + 1) .. p; one that sees none gets zeros.
    heads is a multiple of kv_heads: that many query heads in a row share a kv head.
      max_tokens, max_len   the most new tokens and the most positions that a sequence has, as far as the caller knows (a captured
                            call: the most there may be).  They choose how the work is cut up, not what is computed.
      scale                 of the scores, 1 / sqrt(head_dim) by default
      window                0: no window
      first_key             int32 [sequences]: positions before it are padding
      alibi_slopes          float32 [heads]: slope * (key position - p) is added to the scores
      k_scale, v_scale      of caches of codes
    out may be q.  Rows of out that belong to no sequence are left as they are, uninitialised where this call allocated out.
    Slots that no new token sees may hold anything.  What some new token of a sequence sees must be finite: a NaN or infinity in v reaches
    other new tokens of that sequence, too, also those before it."""
    who = "paged_mha"
    shape, dtype, index, q_str = _first(who, "q", q)
    tokens, heads, head_dim = shape
    cache_shape, cache_strides = _cache(who, k_cache, v_cache, _kept_type(who, k_cache, dtype, k_scale, v_scale), index)
    if cache_shape[3] != head_dim:
        raise RuntimeError(f"paged_mha: caches of head size {cache_shape[3]} beside a q of {head_dim}")
    seqs, columns, pages_stride, table = _table(who, pages, starts, lens, index)
    out, o_str = _output(who, "out", out, q, shape, q_str, dtype, index)
    first = 0 if first_key is None else _array(who, "first_key", first_key, torch.int32, seqs, index)
    slopes = 0 if alibi_slopes is None else _array(who, "alibi_slopes", alibi_slopes, torch.float32, heads, index)
    if max_tokens is None:
        max_tokens = 1 if tokens == seqs else tokens
    args = _pack_mha(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), *table, first, slopes, tokens, seqs, heads,
                     cache_shape[1], head_dim, dtype == torch.bfloat16, cache_shape[0], cache_shape[2], columns, pages_stride, *q_str,
                     *o_str, *cache_strides, window, max_tokens, max_len or 0, 1.0 / math.sqrt(head_dim) if scale is None else scale)
    # (how the call is planned, and with it the scratch, goes by sizes and by the device's number of SMs)
    if k_scale is None and v_scale is None:
        call, size, scales = lib.eet_paged_mha, lib.eet_paged_mha_workspace_bytes, b""
    else:
        call, size = lib.eet_paged_mha_codes, lib.eet_paged_mha_codes_workspace_bytes
        scales = _scales(who, k_cache, k_scale, v_scale, cache_shape, index)
    ws_bytes = _workspace_bytes(size, args + _NO_SCRATCH + scales, index)
    if ws_bytes:
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
        args += _pack_scratch(ws.data_ptr(), ws_bytes)
    else:
        args += _NO_SCRATCH
    _call(call, args + scales, index)
    return out


class PagedMmha:
    """Attention block over a paged cache: RMSNorm, W8A16 (or fp16) QKV projection, rotary positions and append, attention, output
    projection + residual - the flow of EET.LlamaMmha / EET.BaichuanMmha (csrc/op/llama_mmha.cpp:114-266) for sequences of
    different ages, chunks and single tokens in one call, and kv heads that several query heads share.

      QKV_weights     [hidden, (heads + 2 kv_heads) 128] (q, then k, then v), packed int8 or fp16 as MetaDesc.is_int8 says
      Output_weights  [heads 128, hidden]
      kv_head_num     MetaDesc.head_num by default
      freqs           from rotary_frequencies; by default all 128 dims at base 10000, none with alibi_slopes
      alibi_slopes    float32 [heads] instead of rotary positions (the op of Baichuan-13B)
    The caches belong to the caller, a pair for each layer.  MetaDesc.batch_size * max_seq_len is the most tokens of a call.  The
    output is a view of a buffer that the ops of a device share, as the other ops' outputs are."""

    def __init__(self, desc, QKV_weights, QKV_scale, Output_weights, Output_scale, layernorm_weights, kv_head_num=None, freqs=None,
                 interleaved=False, magnitude=1.0, alibi_slopes=None):
        desc._require_half("PagedMmha")
        if desc.tp is not None and desc.tp.size > 1:
            raise RuntimeError("PagedMmha: tensor parallelism is not part of this op")
        self.desc, self.heads = desc, desc.head_num
        self.kv_heads = desc.head_num if kv_head_num is None else int(kv_head_num)
        if self.kv_heads <= 0 or self.heads % self.kv_heads:
            raise RuntimeError(f"PagedMmha: {self.heads} heads are not a multiple of {self.kv_heads} kv heads")
        self.size_per_head = desc.hidden_units // desc.head_num if desc.d_kv == 0 else desc.d_kv
        if self.size_per_head != 128:
            raise RuntimeError("PagedMmha: only head size 128 is supported")
        self.inner_dim, self.qkv_dim = 128 * self.heads, 128 * (self.heads + 2 * self.kv_heads)
        for t, shape, what in ((QKV_weights, (desc.hidden_units, self.qkv_dim), "QKV_weights"),
                               (Output_weights, (self.inner_dim, desc.hidden_units), "Output_weights")):
            if tuple(t.shape) != shape or t.dtype != desc.weight_dtype or not t.is_cuda or not t.is_contiguous():
                raise RuntimeError(f"PagedMmha: {what} must be a contiguous CUDA {desc.weight_dtype} tensor of shape {shape}, got "
                                   f"{tuple(t.shape)} {t.dtype}")
        vectors = [(layernorm_weights, desc.hidden_units, "layernorm_weights")]
        if desc.is_int8:
            vectors += [(QKV_scale, self.qkv_dim, "QKV_scale"), (Output_scale, desc.hidden_units, "Output_scale")]
        self.index = QKV_weights.get_device()
        for t, numel, what in vectors:
            if not torch.is_tensor(t) or t.numel() != numel or t.dtype != torch.float16 or t.get_device() != self.index or \
                    not t.is_contiguous():
                raise RuntimeError(f"PagedMmha: {what} must be a contiguous fp16 tensor of {numel} values on cuda:{self.index}, got " +
                                   (f"{tuple(t.shape)} {t.dtype} on {t.device}" if torch.is_tensor(t) else repr(t)))
        if Output_weights.get_device() != self.index:
            raise RuntimeError("PagedMmha: QKV_weights and Output_weights are on different devices")
        self.qkv_w, self.qkv_s, self.out_w, self.out_s, self.ln_w = QKV_weights, QKV_scale, Output_weights, Output_scale, layernorm_weights
        if alibi_slopes is not None and freqs is not None:
            raise RuntimeError("PagedMmha: rotary positions and ALiBi exclude each other")
        if alibi_slopes is None and freqs is None:
            freqs, magnitude = rotary_frequencies(128, device=desc.device)
        self.freqs, self.interleaved, self.magnitude, self.alibi_slopes = freqs, interleaved, magnitude, alibi_slopes

    def forward(self, input, k_cache, v_cache, pages, starts, lens, max_tokens=None, max_len=None, window=0, first_key=None,
                k_scale=None, v_scale=None):
        """input fp16 [tokens, hidden]: the new tokens of all sequences behind one another; the other arguments as in paged_mha."""
        d = self.desc
        if input.dtype != torch.float16 or input.get_device() != self.index or input.dim() != 2 or input.shape[1] != d.hidden_units or \
                not input.is_contiguous():
            raise RuntimeError(f"PagedMmha: input must be a contiguous fp16 tensor [tokens, hidden] on cuda:{self.index}")
        n, cap = input.shape[0], d.batch_size * d.max_seq_len
        if n > cap:
            raise RuntimeError(f"PagedMmha: {n} tokens, MetaDesc allows {cap}")
        with _on(d.device):
            xn = _pool.rows("layernorm", n, d.hidden_units, cap * d.hidden_units, torch.float16, d.device)
            qkv = _pool.rows("qkv_paged", n, self.qkv_dim, cap * self.qkv_dim, torch.float16, d.device)
            ctx = _pool.rows("dst", n, self.inner_dim, cap * self.inner_dim, torch.float16, d.device).view(n, self.heads, 128)
            out = _pool.rows("self_mask_attn_cache", n, d.hidden_units, cap * d.hidden_units, torch.float16, d.device)
            if n == 0:
                return out
            _norm_head(input, self.ln_w, d.layernorm_eps, xn)
            _forget(out)   # (behind the norm: it may be the input)
            _linear(xn, self.qkv_w, self.qkv_s, qkv)
            q, k, v = qkv.view(n, -1, 128).split((self.heads, self.kv_heads, self.kv_heads), 1)
            q = paged_store(k, v, k_cache, v_cache, pages, starts, lens, q=q, freqs=self.freqs, interleaved=self.interleaved,
                            magnitude=self.magnitude, q_out=q, k_scale=k_scale, v_scale=v_scale)
            # (rows that belong to no sequence go through the block like the others and mean nothing)
            paged_mha(q, k_cache, v_cache, pages, starts, lens, max_tokens=max_tokens, max_len=max_len, window=window,
                      first_key=first_key, alibi_slopes=self.alibi_slopes, out=ctx, k_scale=k_scale, v_scale=v_scale)
            _linear(ctx.view(n, self.inner_dim), self.out_w, self.out_s, out, residual=input)
        return out.view(n, d.hidden_units)

    __call__ = forward

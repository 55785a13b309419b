"""Operators around a prompt: what a layer does with the rows of a prompt chunk outside the sparse path.

  qk_norm_rope        RMS norm of every query and key head and rotation of part of the head, one pass
  kv_cache_write      rows into the quantised paged caches (split arrays, packed rows)
  kv_cache_read       positions of sequences back from those caches as contiguous rows
  prompt_attention    dense causal attention of packed sequences with grouped heads

They take raw torch tensors or `from_torch` handles on one CUDA device, write their outputs in place, return None and run
asynchronously on the current stream, as the operators of `ops`. Rows are bfloat16 or float16. Unlike there, tensors of rows may be
views: the last dim is contiguous and every row starts on a 16-byte boundary (strides a multiple of 8 elements).
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from .compat import Tensor as _Handle
from .compat import unwrap
from .ops import _native, _need, _same_device, _workspace

_ROW_DTYPES = {torch.bfloat16: _lib.PTO_DT_BF16, torch.float16: _lib.PTO_DT_F16}
_LAYOUTS = {"half": _lib.PTO_ROPE_HALF, "interleaved": _lib.PTO_ROPE_INTERLEAVED, "deinterleave": _lib.PTO_ROPE_DEINTERLEAVE}


def _rows(x, what, dims):
    """A tensor of rows: any strides but the last one's, which is 1, on 16-byte boundaries."""
    t = x.torch() if isinstance(x, _Handle) else x
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: input type is not currently supported.")
    _need(t.dim() == dims, f"{what}: {dims} dims expected")
    _need(t.dtype in _ROW_DTYPES, f"{what}: bfloat16 or float16")
    if t.numel() == 0:
        return t
    _need(t.stride(-1) == 1 or t.shape[-1] == 1, f"{what}: the last dim must be contiguous")
    _need(all(s % 8 == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1) and t.data_ptr() % 16 == 0,
          f"{what}: rows must start on 16-byte boundaries (strides a multiple of 8 elements)")
    return t


def _stride(t, dim):
    """Stride of a dim; of one that is never stepped along, 0 (torch gives those any value)."""
    return t.stride(dim) if t.shape[dim] > 1 else 0


class RotaryFrequencies:
    """Frequencies of a rotation, on a device: what `qk_norm_rope` turns positions into angles with. Kept by the caller.

    rotary_dim   dims that are rotated, a multiple of 16; pair i turns by position * base^(-2i / rotary_dim)
    scaling      None, or a dict for contexts longer than the trained one, with `type`:
                 "linear"         factor: positions are divided by it
                 "ntk"            factor: base * factor^(r / (r - 2)), so that the slowest pair alone turns `factor` times slower
                 "yarn"           factor, original_max_position, beta_fast = 32, beta_slow = 1, attention_factor = None: pairs that turn
                                  fewer than beta_slow times over original_max_position are slowed by `factor`, those above beta_fast
                                  kept, a ramp over the pairs between; cos and sin are multiplied by attention_factor, by default
                                  0.1 ln(factor) + 1
                 "by_wavelength"  factor, low_freq_factor, high_freq_factor, original_max_position: the same by wavelength, the ramp in
                                  original_max_position / wavelength between the two factors
    """

    def __init__(self, rotary_dim, base=10000.0, *, scaling=None, device="cuda"):
        _need(int(rotary_dim) >= 16 and int(rotary_dim) % 16 == 0, "rotary_dim: a multiple of 16")
        _need(float(base) > 1.0 and math.isfinite(base), "base must be above 1")
        self.rotary_dim = int(rotary_dim)
        self.inv_freq, self.amplitude = _frequencies(self.rotary_dim, float(base), scaling)
        _need(all(0.0 <= f <= 1.0 for f in self.inv_freq) and math.isfinite(self.amplitude), "scaling: frequencies outside [0, 1]")
        # turns a position, as a 64-bit binary fraction (the scaling by 2^64 is exact)
        bits = [round(f / (2 * math.pi) * 2.0 ** 64) for f in self.inv_freq]
        self.turns = torch.tensor([b - (1 << 64) if b >= 1 << 63 else b for b in bits], dtype=torch.int64, device=device)

    @classmethod
    def of(cls, turns, amplitude=1.0):
        """From a tensor of turns made before (`turns` int64 [rotary_dim / 2])."""
        _need(turns.dtype == torch.int64 and turns.dim() == 1 and turns.shape[0] >= 8 and turns.shape[0] % 8 == 0,
              "turns: int64 [rotary_dim / 2]")
        self = cls.__new__(cls)
        self.rotary_dim, self.inv_freq, self.amplitude, self.turns = 2 * turns.shape[0], None, float(amplitude), turns
        return self


def _frequencies(r, base, scaling):
    """Angles a position of the r/2 pairs (Python floats) and the factor on cos and sin."""
    def powers(b):
        return [b ** (-2.0 * i / r) for i in range(r // 2)]

    freq = powers(base)
    if scaling is None:
        return freq, 1.0
    s = dict(scaling)
    kind, factor = s.pop("type", None), float(s.pop("factor", 1.0))
    _need(factor >= 1.0 and math.isfinite(factor), "scaling: factor must be at least 1")

    def rest(**known):
        _need(set(s) <= set(known), f"scaling: unknown keys {sorted(set(s) - set(known))}")
        for k, v in known.items():
            _need(k in s or v is not None or k == "attention_factor", f"scaling: {k} is missing")
        return [s.get(k, v) for k, v in known.items()]

    if kind == "linear":
        rest()
        return [f / factor for f in freq], 1.0
    if kind == "ntk":
        rest()
        return powers(base * factor ** (r / (r - 2))), 1.0
    if kind == "yarn":
        trained, fast, slow, attention = rest(original_max_position=None, beta_fast=32.0, beta_slow=1.0, attention_factor=None)
        _need(trained > 0 and fast > slow > 0, "scaling: original_max_position > 0 and beta_fast > beta_slow > 0")

        def pair_of(turns):  # the pair that turns this many times over the trained length
            return r * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), r - 1)
        keep = [1.0 - min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0) for i in range(r // 2)]
        amplitude = 0.1 * math.log(factor) + 1.0 if attention is None else float(attention)
        return [f * k + f / factor * (1.0 - k) for f, k in zip(freq, keep)], amplitude
    if kind == "by_wavelength":
        trained, lo, hi = rest(original_max_position=None, low_freq_factor=None, high_freq_factor=None)
        _need(trained > 0 and hi > lo > 0, "scaling: original_max_position > 0 and high_freq_factor > low_freq_factor > 0")
        keep = [min(max((trained * f / (2 * math.pi) - lo) / (hi - lo), 0.0), 1.0) for f in freq]
        return [f * k + f / factor * (1.0 - k) for f, k in zip(freq, keep)], 1.0
    raise ValueError(f"scaling: type {kind!r}: linear, ntk, yarn or by_wavelength expected")


def qk_norm_rope(query, key, positions, rotary, query_out, key_out, *, query_weight=None, key_weight=None, eps=1e-6, layout="half",
                 rope_last=False):
    """RMS norm of every head (where its weight is given) and rotation of `rotary.rotary_dim` of its dims, one pass over the rows.

    query [t, hq, dq], key [t, hk, dk] (or None, with key_out None), positions int32 or int64 [t], rotary a `RotaryFrequencies` or None
    (norm only; positions may then be None); outputs of the inputs' shapes, each its input (in place) or apart from it; weights [dq],
    [dk]. Head dims: multiples of 8 up to 256. `layout`: "half" pairs x[i] with x[i + r/2], "interleaved" x[2i] with x[2i + 1],
    "deinterleave" reads the second and writes the first (what the prologs do to the latent path's rope dims). The rotated dims are
    the head's first, or its last with `rope_last`. Sums and angles in fp32 and wider, one rounding at the end."""
    if _native is not None and type(rotary) is RotaryFrequencies and layout in _LAYOUTS and _native.qk_norm_rope(
            query, key, positions, rotary.turns, query_out, key_out, query_weight, key_weight, eps, _LAYOUTS[layout],
            1 if rope_last else 0, rotary.rotary_dim, rotary.amplitude):
        return None
    q = _rows(query, "query", 3)
    t, hq, dq = q.shape
    qo = _rows(query_out, "query_out", 3)
    _need(qo.shape == q.shape and qo.dtype == q.dtype, "query_out: shape and dtype of query")
    _need((key is None) == (key_out is None), "key and key_out go together")
    k, ko, hk, dk = q, qo, 0, 8
    if key is not None:
        k, ko = _rows(key, "key", 3), _rows(key_out, "key_out", 3)
        hk, dk = k.shape[1], k.shape[2]
        _need(k.shape[0] == t and k.dtype == q.dtype, "key: [t, hk, dk] of the query's dtype")
        _need(ko.shape == k.shape and ko.dtype == k.dtype, "key_out: shape and dtype of key")
    _need(layout in _LAYOUTS, f"layout {layout!r}: half, interleaved or deinterleave expected")
    _need(rotary is None or isinstance(rotary, RotaryFrequencies), "rotary: a RotaryFrequencies or None")
    tensors, wq, wk, pos = [q, qo, k, ko], None, None, None
    if query_weight is not None:
        wq = unwrap(query_weight, "query_weight")
        _need(wq.dtype == q.dtype and tuple(wq.shape) == (dq,), "query_weight: [dq] of the query's dtype")
        tensors.append(wq)
    if key_weight is not None:
        wk = unwrap(key_weight, "key_weight")
        _need(key is not None and wk.dtype == q.dtype and tuple(wk.shape) == (dk,), "key_weight: [dk] of the query's dtype")
        tensors.append(wk)
    if rotary is not None:
        pos = unwrap(positions, "positions")
        _need(pos.dtype in (torch.int32, torch.int64) and tuple(pos.shape) == (t,), "positions: int32 or int64 [t]")
        tensors += [pos, rotary.turns]
    _need(eps >= 0, "eps must not be negative")
    dev = _same_device(tensors)
    strides = (C.c_int64 * 8)(*[_stride(x, i) for x in (q, k, qo, ko) for i in (0, 1)])
    with torch.cuda.device(dev):
        _lib.check(_lib.load().pto_qk_norm_rope(
            q.data_ptr(), k.data_ptr(), pos.data_ptr() if pos is not None else None,
            int(pos is not None and pos.dtype == torch.int64), rotary.turns.data_ptr() if rotary is not None else None,
            wq.data_ptr() if wq is not None else None, wk.data_ptr() if wk is not None else None, qo.data_ptr(), ko.data_ptr(),
            _ROW_DTYPES[q.dtype], t, hq, dq, hk, dk, strides, rotary.rotary_dim if rotary is not None else 0, _LAYOUTS[layout],
            int(bool(rope_last)), rotary.amplitude if rotary is not None else 1.0, float(eps),
            torch.cuda.current_stream(dev).cuda_stream))
    return None


def _cache_form(width, rope, key_nope_2d, key_rope_2d, k_nope_scales, packed_kv_cache):
    """The caches of a write or a read: (split arrays' pointers, scale dtype, packed pointer, rows, tensors)."""
    rows, ptrs, sd, packed, tensors = None, [None] * 3, _lib.PTO_DT_F32, None, []
    if key_nope_2d is not None:
        kn, sc = unwrap(key_nope_2d, "key_nope_2d"), unwrap(k_nope_scales, "k_nope_scales")
        _need(kn.dtype == torch.int8 and kn.numel() % width == 0 and kn.numel() > 0, f"key_nope_2d: int8 [rows, {width}]")
        rows = kn.numel() // width
        _need(sc.dtype in (torch.float32, torch.float16) and sc.numel() == rows * (width // 128),
              f"k_nope_scales: float32 or float16 [rows, {width // 128}]")
        sd = _lib.PTO_DT_F32 if sc.dtype == torch.float32 else _lib.PTO_DT_F16
        tensors += [kn, sc]
        ptrs = [kn.data_ptr(), None, sc.data_ptr()]
        _need(rope == (key_rope_2d is not None), "key_rope_2d goes with the rows' rope dims")
        if rope:
            kr = unwrap(key_rope_2d, "key_rope_2d")
            _need(kr.dtype == torch.bfloat16 and kr.numel() == rows * 64, "key_rope_2d: bfloat16 [rows, 64]")
            tensors.append(kr)
            ptrs[1] = kr.data_ptr()
    else:
        _need(key_rope_2d is None and k_nope_scales is None, "the split caches' three arrays go together")
    if packed_kv_cache is not None:
        pk = unwrap(packed_kv_cache, "packed_kv_cache")
        _need(width == 512, "packed_kv_cache: rows of 512 dims and 64 rope dims")
        _need(pk.dtype == torch.int8 and pk.numel() > 0 and pk.numel() % 656 == 0, "packed_kv_cache: int8 [rows, 656]")
        _need(rows is None or pk.numel() == rows * 656, "packed_kv_cache: as many rows as key_nope_2d")
        rows, packed = pk.numel() // 656, pk.data_ptr()
        tensors.append(pk)
    _need(rows is not None, "no cache: key_nope_2d or packed_kv_cache")
    return ptrs, sd, packed, rows, tensors


def kv_cache_write(key_nope, key_rope, cache_index, key_nope_2d, key_rope_2d, k_nope_scales, *, packed_kv_cache=None):
    """Rows into the quantised paged caches at `cache_index` (int64 [t], distinct; -1: a padding row, not written): int8 with one
    scale per 128 dims, the prologs' arithmetic; rope dims are copied. float16 scales keep their precision for groups whose largest
    magnitude lies between 8e-3 and 8e6; below they lose bits (under 4e-6 the group), above they are infinite.

    key_nope [t, width], width a multiple of 128 (512: latent rows; 128 * hk: the keys or values of hk heads; two heads of 64 share a
    group and its scale); key_rope bfloat16
    [t, 64] or None. Written in place: key_nope_2d int8 [rows, width], key_rope_2d bfloat16 [rows, 64] (None without key_rope),
    k_nope_scales float32 or float16 [rows, width/128], and / or `packed_kv_cache` int8 [rows, 656]: the caches that
    `sparse_flash_attention_quant_d/_p` and `sparse_attention_antiquant_d/_p` read. An index outside the cache is skipped and sets
    PTO_ST_BAD_PAGE in the workspace's status."""
    if _native is not None and _native.kv_cache_write(key_nope, key_rope, cache_index, key_nope_2d, key_rope_2d, k_nope_scales,
                                                      packed_kv_cache):
        return None
    x = _rows(key_nope, "key_nope", 2)
    t, width = x.shape
    _need(width >= 128 and width % 128 == 0, "key_nope: [t, width], width a multiple of 128")
    ci = unwrap(cache_index, "cache_index")
    _need(ci.dtype == torch.int64 and ci.numel() == t, "cache_index: int64 [t]")
    tensors, xr = [x, ci], None
    if key_rope is not None:
        xr = _rows(key_rope, "key_rope", 2)
        _need(x.dtype == torch.bfloat16 and xr.dtype == torch.bfloat16 and tuple(xr.shape) == (t, 64),
              "key_rope: bfloat16 [t, 64] beside bfloat16 key_nope")
        tensors.append(xr)
    _need(packed_kv_cache is None or xr is not None, "packed_kv_cache: its rows have rope dims, key_rope is missing")
    ptrs, sd, packed, rows, caches = _cache_form(width, xr is not None, key_nope_2d, key_rope_2d, k_nope_scales, packed_kv_cache)
    dev = _same_device(tensors + caches)
    with torch.cuda.device(dev):
        ws = _workspace(dev, 256)
        _lib.check(_lib.load().pto_kv_cache_write(
            x.data_ptr(), _stride(x, 0), xr.data_ptr() if xr is not None else None, _stride(xr, 0) if xr is not None else 0,
            ci.data_ptr(), _ROW_DTYPES[x.dtype], t, width, *ptrs, sd, packed, rows, ws.data_ptr(), ws.numel(),
            torch.cuda.current_stream(dev).cuda_stream))
    return None


def kv_cache_read(key_nope_2d, key_rope_2d, k_nope_scales, block_table, cu_seqlens, key_nope_out, key_rope_out, block_size=128, *,
                  first=None, packed_kv_cache=None):
    """Positions of sequences back from the quantised paged caches as contiguous rows: row cu_seqlens[i] + j of the outputs is position
    first[i] + j of sequence i (`first` int32 [b], None: 0), e.g. the earlier context that a chunk's `prompt_attention` needs.

    block_table int32 [b, max_blocks], cu_seqlens int32 [b + 1] (from 0, not decreasing); key_nope_out bfloat16 or float16 [n, width],
    key_rope_out bfloat16 [n, 64] or None (not read); caches as in `kv_cache_write`, one of the two forms. Rows behind the last
    sequence are left as they are. A position without a valid page is written as zeros and sets PTO_ST_BAD_PAGE."""
    if _native is not None and _native.kv_cache_read(key_nope_2d, key_rope_2d, k_nope_scales, block_table, cu_seqlens, key_nope_out,
                                                     key_rope_out, block_size, first, packed_kv_cache):
        return None
    out = _rows(key_nope_out, "key_nope_out", 2)
    n, width = out.shape
    _need(width >= 128 and width % 128 == 0, "key_nope_out: [n, width], width a multiple of 128")
    _need((key_nope_2d is None) != (packed_kv_cache is None), "one cache: key_nope_2d or packed_kv_cache")
    ro = None
    if key_rope_out is not None:
        ro = _rows(key_rope_out, "key_rope_out", 2)
        _need(out.dtype == torch.bfloat16 and ro.dtype == torch.bfloat16 and tuple(ro.shape) == (n, 64),
              "key_rope_out: bfloat16 [n, 64] beside bfloat16 key_nope_out")
    _need(packed_kv_cache is None or out.dtype == torch.bfloat16, "packed_kv_cache: bfloat16 key_nope_out")
    ptrs, sd, packed, rows, tensors = _cache_form(width, key_rope_2d is not None, key_nope_2d, key_rope_2d, k_nope_scales,
                                                  packed_kv_cache)
    _need(ro is None or packed is not None or ptrs[1] is not None, "key_rope_out: key_rope_2d is missing")
    bt, cu = unwrap(block_table, "block_table"), unwrap(cu_seqlens, "cu_seqlens")
    _need(cu.dtype == torch.int32 and cu.dim() == 1 and cu.shape[0] >= 1, "cu_seqlens: int32 [b + 1]")
    b = cu.shape[0] - 1
    _need(bt.dtype == torch.int32 and bt.dim() == 2 and bt.shape[0] == b, "block_table: int32 [b, max_blocks]")
    _need(1 <= int(block_size) < 1 << 31, "block_size must be positive, and a 32-bit number")
    tensors = tensors + [out, bt, cu] + ([ro] if ro is not None else [])
    fs = None
    if first is not None:
        fs = unwrap(first, "first")
        _need(fs.dtype == torch.int32 and tuple(fs.shape) == (b,), "first: int32 [b]")
        tensors.append(fs)
    dev = _same_device(tensors)
    with torch.cuda.device(dev):
        ws = _workspace(dev, 256)
        _lib.check(_lib.load().pto_kv_cache_read(
            *ptrs, sd, packed, rows, bt.data_ptr(), cu.data_ptr(), fs.data_ptr() if fs is not None else None, b, bt.shape[1],
            int(block_size), n, width, out.data_ptr(), _stride(out, 0), ro.data_ptr() if ro is not None else None,
            _stride(ro, 0) if ro is not None else 0, _ROW_DTYPES[out.dtype], ws.data_ptr(), ws.numel(),
            torch.cuda.current_stream(dev).cuda_stream))
    return None


def prompt_attention(query, key, value, cu_seqlens_q, cu_seqlens_k, attention_out, softmax_scale=None, *, causal=True, lse_out=None):
    """Attention of packed sequences over all of their keys: token i of a sequence's lq sees keys j <= i + lk - lq of its lk (all of
    them with causal=False), so a chunk of a prompt comes with its earlier keys in front, and a single token with its whole context.
    Keys and values lie packed, sequence behind sequence: what is in paged caches is read back first (`kv_cache_read`).

    query [tq, hq, dqk], key [tk, hkv, dqk], value [tk, hkv, dv], attention_out [tq, hq, dv]; (dqk, dv) (64, 64), (128, 128) or
    (192, 128) (the latent path after its up-projections); query head h reads key head h / (hq / hkv). cu_seqlens_q, cu_seqlens_k int32
    [b + 1]: where the sequences begin, from 0, not decreasing; rows of the output behind the last sequence are left as they are.
    softmax_scale positive, by default dqk^-0.5. `lse_out` (float32 [hq, tq], optional) receives ln sum exp of the scaled scores, with
    which results over different keys can be joined. A token without a key gets zeros and -inf."""
    if _native is not None and softmax_scale is not None and _native.prompt_attention(
            query, key, value, cu_seqlens_q, cu_seqlens_k, attention_out, softmax_scale, 1 if causal else 0, lse_out):
        return None
    q, k, v, out = _rows(query, "query", 3), _rows(key, "key", 3), _rows(value, "value", 3), _rows(attention_out, "attention_out", 3)
    tq, hq, dqk = q.shape
    tk, hkv, dv = v.shape
    _need(tuple(k.shape) == (tk, hkv, dqk), "key: [tk, hkv, dqk] beside value [tk, hkv, dv]")
    _need((dqk, dv) in ((64, 64), (128, 128), (192, 128)), f"head dims {dqk} / {dv}: 64 / 64, 128 / 128 or 192 / 128 expected")
    _need(hkv >= 1 and hq >= 1 and hq % hkv == 0, "query heads must be a multiple of the key heads")
    _need(tuple(out.shape) == (tq, hq, dv), "attention_out: [tq, hq, dv]")
    _need(q.dtype == k.dtype == v.dtype == out.dtype, "query, key, value and attention_out must share one dtype")
    cq, ck = unwrap(cu_seqlens_q, "cu_seqlens_q"), unwrap(cu_seqlens_k, "cu_seqlens_k")
    _need(cq.dtype == ck.dtype == torch.int32 and cq.dim() == 1 and cq.shape[0] >= 1 and cq.shape == ck.shape,
          "cu_seqlens_q, cu_seqlens_k: int32 [b + 1]")
    scale = dqk ** -0.5 if softmax_scale is None else float(softmax_scale)
    _need(0.0 < scale <= 1e30, "softmax_scale must be positive and finite")
    tensors, lse = [q, k, v, out, cq, ck], None
    if lse_out is not None:
        lse = unwrap(lse_out, "lse_out")
        _need(lse.dtype == torch.float32 and tuple(lse.shape) == (hq, tq), "lse_out: float32 [hq, tq]")
        tensors.append(lse)
    dev = _same_device(tensors)
    b = cq.shape[0] - 1
    if tq == 0 or b == 0:
        return None
    lib = _lib.load()
    nbytes = lib.pto_prompt_attention_workspace_bytes(tq, tk, b, hq, hkv, dv)
    strides = (C.c_int64 * 8)(*[_stride(x, i) for x in (q, k, v, out) for i in (0, 1)])
    with torch.cuda.device(dev):
        ws = _workspace(dev, max(nbytes, 256))
        _lib.check(lib.pto_prompt_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), cq.data_ptr(), ck.data_ptr(), out.data_ptr(),
                                            lse.data_ptr() if lse is not None else None, _ROW_DTYPES[q.dtype], tq, tk, b, hq, hkv,
                                            dqk, dv, strides, scale, int(bool(causal)), ws.data_ptr(), ws.numel(),
                                            torch.cuda.current_stream(dev).cuda_stream))
    return None

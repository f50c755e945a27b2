"""Cached decoding in 8 bits: rows of activations as codes with a scale each, products of them with an 8-bit weight, a key / value cache of
codes and the attention that reads it.

They stand beside ``ops.RMSNorm``, ``ops.Linear`` and ``ops.attention_decode`` for a model that is served: a step of decoding reads every
weight and the whole cache once, so half the bytes are half the time.  The reference has no 8-bit storage (src/dtype.rs:14-21) and its sampling
loop keeps no cache.  Inference only: there are no gradients.  One block of a model, step by step::

    h, rows = q8.rms_norm_add_q8(x, residual, eps)             # the residual stream and what the projection reads
    qkv = q8.linear_q8(rows, w_qkv)                            # w_qkv = q8.quantize_weight_q8(weight), once
    cache.append(k, v, start)                                  # k, v [B, H, T, D]
    o = q8.attention_decode_q8(q, cache, start + T)
    y = q8.linear_q8(q8.quantize_q8(o_rows), w_out)
    u = q8.quantize_q8(up, relu_squared=True)                  # between the products of the MLP

Arithmetic happens in ``libdeers_b200.so``; there is no fallback.  Places and lengths live on the device, so that a captured step of these
operators serves every length; every call allocates its outputs and workspace anew.  A rotation between projection and cache is not among them:
``ops.RotaryPack`` takes one position for the whole batch, so sequences at unlike places are rotated by the caller.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from .errors import DeviceMismatch, DTypeMismatch, LayoutMismatch
from .ops import _DTYPES, _host, _taken, default_scale

BLOCK = _lib.CACHE_BLOCK                      # tokens of a head that share a scale
_CODES = {torch.int8: _lib.I8, torch.float8_e4m3fn: _lib.E4M3}


def _stored(name: str, t: torch.Tensor) -> None:
    if t.dtype not in _DTYPES:
        raise DTypeMismatch(f"{name}: f16 or f32, got {t.dtype}")
    if t.device.type != "cuda":
        raise DeviceMismatch(f"{name}: the op runs on the CUDA device only")


def _code(name: str, dtype: torch.dtype) -> int:
    if dtype not in _CODES:
        raise DTypeMismatch(f"{name}: codes are torch.int8 or torch.float8_e4m3fn, got {dtype}")
    return _CODES[dtype]


class RowsQ8(NamedTuple):
    """Rows [.., C] as 8-bit codes (int8 or e4m3), each standing for ``codes * scale[.., None]``.  Rows of codes start on 16-byte boundaries:
    where C is no multiple of 16 the tensor is a view of padded rows."""
    codes: torch.Tensor
    scale: torch.Tensor

    def values(self) -> torch.Tensor:
        """What the codes stand for, in f32."""
        return self.codes.float() * self.scale[..., None]


def _quantize(name, x, residual, norm, relu_squared, eps, dtype):
    code = _code(name, dtype)
    got = _host.quantize_rows(x, residual, norm, relu_squared, eps, code)
    if got is None:
        if x.dim() < 1 or x.shape[-1] < 1:
            raise LayoutMismatch(f"{name}: rows of at least one element, got {tuple(x.shape)}")
        _stored(name, x)
        if residual is not None:
            if residual.shape != x.shape:
                raise LayoutMismatch(f"{name}: {tuple(residual.shape)} vs {tuple(x.shape)}")
            if residual.dtype != x.dtype:
                raise DTypeMismatch(f"{name}: {residual.dtype} vs {x.dtype}")
            if residual.device != x.device:
                raise DeviceMismatch(f"{name}: {residual.device} vs {x.device}")
            residual = residual.contiguous()
        got = _taken(name, _host.quantize_rows(x.contiguous(), residual, norm, relu_squared, eps, code))
    return got


def rms_norm_add_q8(x, residual=None, eps: float = 1e-5, dtype: torch.dtype = torch.int8):
    """``h = x + residual`` and ``RMSNorm::forward`` of it (src/nn.rs:244-251) over the last axis, the normalised rows as 8-bit codes: returns
    (h, RowsQ8).  x and residual f16 or f32 of one shape; h has their type (and is x itself without a residual).  The norm has no gain, as
    the reference's: one belongs into the rows of the weight that follows.

    scale = max|y| / 127 (int8) or / 448 (e4m3), codes the nearest to y / scale.  A row of zeros has scale 0; a row that holds an
    infinity or a NaN has scale NaN and codes 0."""
    h, codes, scale = _quantize("rms_norm_add_q8", x, residual, True, False, eps, dtype)
    return (x if h is None else h), RowsQ8(codes, scale)


def quantize_q8(x, dtype: torch.dtype = torch.int8, relu_squared: bool = False) -> RowsQ8:
    """Rows of x (f16 or f32) over the last axis as 8-bit codes with a scale each, or those of ``relu(x)^2``
    (src/models/gpt.rs:194-196).  Scales and codes as for ``rms_norm_add_q8``."""
    _, codes, scale = _quantize("quantize_q8", x, None, False, relu_squared, 0.0, dtype)
    return RowsQ8(codes, scale)


def quantize_weight_q8(weight, dtype: torch.dtype = torch.int8) -> RowsQ8:
    """A ``Linear`` weight [in_features, out_features] laid out for ``linear_q8``, once: codes [out_features, in_features], a scale for every
    output channel."""
    if weight.dim() != 2:
        raise LayoutMismatch(f"quantize_weight_q8: a weight is [in_features, out_features], got {tuple(weight.shape)}")
    return quantize_q8(weight.t().contiguous(), dtype)


def linear_q8(rows: RowsQ8, weight: RowsQ8, out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """``x.matmul(weight)`` of ``Linear::forward`` (src/nn.rs:184-190) on codes: [.., in_features] times a weight of ``quantize_weight_q8``
    (codes of the same type) to [.., out_features], f16 or f32: the sum times the product of both scales.  int8 sums are exact (in_features < 131072); e4m3 sums
    are f32 whose additions the tensor core cuts off (off by up to 2^-18.7 of the summands' sizes at 4096 in_features where all have one sign, 2^-23.6
    with random signs), which f16 hides and f32 does not."""
    if out_dtype not in _DTYPES:
        raise DTypeMismatch(f"linear_q8: f16 or f32 comes out, got {out_dtype}")
    out = _DTYPES[out_dtype]
    got = _host.gemm_q8(rows[0], rows[1], weight[0], weight[1], out)
    if got is not None:
        return got
    (a, sa), (b, sb) = rows, weight
    _code("linear_q8", a.dtype)
    if b.dim() != 2 or a.dim() < 1 or a.shape[-1] != b.shape[1] or 0 in b.shape:
        raise LayoutMismatch(f"linear_q8: rows {tuple(a.shape)} vs weight {tuple(b.shape)}")
    if sa.shape != a.shape[:-1] or sb.shape != b.shape[:1]:
        raise LayoutMismatch(f"linear_q8: scales {tuple(sa.shape)} of rows {tuple(a.shape)}, {tuple(sb.shape)} of weight {tuple(b.shape)}")
    if b.dtype != a.dtype:
        raise DTypeMismatch(f"linear_q8: {a.dtype} vs {b.dtype}")
    if sa.dtype != torch.float32 or sb.dtype != torch.float32:
        raise DTypeMismatch(f"linear_q8: scales are f32, got {sa.dtype} and {sb.dtype}")
    if a.device.type != "cuda":
        raise DeviceMismatch("linear_q8: the op runs on the CUDA device only")
    for t in (sa, b, sb):
        if t.device != a.device:
            raise DeviceMismatch(f"linear_q8: {t.device} vs {a.device}")
    return _taken("linear_q8", _host.gemm_q8(_padded(a.reshape(-1, a.shape[-1])), sa.reshape(-1).contiguous(), _padded(b), sb.contiguous(), out)).reshape(*a.shape[:-1], b.shape[0])


def _padded(codes: torch.Tensor) -> torch.Tensor:
    """Rows of codes on 16-byte boundaries: a copy where they are not."""
    if codes.stride(1) == 1 and codes.stride(0) % 16 == 0 and codes.stride(0) >= codes.shape[1] and codes.data_ptr() % 16 == 0:
        return codes
    K = codes.shape[1]
    held = torch.empty((codes.shape[0], (K + 15) // 16 * 16), dtype=codes.dtype, device=codes.device)[:, :K]
    return held.copy_(codes)


class CacheQ8:
    """Keys and values of a batch of sequences as e4m3 codes [B, H, capacity, D] with an f32 scale for every ``BLOCK`` tokens of a head.  D is a
    multiple of 16, at most 256.  How many rows a sequence has is the caller's to keep (one int32 tensor serves all layers)."""

    def __init__(self, k, v, k_scale, v_scale):
        """Takes tensors that hold such a cache (``CacheQ8.new`` makes an empty one); views of larger ones are used in place."""
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        if _host.cache_taken(k, v, k_scale, v_scale):
            return
        if k.dim() != 4 or v.shape != k.shape:
            raise LayoutMismatch(f"CacheQ8: codes are [B, H, capacity, D], got {tuple(k.shape)} and {tuple(v.shape)}")
        blocks = (*k.shape[:2], (k.shape[2] + BLOCK - 1) // BLOCK)
        if tuple(k_scale.shape) != blocks or tuple(v_scale.shape) != blocks:
            raise LayoutMismatch(f"CacheQ8: scales are {blocks}, got {tuple(k_scale.shape)} and {tuple(v_scale.shape)}")
        if 0 in k.shape or k.shape[3] % 16 or k.shape[3] > 256:
            raise LayoutMismatch(f"CacheQ8: head dims are multiples of 16 up to 256, got codes {tuple(k.shape)}")
        for t in (k, v):
            if t.dtype != torch.float8_e4m3fn:
                raise DTypeMismatch(f"CacheQ8: codes are torch.float8_e4m3fn, got {t.dtype}")
            if t.stride(3) != 1 or t.data_ptr() % 16 or any(t.stride(i) % 16 and t.shape[i] > 1 for i in range(3)):
                raise LayoutMismatch("CacheQ8: rows of codes are contiguous and start on 16-byte boundaries")
        for t in (k_scale, v_scale):
            if t.dtype != torch.float32:
                raise DTypeMismatch(f"CacheQ8: scales are f32, got {t.dtype}")
            if t.shape[2] > 1 and t.stride(2) != 1:
                raise LayoutMismatch("CacheQ8: the scales of a head are contiguous")
        if k.device.type != "cuda":
            raise DeviceMismatch("CacheQ8: the cache lives on the CUDA device")
        for t in (v, k_scale, v_scale):
            if t.device != k.device:
                raise DeviceMismatch(f"CacheQ8: {t.device} vs {k.device}")

    @classmethod
    def new(cls, batch: int, heads: int, capacity: int, head_dim: int, device="cuda") -> "CacheQ8":
        if min(batch, heads, capacity, head_dim) < 1 or head_dim % 16 or head_dim > 256:
            raise LayoutMismatch(f"CacheQ8: head dims are multiples of 16 up to 256, got {(batch, heads, capacity, head_dim)}")
        if torch.device(device).type != "cuda":
            raise DeviceMismatch("CacheQ8: the cache lives on the CUDA device")
        codes = [torch.zeros((batch, heads, capacity, head_dim), dtype=torch.float8_e4m3fn, device=device) for _ in range(2)]
        scales = [torch.zeros((batch, heads, (capacity + BLOCK - 1) // BLOCK), dtype=torch.float32, device=device) for _ in range(2)]
        return cls(*codes, *scales)

    def append(self, k, v, start: torch.Tensor, count: Optional[torch.Tensor] = None) -> None:
        """Row t of k and v [B, H, T, D] (f16 or f32) becomes row ``start[b] + t`` of sequence b, for t < ``count[b]`` (all T without it); start and
        count are int32 on the device.  A block of ``BLOCK`` rows keeps one scale: the largest its rows have needed since it was begun; where new
        rows raise it, the block's earlier rows are rounded again.  Codes behind the last new row stay as they are, but not always their block's scale: a
        sequence ends with its newest row.  An infinity or a NaN is kept as NaN.  Rows beyond the capacity, and all rows of a sequence whose
        start is negative, are left out, and ``Context.sync`` reports them; other operators run all the same."""
        if _host.cache_append(self.k, self.v, self.k_scale, self.v_scale, k, v, start, count) is not None:
            return
        B, H, cap, D = self.k.shape
        for t in (k, v):
            if t.dim() != 4 or (t.shape[0], t.shape[1], t.shape[3]) != (B, H, D) or t.shape != k.shape or t.shape[2] > cap:
                raise LayoutMismatch(f"CacheQ8.append: rows {tuple(t.shape)} into a cache {(B, H, cap, D)}")
            _stored("CacheQ8.append", t)
            if t.dtype != k.dtype:
                raise DTypeMismatch(f"CacheQ8.append: {t.dtype} vs {k.dtype}")
            if t.device != self.k.device:
                raise DeviceMismatch(f"CacheQ8.append: {t.device} vs {self.k.device}")
        start, count = _places("CacheQ8.append", start, self.k), count if count is None else _places("CacheQ8.append", count, self.k)
        _taken("CacheQ8.append", _host.cache_append(self.k, self.v, self.k_scale, self.v_scale, k.contiguous(), v.contiguous(), start, count))


def _places(name: str, t: torch.Tensor, of: torch.Tensor) -> torch.Tensor:
    if t.dtype != torch.int32:
        raise DTypeMismatch(f"{name}: places and lengths are int32, got {t.dtype}")
    if tuple(t.shape) != (of.shape[0],):
        raise LayoutMismatch(f"{name}: one place or length for each of {of.shape[0]} sequences, got {tuple(t.shape)}")
    if t.device != of.device:
        raise DeviceMismatch(f"{name}: {t.device} vs {of.device}")
    return t.contiguous()


def attention_decode_q8(q, cache: CacheQ8, lengths: torch.Tensor, scale: Optional[float] = None, causal: bool = True, want_lse: bool = False):
    """``attention_decode`` over a cache of codes: q [B, Hq, Tq, D] (f16 or f32; at most 128 rows; Hq a multiple of the cache's heads, head h reads head
    ``h // (Hq / H)``), ``lengths[b]`` rows of sequence b, the Tq newest of which belong to the queries.  Returns o [B, Hq, Tq, D] (and lse
    [B, Hq, Tq]).  A row that sees no key has o = 0 and lse = -inf; what lies behind a sequence's last row is not read.  Of a batch padded at
    the back to T rows the lengths are ``start + T``: query t then sees rows up to its own, and what the padding's queries see is nobody's.
    The cache is read once for every 8 or 16 query rows of a head's group.  Lengths outside of the capacity are taken as the nearest inside, and
    ``Context.sync`` reports them; other operators run all the same."""
    if scale is None and q.dim() == 4 and q.shape[3]:
        scale = default_scale(q.shape[3])
    held = (cache.k, cache.v, cache.k_scale, cache.v_scale)
    got = _host.attn_decode_q8(*held, q, lengths, scale, causal, want_lse) if scale is not None else None
    if got is not None:
        return got
    B, H, cap, D = cache.k.shape
    if q.dim() != 4 or q.shape[0] != B or q.shape[3] != D or q.shape[1] % H or 0 in q.shape or q.shape[2] > cap:
        raise LayoutMismatch(f"attention_decode_q8: q {tuple(q.shape)} with a cache {(B, H, cap, D)}")
    _stored("attention_decode_q8", q)
    if q.device != cache.k.device:
        raise DeviceMismatch(f"attention_decode_q8: {q.device} vs {cache.k.device}")
    lengths = _places("attention_decode_q8", lengths, cache.k)
    return _taken("attention_decode_q8", _host.attn_decode_q8(*held, q if q.stride(3) == 1 else q.contiguous(), lengths, scale, causal, want_lse))

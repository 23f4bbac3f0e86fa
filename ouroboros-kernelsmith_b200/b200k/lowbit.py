"""Low-precision serving ops: 8-bit activations, a 4-bit paged key/value
cache with the attention that reads it, and products with 4-bit weights.

    h, q, scale = add_rmsnorm_quant(x, residual, w)          # 8-bit rows
    qkv = w4_matmul(q, w_qkv, x_scale=scale, out_dtype=...)  # 4-bit weights
    kv_cache_write(cache, k, v, slots)                       # 4-bit cache
    o = cache_attention(q, cache, page_table, lengths)       # reads it

The calling convention is that of b200k.ops: CUDA tensors, fresh outputs (the
cache is the one operand that is written), the current stream, no host
synchronisation, TypeError / ValueError before a launch, B200KError when one
fails.  Indices that only the device knows (slots, pages, lengths) are checked
by the kernels: a slot outside the pool is not written, and what cannot be
read becomes NaN in the rows that asked for it.

These ops serve: their results carry no gradient, also where an input requires
one.  What is trained through a product with frozen 4-bit weights needs that
product's gradient from elsewhere.
"""
from __future__ import annotations

import math

import torch

from . import _lib as L
from .ops import _DT, _cuda, _dev, _dtype_id, _p, _raw_stream, _rows, _same_dtype, _vec

__all__ = ["rmsnorm_quant", "add_rmsnorm_quant", "KVCache4", "kv_cache_write", "kv_cache_read",
           "cache_attention", "W4Weight", "w4_pack", "w4_quantize", "w4_matmul"]

_Q8 = {torch.int8: L.I8, torch.float8_e4m3fn: L.E4M3}
_DT16 = {torch.float16: L.F16, torch.bfloat16: L.BF16}


_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _call(dev, fn, name, *args):
    """fn(*args, stream) on dev's current stream, with dev made current; raises
    B200KError when it fails.  The usual case, dev already current, takes no
    context manager: these calls are short beside the host's part of them."""
    if _raw_stream is not None and _device() == dev.index:
        st = fn(*args, _raw_stream(dev.index))
    else:
        with _dev(dev) as stream:
            st = fn(*args, stream)
    L.check(st, name)


def _new(m, n, dtype, dev):
    """A fresh contiguous [m, n] (empty_strided takes the least time on the host)."""
    return torch.empty_strided((m, n), (n, 1), dtype=dtype, device=dev)


def _matrix(t, n):
    """_rows, which a contiguous matrix need not pay for."""
    return (t, n) if t.dim() == 2 and t.is_contiguous() and t.shape[1] == n else _rows(t, n)


def _dt16(t: torch.dtype, what: str) -> int:
    try:
        return _DT16[t]
    except KeyError:
        raise TypeError(f"b200k: {what} must be float16 or bfloat16, got {t}")


# --------------------------------------------------------------------------
# RMS norm with an 8-bit output (b2k_norm_quant)
def _norm_quant(x, residual, w, dtype, group, eps):
    dev = _cuda(x, residual, w)
    _same_dtype(x, residual, w)
    dt = _dtype_id(x)
    try:
        qt = _Q8[dtype]
    except KeyError:
        raise TypeError(f"b200k: quantised dtype must be int8 or float8_e4m3fn, got {dtype}")
    if group not in (None, 32, 64, 128):
        raise ValueError(f"b200k: group must be None, 32, 64 or 128, got {group}")
    n = x.shape[-1]
    x2, ldx = _matrix(x, n)
    m = x2.shape[0]
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"b200k: residual shape {tuple(residual.shape)} != {tuple(x.shape)}")
        r2, ldr = _matrix(residual, n)
        h = _new(m, n, x.dtype, dev)
    else:
        r2, ldr, h = None, 0, None
    w1 = _vec(w, n, "weight")
    ns = 1 if group is None else (n + group - 1) // group
    q = _new(m, n, dtype, dev)
    scale = _new(m, ns, torch.float32, dev)
    _call(dev, L.lib.b2k_norm_quant, "b2k_norm_quant", _p(x2), ldx, _p(r2), ldr, _p(w1), _p(h), n,
          _p(q), n, _p(scale), ns, m, n, dt, qt, group or 0, eps)
    if x.dim() != 2:
        q = q.view(x.shape)
        scale = scale.view(x.shape[:-1] + (ns,))
        h = h.view(x.shape) if h is not None else None
    return h, q, scale


def rmsnorm_quant(x, w, *, dtype: torch.dtype = torch.int8, group: int | None = None,
                  eps: float = 1e-6):
    """RMS norm of x's rows, times w, in 8 bits: (q, scale) with
    y = (x*w) * rsqrt(mean(x^2) + eps) in fp32, scale = max|y| / Q and
    q = round(y * Q / max|y|), Q = 127 (int8) or 448 (float8_e4m3fn).  scale is
    fp32, [..., 1] per row or [..., ceil(n / group)] per `group` (32, 64, 128)
    columns; a maximum below 1e-30 gives scale 0 and zeros, a NaN a NaN scale.
    int8 rows with a scale per row are what dequant_int8 reads."""
    _, q, scale = _norm_quant(x, None, w, dtype, group, eps)
    return q, scale


def add_rmsnorm_quant(x, residual, w, *, dtype: torch.dtype = torch.int8,
                      group: int | None = None, eps: float = 1e-6):
    """rmsnorm_quant of h = T(x + residual): (h, q, scale), h the residual
    stream for the next block (as in fused_add_norm)."""
    return _norm_quant(x, residual, w, dtype, group, eps)


class _Handle:
    """What the kernels are called with is taken from the tensors once, when the
    handle is made, so its attributes stay what they are."""

    __slots__ = ()

    def _fill(self, **values):
        for name, value in values.items():
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError(f"b200k: {type(self).__name__}.{name} cannot be set; make a new "
                             f"{type(self).__name__}")


# --------------------------------------------------------------------------
# the 4-bit cache (b2k_kv4_write, b2k_kv4_read, b2k_kv4_attention)
class KVCache4(_Handle):
    """A paged key/value cache in 4 bits: `data`, uint8
    [pages, kv_heads, page_size / 16, 16 * (D + 8 * D / group)].

    Each 16 tokens of a head lie together: the keys' rows of D / 2 bytes,
    their (s, lo) pairs of float16 for every `group` dimensions, the values'
    rows, their pairs.  A value row holds dimension i in nibble i (low bits
    first); a key row holds words of eight dimensions, word j of quarter c
    being dimensions 32 j + 8 c .. + 7.  A group stands for lo + n * s with
    s = f16((max - min) / 15), lo = f16(min), n = round((x - lo) / s) in 0..15;
    magnitudes above 65408 saturate and a NaN makes its group NaN.  Slot
    t = page * page_size + offset names a token."""

    __slots__ = ("data", "pages", "kv_heads", "page_size", "head_dim", "group", "_args", "_sizes")

    def __init__(self, data: torch.Tensor, head_dim: int, group: int = 32):
        if head_dim not in (64, 128, 256):
            raise ValueError(f"b200k: head_dim must be 64, 128 or 256, got {head_dim}")
        if group not in (32, 64, 128) or group > head_dim:
            raise ValueError(f"b200k: group must be 32, 64 or 128 and at most head_dim, got {group}")
        if not isinstance(data, torch.Tensor) or not data.is_cuda:
            raise ValueError("b200k: every operand must be a CUDA tensor (no CPU path exists)")
        if data.dtype != torch.uint8:
            raise TypeError(f"b200k: cache data must be uint8, got {data.dtype}")
        micro = 16 * (head_dim + 8 * head_dim // group)
        if data.dim() != 4 or data.shape[1] < 1 or data.shape[2] < 1 or data.shape[3] != micro \
                or not data.is_contiguous():
            raise ValueError("b200k: cache data must be contiguous [pages, kv_heads, "
                             f"page_size / 16, {micro}], got {tuple(data.shape)}")
        pages, kv_heads, page_size = data.shape[0], data.shape[1], 16 * data.shape[2]
        self._fill(data=data, pages=pages, kv_heads=kv_heads, page_size=page_size,
                   head_dim=head_dim, group=group,
                   _args=(data.data_ptr(), pages, kv_heads, page_size, head_dim, group),
                   _sizes={})  # workspace bytes of cache_attention by (B, Sq, H)

    @classmethod
    def zeros(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, group: int = 32,
              device="cuda") -> "KVCache4":
        """A pool of `pages` pages of `page_size` (a multiple of 16) tokens."""
        if page_size < 16 or page_size % 16:
            raise ValueError(f"b200k: page_size must be a multiple of 16, got {page_size}")
        if group not in (32, 64, 128):
            raise ValueError(f"b200k: group must be 32, 64 or 128, got {group}")
        return cls(torch.zeros((pages, kv_heads, page_size // 16,
                                16 * (head_dim + 8 * head_dim // group)),
                               dtype=torch.uint8, device=device), head_dim, group)


def _check_cache(cache):
    if not isinstance(cache, KVCache4):
        raise TypeError(f"b200k: expected a KVCache4, got {type(cache).__name__}")


def _check_slots(slots, n):
    if slots.dtype != torch.int64:
        raise TypeError(f"b200k: slots must be int64, got {slots.dtype}")
    if n is not None and slots.numel() != n:
        raise ValueError(f"b200k: {slots.numel()} slots for {n} tokens")
    return slots if slots.dim() == 1 and slots.is_contiguous() else slots.reshape(-1).contiguous()


def kv_cache_write(cache: KVCache4, k, v, slots) -> None:
    """Quantises the keys and values k, v [..., kv_heads, D] (any strides, unit
    innermost) of new tokens into the cache's `slots` (int64, one per token,
    distinct).  A negative slot is padding and is skipped, as is one past the
    pool."""
    _check_cache(cache)
    dev = _cuda(cache.data, k, v, slots)
    _same_dtype(k, v)
    dt = _dt16(k.dtype, "k and v")
    hk, d = cache.kv_heads, cache.head_dim
    for t in (k, v):
        if t.shape[-2:] != (hk, d):
            raise ValueError(f"b200k: k and v must be [..., {hk}, {d}], got {tuple(t.shape)}")
    if k.shape != v.shape:
        raise ValueError(f"b200k: k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    if k.dim() != 3:
        k, v = k.reshape(-1, hk, d), v.reshape(-1, hk, d)
    if k.stride(2) != 1:
        k = k.contiguous()
    if v.stride(2) != 1:
        v = v.contiguous()
    n = k.shape[0]
    s1 = _check_slots(slots, n)
    (ldk, hdk, _), (ldv, hdv, _) = k.stride(), v.stride()
    _call(dev, L.lib.b2k_kv4_write, "b2k_kv4_write", k.data_ptr(), ldk, hdk, v.data_ptr(), ldv, hdv,
          s1.data_ptr(), n, *cache._args, dt)


def kv_cache_read(cache: KVCache4, slots, *, dtype: torch.dtype = torch.bfloat16):
    """The keys and values that the cache's `slots` (int64, any shape) stand
    for: (k, v) of `dtype` (float16 or bfloat16), slots.shape + (kv_heads, D).
    A negative slot reads zeros, one past the pool NaN."""
    _check_cache(cache)
    dev = _cuda(cache.data, slots)
    dt = _dt16(dtype, "dtype")
    s1 = _check_slots(slots, None)
    k = torch.empty((*slots.shape, cache.kv_heads, cache.head_dim), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    _call(dev, L.lib.b2k_kv4_read, "b2k_kv4_read", *cache._args, s1.data_ptr(), s1.shape[0],
          k.data_ptr(), v.data_ptr(), dt)
    return k, v


def cache_attention(q, cache: KVCache4, page_table, lengths, *, scale: float | None = None,
                    causal: bool = True, return_lse: bool = False):
    """Attention of q [B, Sq, H, D] over the cached tokens of B sequences.
    page_table int32 [B, W]: the pages of each sequence in order (entries past
    its length are not read); lengths int32 [B]: its tokens in the cache, the
    Sq new ones included.  H is a multiple of the cache's heads; head h reads
    h // (H // kv_heads).  With `causal`, query i sees tokens up to
    lengths - Sq + i; a row that sees none is zeros (log-sum -inf).  scale
    defaults to D ** -0.5.  Returns o [B, Sq, H, D] in q's dtype, and with
    return_lse also the log of the sum of exponentials, fp32 [B, H, Sq].  A
    length beyond the table gives NaN for its sequence; a page outside the pool
    among the tokens read for the rows that see it, and for rows computed with
    them; a value that is not finite in the dimensions of its group, for the rows
    that see its token.  No gradient."""
    _check_cache(cache)
    dev = _cuda(q, cache.data, page_table, lengths)
    dt = _dt16(q.dtype, "q")
    if q.dim() != 4 or q.shape[3] != cache.head_dim:
        raise ValueError(f"b200k: q must be [B, Sq, H, {cache.head_dim}], got {tuple(q.shape)}")
    b, sq, h, d = q.shape
    hk = cache.kv_heads
    if h % hk:
        raise ValueError(f"b200k: {h} heads are no multiple of the cache's {hk}")
    if page_table.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise TypeError("b200k: page_table and lengths must be int32")
    if page_table.dim() != 2 or page_table.shape[0] != b or lengths.shape != (b,):
        raise ValueError(f"b200k: page_table {tuple(page_table.shape)} and lengths "
                         f"{tuple(lengths.shape)} do not match {b} sequences")
    if q.stride(3) != 1:
        q = q.contiguous()
    page_table, lengths = page_table.contiguous(), lengths.contiguous()
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((b, h, sq), dtype=torch.float32, device=dev) if return_lse else None
    nws = cache._sizes.get((b, sq, h))
    if nws is None:
        with _dev(dev):
            nws = L.lib.b2k_kv4_attention_workspace(b, sq, h, hk, d)
        cache._sizes[(b, sq, h)] = nws
    ws = _new(1, nws, torch.uint8, dev) if nws > 0 else None
    _call(dev, L.lib.b2k_kv4_attention, "b2k_kv4_attention", q.data_ptr(), *q.stride()[:3], o.data_ptr(),
          _p(lse), *cache._args, page_table.data_ptr(), page_table.shape[1], lengths.data_ptr(), b, sq, h,
          d ** -0.5 if scale is None else scale, 1 if causal else 0, dt, _p(ws), nws)
    return (o, lse) if return_lse else o


# --------------------------------------------------------------------------
# 4-bit weights (b2k_w4_pack, b2k_w4_quantize, b2k_w4_matmul)
class W4Weight(_Handle):
    """Weights [n, k] in 4 bits, laid out for w4_matmul: w = scale * (i - zero)
    for integers i in 0..15, scale and zero (8 without zeros) per row and group
    of 32, 64 or 128 columns.

    tiles uint8 [ceil(n/16), ceil(k/128), 16, 64]: rows of 128 columns, word j
    (32 bits, the first column in the low ones) of quarter c holding columns
    32 j + 8 c .. + 7; scales and zeros (float16 or bfloat16)
    [ceil(n/16), ceil(k/128), 128 / group, 16].  w4_pack and w4_quantize
    make them."""

    __slots__ = ("tiles", "scales", "zeros", "n", "k", "group", "_args", "_sizes")

    def __init__(self, tiles, scales, zeros, n: int, k: int):
        _cuda(tiles, scales, zeros)
        if tiles.dtype != torch.uint8:
            raise TypeError(f"b200k: tiles must be uint8, got {tiles.dtype}")
        st = _dt16(scales.dtype, "scales")
        nt, kt = (n + 15) // 16, (k + 127) // 128
        if n < 0 or k < 0 or tuple(tiles.shape) != (nt, kt, 16, 64):
            raise ValueError(f"b200k: tiles of [{n}, {k}] must be {(nt, kt, 16, 64)}, got "
                             f"{tuple(tiles.shape)}")
        if scales.dim() != 4 or scales.shape[2] not in (1, 2, 4) or \
                tuple(scales.shape) != (nt, kt, scales.shape[2], 16):
            raise ValueError(f"b200k: scales of [{n}, {k}] must be [{nt}, {kt}, 128 / group, 16], "
                             f"got {tuple(scales.shape)}")
        if zeros is not None and (zeros.shape != scales.shape or zeros.dtype != scales.dtype):
            raise ValueError("b200k: zeros must have the scales' shape and dtype")
        for t in (tiles, scales, zeros):
            if t is not None and (not t.is_contiguous() or t.data_ptr() % 16):
                raise ValueError("b200k: tiles, scales and zeros must be contiguous and 16-byte "
                                 "aligned")
        group = 128 // scales.shape[2]
        self._fill(tiles=tiles, scales=scales, zeros=zeros, n=n, k=k, group=group,
                   _args=(_p(tiles), _p(scales), _p(zeros), st, group),
                   _sizes={})  # workspace bytes of w4_matmul by (rows, x's type)


def _w4_empty(n, k, group, stype, with_zeros, dev):
    nt, kt = (n + 15) // 16, (k + 127) // 128
    tiles = torch.empty((nt, kt, 16, 64), dtype=torch.uint8, device=dev)
    scales = torch.empty((nt, kt, 128 // group, 16), dtype=stype, device=dev)
    return tiles, scales, torch.empty_like(scales) if with_zeros else None


def _check_group(group):
    if group not in (32, 64, 128):
        raise ValueError(f"b200k: group must be 32, 64 or 128, got {group}")


def w4_pack(q, scales, zeros=None, *, group: int = 128) -> W4Weight:
    """Lays out given 4-bit weights: q uint8 [n, k] of integers 0..15, scales
    (and zeros) float16 or bfloat16 [n, ceil(k / group)]."""
    dev = _cuda(q, scales, zeros)
    _check_group(group)
    if q.dtype != torch.uint8 or q.dim() != 2:
        raise TypeError(f"b200k: q must be a uint8 matrix, got {q.dtype} {tuple(q.shape)}")
    st = _dt16(scales.dtype, "scales")
    n, k = q.shape
    want = (n, (k + group - 1) // group)
    if tuple(scales.shape) != want:
        raise ValueError(f"b200k: scales must be {want}, got {tuple(scales.shape)}")
    if zeros is not None and (zeros.shape != scales.shape or zeros.dtype != scales.dtype):
        raise ValueError("b200k: zeros must have the scales' shape and dtype")
    q, scales = q.contiguous(), scales.contiguous()
    zeros = None if zeros is None else zeros.contiguous()
    out = _w4_empty(n, k, group, scales.dtype, zeros is not None, dev)
    with _dev(dev) as stream:
        L.check(L.lib.b2k_w4_pack(_p(q), k, _p(scales), _p(zeros), want[1], n, k, group, st,
                                  _p(out[0]), _p(out[1]), _p(out[2]), stream), "b2k_w4_pack")
    return W4Weight(*out, n, k)


def w4_quantize(w, *, group: int = 128, zeros: bool = False,
                scale_dtype: torch.dtype = torch.float16) -> W4Weight:
    """Rounds weights [n, k] to 4 bits.  Without zeros a group's scale is
    max|w| / 7 and its integers round(w / scale) + 8 in 1..15; with them its
    range, widened to hold 0, is divided into 15 steps and the zero is the
    integer that stands for 0.  Integers go by the scale as rounded to
    scale_dtype."""
    dev = _cuda(w)
    dt = _dtype_id(w)
    _check_group(group)
    st = _dt16(scale_dtype, "scale_dtype")
    if w.dim() != 2:
        raise ValueError(f"b200k: w must be a matrix, got {tuple(w.shape)}")
    n, k = w.shape
    w2, ldw = _rows(w, k)
    out = _w4_empty(n, k, group, scale_dtype, zeros, dev)
    with _dev(dev) as stream:
        L.check(L.lib.b2k_w4_quantize(_p(w2), ldw, n, k, dt, group, st, _p(out[0]), _p(out[1]),
                                      _p(out[2]), stream), "b2k_w4_quantize")
    return W4Weight(*out, n, k)


def w4_matmul(x, weight: W4Weight, *, x_scale=None, out_dtype: torch.dtype | None = None):
    """x [..., k] times 4-bit weights: y [..., n] = x W^T with fp32 sums.  x is
    float32 / float16 / bfloat16, or int8 / float8_e4m3fn with fp32 x_scale
    [..., 1] or [..., ceil(k / g)] for groups of g = 32, 64 or 128 columns, a
    multiple of the weight's group (what rmsnorm_quant returns).  out_dtype
    defaults to x's dtype (bfloat16 for 8-bit x).  Meant for few rows: the
    weights are read once for every 32 of them (8 of float32, whose products keep
    float32's precision; those of 16-bit and 8-bit x are good to about 2^-17 of the
    result beside columns 20 to 100 times the others).  A row that holds an infinity
    or a NaN comes out NaN.  No gradient, neither to x nor to the weights."""
    if not isinstance(weight, W4Weight):
        raise TypeError(f"b200k: expected a W4Weight, got {type(weight).__name__}")
    dev = _cuda(x, weight.tiles, x_scale)
    n, k, group = weight.n, weight.k, weight.group
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"b200k: x {tuple(x.shape)} does not end in {k} columns")
    if x.numel():
        x2, ldx = _matrix(x, k)
        m = x2.shape[0]
    else:  # no rows, or no columns
        x2, ldx, m = x, k, math.prod(x.shape[:-1])
    xg, ldxs, xs = 0, 0, None
    if x.dtype in _Q8:
        xt = _Q8[x.dtype]
        if x_scale is None:
            raise ValueError("b200k: x of 8 bits needs x_scale")
        if x_scale.dtype != torch.float32:
            raise TypeError(f"b200k: x_scale must be float32, got {x_scale.dtype}")
        ns = x_scale.shape[-1] if x_scale.dim() else 1
        if x_scale.numel() != m * ns or (x_scale.dim() > 1 and x_scale.shape[:-1] != x.shape[:-1]):
            raise ValueError(f"b200k: x_scale {tuple(x_scale.shape)} does not match x "
                             f"{tuple(x.shape)}")
        if ns != 1:
            xg = next((g for g in (32, 64, 128) if (k + g - 1) // g == ns), -1)
            if xg < 0 or xg % group:
                raise ValueError(f"b200k: x_scale has {ns} groups for {k} columns: expected one, "
                                 f"or groups of a multiple of {group} up to 128")
        xs = x_scale if x_scale.is_contiguous() else x_scale.contiguous()
        ldxs = ns
        out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
    else:
        xt = _dtype_id(x)
        if x_scale is not None:
            raise ValueError("b200k: x_scale goes with x of 8 bits")
        out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in _DT:
        raise TypeError(f"b200k: unsupported out_dtype {out_dtype}")
    y = _new(m, n, out_dtype, dev)
    nws = weight._sizes.get((m, xt))
    if nws is None:
        with _dev(dev):
            nws = L.lib.b2k_w4_matmul_workspace(m, n, k, group, xt)
        weight._sizes[(m, xt)] = nws
    ws = _new(1, nws, torch.uint8, dev) if nws > 0 else None
    _call(dev, L.lib.b2k_w4_matmul, "b2k_w4_matmul", x2.data_ptr(), ldx, xt, _p(xs), ldxs, xg,
          *weight._args, m, n, k, y.data_ptr(), n, _DT[out_dtype], _p(ws), nws)
    return y if x.dim() == 2 else y.view(x.shape[:-1] + (n,))

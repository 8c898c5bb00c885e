"""Operators of a transformer served in low precision: linear layers in 8-bit floating point with one
scale per block of 128, norms of queries and keys with the rotation of their positions, and attention
over a paged cache of keys and values held in 4 bits.

Tensors are CUDA tensors of fp32, fp16 or bf16, all of a call on one device; a call is enqueued on that
device's current stream.  Sums, statistics and softmax are fp32, the result is rounded once; what
`kv4_attention` holds in fewer bits its docstring says.  There is no backward pass and no
forward-mode derivative: inputs that ask for gradients are refused while gradients are recorded, inputs with
a tangent always.
"""
import struct
from typing import NamedTuple

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _lib
from ._lib import ModiffError

FP8_BLOCK = 128
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


_Tensor, _grad_enabled = torch.Tensor, torch.is_grad_enabled
# what torch.cuda.current_stream(device).cuda_stream and torch.cuda.current_device() wrap
_stream, _current = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _device(name, *tensors):
    """The device that all `tensors` (None allowed) are on; CUDA tensors, none of which needs gradients or
    carries a tangent."""
    device, grad = -2, _grad_enabled()
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, _Tensor):
            raise ModiffError(f"{name}: every tensor must be a CUDA tensor (there is no CPU fallback)")
        d = t.get_device()
        if d != device:
            if d < 0:
                raise ModiffError(f"{name}: every tensor must be a CUDA tensor (there is no CPU fallback)")
            if device >= 0:
                raise ModiffError(f"{name}: tensors on cuda:{device} and cuda:{d}")
            device = d
        if grad and t.requires_grad:
            raise ModiffError(f"{name} has no backward pass: call it under torch.no_grad() or detach its inputs")
    if _forward_ad._current_level >= 0:                        # inside a dual_level or torch.func.jvp
        for t in tensors:
            if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
                raise ModiffError(f"{name} has no forward-mode derivative: an input carries a tangent")
    return device


def _dtype(name, x):
    dt = _DTYPES.get(x.dtype)
    if dt is None:
        raise ModiffError(f"{name}: fp32, fp16 or bf16 tensors, got {x.dtype}")
    return dt


# the arguments of the entry points as 64-bit words, without the stream, which is the last
_CACHE = "4Q4i"
_PACK = {name: struct.Struct(words + "q").pack for name, words in (
    ("modiff_fp8_quantize", "9q"), ("modiff_fp8_linear", "15q"), ("modiff_fp8_linear_x", "14q"),
    ("modiff_qk_norm_rope", "25qdq"), ("modiff_kv4_append", _CACHE + "14q"), ("modiff_kv4_read", _CACHE + "8q"),
    ("modiff_kv4_attention", _CACHE + "11qd5q"))}
_PACK_BYTES = struct.Struct(_CACHE + "7q").pack


def _call(device, entry, *args, nbytes=0, nops=0, more=0):
    """One entry point on `device`'s current stream, whatever the current device is; `more` kernels
    beyond its first."""
    words = _PACK[entry](*args, _stream(device))
    if device == _current():
        _lib.call_words(entry, words, nbytes, nops, more)
    else:
        with torch.cuda.device(device):
            _lib.call_words(entry, words, nbytes, nops, more)


# ------------------------------------------------------------------------------- 8-bit linear layers
class Fp8Rows(NamedTuple):
    """Rows quantised by `fp8_quantize`: e4m3 codes [..., k] (row pitch a multiple of 16), fp32 scales
    [..., ceil(k / 128)] (in memory block by block, the rows of a block next to each other) and the type
    of the rows, which is the type of the layers' outputs."""
    codes: torch.Tensor
    scale: torch.Tensor
    dtype: torch.dtype


def _rows(name, x):
    """[..., k] as (address, row pitch, rows, k, the tensor that holds them); a copy only if it must be."""
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ModiffError(f"{name}: rows of at least one channel, got shape {tuple(x.shape)}")
    k = x.shape[-1]
    if x.dim() != 2:
        x = x.reshape(-1, k)
    if k > 1 and x.stride(1) != 1:
        x = x.contiguous()
    return x.data_ptr(), x.stride(0), x.shape[0], k, x


def fp8_quantize(x):
    """x [..., k] -> `Fp8Rows`: per row and block of 128 channels scale = max|x| / 448 (as a product with
    the fp32 number 1 / 448; 1 where it is 0) and codes e4m3(x / scale).  Quantise once what several
    layers read."""
    device = _device("fp8_quantize", x)
    dt = _dtype("fp8_quantize", x)
    at, pitch, rows, k, keep = _rows("fp8_quantize", x)
    blocks, kp = -(-k // FP8_BLOCK), -(-k // 16) * 16
    lead = tuple(x.shape[:-1])
    codes = x.new_empty(lead + (kp,), dtype=torch.float8_e4m3fn)
    row4 = -(-rows // 4) * 4
    scale = x.new_empty((blocks, row4), dtype=torch.float32)
    if rows:
        _call(device, 'modiff_fp8_quantize', at, pitch, rows, k, dt, codes.data_ptr(), kp, scale.data_ptr(), row4,
              nbytes=rows * (k * x.element_size() + kp + 4 * blocks))
    scale = scale[:, :rows].t()
    return Fp8Rows(codes[..., :k], scale if len(lead) == 1 else scale.view(lead + (blocks,)), x.dtype)


def fp8_pack_weight(w):
    """A weight matrix [n, k] -> (e4m3 codes [n, k] with a row pitch of a multiple of 16, fp32 scales
    [ceil(n / 128), ceil(k / 128)]), one scale per 128 x 128 block.  Once per weight version."""
    if isinstance(w, torch.Tensor):
        w = w.detach()
    device = _device("fp8_pack_weight", w)
    dt = _dtype("fp8_pack_weight", w)
    if w.dim() != 2 or w.numel() == 0:
        raise ModiffError(f"fp8_pack_weight: a matrix [n, k], got shape {tuple(w.shape)}")
    at, pitch, n, k, keep = _rows("fp8_pack_weight", w)
    kp = -(-k // 16) * 16
    codes = torch.empty((n, kp), dtype=torch.float8_e4m3fn, device=w.device)
    scale = torch.empty((-(-n // FP8_BLOCK), -(-k // FP8_BLOCK)), dtype=torch.float32, device=w.device)
    with torch.cuda.device(device):
        _lib.call('modiff_fp8_pack_weight', at, pitch, n, k, dt, codes.data_ptr(), kp, scale.data_ptr(),
                  scale.shape[1], _stream(device), nbytes=n * (k * w.element_size() + kp))
    return codes[:, :k], scale


def fp8_linear(x, w, w_scale, bias=None):
    """y = x w^T (+ bias) with x (a tensor [..., k], or `Fp8Rows`) and w (`fp8_pack_weight`) as 8-bit
    floating-point codes with one scale per block of 128 channels (and 128 weight rows).  y [..., n] and
    bias have the type of x."""
    ready = isinstance(x, Fp8Rows)
    src = x.codes if ready else x
    device = _device("fp8_linear", src, w, w_scale, bias)
    if w.dtype is not torch.float8_e4m3fn or w.dim() != 2 or w.numel() == 0:
        raise ModiffError("fp8_linear: weight codes are a float8_e4m3fn matrix [n, k] (fp8_pack_weight)")
    n, k = w.shape
    w_pitch, step = w.stride()
    if n == 1:
        w_pitch = -(-k // 16) * 16
    if (k > 1 and step != 1) or w_pitch % 16 or w_pitch < k or w.data_ptr() % 16:
        raise ModiffError("fp8_linear: weight rows start at multiples of 16 bytes (fp8_pack_weight lays them "
                          f"out so); got strides {w.stride()} for {k} channels")
    blocks = -(-k // FP8_BLOCK)
    if w_scale.dtype != torch.float32 or w_scale.shape != (-(-n // FP8_BLOCK), blocks):
        raise ModiffError(f"fp8_linear: fp32 weight scales of shape {(-(-n // FP8_BLOCK), blocks)}, got "
                          f"{w_scale.dtype} {tuple(w_scale.shape)}")
    if not w_scale.is_contiguous():
        w_scale = w_scale.contiguous()
    dtype = x.dtype
    dt = _DTYPES.get(dtype)
    if dt is None:
        raise ModiffError(f"fp8_linear: fp32, fp16 or bf16 rows, got {dtype}")
    if src.dim() < 1 or src.shape[-1] != k:
        raise ModiffError(f"fp8_linear: rows of shape {tuple(src.shape)} for weights {tuple(w.shape)}")
    if bias is not None:
        if bias.dtype != dtype or bias.shape != (n,):
            raise ModiffError(f"fp8_linear: bias of {n} values of {dtype}, got {tuple(bias.shape)} {bias.dtype}")
        bias = bias.contiguous()
    if not ready:
        return _fp8_linear_rows(device, x, w, n, k, w_pitch, w_scale, blocks, bias, dt)
    lead = tuple(src.shape[:-1])
    y = torch.empty(lead + (n,), dtype=dtype, device=src.device)
    if y.numel():
        kp = -(-k // 16) * 16
        rows = lead[0] if len(lead) == 1 else y.numel() // n
        if rows > 0x7fffff00:
            raise ModiffError("fp8_linear: too many rows")
        _device("fp8_linear", src, x.scale)
        if x.scale.dtype != torch.float32 or tuple(x.scale.shape) != lead + (blocks,):
            raise ModiffError(f"fp8_linear: fp32 scales of shape {lead + (blocks,)}, got {tuple(x.scale.shape)}")
        row4 = -(-rows // 4) * 4
        if (src.dtype != torch.float8_e4m3fn or src.data_ptr() % 16 or not _pitched(src, kp, 1)
                or x.scale.data_ptr() % 16 or not _pitched(x.scale, 1, row4)):
            raise ModiffError("fp8_linear: rows of codes as fp8_quantize lays them out")
        _call(device, 'modiff_fp8_linear', src.data_ptr(), kp, x.scale.data_ptr(), row4, w.data_ptr(), w_pitch,
              w_scale.data_ptr(), blocks, 0 if bias is None else bias.data_ptr(), y.data_ptr(), n, rows, k, n, dt,
              nbytes=rows * kp + n * k + y.numel() * y.element_size(), nops=2 * rows * n * k)
    return y


def _fp8_linear_rows(device, x, w, n, k, w_pitch, w_scale, blocks, bias, dt):
    """`fp8_linear` of a tensor: quantised inside the product, or into a workspace before it."""
    at, pitch, rows, _, keep = _rows("fp8_linear", x)
    if rows > 0x7fffff00:
        raise ModiffError("fp8_linear: too many rows")
    y = keep.new_empty((rows, n))
    if rows:
        size = _lib.lib().modiff_fp8_linear_bytes(rows, k, n)
        work = keep.new_empty(size, dtype=torch.uint8) if size else None
        _call(device, 'modiff_fp8_linear_x', at, pitch, w.data_ptr(), w_pitch, w_scale.data_ptr(), blocks,
              0 if bias is None else bias.data_ptr(), y.data_ptr(), n, rows, k, n, dt,
              0 if work is None else work.data_ptr(),
              nbytes=rows * (k + n) * x.element_size() + n * k, nops=2 * rows * n * k, more=int(size > 0))
    return y if x.dim() == 2 else y.view(*x.shape[:-1], n)


def _pitched(t, pitch, step):
    """Whether the leading dimensions of `t` walk rows `pitch` apart without a gap, its last one `step`."""
    if t.shape[-1] > 1 and t.stride(-1) != step:
        return False
    for d in range(t.dim() - 2, -1, -1):
        if t.shape[d] > 1 and t.stride(d) != pitch:
            return False
        pitch *= t.shape[d]
    return True


# --------------------------------------------------------------------- norms of queries and keys
def _tokens(name, x):
    """[..., heads, d] as [tokens, heads, d] with the channels contiguous (a copy only if it must be)."""
    if x.dim() != 3:
        if x.dim() < 3:
            raise ModiffError(f"{name}: tensors [..., heads, d], got shape {tuple(x.shape)}")
        x = x.flatten(0, -3)
    return x if x.stride(2) == 1 or x.shape[2] == 1 else x.contiguous()


def _norm_weight(name, w, d):
    """Address of a weight, and the tensor that holds it."""
    if w is None:
        return 0, None
    if w.dtype is not torch.float32 or w.shape != (d,):
        raise ModiffError(f"{name}: fp32 weights of {d} values, got {tuple(w.shape)} {w.dtype}")
    w = w.contiguous()
    return w.data_ptr(), w


def _norm_side(name, x, out):
    """One of q and k: (input, its copy if one had to be made, result, arguments of the entry point)."""
    x3 = _tokens(name, x)
    if out is None:
        out = torch.empty_like(x3) if x3 is x else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif out.shape != x.shape or out.dtype is not x.dtype:
        raise ModiffError(f"{name}: out {tuple(out.shape)} {out.dtype} for {tuple(x.shape)} {x.dtype}")
    flat = out
    if out.dim() != 3:
        try:
            flat = out.view(-1, *out.shape[-2:]) if out.numel() else out.flatten(0, -3)
        except RuntimeError:
            raise ModiffError(f"{name}: out needs leading dimensions that merge, got strides {out.stride()}") from None
    x_token, x_head, _ = x3.stride()
    y_token, y_head, step = flat.stride()
    if step != 1:
        raise ModiffError(f"{name}: out needs contiguous channels, got strides {out.stride()}")
    return x3, out, (x3.data_ptr(), x_token, x_head, flat.data_ptr(), y_token, y_head, x3.shape[1])


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions=None, eps=1e-6, interleaved=False, out=None):
    """Root-mean-square norm of every head of q [..., heads, d] and k [..., kv_heads, d] (k may be None),
    times the weights fp32 [d] (None: ones), and the rotation of the first 2 * cos.shape[1] channels by
    the angles in row `positions` (int32 / int64, one per token; None: the token's own number) of the
    fp32 tables cos and sin, one pass over both.  Pairs are (i, half + i), or (2i, 2i + 1) with
    `interleaved`.  q and k may be slices of one projection; `out` = (q, k) writes in place (`out` may
    be the inputs or apart from them, not overlap them otherwise).  A position outside the tables gives a
    row of NaN.  Returns (q', k')."""
    name = "qk_norm_rope"
    if out is not None and (len(out) != 2 or (out[1] is None) != (k is None)):
        raise ModiffError(f"{name}: out is a pair like (q, k)")
    device = _device(name, q, k, q_weight, k_weight, cos, sin, positions, *(out or ()))
    dt = _dtype(name, q)
    d = q.shape[-1] if q.dim() else 0
    if k is not None and (k.dtype is not q.dtype or k.shape[-1] != d or k.shape[:-2] != q.shape[:-2]):
        raise ModiffError(f"{name}: q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} differ in more "
                          "than their heads")
    if d % 2 or not 2 <= d <= 256:
        raise ModiffError(f"{name}: heads of an even number of channels up to 256, got {d}")
    qw, q_weight = _norm_weight(name, q_weight, d)
    kw, k_weight = _norm_weight(name, k_weight, d)
    shape = cos.shape
    if (cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or len(shape) != 2 or sin.shape != shape
            or 2 * shape[1] > d):
        raise ModiffError(f"{name}: fp32 tables [rows, at most {d // 2}], got {tuple(cos.shape)} and "
                          f"{tuple(sin.shape)}")
    cos, sin = cos.contiguous(), sin.contiguous()
    rows, half = shape
    q3, q_out, q_args = _norm_side(name, q, None if out is None else out[0])
    n = q3.shape[0]
    k3, k_out, k_args = None, None, (0, 0, 0, 0, 0, 0, 0)
    if k is not None:
        k3, k_out, k_args = _norm_side(name, k, None if out is None else out[1])
    wide, at = 0, 0
    if positions is not None:
        wide = int(positions.dtype is torch.int64)
        if not (wide or positions.dtype is torch.int32) or positions.numel() != n:
            raise ModiffError(f"{name}: {n} positions of int32 or int64, got {tuple(positions.shape)} "
                              f"{positions.dtype}")
        positions = positions.contiguous()
        at = positions.data_ptr()
    elif half and rows < n:
        raise ModiffError(f"{name}: tables of {rows} rows for {n} tokens")
    if n:
        _call(device, 'modiff_qk_norm_rope', *q_args, *k_args, qw, kw, cos.data_ptr(), sin.data_ptr(), rows, at, wide, n,
              d, 2 * half, int(bool(interleaved)), eps, dt,
              nbytes=2 * n * (q_args[6] + k_args[6]) * d * q.element_size())
    return q_out, k_out


# ------------------------------------------------------------------------------ the 4-bit cache
class KV4Cache(NamedTuple):
    """A paged cache of keys and values in 4 bits (`kv4_cache` makes an empty one): codes uint8 [pages,
    kv_heads, page_size, d / 2], channel 2i in the low half of byte i, and fp16 (scale, minimum) [pages,
    kv_heads, page_size, 2].  A token's value of channel c is scale * code[c] + minimum, with the scale
    (largest - smallest value) / 15 (as a product with the fp32 number 1 / 15)."""
    k_codes: torch.Tensor
    k_params: torch.Tensor
    v_codes: torch.Tensor
    v_params: torch.Tensor


def kv4_cache(pages, kv_heads, page_size, head_dim, device):
    """An empty `KV4Cache`.  page_size is a multiple of 16, head_dim 64, 128, 192 or 256; a token takes
    head_dim + 8 bytes per head."""
    if pages < 1 or kv_heads < 1 or page_size < 16 or page_size % 16 or head_dim not in (64, 128, 192, 256):
        raise ModiffError(f"kv4_cache: {pages} pages of {page_size} tokens (a multiple of 16), {kv_heads} heads of "
                          f"{head_dim} channels (64, 128, 192 or 256)")
    shape = (pages, kv_heads, page_size)
    codes = [torch.zeros(shape + (head_dim // 2,), dtype=torch.uint8, device=device) for _ in range(2)]
    params = [torch.zeros(shape + (2,), dtype=torch.float16, device=device) for _ in range(2)]
    return KV4Cache(codes[0], params[0], codes[1], params[1])


def _cache(name, cache, table, lengths):
    """(the cache as the entry points take it, its heads and channels, table and lengths without gaps)"""
    kc, kp, vc, vp = cache
    shape, par = kc.shape, kp.shape
    if (len(shape) != 4 or shape[1] == 0 or kc.dtype is not torch.uint8 or vc.dtype is not torch.uint8 or vc.shape != shape
            or kp.dtype is not torch.float16 or vp.dtype is not torch.float16 or par != (*shape[:3], 2) or vp.shape != par
            or not (kc.is_contiguous() and vc.is_contiguous() and kp.is_contiguous() and vp.is_contiguous())):
        raise ModiffError(f"{name}: a cache is contiguous uint8 codes [pages, heads, page_size, d / 2] and fp16 "
                          f"[pages, heads, page_size, 2], got {tuple(kc.shape)} {kc.dtype}, {tuple(kp.shape)} {kp.dtype}")
    where = table.shape
    if (len(where) != 2 or table.dtype is not torch.int32 or lengths.dtype is not torch.int32
            or lengths.shape != where[:1] or where[1] == 0):
        raise ModiffError(f"{name}: int32 table [batch, pages] and lengths [batch], got {tuple(table.shape)} "
                          f"{table.dtype} and {tuple(lengths.shape)} {lengths.dtype}")
    pages, heads, size, half = shape
    return ((kc.data_ptr(), vc.data_ptr(), kp.data_ptr(), vp.data_ptr(), pages, heads, size, 2 * half), heads, 2 * half,
            table.contiguous(), lengths.contiguous())


def kv4_append(cache, k, v, table, lengths):
    """Writes k and v [batch, n, kv_heads, d] as the last n positions of every sequence: token i of
    sequence b at position lengths[b] - n + i, i.e. at that offset of the pages `table`[b] names.
    `lengths` counts the new tokens; positions below 0 (shorter sequences of a padded batch) and page
    numbers outside the cache are skipped.  No two sequences may name the same place."""
    name = "kv4_append"
    device = _device(name, k, v, table, lengths, *cache)
    c, heads, dim, table, lengths = _cache(name, cache, table, lengths)
    dt = _dtype(name, k)
    b, per = table.shape
    shape = k.shape
    if (len(shape) != 4 or v.shape != shape or v.dtype is not k.dtype or shape[0] != b or shape[2] != heads
            or shape[3] != dim):
        raise ModiffError(f"{name}: k and v [{b}, n, {heads}, {dim}] of one type, got {tuple(k.shape)} {k.dtype} "
                          f"and {tuple(v.shape)} {v.dtype}")
    ks, vs = k.stride(), v.stride()
    if ks[3] != 1:
        k = k.contiguous()
        ks = k.stride()
    if vs[3] != 1:
        v = v.contiguous()
        vs = v.stride()
    rows = b * shape[1] * heads
    if rows:
        _call(device, 'modiff_kv4_append', *c, k.data_ptr(), *ks[:3], v.data_ptr(), *vs[:3], table.data_ptr(),
              lengths.data_ptr(), b, shape[1], per, dt, nbytes=2 * rows * (dim * k.element_size() + dim // 2 + 4))


def kv4_read(cache, table, lengths, n, dtype=torch.float32):
    """The last n positions of every sequence as values: (k, v) [batch, n, kv_heads, d], zeros for
    positions below 0 and pages outside the cache."""
    name = "kv4_read"
    device = _device(name, table, lengths, *cache)
    c, heads, dim, table, lengths = _cache(name, cache, table, lengths)
    if dtype not in _DTYPES or n < 0:
        raise ModiffError(f"{name}: n >= 0 tokens as fp32, fp16 or bf16, got {n} and {dtype}")
    b, per = table.shape
    k = table.new_empty((b, n, heads, dim), dtype=dtype)
    v = torch.empty_like(k)
    rows = b * n * heads
    if rows:
        _call(device, 'modiff_kv4_read', *c, table.data_ptr(), lengths.data_ptr(), b, n, per, k.data_ptr(), v.data_ptr(),
              _DTYPES[dtype], nbytes=2 * rows * (dim * k.element_size() + dim // 2 + 4))
    return k, v


def kv4_attention(q, cache, table, lengths, scale=None, causal=True, window=0, sinks=0):
    """Attention of q [batch, n, heads, d] over the cached tokens of every sequence:
    out[b, i, h] = sum_t softmax_t(scale * q[b, i, h] . k_t) v_t; `heads` is a multiple of the cache's
    heads, which consecutive query heads share.  Query i of sequence b stands at position
    lengths[b] - n + i and sees the positions up to its own; with `window` > 0 only the last `window` of
    them and the first `sinks` of the sequence (tokens outside are not read).  causal=False: every query
    sees all lengths[b] tokens.  A row that sees nothing is 0.  A cached scale or minimum that is not finite
    (`kv4_append` writes NaN for a row that holds one) makes the rows that see its key NaN, those that see its
    value not finite, and no others.  scale defaults to d ** -0.5.

    fp32 and fp16: queries and weights count with 22 bits (of a row's largest element), codes exactly, the rest is
    fp32.  bf16: weights are rounded to fp16, 2^-11 of each at most, and sums of query times code keep 17 bits; from
    41 query rows per key head on (d <= 128) keys and values are rounded to fp16 as well, once each, so that a
    score is off by up to scale 2^-11 sum |q k|."""
    name = "kv4_attention"
    device = _device(name, q, table, lengths, *cache)
    c, kv_heads, dim, table, lengths = _cache(name, cache, table, lengths)
    dt = _dtype(name, q)
    b, per = table.shape
    shape = q.shape
    if len(shape) != 4 or shape[0] != b or shape[3] != dim or shape[2] == 0 or shape[2] % kv_heads:
        raise ModiffError(f"{name}: q [{b}, n, a multiple of {kv_heads}, {dim}], got {tuple(shape)}")
    window, sinks = int(window), int(sinks)
    if window < 0 or sinks < 0 or (window and not causal) or (sinks and not window):
        raise ModiffError(f"{name}: window {window} and sinks {sinks}: a window needs causal positions, sinks need "
                          "a window")
    if q.is_contiguous():
        out = torch.empty_like(q)
    else:
        out = torch.empty(shape, dtype=q.dtype, device=q.device)
        if q.stride(3) != 1:
            q = q.contiguous()
    n, heads = shape[1], shape[2]
    if b * n:
        window, sinks = min(window, 1 << 30), min(sinks, 1 << 30)
        size = _lib.lib().modiff_packed_call(7, _PACK_BYTES(*c, b, n, heads, per, window, sinks, dt))
        work = q.new_empty(size, dtype=torch.uint8) if size else None
        _call(device, 'modiff_kv4_attention', *c, q.data_ptr(), *q.stride()[:3], table.data_ptr(), lengths.data_ptr(),
              out.data_ptr(), b, n, heads, per, dim ** -0.5 if scale is None else scale, 1 if causal else 0, window,
              sinks, dt, 0 if work is None else work.data_ptr(), more=int(size > 0))
    return out

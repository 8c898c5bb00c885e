"""Plain restatements of the low-precision transformer operators: 8-bit floating-point linear layers,
norms with rotation, the 4-bit cache and its attention.  Scales and codes in fp32, as they are defined;
everything that is summed in 64 bits."""
import math

import torch

BLOCK = 128


def half_step(dtype):
    """Largest relative error of one rounding to nearest."""
    return torch.finfo(dtype).eps / 2


def e4m3_rows(x):
    """[rows, k] -> codes as fp32 values [rows, k], scales [rows, blocks]."""
    rows, k = x.shape
    kb = -(-k // BLOCK)
    xp = torch.zeros(rows, kb * BLOCK)
    xp[:, :k] = x.float().cpu()
    xb = xp.view(rows, kb, BLOCK)
    top = xb.abs().amax(-1)
    s = top * torch.tensor(1.0 / 448.0)
    s = torch.where(s == 0, torch.ones_like(s), s)
    codes = (xb / s[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()
    return codes.view(rows, -1)[:, :k], s


def e4m3_blocks(w):
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    wp = torch.zeros(nb * BLOCK, kb * BLOCK)
    wp[:n, :k] = w.float().cpu()
    blocks = wp.view(nb, BLOCK, kb, BLOCK)
    top = blocks.abs().amax(dim=(1, 3))
    s = top * torch.tensor(1.0 / 448.0)
    s = torch.where(s == 0, torch.ones_like(s), s)
    codes = (blocks / s[:, None, :, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()
    return codes.view(nb * BLOCK, kb * BLOCK)[:n, :k], s


def linear(codes, scale, w_codes, w_scale, bias=None):
    """(y, sum of the terms' magnitudes) in 64 bits."""
    k, n = codes.shape[1], w_codes.shape[0]
    x = codes.double() * scale.double().repeat_interleave(BLOCK, 1)[:, :k]
    w = w_codes.double() * w_scale.double().repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size


def linear_tolerance(y, size, k, dtype):
    """Four MMAs of 32 exact products and an accumulator a block, each at least 24 bits of the largest
    addend: 4 * 33 * 2^-23 of a block's magnitudes; scale product, scaling, addition and bias 2^-24 each
    per block; one rounding of the result."""
    kb = -(-k // BLOCK)
    return size * (132 * 2.0 ** -23 + (kb + 4) * 2.0 ** -24) + y.abs() * half_step(dtype)


def norm_rope(x, w, cos, sin, positions, eps, interleaved):
    """x [tokens, heads, d] -> (y, sum of the terms' magnitudes) in 64 bits."""
    x = x.double().cpu()
    x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        x = x * w.double().cpu()
    cos, sin = cos.double().cpu(), sin.double().cpu()
    half = cos.shape[1]
    at = torch.arange(x.shape[0]) if positions is None else positions.long().cpu().flatten()
    bad = (at < 0) | (at >= cos.shape[0])
    if half == 0:
        bad = torch.zeros_like(bad)
    at = at.clamp(0, max(0, cos.shape[0] - 1))
    c, s = (t[at][:, None] if half else torch.zeros(x.shape[0], 1, 0, dtype=torch.float64) for t in (cos, sin))
    i = torch.arange(half)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, half + i)
    a, b = x[..., first], x[..., second]
    y, size = x.clone(), x.abs()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = (a * c).abs() + (b * s).abs()
    size[..., second] = (b * c).abs() + (a * s).abs()
    y[bad] = math.nan
    return y, size


def norm_tolerance(y, size, d, dtype):
    """The mean of d squares is off by at most (d + 2) 2^-24, its root by half of that; root, division
    and three products a term, one addition; one rounding of the result."""
    return size * (d / 2 + 8) * 2.0 ** -24 + y.abs() * half_step(dtype)


def quantise_4bit(x):
    x = x.float().cpu().clamp(-65504.0, 65504.0)
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s, m = ((high - low) * torch.tensor(1.0 / 15.0)).half(), low.half()
    sf = s.float()
    q = torch.where(sf > 0, (x - m.float()) / torch.where(sf > 0, sf, torch.ones_like(sf)), torch.zeros_like(x))
    q = torch.nan_to_num(q, 0.0).round().clamp(0, 15).to(torch.uint8)
    return q[..., 0::2] | (q[..., 1::2] << 4), torch.cat([s, m], -1)


def values_4bit(codes, params):
    """(codes as numbers, scale, minimum) in 64 bits."""
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    return q, params[..., 0].double(), params[..., 1].double()


def attention(q, cache, table, lengths, scale, causal=True, window=0, sinks=0):
    """(out, tolerance) [batch, n, heads, d] in 64 bits, on the CPU, one row at a time."""
    dtype = q.dtype
    kc, kp, vc, vp = (t.cpu() for t in cache)
    table, lengths = table.cpu(), lengths.cpu()
    pages, kv_heads, size, _ = kc.shape
    b, n, heads, d = q.shape
    q = q.double().cpu()
    group = heads // kv_heads
    out = torch.zeros(b, n, heads, d, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for i in range(b):
        length = min(max(int(lengths[i]), 0), table.shape[1] * size)
        t = torch.arange(length)
        page = table[i].long()[t // size]
        there = (page >= 0) & (page < pages)
        page = page.clamp(0, pages - 1)
        for h in range(kv_heads):
            kq, ks, km = values_4bit(kc[page, h, t % size], kp[page, h, t % size])
            vq, vs, vm = values_4bit(vc[page, h, t % size], vp[page, h, t % size])
            for r in range(n):
                sees = there.clone()
                if causal:
                    at = length - n + r
                    sees &= t <= at
                    if window:
                        sees &= (t > at - window) | (t < sinks)
                if not bool(sees.any()):
                    continue
                rows = q[i, r, h * group:(h + 1) * group]
                kq_, ks_, km_ = kq[sees], ks[sees], km[sees]
                score = scale * (ks_ * (rows @ kq_.t()) + km_ * rows.sum(-1, keepdim=True))
                p = torch.softmax(score, -1)
                v = vs[sees, None] * vq[sees] + vm[sees, None]
                out[i, r, h * group:(h + 1) * group] = p @ v
                # a score: d exact products and the row's sum in fp32 (or q in 22 bits), scale and minimum
                off = abs(scale) * (d + 16) * 2.0 ** -22 * (
                    ks_ * (rows.abs() @ kq_.t()) + km_.abs() * rows.abs().sum(-1, keepdim=True)).amax(-1)
                # its weight: exp2 (2^-21) and, against the codes, one rounding to fp16 for bf16 (22 bits
                # otherwise); the sums over the tokens
                much = p @ (vs[sees, None] * vq[sees] + vm[sees, None].abs())
                many = d <= 128 and n * group > {torch.bfloat16: 40, torch.float16: 63}.get(dtype, n * group)
                weight = 2.0 ** -20 + (2.0 ** -11 if many or dtype == torch.bfloat16 else 2.0 ** -21)
                if many:
                    # many rows: keys and values as fp16 numbers, one rounding (half a step, 2^-11) each, and
                    # weights that fp16's smallest step, 2^-24, may round by 2^-25 where 2^5 stands for 1
                    k = ks_[:, None] * kq_ + km_[:, None]
                    off = off + abs(scale) * 2.0 ** -11 * (rows.abs() @ k.abs().t()).amax(-1)
                    much = torch.maximum(much, p @ v.abs())
                    weight = weight + 2.0 ** -11
                    tol[i, r, h * group:(h + 1) * group] = len(k) * 2.0 ** -30 * v.abs().amax(0)
                err = (2 * off + weight + (len(p[0]) + 8) * 2.0 ** -23)[:, None] * much
                tol[i, r, h * group:(h + 1) * group] += err + (p @ v).abs() * half_step(dtype)
    # what fp16 cannot hold: outputs below its normal range
    return out, tol + (2.0 ** -25 if dtype == torch.float16 else 0.0)

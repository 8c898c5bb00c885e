"""Low-precision transformer operators: how far attention over the 4-bit cache is from 64 bits, as a norm over
all outputs, whichever kernel serves a call; cached rows that are not finite; and tangents."""
import math

import pytest
import torch

import lowp_reference as ref
from modiff_b200 import ModiffError, ops

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _cache_of(cuda, k, v, page, seed):
    """k, v [batch, tokens, heads, d] as a cache whose pages lie in random order."""
    b, tokens, heads, d = k.shape
    per = -(-tokens // page)
    table = torch.randperm(b * per, generator=_gen(seed)).view(b, per).int()
    parts = []
    for x in (k, v):
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, per * page - tokens))
        codes, params = ref.quantise_4bit(x.view(b * per, page, heads, d).transpose(1, 2))
        order = table.flatten().long().argsort()
        parts += [codes[order].contiguous().to(cuda), params[order].contiguous().to(cuda)]
    return ops.KV4Cache(*parts), table.to(cuda)


def _attention(q, cache, table, lengths, scale, window=0, sinks=0, causal=True):
    """(out, variance) in 64 bits.  The variance is that of independent roundings of keys, values and weights to
    fp16, once each: a rounding is uniform within half a step, at most 2^-11 of the value, so of variance (2^-11)^2 / 3
    at most.  A weight's and a value's act on p v; a key's on the score, d score = scale sum(q dk), and the score's on
    p (v - out)."""
    kc, kp, vc, vp = (t.cpu() for t in cache)
    pages, kv_heads, size, _ = kc.shape
    b, n, heads, d = q.shape
    group, q = heads // kv_heads, q.double().cpu()
    out, var = torch.zeros(b, n, heads, d, dtype=torch.float64), torch.zeros(b, n, heads, d, dtype=torch.float64)
    unit = 2.0 ** -22 / 3
    for i, length in enumerate(lengths):
        t = torch.arange(length)
        page = table.cpu()[i].long()[t // size]
        at = (length - n + torch.arange(n))[:, None]
        sees = (t <= at) if causal else torch.ones(n, length, dtype=torch.bool)
        if window:
            sees = sees & ((t > at - window) | (t < sinks))
        for h in range(kv_heads):
            k, v = (s[:, None] * c + m[:, None] for c, s, m in (
                ref.values_4bit(kc[page, h, t % size], kp[page, h, t % size]),
                ref.values_4bit(vc[page, h, t % size], vp[page, h, t % size])))
            for j in range(h * group, (h + 1) * group):
                x = q[i, :, j]
                p = torch.softmax((scale * x @ k.t()).masked_fill(~sees, -math.inf), -1)
                p = torch.where(sees.any(1, keepdim=True), p, torch.zeros_like(p))
                y, p2 = p @ v, p * p
                score = p2 * (scale ** 2 * unit) * (x * x @ (k * k).t())
                out[i, :, j] = y
                var[i, :, j] = 2 * unit * (p2 @ (v * v)) + (score @ (v * v) - 2 * y * (score @ v)
                                                            + y * y * score.sum(1, keepdim=True))
    return out, var


CASES = [  # tokens of every sequence, queries, heads, key heads, channels, page, mask
    ([900, 310], 1, 8, 2, 128, 16, {}), ([500], 5, 8, 1, 64, 32, {}), ([700], 3, 4, 2, 256, 16, {}),
    ([640, 333], 15, 8, 2, 128, 16, dict(window=130, sinks=3)),                        # 60 rows a key head
    ([640, 333], 16, 8, 2, 128, 16, dict(window=130, sinks=3)),                        # 64
    ([900, 500], 200, 4, 2, 128, 64, {}), ([513], 300, 2, 1, 64, 16, dict(causal=False)),
    ([1200], 257, 2, 1, 128, 48, dict(window=400, sinks=5)), ([5000], 33, 4, 1, 64, 64, {}),
    ([130, 129, 64], 64, 2, 2, 128, 16, {}), ([300], 100, 2, 1, 192, 16, {}), ([300], 100, 2, 1, 256, 32, {})]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["even", "growing", "sizes"])
@pytest.mark.parametrize("lengths,n,heads,kv_heads,d,page,kw", CASES)
def test_kv4_attention_error_as_a_norm(cuda, lengths, n, heads, kv_heads, d, page, kw, kind, dtype):
    """fp32 and fp16: 22 bits of every weight, exact codes, fp32 otherwise.  The sums over the tokens are cut at 2^-23
    of them a step of 16 tokens, 2^-23 * 5000 / 16 = 2^-14.7 at the very worst where nothing cancels, an eighth of
    fp16's rounding (0.84 * 2^-12 in the mean): 1.01 of it together, and the test leaves a tenth.  fp32 is held to
    2^-16 of the result, four times that of scores of magnitude 64 with sums cut at 2^-23 (64 * 2^-23 = 2^-17, with
    signs an eighth of it in the mean, times two for numerator and sum).
    bf16: the output's rounding, and keys, values and weights as fp16 numbers, as variances; a tenth and a half more
    than the model, whose roundings are taken as large as they can be."""
    b, tokens = len(lengths), max(lengths)
    g = _gen(n + d)
    k, v = (torch.randn(b, tokens, kv_heads, d, generator=g) * 1.5 + 0.3 for _ in range(2))
    q = 2 * torch.randn(b, n, heads, d, generator=g)
    if kind == "growing":                     # scores that rise by 60 over the tokens: maxima found late
        u = torch.randn(d, generator=g)
        u = u / u.norm()
        rise = 60 * d ** 0.5 / 8 * torch.arange(tokens) / tokens
        k, q = 0.5 * k + rise[None, :, None, None] * u, q * 0.5 + 8 * u
    elif kind == "sizes":                     # values whose scales lie far apart, some of them constant
        v = v * torch.exp(2 * torch.randn(b, tokens, kv_heads, 1, generator=g))
        v[:, 7::50] = 1.25
    q = q.to(dtype)
    cache, table = _cache_of(cuda, k, v, page, n)
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    got = ops.kv4_attention(q.to(cuda), cache, table, lens, **kw)
    want, var = _attention(q, cache, table, lengths, d ** -0.5, **kw)
    off = float((got.double().cpu() - want).norm())
    rounding = float((want.to(dtype).double() - want).norm())
    if dtype == torch.float32:
        assert off <= 2.0 ** -16 * float(want.norm())
    elif dtype == torch.float16:
        assert off <= 1.1 * rounding, off / rounding
    else:
        most = ((1.1 * rounding) ** 2 + 1.5 ** 2 * float(var.sum())) ** 0.5
        assert off <= most, off / most


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("n,d", [(4, 64), (4, 256), (40, 128), (100, 64)])
def test_kv4_attention_meets_cached_rows_that_are_not_finite(cuda, n, d, which, value, dtype):
    """A key whose scale (0) or minimum (1) is not finite makes the rows that see it NaN, such a value makes them not
    finite; the rows that do not see it are what they were."""
    lengths = [150, 90]
    g = _gen(d + n)
    k, v = (torch.randn(2, 150, 2, d, generator=g) for _ in range(2))
    cache, table = _cache_of(cuda, k, v, 16, 3)
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    q = torch.randn(2, n, 4, d, generator=g).to(dtype).to(cuda)
    clean = ops.kv4_attention(q, cache, table, lens)
    assert torch.isfinite(clean).all()
    at = 150 - n // 2                                      # seen by the later half of the queries
    place = (int(table[0, at // 16]), 1, at % 16, which)
    for params, key in ((cache.k_params, True), (cache.v_params, False)):
        before = params[place].clone()
        params[place] = value
        got = ops.kv4_attention(q, cache, table, lens)
        params[place] = before
        met, rest = got[0, n - n // 2:, 2:], [got[1], got[0, :n - n // 2], got[0, :, :2]]
        assert not torch.isfinite(met).any() and (not key or torch.isnan(met).all())
        for a, c in zip(rest, [clean[1], clean[0, :n - n // 2], clean[0, :, :2]]):
            assert torch.equal(a, c)
    assert torch.equal(ops.kv4_attention(q, cache, table, lens), clean)


@gpu
def test_tangents_are_refused(cuda):
    """There is no forward-mode derivative either: a tangent is refused, not dropped."""
    import torch.autograd.forward_ad as fwd
    x = torch.randn(4, 256, device=cuda)
    w, ws = ops.fp8_pack_weight(torch.randn(8, 256, device=cuda))
    cos = torch.ones(4, 32, device=cuda)
    q = torch.randn(1, 4, 2, 64, device=cuda)
    cache = ops.kv4_cache(2, 2, 16, 64, cuda)
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device=cuda), torch.full((1,), 4, dtype=torch.int32, device=cuda)
    calls = (lambda f: ops.fp8_quantize(f(x)), lambda f: ops.fp8_linear(f(x), w, ws),
             lambda f: ops.fp8_linear(x, w, ws, f(torch.zeros(8, device=cuda))),
             lambda f: ops.qk_norm_rope(f(q), None, None, None, cos, cos),
             lambda f: ops.qk_norm_rope(q, None, None, None, f(cos), cos),
             lambda f: ops.kv4_append(cache, q, f(q), table, lens),
             lambda f: ops.kv4_attention(f(q), cache, table, lens))
    with fwd.dual_level():
        for call in calls:
            with pytest.raises(ModiffError, match="tangent"):
                call(lambda t: fwd.make_dual(t, torch.ones_like(t)))
            call(lambda t: t)                              # nothing to refuse
    for call in calls:
        call(lambda t: t)
    with pytest.raises(ModiffError, match="tangent"):
        torch.func.jvp(lambda t: ops.fp8_linear(t, w, ws), (x,), (x,))

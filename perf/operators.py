"""The operators of a transformer served in low precision, as cases to be timed.

Four operators that such a block runs one after the other: the projection (8-bit floating-point codes
with one scale per block of 128), the norms of queries and keys with the rotation of their positions,
the write into a cache of keys and values held in 4 bits, and the attention that reads that cache.

Ranges: 1 to 16384 rows of 16 to 10240 channels for the projection; 1 to 65536 tokens, 1 to 64 heads
of 32 to 256 channels for the norms; 1 to 8192 tokens written; caches of 1 to 131072 tokens read by
1 to 1024 queries a sequence, with and without a window, for the attention.

Formulas.  Projection: a row's block of 128 channels has the scale s = max|x| / 448 (1 where that is
0), in fp32, and the codes e4m3(x / s); weights have one scale per 128 x 128 block;
y = sum over blocks of s_x s_w sum(code_x code_w) + bias.  Norm: y = x / sqrt(mean(x^2) + eps) * w over
a head's channels, then (a, b) -> (a cos - b sin, b cos + a sin) for the pairs of its first channels.
Cache: a token's channels of one head have m = fp16(min x), s = fp16((max x - min x) / 15) and the
codes round((x - m) / s) in 0 .. 15 (0 where s is 0), two to a byte, the even channel in the low half;
values beyond +-65504 count as +-65504.  Attention: softmax over the visible tokens of
scale * q . (s_k code_k + m_k), times s_v code_v + m_v; query i of n stands at position length - n + i
and sees no later position, and with a window none more than window - 1 back except the first `sinks`.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
BLOCK = 128            # channels (and rows of a weight) that share one scale
E4M3_MAX = 448.0
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
EPS = 1e-6


# ------------------------------------------------------------------------------------------ cases
def _linear(rows, k, n, dtype, bias=True):
    return dict(op="linear", rows=rows, k=k, n=n, dtype=dtype, bias=bias)


def _norm(tokens, q_heads, k_heads, dim, rot, dtype, interleaved=False, gather=True):
    return dict(op="norm", tokens=tokens, q_heads=q_heads, k_heads=k_heads, dim=dim, rot=rot,
                dtype=dtype, interleaved=interleaved, gather=gather)


def _append(batch, new, longest, kv_heads, dim, page, dtype):
    return dict(op="append", batch=batch, new=new, longest=longest, kv_heads=kv_heads, dim=dim,
                page=page, dtype=dtype)


def _attention(batch, new, longest, heads, kv_heads, dim, page, dtype, window=0, sinks=0, causal=True):
    return dict(op="attention", batch=batch, new=new, longest=longest, heads=heads, kv_heads=kv_heads,
                dim=dim, page=page, dtype=dtype, window=window, sinks=sinks, causal=causal)


def _named(name, case):
    return dict(case, name=name)


def listed():
    return [
        # one token of one user through a projection of 1280 channels: latency
        _named("linear_1x1280x1280_bf16", _linear(1, 1280, 1280, "bf16")),
        # two prompts of 77 text tokens to the keys of a cross attention, in the UNet's own type
        _named("linear_154x768x640_fp32", _linear(154, 768, 640, "fp32", bias=False)),
        # a step of 64 users through a large layer: the weights' bytes decide
        _named("linear_64x8192x8192_bf16", _linear(64, 8192, 8192, "bf16", bias=False)),
        # the second layer of a feed-forward over a large batch of image tokens: arithmetic decides
        _named("linear_16384x5120x5120_bf16", _linear(16384, 5120, 5120, "bf16")),
        # one token, 32 query and 8 key heads, position read from a table: latency
        _named("norm_1x40x128_bf16", _norm(1, 32, 8, 128, 128, "bf16")),
        # 16 images of 64x64 tokens, 8 heads of 40 channels, a row of angles for every token
        _named("norm_65536x16x40_fp32", _norm(65536, 8, 8, 40, 40, "fp32", gather=False)),
        # a step of 64 users: one token each
        _named("append_64x1_bf16", _append(64, 1, 8192, 8, 128, 64, "bf16")),
        # prompts of four users, ragged
        _named("append_4x2048_fp16", _append(4, 2048, 4001, 8, 128, 16, "fp16")),
        # the next token of a short conversation: latency
        _named("attention_1x1_of_200_fp16", _attention(1, 1, 200, 32, 8, 128, 64, "fp16")),
        # a step of 64 users with 4096 to 8192 tokens behind them: the cache's bytes decide
        _named("attention_64x1_of_8192_bf16", _attention(64, 1, 8192, 32, 8, 128, 64, "bf16")),
        # one user with a long document, few heads: the cache has to be split to fill the machine
        _named("attention_1x1_of_131072_bf16", _attention(1, 1, 131072, 32, 4, 128, 64, "bf16")),
        # a piece of four prompts over what is cached, with a window and four sinks
        _named("attention_4x1000_of_8000_bf16", _attention(4, 1000, 8000, 32, 8, 128, 64, "bf16",
                                                           window=2048, sinks=4)),
    ]


def _between(rng, lo, hi):
    """A whole number, uniform over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["linear"] * 4 + ["norm"] * 2 + ["append"] * 2 + ["attention"] * 4)
    dtype = rng.choice(["fp32", "fp16", "bf16", "bf16"])
    if op == "linear":
        k, n = _between(rng, 16, 10240), _between(rng, 16, 10240)
        if rng.random() < 0.6:                 # most layers' widths are multiples of 64, some are odd
            k, n = -(-k // 64) * 64, -(-n // 64) * 64
        if k * n > 8192 * 8192:
            n = 8192 * 8192 // k
        return _linear(_between(rng, 1, min(16384, 16384 * 5120 * 5120 // (k * n))), k, n, dtype,
                       rng.random() < 0.5)
    if op == "norm":
        dim = rng.choice([32, 40, 64, 80, 96, 128, 128, 160, 256])
        k_heads = rng.choice([1, 2, 3, 8])
        q_heads = k_heads * rng.choice([1, 2, 4, 5, 8])
        tokens = _between(rng, 1, 65536 * 16 * 40 // ((q_heads + k_heads) * dim))
        return _norm(tokens, q_heads, k_heads, dim, rng.choice([dim, dim, dim // 2]), dtype,
                     rng.random() < 0.4, rng.random() < 0.6)
    dim = rng.choice([64, 128, 128, 192, 256])
    page = rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    batch = _between(rng, 1, 64)
    if op == "append":
        longest = _between(rng, 2, 8192)
        return _append(batch, min(longest, _between(rng, 1, max(1, 8192 // batch))), longest, kv_heads,
                       dim, page, dtype)
    heads = kv_heads * rng.choice([1, 2, 4, 7, 8])
    longest = _between(rng, 1, min(131072, 64 * 8192 * 8 * 128 // (batch * kv_heads * dim)))
    most = 4 * 1000 * 32 * 2048 * 128 // (batch * heads * longest * dim)
    new = 1 if rng.random() < 0.5 else min(longest, _between(rng, 1, max(1, min(1024, most))))
    window = _between(rng, 1, longest) if rng.random() < 0.4 else 0
    causal = window > 0 or rng.random() < 0.8
    return _attention(batch, new, longest, heads, kv_heads, dim, page, dtype, window,
                      rng.choice([0, 1, 4, 16]) if window else 0, causal)


# ----------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """Tokens of every sequence, the new ones among them: the longest first, down to half of it."""
    b, top = case["batch"], case["longest"]
    return [max(1, top - i * (top // 2) // b) for i in range(b)]


def _quantise_blocks(w):
    """Weights [n, k] -> codes with a row pitch of a multiple of 16, scales [n / 128, k / 128]."""
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    padded = torch.zeros(nb * BLOCK, kb * BLOCK, device=w.device)
    padded[:n, :k] = w
    blocks = padded.view(nb, BLOCK, kb, BLOCK)
    top = blocks.abs().amax(dim=(1, 3))
    scale = torch.where(top > 0, top / E4M3_MAX, torch.ones_like(top))
    codes = (blocks / scale[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    out = torch.zeros(n, -(-k // 16) * 16, dtype=torch.uint8, device=w.device)
    out[:, :k] = codes.view(nb * BLOCK, kb * BLOCK)[:n, :k].view(torch.uint8)
    return out.view(torch.float8_e4m3fn)[:, :k], scale


def _quantise_4bit(x):
    """[..., dim] -> packed codes [..., dim / 2], (scale, minimum) fp16 [..., 2]."""
    x = x.float().clamp(-65504.0, 65504.0)
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s, m = ((high - low) / 15.0).half(), low.half()
    sf = s.float()
    q = torch.where(sf > 0, (x - m.float()) / torch.where(sf > 0, sf, torch.ones_like(sf)),
                    torch.zeros_like(x))
    q = q.round().clamp(0.0, 15.0).to(torch.uint8)
    return q[..., 0::2] | (q[..., 1::2] << 4), torch.cat([s, m], -1)


def _dequantise_4bit(codes, params):
    low, high = (codes & 15).float(), (codes >> 4).float()
    q = torch.stack([low, high], -1).flatten(-2)
    return q * params[..., 0:1].float() + params[..., 1:2].float()


def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device=DEVICE)

    t = TYPES[case["dtype"]]
    state = dict(case=case)
    if case["op"] == "linear":
        # activations with a few strong channels, as a normalised layer's input has
        x = normal(case["rows"], case["k"]) * torch.exp(0.5 * normal(1, case["k"]))
        state["x"] = x.to(t)
        state["w"], state["w_scale"] = _quantise_blocks(normal(case["n"], case["k"]) * case["k"] ** -0.5)
        state["bias"] = normal(case["n"]).to(t) if case["bias"] else None
    elif case["op"] == "norm":
        hq, hk, d, n = case["q_heads"], case["k_heads"], case["dim"], case["tokens"]
        qkv = (2.0 * normal(n, (hq + 2 * hk) * d)).to(t)     # what a fused projection has written
        state["q"] = qkv[:, :hq * d].unflatten(1, (hq, d))
        state["k"] = qkv[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
        state["q_weight"], state["k_weight"] = 1.0 + 0.1 * normal(d), 1.0 + 0.1 * normal(d)
        rows = 8192 if case["gather"] else n
        half = case["rot"] // 2
        freq = 10000.0 ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)
        angle = torch.arange(rows, device=DEVICE, dtype=torch.float64)[:, None] * freq
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
        state["positions"] = (torch.randint(0, rows, (n,), generator=g, device=DEVICE, dtype=torch.int32)
                              if case["gather"] else None)
    else:
        b, page, kv, d = case["batch"], case["page"], case["kv_heads"], case["dim"]
        per = -(-case["longest"] // page)
        total = b * per + 3
        for name in ("k", "v"):
            spread = torch.exp(0.3 * normal(kv, 1, d))
            shift = normal(kv, 1, d) if name == "k" else torch.zeros(kv, 1, d, device=DEVICE)
            parts = [_quantise_4bit(normal(min(512, total - at), kv, page, d) * spread + 0.5 * shift)
                     for at in range(0, total, 512)]
            state[name + "_codes"] = torch.cat([p[0] for p in parts])
            state[name + "_params"] = torch.cat([p[1] for p in parts])
            del parts
        table = torch.randperm(total, generator=g, device=DEVICE)[:b * per].view(b, per).to(torch.int32)
        lengths = torch.tensor(_lengths(case), dtype=torch.int32, device=DEVICE)
        used = torch.arange(per, device=DEVICE)[None] * page < lengths[:, None]
        state["table"] = torch.where(used, table, torch.full_like(table, -1))
        state["lengths"] = lengths
        if case["op"] == "append":
            for name in ("k", "v"):
                state[name] = normal(b, case["new"], kv, d).to(t)
        else:
            gain = 1.0 + 2.0 * uniform(1, 1, case["heads"], 1)   # some heads look sharply, some evenly
            state["q"] = (gain * normal(b, case["new"], case["heads"], d)).to(t)
    return state


# --------------------------------------------------------------------------------------- one pass
def run(state):
    return _RUN[state["case"]["op"]](state)


def _run_linear(s):
    if own:
        from modiff_b200 import ops
        return ops.fp8_linear(s["x"], s["w"], s["w_scale"], s["bias"])
    x, w, scale = s["x"].float(), s["w"].float(), s["w_scale"]
    (rows, k), n = x.shape, w.shape[0]
    kb = -(-k // BLOCK)
    x = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).view(rows, kb, BLOCK)
    top = x.abs().amax(-1, keepdim=True)
    sx = torch.where(top > 0, top / E4M3_MAX, torch.ones_like(top))
    x = (x / sx).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).float() * sx
    w = w * scale.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    y = x.flatten(1)[:, :k] @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def _norm_plain(x, weight, cos, sin, interleaved):
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight
    rot, rest = y[..., :2 * cos.shape[-1]], y[..., 2 * cos.shape[-1]:]
    c, s = cos[:, None], sin[:, None]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if interleaved else rot.chunk(2, -1)
    a, b = a * c - b * s, b * c + a * s
    rot = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([rot, rest], -1).to(x.dtype)


def _run_norm(s):
    flip = s["case"]["interleaved"]
    if own:
        from modiff_b200 import ops
        return ops.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"],
                                s["positions"], eps=EPS, interleaved=flip)
    cos, sin = s["cos"], s["sin"]
    if s["positions"] is not None:
        at = s["positions"].long()
        cos, sin = cos[at], sin[at]
    return (_norm_plain(s["q"], s["q_weight"], cos, sin, flip),
            _norm_plain(s["k"], s["k_weight"], cos, sin, flip))


def _own_cache(s):
    from modiff_b200 import ops
    return ops.KV4Cache(s["k_codes"], s["k_params"], s["v_codes"], s["v_params"])


def _places(s, new):
    """Page and offset of the last `new` tokens of every sequence, and which of them exist."""
    page = s["case"]["page"]
    at = s["lengths"].long()[:, None] - new + torch.arange(new, device=DEVICE)
    there = at >= 0
    at = at.clamp(min=0)
    return s["table"].long().gather(1, at // page), at % page, there


def _run_append(s):
    new = s["case"]["new"]
    if own:
        from modiff_b200 import ops
        cache = _own_cache(s)
        ops.kv4_append(cache, s["k"], s["v"], s["table"], s["lengths"])
        return ops.kv4_read(cache, s["table"], s["lengths"], new)
    pages, offsets, there = _places(s, new)
    out = []
    for name in ("k", "v"):
        codes, params = _quantise_4bit(s[name])
        s[name + "_codes"][pages[there], :, offsets[there]] = codes[there]
        s[name + "_params"][pages[there], :, offsets[there]] = params[there]
        x = _dequantise_4bit(s[name + "_codes"][pages, :, offsets], s[name + "_params"][pages, :, offsets])
        out.append(torch.where(there[..., None, None], x, torch.zeros_like(x)))
    return tuple(out)


def _visible(case, lengths, tokens):
    """[batch, new, tokens]: whether a query sees a token."""
    t = torch.arange(tokens, device=DEVICE)[None, None]
    lengths = lengths.long()[:, None, None]
    sees = (t < lengths).expand(-1, case["new"], -1)
    if case["causal"]:
        at = lengths - case["new"] + torch.arange(case["new"], device=DEVICE)[None, :, None]
        sees = sees & (t <= at)
        if case["window"]:
            sees = sees & ((t > at - case["window"]) | (t < case["sinks"]))
    return sees


def _run_attention(s):
    c = s["case"]
    scale = c["dim"] ** -0.5
    if own:
        from modiff_b200 import ops
        return ops.kv4_attention(s["q"], _own_cache(s), s["table"], s["lengths"], scale,
                                 causal=c["causal"], window=c["window"], sinks=c["sinks"])
    b, new, kv, d = c["batch"], c["new"], c["kv_heads"], c["dim"]
    rep = c["heads"] // kv
    pages = s["table"].long().clamp(min=0)
    k, v = (_dequantise_4bit(s[x + "_codes"][pages], s[x + "_params"][pages]).transpose(1, 2).flatten(2, 3)
            for x in ("k", "v"))                                         # [batch, kv, tokens, dim]
    sees = _visible(c, s["lengths"], k.shape[2])
    q = s["q"].float().view(b, new, kv, rep, d).permute(0, 2, 3, 1, 4).reshape(b, kv, rep * new, d)
    score = (q @ k.transpose(2, 3)).view(b, kv, rep, new, -1) * scale
    score.masked_fill_(~sees[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.view(b, kv, rep * new, -1) @ v).view(b, kv, rep, new, d)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    return out.permute(0, 3, 1, 2, 4).reshape(b, new, c["heads"], d).to(s["q"].dtype)


_RUN = {"linear": _run_linear, "norm": _run_norm, "append": _run_append, "attention": _run_attention}


# ------------------------------------------------------------------------------------------- work
def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        scales = 4 * -(-n // BLOCK) * -(-k // BLOCK)
        return {"bytes": size * m * k + n * k + scales + size * m * n + (size * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    if case["op"] == "norm":
        x = case["tokens"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        angles = 4 * case["rot"] * min(case["tokens"], 8192 if case["gather"] else case["tokens"])
        return {"bytes": 2 * size * x + angles + (4 * case["tokens"] if case["gather"] else 0),
                "flops": 8 * x}
    kv, d, new = case["kv_heads"], case["dim"], case["new"]
    row = 2 * (d // 2 + 4)                       # codes, scale and minimum of a key and a value
    if case["op"] == "append":
        n = sum(min(new, length) for length in _lengths(case)) * kv
        return {"bytes": n * (2 * d * size + 2 * row + 8 * d), "flops": 10 * n * d}
    tokens = pairs = 0
    for length in _lengths(case):
        at = np.arange(max(0, length - new), length) if case["causal"] else np.full(new, length - 1)
        seen = at + 1
        first = np.zeros_like(at)
        if case["window"]:
            first = np.maximum(at - case["window"] + 1, 0)
            seen = at + 1 - first + np.minimum(first, case["sinks"])
        tokens += int(length - first[0] + min(int(first[0]), case["sinks"]))
        pairs += int(seen.sum())
    return {"bytes": tokens * kv * row + 2 * size * case["batch"] * new * case["heads"] * d,
            "flops": 4 * pairs * case["heads"] * d}


# -------------------------------------------------------------------------------- in 64 bits, apart
def exact(case, seed):
    """What run() returns, from the formulas above in 64 bits.  Scales, minima and quotients are what
    the formulas say they are, numbers of 32 and 16 bits; everything that is summed is not."""
    s = prepare(case, seed)
    return {"linear": _exact_linear, "norm": _exact_norm, "append": _exact_append,
            "attention": _exact_attention}[case["op"]](case, s)


def _exact_linear(case, s):
    m, k, n = case["rows"], case["k"], case["n"]
    y = torch.zeros(m, n, dtype=torch.float64, device=DEVICE)
    for at in range(0, k, BLOCK):
        x = s["x"][:, at:at + BLOCK].to(torch.float32)
        sx = x.abs().max(dim=1).values / torch.tensor(E4M3_MAX, device=DEVICE)
        sx[sx == 0] = 1.0
        quotient = torch.div(x, sx.unsqueeze(1)).clip(-E4M3_MAX, E4M3_MAX)
        part = quotient.to(torch.float8_e4m3fn).double() @ s["w"][:, at:at + BLOCK].double().T
        sw = s["w_scale"][:, at // BLOCK].double()
        y += part * sx.double().unsqueeze(1) * sw[torch.arange(n, device=DEVICE) // BLOCK]
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_norm(case, s):
    out = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        x = x.double()
        x = x / (x.pow(2).sum(-1, keepdim=True) / case["dim"] + EPS).sqrt() * w.double()
        half = case["rot"] // 2
        i = torch.arange(half, device=DEVICE)
        first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, half + i)
        at = torch.arange(case["tokens"], device=DEVICE) if s["positions"] is None else s["positions"].long()
        turn = torch.complex(s["cos"].double(), s["sin"].double())[at].unsqueeze(1)
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        out.append(x)
    return tuple(out)


def _exact_append(case, s):
    out = []
    for x in (s["k"], s["v"]):
        x = x.to(torch.float32)
        low, high = x.min(-1).values, x.max(-1).values
        step = (high - low).div(torch.tensor(15.0, device=DEVICE)).to(torch.float16)
        low = low.to(torch.float16)
        at = torch.div(x - low.float().unsqueeze(-1), step.float().unsqueeze(-1))
        at = torch.where(step.unsqueeze(-1) == 0, torch.zeros_like(at), at)
        value = at.round().clip(0, 15).double() * step.double().unsqueeze(-1) + low.double().unsqueeze(-1)
        for b, length in enumerate(_lengths(case)):
            value[b, :max(0, case["new"] - length)] = 0
        out.append(value)
    return tuple(out)


def _exact_attention(case, s):
    b, new, heads, d, page = case["batch"], case["new"], case["heads"], case["dim"], case["page"]
    out = torch.zeros(b, new, heads, d, dtype=torch.float64, device=DEVICE)
    shift = torch.tensor([0, 4], dtype=torch.uint8, device=DEVICE)
    for i, length in enumerate(_lengths(case)):
        ids = s["table"][i, :-(-length // page)].long()
        for h in range(heads):
            j = h // (heads // case["kv_heads"])
            k, v = ((((s[x + "_codes"][ids, j].unsqueeze(-1) >> shift) & 15).reshape(-1, d).double()
                     * s[x + "_params"][ids, j, :, 0].double().reshape(-1, 1)
                     + s[x + "_params"][ids, j, :, 1].double().reshape(-1, 1))[:length] for x in ("k", "v"))
            for at in range(0, new, 256):
                rows = torch.arange(at, min(new, at + 256), device=DEVICE)
                pos = (length - new + rows).unsqueeze(1)
                t = torch.arange(length, device=DEVICE).unsqueeze(0)
                hidden = torch.zeros(len(rows), length, dtype=torch.bool, device=DEVICE)
                if case["causal"]:
                    hidden |= t > pos
                if case["window"]:
                    hidden |= (t <= pos - case["window"]) & (t >= case["sinks"])
                score = s["q"][i, rows, h].double() @ k.T * (float(d) ** -0.5)
                score[hidden] = -math.inf
                p = torch.softmax(score, -1)
                p[hidden.all(-1)] = 0
                out[i, rows, h] = p @ v
    return out

"""Low-precision transformer operators: cached rows that are not finite."""
import math

import pytest
import torch

import lowp_reference as ref
from modiff_b200 import ops

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

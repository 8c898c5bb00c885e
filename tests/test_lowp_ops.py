"""Low-precision transformer operators (linear layers in 8-bit floating point, norms of queries and keys
with their rotation, the 4-bit cache and its attention) against plain restatements in 64 bits."""
import ctypes as C
import math

import pytest
import torch

import lowp_reference as ref
from modiff_b200 import ModiffError, _lib, lowp_ops, ops

TYPES = [torch.float32, torch.float16, torch.bfloat16]
gpu = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _close(got, want, tol):
    got = got.double().cpu()
    assert got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    off = (got - want).abs()[~nan] - tol[~nan]
    assert off.numel() == 0 or float(off.max()) <= 0, f"{float(off.max()):.3g} beyond the tolerance"


# ------------------------------------------------------------------------------- what is refused
def test_cpu_tensors_are_refused():
    x = torch.randn(2, 128)
    codes = torch.zeros(128, 128, dtype=torch.float8_e4m3fn)
    cache = ops.kv4_cache(2, 1, 16, 64, "cpu")
    table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    kv = torch.randn(1, 1, 1, 64)
    for call in (lambda: ops.fp8_quantize(x), lambda: ops.fp8_pack_weight(x),
                 lambda: ops.fp8_linear(x, codes, torch.ones(1, 1)),
                 lambda: ops.qk_norm_rope(kv, kv, None, None, torch.ones(1, 32), torch.ones(1, 32)),
                 lambda: ops.kv4_append(cache, kv, kv, table, lengths),
                 lambda: ops.kv4_read(cache, table, lengths, 1),
                 lambda: ops.kv4_attention(kv, cache, table, lengths)):
        with pytest.raises(ModiffError, match="CUDA"):
            call()


def test_cache_shapes_are_checked():
    for args in ((0, 1, 16, 64), (1, 0, 16, 64), (1, 1, 24, 64), (1, 1, 0, 64), (1, 1, 16, 80), (1, 1, 16, 320)):
        with pytest.raises(ModiffError):
            ops.kv4_cache(*args, "cpu")


def test_entry_points_refuse_bad_arguments_without_a_device():
    """The C entry points check before they touch a device: made-up addresses are never followed."""
    lib = _lib.lib()
    a = 1 << 20                                            # an aligned address nobody reads
    s2, s3 = (64, 64), (64, 64, 64)

    def cache(pages=4, heads=2, size=16, dim=64, at=a):
        return C.byref(_lib.Kv4CacheStruct(at, a, a, a, pages, heads, size, dim))

    def attend(c, q=a, heads=4, count=1, pages=1, causal=1, window=0, sinks=0, dtype=0):
        return lib.modiff_kv4_attention(q, *s3, c, a, a, a, 1, count, heads, pages, 1.0, causal, window, sinks, dtype,
                                        None, None)

    for rc in (attend(cache(size=24)), attend(cache(dim=96)), attend(cache(pages=0)), attend(cache(at=a + 8)),
               attend(cache(at=None)), attend(cache(), heads=3), attend(cache(), window=-1),
               attend(cache(), causal=0, window=4), attend(cache(), dtype=3), attend(cache(), q=None),
               attend(cache(), pages=0), attend(cache(), pages=1 << 28), attend(cache(), count=1 << 29),
               lib.modiff_kv4_append(cache(), a, *s3, a, *s3, a, a, 1, -1, 1, 0, None),
               lib.modiff_kv4_append(cache(), a + 1, *s3, a, *s3, a, a, 1, 1, 1, 0, None),
               lib.modiff_kv4_read(cache(), a, a, 1, 1, 1, a + 4, a, 0, None),
               lib.modiff_fp8_quantize(a, 64, 1, 0, 0, a, 64, a, 4, None),
               lib.modiff_fp8_quantize(a, 64, 1, 64, 0, a, 72, a, 4, None),
               lib.modiff_fp8_quantize(a, 64, 1, 64, 0, a, 48, a, 4, None),
               lib.modiff_fp8_quantize(a, 64, 1, 64, 0, a, 64, a, 6, None),
               lib.modiff_fp8_quantize(a, 64, 5, 64, 0, a, 64, a, 4, None),
               lib.modiff_fp8_pack_weight(a, 64, 1, 64, 0, a, 128, a, 1, None),
               lib.modiff_fp8_linear(a, 64, a, 4, a, 72, a, 1, None, a, 8, 1, 64, 8, 0, None),
               lib.modiff_fp8_linear(a, 64, a, 4, a, 64, a, 1, None, a, 7, 1, 64, 8, 0, None),
               lib.modiff_fp8_linear(a + 8, 64, a, 4, a, 64, a, 1, None, a, 8, 1, 64, 8, 0, None),
               lib.modiff_fp8_linear(a, 64, a, 4, a, 64, a, 1, None, a, 8, 1, 64, 8, 7, None),
               lib.modiff_fp8_linear(a, 64, a, 5, a, 64, a, 1, None, a, 8, 1, 64, 8, 0, None),
               lib.modiff_fp8_linear_x(a, 64, a, 64, a, 1, None, a, 8, 40, 64, 8, 0, None, None),
               lib.modiff_fp8_linear_x(a, 64, a, 72, a, 1, None, a, 8, 40, 64, 8, 0, a, None),
               lib.modiff_fp8_linear_x(None, 64, a, 64, a, 1, None, a, 8, 1, 64, 8, 0, a, None),
               lib.modiff_qk_norm_rope(a, *s2, a, *s2, 1, a, *s2, a, *s2, 1, None, None, a, a, 8, a, 0, 8, 63, 32, 0, 1e-6,
                                       0, None),
               lib.modiff_qk_norm_rope(a, *s2, a, *s2, 1, a, *s2, a, *s2, 1, None, None, a, a, 8, a, 0, 8, 64, 66, 0, 1e-6,
                                       0, None),
               lib.modiff_qk_norm_rope(a, *s2, a, *s2, 1, a, *s2, a, *s2, 1, None, None, a, a, 7, None, 0, 8, 64, 64, 0,
                                       1e-6, 0, None),
               lib.modiff_qk_norm_rope(a, *s2, a, *s2, 1, a, *s2, a, *s2, 1, None, None, None, a, 8, a, 0, 8, 64, 64, 0,
                                       1e-6, 0, None)):
        assert rc == 1 and lib.modiff_last_error()
    # nothing to do is not an error, and touches nothing
    assert lib.modiff_fp8_quantize(None, 64, 0, 64, 0, None, 64, None, 1, None) == 0
    assert lib.modiff_kv4_append(cache(), a, *s3, a, *s3, a, a, 1, 0, 1, 0, None) == 0


def test_arguments_as_words():
    """Words for every entry of the packed call, and its refusals."""
    lib = _lib.lib()
    cache = {"modiff_kv4_append", "modiff_kv4_read", "modiff_kv4_attention", "modiff_kv4_attention_bytes"}
    for name in _lib.PACKED:
        pack = lowp_ops._PACK.get(name, lowp_ops._PACK_BYTES).__self__
        assert pack.size == 8 * len(_lib.SIGNATURES[name][1]) + (40 if name in cache else 0)
    assert lib.modiff_packed_call(0, None) == 1 and lib.modiff_packed_call(99, bytes(8 * 30)) == 1
    assert lib.modiff_packed_call(0, bytes(80)) == 1 and lib.modiff_last_error()      # no shape
    words = lowp_ops._PACK_BYTES(0, 0, 0, 0, 64, 2, 64, 128, 1, 1, 8, 64, 0, 0, 1)
    c = C.byref(_lib.Kv4CacheStruct(None, None, None, None, 64, 2, 64, 128))
    assert lib.modiff_packed_call(7, words) == lib.modiff_kv4_attention_bytes(c, 1, 1, 8, 64, 0, 0, 1) > 0


def test_entry_points_refuse_sizes_beyond_their_index_types():
    lib = _lib.lib()
    a, most = 1 << 20, 0x7fffff00
    s2, s3 = (64, 64), (64, 64, 64)
    cache = C.byref(_lib.Kv4CacheStruct(a, a, a, a, 4, 1 << 20, 16, 64))
    for rc in (lib.modiff_fp8_linear(a, 16, a, most + 4, a, 16, a, 1, None, a, 1, most + 1, 16, 1, 0, None),
               lib.modiff_fp8_linear_x(a, 16, a, 16, a, 1, None, a, 1, most + 1, 16, 1, 0, a, None),
               lib.modiff_fp8_quantize(a, 16, 1 << 40, 16, 0, a, 16, a, 1 << 40, None),
               lib.modiff_fp8_quantize(a, 1 << 31, 1, most + 1, 0, a, 1 << 31, a, 4, None),
               lib.modiff_kv4_append(cache, a, *s3, a, *s3, a, a, 64, 32, 1, 0, None),
               lib.modiff_kv4_read(cache, a, a, 64, 32, 1, a, a, 0, None),
               lib.modiff_qk_norm_rope(a, *s2, a, *s2, 1, None, *s2, None, *s2, 0, None, None, a, a, 8, a, 0, 1 << 31, 64, 64,
                                       0, 1e-6, 0, None),
               lib.modiff_qk_norm_rope(a, *s2, a, *s2, 1, None, *s2, None, *s2, 0, None, None, a, a, 8, a + 4, 1, 1, 64, 64,
                                       0, 1e-6, 0, None)):
        assert rc == 1 and lib.modiff_last_error()
    assert lib.modiff_fp8_linear_bytes(most + 1, 16, 1) == 0


@gpu
def test_arguments_are_checked(cuda):
    x = torch.randn(4, 256, device=cuda)
    w, ws = ops.fp8_pack_weight(torch.randn(8, 256, device=cuda))
    cos = torch.ones(4, 32, device=cuda)
    q = torch.randn(1, 4, 2, 64, device=cuda)
    cache = ops.kv4_cache(2, 1, 16, 64, cuda)
    table, lengths = torch.zeros(1, 1, dtype=torch.int32, device=cuda), torch.ones(1, dtype=torch.int32, device=cuda)
    kv = torch.randn(1, 1, 1, 64, device=cuda)
    odd, _ = ops.fp8_pack_weight(torch.randn(8, 250, device=cuda))
    for call in (lambda: ops.fp8_linear(x[:, :128], w, ws), lambda: ops.fp8_linear(x, w, ws[:, :1]),
                 lambda: ops.fp8_linear(x, w.float(), ws), lambda: ops.fp8_linear(x.double(), w, ws),
                 lambda: ops.fp8_linear(x, w, ws, torch.zeros(8, device=cuda, dtype=torch.half)),
                 lambda: ops.fp8_linear(x, w, ws, torch.zeros(9, device=cuda)),
                 lambda: ops.fp8_linear(x[:, :250], odd.contiguous(), ws),
                 lambda: ops.fp8_linear(x, w, ws.cpu()),
                 lambda: ops.fp8_linear(x.clone().requires_grad_(), w, ws),
                 lambda: ops.fp8_quantize(x[:, :0]), lambda: ops.fp8_pack_weight(x[0]),
                 lambda: ops.qk_norm_rope(q, q.half(), None, None, cos, cos),
                 lambda: ops.qk_norm_rope(q, None, None, None, cos[:3], cos[:3]),
                 lambda: ops.qk_norm_rope(q[..., :63], None, None, None, cos, cos),
                 lambda: ops.qk_norm_rope(q, None, torch.ones(64, device=cuda).half(), None, cos, cos),
                 lambda: ops.qk_norm_rope(q, None, None, None, cos, cos, positions=torch.zeros(3, device=cuda).int()),
                 lambda: ops.qk_norm_rope(q, None, None, None, cos, cos, positions=torch.zeros(4, device=cuda)),
                 lambda: ops.qk_norm_rope(q, None, None, None, cos, cos, out=(q[..., ::2], None)),
                 lambda: ops.kv4_append(cache, kv, kv.half(), table, lengths),
                 lambda: ops.kv4_append(cache, kv.expand(1, 1, 2, 64), kv.expand(1, 1, 2, 64), table, lengths),
                 lambda: ops.kv4_append(cache, kv, kv, table.long(), lengths),
                 lambda: ops.kv4_attention(kv, cache, table, lengths, sinks=2),
                 lambda: ops.kv4_attention(kv, cache, table, lengths, causal=False, window=4),
                 lambda: ops.kv4_attention(kv[..., :32], cache, table, lengths),
                 lambda: ops.kv4_attention(kv, cache, table, torch.ones(2, dtype=torch.int32, device=cuda)),
                 lambda: ops.kv4_read(cache, table, lengths, 1, torch.float64)):
        with pytest.raises(ModiffError):
            call()
    with torch.no_grad():
        ops.fp8_linear(x.clone().requires_grad_(), w, ws)


# --------------------------------------------------------------------------- 8-bit linear layers
@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 5), (1, 128), (7, 130), (33, 1280), (5, 2001), (300, 320)])
def test_fp8_quantize_bits(cuda, rows, k, dtype):
    x = (torch.randn(rows, k, generator=_gen(rows + k)) * torch.randn(rows, 1, generator=_gen(k)).exp()).to(dtype)
    if k >= 128:
        x[0, :128] = 0                                     # an empty block
        x[-1, :64] *= 2.0 ** -12                           # codes below e4m3's normal range
    codes, scale, t = ops.fp8_quantize(x.to(cuda))
    want, s = ref.e4m3_rows(x)
    assert t == dtype and torch.equal(scale.cpu(), s) and torch.equal(codes.float().cpu(), want)


@gpu
def test_fp8_quantize_extremes_and_strides(cuda):
    x = torch.randn(6, 300, generator=_gen(2))
    x[0, 5], x[1, 140], x[2, 299], x[3, 0] = math.inf, -math.inf, math.nan, 3.4e38
    x[4] *= 1e-38
    x[5] = 1e-45                                           # the smallest number: its scale is one too
    codes, scale, _ = ops.fp8_quantize(x.to(cuda))
    want, s = ref.e4m3_rows(x)
    y, z = codes.float().cpu() * scale.cpu().repeat_interleave(128, 1)[:, :300], want * s.repeat_interleave(128, 1)[:, :300]
    clean = torch.ones(6, 300, dtype=torch.bool)
    clean[0, :128] = clean[1, 128:256] = clean[2, 256:] = False
    assert torch.equal(y[clean], z[clean])
    for r, c in ((0, 5), (1, 140), (2, 299)):              # not a number where one was none
        assert torch.isnan(y[r, c])
    wide = torch.randn(9, 700, generator=_gen(3), dtype=torch.float32).to(cuda)
    for view in (wide[:, 3:303], wide[::2, :300], wide.t()[:300, :], wide.view(3, 3, 700)[..., 64:192]):
        got, plain = ops.fp8_quantize(view), ops.fp8_quantize(view.contiguous())
        assert got.codes.shape == view.shape
        assert torch.equal(got.codes.float(), plain.codes.float()) and torch.equal(got.scale, plain.scale)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k", [(1, 1), (5, 130), (128, 128), (300, 77), (129, 640)])
def test_fp8_pack_weight_bits(cuda, n, k, dtype):
    w = torch.randn(n, k, generator=_gen(n * k)).to(dtype)
    codes, scale = ops.fp8_pack_weight(w.to(cuda))
    want, s = ref.e4m3_blocks(w)
    assert codes.shape == (n, k) and torch.equal(codes.float().cpu(), want) and torch.equal(scale.cpu(), s)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k,n", [
    (1, 1, 1), (1, 16, 8), (2, 128, 128), (15, 77, 130), (16, 1280, 640), (17, 300, 33), (31, 2001, 129),
    (64, 5120, 320), (65, 640, 1280), (100, 33, 7), (154, 768, 640), (129, 129, 257), (257, 1000, 520),
    (1000, 320, 2560), (2500, 1411, 1030), (4096, 640, 768), (1300, 129, 1001), (65, 136, 20000), (64, 256, 9600),
    (512, 1000, 1000), (70, 4200, 2049), (8, 2048, 130)])
def test_fp8_linear(cuda, rows, k, n, dtype):
    g = _gen(rows + 3 * k + 7 * n)
    x = (torch.randn(rows, k, generator=g) * torch.randn(1, k, generator=g).exp()).to(dtype)
    w = torch.randn(n, k, generator=g) * torch.randn(n, 1, generator=g).exp()
    bias = torch.randn(n, generator=g).to(dtype)
    codes, scale = ops.fp8_pack_weight(w.to(cuda))
    packed = (codes.float().cpu(), scale.cpu())
    for b in (bias, None):
        got = ops.fp8_linear(x.to(cuda), codes, scale, None if b is None else b.to(cuda))
        assert got.dtype == dtype and got.shape == (rows, n)
        y, size = ref.linear(*ref.e4m3_rows(x), *packed, b)
        _close(got, y, ref.linear_tolerance(y, size, k, dtype))
    again = ops.fp8_linear(x.to(cuda), codes, scale)
    assert torch.equal(got, again)                         # no order that changes from call to call
    assert _lib.device_status() == 0


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pitch", [1001, 1002, 1004, 1016])
@pytest.mark.parametrize("rows", [3, 100, 1300])
def test_fp8_linear_writes_nothing_beside_its_rows(cuda, rows, pitch, dtype):
    """Results as a part of wider rows, on every alignment that a row can start on."""
    k, n = 200, 1001
    x = torch.randn(rows, k, generator=_gen(rows)).to(cuda, dtype)
    w, s = ops.fp8_pack_weight(torch.randn(n, k, generator=_gen(1)).to(cuda))
    y = torch.full((rows + 1, pitch), 7.0, dtype=dtype, device=cuda)
    q = ops.fp8_quantize(x)
    assert _lib.lib().modiff_fp8_linear(
        q.codes.data_ptr(), 208, q.scale.data_ptr(), -(-rows // 4) * 4, w.data_ptr(), 208, s.data_ptr(), 2, None,
        y.data_ptr(), pitch, rows, k, n, TYPES.index(dtype), torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(y[:rows, :n], ops.fp8_linear(q, w, s))
    assert (y[:rows, n:] == 7).all() and (y[rows] == 7).all()


@gpu
def test_fp8_linear_shapes_and_shared_rows(cuda):
    x = torch.randn(3, 5, 200, generator=_gen(5)).to(cuda).bfloat16()
    w, s = ops.fp8_pack_weight(torch.randn(48, 200, generator=_gen(6)).to(cuda))
    plain = ops.fp8_linear(x.view(15, 200), w, s)
    rows = ops.fp8_quantize(x)
    assert torch.equal(ops.fp8_linear(x, w, s), plain.view(3, 5, 48))
    assert torch.equal(ops.fp8_linear(rows, w, s), plain.view(3, 5, 48))
    assert torch.equal(ops.fp8_linear(x[1, 2], w, s), plain[7])
    assert ops.fp8_linear(x[:0], w, s).shape == (0, 5, 48)
    with pytest.raises(ModiffError):                       # rows that are not laid out as they came
        ops.fp8_linear(ops.Fp8Rows(rows.codes[:, ::2], rows.scale[:, ::2], rows.dtype), w, s)


@gpu
def test_fp8_linear_not_a_number_stays_in_its_row(cuda):
    x = torch.randn(130, 256, generator=_gen(8))
    x[3, 7], x[129, 200] = math.nan, math.inf
    w, s = ops.fp8_pack_weight(torch.randn(64, 256, generator=_gen(9)).to(cuda))
    for lo, hi in ((0, 130), (0, 4), (128, 130)):
        bad = torch.isnan(ops.fp8_linear(x[lo:hi].to(cuda), w, s)).cpu()
        want = torch.tensor([r in (3, 129) for r in range(lo, hi)])
        assert torch.equal(bad.all(1), want) and torch.equal(bad.any(1), want)


# --------------------------------------------------------------------- norms of queries and keys
@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hk,d,rot", [
    (1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (3, 5, 1, 40, 40), (77, 8, 8, 40, 20), (5, 7, 0, 6, 4), (130, 3, 2, 66, 34),
    (9, 4, 4, 80, 0), (1500, 8, 2, 64, 64), (2, 2, 1, 256, 128), (11, 3, 3, 250, 2), (700, 16, 4, 128, 64)])
def test_qk_norm_rope(cuda, tokens, hq, hk, d, rot, interleaved, dtype):
    g = _gen(tokens * 5 + d + rot)
    qkv = (3 * torch.randn(tokens, (hq + 2 * hk) * d, generator=g)).to(dtype)
    q, k = qkv[:, :hq * d].unflatten(1, (hq, d)), qkv[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d)) if hk else None
    wq, wk = 1 + 0.2 * torch.randn(d, generator=g), torch.randn(d, generator=g)
    angle = torch.randn(2000, rot // 2, generator=g) * 3
    cos, sin = angle.cos(), angle.sin()
    at = torch.randint(0, 2000, (tokens,), generator=g)
    dev = qkv.to(cuda)
    q_, k_ = (dev[:, :hq * d].unflatten(1, (hq, d)), dev[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d)) if hk else None)
    for pos, weights in ((at.int(), (wq, wk)), (at, (None, None)), (None, (wq, None))):
        got = ops.qk_norm_rope(q_, k_, *(None if w is None else w.to(cuda) for w in weights), cos.to(cuda), sin.to(cuda),
                               None if pos is None else pos.to(cuda), eps=1e-5, interleaved=interleaved)
        for y, x, w in zip(got, (q, k), weights):
            if x is None:
                assert y is None
                continue
            want, size = ref.norm_rope(x, w, cos, sin, pos, 1e-5, interleaved)
            assert y.dtype == dtype
            # the smallest of fp16's results lie below its normal range
            _close(y, want, ref.norm_tolerance(want, size, d, dtype) + (2.0 ** -25 if dtype == torch.float16 else 0))
    # in place, on the projection's own memory: the values behind the keys stay as they were
    got = ops.qk_norm_rope(q_, k_, None, None, cos.to(cuda), sin.to(cuda), interleaved=interleaved)
    ops.qk_norm_rope(q_, k_, None, None, cos.to(cuda), sin.to(cuda), interleaved=interleaved, out=(q_, k_))
    assert torch.equal(q_, got[0]) and (hk == 0 or torch.equal(k_, got[1]))
    assert torch.equal(dev[:, (hq + hk) * d:].cpu(), qkv[:, (hq + hk) * d:])


@gpu
def test_qk_norm_rope_far_and_bad_positions(cuda):
    q = torch.randn(2, 3, 4, 64, generator=_gen(1)).to(cuda)
    cos = torch.randn(100, 32, generator=_gen(2)).to(cuda)
    at = torch.tensor([[0, 99, 100], [-1, 2 ** 40, 50]], device=cuda)
    y, none = ops.qk_norm_rope(q, None, None, None, cos, cos, at)
    want, size = ref.norm_rope(q.cpu().flatten(0, 1), None, cos, cos, at, 1e-6, False)
    assert none is None and torch.isnan(want).any()
    _close(y.flatten(0, 1), want, ref.norm_tolerance(want, size, 64, torch.float32))
    zero = ops.qk_norm_rope(torch.zeros_like(q), None, None, None, cos, cos, torch.zeros(6, device=cuda).int())[0]
    assert torch.equal(zero, torch.zeros_like(zero))
    assert ops.qk_norm_rope(q[:, :0], q[:, :0], None, None, cos, cos)[1].shape == (2, 0, 4, 64)


# ------------------------------------------------------------------------------- the 4-bit cache
def _filled(cuda, batch, per, kv_heads, page, d, seed, spare=2):
    """A cache of random content (every place, also those that no sequence owns), tables of its pages in
    random order."""
    g = _gen(seed)
    total = batch * per + spare
    parts = [ref.quantise_4bit(torch.randn(total, kv_heads, page, d, generator=g) * 1.5 + 0.3) for _ in range(2)]
    cache = ops.KV4Cache(*(t.to(cuda) for p in parts for t in p))
    table = torch.randperm(total, generator=g)[:batch * per].view(batch, per).int().to(cuda)
    return cache, table


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,n,lengths,kv_heads,page,d", [
    (1, 1, [1], 1, 16, 64), (3, 1, [5, 0, 33], 2, 16, 128), (2, 40, [40, 17], 3, 16, 192), (4, 7, [7, 64, 3, 50], 1, 32, 256),
    (2, 100, [111, 100], 8, 64, 128), (1, 33, [48], 5, 48, 64)])
def test_kv4_append_bits(cuda, batch, n, lengths, kv_heads, page, d, dtype):
    per = 4 if page < 32 else 3
    cache, table = _filled(cuda, batch, per, kv_heads, page, d, n)
    before = [t.clone() for t in cache]
    g = _gen(d)
    k, v = (torch.randn(batch, n, kv_heads, d, generator=g).mul(4).to(dtype) for _ in range(2))
    k[0, 0, 0], v[-1, -1, -1, :] = 0.25, 70000.0 if dtype != torch.float16 else math.inf
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    ops.kv4_append(cache, k.to(cuda), v.to(cuda), table, lens)
    want = [t.cpu().clone() for t in before]
    for b in range(batch):
        for i in range(n):
            at = lengths[b] - n + i
            if at < 0 or at // page >= per:
                continue
            place = (int(table[b, at // page]), slice(None), at % page)
            for x, c, p in ((k, 0, 1), (v, 2, 3)):
                want[c][place], want[p][place] = ref.quantise_4bit(x[b, i])
    for got, w in zip(cache, want):                        # every other place as it was
        assert torch.equal(got.cpu().view(torch.uint8), w.view(torch.uint8))
    rk, rv = ops.kv4_read(cache, table, lens, n)
    for got, x in ((rk, k), (rv, v)):
        codes, params = ref.quantise_4bit(x)
        q, s, m = ref.values_4bit(codes, params)
        value = s[..., None] * q + m[..., None]
        for b in range(batch):
            value[b, :max(0, n - lengths[b])] = 0
        assert float((got.double().cpu() - value).abs().max()) <= 2.0 ** -24 * float(value.abs().max())
    half = ops.kv4_read(cache, table, lens, n, torch.bfloat16)[0]
    assert torch.equal(half, rk.bfloat16())


@gpu
def test_kv4_append_odd_inputs(cuda):
    cache, table = _filled(cuda, 2, 2, 2, 16, 64, 4)
    before = [t.clone() for t in cache]
    lens = torch.tensor([20, 9], dtype=torch.int32, device=cuda)
    kv = torch.randn(2, 2, 3, 2, 70, generator=_gen(5)).to(cuda)
    k, v = kv[0, ..., 3:67], kv[1, ..., 3:67]              # neither aligned nor contiguous
    bad = table.clone()
    bad[0, 1], bad[1, 0] = -1, 6                           # no such page: nothing is written
    ops.kv4_append(cache, k, v, bad, lens)
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    assert float(ops.kv4_read(cache, bad, lens, 3)[0].abs().max()) == 0
    for odd in (-5, -2 ** 31, 2 ** 31 - 1, 33):            # lengths that name no place of the table
        ops.kv4_append(cache, k, v, table, torch.full_like(lens, odd) if odd != 33 else lens * 0)
        assert all(torch.equal(a, b) for a, b in zip(cache, before))
    ops.kv4_append(cache, k, v, table, lens)
    other = ops.KV4Cache(*(t.clone() for t in before))
    ops.kv4_append(other, k.contiguous(), v.contiguous(), table, lens)
    assert all(torch.equal(a, b) for a, b in zip(cache, other))
    k = k.contiguous()
    k[0, 0, 0, 5] = math.nan
    ops.kv4_append(cache, k, v, table, lens)
    rk = ops.kv4_read(cache, table, lens, 3)[0]
    bad_rows = torch.isnan(rk).any(-1)
    assert bool(torch.isnan(rk[0, 0, 0]).all()) and int(bad_rows.sum()) == 1
    assert ops.kv4_append(cache, k[:, :0], v[:, :0], table, lens) is None


@gpu
@pytest.mark.parametrize("k", [1, 100, 128, 300])
def test_fp8_quantize_writes_nothing_beyond_its_rows(cuda, k):
    """Codes as a part of wider rows: zeros up to the next multiple of 16, nothing behind that."""
    rows, pitch, k16 = 5, 512, -(-k // 16) * 16
    x = torch.randn(rows, k, generator=_gen(k)).to(cuda)
    codes = torch.full((rows + 1, pitch), 0x55, dtype=torch.uint8, device=cuda)
    scale = torch.full((-(-k // 128) + 1, 8), -1.0, device=cuda)
    assert _lib.lib().modiff_fp8_quantize(x.data_ptr(), k, rows, k, 0, codes.data_ptr(), pitch, scale.data_ptr(), 8,
                                          torch.cuda.current_stream().cuda_stream) == 0
    want = ops.fp8_quantize(x)
    assert torch.equal(codes[:rows, :k], want.codes.view(torch.uint8))
    assert torch.equal(scale[:-1, :rows].t(), want.scale)
    assert not codes[:rows, k:k16].any() and (codes[:rows, k16:] == 0x55).all() and (codes[rows] == 0x55).all()
    assert (scale[-1] == -1).all()


# ------------------------------------------------------------------------------ cached attention
def _attend(cuda, lengths, n, heads, kv_heads, page, d, dtype, seed=0, gain=2.0, per=None, **kw):
    batch = len(lengths)
    per = per or max(1, -(-max(lengths) // page))
    cache, table = _filled(cuda, batch, per, kv_heads, page, d, seed + d)
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    q = (gain * torch.randn(batch, n, heads, d, generator=_gen(seed))).to(dtype)
    got = ops.kv4_attention(q.to(cuda), cache, table, lens, **kw)
    want, tol = ref.attention(q, cache, table, lens, **{"scale": d ** -0.5, **kw})
    assert got.dtype == dtype
    _close(got, want, tol)
    return q, cache, table, lens, got


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("lengths,n,heads,kv_heads,page", [
    ([1], 1, 1, 1, 16), ([0, 3, 65], 1, 8, 2, 16), ([200], 1, 5, 1, 64), ([63, 64, 129], 2, 14, 2, 32),
    ([70, 5], 9, 8, 4, 16), ([40], 40, 2, 2, 48), ([300, 90], 33, 3, 1, 128)])
def test_kv4_attention(cuda, lengths, n, heads, kv_heads, page, d, dtype):
    _attend(cuda, lengths, n, heads, kv_heads, page, d, dtype, seed=n)


@gpu
@pytest.mark.parametrize("dtype,gain", [(torch.float32, 2.0), (torch.float16, 2.0), (torch.float16, 0.01)])
@pytest.mark.parametrize("lengths,n,heads,kv_heads,d", [
    ([4000], 1, 8, 2, 128), ([900, 10], 2, 10, 5, 64), ([1, 30], 1, 7, 1, 256), ([600], 7, 8, 1, 128),
    ([16000] * 4, 1, 64, 64, 64)])
def test_kv4_attention_is_as_exact_as_its_type(cuda, lengths, n, heads, kv_heads, d, dtype, gain):
    """Few query rows.  Root mean squares: weights of 22 bits (2^-23 of each), scores of magnitude 16 at most
    from products and sums in fp32 that are cut at 2^-23 of sums no larger than 16 times the score (their error
    is that of the weight: 16 * 16 * 2^-23 = 2^-15 at worst, in the mean over signs and sizes an eighth), sums
    of numbers of both signs, rounded at every sixteen tokens (the errors of 16000 tokens' sums, of either sign,
    are 2^-24 sqrt(16000 / 16) = 2^-19 of a part of the sum at worst).  So 2^-18 in all; beside fp16's rounding, 0.84 * 2^-12 in the mean over a binade,
    that adds less than a thousandth, and the test leaves a tenth."""
    q, cache, table, lens, got = _attend(cuda, lengths, n, heads, kv_heads, 16, d, dtype, seed=11, gain=gain)
    want, _ = ref.attention(q, cache, table, lens, d ** -0.5)
    off = (got.double().cpu() - want).norm()
    if dtype == torch.float32:
        assert off <= 2.0 ** -18 * want.norm()
    else:
        assert off <= 1.1 * (want.half().double() - want).norm()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,kw", [
    (1, dict(window=1)), (1, dict(window=50)), (1, dict(window=70, sinks=4)), (1, dict(window=64, sinks=100)),
    (5, dict(window=3, sinks=1)), (30, dict(window=17)), (30, dict(window=100, sinks=33)),
    (150, dict(window=65, sinks=4)), (7, dict(window=10 ** 9, sinks=3)), (1, dict(causal=False)),
    (20, dict(causal=False)), (300, dict(causal=False))])
def test_kv4_attention_masks(cuda, n, kw, dtype):
    _attend(cuda, [290, 0, 131, 12], n, 6, 2, 16, 64, dtype, seed=n, **kw)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths,n,heads,kv_heads,d,kw", [
    ([6000, 17], 1, 8, 1, 128, {}), ([5000], 3, 8, 2, 64, {}), ([4500], 1, 4, 1, 256, dict(window=3000, sinks=200)),
    ([2100], 40, 4, 1, 128, {})])
def test_kv4_attention_split_over_tokens(cuda, lengths, n, heads, kv_heads, d, kw, dtype):
    """Long caches of few sequences: parts of the tokens in several blocks, joined afterwards."""
    q, cache, table, lens, got = _attend(cuda, lengths, n, heads, kv_heads, 64, d, dtype, **kw)
    for _ in range(3):
        assert torch.equal(ops.kv4_attention(q.to(cuda), cache, table, lens, **kw), got)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths,n,heads,kv_heads,page,d,kw", [
    ([64], 64, 1, 1, 16, 64, {}), ([128], 128, 1, 1, 64, 128, {}), ([129, 700], 129, 2, 2, 48, 128, {}),
    ([257], 257, 1, 1, 16, 64, dict(causal=False)), ([500, 130, 0, 3], 130, 6, 2, 32, 128, {}),
    ([400], 65, 8, 1, 128, 128, dict(window=30, sinks=2)), ([900], 300, 2, 1, 64, 64, dict(window=200, sinks=140)),
    ([6000], 33, 4, 1, 64, 128, {}), ([4100], 16, 8, 1, 64, 64, dict(window=3000, sinks=5))])
def test_kv4_attention_of_many_rows(cuda, lengths, n, heads, kv_heads, page, d, kw, dtype):
    q, cache, table, lens, got = _attend(cuda, lengths, n, heads, kv_heads, page, d, dtype, seed=n, **kw)
    for _ in range(2):
        assert torch.equal(ops.kv4_attention(q.to(cuda), cache, table, lens, **kw), got)
    assert _lib.device_status() == 0


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0])
def test_kv4_attention_scale(cuda, scale, dtype):
    for n in (1, 70):
        _attend(cuda, [150, 71], n, 2, 2, 16, 64, dtype, seed=5, gain=0.7, scale=scale)


@gpu
@pytest.mark.parametrize("n", [1, 20, 40])
def test_kv4_attention_never_meets_hidden_tokens(cuda, n):
    """Infinities and NaN behind the last token, outside the window and in pages that are not there."""
    lengths, page, d = [100, 37], 16, 64
    cache, table = _filled(cuda, 2, 8, 2, page, d, 3)
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    q = torch.randn(2, n, 4, d, generator=_gen(7)).to(cuda)
    if n == 40:
        q = q.half()                                       # rows enough for the kernel of many rows
    kw = dict(window=n + 30, sinks=2)
    clean = ops.kv4_attention(q, cache, table, lens, **kw)
    for b, length in enumerate(lengths):
        for t in range(8 * page):
            if t >= length or (2 <= t <= length - n - kw["window"]):
                for p in (cache.k_params, cache.v_params):
                    p[int(table[b, t // page]), :, t % page] = math.nan if t % 2 else math.inf
    table[0, 100 // page + 1:] = -1                        # never read
    table[1, 37 // page + 1:] = 2 ** 31 - 1
    assert torch.equal(ops.kv4_attention(q, cache, table, lens, **kw), clean)
    if n == 40:                                            # a value that only the later queries may meet
        cache.v_params[int(table[0, 80 // page]), :, 80 % page, 1] = math.nan
        got = ops.kv4_attention(q, cache, table, lens, **kw)
        assert bool(torch.isnan(got[0, 20:]).all()) and torch.equal(got[0, :20], clean[0, :20])
        assert torch.equal(got[1], clean[1])
    # a page that is missing in the middle: its tokens are not seen
    table[0, 5] = 18
    got = ops.kv4_attention(q, cache, table, lens)
    want, tol = ref.attention(q.cpu(), cache, table, lens, d ** -0.5)
    ok = ~torch.isnan(want).any(-1)
    _close(got[ok.to(cuda)], want[ok], tol[ok])


@gpu
def test_kv4_attention_scales_of_any_size(cuda):
    """Tokens whose values are tiny, huge or constant, and queries far from 1."""
    g = _gen(11)
    lengths, page, d = [200], 16, 128
    size = torch.exp(8 * torch.randn(1, 200, 1, 1, generator=g)).clamp(1e-6, 3e4)
    for dtype, gain in ((torch.float32, 1e-3), (torch.float32, 3.0), (torch.bfloat16, 1e4), (torch.float16, 0.5)):
        cache = ops.kv4_cache(14, 2, page, d, cuda)
        table = torch.arange(13, dtype=torch.int32, device=cuda)[None].flip(1).contiguous()
        lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
        k = torch.randn(1, 200, 2, d, generator=g) / max(1.0, gain)
        v = torch.randn(1, 200, 2, d, generator=g) * size
        v[:, 50:60] = 7.5                                  # a scale of 0
        ops.kv4_append(cache, k.to(cuda), v.to(cuda), table, lens)
        q = (gain * torch.randn(1, 1, 8, d, generator=g)).to(dtype)
        got = ops.kv4_attention(q.to(cuda), cache, table, lens)
        want, tol = ref.attention(q, cache, table, lens, d ** -0.5)
        _close(got, want, tol)
    constant = ops.kv4_cache(1, 1, 16, 64, cuda)           # all scales 0
    one = torch.full((1, 3, 1, 64), 2.0, device=cuda)
    tab, lens = torch.zeros(1, 1, dtype=torch.int32, device=cuda), torch.tensor([3], dtype=torch.int32, device=cuda)
    ops.kv4_append(constant, one, one, tab, lens)
    assert torch.equal(ops.kv4_attention(one[:, :1], constant, tab, lens), one[:, :1])


@gpu
def test_kv4_attention_strided_queries_and_empty_batches(cuda):
    cache, table = _filled(cuda, 2, 3, 2, 16, 64, 1)
    lens = torch.tensor([40, 20], dtype=torch.int32, device=cuda)
    qkv = torch.randn(2, 5, 8 * 64 + 3, generator=_gen(2)).to(cuda).half()
    q = qkv[..., 3:3 + 4 * 64].unflatten(2, (4, 64))
    plain = ops.kv4_attention(q.contiguous(), cache, table, lens)
    assert torch.equal(ops.kv4_attention(q, cache, table, lens), plain)
    assert torch.equal(ops.kv4_attention(q.transpose(1, 2).contiguous().transpose(1, 2), cache, table, lens), plain)
    assert ops.kv4_attention(q[:, :0], cache, table, lens).shape == (2, 0, 4, 64)
    assert ops.kv4_attention(q[:0], cache, table[:0], lens[:0]).shape == (0, 5, 4, 64)
    none = ops.kv4_attention(q, cache, table, lens * 0)
    assert torch.equal(none, torch.zeros_like(none))
    more = ops.kv4_attention(q, cache, table, lens * 0 + 10 ** 9)   # more than the table holds
    assert torch.equal(more, ops.kv4_attention(q, cache, table, lens * 0 + 48))
    nan = q.clone()
    nan[0, 1, 2, 3] = math.nan
    bad = torch.isnan(ops.kv4_attention(nan, cache, table, lens))
    assert bool(bad[0, 1, 2].all()) and int(bad.any(-1).sum()) == 1


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("n,page", [(2, 16), (100, 64)])
def test_kv4_attention_of_queries_that_are_not_finite(cuda, n, page, value, dtype):
    """All keys of one sign, so that every score of such a query is the same infinity: not a number where
    the query sees anything, 0 where it does not, nothing in the rows beside it."""
    d, lens = 128, torch.tensor([150, 1], dtype=torch.int32, device=cuda)
    cache = ops.kv4_cache(-(-150 // page) * 2, 2, page, d, cuda)
    table = torch.arange(cache.k_codes.shape[0], dtype=torch.int32, device=cuda).view(2, -1)
    k = 0.5 + torch.rand(2, 150, 2, d, generator=_gen(4)).to(cuda)
    ops.kv4_append(cache, k, k, table, torch.tensor([150, 150], dtype=torch.int32, device=cuda))
    q = torch.randn(2, n, 4, d, generator=_gen(5)).to(dtype).to(cuda)
    clean = ops.kv4_attention(q, cache, table, lens)
    q[0, 1, 2, 5] = q[1, 0, 3, 7] = value                  # the second one stands before its sequence begins
    got = ops.kv4_attention(q, cache, table, lens)
    assert torch.isnan(got[0, 1, 2]).all() and not got[1, 0, 3].any()
    clean[0, 1, 2] = got[0, 1, 2] = 0
    assert torch.equal(got, clean)


@gpu
def test_kv4_cache_beyond_32_bits(cuda):
    """Pages whose bytes lie more than 2^32 behind the cache's beginning."""
    pages = 140000
    cache = ops.kv4_cache(pages, 8, 64, 128, cuda)         # 4.6 GB of codes each
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device=cuda)
    lens = torch.tensor([170], dtype=torch.int32, device=cuda)
    g = _gen(3)
    k, v = (torch.randn(1, 170, 8, 128, generator=g).to(cuda) for _ in range(2))
    ops.kv4_append(cache, k, v, table, lens)
    q = torch.randn(1, 2, 8, 128, generator=g).to(cuda)
    got = ops.kv4_attention(q, cache, table, lens)
    small = ops.KV4Cache(*(t[table[0].long()].contiguous() for t in cache))
    order = torch.arange(3, dtype=torch.int32, device=cuda)[None]
    assert torch.equal(got, ops.kv4_attention(q, small, order, lens))
    want, tol = ref.attention(q.cpu(), small, order, lens, 128 ** -0.5)
    _close(got, want, tol)
    assert torch.equal(ops.kv4_read(cache, table, lens, 170)[0], ops.kv4_read(small, order, lens, 170)[0])


# ------------------------------------------------------------------------------------ together
def _block(cuda, dtype):
    """Weights and cache of one attention block: 8 query and 2 key heads of 64 channels."""
    g = _gen(21)
    w = {n: ops.fp8_pack_weight(torch.randn(o, i, generator=g).mul(i ** -0.5).to(cuda))
         for n, o, i in (("qkv", 12 * 64, 200), ("out", 200, 8 * 64))}
    angle = torch.arange(300)[:, None] * 10000.0 ** (-torch.arange(32) / 32)
    return dict(w=w, cos=angle.cos().to(cuda), sin=angle.sin().to(cuda), norm=torch.ones(64, device=cuda),
                cache=ops.kv4_cache(12, 2, 16, 64, cuda),
                table=torch.randperm(12, generator=g)[:10].view(2, 5).int().to(cuda), dtype=dtype)


def _step(s, x, lens):
    """x [2, n, 200] through projection, norms, cache, attention and projection."""
    n = x.shape[1]
    qkv = ops.fp8_linear(x, *s["w"]["qkv"]).unflatten(2, (12, 64))
    at = (lens[:, None] - n + torch.arange(n, device=x.device)).clamp(min=0).int()
    q, k = ops.qk_norm_rope(qkv[:, :, :8], qkv[:, :, 8:10], s["norm"], s["norm"], s["cos"], s["sin"], at)
    ops.kv4_append(s["cache"], k, qkv[:, :, 10:], s["table"], lens)
    y = ops.kv4_attention(q, s["cache"], s["table"], lens, window=48, sinks=4)
    return qkv, at, q, k, y, ops.fp8_linear(y.flatten(2), *s["w"]["out"])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_a_block_of_all_operators(cuda, dtype):
    """A padded prompt and ten single tokens: every operator against the reference of its own inputs."""
    s = _block(cuda, dtype)
    g = _gen(22)
    lens = torch.tensor([60, 33], dtype=torch.int32, device=cuda)
    for step in range(11):
        n = 60 if step == 0 else 1
        x = torch.randn(2, n, 200, generator=g).to(dtype).to(cuda)
        qkv, at, q, k, y, out = _step(s, x, lens)
        for a, b, name in ((x, qkv.flatten(2), "qkv"), (y.flatten(2), out, "out")):
            codes, scale = s["w"][name]
            rows = a.flatten(0, 1)
            want, size = ref.linear(*ref.e4m3_rows(rows), codes.float().cpu(), scale.cpu())
            _close(b.flatten(0, 1), want, ref.linear_tolerance(want, size, rows.shape[1], dtype))
        tiny = 2.0 ** -25 if dtype == torch.float16 else 0
        for a, b in ((qkv[:, :, :8], q), (qkv[:, :, 8:10], k)):
            want, size = ref.norm_rope(a.flatten(0, 1), s["norm"], s["cos"], s["sin"], at, 1e-6, False)
            _close(b.flatten(0, 1), want, ref.norm_tolerance(want, size, 64, dtype) + tiny)
        want, tol = ref.attention(q.cpu(), s["cache"], s["table"], lens, 64 ** -0.5, window=48, sinks=4)
        _close(y, want, tol)
        lens = lens + 1
    assert _lib.device_status() == 0


@gpu
def test_captured_steps_and_other_streams(cuda):
    """A captured step replayed with new inputs equals the eager one; two graphs and a second stream do
    not share what they write."""
    s, t = _block(cuda, torch.bfloat16), _block(cuda, torch.bfloat16)
    lens = torch.tensor([1, 1], dtype=torch.int32, device=cuda)
    x = torch.randn(2, 1, 200, generator=_gen(1)).bfloat16().to(cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(s, x, lens)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(s, x, lens)[-1]
        graphs.append((graph, out))
    for i in range(1, 40):
        lens.fill_(i)
        x.copy_(torch.randn(2, 1, 200, generator=_gen(i)))
        for graph, _ in graphs:
            graph.replay()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            want = _step(t, x, lens)[-1]
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want), i

"""Low-precision transformer operators captured into CUDA graphs, on two streams at once and from two threads: every
form that takes a workspace or launches more than one kernel."""
import threading

import pytest
import torch

from modiff_b200 import _lib, ops

gpu = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _linear(cuda, rows, k, n, dtype):
    g = _gen(rows + k)
    w = ops.fp8_pack_weight(torch.randn(n, k, generator=g).to(cuda))
    x = torch.randn(rows, k, generator=g).to(dtype).to(cuda)
    return x, lambda: ops.fp8_linear(x, *w)


def _attention(cuda, lengths, n, heads, kv_heads, d, dtype, **kw):
    g = _gen(sum(lengths) + n)
    b, per = len(lengths), -(-max(lengths) // 64)
    cache = ops.kv4_cache(b * per, kv_heads, 64, d, cuda)
    table = torch.randperm(b * per, generator=g).view(b, per).int().to(cuda)
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    k, v = (torch.randn(b, max(lengths), kv_heads, d, generator=g).to(dtype).to(cuda) for _ in range(2))
    ops.kv4_append(cache, k, v, table, torch.full_like(lens, max(lengths)))
    q = torch.randn(b, n, heads, d, generator=g).to(dtype).to(cuda)
    return q, lambda: ops.kv4_attention(q, cache, table, lens, **kw)


# rows quantised in the product, in front of it, tiles of two SMs; one part, parts that are joined, few and many rows
FORMS = [(_linear, (3, 256, 384, torch.bfloat16)), (_linear, (40, 1000, 520, torch.float32)),
         (_linear, (1300, 640, 1280, torch.float16)), (_attention, ([150, 40], 1, 8, 2, 64, torch.float32)),
         (_attention, ([6000, 700], 1, 8, 2, 128, torch.bfloat16)), (_attention, ([5000], 2, 8, 2, 256, torch.float16)),
         (_attention, ([900, 500], 150, 4, 2, 128, torch.bfloat16)), (_attention, ([6000], 33, 4, 1, 128, torch.float16)),
         (_attention, ([6000], 33, 4, 1, 64, torch.bfloat16))]


@gpu
def test_two_graphs_of_every_form(cuda):
    """Two graphs of all forms, their workspaces in one pool, replayed in turn with new inputs, equal eager calls."""
    forms = [make(cuda, *args) for make, args in FORMS]
    for _, run in forms:
        run()
    torch.cuda.synchronize()
    pool, graphs = torch.cuda.graph_pool_handle(), []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs = [run() for _, run in forms]
        graphs.append((graph, outs))
    for i in range(6):
        for x, _ in forms:
            x.copy_(torch.randn(x.shape, generator=_gen(i)).to(x.dtype))
        want = [run() for _, run in forms]
        graph, outs = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
    assert _lib.device_status() == 0


@gpu
def test_weights_packed_right_before_they_are_read(cuda):
    """The product may begin while its quantiser runs, but not before the weights are there."""
    x = torch.randn(100, 2048, generator=_gen(1)).bfloat16().to(cuda)
    weights = [torch.randn(1024, 2048, generator=_gen(i)).to(cuda) for i in range(4)]
    want = [ops.fp8_linear(x, *ops.fp8_pack_weight(w)) for w in weights]
    torch.cuda.synchronize()
    codes, scale = (t.clone() for t in ops.fp8_pack_weight(weights[0]))
    got = []
    for i in (1, 2, 3, 0):
        c, s = ops.fp8_pack_weight(weights[i])
        codes.copy_(c)
        scale.copy_(s)
        got.append((i, ops.fp8_linear(x, codes, scale)))
    for i, y in got:
        assert torch.equal(y, want[i])


@gpu
def test_all_forms_on_two_streams_and_from_two_threads(cuda):
    forms = [make(cuda, *args) for make, args in FORMS]
    want = [run() for _, run in forms]
    torch.cuda.synchronize()
    bad = []

    def work(order):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream), torch.no_grad():
            got = [(i, forms[i][1]()) for _ in range(8) for i in order]
        stream.synchronize()
        bad.extend(i for i, y in got if not torch.equal(y, want[i]))

    threads = [threading.Thread(target=work, args=(o,)) for o in (range(len(forms)), range(len(forms) - 1, -1, -1))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad and _lib.device_status() == 0

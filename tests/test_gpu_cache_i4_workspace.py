"""The scratch of a QuantizedKVCache on the device: none is made while a graph is captured, and one eager step of any length makes all of it."""
import pytest
import torch

from flh_amd.quantized_model import QuantizedKVCache

pytestmark = pytest.mark.gpu


def step(gen, t, hq=8, hkv=2, d=128, b=2):
    x = [torch.randn(b, t, h, d, generator=gen, device="cuda").half() for h in (hq, hkv, hkv)]
    return (*x, torch.ones(b, t, d, device="cuda").half(), torch.zeros(b, t, d, device="cuda").half())


def test_a_capture_makes_no_scratch():
    gen = torch.Generator("cuda").manual_seed(1)
    cache, x = QuantizedKVCache(1, 2, 2, 600, 128, "cuda"), step(gen, 5)
    with pytest.raises(RuntimeError, match="workspace"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            cache.layer(0).attend(*x)
    torch.cuda.synchronize()


@pytest.mark.parametrize("first,t", [(1, 5), (5, 1), (300, 9)])
def test_a_step_captured_behind_an_eager_one_of_another_length(first, t):
    gen = torch.Generator("cuda").manual_seed(t)
    cache, eager = (QuantizedKVCache(1, 2, 2, 600, 128, "cuda") for _ in range(2))
    x = step(gen, t)
    for c in (cache, eager):
        gen_first = torch.Generator("cuda").manual_seed(0)
        c.layer(0).attend(*step(gen_first, first))
        c.advance(first)
    eager.layer(0).attend(*x)                                          # (every kernel has run before the capture)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.layer(0).attend(*x)
    for n in ([first, first], [400, 77], [0, -1]):
        for c in (cache, eager):
            c.lengths.copy_(torch.tensor(n))
        for a, b in zip(x, step(gen, t)):
            a.copy_(b)
        graph.replay()
        want = eager.layer(0).attend(*x)
        torch.cuda.synchronize()
        assert torch.equal(out, want), n
        for a, b in zip(cache.layers[0], eager.layers[0]):
            assert torch.equal(a, b)

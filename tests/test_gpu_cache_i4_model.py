"""The W4A4 model on a key / value cache in 4 bits: the decoder layer's attention from its own projections against float64 over what the cache
holds, prompts in blocks and token by token, padded batches, a captured step over many lengths, the way to a cache in fp16."""
import pytest
import torch

from flh_amd.quantized_model import DraftTree, LlamaShape, QuantizedKVCache, W4A4LlamaModel

pytestmark = pytest.mark.gpu

SHAPE = LlamaShape(1024, 8, 2, 2048, 2, 512, 1e-5, 10000.0)           # heads of 128
SMALL = LlamaShape(512, 8, 8, 1024, 2, 512, 1e-5, 10000.0)            # of 64
H16 = 2.0 ** -11


def make(activation="group", fused=True, shape=SHAPE):
    return W4A4LlamaModel.random_init(shape, activation=activation, weight_group_size=128, fused=fused, device="cuda", seed=3)


def tokens(b, t, seed=1):
    return torch.randint(0, 512, (b, t), device="cuda", generator=torch.Generator("cuda").manual_seed(seed))


def rotate64(x, cos, sin):
    x, c, s = x.double(), cos.double()[:, :, None], sin.double()[:, :, None]
    half = x.size(-1) // 2
    return x * c + torch.cat((-x[..., half:], x[..., :half]), -1) * s


@pytest.mark.parametrize("shape,activation,fused,t", [(SHAPE, "token", True, 1), (SHAPE, "group", True, 1), (SHAPE, "group", False, 1),
                                                      (SHAPE, "token", True, 9), (SHAPE, "group", True, 70), (SHAPE, "group", False, 5),
                                                      (SMALL, "group", True, 1), (SMALL, "group", True, 40)])
def test_the_layer_attends_to_what_the_cache_holds(shape, activation, fused, t):
    model, b, d, heads = make(activation, fused, shape), 2, shape.head_dim, shape.num_heads
    cache = model.new_cache(b, 160, bits=4)
    with torch.no_grad():
        model.append(tokens(b, 50), cache)
    cache.lengths.copy_(torch.tensor([50, 33]))
    layer = model.layers[1]
    x = torch.randn(b, t, shape.hidden_size, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).half()
    positions = cache.lengths[:, None] + torch.arange(t, device="cuda")
    cos, sin = (v.view(b, t, d) for v in model._rotary(positions.reshape(-1), cache))
    layer.record = {}
    with torch.no_grad():
        layer.attention(x, cos, sin, cache.layer(1))
    rec, layer.record = layer.record, None
    q, k, v = (rec[n + "_proj"].view(b, t, -1, d) for n in "qkv")
    got = rec["attn_out.input"].double().view(b, t, heads, d)
    qr, kr = rotate64(q, cos, sin), rotate64(k, cos, sin)
    keys, values = (c.double() for c in cache.read(1, torch.zeros_like(cache.lengths), 160))
    rep = heads // shape.num_kv_heads
    for i, n in enumerate((50, 33)):
        # the new rows are in their slots: a 4-bit code is off by half a step, 1 / 14 of the rotated row's largest, over d channels that
        # the Hadamard rotation mixes with 1 / sqrt(d) each; that largest is at most sqrt(d) of the row's
        assert ((keys[i, :, n:n + t] - kr[i].transpose(0, 1)).norm(dim=-1) <= kr[i].transpose(0, 1).norm(dim=-1) * d ** 0.5 / 13).all()
        step = v[i].double().abs().amax(-1).t()[..., None] / 7
        assert ((values[i, :, n:n + t] - v[i].double().transpose(0, 1)).abs() <= step * (0.5 + 8 * H16)).all()
        seen = torch.arange(n + t, device="cuda") < n + 1 + torch.arange(t, device="cuda")[:, None]
        for h in range(heads):
            kk, vv = keys[i, h // rep, :n + t], values[i, h // rep, :n + t]
            p = torch.softmax(((qr[i, :, h] @ kk.t()) / d ** 0.5).masked_fill(~seen, -torch.inf), -1)
            want = p @ vv
            # the result, the probabilities, the queries (of a block) and the keys read back are rounded to fp16: the latter two move a score by
            # 2^-11 of its terms each, a probability by twice that
            size = (qr[i, :, h].abs().sum(-1) * kk.abs().max()).max().item() / d ** 0.5
            tol = H16 * want.abs() + (H16 + 4 * H16 * size + 1e-4) * (p @ vv.abs()) + 1e-6
            assert ((got[i, :, h] - want).abs() <= tol).all(), (i, h, ((got[i, :, h] - want).abs() / tol).max())


def test_blocks_and_tokens_give_the_same_first_layer():
    """The first layer's keys and values do not depend on how a prompt comes (the layers behind see attention's roundings)."""
    model, ids = make(), tokens(2, 40)
    caches = [model.new_cache(2, 64, bits=4) for _ in range(3)]
    with torch.no_grad():
        model.append(ids, caches[0])
        for part in ids.split(17, 1):
            last = model.append(part, caches[1])
        for i in range(40):
            step = model.append(ids[:, i:i + 1], caches[2])
    for cache in caches[1:]:
        assert torch.equal(cache.lengths, caches[0].lengths) and cache.lengths.tolist() == [40, 40]
        for a, b in zip(cache.layers[0], caches[0].layers[0]):
            assert torch.equal(a, b)
    assert last.shape == (2, 6, 512) and step.shape == (2, 1, 512) and torch.isfinite(step).all()


def test_padded_batch_and_places_that_take_no_part():
    model = make()
    ids, counts = tokens(3, 20), torch.tensor([20, 7, 0], device="cuda")
    cache, alone = model.new_cache(3, 64, bits=4), model.new_cache(1, 64, bits=4)
    with torch.no_grad():
        model.append(ids, cache, counts=counts)
        assert cache.lengths.tolist() == [20, 7, 0]
        cache.lengths[2] = -1
        held = [t[2].clone() for t in cache.layers[1]]
        more = tokens(3, 1, seed=5)
        out = model.append(more, cache)
        assert cache.lengths.tolist() == [21, 8, -1]
        for a, b in zip(cache.layers[1], held):
            assert torch.equal(a[2], b)
        model.append(ids[1:2, :7], alone)
        single = model.append(more[1:2], alone)
    # the padded row's sequence is the one that came alone: the same codes in the first layer, and what the padding left is overwritten
    for a, b in zip(cache.layers[0], alone.layers[0]):
        assert torch.equal(a[1, :, :8], b[0, :, :8])
    assert torch.isfinite(out[:2]).all() and torch.isfinite(single).all()
    cache.lengths[0] = 64                                             # full: takes no part, and keeps its length
    with torch.no_grad():
        model.append(more, cache)
    assert cache.lengths.tolist() == [64, 9, -1]


@pytest.mark.parametrize("shape,t", [(SHAPE, 1), (SMALL, 1), (SHAPE, 5)])
def test_a_captured_step_serves_every_length(shape, t):
    model, ids = make(shape=shape), tokens(2, 30)
    eager, cache = model.new_cache(2, 200, bits=4), model.new_cache(2, 200, bits=4)
    static = torch.zeros(2, t, dtype=torch.int64, device="cuda")
    with torch.no_grad():
        for c in (eager, cache):
            model.append(ids, c)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            model.append(static, cache)                               # (every kernel runs once before the capture)
        torch.cuda.current_stream().wait_stream(side)
        cache.lengths.sub_(t)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = model.append(static, cache)
        for step in range(6):
            new = tokens(2, t, seed=10 + step)
            static.copy_(new)
            graph.replay()
            want = model.append(new, eager)                           # (eager work between the replays)
            torch.cuda.synchronize()
            assert torch.equal(out, want), step
            assert torch.equal(cache.lengths, eager.lengths)
        if t == 1:
            cache.lengths.copy_(torch.tensor([150, 64]))
            eager.lengths.copy_(torch.tensor([150, 64]))
            graph.replay()
            assert torch.equal(out, model.append(new, eager))
    for a, b in zip(cache.layers, eager.layers):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_to_static_serves_drafts():
    model, ids = make(), tokens(2, 30)
    cache = model.new_cache(2, 64, bits=4)
    with torch.no_grad():
        model.append(ids, cache)
        static = cache.to_static(q_heads=SHAPE.num_heads, max_positions=80)
        assert static.lengths.tolist() == [30, 30] and static.lengths is not cache.lengths
        for i in range(2):
            keys, values = cache.read(i, torch.tensor([5, 0], device="cuda"), 20)
            assert torch.equal(static.keys[i][0, :, 5:25], keys[0]) and torch.equal(static.values[i][1, :, :20], values[1])
        tree = DraftTree([-1, 0, 1])
        new = tokens(2, 3, seed=7)
        drafted = model.tree_step(new, tree, static)
        chained = model.append(new, cache)
    assert drafted.shape == chained.shape and torch.isfinite(drafted).all()
    # (the chain's own keys are fp16 in one and 4 bits in the other: loosely alike)
    assert torch.nn.functional.cosine_similarity(drafted.float(), chained.float(), dim=-1).min() > 0.5


def test_memory_is_a_quarter():
    cache = QuantizedKVCache(2, 3, 8, 256, 128, "cuda")
    held = sum(t.numel() * t.element_size() for layer in cache.layers for t in layer)
    assert held == 2 * 2 * 3 * 8 * 256 * (64 + 2)                     # 66 bytes a row of 128 values, where fp16 takes 256

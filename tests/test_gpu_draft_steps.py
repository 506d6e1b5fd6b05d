"""Steps of the W4A4 model over drafted tokens: the decoder layer's attention from its own projections against float64, a generation with
drafts against the state it leaves, and a captured step at several lengths."""
import pytest
import torch

from flh_amd.quantized_model import DraftTree, LlamaShape, W4A4LlamaModel

pytestmark = pytest.mark.gpu

SHAPE = LlamaShape(1024, 8, 2, 2048, 2, 512, 1e-5, 10000.0)           # heads of 128
PARENTS = [-1, 0, 0, 1, 1, 2, 5, 6]


def make(activation, fused=True, shape=SHAPE):
    return W4A4LlamaModel.random_init(shape, activation=activation, weight_group_size=128, fused=fused, device="cuda", seed=3)


def prompted(model, batch=2, length=70, max_len=160):
    ids = torch.randint(0, 512, (batch, length), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    cache = model.new_cache(batch, max_len)
    with torch.no_grad():
        model(ids, cache.advance(length), cache)
    return cache


def rotate64(x, cos, sin):
    x, c, s = x.double(), cos.double()[:, :, None], sin.double()[:, :, None]
    half = x.size(-1) // 2
    return x * c + torch.cat((-x[..., half:], x[..., :half]), -1) * s


@pytest.mark.parametrize("activation,fused", [("token", True), ("group", True), ("group", False)])
def test_the_layer_attends_to_cache_and_tree(activation, fused):
    model = make(activation, fused)
    cache = prompted(model)
    cache.begin_drafts()
    cache.lengths.copy_(torch.tensor([70, 33]))
    tree, layer, t = DraftTree(PARENTS), model.layers[1], len(PARENTS)
    x = torch.randn(2, t, SHAPE.hidden_size, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).half()
    positions = cache.lengths[:, None] + tree.depths
    cos, sin = (v.view(2, t, 128) for v in model._rotary(positions.view(-1), cache))
    before = [c.clone() for c in (cache.keys[1], cache.values[1])]
    layer.record = {}
    with torch.no_grad():
        layer.attention(x, cos, sin, cache.tree_layer(1, tree))
    rec, layer.record = layer.record, None
    q, k, v = (rec[n + "_proj"].view(2, t, -1, 128) for n in "qkv")
    got = rec["attn_out.input"].double().view(2, t, 8, 128)
    qr, kr = rotate64(q, cos, sin), rotate64(k, cos, sin)
    for b, n in enumerate((70, 33)):
        keys, values = before[0][b].double(), before[1][b].double()
        keys[:, n:n + t], values[:, n:n + t] = kr[b].half().transpose(0, 1).double(), v[b].transpose(0, 1).double()
        assert torch.equal(cache.values[1][b], values.half())
        assert (cache.keys[1][b].double() - keys).abs().max() <= 2.0 ** -10 * keys.abs().max()   # a neighbour at most
        seen = torch.cat((torch.ones(t, n, dtype=torch.bool, device="cuda"), tree.mask), 1)
        for h in range(8):
            kk, vv = keys[h // 4, :n + t], values[h // 4, :n + t]
            p = torch.softmax(((qr[b, :, h] @ kk.t()) / 128 ** 0.5).masked_fill(~seen, -torch.inf), -1)
            # the result and the probabilities rounded to fp16; a key that is a neighbour moves a score by 2^-10 of its size
            size = (qr[b, :, h].abs() @ kk.abs().t()).max().item() / 128 ** 0.5
            assert ((got[b, :, h] - p @ vv).abs() <= vv.abs().max() * (2.0 ** -10 + size * 2.0 ** -10 + 1e-4)).all()


def test_a_generation_with_drafts_leaves_the_accepted_rows():
    model = make("group")
    cache = prompted(model)
    lengths = cache.begin_drafts()
    tree, t = DraftTree(PARENTS), len(PARENTS)
    gen = torch.Generator("cuda").manual_seed(5)
    want = [70, 70]
    with torch.no_grad():
        for step in range(3):
            tokens = torch.randint(0, 512, (2, t), device="cuda", generator=gen)
            logits = model.tree_step(tokens, tree, cache)
            assert logits.shape == (2, t, 512) and torch.isfinite(logits).all()
            chosen = logits.argmax(-1)
            # drafts that the model agrees with: the branch 0, 2, 5 of the first sequence, none of the second
            chosen[0, 0], chosen[0, 2], chosen[1, 0] = tokens[0, 2], tokens[0, 5], -5
            chosen[0, 5] = -7
            if tokens[0, 1] == tokens[0, 2]:
                tokens[0, 1] = (tokens[0, 1] + 1) % 512
            held = [c.clone() for c in cache.keys + cache.values]
            path, accepted, following = cache.commit(tokens, tree, chosen)
            assert path[:, :4].tolist() == [[0, 2, 5, -1], [0, -1, -1, -1]] and following.tolist() == [-7, -5]
            for old, new in zip(held, cache.keys + cache.values):
                n = want[0]
                assert torch.equal(new[0, :, n:n + 3], old[0, :, [n, n + 2, n + 5]])
                assert torch.equal(new[0, :, n + 3:], old[0, :, n + 3:]) and torch.equal(new[1], old[1])
            want = [want[0] + 3, want[1] + 1]
            assert lengths is cache.lengths and lengths.tolist() == want
    with pytest.raises(ValueError, match="lengths of their own"):
        cache.advance(1)
    with pytest.raises(ValueError, match="lengths of their own"):
        model(tokens[:, :1], torch.tensor([75], device="cuda"), cache)


@pytest.mark.parametrize("activation", ["token", "group"])
def test_a_captured_step_serves_every_length(activation):
    model = make(activation)
    cache = prompted(model, length=90)
    cache.begin_drafts()
    tree, t = DraftTree(PARENTS), len(PARENTS)
    ids = torch.randint(0, 512, (2, t), device="cuda", generator=torch.Generator("cuda").manual_seed(6))
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                model.tree_step(ids, tree, cache)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = model.tree_step(ids, tree, cache)
        for lengths in ([90, 61], [20, -1], [64, 152], [1, 90]):
            cache.lengths.copy_(torch.tensor(lengths))
            ids.random_(0, 512)
            start = [c.clone() for c in cache.keys + cache.values]
            graph.replay()
            torch.cuda.synchronize()
            got, rows = logits.clone(), [c.clone() for c in cache.keys + cache.values]
            for c, x in zip(cache.keys + cache.values, start):
                c.copy_(x)
            eager = model.tree_step(ids, tree, cache)
            assert torch.equal(got, eager)
            for a, b in zip(rows, cache.keys + cache.values):
                assert torch.equal(a, b)


def test_a_chain_writes_what_a_block_of_tokens_writes():
    """A chain of four nodes against a block of four tokens, in the first layer, whose inputs are the same: the values' bits, and keys
    that differ by the block's two further roundings (each product, half a step of at most the row's largest value; and its sum's)."""
    model = make("group")
    a, b = prompted(model), prompted(model)
    ids = torch.randint(0, 512, (2, 4), device="cuda", generator=torch.Generator("cuda").manual_seed(7))
    with torch.no_grad():
        model(ids, a.advance(4), a)
        b.begin_drafts()
        logits = model.tree_step(ids, DraftTree([-1, 0, 1, 2]), b)
    assert torch.isfinite(logits).all()
    assert torch.equal(a.values[0][:, :, :74], b.values[0][:, :, :74])
    ka, kb = a.keys[0][:, :, :74].double(), b.keys[0][:, :, :74].double()
    top = kb.abs().amax(-1, keepdim=True) * 2 ** 0.5                    # (a channel before its rotation: at most the pair's length)
    assert ((ka - kb).abs() <= 4 * 2.0 ** -11 * top).all()


def test_refusals():
    for parents in ([], [0], [-1, 1], [-1, 0, 2], [-1, -1], [-1] * 257):
        with pytest.raises(ValueError):
            DraftTree(parents)
    model = make("group")
    cache = prompted(model)
    tree = DraftTree([-1, 0])
    ids = torch.zeros(2, 2, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="begin_drafts"):
        model.tree_step(ids, tree, cache)
    with pytest.raises(ValueError, match="begin_drafts"):
        cache.commit(ids, tree, ids)
    cache.begin_drafts()
    with pytest.raises(ValueError, match="nodes"):
        model.tree_step(ids[:, :1], tree, cache)
    with pytest.raises(ValueError, match="sequences"):
        model.tree_step(ids[:1], tree, cache)

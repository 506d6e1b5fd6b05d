"""Steps over drafted tokens on a cache that is cut on the way: the positions behind a cut go on counting, the kept keys stay as they
were rotated, a sequence past the rotary table or out of the batch takes no part and loses nothing."""
import pytest
import torch

from flh_amd.quantized_model import DraftTree, LlamaShape, W4A4LlamaModel

pytestmark = pytest.mark.gpu

SHAPE = LlamaShape(1024, 8, 2, 2048, 2, 512, 1e-5, 10000.0)           # heads of 128
PARENTS = [-1, 0, 0, 1, 1, 2, 5, 6]
T, SLOTS = len(PARENTS), 160


def make(activation="group", shape=SHAPE):
    return W4A4LlamaModel.random_init(shape, activation=activation, weight_group_size=128, fused=True, device="cuda", seed=3)


def prompted(model, length=100, **more):
    ids = torch.randint(0, 512, (2, length), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    cache = model.new_cache(2, SLOTS, **more)
    with torch.no_grad():
        model(ids, cache.advance(length), cache)
    cache.begin_drafts()
    return cache


def sums(seed=2):
    return torch.rand(2, 2, 2, SLOTS, device="cuda", generator=torch.Generator("cuda").manual_seed(seed))


def tokens(seed):
    return torch.randint(0, 512, (2, T), device="cuda", generator=torch.Generator("cuda").manual_seed(seed))


def rotated(k, positions):
    """k [B, T, H, 128] of the projections, positions [B, T] -> float64, with the model's fp16 table at these positions"""
    inv = 1.0 / (10000.0 ** (torch.arange(0, 128, 2, device="cuda", dtype=torch.float32) / 128))
    angle = torch.cat((positions.float()[..., None] * inv,) * 2, -1)
    cos, sin, x = angle.cos().half().double()[:, :, None], angle.sin().half().double()[:, :, None], k.double()
    return x * cos + torch.cat((-x[..., 64:], x[..., :64]), -1) * sin


@pytest.mark.parametrize("activation", ["group", "token"])
def test_positions_go_on_counting_behind_a_cut(activation):
    model = make(activation)
    cache = prompted(model, max_positions=400)
    lengths, cut, tree = cache.lengths, cache.cut, DraftTree(PARENTS)
    lengths.copy_(torch.tensor([100, 61]))
    before = [c.clone() for c in cache.keys + cache.values]
    w = sums()
    kept, left = cache.evict(w, 40, 8)
    assert lengths is cache.lengths and lengths.tolist() == [40, 40] and cut.tolist() == [60, 21]
    for old, new, at in zip(before, cache.keys + cache.values, [*kept, *kept]):
        assert torch.equal(new[:, :, :40], old.gather(2, at[..., None].expand(-1, -1, -1, 128)))
    assert torch.equal(left[..., :40], w.gather(3, kept)) and not left[..., 40:].any()
    want = torch.tensor([100, 61], device="cuda")
    layer = model.layers[0]
    with torch.no_grad():
        for step in range(2):
            ids, n = tokens(step), lengths.tolist()
            layer.record = {}
            logits = model.tree_step(ids, tree, cache)
            rec, layer.record = layer.record, None
            assert torch.isfinite(logits).all()
            keys = rotated(rec["k_proj"].view(2, T, 2, 128), want[:, None] + tree.depths).transpose(1, 2)
            for b in range(2):
                got = cache.keys[0][b, :, n[b]:n[b] + T].double()
                # a neighbour at most; and float32's rounding of two products, each at most as large as the largest channel, and their sum
                slack = 4 * 2.0 ** -24 * rec["k_proj"].double().abs().max()
                assert ((got - keys[b]).abs() <= 2.0 ** -10 * keys[b].abs().clamp(min=2.0 ** -14) + slack).all()
            chosen = torch.full_like(ids, -5)
            chosen[0, 0], chosen[0, 2] = ids[0, 2], ids[0, 5]
            ids[0, 1] = (ids[0, 2] + 1) % 512                          # (not the branch's token)
            _, accepted, _ = cache.commit(ids, tree, chosen)
            assert accepted.tolist() == [3, 1]
            want = want + accepted
            assert torch.equal(cache.next_positions(), want)
    cache.evict(sums(), 40, 0)
    assert lengths.tolist() == [40, 40] and torch.equal(cache.next_positions(), want)


def test_sequences_that_take_no_part_lose_nothing():
    """One whose next positions pass the table; one that waits, whose sums survive the cut of the other."""
    model, tree = make(), DraftTree(PARENTS)
    cache = prompted(model, max_positions=164)
    cache.lengths.copy_(torch.tensor([100, -1]))
    w = sums()
    _, left = cache.evict(w, 50, 8)
    assert cache.lengths.tolist() == [50, -1] and cache.cut.tolist() == [50, 0]
    assert torch.equal(left[:, 1], w[:, 1]) and not left[:, 0, :, 50:].any()
    cache.lengths.copy_(torch.tensor([107, 156 - 4]))                  # positions 157 .. 164: one too many; slots 152 .. 159
    before = [c.clone() for c in cache.keys + cache.values]
    ids = tokens(1)
    with torch.no_grad():
        model.tree_step(ids, tree, cache)
    for old, new in zip(before, cache.keys + cache.values):
        assert torch.equal(new[0], old[0]) and not torch.equal(new[1, :, 152:], old[1, :, 152:])
    path, accepted, following = cache.commit(ids, tree, torch.full_like(ids, -5))
    assert accepted.tolist() == [0, 1] and following.tolist() == [-1, -5] and cache.lengths.tolist() == [107, 153]
    cache.lengths.copy_(torch.tensor([106, -1]))                       # positions 156 .. 163: the last ones
    with torch.no_grad():
        model.tree_step(ids, tree, cache)
    _, accepted, _ = cache.commit(ids, tree, torch.full_like(ids, -5))
    assert accepted.tolist() == [1, 0]


def test_a_step_captured_in_front_of_a_cut_serves_behind_it():
    model, tree = make(), DraftTree(PARENTS)
    cache, other = (prompted(model, max_positions=400) for _ in range(2))
    ids, chosen = tokens(7), torch.full((2, T), -5, device="cuda")
    chosen[0, 0], chosen[0, 2] = ids[0, 2], ids[0, 5]
    ids[0, 1] = (ids[0, 2] + 1) % 512
    with torch.no_grad():
        for c in (cache, other):
            model.tree_step(ids, tree, c)
            c.commit(ids, tree, chosen)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = model.tree_step(ids, tree, cache)
            cache.commit(ids, tree, chosen)
        for step in range(4):
            graph.replay()
            torch.cuda.synchronize()
            eager = model.tree_step(ids, tree, other)
            other.commit(ids, tree, chosen)
            assert torch.equal(logits, eager)
            for a, b in zip([*cache.keys, *cache.values, cache.lengths, cache.cut], [*other.keys, *other.values, other.lengths, other.cut]):
                assert torch.equal(a, b)
            if step % 2 == 0:
                for c in (cache, other):
                    c.evict(sums(step), 60, 10)
        assert cache.next_positions().tolist() == [100 + 3 * 5, 100 + 5]


def test_a_place_takes_a_new_prompt_as_chains():
    """A finished sequence's place: its length (and cut) zero, the other one out of the steps; the prompt as chains of up to 256 tokens,
    all accepted.  The first layer's rows have the bits that one chain of the whole prompt leaves."""
    model = make()
    cache, other = prompted(model, max_positions=400), prompted(model, max_positions=400)
    cache.evict(sums(), 60, 10)
    waiting = [c[1].clone() for c in cache.keys + cache.values]
    ids = torch.randint(0, 512, (2, 120), device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    with torch.no_grad():
        for c, pieces in ((cache, (70, 50)), (other, (120,))):
            c.lengths.copy_(torch.tensor([0, -1]))
            c.cut.zero_()
            at = 0
            for n in pieces:
                chain, part = DraftTree(range(-1, n - 1)), ids[:, at:at + n].contiguous()
                model.tree_step(part, chain, c)
                _, accepted, _ = c.commit(part, chain, torch.cat((part[:, 1:], part[:, :1]), 1))
                assert accepted.tolist() == [n, 0]
                at += n
            assert c.lengths.tolist() == [120, -1]
    for a, b in zip((cache.keys[0], cache.values[0]), (other.keys[0], other.values[0])):
        assert torch.equal(a[0, :, :120], b[0, :, :120])
    for a, b in zip(waiting, cache.keys + cache.values):
        assert torch.equal(a, b[1])


def test_refusals():
    model = make()
    with pytest.raises(ValueError, match="below max_len"):
        model.new_cache(2, SLOTS, max_positions=SLOTS - 1)
    cache = prompted(model)
    with pytest.raises(ValueError, match="max_positions"):
        cache.evict(sums(), 40, 8)
    cache = model.new_cache(2, SLOTS, max_positions=SLOTS)
    with pytest.raises(ValueError, match="begin_drafts"):
        cache.evict(sums(), 40, 8)
    cache.begin_drafts()
    with pytest.raises(RuntimeError, match="weights"):
        cache.evict(sums()[:1].contiguous(), 40, 8)


@pytest.mark.parametrize("batch,nodes,hidden", [(2, 4, 1024), (1, 1, 1024), (1, 1, 4096), (1, 2, 4096), (2, 1, 4096), (3, 1, 4096),
                                                (1, 17, 4096), (3, 43, 1024), (1, 256, 1024), (2, 256, 1024)])
@pytest.mark.parametrize("activation", ["group", "token"])
def test_nodes_that_see_only_themselves_are_steps_of_one_token(activation, batch, nodes, hidden):
    """A node that sees nothing but itself attends to its own value, exactly: its logits have the bits of a first token's step, whichever
    launches a step of that many tokens takes."""
    model = make(activation, LlamaShape(hidden, hidden // 128, hidden // 512, 2 * hidden, 1 if hidden > 1024 else 2, 512, 1e-5, 10000.0))
    ids = torch.randint(0, 512, (batch, nodes), device="cuda", generator=torch.Generator("cuda").manual_seed(9))
    tree = DraftTree([-1] + [0] * (nodes - 1))
    tree.mask.copy_(torch.eye(nodes, dtype=torch.bool))
    first, cache = model.new_cache(batch * nodes, 2), model.new_cache(batch, nodes)
    cache.begin_drafts()
    with torch.no_grad():
        want = model(ids.view(-1, 1), first.advance(1), first)
        got = model.tree_step(ids, tree, cache)
    assert torch.equal(got.view(batch * nodes, 1, -1), want)

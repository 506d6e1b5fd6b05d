"""Batches of padded rows on caches in 4 bits: `counts` says how many of each sequence's tokens are its own, the others are not written and give zeros, and
a sequence takes part where its own fit the cache.  What counts is held to the operators' other tests' evaluations and tolerances."""
import pytest
import torch

from flh_amd.quantized_model import LlamaShape, W4A4LlamaModel
from test_gpu_cache_i4 import attend64, close, normal, packed, quantised, random_cache, rotary, turned, unpacked

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["default", "ctypes"])
def ops(request):
    if request.param == "ctypes":
        from flh_amd import _ops
        return _ops
    import flh_amd
    return flh_amd._CUDA


def own(n, count, T, max_len):
    """Tokens that a sequence of length n takes."""
    return count if 0 <= count <= T and 0 <= n <= max_len - count else 0


@pytest.mark.parametrize("B,T,Hq,Hkv,d,max_len,lengths,counts", [
    (4, 7, 8, 2, 128, 40, [33, 38, 40, 0], [7, 2, 0, 5]),
    (6, 9, 3, 3, 64, 20, [18, 19, -1, 4, 4, 2 ** 62], [3, 1, 2, -1, 10, 1]),       # one does not fit, one is alone at the end, the others are out of range
    (2, 30, 12, 4, 128, 20, [0, 15], [20, 5])])                                    # rows longer than the cache
def test_write(ops, B, T, Hq, Hkv, d, max_len, lengths, counts):
    gen = torch.Generator().manual_seed(T)
    q, k, v = normal(gen, B, T, Hq, d), normal(gen, B, T, Hkv, d), normal(gen, B, T, Hkv, d)
    cos, sin = rotary(gen, B, T, d)
    cache = random_cache(gen, B, Hkv, max_len, d)
    want = [c.clone() for c in cache]
    (kc, ks), (vc, vs) = quantised(turned(k, cos, sin)), quantised(v.float())
    for b, n in enumerate(lengths):
        m = own(n, counts[b], T, max_len)
        if m:
            for at, new in zip(want, (packed(kc[b]), ks[b], packed(vc[b]), vs[b])):
                at[b, :, n:n + m] = new[:m].transpose(0, 1)
    dev = [t.cuda() for t in cache]
    got = ops.rope_quantize_kv_cache_(*(t.cuda() for t in (q, k, v, cos, sin)), torch.tensor(lengths).cuda(), *dev, counts=torch.tensor(counts).cuda())
    assert torch.equal(got.cpu(), turned(q, cos, sin).half())
    for a, b in zip(dev, want):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("B,T,Hq,Hkv,d,max_len", [
    (4, 7, 32, 8, 128, 900),                                           # shared by workgroups, joined
    (3, 40, 12, 4, 64, 2000),                                          # .. three queries per head, several blocks
    (150, 3, 2, 1, 128, 1500),                                         # .. more sequences than lanes
    (6, 100, 16, 16, 128, 300),                                        # four waves a block
    (20, 65, 32, 32, 128, 200),                                        # two
    (64, 65, 32, 32, 128, 150),                                        # one
    (20, 70, 96, 32, 64, 200)])
def test_block(ops, B, T, Hq, Hkv, d, max_len):
    gen = torch.Generator().manual_seed(B + T)
    counts = [(0, T, 1, T - 1, T // 2, T // 3, T + 1, -1)[(3 * b) % 8] for b in range(B)]
    # at the very end, one past it, anywhere, and out of range
    lengths = [(max_len - counts[b], max_len - counts[b] + 1, (37 * b) % (max_len - T), -1, max_len - T, 0)[b % 6] for b in range(B)]
    cache = random_cache(gen, B, Hkv, max_len, d)
    q = normal(gen, B, T, Hq, d, scale=2.0)
    rep = Hq // Hkv
    for b, n in enumerate(lengths):
        m = own(n, counts[b], T, max_len)
        if m:
            q[b, m:] = float("nan")
            cache[1][b, :, n + m:], cache[3][b, :, n + m:] = float("inf"), float("nan")
    dev = [t.cuda() for t in cache]
    x = (q.cuda(), torch.tensor(lengths).cuda(), *dev)
    out = ops.prefill_attention_i4(*x, counts=torch.tensor(counts).cuda())
    got = out.view(B, T, Hq, d).cpu()
    ws = torch.full((64 << 20,), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(ops.prefill_attention_i4(*x, counts=torch.tensor(counts).cuda(), workspace=ws), out)
    looked_at = range(B) if B <= 6 else range(0, B, max(1, B // 20))
    for b in range(B):
        m = own(lengths[b], counts[b], T, max_len)
        assert (got[b, m:] == 0).all(), b
        if not m or b not in looked_at:
            assert torch.isfinite(got[b]).all()
            continue
        n = lengths[b]
        limits = torch.arange(n + 1, n + m + 1).repeat_interleave(rep)
        for g in range(Hkv) if B <= 6 else (0, Hkv - 1):
            rows = q[b, :m, g * rep:(g + 1) * rep].reshape(m * rep, d)
            w, tol = attend64(rows, unpacked(cache[0][b, g, :n + m]), cache[1][b, g, :n + m], unpacked(cache[2][b, g, :n + m]), cache[3][b, g, :n + m],
                              limits, d ** -0.5)
            close(got[b, :m, g * rep:(g + 1) * rep].reshape(m * rep, d), w, tol, (b, g, n, m))


@pytest.mark.parametrize("B,T,H", [(3, 9, 4), (20, 65, 32), (64, 65, 32)])
def test_whole_rows_are_what_they_are_without_counts(ops, B, T, H):
    gen = torch.Generator().manual_seed(T)
    cache = [t.cuda() for t in random_cache(gen, B, H, 300, 128)]
    q, lengths = normal(gen, B, T, H, 128).cuda(), torch.tensor([(61 * b) % 236 for b in range(B)]).cuda()
    counts = torch.full((B,), T).cuda()
    assert torch.equal(ops.prefill_attention_i4(q, lengths, *cache, counts=counts), ops.prefill_attention_i4(q, lengths, *cache))


def test_counts_are_checked(ops):
    gen = torch.Generator().manual_seed(1)
    cache = [t.cuda() for t in random_cache(gen, 2, 2, 64, 128)]
    q, kv, one, n = (t.cuda() for t in (normal(gen, 2, 3, 4, 128), normal(gen, 2, 3, 2, 128), normal(gen, 2, 3, 128), torch.zeros(2, dtype=torch.int64)))
    for bad in (torch.zeros(2, dtype=torch.int64), n.int(), n[:1], torch.zeros(4, dtype=torch.int64).cuda()[::2], n.view(1, 2)):
        with pytest.raises(RuntimeError, match="counts"):
            ops.rope_quantize_kv_cache_(q, kv, kv, one, one, n, *cache, counts=bad)
        with pytest.raises(RuntimeError, match="counts"):
            ops.prefill_attention_i4(q, n, *cache, counts=bad)


SHAPE = LlamaShape(1024, 8, 2, 2048, 2, 512, 1e-5, 10000.0)
SMALL = LlamaShape(512, 8, 8, 1024, 2, 512, 1e-5, 10000.0)


@pytest.mark.parametrize("shape", [SHAPE, SMALL])
def test_the_model_takes_tokens_up_to_the_end_of_the_cache(shape):
    """Three sequences, two of which have room for their own tokens and not for the padding."""
    model = W4A4LlamaModel.random_init(shape, activation="group", weight_group_size=128, fused=True, device="cuda", seed=3)
    ids = torch.randint(0, 512, (3, 40), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    cache, counts = model.new_cache(3, 64, bits=4), torch.tensor([10, 4, 0], device="cuda")
    more = torch.randint(0, 512, (3, 10), device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    with torch.no_grad():
        model.append(ids, cache)
        cache.lengths.copy_(torch.tensor([40, 30, 40]))
        model.append(ids[:, :30], cache, counts=torch.tensor([4, 30, 24], device="cuda"))
        assert cache.lengths.tolist() == [44, 60, 64]
        held = [t[2].clone() for t in cache.layers[1]]
        out = model.append(more, cache, counts=counts)
        assert cache.lengths.tolist() == [54, 64, 64]
        for a, b in zip(cache.layers[1], held):
            assert torch.equal(a[2], b)
        alone = model.new_cache(1, 64, bits=4)
        model.append(ids[1:2, :30], alone)
        model.append(ids[1:2, :30], alone)
        want = model.append(more[1:2, :4], alone)
        assert alone.lengths.tolist() == [64]
    for a, b in zip(cache.layers[0], alone.layers[0]):
        assert torch.equal(a[1], b[0])
    assert torch.isfinite(out[1, :4]).all() and torch.nn.functional.cosine_similarity(out[1, :4].float(), want[0].float(), dim=-1).min() > 0.5
    # single tokens: one sequence's is padding
    with torch.no_grad():
        cache.lengths[1] = 50
        held = [t[1].clone() for t in cache.layers[1]]
        model.append(more[:, :1], cache, counts=torch.tensor([1, 0, 1], device="cuda"))
    assert cache.lengths.tolist() == [55, 50, 64]
    for a, b in zip(cache.layers[1], held):
        assert torch.equal(a[1], b)


@pytest.mark.parametrize("t", [1, 9])
def test_a_captured_step_follows_the_counts(t):
    model = W4A4LlamaModel.random_init(SHAPE, activation="group", weight_group_size=128, fused=True, device="cuda", seed=3)
    ids = torch.randint(0, 512, (2, 30), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    eager, cache = model.new_cache(2, 60, bits=4), model.new_cache(2, 60, bits=4)
    static, counts = ids[:, :t].clone(), torch.tensor([t, 0], device="cuda")
    with torch.no_grad():
        for c in (eager, cache):
            model.append(ids, c)
            model.append(static, c, counts=counts)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = model.append(static, cache, counts=counts)
        for step, n in enumerate(([t, t], [t // 2, 1], [0, t], [t, t], [t, 0], [t, t])):
            counts.copy_(torch.tensor(n))
            static.copy_(ids[:, step:step + t])
            graph.replay()
            want = model.append(static, eager, counts=counts)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(cache.lengths, eager.lengths), step
    for a, b in zip(cache.layers, eager.layers):
        for x, y in zip(a, b):
            assert torch.equal(x, y)

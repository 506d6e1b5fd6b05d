"""Paths of the operators on caches that only large calls, or the edges of a rule, take: an eviction that moves whole rows, the
selection staged in LDS up to its limit, column sums without a second launch, the rotated queries' low halves, a captured commit."""
import numpy as np
import pytest
import torch

from test_gpu_cache_operators import (H16, H32, attend64, commit_oracle, equal_bits, evict_oracle, normal, ops, rotate64,  # noqa: F401
                                      weights_tolerance)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("L,B,Hkv,d,max_len,lengths,budget,recent", [(32, 2, 4, 128, 300, [300, 211], 140, 20),
                                                                    (20, 3, 5, 64, 333, [333, 90, 170], 128, 128),
                                                                    (16, 16, 1, 128, 700, [700 - 20 * i for i in range(16)], 600, 0)])
def test_an_eviction_that_moves_whole_rows(ops, L, B, Hkv, d, max_len, lengths, budget, recent):
    assert 2 * L * B * Hkv >= 512                                      # two workgroups per compute unit: rows are not cut into slices
    gen = torch.Generator().manual_seed(L)
    print(f"case evict L={L} B={B} Hkv={Hkv} d={d} budget={budget}", flush=True)
    w = torch.rand(L, B, Hkv, max_len, generator=gen)
    w[:, :, :, :40] += 1.0                                             # rows in front that stay where they are
    caches = [normal(gen, B, Hkv, max_len, d) for _ in range(2 * L)]
    kept, new_w, new, ref = evict_oracle(caches, w.numpy(), lengths, budget, recent, max_len)
    dev = [c.cuda() for c in caches]
    got = ops.evict_kv_cache_(dev[:L], dev[L:], w.cuda(), torch.tensor(lengths).cuda(), budget, recent)
    for g, r in zip(got, (kept, new_w, new)):
        assert np.array_equal(g.cpu().numpy(), r)
    for g, r in zip(dev, ref):
        assert equal_bits(g, r)


@pytest.mark.parametrize("max_len,n", [(14200, 14200), (16384, 16384), (16385, 16385), (16384, 9)])
def test_an_eviction_at_the_limit_of_what_is_staged(ops, max_len, n):
    gen = torch.Generator().manual_seed(n)
    print(f"case evict max_len={max_len} n={n}", flush=True)
    w = torch.exp(20 * torch.rand(1, 1, 2, max_len, generator=gen))
    caches = [normal(gen, 1, 2, max_len, 8) for _ in range(2)]
    kept, new_w, new, ref = evict_oracle(caches, w.numpy(), [n], 4000, 300, max_len)
    dev = [c.cuda() for c in caches]
    got = ops.evict_kv_cache_(*dev, w.cuda(), torch.tensor([n]).cuda(), 4000, 300)
    for g, r in zip(got, (kept, new_w, new)):
        assert np.array_equal(g.cpu().numpy(), r)
    for g, r in zip(dev, ref):
        assert equal_bits(g, r)


@pytest.mark.parametrize("T,past,Hq", [(130, 0, 32), (200, 33, 32)])
def test_column_sums_of_many_heads_at_once(ops, T, past, Hq):
    """2048 blocks of slots or more: one chunk of queries, several tiles of 64 in it, added straight to the weights."""
    B, Hkv, d, n = 64, 32, 128, past + T
    gen = torch.Generator("cuda").manual_seed(T)
    print(f"case prefill weights B={B} T={T} Hkv={Hkv} past={past}", flush=True)
    q, kc, vc = (torch.randn(s, device="cuda", generator=gen).half() for s in ((B, T, Hq, d), (B, Hkv, n, d), (B, Hkv, n, d)))
    weights = torch.rand(B, Hkv, n, device="cuda", generator=gen)
    dev = weights.clone()
    ops.prefill_attention_weights(q, kc, vc, past, dev)
    q, kc, vc, weights = (x.cpu() for x in (q, kc, vc, weights))
    assert (dev.cpu().double().sum(-1) - weights.double().sum(-1) - T * Hq / Hkv).abs().max() <= 1e-2   # a probability of one a query
    seen = torch.ones(T, n, dtype=torch.bool).tril(past)
    for b, g in ((0, 0), (0, 31), (31, 7), (63, 0), (63, 31)):
        added, sizes = 0, 0
        for h in range(g * Hq // Hkv, (g + 1) * Hq // Hkv):
            _, p, size = attend64(q[b, :, h].double(), kc[b, g].double(), vc[b, g].double(), seen, d ** -0.5)
            added, sizes = added + p.sum(0), max(sizes, size)
        total = weights[b, g].double() + added
        tol = weights_tolerance(sizes, d, n, T * Hq // Hkv, added, total)
        assert ((dev[b, g].cpu().double() - total).abs() <= tol).all()


@pytest.mark.parametrize("T", [1, 40, 100])                            # one, two and four groups of 32 query rows
@pytest.mark.parametrize("d", [64, 128])
def test_rotated_queries_are_not_rounded_to_fp16(ops, T, d):
    """Two cached slots: a key made of the signs of the rotated query's rounding errors, with one channel that makes its score nothing,
    and a zero key; values 1 and -1.  Rounding the query moves the first score by the sum of all its errors."""
    gen = torch.Generator().manual_seed(d + T)
    B, H, max_len = 2, 4, 128
    q = normal(gen, B, 1, H, d, scale=8.0).expand(B, T, H, d).contiguous()
    q[..., 0] = q[..., 0].sign() * 24 + (q[..., 0] == 0) * 24
    angle = torch.rand(B, 1, d // 2, generator=gen, dtype=torch.float64) * 6.28
    angle[..., 0] = 0.0                                                # (channel 0 keeps its 24)
    angle = torch.cat((angle, angle), -1).expand(B, T, d)
    cos, sin = angle.cos().half().contiguous(), angle.sin().half().contiguous()
    qr = rotate64(q, cos, sin)                                         # [B, T, H, d]
    kc, vc = torch.zeros(B, H, max_len, d).half(), torch.zeros(B, H, max_len, d).half()
    for b in range(B):
        for h in range(H):
            x = qr[b, 0, h]
            k = (x.half().double() - x).sign()
            k[0] = 0
            k[0] = -(x @ k) / x[0]
            kc[b, h, 0] = k.half()
    vc[:, :, 0], vc[:, :, 1] = 1.0, -1.0
    new = normal(gen, B, T, H, d)
    mask, lengths = torch.zeros(T, T, dtype=torch.bool), torch.full((B,), 2)
    out = ops.tree_attention(*(t.cuda() for t in (q, new, new, cos, sin, lengths, mask, kc, vc))).cpu().double().view(B, T, H, d)
    beyond = 0
    for b in range(B):
        for h in range(H):
            k, v = kc[b, h, :2].double(), vc[b, h, :2].double()
            seen = torch.ones(T, 2, dtype=torch.bool)
            ref, _, size = attend64(qr[b, :, h], k, v, seen, d ** -0.5)
            rounded, _, _ = attend64(qr[b, :, h].half().double(), k, v, seen, d ** -0.5)
            # the result and two probabilities rounded to fp16; a score of d + 4 float32 steps and the low half's rounding, half of which
            # a difference of two probabilities (each moves by at most a quarter) sees
            tol = H16 + 2 * H16 + 0.5 * size * ((d + 4) * H32 + 2 ** -22) + 1e-5
            assert ((out[b, :, h] - ref).abs() <= tol).all()
            beyond += ((rounded - ref).abs() > tol).all().item()
    assert beyond == B * H                                             # ... which a rounded query is outside of


@pytest.mark.parametrize("layers", [2, 130])
def test_a_captured_commit(ops, layers):
    gen = torch.Generator().manual_seed(layers)
    rng = np.random.default_rng(layers)
    B, T, Hkv, d, max_len = 3, 20, 2, 64, 90
    tokens, chosen = torch.zeros(B, T, dtype=torch.int64).cuda(), torch.zeros(B, T, dtype=torch.int64).cuda()
    parents = np.array([-1] + [int(rng.integers(max(0, i - 3), i)) for i in range(1, T)])
    up, lengths = torch.from_numpy(parents).cuda(), torch.zeros(B, dtype=torch.int64).cuda()
    dev = [normal(gen, B, Hkv, max_len, d).cuda() for _ in range(2 * layers)]
    ops.tree_commit_(tokens, up, chosen, lengths, dev[:layers], dev[layers:])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.tree_commit_(tokens, up, chosen, lengths, dev[:layers], dev[layers:])
    for lens in ([5, 70, 33], [-1, 0, 71], [70, 69, 1]):
        t, c = rng.integers(0, 2, (B, T)), rng.integers(0, 2, (B, T))
        for to, x in ((tokens, t), (chosen, c), (lengths, np.array(lens))):
            to.copy_(torch.from_numpy(x))
        caches = [x.cpu() for x in dev]
        torch.zeros(1000, device="cuda").add_(1)
        graph.replay()
        torch.cuda.synchronize()
        path, accepted, following, new, ref = commit_oracle(t, parents, c, lens, caches, max_len)
        for g, r in zip(got, (path, accepted, following, new)):
            assert np.array_equal(g.cpu().numpy(), r)
        for g, r in zip(dev, ref):
            assert equal_bits(g, r)

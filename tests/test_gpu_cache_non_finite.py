"""Attention weights where a query or a cached key is no number: every slot that such a query sees gets NaN, all others keep the
sums of the other queries."""
import pytest
import torch

from test_gpu_cache_operators import attend64, normal, ops, weights_tolerance  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("B,T,Hq,Hkv,past,odd", [(1, 100, 4, 2, 30, 37), (2, 70, 2, 2, 0, 1), (1, 300, 4, 1, 77, 255), (1, 5, 2, 1, 200, 0),
                                                  (1, 130, 2, 1, 64, 129)])
def test_a_prompt_with_one_odd_query(ops, B, T, Hq, Hkv, past, odd, value):
    gen = torch.Generator().manual_seed(T)
    d, n = 128, past + T
    print(f"case prefill weights, odd query B={B} T={T} Hq={Hq} Hkv={Hkv} past={past} {odd} {value}", flush=True)
    q = normal(gen, B, T, Hq, d, scale=2.0)
    kc, vc = normal(gen, B, Hkv, n + 3, d), normal(gen, B, Hkv, n + 3, d)
    weights = torch.rand(B, Hkv, n + 3, generator=gen)
    head, rep = Hq - 1, Hq // Hkv                                      # the last head of the first sequence
    if value != value:
        q[0, odd, head] = value
    else:
        q[0, odd, head, 5] = value                                     # scores of either infinity
        kc[0, -1, :2, 5] = torch.tensor([1.0, -1.0]).half()
    dev = weights.cuda()
    ops.prefill_attention_weights(q.cuda(), kc.cuda(), vc.cuda(), past, dev)
    got = dev.cpu()
    assert torch.equal(got[:, :, n:], weights[:, :, n:])
    seen = torch.ones(T, n, dtype=torch.bool).tril(past)
    for b in range(B):
        for g in range(Hkv):
            added, sizes = 0, 0
            for h in range(g * rep, (g + 1) * rep):
                rows = [t for t in range(T) if not (b == 0 and h == head and t == odd)]
                _, p, size = attend64(q[b, rows, h].double(), kc[b, g, :n].double(), vc[b, g, :n].double(), seen[rows], d ** -0.5)
                added, sizes = added + p.sum(0), max(sizes, size)
            total = weights[b, g, :n].double() + added
            tol = weights_tolerance(sizes, d, n, T * rep, added, total)
            spoilt = past + odd + 1 if b == 0 and g == Hkv - 1 else 0
            assert torch.isnan(got[b, g, :spoilt]).all()
            assert ((got[b, g, spoilt:n].double() - total[spoilt:]).abs() <= tol[spoilt:]).all()


@pytest.mark.parametrize("B,Hq,Hkv,d,n,slot", [(2, 8, 2, 128, 300, 5), (1, 4, 4, 64, 1000, 999), (1, 70, 1, 128, 130, 64)])
def test_a_decode_step_over_a_key_that_is_no_number(ops, B, Hq, Hkv, d, n, slot):
    gen = torch.Generator().manual_seed(n)
    print(f"case decode weights, odd key B={B} Hq={Hq} Hkv={Hkv} d={d} {n} {slot}", flush=True)
    q, kc, vc = normal(gen, B, Hq, d), normal(gen, B, Hkv, n + 7, d), normal(gen, B, Hkv, n + 7, d)
    kc[0, 0, slot, 3] = float("nan")
    weights = torch.rand(B, Hkv, n + 7, generator=gen)
    dev, clean = weights.cuda(), weights.cuda()
    lengths = torch.tensor([n] * B).cuda()
    out = ops.decode_attention_weights(q.cuda(), kc.cuda(), vc.cuda(), lengths, dev)
    kc[0, 0, slot, 3] = 0
    ref = ops.decode_attention_weights(q.cuda(), kc.cuda(), vc.cuda(), lengths, clean)
    assert torch.isnan(out[0, :Hq // Hkv]).all() and torch.isnan(dev[0, 0, :n]).all()
    dev[0, 0, :n] = clean[0, 0, :n]                                    # everything else has the bits it has without the NaN
    out[0, :Hq // Hkv] = ref[0, :Hq // Hkv]
    assert torch.equal(dev, clean) and torch.equal(out, ref)

"""Attention over caches in 4 bits where one wave adds up hundreds of thousands of keys with nearly the same probability: the result grows with the
root of their number, what the accumulators hold beside it must not grow with the number itself.

The tolerance, of the 2-norm over some queries and all channels, counts independent roundings (codes are random and symmetric, so the squares of the
weighted codes add up to the square of the result): half a step of fp16 is at most 2^-11 of a value and evenly spread, 2^-11 / sqrt(3) in the mean
square, once for every weight and once for the result, sqrt(2 / 3) 2^-11 together.  A matrix instruction takes sixteen keys or more and rounds what has been added up
to float32, at most 2^-24 of it: of the result's own size, and of the eight that each code has on top, which is allowed to stay for 1024 keys of a wave: sqrt(n / 16)
2^-24 (1 + 8 1024 / (sqrt(n) r)) of the result for codes of root mean square r.  The cut of the products' low bits, 2^-18 of a weight for each instruction, is sqrt(n /
16) 2^-18 / (sqrt(n) r).  A weight's scale is up to twice another's, which counts as a factor of two for the last two; a score's rounding moves a probability by its
own size, below 2^-14 for the queries here."""
import pytest
import torch

from test_gpu_cache_i4 import hadamard64, packed

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["default", "ctypes"])
def ops(request):
    if request.param == "ctypes":
        from flh_amd import _ops
        return _ops
    import flh_amd
    return flh_amd._CUDA


def symmetric(gen, H, n, d):
    """Codes of -7 .. 7 and scales of 0.1 .. 0.2 (CPU): (codes int8, bytes, scales), one sequence"""
    codes = torch.randint(-7, 8, (1, H, n, d), generator=gen, dtype=torch.int8)
    return codes, packed(codes), (0.1 + 0.1 * torch.rand(1, H, n, generator=gen)).half()


def tolerance(n):
    r = (sum(c * c for c in range(-7, 8)) / 15) ** 0.5
    return (2 / 3) ** 0.5 * 2.0 ** -11 + (n / 16) ** 0.5 * 2.0 ** -24 * (1 + 2 * 8 * 1024 / (n ** 0.5 * r)) + 2 * 2.0 ** -18 / (4 * r) + 2.0 ** -14


def off(got, want):
    return ((got.double().cpu() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("n", [1500, 250000])
@pytest.mark.parametrize("d,rep", [(128, 64), (64, 128)])
def test_blocks_behind_many_keys_of_one_weight(ops, d, rep, n):
    gen = torch.Generator().manual_seed(n + d)
    T = 1024
    assert T * rep // 32 >= 2048 * (128 // d)                          # (a wave has rows of its own, and all keys)
    (kc, kb, ks), (vc, vb, vs) = symmetric(gen, 1, n + T, d), symmetric(gen, 1, n + T, d)
    q = (torch.randn(1, T, rep, d, generator=gen) * 1e-3).half()
    got = ops.prefill_attention_i4(q.cuda(), torch.tensor([n]).cuda(), kb.cuda(), ks.cuda(), vb.cuda(), vs.cuda()).view(T, rep, d)
    ts, k, v = torch.arange(5, T, 97), kc[0, 0].double() * ks[0, 0].double()[:, None], vc[0, 0].double() * vs[0, 0].double()[:, None]
    for h in (0, rep - 1):
        s = (q[0, ts, h].double() @ k.t()) * d ** -0.5
        p = torch.softmax(s.masked_fill(torch.arange(n + T) > n + ts[:, None], -torch.inf), -1)
        x = off(got[ts, h], p @ v)
        assert x <= tolerance(n), h


@pytest.mark.parametrize("d,n", [(64, 400000), (128, 120000)])
def test_tokens_behind_many_keys_of_one_weight(ops, d, n):
    """512 heads of the same codes and scales, one to a workgroup, whose waves take a quarter of its keys each."""
    gen = torch.Generator().manual_seed(d)
    H = 512
    (kc, kb, ks), (vc, vb, vs) = symmetric(gen, 1, n + 1, d), symmetric(gen, 1, n + 1, d)
    q = (torch.randn(1, H, d, generator=gen) * 1e-3).half()
    one, zero, new = torch.ones(1, d).half(), torch.zeros(1, d).half(), torch.zeros(1, H, d).half()
    cache = [t.cuda().expand(1, H, *t.shape[2:]).contiguous() for t in (kb, ks, vb, vs)]
    got = ops.decode_attention_rope_i4(*(t.cuda() for t in (q, new, new, one, zero, torch.tensor([n]))), *cache)
    k, v = kc[0, 0].double() * ks[0, 0].double()[:, None], vc[0, 0].double() * vs[0, 0].double()[:, None]
    k[n] = v[n] = 0                                                    # (the new token's)
    heads = torch.arange(3, H, 101)
    p = torch.softmax((q[0, heads].double() @ hadamard64(d) @ k.t()) * d ** -0.5, -1)
    x = off(got[0, heads], p @ v)
    assert x <= tolerance(n)

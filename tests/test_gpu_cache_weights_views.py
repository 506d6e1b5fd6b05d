import pytest
import torch

from test_gpu_cache_operators import normal, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def test_one_layers_view_of_the_sums(ops):
    """The sums of all layers as eviction takes them, one layer's view at a time: 8 bytes behind a 16-byte boundary here."""
    gen = torch.Generator().manual_seed(0)
    L, B, Hq, Hkv, d, max_len, past, T = 3, 1, 4, 2, 128, 41, 9, 30
    kc, vc = normal(gen, B, Hkv, max_len, d).cuda(), normal(gen, B, Hkv, max_len, d).cuda()
    sums = torch.rand(L, B, Hkv, max_len, generator=gen).cuda()
    assert sums[1].data_ptr() % 16 == 8
    want = sums.clone()
    lengths, q, qs = torch.tensor([33]).cuda(), normal(gen, B, Hq, d).cuda(), normal(gen, B, T, Hq, d).cuda()
    own = want[1].clone()
    a, b = ops.decode_attention_weights(q, kc, vc, lengths, own), ops.prefill_attention_weights(qs, kc, vc, past, own)
    want[1] = own
    assert torch.equal(ops.decode_attention_weights(q, kc, vc, lengths, sums[1]), a)
    assert torch.equal(ops.prefill_attention_weights(qs, kc, vc, past, sums[1]), b)
    assert torch.equal(sums, want)

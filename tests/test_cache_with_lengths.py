"""A StaticKVCache whose sequences have lengths of their own (host side)."""
import pytest
import torch

from flh_amd.quantized_model import StaticKVCache


def test_one_common_length_is_refused_once_the_sequences_have_their_own():
    cache = StaticKVCache(2, 2, 2, 16, 8, "cpu")
    cache.advance(3)
    cache.layer(1)
    assert cache.begin_drafts().tolist() == [3, 3] and cache.cut is None
    for call in (lambda: cache.advance(1), lambda: cache.layer(0)):
        with pytest.raises(ValueError, match="lengths of their own"):
            call()


def test_lengths_of_a_step_over_a_cache_that_has_been_cut():
    cache = StaticKVCache(1, 4, 2, 16, 8, "cpu", max_positions=40)
    cache.begin_drafts()
    cache.lengths.copy_(torch.tensor([10, 10, -3, 2 ** 63 - 1]))
    cache.cut.copy_(torch.tensor([25, 26, 100, 7]))
    assert cache.step_lengths(5).tolist() == [10, -1, -1, 2 ** 63 - 1]   # positions 35 .. 39 are the table's last
    assert cache.next_positions()[:2].tolist() == [35, 36]

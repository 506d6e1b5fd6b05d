"""Padded batches on a QuantizedKVCache, without a device: which sequences move on, and what the C entries refuse."""
import pytest
import torch

from flh_amd import _lib
from flh_amd.quantized_model import QuantizedKVCache


def test_a_sequence_moves_on_by_its_own_tokens_where_they_fit():
    cache = QuantizedKVCache(1, 7, 1, 10, 64, "cpu")
    cache.lengths.copy_(torch.tensor([8, 8, 10, 0, -1, 3, 3]))
    cache.advance(5, counts=torch.tensor([2, 3, 0, 5, 1, 6, -1]))
    assert cache.lengths.tolist() == [10, 8, 10, 5, -1, 3, 3]          # (8 + 3 do not fit; counts of 6 and -1 of 5 tokens are none)


def test_single_tokens_of_padding_take_no_part():
    cache = QuantizedKVCache(1, 3, 1, 10, 64, "cpu")
    cache.lengths.copy_(torch.tensor([4, 5, 9]))
    counts = torch.tensor([1, 0, 1])
    assert cache.step_lengths(1, counts).tolist() == [4, -1, 9]
    assert cache.step_lengths(1) is cache.lengths and cache.step_lengths(2, counts) is cache.lengths


A = [0x1000000 * (i + 1) for i in range(13)]


@pytest.mark.parametrize("name,count,outputs,sizes", [
    ("flh_rope_quant_kv_cache_i4_counts", 12, (7, 8, 9, 10, 11), (2, 3, 8, 2, 128, 64, None)),
    ("flh_prefill_attention_i4_counts", 8, (7,), (2, 3, 8, 2, 128, 4096, 0.1, A[12], 1 << 23, None))])
def test_outputs_do_not_lie_on_the_counts(name, count, outputs, sizes):
    lib = _lib.load()
    at = 6 if name.startswith("flh_rope") else 2
    for o in outputs:
        p = A[:count]
        p[at] = p[o] + 8
        assert getattr(lib, name)(*p, *sizes) == -1 and b"shares memory" in lib.flh_last_error(), lib.flh_last_error()


@pytest.mark.parametrize("B,refused", [(1024, False), (1025, True)])
def test_outputs_of_large_batches_are_their_own(B, refused):
    """More than 1024 sequences go in several pairs of launches: an output of the first must not lie on what the next one reads."""
    lib = _lib.load()
    place = [(i + 2) << 40 for i in range(12)]

    def call(out, workspace_bytes):
        p = place[:11]
        p[10] = out
        return lib.flh_decode_attention_rope_i4(*p, B, 8, 2, 128, 64, 0.1, place[11], workspace_bytes, None)

    for out in (place[0] + 16, place[1], place[2] + 64, place[3], place[4]):
        if refused:
            assert call(out, 1 << 40) == -1 and b"shares memory" in lib.flh_last_error(), lib.flh_last_error()
        assert call(out, 64) == -1 and b"workspace" in lib.flh_last_error()       # (never launched here)

"""Sizes at the C entries of the operators on caches that their 32-bit counts do not hold (no device here: nothing is launched)."""
import pytest

from flh_amd import _lib

MAX = 2 ** 32 - 1


@pytest.mark.parametrize("name,args", [
    ("flh_prefill_attention_weights_workspace_bytes", (1, 1, 8, 2, MAX)),          # the number of slots wraps to none
    ("flh_prefill_attention_weights_workspace_bytes", (1, MAX, 8, 2, 0)),
    ("flh_prefill_attention_weights_workspace_bytes", (MAX, MAX, MAX, 1, 0)),
    ("flh_prefill_attention_weights_workspace_bytes", (MAX, 1, MAX, MAX, 2 ** 20)),
    ("flh_tree_attention_workspace_bytes", (1, 2 ** 20, 2 ** 19, 1, 128)),         # 2^32 blocks of rows
    ("flh_tree_attention_workspace_bytes", (MAX, 256, MAX, MAX, 128)),
    ("flh_tree_attention_workspace_bytes", (MAX, MAX, MAX, 1, MAX)),
    ("flh_tree_attention_workspace_bytes", (2, 8, 8, 0, 128)),
    ("flh_decode_attention_weights_workspace_bytes", (1, 8, 8, 128, MAX)),
    ("flh_decode_attention_weights_workspace_bytes", (MAX, MAX, 1, 128, MAX))])
def test_workspace_sizes_of_calls_that_are_refused(name, args):
    assert getattr(_lib.load(), name)(*args) == 0


@pytest.mark.parametrize("name,args,least", [
    ("flh_prefill_attention_weights_workspace_bytes", (2, 100, 8, 2, 30), 2 * 100 * 8 * 4),
    ("flh_tree_attention_workspace_bytes", (2, 8, 8, 2, 128), 2 * 2 * 32 * 130 * 4),
    ("flh_decode_attention_weights_workspace_bytes", (2, 8, 2, 64, 101), 2 * 8 * 104 * 4 + 2 * 2 * 32 * 66 * 4)])
def test_workspace_sizes_of_calls_that_run(name, args, least):
    assert least <= getattr(_lib.load(), name)(*args) < 2 ** 30

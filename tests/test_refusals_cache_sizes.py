"""Sizes at the C entries of the operators on caches that their 32-bit counts do not hold (no device here: nothing is launched)."""
import ctypes

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


OK, BIG = 0x10000, 1 << 60
CACHES = ((ctypes.c_void_p * 1)(1 << 50), (ctypes.c_void_p * 1)(1 << 56))


@pytest.mark.parametrize("name,args", [
    ("flh_tree_attention_f16", (*[OK] * 7, 0, OK, OK, OK, 1 << 20, 1, 4, 4, 128, 64, 0.1, OK, BIG, None)),
    ("flh_decode_attention_weights_f16", (*[OK] * 6, 1 << 20, 4, 4, 128, 64, 0.1, OK, BIG, None)),
    ("flh_decode_attention_weights_f16", (*[OK] * 6, 1 << 21, 4, 4, 64, 256, 0.1, OK, BIG, None)),
    ("flh_prefill_attention_weights_f16", (*[OK] * 5, 1 << 22, 1, 4, 4, 128, 0, 64, 0.1, OK, BIG, None)),
    ("flh_tree_commit", (OK, OK, 0, OK, 2 * OK, OK, OK, OK, 3 * OK, 1, *CACHES, 1 << 24, 8, 2, 8, 16, None)),
    ("flh_evict_kv_cache", (1, *CACHES, OK, OK, OK, 2 * OK, 2 * OK, 1 << 22, 2, 8, 16, 8, 4, None))])
def test_launches_of_more_items_than_32_bits_count(name, args):
    """Refused in front of the first launch, not by the runtime behind the one that has written the caches."""
    lib = _lib.load()
    assert getattr(lib, name)(*args) == -1 and b"too large" in lib.flh_last_error(), lib.flh_last_error()


@pytest.mark.parametrize("name,args", [
    ("flh_decode_attention_weights_f16", (OK, OK, OK, OK, OK, "weights", 1, 8, 2, 128, 64, 0.1, OK, 4, None)),
    ("flh_prefill_attention_weights_f16", (OK, OK, OK, OK, "weights", 1, 4, 8, 2, 128, 0, 64, 0.1, OK, 4, None))])
def test_sums_of_weights_are_aligned_as_floats(name, args):
    lib = _lib.load()
    for at, message in ((OK + 2, b"4-byte aligned"), (OK + 4, b"workspace"), (OK + 8, b"workspace")):
        assert getattr(lib, name)(*(at if x == "weights" else x for x in args)) == -1
        assert message in lib.flh_last_error(), lib.flh_last_error()


AT = [(i + 2) << 32 for i in range(12)]                                # places far from one another


@pytest.mark.parametrize("k,v", [(AT[0], AT[0]), (AT[0], AT[0] + 16), (AT[0] + 2 * 2 * 64 * 128 * 2 - 16, AT[0])])
def test_the_caches_of_a_tree_share_no_memory(k, v):
    lib = _lib.load()
    assert lib.flh_tree_attention_f16(*[OK] * 7, 0, k, v, OK, 2, 8, 8, 2, 128, 64, 0.1, OK, BIG, None) == -1
    assert b"share memory" in lib.flh_last_error()


@pytest.mark.parametrize("shift", [0, 16, 1 * 4 * 8 * 128 * 2 - 16, -16])
def test_the_output_of_a_prompt_with_weights_is_not_its_queries(shift):
    lib = _lib.load()
    assert lib.flh_prefill_attention_weights_f16(AT[0], AT[1], AT[2], AT[0] + shift, AT[3], 1, 4, 8, 2, 128, 0, 64, 0.1, OK, BIG, None) == -1
    assert b"memory of its own" in lib.flh_last_error()


@pytest.mark.parametrize("one,other,shift,message", [(4, 0, 0, b"with an input"), (4, 2, 8, b"with an input"), (5, 1, 56, b"with an input"),
                                                     (6, 3, 8, b"with an input"), (4, 3, -8, b"with an input"),
                                                     (5, 4, 8, b"two outputs"), (6, 5, 0, b"two outputs"), (7, 6, 8, b"two outputs")])
def test_the_outputs_of_a_commit_are_in_memory_of_their_own(one, other, shift, message):
    at = AT[:8]                                                        # tokens, parents, chosen, lengths; path, accepted, next, new lengths
    at[one] = at[other] + shift
    lib = _lib.load()
    assert lib.flh_tree_commit(*at[:2], 0, *at[2:], 1, *CACHES, 2, 8, 2, 8, 16, None) == -1
    assert message in lib.flh_last_error(), lib.flh_last_error()


@pytest.mark.parametrize("one,other,shift,message", [(2, 0, 0, b"with an input"), (3, 0, 4, b"with an input"), (4, 1, 8, b"with an input"),
                                                     (3, 2, 8, b"two outputs"), (4, 3, 0, b"two outputs")])
def test_the_outputs_of_an_eviction_are_in_memory_of_their_own(one, other, shift, message):
    at = AT[:5]                                                        # weights, lengths; kept, new weights, new lengths
    at[one] = at[other] + shift
    lib = _lib.load()
    assert lib.flh_evict_kv_cache(1, *CACHES, *at, 2, 2, 8, 16, 8, 4, None) == -1
    assert message in lib.flh_last_error(), lib.flh_last_error()


def test_a_decode_step_over_caches_without_slots_is_refused():
    """(zeros are documented where there is nothing to see: success without writing them is not that)"""
    lib = _lib.load()
    assert lib.flh_decode_attention_weights_f16(*AT[:6], 2, 8, 2, 128, 0, 0.1, OK, BIG, None) == -1
    assert b"no slots" in lib.flh_last_error()

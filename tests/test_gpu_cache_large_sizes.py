"""Caches with an axis that the C ABI's 32-bit sizes do not hold (68 GB at least; here of no sequences, which takes no memory)."""
import pytest
import torch

from test_gpu_cache_operators import ops  # noqa: F401

pytestmark = pytest.mark.gpu


def test_slots_beyond_32_bits_are_refused(ops):
    max_len = 2 ** 32 + 64                                             # 64 when cut to 32 bits
    z = lambda *s, dtype=torch.float16: torch.empty(*s, dtype=dtype, device="cuda")
    cache, lengths = z(0, 2, max_len, 8), z(0, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="too large"):
        ops.evict_kv_cache_(cache, cache.clone(), z(1, 0, 2, max_len, dtype=torch.float32), lengths, 32, 4)
    tokens = z(0, 4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="too large"):
        ops.tree_commit_(tokens, tokens, tokens, lengths, cache, cache.clone())

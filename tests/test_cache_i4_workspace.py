"""The scratch that a QuantizedKVCache keeps for its attention (CPU: sizes alone): one tensor, whatever the steps' lengths."""
import pytest
import torch

from flh_amd import _lib
from flh_amd.quantized_model import QuantizedKVCache, decoder_layer


def needs(batch, t, q_heads, kv_heads, d, max_len):
    lib = _lib.load()
    return (lib.flh_decode_attention_i4_workspace_bytes(batch, q_heads, kv_heads, d, max_len) if t == 1 else
            lib.flh_prefill_attention_i4_workspace_bytes(batch, t, q_heads, kv_heads, d, max_len))


class Recorder:
    """Stands in for the operators: keeps the scratch that each call is given."""

    def __init__(self):
        self.given = []

    def rope_quantize_kv_cache_(self, q, *_, counts):
        return q

    def prefill_attention_i4(self, q, *_, workspace, counts):
        self.given.append(workspace)
        return q.flatten(2)

    def decode_attention_rope_i4(self, q, *_, workspace):
        self.given.append(workspace)
        return q


@pytest.fixture
def ops(monkeypatch):
    recorder = Recorder()
    monkeypatch.setattr(decoder_layer, "_ops", lambda: recorder)
    return recorder


def attend(cache, t, q_heads):
    codes = cache.layers[0][0]
    b, kv_heads, d = codes.size(0), codes.size(1), cache.head_dim
    q, kv, rows = (torch.empty(1).half().expand(b, t, *s) for s in ((q_heads, d), (kv_heads, d), (d,)))
    cache.layer(0).attend(q, kv, kv, rows, rows)


@pytest.mark.parametrize("batch,q_heads,kv_heads,d,max_len", [(1, 32, 8, 128, 3000), (1, 28, 4, 128, 3000), (3, 16, 16, 64, 900), (1, 2, 1, 64, 3000),
                                                              (300, 4, 4, 128, 70), (2, 40, 2, 128, 5), (1, 64, 1, 128, 1)])
def test_steps_of_every_length_share_one(ops, batch, q_heads, kv_heads, d, max_len):
    cache = QuantizedKVCache(2, batch, kv_heads, max_len, d, "cpu")
    for t in (*range(1, min(max_len, 60) + 1), *range(max_len, 60, -7), max_len):
        attend(cache, t, q_heads)
        assert ops.given[-1].numel() >= needs(batch, t, q_heads, kv_heads, d, max_len)
    kept = {ws.data_ptr(): ws.numel() for ws in ops.given}             # (all of them are still held here)
    assert len(kept) == 1
    # (pieces of what 512 workgroups and one a block take, no more than 256 blocks, 32 rows of d + 2 floats each; the decode step's of 16)
    assert sum(kept.values()) <= max(768 * 32 * (d + 2) * 4, needs(batch, 1, q_heads, kv_heads, d, max_len))

"""Two threads that launch on one stream through the ctypes route, which gives the interpreter up during a call: the launches of one
call must not come between those of another that has the same default workspace (a stand-in library, no device)."""
import threading
import time

import pytest
import torch

from flh_amd import _ops


class OnDevice(torch.Tensor):
    """Host memory that says it is on a device."""
    is_cuda = property(lambda self: True)


def dev(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnDevice)


def calls():
    B, T, Hq, Hkv, d, n = 1, 3, 2, 2, 128, 16
    cache, new, row = dev(B, Hkv, n, d), dev(B, T, Hkv, d), dev(B, T, d)
    lengths, weights = dev(B, dtype=torch.int64), dev(B, Hkv, n, dtype=torch.float32)
    return {
        "decode_attention": lambda ws: _ops.decode_attention(dev(B, Hq, d), cache, cache, 4, workspace=ws),
        "decode_attention_rope": lambda ws: _ops.decode_attention_rope(dev(B, Hq, d), dev(B, Hkv, d), dev(B, Hkv, d), dev(d), dev(d),
                                                                       lengths, cache, cache, 4, workspace=ws),
        "tree_attention": lambda ws: _ops.tree_attention(dev(B, T, Hq, d), new, new, row, row, lengths, dev(T, T, dtype=torch.bool),
                                                         cache, cache, workspace=ws),
        "decode_attention_weights": lambda ws: _ops.decode_attention_weights(dev(B, Hq, d), cache, cache, lengths, weights, workspace=ws),
        "prefill_attention_weights": lambda ws: _ops.prefill_attention_weights(dev(B, T, Hq, d), cache, cache, 0, weights, workspace=ws),
    }


@pytest.fixture
def launches(monkeypatch):
    """What the stand-in library saw: (thread, enters / leaves, workspace address)."""
    seen = []

    def entry(*args):
        at = args[-3]                                                  # workspace, its bytes, stream
        seen.append((threading.get_ident(), "enters", at))
        time.sleep(0.05)
        seen.append((threading.get_ident(), "leaves", at))
        return 0

    class Library:
        def __getattr__(self, name):
            return (lambda *args: 1000) if name.endswith("_workspace_bytes") else entry

    monkeypatch.setattr(_ops._lib, "load", lambda: Library())
    monkeypatch.setattr(_ops, "_stream", lambda t: 0)
    monkeypatch.setattr(_ops, "_run", lambda name, device, *args: entry(*args))
    monkeypatch.setattr(_ops, "_attention_workspaces", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return seen


def both(call, *args):
    threads = [threading.Thread(target=call, args=(a,)) for a in args]
    for t in threads:
        t.start()
    for t in threads:
        t.join()


@pytest.mark.parametrize("name", ["decode_attention", "decode_attention_rope", "tree_attention", "decode_attention_weights",
                                  "prefill_attention_weights"])
def test_calls_with_the_default_workspace_do_not_interleave(launches, name):
    both(calls()[name], None, None)
    assert len(launches) == 4 and len({at for _, _, at in launches}) == 1
    assert [what for _, what, _ in launches] == ["enters", "leaves"] * 2, launches
    assert launches[0][0] == launches[1][0] and launches[2][0] == launches[3][0]


def test_calls_with_workspaces_of_their_own_do_not_wait(launches):
    both(calls()["tree_attention"], *(dev(1 << 21, dtype=torch.uint8) for _ in range(2)))
    assert [what for _, what, _ in launches] == ["enters", "enters", "leaves", "leaves"], launches

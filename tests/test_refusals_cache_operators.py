"""What the operators on caches refuse, found on the host before any launch (no device here: the addresses are never used)."""
import ctypes

import pytest
import torch

from flh_amd import _lib, _ops

OK, ODD = 0x10000, 0x10008


def call(name, args, message):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == -1, (name, args)
    assert message in lib.flh_last_error(), lib.flh_last_error()


def tree(at=None, value=None, mask_per_sequence=0, B=2, T=8, Hq=8, Hkv=2, d=128, max_len=64, scale=0.1, ws=OK, ws_bytes=1 << 40):
    p = [OK] * 7
    caches = [OK] * 3
    if at is not None:
        (p if at < 7 else caches)[at if at < 7 else at - 7] = value
    return (*p, mask_per_sequence, *caches, B, T, Hq, Hkv, d, max_len, scale, ws, ws_bytes, None)


@pytest.mark.parametrize("more,message", [
    (dict(at=0, value=None), b"null pointer"), (dict(at=6, value=None), b"null pointer"), (dict(at=5, value=None), b"null pointer"),
    (dict(at=0, value=ODD), b"16-byte aligned"), (dict(at=9, value=ODD), b"16-byte aligned"), (dict(at=3, value=ODD), b"16-byte aligned"),
    (dict(d=96), b"head_dim (96) must be 64 or 128"), (dict(Hq=7), b"do not divide"), (dict(Hkv=0), b"do not divide"),
    (dict(T=257), b"257 nodes"), (dict(scale=0.0), b"scale"), (dict(scale=float("nan")), b"scale"), (dict(scale=float("inf")), b"scale"), (dict(scale=1e16), b"scale"),
    (dict(B=1 << 20, T=256), b"too large"), (dict(ws=None), b"workspace"), (dict(ws=ODD), b"workspace"), (dict(ws_bytes=8), b"workspace")])
def test_tree_attention(more, message):
    call("flh_tree_attention_f16", tree(**more), message)


@pytest.mark.parametrize("name,args,message", [
    ("flh_decode_attention_weights_f16", (OK, OK, OK, None, OK, OK, 1, 8, 2, 128, 64, 0.1, OK, 1 << 40, None), b"null pointer"),
    ("flh_decode_attention_weights_f16", (OK, ODD, OK, OK, OK, OK, 1, 8, 2, 128, 64, 0.1, OK, 1 << 40, None), b"16-byte aligned"),
    ("flh_decode_attention_weights_f16", (OK, OK, OK, OK, OK, OK, 1, 8, 2, 80, 64, 0.1, OK, 1 << 40, None), b"head_dim (80)"),
    ("flh_decode_attention_weights_f16", (OK, OK, OK, OK, OK, OK, 1, 8, 3, 128, 64, 0.1, OK, 1 << 40, None), b"do not divide"),
    ("flh_decode_attention_weights_f16", (OK, OK, OK, OK, OK, OK, 1, 8, 2, 128, 64, 0.1, OK, 4, None), b"workspace"),
    ("flh_decode_attention_weights_f16", (OK, OK, OK, OK, OK, OK, 1, 8, 2, 128, 64, -1.0, OK, 1 << 40, None), b"scale"),
    ("flh_prefill_attention_weights_f16", (OK, OK, OK, OK, None, 1, 4, 8, 2, 128, 0, 64, 0.1, OK, 1 << 40, None), b"null pointer"),
    ("flh_prefill_attention_weights_f16", (OK, OK, OK, OK, OK, 1, 4, 8, 2, 64, 0, 64, 0.1, OK, 1 << 40, None), b"head_dim (64) must be 128"),
    ("flh_prefill_attention_weights_f16", (OK, OK, OK, OK, OK, 1, 4, 8, 2, 128, 61, 64, 0.1, OK, 1 << 40, None), b"exceeds the cache length"),
    ("flh_prefill_attention_weights_f16", (OK, OK, OK, OK, OK, 1, 4, 8, 2, 128, 0, 64, 0.1, OK, 8, None), b"workspace")])
def test_attention_weights(name, args, message):
    call(name, args, message)


def pointers(*values):
    return (ctypes.c_void_p * len(values))(*values)


def commit(k=(OK,), v=(2 * OK,), T=8, Hkv=2, d=128, max_len=64, new=4 * OK, layers=None):
    return (OK, OK, 0, OK, 3 * OK, OK, OK, OK, new, len(k) if layers is None else layers, pointers(*k), pointers(*v), 1, T, Hkv, d, max_len, None)


@pytest.mark.parametrize("more,message", [(dict(T=0), b"0 nodes"), (dict(T=257), b"257 nodes"), (dict(new=3 * OK), b"memory of their own"),
                                          (dict(k=(None,)), b"null pointer"), (dict(v=(ODD,)), b"16-byte aligned"), (dict(d=100), b"head_dim (100)"),
                                          (dict(d=1024), b"head_dim (1024)"), (dict(max_len=0), b"must be positive"),
                                          (dict(k=(1 << 20,), v=(1 << 20,)), b"share memory"),
                                          (dict(k=(1 << 20, 1 << 30), v=(1 << 40, (1 << 20) + 1024)), b"share memory")])
def test_tree_commit(more, message):
    call("flh_tree_commit", commit(**more), message)


def evict(k=(OK,), v=(1 << 30,), w=1 << 31, n=1 << 32, new_w=1 << 33, new_n=1 << 34, max_len=64, budget=32, recent=4, layers=None, Hkv=2):
    return (len(k) if layers is None else layers, pointers(*k), pointers(*v), w, n, OK, new_w, new_n, 1, Hkv, 128, max_len, budget, recent, None)


@pytest.mark.parametrize("more,message", [(dict(w=None), b"null pointer"), (dict(budget=0), b"budget (0)"), (dict(budget=65), b"budget (65)"),
                                          (dict(recent=33), b"recent (33)"), (dict(new_w=1 << 31), b"memory of their own"),
                                          (dict(new_n=1 << 32), b"memory of their own"), (dict(layers=0), b"no layers"),
                                          (dict(k=(None,)), b"null pointer"), (dict(k=(1 << 30,)), b"share memory"), (dict(Hkv=0), b"must be positive")])
def test_evict(more, message):
    call("flh_evict_kv_cache", evict(**more), message)


def routes():
    import flh_amd
    return [_ops, flh_amd._CUDA]


@pytest.mark.parametrize("route", [0, 1])
def test_tensors_off_the_device_are_refused(route):
    ops = routes()[route]
    z = lambda *s, dtype=torch.float16: torch.zeros(*s, dtype=dtype)
    n, cache, w = z(1, dtype=torch.int64), z(1, 2, 16, 128), z(1, 2, 16, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.tree_attention(z(1, 4, 8, 128), z(1, 4, 2, 128), z(1, 4, 2, 128), z(1, 4, 128), z(1, 4, 128), n, z(4, 4, dtype=torch.bool), cache, cache)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.decode_attention_weights(z(1, 8, 128), cache, cache, n, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.prefill_attention_weights(z(1, 4, 8, 128), cache, cache, 0, w)
    t = z(1, 4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.tree_commit_(t, t, t, n, cache, cache)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.evict_kv_cache_([cache], [cache], w[None], n, 4, 0)

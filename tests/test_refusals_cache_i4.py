"""What the operators on caches in 4 bits refuse, found on the host before any launch (no device here: the addresses are never used)."""
import pytest
import torch

from flh_amd import _lib, _ops
from flh_amd.quantized_model import LlamaShape, QuantizedKVCache, StaticKVCache, W4A4LlamaModel

A = [0x1000000 * (i + 1) for i in range(12)]                           # addresses far apart
ODD = 0x1000008


def call(name, args, message):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == -1, (name, args)
    assert message in lib.flh_last_error(), lib.flh_last_error()


def with_(pointers, at, value):
    p = list(pointers)
    if at is not None:
        p[at] = value
    return p


def write(at=None, value=None, B=2, T=3, Hq=8, Hkv=2, d=128, max_len=64):
    return (*with_(A[:11], at, value), B, T, Hq, Hkv, d, max_len, None)


def read(at=None, value=None, B=2, rows=3, Hkv=2, d=128, max_len=64):
    return (*with_(A[:7], at, value), B, rows, Hkv, d, max_len, None)


def decode(at=None, value=None, B=2, Hq=8, Hkv=2, d=128, max_len=64, scale=0.1, ws=A[11], ws_bytes=1 << 23):
    return (*with_(A[:11], at, value), B, Hq, Hkv, d, max_len, scale, ws, ws_bytes, None)


def prefill(at=None, value=None, B=2, T=3, Hq=8, Hkv=2, d=128, max_len=4096, scale=0.1, ws=A[11], ws_bytes=1 << 23):
    return (*with_(A[:7], at, value), B, T, Hq, Hkv, d, max_len, scale, ws, ws_bytes, None)


NAMES = {"write": ("flh_rope_quant_kv_cache_i4", write), "read": ("flh_dequant_kv_cache_i4", read),
         "decode": ("flh_decode_attention_rope_i4", decode), "prefill": ("flh_prefill_attention_i4", prefill)}


@pytest.mark.parametrize("kind,count", [("write", 11), ("read", 7), ("decode", 11), ("prefill", 7)])
def test_null_pointers(kind, count):
    name, args = NAMES[kind]
    for at in range(count):
        call(name, args(at=at, value=None), b"null pointer")


@pytest.mark.parametrize("kind,aligned", [("write", (0, 1, 2, 3, 4, 6, 7, 9)), ("read", (0, 2, 5, 6)), ("decode", (0, 1, 2, 3, 4, 6, 8, 10)),
                                          ("prefill", (0, 2, 4, 6))])
def test_alignment(kind, aligned):
    name, args = NAMES[kind]
    for at in aligned:
        call(name, args(at=at, value=ODD), b"16-byte aligned")


@pytest.mark.parametrize("kind", list(NAMES))
def test_sizes(kind):
    name, args = NAMES[kind]
    call(name, args(d=96), b"head_dim (96)")
    call(name, args(d=256), b"head_dim (256)")
    call(name, args(Hkv=0), b"head" if kind in ("write", "read") else b"do not divide")
    call(name, args(max_len=0), b"cache")
    big = {"write": dict(T=1 << 28), "read": dict(rows=1 << 30), "decode": dict(B=1 << 22), "prefill": dict(T=1 << 26)}[kind]
    call(name, args(**big), b"too")
    call(name, args(B=1 << 30, max_len=1 << 31), b"too")
    if kind in ("decode", "prefill"):
        call(name, args(Hq=7), b"do not divide")
        call(name, args(Hq=0), b"do not divide")
        for scale in (0.0, -1.0, float("nan"), float("inf"), 1e16):
            call(name, args(scale=scale), b"scale")
        call(name, args(ws=None), b"workspace")
        call(name, args(ws=ODD), b"workspace")
        call(name, args(ws_bytes=64), b"workspace")
        call(name, args(max_len=1 << 26), b"too large")


def test_shared_memory():
    call("flh_rope_quant_kv_cache_i4", write(at=9, value=A[7]), b"share memory")             # the caches
    call("flh_rope_quant_kv_cache_i4", write(at=8, value=A[7] + 64), b"share memory")        # codes and scales
    call("flh_rope_quant_kv_cache_i4", write(at=6, value=A[0] + 16), b"shares memory")       # queries, but not in place
    call("flh_rope_quant_kv_cache_i4", write(at=6, value=A[1]), b"shares memory")
    call("flh_rope_quant_kv_cache_i4", write(at=10, value=A[5]), b"shares memory")
    call("flh_dequant_kv_cache_i4", read(at=6, value=A[5]), b"two outputs")
    call("flh_dequant_kv_cache_i4", read(at=5, value=A[0] + 256), b"shares memory")
    call("flh_decode_attention_rope_i4", decode(at=8, value=A[6]), b"share memory")
    call("flh_decode_attention_rope_i4", decode(at=10, value=A[6]), b"share memory")
    call("flh_decode_attention_rope_i4", decode(at=10, value=A[11]), b"share memory")        # output and workspace
    call("flh_decode_attention_rope_i4", decode(at=7, value=A[5]), b"shares memory")
    call("flh_decode_attention_rope_i4", decode(at=10, value=A[5] - A[5] % 16), b"shares memory")   # output and lengths
    call("flh_prefill_attention_i4", prefill(at=6, value=A[0]), b"shares memory")
    call("flh_prefill_attention_i4", prefill(at=6, value=A[11]), b"workspace")
    call("flh_prefill_attention_i4", prefill(at=2, value=A[11]), b"shares memory")


def test_nothing_to_do():
    lib = _lib.load()
    for name, args in (("flh_rope_quant_kv_cache_i4", write(B=0)), ("flh_rope_quant_kv_cache_i4", write(T=0)), ("flh_dequant_kv_cache_i4", read(rows=0)),
                       ("flh_dequant_kv_cache_i4", read(B=0)), ("flh_decode_attention_rope_i4", decode(B=0)), ("flh_prefill_attention_i4", prefill(T=0)),
                       ("flh_prefill_attention_i4", prefill(B=0))):
        assert getattr(lib, name)(*args) == 0, name


def test_workspace_sizes():
    lib = _lib.load()
    decode_bytes, prefill_bytes = lib.flh_decode_attention_i4_workspace_bytes, lib.flh_prefill_attention_i4_workspace_bytes
    assert decode_bytes(2, 8, 2, 128, 64) == (512 + 4) * 16 * 130 * 4
    assert decode_bytes(2, 40, 2, 64, 64) == (512 + 8) * 16 * 66 * 4
    assert prefill_bytes(1, 4096, 32, 8, 128, 4096) == 0 and prefill_bytes(2, 3, 8, 2, 128, 64) == 0
    assert 0 < prefill_bytes(2, 3, 8, 2, 128, 4096) <= 512 * 32 * 130 * 4
    for f, args in ((decode_bytes, (2, 7, 2, 128, 64)), (decode_bytes, (2, 8, 0, 128, 64)), (decode_bytes, (2, 8, 2, 80, 64)), (decode_bytes, (2, 8, 2, 128, 0)),
                    (decode_bytes, (2 ** 32 - 1, 2 ** 32 - 1, 1, 128, 2 ** 32 - 1)), (prefill_bytes, (2, 3, 8, 3, 128, 64)), (prefill_bytes, (0, 3, 8, 2, 128, 64)),
                    (prefill_bytes, (2 ** 32 - 1, 2 ** 32 - 1, 2 ** 32 - 1, 1, 128, 2 ** 32 - 1))):
        assert f(*args) == 0, args


def cpu_cache(B=2, Hkv=2, S=8, d=128):
    return [torch.zeros(B, Hkv, S, d // 2, dtype=torch.uint8), torch.zeros(B, Hkv, S).half(), torch.zeros(B, Hkv, S, d // 2, dtype=torch.uint8),
            torch.zeros(B, Hkv, S).half()]


@pytest.mark.parametrize("name", ["rope_quantize_kv_cache_", "dequantize_kv_cache", "decode_attention_rope_i4", "prefill_attention_i4"])
@pytest.mark.parametrize("route", ["default", "ctypes"])
def test_tensors_of_the_host_are_refused(name, route):
    if route == "default":
        import flh_amd
        ops = flh_amd._CUDA
    else:
        ops = _ops
    n, cache = torch.zeros(2, dtype=torch.int64), cpu_cache()
    q, kv, one = torch.zeros(2, 3, 4, 128).half(), torch.zeros(2, 3, 2, 128).half(), torch.zeros(2, 3, 128).half()
    args = {"rope_quantize_kv_cache_": (q, kv, kv, one, one, n, *cache), "dequantize_kv_cache": (*cache, n, 3),
            "decode_attention_rope_i4": (q[:, 0], kv[:, 0], kv[:, 0], one[:, 0], one[:, 0], n, *cache), "prefill_attention_i4": (q, n, *cache)}[name]
    with pytest.raises(RuntimeError, match="CUDA"):
        getattr(ops, name)(*args)


def test_model_refusals():
    shape = LlamaShape(256, 2, 2, 256, 1, 16, 1e-5, 10000.0)
    model = W4A4LlamaModel(shape, device="cpu")
    cache = model.new_cache(2, 8, bits=4)
    assert isinstance(cache, QuantizedKVCache) and isinstance(model.new_cache(2, 8), StaticKVCache)
    ids = torch.zeros(2, 1, dtype=torch.int64)
    for bad, match in ((lambda: model.new_cache(2, 8, bits=8), "16 or 4 bits"), (lambda: model.new_cache(2, 8, max_positions=9, bits=4), "not cut"),
                       (lambda: QuantizedKVCache(1, 1, 1, 8, 32, "cpu"), "64 or 128"), (lambda: model(ids, torch.zeros(1, dtype=torch.int64), cache), "append"),
                       (lambda: model.tree_step(ids, [0], cache), "drafts"), (lambda: model.append(ids, model.new_cache(2, 8)), "4 bits"),
                       (lambda: model.append(ids[:1], cache), "sequences"), (lambda: model.append(torch.zeros(2, 9, dtype=torch.int64), cache), "slots"),
                       (lambda: model.append(ids, cache, counts=torch.zeros(1, dtype=torch.int64)), "counts"),
                       (lambda: model.append(ids, cache, counts=torch.zeros(2)), "counts")):
        with pytest.raises(ValueError, match=match):
            bad()


def test_lengths_move_on():
    cache = QuantizedKVCache(1, 4, 1, 10, 64, "cpu")
    cache.lengths.copy_(torch.tensor([0, -1, 8, 7]))
    lengths = cache.lengths
    cache.advance(3)
    assert lengths.tolist() == [3, -1, 8, 10] and cache.lengths is lengths    # (8 + 3 do not fit: no part)
    cache.advance(5, counts=torch.tensor([2, 5, 5, 0]))
    assert lengths.tolist() == [5, -1, 8, 10]

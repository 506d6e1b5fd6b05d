"""The operators on caches in 4 bits on streams of their own, in graphs, at offsets beyond 32 bits, and the calls their Python side refuses."""
import pytest
import torch

from test_gpu_cache_i4 import check_decode, check_prefill, decode_case, normal, packed, prefill_case, quantised, random_cache, rotary, turned

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["default", "ctypes"])
def ops(request):
    if request.param == "ctypes":
        from flh_amd import _ops
        return _ops
    import flh_amd
    return flh_amd._CUDA


def test_capture_needs_a_workspace(ops):
    gen = torch.Generator().manual_seed(1)
    q, k, v, cos, sin, lengths, cache = decode_case(gen, 2, 8, 2, 128, 600, [100, 500])
    x, dev = [t.cuda() for t in (q, k, v, cos, sin, lengths)], [t.cuda() for t in cache]
    block = normal(gen, 2, 5, 8, 128).cuda()
    ops.decode_attention_rope_i4(*x, *dev)
    ops.prefill_attention_i4(block, x[5], *dev)
    for call in (lambda: ops.decode_attention_rope_i4(*x, *dev), lambda: ops.prefill_attention_i4(block, x[5], *dev)):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="workspace"):
            with torch.cuda.graph(graph):
                call()
    torch.cuda.synchronize()
    small = torch.empty(64, dtype=torch.uint8, device="cuda")
    with pytest.raises(RuntimeError, match="workspace"):
        ops.decode_attention_rope_i4(*x, *dev, workspace=small)


@pytest.mark.parametrize("T", [1, 5, 70])
def test_replays_follow_lengths_and_inputs(ops, T):
    """A captured write, attention and read, replayed for other tokens and lengths with eager work between, gives the eager bits."""
    gen = torch.Generator().manual_seed(T)
    B, Hq, Hkv, d, max_len = 3, 8, 2, 128, 900
    cache = random_cache(gen, B, Hkv, max_len, d)
    ours, eager = [t.cuda() for t in cache], [t.cuda() for t in cache]
    lengths, ws = torch.tensor([0, 100, 500]).cuda(), torch.empty(64 << 20, dtype=torch.uint8, device="cuda")

    def new():
        x = [normal(gen, B, T, Hq, d, scale=2.0), normal(gen, B, T, Hkv, d), normal(gen, B, T, Hkv, d), *rotary(gen, B, T, d)]
        return [t.cuda() for t in x]

    def step(x, n, cache, workspace):
        if T == 1:
            out = ops.decode_attention_rope_i4(*(y[:, 0] for y in x), n, *cache, workspace=workspace)
        else:
            out = ops.prefill_attention_i4(ops.rope_quantize_kv_cache_(*x, n, *cache), n, *cache, workspace=workspace)
        return (out, *ops.dequantize_kv_cache(*cache, n, T))

    x = new()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, lengths, [t.clone() for t in ours], ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, lengths, ours, ws)
    for n in ([0, 100, 500], [T, 100 + T, 500 + T], [820, -1, 64 - T if T < 64 else 3], [899, 831, 0]):
        for a, b in zip(x, new()):
            a.copy_(b)
        lengths.copy_(torch.tensor(n))
        graph.replay()
        want = step(x, lengths, eager, None)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), n
        for a, b in zip(ours, eager):
            assert torch.equal(a, b), n


def test_streams_have_workspaces_of_their_own(ops):
    """The same calls on two streams at once, each with its default workspace."""
    gen = torch.Generator().manual_seed(4)
    cases = [decode_case(gen, 4, 32, 8, 128, 3000, [2999, 2000, 10, 1500]) for _ in range(2)]
    dev = [[t.cuda() for t in c[:6]] + [t.cuda() for t in c[6]] for c in cases]
    alone = [ops.decode_attention_rope_i4(*d) for d in dev]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in dev]
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(ops.decode_attention_rope_i4(*dev[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in outs[i])


def test_offsets_beyond_32_bits(ops):
    """Codes of 4.6 GB each: the last sequence's rows lie behind 2^32 bytes."""
    B, Hkv, max_len, d = 9, 8, 1 << 20, 128
    free, _ = torch.cuda.mem_get_info()
    if free < 30 << 30:
        pytest.skip("not enough memory")
    big = [torch.zeros(B, Hkv, max_len, d // 2, dtype=torch.uint8, device="cuda"), torch.full((B, Hkv, max_len), float("nan"), device="cuda").half(),
           torch.zeros(B, Hkv, max_len, d // 2, dtype=torch.uint8, device="cuda"), torch.full((B, Hkv, max_len), float("nan"), device="cuda").half()]
    assert big[0].numel() > 1 << 32
    gen = torch.Generator().manual_seed(6)
    n = 300
    small = random_cache(gen, 1, Hkv, n, d)
    # the last sequence holds n slots; another's tokens go to its very last slots
    for a, b in zip(big, small):
        a[B - 1, :, :n] = b[0].cuda()
    lengths = torch.full((B,), -1, dtype=torch.int64)
    lengths[B - 1], lengths[B - 2] = n, max_len - 1
    q, k, v = normal(gen, B, 8, d, scale=2.0), normal(gen, B, Hkv, d), normal(gen, B, Hkv, d)
    cos, sin = rotary(gen, B, d)
    last = [t.cuda() for t in (q[B - 1:], k[B - 1:], v[B - 1:], cos[B - 1:], sin[B - 1:], torch.tensor([n]))]
    held = [torch.cat((t, torch.zeros_like(t[:, :, :64])), 2).cuda() for t in small]
    want = ops.decode_attention_rope_i4(*last, *held)
    lengths[B - 2] = -1
    out = ops.decode_attention_rope_i4(*(t.cuda() for t in (q, k, v, cos, sin, lengths)), *big)
    # (the same sums in another order: two roundings of the result)
    assert (out[B - 1].double() - want[0].double()).abs().max() <= 2.0 ** -10 * want.abs().max().item() and (out[:B - 1] == 0).all()
    for a, b in zip(big, held):
        assert torch.equal(a[B - 1, :, :n + 1], b[0, :, :n + 1])
    # a block behind it, and read back; the first row goes to the last slots of the sequence in front
    T = 40
    lengths = torch.full((B,), -1, dtype=torch.int64)
    lengths[B - 1], lengths[B - 2] = n + 1, max_len - T
    x = [normal(gen, B, T, 8, d, scale=2.0), normal(gen, B, T, Hkv, d), normal(gen, B, T, Hkv, d), *rotary(gen, B, T, d)]
    lengths = lengths.cuda()
    rotated = ops.rope_quantize_kv_cache_(*(t.cuda() for t in x), lengths, *big)
    (kc, ks), (vc, vs) = quantised(turned(x[1], x[3], x[4])), quantised(x[2].float())
    for b, at in ((B - 1, n + 1), (B - 2, max_len - T)):
        for a, new in zip(big, (packed(kc[b]), ks[b], packed(vc[b]), vs[b])):
            assert torch.equal(a[b, :, at:at + T].cpu(), new.transpose(0, 1))
    keys, values = ops.dequantize_kv_cache(*big, lengths, T)
    assert torch.equal(values[B - 2].cpu(), (quantised(x[2][B - 2].float())[0].float() * vs[B - 2].float()[..., None]).half().transpose(0, 1))
    lengths[B - 2] = -1
    got = ops.prefill_attention_i4(rotated, lengths, *big)
    cut = [a[B - 1:, :, :n + 1 + T].contiguous() for a in big]
    want = ops.prefill_attention_i4(rotated[B - 1:].contiguous(), torch.tensor([n + 1]).cuda(), *cut)
    assert (got[B - 1].double() - want[0].double()).abs().max() <= 2.0 ** -10 * want.abs().max().item() and (got[:B - 1] == 0).all()


def test_long_caches_of_few_sequences(ops):
    """The last tiles of caches that are much longer than the sequences, and blocks that are split over workgroups."""
    gen = torch.Generator().manual_seed(12)
    check_decode(ops, decode_case(gen, 2, 4, 1, 128, 50000, [40001, 3]))
    q, cache = prefill_case(gen, 1, 6, 4, 1, 64, 30000, [29000])
    check_prefill(ops, q, [29000], cache)


@pytest.mark.parametrize("change,match", [
    (dict(k_codes=lambda t: t.char()), "uint8"), (dict(k_scales=lambda t: t.float()), "float16"), (dict(v_codes=lambda t: t[:, :, :-1]), "contiguous|B, Hkv"),
    (dict(v_scales=lambda t: t[:, :1].contiguous()), "B, Hkv"), (dict(lengths=lambda t: t.int()), "int64"), (dict(lengths=lambda t: t[:1].contiguous()), "int64"),
    (dict(q=lambda t: t.bfloat16()), "float16"), (dict(cos=lambda t: t[:1].contiguous()), "cos"), (dict(k=lambda t: t[..., :64].contiguous()), "expected"),
    (dict(q=lambda t: t[..., :3, :].contiguous()), "multiple")])
def test_refusals(ops, change, match):
    gen = torch.Generator().manual_seed(2)
    q, k, v, cos, sin, lengths, cache = decode_case(gen, 2, 4, 2, 128, 64, [5, 6])
    args = dict(zip(("q", "k", "v", "cos", "sin", "lengths", "k_codes", "k_scales", "v_codes", "v_scales"), [t.cuda() for t in (q, k, v, cos, sin, lengths, *cache)]))
    before = [args[n].clone() for n in ("k_codes", "k_scales", "v_codes", "v_scales")]
    for name, f in change.items():
        args[name] = f(args[name])
    with pytest.raises(RuntimeError, match=match):
        ops.decode_attention_rope_i4(*args.values())
    if set(change) & {"k_codes", "k_scales", "v_codes", "v_scales", "lengths"}:
        with pytest.raises(RuntimeError, match=match):
            ops.prefill_attention_i4(args["q"][:, None].contiguous(), args["lengths"], *list(args.values())[6:])
        with pytest.raises(RuntimeError, match=match):
            ops.dequantize_kv_cache(*list(args.values())[6:], args["lengths"], 3)
        with pytest.raises(RuntimeError, match=match):
            ops.rope_quantize_kv_cache_(*(args[n][:, None].contiguous() for n in ("q", "k", "v", "cos", "sin")), args["lengths"], *list(args.values())[6:])
    if "k_codes" not in change:
        assert torch.equal(args["k_codes"], before[0])

"""Attention over caches in 4 bits where the calls take other ways than at small sizes and magnitudes: blocks whose waves have rows of their own, ragged
batches whose long sequences are shared by many workgroups, scores and values that grow along the cache, and scales out of a query's sight that are
larger than those in it.  Tolerances are those of the operators' other tests; what each query sees is evaluated by itself where what it does not see
must not count."""
import pytest
import torch

from test_gpu_cache_i4 import attend64, check_decode, check_prefill, close, decode_case, hadamard64, normal, prefill_case, random_cache, turned, unpacked

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["default", "ctypes"])
def ops(request):
    if request.param == "ctypes":
        from flh_amd import _ops
        return _ops
    import flh_amd
    return flh_amd._CUDA


@pytest.mark.parametrize("B,T,Hq,Hkv,d,max_len,lengths", [
    (64, 65, 32, 32, 128, 200, [(i * 31) % 136 - 1 for i in range(64)]),         # three blocks of rows, a fourth wave without; the first takes no part
    (20, 70, 96, 32, 64, 333, [(i * 71) % 270 - 3 for i in range(20)]),          # three queries per head: blocks that end inside a token
    (130, 1, 32, 32, 128, 70, [i % 71 for i in range(130)]),                     # a single row in each; one token past the end takes no part
    (4, 1100, 32, 32, 64, 1200, [0, 63, 100, 101])])
def test_waves_with_rows_of_their_own(ops, B, T, Hq, Hkv, d, max_len, lengths):
    assert B * Hkv * -(-T * (Hq // Hkv) // 32) >= 4096
    gen = torch.Generator().manual_seed(T + B)
    q, cache = prefill_case(gen, B, T, Hq, Hkv, d, max_len, lengths)
    check_prefill(ops, q, lengths, cache)


@pytest.mark.parametrize("B,T,Hq,Hkv,d,max_len,lengths", [
    (20, 65, 32, 32, 128, 300, [(i * 31) % 237 - 1 for i in range(20)]),         # three blocks of rows: two waves without; one takes no part
    (13, 33, 40, 40, 128, 200, [(i * 47) % 169 for i in range(13)]),             # pairs that are no multiple of eight
    (37, 17, 28, 28, 128, 100, [(i * 13) % 90 - 2 for i in range(37)]),          # one block: a pair of waves without, in every workgroup
    (33, 10, 160, 32, 64, 150, [(i * 29) % 141 for i in range(33)]),             # five queries per head
    (10, 65, 96, 32, 64, 333, [(i * 71) % 270 - 3 for i in range(10)])])
def test_waves_in_pairs(ops, B, T, Hq, Hkv, d, max_len, lengths):
    blocks = B * Hkv * -(-T * (Hq // Hkv) // 32)
    assert 1024 * (128 // d) <= blocks < 2048 * (128 // d)
    gen = torch.Generator().manual_seed(T + B)
    q, cache = prefill_case(gen, B, T, Hq, Hkv, d, max_len, lengths)
    check_prefill(ops, q, lengths, cache)


@pytest.mark.parametrize("B,H,d", [(70, 32, 64), (70, 32, 128), (35, 32, 64), (17, 32, 128), (20, 6, 128)])
def test_waves_with_rows_of_their_own_non_finite(ops, B, H, d):
    gen = torch.Generator().manual_seed(7)
    T, n = 33, 50
    q, cache = prefill_case(gen, B, T, H, H, d, 100, [n] * B)
    cache[1][3, 5, n + 20] = float("nan")                              # a key that the queries from the twentieth on see, in one head
    cache[3][9, 0, n + 4] = float("inf")                               # a value
    q[11, 30, 2, 7] = float("nan")
    out = ops.prefill_attention_i4(q.cuda(), torch.tensor([n] * B).cuda(), *(t.cuda() for t in cache)).cpu().view(B, T, H, d)
    finite = torch.isfinite(out).all(-1)
    want = torch.ones(B, T, H, dtype=torch.bool)
    want[3, 20:, 5] = want[9, 4:, 0] = want[11, 30, 2] = False
    held = torch.where(unpacked(cache[2][9, 0, n + 4]) == 0)[0]        # (a code of zero times an infinite scale is NaN as well)
    assert held.numel() < d and torch.equal(finite, want)


@pytest.mark.parametrize("B,T,Hq,Hkv,d,max_len,lengths", [
    (4, 5, 32, 8, 128, 9000, [8990, 100, 0, 640]),                     # one sequence has most of the tiles
    (4, 5, 32, 8, 128, 9000, [100, -1, 8990, 9000]),                   # .. and some take no part
    (3, 40, 12, 4, 64, 5000, [64, 4960, 2000]),                        # several blocks of rows share a sequence's parts
    (150, 1, 2, 1, 128, 3000, [2999 if i in (0, 63, 64, 149) else (i * 7) % 300 - 2 for i in range(150)]),   # more sequences than lanes
    (256, 1, 4, 1, 64, 2000, [1999 if i == 200 else i for i in range(256)])])    # the most that are shared
def test_ragged_parts(ops, B, T, Hq, Hkv, d, max_len, lengths):
    gen = torch.Generator().manual_seed(T + B)
    q, cache = prefill_case(gen, B, T, Hq, Hkv, d, max_len, lengths)
    out = check_prefill(ops, q, lengths, cache)
    ws = torch.full((64 << 20,), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(out, ops.prefill_attention_i4(q.cuda(), torch.tensor(lengths).cuda(), *(t.cuda() for t in cache), workspace=ws))


def test_parts_on_two_streams(ops):
    """Calls whose parts are joined by a second launch, on two streams at once, each with its default workspace."""
    gen = torch.Generator().manual_seed(4)
    cases = [prefill_case(gen, 3, 9, 32, 8, 128, 3000, lengths) for lengths in ([2990, 100, 1500], [700, 2991, 0])]
    dev = [(q.cuda(), torch.tensor(n).cuda(), *(t.cuda() for t in cache)) for (q, cache), n in zip(cases, ([2990, 100, 1500], [700, 2991, 0]))]
    alone = [ops.prefill_attention_i4(*d) for d in dev]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in dev]
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(ops.prefill_attention_i4(*dev[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in outs[i])


def growing(cache, n, keys, values):
    """Scales that change by 2^keys and 2^values over the first n slots."""
    at = torch.arange(n) / max(n - 1, 1)
    cache[1][:, :, :n] = (0.01 * torch.exp2(keys * at if keys > 0 else -keys * (1 - at))).half()
    cache[3][:, :, :n] = (2.0 ** -12 * torch.exp2(values * at if values > 0 else -values * (1 - at))).half()


@pytest.mark.parametrize("keys,values", [(7, 0), (-7, 0), (0, 26), (0, -26), (6, 24), (6, -24), (-6, 24)])
@pytest.mark.parametrize("B,T,Hq,Hkv,n", [(1, 9, 8, 2, 900), (2, 70, 8, 4, 400), (70, 33, 32, 32, 300)])
def test_blocks_of_growing_scales(ops, B, T, Hq, Hkv, n, keys, values):
    """References that are raised on the way, and ones that the first tile sets above all others."""
    gen = torch.Generator().manual_seed(n)
    cache = random_cache(gen, B, Hkv, n + T, 128)
    growing(cache, n + T, keys, values)
    q = normal(gen, B, T, Hq, 128, scale=2.0)
    if B > 8:                                                          # (the others are for the number of rows; evaluated for one)
        lengths = [-1] * B
        lengths[5] = n
    else:
        lengths = [n - 3 * b for b in range(B)]
    check_prefill(ops, q, lengths, cache)


@pytest.mark.parametrize("keys,values", [(7, 0), (-7, 0), (0, 26), (0, -26), (6, 24), (6, -24), (-6, 24)])
@pytest.mark.parametrize("B,Hq,Hkv,d,n", [(1, 8, 2, 128, 900), (2, 40, 2, 64, 1400), (70, 8, 4, 128, 200)])
def test_tokens_of_growing_scales(ops, B, Hq, Hkv, d, n, keys, values):
    gen = torch.Generator().manual_seed(n)
    case = decode_case(gen, B, Hq, Hkv, d, n + 1, [n - b for b in range(B)])
    growing(case[6], n + 1, keys, values)
    check_decode(ops, case)


class Negated:
    """The operators on caches whose values' scales have the other sign, and their outputs with the other sign.  Everything the tolerance counts is the
    same size for either sign (the bits differ: the matrix instruction does not round both sides of zero alike)."""

    def __init__(self, ops):
        self.ops = ops

    def prefill_attention_i4(self, q, lengths, kc, ks, vc, vs):
        return -self.ops.prefill_attention_i4(q, lengths, kc, ks, vc, -vs)

    def decode_attention_rope_i4(self, *x):
        vs = -x[9]
        out = self.ops.decode_attention_rope_i4(*x[:9], vs)
        x[9].copy_(vs.abs())                                           # (the new token's scale is positive)
        return -out


@pytest.mark.parametrize("values", [26, -26])
def test_scales_of_either_sign(ops, values):
    """Values whose scales are negative, large enough that weights leave fp16's range on the way."""
    gen = torch.Generator().manual_seed(12)
    B, T, Hq, Hkv, n, d = 2, 20, 8, 2, 700, 128
    cache = random_cache(gen, B, Hkv, n + T, d)
    growing(cache, n + T, 0, values)
    q, lengths = normal(gen, B, T, Hq, d, scale=2.0), [n, n - 40]
    check_prefill(Negated(ops), q, lengths, cache)
    case = decode_case(gen, B, Hq, Hkv, d, n + T, lengths)
    case[2].zero_()                                                    # (the new token's value would count with the other sign)
    check_decode(Negated(ops), (*case[:6], cache))


@pytest.mark.parametrize("big", [60000.0, float("inf"), float("nan")])
@pytest.mark.parametrize("B,T,Hq,Hkv", [(1, 30, 8, 2), (70, 33, 32, 32)])
def test_scales_out_of_sight(ops, B, T, Hq, Hkv, big):
    """Values of 2^-9 in sight, the largest there are behind them in the same tile: every query has the precision of what it sees."""
    gen = torch.Generator().manual_seed(T)
    n, d, rep = 64, 128, Hq // Hkv
    cache = random_cache(gen, B, Hkv, n + T, d)
    cache[3][:, :, :n + 20] = 2.0 ** -10
    cache[3][:, :, n + 20:] = big
    cache[1][:, :, n + 20:] = big if big != big else 60000.0
    q = normal(gen, B, T, Hq, d)
    got = ops.prefill_attention_i4(q.cuda(), torch.full((B,), n).cuda(), *(t.cuda() for t in cache)).cpu().view(B, T, Hq, d)
    for t in (0, 7, 19):
        for g in range(Hkv):
            m = n + t + 1
            x, tol = attend64(q[0, t, g * rep:(g + 1) * rep], unpacked(cache[0][0, g, :m]), cache[1][0, g, :m], unpacked(cache[2][0, g, :m]),
                              cache[3][0, g, :m], [m] * rep, d ** -0.5)
            close(got[0, t, g * rep:(g + 1) * rep], x, tol, (t, g))


def check_huge(got, q, kc, ks, vc, vs, scale):
    """One query's output where scores are so large that their rounding decides between keys next to the largest: a mean of values, and the value of the
    key with the largest score where that one is out of all others' reach."""
    v = vc.double() * vs.double()[:, None]
    s = (kc.double() @ q.double()) * ks.double() * scale
    bound = (4 * q.numel() + 32) * 2.0 ** -24 * scale * ((kc.double().abs() + 8) @ q.double().abs() * ks.double()).max() + 60
    first, second = torch.topk(s, 2).values
    assert torch.isfinite(got).all() and (got.double().abs() <= v.abs().max() * 1.01).all()
    if first - second > 2 * bound:                                     # (every other key's probability is below 2^-60)
        x = v[s.argmax()]
        assert ((got.double() - x).abs() <= 4 * 2.0 ** -11 * x.abs() + 40 * 2.0 ** -18 * vs[s.argmax()].double()).all()
        return 1
    return 0


@pytest.mark.parametrize("qscale,key,scale", [(100.0, 1.0, 1e3), (1e4, 100.0, 1.0), (1e4, 1e4, 1.0), (1e4, 1e4, 1e9)])
def test_huge_scores(ops, qscale, key, scale):
    gen = torch.Generator().manual_seed(3)
    T, Hq, Hkv, d, n = 9, 8, 2, 128, 900
    cache = random_cache(gen, 1, Hkv, n + T, d)
    cache[1].mul_(key)
    q = normal(gen, 1, T, Hq, d, scale=qscale)
    dev = [t.cuda() for t in cache]
    got = ops.prefill_attention_i4(q.cuda(), torch.tensor([n]).cuda(), *dev, scale=scale).cpu().view(T, Hq, d)
    sure = 0
    for t in range(T):
        for h in range(Hq):
            g, m = h // (Hq // Hkv), n + t + 1
            sure += check_huge(got[t, h], q[0, t, h], unpacked(cache[0][0, g, :m]), cache[1][0, g, :m], unpacked(cache[2][0, g, :m]), cache[3][0, g, :m], scale)
    assert sure > T * Hq // 2
    one, zero = torch.ones(1, d).half(), torch.zeros(1, d).half()      # no turn; the queries' rotation is undone in front
    x = (q[:, 0].double() @ hadamard64(d)).half()
    kn, vn = normal(gen, 1, Hkv, d), normal(gen, 1, Hkv, d)
    got = ops.decode_attention_rope_i4(*(t.cuda() for t in (x, kn, vn, one, zero, torch.tensor([n]))), *dev, scale=scale).cpu()
    cache = [t.cpu() for t in dev]
    y = turned(x, one, zero, torch.float64)
    sure = 0
    for h in range(Hq):
        g, m = h // (Hq // Hkv), n + 1
        sure += check_huge(got[0, h], y[0, h], unpacked(cache[0][0, g, :m]), cache[1][0, g, :m], unpacked(cache[2][0, g, :m]), cache[3][0, g, :m], scale)
    assert sure > Hq // 2

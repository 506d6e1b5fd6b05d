"""The operators on caches with lengths of their own -- attention of drafted trees, their commit, attention weights, eviction --
against plain float64 evaluations, at the sizes and masks where they can go wrong.

Tolerances count roundings (half a step of fp16 is 2^-11, of float32 2^-24, relative).  Attention output: the result and the
probabilities are rounded to fp16, and with the rotary embedding inside the query too, which moves a score by at most
scale * sum |q| |k| * 2^-11 and with it a probability by twice that (numerator and sum); probabilities below the smallest normal fp16
are off by 2^-25 of the largest one each.  Weights: the same with float32 steps, d of them in a score."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

H16, H32 = 2.0 ** -11, 2.0 ** -24


@pytest.fixture(params=["default", "ctypes"])
def ops(request):
    """Both routes to the library."""
    if request.param == "ctypes":
        from flh_amd import _ops
        return _ops
    import flh_amd
    return flh_amd._CUDA


def normal(gen, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).half()


def rotate64(x, cos, sin):
    """x [B, T, H, d], cos / sin [B, T, d] -> float64"""
    x, c, s = x.double(), cos.double()[:, :, None], sin.double()[:, :, None]
    half = x.size(-1) // 2
    return x * c + torch.cat((-x[..., half:], x[..., :half]), -1) * s


def attend64(q, k, v, seen, scale):
    """q [R, d], k / v [n, d] float64, seen [R, n] -> (out, probabilities, largest sum |q| |k| * scale)"""
    k, v = torch.where(seen.any(0)[:, None], k, 0.0), torch.where(seen.any(0)[:, None], v, 0.0)
    s = torch.where(seen, (q @ k.t()) * scale, -torch.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = torch.where(total > 0, e / total, 0.0)
    size = (torch.where(seen, (q.abs() @ k.abs().t()) * scale, 0.0)).max().item() if seen.numel() else 0.0
    return p @ v, p, size


def random_mask(gen, kind, B, T):
    """bool [T, T] or [B, T, T]: ancestors of random trees, a chain, or anything (rows without a node among it)."""
    def one():
        if kind == "chain":
            return torch.ones(T, T, dtype=torch.bool).tril()
        if kind == "random":
            m = torch.rand(T, T, generator=gen) < 0.4
            m[:: 3] = False
            return m
        m = torch.eye(T, dtype=torch.bool)
        for i in range(1, T):
            m[i] |= m[int(torch.randint(0, i, (1,), generator=gen))]
        return m
    if kind.endswith("each"):
        return torch.stack([one() for _ in range(B)])
    return one()


def tree_case(gen, B, T, Hq, Hkv, d, lengths, max_len, kind, qscale=1.0):
    q, k, v = normal(gen, B, T, Hq, d, scale=qscale), normal(gen, B, T, Hkv, d), normal(gen, B, T, Hkv, d)
    angle = torch.rand(B, T, d // 2, generator=gen, dtype=torch.float64) * 6.28
    angle = torch.cat((angle, angle), -1)
    mask = random_mask(gen, kind, B, T)
    kc, vc = normal(gen, B, Hkv, max_len, d), normal(gen, B, Hkv, max_len, d)
    for b, n in enumerate(lengths):                                    # what lies behind a sequence is not looked at
        n = min(n, max_len)
        kc[b, :, max(n, 0):] = float("nan")
        vc[b, :, max(n, 0):] = float("inf") if b % 2 else float("nan")
    return q, k, v, angle.cos().half(), angle.sin().half(), torch.tensor(lengths), mask, kc, vc


def tree_oracle(case, scale=None):
    """(out [B, T, Hq, d], tolerance, caches)"""
    q, k, v, cos, sin, lengths, mask, kc, vc = case
    B, T, Hq, d = q.shape
    Hkv, max_len = kc.size(1), kc.size(2)
    scale = d ** -0.5 if scale is None else scale
    kc, vc = kc.clone(), vc.clone()
    qr, kr = rotate64(q, cos, sin), rotate64(k, cos, sin).half()
    out = torch.zeros(B, T, Hq, d, dtype=torch.float64)
    tol = torch.zeros(B, 1, Hq, 1, dtype=torch.float64)
    for b, n in enumerate(lengths.tolist()):
        if n < 0 or n + T > max_len:
            continue
        kc[b, :, n:n + T], vc[b, :, n:n + T] = kr[b].transpose(0, 1), v[b].transpose(0, 1)
        seen = torch.cat((torch.ones(T, n, dtype=torch.bool), mask[b] if mask.dim() == 3 else mask), 1)
        for h in range(Hq):
            g = h // (Hq // Hkv)
            out[b, :, h], _, size = attend64(qr[b, :, h], kc[b, g, :n + T].double(), vc[b, g, :n + T].double(), seen, scale)
            top = vc[b, g, :n + T].double().abs().max().item()
            # result, probabilities, the query's rounding (and float32's, far below), small probabilities
            tol[b, 0, h, 0] = top * (H16 + H16 + 2 * size * H16 + (n + T) * 2.0 ** -25 + 1e-5)
    return out, tol, kc, vc


def equal_bits(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.int16), b.cpu().contiguous().view(torch.int16))


def near_keys(got, ref):
    """Cached keys: float32's rotation against float64's may round to the other neighbour where it lies on a border."""
    same = got.cpu().view(torch.int16) == ref.view(torch.int16)
    g, r = got.cpu().double(), ref.double()
    step = torch.maximum(r.abs(), torch.tensor(2.0 ** -14, dtype=torch.float64)) * 2 * H16
    assert torch.isfinite(g[~same]).all() and ((g - r).abs()[~same] <= 1.001 * step[~same]).all()
    assert (~same).sum().item() <= 1 + 2e-3 * same.numel()


def run_tree(ops, case, **more):
    dev = [t.cuda() for t in case]
    before = [t.clone() for t in dev[:7]]
    out = ops.tree_attention(*dev, **more)
    torch.cuda.synchronize()
    for a, b in zip(dev[:7], before):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    return out, dev[7], dev[8]


def check_tree(ops, case, **more):
    out, kc, vc = run_tree(ops, case, **more)
    ref, tol, rk, rv = tree_oracle(case, more.get("scale"))
    B, T, Hq, d = case[0].shape
    got = out.cpu().double().view(B, T, Hq, d)
    assert torch.isfinite(got).all()
    worst = ((got - ref).abs() - tol).max().item()
    assert worst <= 0, worst
    norm = ref.norm().item()
    if norm:
        assert (got - ref).norm().item() <= 4 * H16 * norm
    near_keys(kc, rk)
    assert equal_bits(vc, rv)
    return out, kc, vc


TREES = [
    # B, T, Hq, Hkv, d, lengths, max_len, mask
    (1, 1, 8, 8, 128, [0], 64, "chain"),                               # nothing but the node itself
    (1, 1, 32, 8, 128, [63], 64, "chain"),                             # the cache filled to its last slot
    (1, 8, 32, 8, 128, [120], 256, "tree"),
    (3, 7, 8, 2, 128, [64, 1, 129], 300, "tree-each"),
    (2, 26, 8, 8, 128, [500, 333], 640, "tree"),
    (2, 33, 4, 4, 64, [0, 65], 128, "random"),                         # rows that see nothing at all
    (2, 63, 16, 4, 64, [1000, 777], 1063, "tree-each"),
    (4, 5, 12, 4, 64, [-1, 100, 124, 123], 128, "tree"),               # no sequence, and one whose tree does not fit
    (4, 3, 4, 2, 128, [2 ** 63 - 1, -2 ** 63, 7, 2 ** 32 + 5], 64, "tree"),
    (1, 64, 32, 4, 128, [2049], 2200, "tree"),
    (1, 256, 2, 1, 128, [70], 400, "random-each"),
    (2, 100, 3, 1, 64, [31, 32], 200, "tree"),
    (5, 17, 16, 1, 128, [15, 16, 17, 0, 255], 300, "random-each"),
    (70, 3, 2, 1, 64, [i % 20 for i in range(70)], 32, "tree"),       # more sequences than lanes of a wave
    (1, 2, 64, 1, 128, [4097], 4100, "chain"),
]


@pytest.mark.parametrize("B,T,Hq,Hkv,d,lengths,max_len,kind", TREES, ids=lambda v: str(v) if not isinstance(v, list) else f"n{v[0]}")
def test_tree_attention(ops, B, T, Hq, Hkv, d, lengths, max_len, kind):
    gen = torch.Generator().manual_seed(B * 1000 + T)
    print(f"case tree B={B} T={T} Hq={Hq} Hkv={Hkv} d={d} max={max_len} {kind}", flush=True)
    check_tree(ops, tree_case(gen, B, T, Hq, Hkv, d, lengths, max_len, kind))


def test_tree_attention_workspace_scale_and_peaks(ops):
    from flh_amd import _lib
    gen = torch.Generator().manual_seed(1)
    B, T, Hq, Hkv, d = 2, 9, 8, 2, 128
    case = tree_case(gen, B, T, Hq, Hkv, d, [300, 211], 512, "tree", qscale=8.0)      # one slot has most of the weight
    need = _lib.load().flh_tree_attention_workspace_bytes(B, T, Hq, Hkv, d)
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
    a, _, _ = check_tree(ops, case, workspace=ws)
    b, _, _ = run_tree(ops, case)
    assert torch.equal(a, b)                                           # the same bits whatever the workspace held
    check_tree(ops, case, scale=0.01)
    flat = (case[0] * 0, *case[1:])
    check_tree(ops, flat)


@pytest.mark.parametrize("T,Hq,Hkv,d", [(9, 4, 2, 128), (40, 4, 1, 64), (70, 2, 1, 128), (20, 2, 1, 128), (200, 1, 1, 64), (219, 1, 1, 128)])
def test_tree_values_that_some_queries_do_not_see(ops, T, Hq, Hkv, d):
    """Keys and values of the tree that are infinite or NaN reach the queries that see them, and no others."""
    gen = torch.Generator().manual_seed(T)
    case = list(tree_case(gen, 1, T, Hq, Hkv, d, [37], 256, "tree"))
    mask = case[6]
    odd = [T - 1, T // 2, T // 3]
    ref_case = [t.clone() for t in case]
    case[1][0, odd[0]] = float("nan")                                  # a key
    case[2][0, odd[1], :, 3] = float("inf")                            # one channel of the values
    case[2][0, odd[2], :, d - 5] = float("nan")
    ref_case[6][:, odd[0]] = False                                     # (queries that see the key are not compared)
    out, _, vc = run_tree(ops, case)
    got = out.cpu().double().view(1, T, Hq, d)
    ref, tol, _, _ = tree_oracle(ref_case)
    for t in range(T):
        if mask[t, odd[0]]:
            assert torch.isnan(got[0, t]).all()
            continue
        skip = [c for j, c in ((odd[1], 3), (odd[2], d - 5)) if mask[t, j]]
        for j, c in ((odd[1], 3), (odd[2], d - 5)):
            if mask[t, j]:
                assert not torch.isfinite(got[0, t, :, c]).any()
        rest = [c for c in range(d) if c not in skip]
        assert ((got[0, t] - ref[0, t]).abs() <= tol[0, 0])[:, rest].all()
    assert torch.isinf(vc[0, :, 37 + odd[1], 3]).all() and torch.isnan(vc[0, :, 37 + odd[2], d - 5]).all()


def test_tree_attention_zero_sizes(ops):
    z = lambda *s, dtype=torch.float16: torch.zeros(*s, dtype=dtype, device="cuda")
    for B, T in ((0, 4), (2, 0)):
        out = ops.tree_attention(z(B, T, 8, 128), z(B, T, 2, 128), z(B, T, 2, 128), z(B, T, 128), z(B, T, 128),
                                 z(B, dtype=torch.int64), z(T, T, dtype=torch.bool), z(B, 2, 64, 128), z(B, 2, 64, 128))
        assert tuple(out.shape) == (B, T, 8 * 128)


def test_tree_of_one_node_is_a_decode_step(ops):
    """A chain of one node against the decode step's operator, whose rotation rounds three times."""
    gen = torch.Generator().manual_seed(2)
    B, Hq, Hkv, d, n = 2, 32, 8, 128, 200
    case = tree_case(gen, B, 1, Hq, Hkv, d, [n] * B, 256, "chain")
    case = (*case[:3], case[3][:1].expand(B, 1, d).contiguous(), case[4][:1].expand(B, 1, d).contiguous(), *case[5:])
    out, kc, vc = run_tree(ops, case)
    dev = [t.cuda() for t in case]
    import flh_amd
    ref = flh_amd._CUDA.decode_attention_rope(dev[0][:, 0], dev[1][:, 0], dev[2][:, 0], dev[3][0, 0], dev[4][0, 0],
                                              torch.tensor([n], device="cuda"), dev[7], dev[8], n + 1)
    assert (out.view(B, Hq, d).float() - ref.float()).norm() <= 8 * H16 * ref.float().norm()
    assert equal_bits(vc, dev[8])


def test_tree_attention_in_a_graph_serves_every_length(ops):
    from flh_amd import _lib
    gen = torch.Generator().manual_seed(3)
    B, T, Hq, Hkv, d, max_len = 3, 12, 8, 2, 128, 700
    ws = torch.empty(_lib.load().flh_tree_attention_workspace_bytes(B, T, Hq, Hkv, d), dtype=torch.uint8, device="cuda")
    dev = [t.cuda() for t in tree_case(gen, B, T, Hq, Hkv, d, [1, 1, 1], max_len, "tree")]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.tree_attention(*dev, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.tree_attention(*dev, workspace=ws)
    for lengths in ([5, 300, 688], [0, -1, 64], [688, 689, 128], [77, 200, 511]):
        case = tree_case(gen, B, T, Hq, Hkv, d, lengths, max_len, "tree")
        for to, x in zip(dev, case):
            to.copy_(x)
        torch.zeros(1000, device="cuda").add_(1)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        for to, x in zip(dev[7:], case[7:]):
            to.copy_(x)
        eager = ops.tree_attention(*dev, workspace=ws.clone())
        assert torch.equal(got, eager), lengths
        ref, tol, _, _ = tree_oracle(case)
        assert ((got.cpu().double().view(ref.shape) - ref).abs() <= tol).all()


def test_operators_follow_the_current_stream(ops):
    """Inputs made on a side stream behind a long kernel, the operator there too."""
    gen = torch.Generator().manual_seed(4)
    case = tree_case(gen, 1, 8, 8, 2, 128, [150], 256, "tree")
    dev = [t.cuda() for t in case]
    ref, kc, vc = run_tree(ops, case)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(8):
            big = big @ big * 1e-3
        late = [t.clone() for t in dev]
        out = ops.tree_attention(*late)
    stream.synchronize()
    assert torch.equal(out, ref) and equal_bits(late[7], kc)


# ---------------------------------------------------------------------------------------------------- commit
def commit_oracle(tokens, parents, chosen, lengths, caches, max_len):
    B, T = tokens.shape
    path = np.full((B, T), -1)
    accepted, following, new = np.zeros(B, int), np.full(B, -1), np.array(lengths)
    caches = [c.clone() for c in caches]
    for b in range(B):
        if lengths[b] < 0 or lengths[b] + T > max_len:
            continue
        par = parents[b] if parents.ndim == 2 else parents
        p = [0]
        while True:
            c = [i for i in range(p[-1] + 1, T) if par[i] == p[-1] and tokens[b, i] == chosen[b, p[-1]]]
            if not c:
                break
            p.append(c[0])
        path[b, :len(p)], accepted[b], following[b], new[b] = p, len(p), chosen[b, p[-1]], lengths[b] + len(p)
        for cache in caches:
            cache[b, :, lengths[b]:lengths[b] + len(p)] = cache[b][:, [lengths[b] + i for i in p]].clone()
    return path, accepted, following, new, caches


@pytest.mark.parametrize("B,T,layers,Hkv,d,max_len,per_sequence", [(1, 1, 2, 2, 128, 16, True), (3, 8, 2, 2, 128, 40, True),
                                                                  (4, 64, 1, 1, 64, 128, False), (2, 256, 2, 2, 128, 300, True),
                                                                  (2, 65, 130, 1, 8, 70, False), (5, 30, 3, 3, 24, 64, True)])
def test_tree_commit(ops, B, T, layers, Hkv, d, max_len, per_sequence):
    rng = np.random.default_rng(T)
    gen = torch.Generator().manual_seed(T)
    # chains and bushes; few different tokens, so that siblings share them
    parents = np.stack([[-1] + [int(rng.integers(max(0, i - 3), i)) for i in range(1, T)] for _ in range(B)])
    parents = parents if per_sequence else parents[0]
    tokens, chosen = rng.integers(0, 2, (B, T)), rng.integers(0, 2, (B, T))
    lengths = [int(x) for x in rng.integers(0, max_len - T + 1, B)]
    if B > 2:
        lengths[1], lengths[2] = -1, max_len - T + 1
    if B > 3:
        lengths[3] = 2 ** 63 - 1
    caches = [normal(gen, B, Hkv, max_len, d) for _ in range(2 * layers)]
    path, accepted, following, new, ref = commit_oracle(tokens, parents, chosen, lengths, caches, max_len)
    dev = [torch.from_numpy(x).cuda() for x in (tokens, parents, chosen)]
    on_gpu = [c.cuda() for c in caches]
    got = ops.tree_commit_(*dev, torch.tensor(lengths).cuda(), on_gpu[:layers], on_gpu[layers:])
    for g, r in zip(got, (path, accepted, following, new)):
        assert g.dtype == torch.int64 and np.array_equal(g.cpu().numpy(), r)
    for g, r in zip(on_gpu, ref):
        assert equal_bits(g, r)


def test_tree_commit_with_parents_that_are_none(ops):
    """Parents that are not a lower index are nobody's; a chain of 256 nodes is accepted whole."""
    B, T, max_len = 2, 256, 256
    parents = torch.arange(-1, T - 1).expand(B, T).clone()
    tokens = torch.arange(T).expand(B, T).clone()
    chosen = torch.arange(1, T + 1).expand(B, T).clone()
    parents[1, 5:] = torch.tensor([5, 9, -7, 2 ** 40, 4] + [300] * (T - 10))
    gen = torch.Generator().manual_seed(0)
    caches = [normal(gen, B, 1, max_len, 128) for _ in range(2)]
    path, accepted, following, new, ref = commit_oracle(tokens.numpy(), parents.numpy(), chosen.numpy(), [0, 0], caches, max_len)
    dev = [c.cuda() for c in caches]
    got = ops.tree_commit_(tokens.cuda(), parents.cuda(), chosen.cuda(), torch.zeros(B, dtype=torch.int64).cuda(), *dev)
    assert accepted.tolist() == [256, 5]
    for g, r in zip(got, (path, accepted, following, new)):
        assert np.array_equal(g.cpu().numpy(), r)
    for g, r in zip(dev, ref):
        assert equal_bits(g, r)


# ---------------------------------------------------------------------------------------------------- attention weights
def weights_tolerance(size, d, n, rows, added, total):
    """float32: d steps in a score, its scaling and the exponential's argument, sums over n slots and `rows` queries."""
    return (2 * (d + 4) * H32 * size + (n + rows + 16) * H32) * added + rows * H32 * total + 1e-30


@pytest.mark.parametrize("B,Hq,Hkv,d,lengths,max_len", [(1, 32, 8, 128, [2048], 2048), (3, 8, 8, 128, [1, 64, 65], 100),
                                                        (4, 16, 4, 64, [0, 777, -3, 1001], 1000), (3, 4, 2, 128, [2 ** 63 - 1, 30, 2 ** 32 + 1], 64), (2, 12, 4, 64, [333, 31], 400),
                                                        (5, 64, 2, 128, [129, 500, 2, 1023, 1024], 1024), (1, 3, 1, 128, [4500], 4501),
                                                        (66, 2, 2, 64, [i for i in range(66)], 70), (1, 128, 1, 128, [300], 320),
                                                        (2, 320, 1, 64, [70, 33], 80)])
def test_decode_attention_weights(ops, B, Hq, Hkv, d, lengths, max_len):
    gen = torch.Generator().manual_seed(B + Hq)
    print(f"case decode weights B={B} Hq={Hq} Hkv={Hkv} d={d} max={max_len}", flush=True)
    q = normal(gen, B, Hq, d, scale=2.0)
    kc, vc = normal(gen, B, Hkv, max_len, d), normal(gen, B, Hkv, max_len, d)
    for b, n in enumerate(lengths):
        kc[b, :, max(min(n, max_len), 0):], vc[b, :, max(min(n, max_len), 0):] = float("nan"), float("inf")
    weights = torch.rand(B, Hkv, max_len, generator=gen)
    args = [q.cuda(), kc.cuda(), vc.cuda(), torch.tensor(lengths).cuda()]
    dev = weights.cuda()
    out = ops.decode_attention_weights(*args, dev)
    again = weights.cuda()
    assert torch.equal(ops.decode_attention_weights(*args, again), out) and torch.equal(again, dev)   # a fixed order
    got, gw = out.cpu().double(), dev.cpu().double()
    for b, n in enumerate(lengths):
        if not 0 < n <= max_len:
            assert (got[b] == 0).all() and torch.equal(dev[b].cpu(), weights[b])
            continue
        assert torch.equal(dev[b, :, n:].cpu(), weights[b, :, n:])
        for g in range(Hkv):
            rows = slice(g * Hq // Hkv, (g + 1) * Hq // Hkv)
            k, v = kc[b, g, :n].double(), vc[b, g, :n].double()
            ref, p, size = attend64(q[b, rows].double(), k, v, torch.ones(Hq // Hkv, n, dtype=torch.bool), d ** -0.5)
            assert ((got[b, rows] - ref).abs() <= v.abs().max() * (2 * H16 + n * 2.0 ** -25 + 1e-5)).all()
            added = p.sum(0)
            total = weights[b, g, :n].double() + added
            assert ((gw[b, g, :n] - total).abs() <= weights_tolerance(size, d, n, Hq // Hkv, added, total)).all()


@pytest.mark.parametrize("B,T,Hq,Hkv,past,max_len", [(1, 300, 8, 8, 77, 400), (2, 129, 8, 2, 0, 129), (1, 1, 4, 1, 0, 64), (1, 1, 4, 4, 63, 64),
                                                     (1, 513, 4, 1, 100, 700), (3, 40, 12, 4, 500, 600), (1, 1000, 2, 1, 0, 1000),
                                                     (1, 64, 32, 2, 64, 128), (1, 7, 6, 1, 2000, 2100)])
def test_prefill_attention_weights(ops, B, T, Hq, Hkv, past, max_len):
    import flh_amd
    d = 128
    gen = torch.Generator().manual_seed(T + past)
    print(f"case prefill weights B={B} T={T} Hq={Hq} Hkv={Hkv} past={past}", flush=True)
    q = normal(gen, B, T, Hq, d, scale=2.0)
    kc, vc = normal(gen, B, Hkv, max_len, d), normal(gen, B, Hkv, max_len, d)
    n = past + T
    kc[:, :, n:], vc[:, :, n:] = float("nan"), float("nan")
    weights = torch.rand(B, Hkv, max_len, generator=gen)
    args = [q.cuda(), kc.cuda(), vc.cuda(), past]
    dev = weights.cuda()
    out = ops.prefill_attention_weights(*args, dev)
    again = weights.cuda()
    assert torch.equal(ops.prefill_attention_weights(*args, again), out) and torch.equal(again, dev)
    assert torch.equal(out, flh_amd._CUDA.prefill_attention(*args))    # the bits of the operator without weights
    assert torch.equal(dev[:, :, n:].cpu(), weights[:, :, n:])
    seen = torch.ones(T, n, dtype=torch.bool).tril(past)
    for b in range(B):
        for g in range(Hkv):
            added, sizes = 0, 0
            for h in range(g * Hq // Hkv, (g + 1) * Hq // Hkv):
                _, p, size = attend64(q[b, :, h].double(), kc[b, g, :n].double(), vc[b, g, :n].double(), seen, d ** -0.5)
                added, sizes = added + p.sum(0), max(sizes, size)
            total = weights[b, g, :n].double() + added
            tol = weights_tolerance(sizes, d, n, T * Hq // Hkv, added, total)
            assert ((dev[b, g, :n].cpu().double() - total).abs() <= tol).all()


def test_attention_weights_in_a_graph(ops):
    from flh_amd import _lib
    gen = torch.Generator().manual_seed(5)
    B, Hq, Hkv, d, max_len = 2, 8, 2, 128, 300
    q, kc, vc = (t.cuda() for t in (normal(gen, B, Hq, d), normal(gen, B, Hkv, max_len, d), normal(gen, B, Hkv, max_len, d)))
    lengths, weights = torch.tensor([10, 20]).cuda(), torch.zeros(B, Hkv, max_len).cuda()
    ws = torch.empty(_lib.load().flh_decode_attention_weights_workspace_bytes(B, Hq, Hkv, d, max_len), dtype=torch.uint8, device="cuda")
    ops.decode_attention_weights(q, kc, vc, lengths, weights, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.decode_attention_weights(q, kc, vc, lengths, weights, workspace=ws)
    for lens in ([300, 1], [150, 151], [0, 64]):
        lengths.copy_(torch.tensor(lens))
        weights.zero_()
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.zeros_like(weights)
        for _ in range(2):
            ref = ops.decode_attention_weights(q, kc, vc, lengths, eager, workspace=ws.clone())
        assert torch.equal(out, ref) and torch.equal(weights, eager)
        sums = weights.sum(-1).cpu()                                   # probabilities add up to one a query
        want = torch.tensor([[2.0 * Hq / Hkv if n else 0.0] * Hkv for n in lens])
        assert ((sums - want).abs() <= 1e-4).all()


# ---------------------------------------------------------------------------------------------------- eviction
def evict_oracle(caches, weights, lengths, budget, recent, max_len):
    L, B, Hkv = weights.shape[:3]
    kept = np.full((L, B, Hkv, budget), -1)
    new_w, new = np.zeros_like(weights), np.array(lengths)
    caches = [c.clone() for c in caches]
    for b, n in enumerate(lengths):
        if n < 0 or n > max_len:
            continue
        new[b] = min(n, budget)
        for l in range(L):
            for g in range(Hkv):
                w = weights[l, b, g]
                keep = list(range(n))
                if n > budget:
                    key = [(-np.inf, i) if np.isnan(w[i]) else (-w[i] + 0.0, i) for i in range(n - recent)]
                    nans = [i for i in range(n - recent) if np.isnan(w[i])]
                    rest = [i for _, i in sorted((k, i) for k, i in key if not np.isnan(w[i]))]
                    keep = sorted((nans + rest)[:budget - recent]) + list(range(n - recent, n))
                kept[l, b, g, :len(keep)] = keep
                new_w[l, b, g, :len(keep)] = w[keep]
                for c in (caches[l], caches[L + l]):
                    c[b, g, :len(keep)] = c[b, g, keep].clone()
    return kept, new_w, new, caches


@pytest.mark.parametrize("L,B,Hkv,d,max_len,lengths,budget,recent,kind",
                         [(1, 1, 1, 128, 64, [64], 32, 4, "random"), (2, 3, 2, 128, 300, [300, 100, 257], 100, 100, "random"),
                          (3, 2, 2, 64, 700, [513, 700], 511, 0, "ties"), (130, 1, 1, 8, 40, [33], 17, 5, "ties"),
                          (1, 4, 1, 128, 64, [-1, 0, 65, 10], 10, 3, "random"), (1, 2, 1, 64, 64, [2 ** 63 - 1, 2 ** 32 + 9], 10, 3, "random"), (2, 2, 2, 128, 1025, [1025, 1024], 1024, 7, "equal"),
                          (1, 1, 2, 128, 2100, [2100], 1, 0, "random"), (1, 2, 1, 24, 500, [400, 500], 130, 20, "odd"),
                          (1, 1, 1, 128, 5000, [4999], 2500, 100, "front"), (1, 1, 1, 64, 9000, [9000], 4500, 1, "log")])
def test_evict(ops, L, B, Hkv, d, max_len, lengths, budget, recent, kind):
    gen = torch.Generator().manual_seed(budget)
    print(f"case evict L={L} B={B} d={d} max={max_len} budget={budget} recent={recent} {kind}", flush=True)
    w = torch.rand(L, B, Hkv, max_len, generator=gen)
    if kind == "ties":
        w = (w * 8).floor() / 8
    elif kind == "equal":
        w.fill_(0.25)
    elif kind == "front":
        w = w + torch.arange(max_len, 0, -1)                            # the first slots stay where they are
    elif kind == "log":
        w = torch.exp(40 * (w - 0.8))
    elif kind == "odd":                                                # signs, zeros of both, infinities, NaN
        w = w - 0.5
        w[..., ::7], w[..., 1::7], w[..., 3::50], w[..., 4::60], w[..., 5::70] = 0.0, -0.0, float("inf"), -float("inf"), float("nan")
    caches = [normal(gen, B, Hkv, max_len, d) for _ in range(2 * L)]
    kept, new_w, new, ref = evict_oracle(caches, w.numpy(), lengths, budget, recent, max_len)
    dev = [c.cuda() for c in caches]
    wd, ld = w.cuda(), torch.tensor(lengths).cuda()
    got = ops.evict_kv_cache_(dev[:L], dev[L:], wd, ld, budget, recent)
    assert np.array_equal(got[0].cpu().numpy(), kept)
    assert np.array_equal(got[1].cpu().numpy(), new_w, equal_nan=True)
    assert np.array_equal(got[2].cpu().numpy(), new)
    assert torch.equal(wd.cpu().nan_to_num(9.0), w.nan_to_num(9.0)) and ld.tolist() == lengths
    for g, r in zip(dev, ref):
        assert equal_bits(g, r)                                        # the rows behind the budget among them


def test_evict_a_single_pair_of_tensors(ops):
    gen = torch.Generator().manual_seed(6)
    k, v = normal(gen, 1, 2, 50, 64).cuda(), normal(gen, 1, 2, 50, 64).cuda()
    w = torch.rand(1, 1, 2, 50, generator=gen).cuda()
    kk, vv = k.clone(), v.clone()
    kept, _, n = ops.evict_kv_cache_(k, v, w, torch.tensor([50]).cuda(), 20, 4)
    assert n.tolist() == [20] and tuple(kept.shape) == (1, 1, 2, 20)
    at = kept[0][..., None].expand(1, 2, 20, 64)
    assert torch.equal(k[:, :, :20], kk.gather(2, at)) and torch.equal(v[:, :, :20], vv.gather(2, at))


# ---------------------------------------------------------------------------------------------------- sizes
def test_offsets_beyond_32_bits(ops):
    """A cache whose last heads lie more than 4 GiB behind its start, against the same slots in a small one: the same bits."""
    gen = torch.Generator().manual_seed(8)
    B, T, Hq, Hkv, d, n, small, large = 1, 6, 34, 17, 128, 100, 128, 1 << 20
    case = [t.cuda() for t in tree_case(gen, B, T, Hq, Hkv, d, [n], small, "tree")]
    big = [torch.empty(B, Hkv, large, d, dtype=torch.float16, device="cuda") for _ in range(2)]
    for b, s in zip(big, case[7:]):
        b[:, :, :small] = s
    assert big[0].stride(1) * (Hkv - 1) * 2 >= 2 ** 32

    def same():
        return all(equal_bits(b[:, :, :small], s) for b, s in zip(big, case[7:]))
    assert torch.equal(ops.tree_attention(*case[:7], *big), ops.tree_attention(*case))
    assert same()
    parents, tokens = torch.tensor([-1, 0, 0, 1, 2, 4]).cuda(), torch.arange(6)[None].cuda()
    chosen = torch.tensor([[2, 9, 4, 9, 5, 9]]).cuda()
    got = ops.tree_commit_(tokens, parents, chosen, case[5], *big)
    ref = ops.tree_commit_(tokens, parents, chosen, case[5], *case[7:])
    assert all(torch.equal(a, b) for a, b in zip(got, ref)) and got[1].tolist() == [4] and same()
    q = normal(gen, B, Hq, d).cuda()
    w = torch.rand(B, Hkv, small, generator=gen).cuda()
    wide = torch.zeros(B, Hkv, large, device="cuda")
    wide[:, :, :small] = w
    assert torch.equal(ops.decode_attention_weights(q, *big, got[3], wide), ops.decode_attention_weights(q, *case[7:], got[3], w))
    assert torch.equal(wide[:, :, :small], w)
    qs = normal(gen, B, 40, Hq, d).cuda()
    assert torch.equal(ops.prefill_attention_weights(qs, *big, 60, wide), ops.prefill_attention_weights(qs, *case[7:], 60, w))
    assert torch.equal(wide[:, :, :small], w)
    got = ops.evict_kv_cache_(*big, wide[None], got[3], 50, 9)         # (weights of more slots than are staged at once)
    ref = ops.evict_kv_cache_(*case[7:], w[None], ref[3], 50, 9)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1][..., :small], ref[1]) and torch.equal(got[2], ref[2]) and same()
    assert not got[1][..., small:].any()


# ---------------------------------------------------------------------------------------------------- together
def test_a_generation_with_a_bounded_cache_and_drafts(ops):
    """A prompt with weights, a cut, decode steps with weights, another cut, a drafted tree and its commit, all on one cache:
    every step against float64 on the state that the one before left."""
    gen = torch.Generator().manual_seed(7)
    B, Hq, Hkv, d, max_len, prompt, budget = 2, 8, 2, 128, 256, 200, 96
    kc, vc = normal(gen, B, Hkv, max_len, d).cuda(), normal(gen, B, Hkv, max_len, d).cuda()
    weights = torch.zeros(B, Hkv, max_len).cuda()
    ops.prefill_attention_weights(normal(gen, B, prompt, Hq, d).cuda(), kc, vc, 0, weights)
    assert (weights[:, :, :prompt].sum(-1).cpu() - prompt * Hq / Hkv).abs().max() < 0.05
    lengths = torch.tensor([prompt] * B).cuda()
    kept, w, lengths = ops.evict_kv_cache_(kc, vc, weights[None].contiguous(), lengths, budget, 16)
    weights = w[0]
    assert lengths.tolist() == [budget] * B
    for step in range(3):
        lengths = lengths + 1
        q = normal(gen, B, Hq, d).cuda()
        before = weights.clone()
        out = ops.decode_attention_weights(q, kc, vc, lengths, weights)
        n = budget + step + 1
        for b in range(B):
            for h in range(Hq):
                k, v = kc[b, h // 4, :n].cpu().double(), vc[b, h // 4, :n].cpu().double()
                ref, _, _ = attend64(q[b, h:h + 1].cpu().double(), k, v, torch.ones(1, n, dtype=torch.bool), d ** -0.5)
                assert ((out[b, h].cpu().double() - ref[0]).abs() <= v.abs().max() * (2 * H16 + n * 2.0 ** -25 + 1e-5)).all()
        assert (weights - before >= 0).all() and torch.equal(weights[:, :, n:], before[:, :, n:])
    kept, w, lengths = ops.evict_kv_cache_(kc, vc, weights[None].contiguous(), lengths, budget, 3)
    assert (kept[..., -3:].cpu() == torch.arange(budget, budget + 3)).all()
    T = 11
    case = tree_case(gen, B, T, Hq, Hkv, d, [budget] * B, max_len, "tree")
    case = (*case[:5], lengths.cpu(), case[6], kc.cpu(), vc.cpu())
    _, kc, vc = check_tree(ops, case)
    parents = torch.tensor([-1, 0, 0, 1, 1, 2, 2, 5, 5, 7, 7]).cuda()
    tokens = torch.arange(T).expand(B, T).contiguous().cuda()
    chosen = torch.tensor([[2, 9, 6, 9, 9, 9, 9, 9, 9, 9, 9], [2, 9, 5, 9, 9, 8, 9, 9, 3, 9, 9]]).cuda()
    keys = kc.clone()
    path, accepted, following, lengths = ops.tree_commit_(tokens, parents, chosen, lengths, kc, vc)
    assert accepted.tolist() == [3, 4] and following.tolist() == [9, 3] and lengths.tolist() == [budget + 3, budget + 4]
    assert path[1, :5].tolist() == [0, 2, 5, 8, -1]
    assert torch.equal(kc[1, :, budget + 3], keys[1, :, budget + 8]) and torch.equal(kc[0, :, budget + 3:], keys[0, :, budget + 3:])

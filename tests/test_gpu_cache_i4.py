"""The operators on a key / value cache held in 4 bits -- write, read, decode step, attention of a block -- against plain evaluations: codes
bit for bit against the same float32 expression on the CPU, attention against float64 over what the cache holds.

Tolerances count roundings (half a step of fp16 is 2^-11 of a value, of float32 2^-24).  Attention: the result and every probability times its
value's scale are rounded to fp16: 2^-11 of |out| and of sum p |v|; a weight below the smallest normal fp16 is off by 2^-25, where the
largest is 2^10 or more when its reference is set: 2^-35 of the largest p vs, times codes of up to 8, counted as 2^-30 of the largest |v| per key.  A
score is a float32 sum of d products (twice, high and low halves of the query) of the query with codes + 8, less eight times the query's sum: (4 d + 32)
half steps of scale * sum |q| (|code| + 8) ks, which a probability takes twice (numerator and sum).  The sums of p vs (code + 8), and of p vs 8, which
is taken off: codes enter the matrix instructions as subnormals of 2^-20, whose products are lined up by the exponent of the smallest normal number, 2^-14, and
cut at 24 bits from there, so each instruction is off by up to 2^-24 2^-14 / 2^-20 = 2^-18 of the largest p vs among its sixteen (or eight times two) keys, and
by float32 steps of what has been added up, at most 2^-24 16 = 2^-20 of the largest again: per sixteen keys, and once for the last, two instructions with
5/4 2^-18 each."""
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


# ------------------------------------------------------------------------------------------------ the plain evaluations (CPU)
def normal(gen, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).half()


def rotary(gen, *shape):
    angle = torch.rand(*shape[:-1], shape[-1] // 2, generator=gen, dtype=torch.float64) * 6.28
    angle = torch.cat((angle, angle), -1)
    return angle.cos().half(), angle.sin().half()


def turned(x, cos, sin, dtype=torch.float32):
    """x [..., H, d], cos / sin [..., d]: rotary embedding and Hadamard rotation, one rounding per step"""
    x, c, s = x.to(dtype), cos.to(dtype).unsqueeze(-2), sin.to(dtype).unsqueeze(-2)
    d = x.size(-1)
    x = x * c + torch.cat((-x[..., d // 2:], x[..., :d // 2]), -1) * s
    stride = 1
    while stride < d:
        pair = x.reshape(*x.shape[:-1], d // (2 * stride), 2, stride)
        a, b = pair[..., 0, :], pair[..., 1, :]
        x = torch.stack((a + b, a - b), -2).reshape(x.shape)
        stride *= 2
    return x * torch.tensor(d ** -0.5, dtype=dtype)


def quantised(y):
    """float32 rows -> codes int8 [..., d], scales fp16"""
    s = (y.abs().amax(-1) * torch.tensor(1 / 7, dtype=torch.float32)).half()
    s = torch.where(s == 0, torch.ones_like(s), s)
    bad = ~torch.isfinite(y).all(-1) | ~torch.isfinite(s)
    c = torch.round(y / s.float().unsqueeze(-1)).clamp(-8, 7)
    c = torch.where(bad.unsqueeze(-1), torch.zeros_like(c), c)
    return c.to(torch.int8), torch.where(bad, torch.full_like(s, float("nan")), s)


def packed(codes):
    c = codes.to(torch.int16) & 15
    return (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8)


def unpacked(b):
    c = torch.stack((b & 15, b >> 4), -1).flatten(-2).to(torch.int16)
    return torch.where(c > 7, c - 16, c)


def hadamard64(d):
    m = torch.ones(1, 1, dtype=torch.float64)
    while m.size(0) < d:
        m = torch.cat((torch.cat((m, m), 1), torch.cat((m, -m), 1)), 0)
    return m / d ** 0.5


def random_cache(gen, B, Hkv, max_len, d, spread=1.0):
    """Any codes (-8 among them), scales that differ by up to `spread`."""
    codes = [torch.randint(0, 256, (B, Hkv, max_len, d // 2), generator=gen, dtype=torch.uint8) for _ in range(2)]
    scales = [((torch.rand(B, Hkv, max_len, generator=gen) * spread + 0.2) * 0.3).half() for _ in range(2)]
    return codes[0], scales[0], codes[1], scales[1]


def attend64(q, kc, ks, vc, vs, limits, scale):
    """q [R, d] over codes [n, d] and scales [n], query r over the first limits[r] keys -> (out, tolerance) [R, d]"""
    n, d = kc.shape
    seen = torch.arange(n) < torch.as_tensor(limits)[:, None]
    q, any_ = q.double(), seen.any(0)
    ks, vs = torch.where(any_, ks.double(), 0.0), torch.where(any_, vs.double(), 0.0)
    k, v = kc.double() * ks[:, None], vc.double() * vs[:, None]
    s = torch.where(seen, (q @ k.t()) * scale, -torch.inf)
    p = torch.softmax(s, -1)
    size = torch.where(seen, (q.abs() @ ((kc.double().abs() + 8) * ks[:, None].abs()).t()) * scale, 0.0).amax(-1, keepdim=True)
    spread = p @ v.abs()
    out = p @ v
    tol = H16 * out.abs() + (H16 + 2 * (4 * d + 32) * H32 * (1 + size)) * spread + n * 2.0 ** -30 * v.abs().max() + 1e-7
    tol = tol + (n // 16 + 4) * 2.5 * 2.0 ** -18 * (p * vs).amax(-1, keepdim=True)   # (a tile has four such steps, also a short one)
    return out, tol


def close(got, want, tol, what=""):
    got = got.double().cpu()
    off = (got - want).abs() - tol
    assert torch.isfinite(got).all() and (off <= 0).all(), (what, off.max().item(), ((got - want).abs() / tol).max().item())


# ------------------------------------------------------------------------------------------------ write
@pytest.mark.parametrize("B,T,Hq,Hkv,d,max_len,lengths", [
    (1, 1, 1, 1, 128, 1, [0]),
    (3, 7, 32, 8, 64, 517, [500, 0, 510]),
    (2, 33, 12, 4, 128, 101, [0, 68]),
    (4, 5, 3, 3, 128, 40, [35, -1, 36, 0]),                            # the second and third take no part
    (2, 9, 7, 1, 64, 31, [2 ** 62, 22]),
    (1, 300, 32, 8, 128, 600, [299])])
def test_write(ops, B, T, Hq, Hkv, d, max_len, lengths):
    gen = torch.Generator().manual_seed(B * 1000 + T)
    q, k, v = normal(gen, B, T, Hq, d, scale=2.0), normal(gen, B, T, Hkv, d), normal(gen, B, T, Hkv, d)
    k[..., 5::37] *= 8
    k[0, 0, 0] = 0                                                     # a row of zeros
    v[0, -1, 0] = 0
    v[0, 0, -1] = 6e-8                                                 # a row whose scale is the smallest there is
    v[0, 0, -1, 3] = 6e-7
    cos, sin = rotary(gen, B, T, d)
    cache = random_cache(gen, B, Hkv, max_len, d)
    want = [c.clone() for c in cache]
    (kc, ks), (vc, vs) = quantised(turned(k, cos, sin)), quantised(v.float())
    for b, n in enumerate(lengths):
        if 0 <= n <= max_len - T:
            for at, new in zip(want, (packed(kc[b]), ks[b], packed(vc[b]), vs[b])):
                at[b, :, n:n + T] = new.transpose(0, 1)
    dev = [t.cuda() for t in cache]
    qd = q.cuda()
    got = ops.rope_quantize_kv_cache_(qd, k.cuda(), v.cuda(), cos.cuda(), sin.cuda(), torch.tensor(lengths).cuda(), *dev)
    assert torch.equal(qd.cpu(), q)
    assert torch.equal(got.cpu(), turned(q, cos, sin).half())
    for a, b, name in zip(dev, want, ("k_codes", "k_scales", "v_codes", "v_scales")):
        assert torch.equal(a.cpu(), b), name


def test_write_borders(ops):
    """Values in the middle between two codes go to the even one; -8 does not occur with a normal scale, and does with a subnormal one."""
    d = 128
    v = torch.zeros(1, 4, 1, d)
    v[0, 0, 0, :15] = torch.arange(-7, 8) * 0.5 * 0.25                # scale 0.25: quotients at k / 2 ...
    v[0, 0, 0, 20] = 7 * 0.25
    v[0, 1, 0, :13] = torch.arange(-6, 7) * 1.0 + 0.5
    v[0, 1, 0, 14] = -7.0
    v[0, 2, 0, 0], v[0, 2, 0, 1] = 5.9604645e-08 * 10, -5.9604645e-08 * 10   # scale 2^-24 (10 / 7 rounded): quotients of 10
    v[0, 3, 0, 7] = 65504.0
    v = v.half()
    zero = torch.zeros(1, 4, 1, d).half()
    cos, sin = torch.ones(1, 4, d).half(), torch.zeros(1, 4, d).half()
    cache = [torch.zeros(1, 1, 4, 64, dtype=torch.uint8).cuda(), torch.zeros(1, 1, 4).half().cuda(), torch.zeros(1, 1, 4, 64, dtype=torch.uint8).cuda(),
             torch.zeros(1, 1, 4).half().cuda()]
    ops.rope_quantize_kv_cache_(zero.cuda(), zero.cuda(), v.cuda(), cos.cuda(), sin.cuda(), torch.zeros(1, dtype=torch.int64).cuda(), *cache)
    codes, scales = unpacked(cache[2].cpu())[0, 0], cache[3].cpu()[0, 0]
    assert codes[0, :15].tolist() == [-4, -3, -2, -2, -2, -1, 0, 0, 0, 1, 2, 2, 2, 3, 4] and codes[0, 20] == 7 and scales[0] == 0.25
    assert codes[1, :13].tolist() == [-6, -4, -4, -2, -2, 0, 0, 2, 2, 4, 4, 6, 6] and scales[1] == 1.0
    assert codes[2, 0] == 7 and codes[2, 1] == -8 and scales[2].item() == 2.0 ** -24
    assert codes[3, 7] == 7 and scales[3].item() == 65504 / 7 // 8 * 8 + (8 if 65504 / 7 % 8 >= 4 else 0)
    assert (cache[1] == 1).all() and (cache[0] == 0).all()            # keys of zeros


def test_write_in_place_and_non_finite():
    """The C entry takes q as q_out; rows that are not finite are held as NaN, and rows whose scale would not be."""
    from flh_amd import _lib
    gen = torch.Generator().manual_seed(3)
    B, T, Hq, Hkv, d, max_len = 1, 4, 4, 2, 64, 9
    q, k, v = normal(gen, B, T, Hq, d), normal(gen, B, T, Hkv, d), normal(gen, B, T, Hkv, d)
    k[0, 1, 0, 9] = float("nan")
    k[0, 2, 1, 60] = float("inf")
    k[0, 3, 0] = 60000.0                                               # its rotation has one value of 480000: scale beyond fp16
    k[0, 3, 0, 0] = 65504.0
    v[0, 0, 1, 63] = -float("inf")
    v[0, 2, 0, 0] = float("nan")
    cos, sin = torch.ones(B, T, d).half(), torch.zeros(B, T, d).half()
    cache = random_cache(gen, B, Hkv, max_len, d)
    dev = [t.cuda() for t in cache]
    qd, kd, vd, cd, sd, ld = q.cuda(), k.cuda(), v.cuda(), cos.cuda(), sin.cuda(), torch.tensor([5]).cuda()
    lib = _lib.load()
    _lib.check(lib.flh_rope_quant_kv_cache_i4(qd.data_ptr(), kd.data_ptr(), vd.data_ptr(), cd.data_ptr(), sd.data_ptr(), ld.data_ptr(), qd.data_ptr(),
                                              *(t.data_ptr() for t in dev), B, T, Hq, Hkv, d, max_len, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(qd.cpu(), turned(q, cos, sin).half())
    (kc, ks), (vc, vs) = quantised(turned(k, cos, sin)), quantised(v.float())
    assert torch.isnan(ks).sum() == 3 and torch.isnan(vs).sum() == 2
    for at, new in zip(dev, (packed(kc), ks, packed(vc), vs)):
        assert torch.equal(at.cpu()[:, :, 5:9].nan_to_num(-1.0) if at.dtype == torch.float16 else at.cpu()[:, :, 5:9],
                           new.transpose(1, 2).nan_to_num(-1.0) if at.dtype == torch.float16 else new.transpose(1, 2))


# ------------------------------------------------------------------------------------------------ read
@pytest.mark.parametrize("B,Hkv,d,max_len,rows,first", [
    (1, 1, 128, 1, 1, [0]), (3, 5, 64, 77, 40, [0, 37, 30]), (2, 8, 128, 33, 10, [-4, 30]), (2, 2, 128, 20, 25, [2 ** 62, -2 ** 62]),
    (4, 8, 128, 257, 257, [0, 0, 0, 0])])
def test_read(ops, B, Hkv, d, max_len, rows, first):
    gen = torch.Generator().manual_seed(rows)
    cache = random_cache(gen, B, Hkv, max_len, d, spread=50.0)
    keys, values = ops.dequantize_kv_cache(*(t.cuda() for t in cache), torch.tensor(first).cuda(), rows)
    k, v = (unpacked(cache[i]).double() * cache[i + 1].double().unsqueeze(-1) for i in (0, 2))
    k = k @ hadamard64(d)
    for b, f in enumerate(first):
        for i in range(rows):
            if 0 <= f + i < max_len:
                assert torch.equal(values[b, :, i].cpu(), v[b, :, f + i].half())       # (eleven and four bits: rounded once)
                got, want = keys[b, :, i].double().cpu(), k[b, :, f + i]
                assert ((got - want).abs() <= (H16 + 2 * H32) * want.abs() + 2.0 ** -25).all()
            else:
                assert (keys[b, :, i] == 0).all() and (values[b, :, i] == 0).all()


def test_read_gives_what_was_written(ops):
    """Written, read back: within half a code's step of the rotated row (a scale rounded to fp16 makes the step 2^-11 wider)."""
    gen = torch.Generator().manual_seed(8)
    B, T, Hkv, d = 2, 50, 4, 128
    k, v, q = normal(gen, B, T, Hkv, d), normal(gen, B, T, Hkv, d), normal(gen, B, T, 8, d)
    cos, sin = rotary(gen, B, T, d)
    cache = [t.cuda() for t in random_cache(gen, B, Hkv, 64, d)]
    lengths = torch.tensor([0, 14]).cuda()
    ops.rope_quantize_kv_cache_(q.cuda(), k.cuda(), v.cuda(), cos.cuda(), sin.cuda(), lengths, *cache)
    keys, values = ops.dequantize_kv_cache(*cache, lengths, T)
    y = turned(k, cos, sin, torch.float64)
    plain = (y @ hadamard64(d)).transpose(1, 2)                        # the rotary embedding alone
    step = y.abs().amax(-1, keepdim=True).transpose(1, 2) / 7 * (1 + 2 * H16)
    back = keys.double().cpu() @ hadamard64(d) - plain @ hadamard64(d)
    assert (back.abs() <= step * 0.5 + 7 * step * H16 + d ** 0.5 * H16 * plain.abs().amax(-1, keepdim=True)).all()
    step = v.double().abs().amax(-1, keepdim=True).transpose(1, 2) / 7 * (1 + 2 * H16)
    assert ((values.double().cpu() - v.double().transpose(1, 2)).abs() <= step * 0.5 + 7 * step * H16 + H16 * values.double().cpu().abs()).all()


# ------------------------------------------------------------------------------------------------ decode
def decode_case(gen, B, Hq, Hkv, d, max_len, lengths, qscale=2.0, spread=1.0):
    q, k, v = normal(gen, B, Hq, d, scale=qscale), normal(gen, B, Hkv, d), normal(gen, B, Hkv, d)
    cos, sin = rotary(gen, B, d)
    cache = random_cache(gen, B, Hkv, max_len, d, spread)
    for b, n in enumerate(lengths):                                    # what lies behind a sequence is not looked at
        if n < max_len:
            cache[1][b, :, max(n, 0):] = float("nan")
            cache[3][b, :, max(n, 0):] = float("nan") if b % 2 else float("inf")
    return q, k, v, cos, sin, torch.tensor(lengths), cache


def check_decode(ops, case, scale=None, **more):
    q, k, v, cos, sin, lengths, cache = case
    B, Hq, d = q.shape
    Hkv, max_len = cache[0].size(1), cache[0].size(2)
    dev = [t.cuda() for t in cache]
    inputs = [t.cuda() for t in (q, k, v, cos, sin, lengths)]
    out = ops.decode_attention_rope_i4(*inputs, *dev, **({} if scale is None else {"scale": scale}), **more)
    for a, b in zip(inputs, (q, k, v, cos, sin, lengths)):
        assert torch.equal(a.cpu(), b)
    want = [t.clone() for t in cache]
    (kc, ks), (vc, vs) = quantised(turned(k, cos, sin)), quantised(v.float())
    qt = turned(q, cos, sin, torch.float64)
    for b, n in enumerate(lengths.tolist()):
        if not 0 <= n < max_len:
            assert (out[b] == 0).all()
            continue
        for at, new in zip(want, (packed(kc[b]), ks[b], packed(vc[b]), vs[b])):
            at[b, :, n] = new
        for g in range(Hkv):
            heads = slice(g * (Hq // Hkv), (g + 1) * (Hq // Hkv))
            x, tol = attend64(qt[b, heads], unpacked(want[0][b, g, :n + 1]), want[1][b, g, :n + 1], unpacked(want[2][b, g, :n + 1]),
                              want[3][b, g, :n + 1], [n + 1] * (Hq // Hkv), d ** -0.5 if scale is None else scale)
            close(out[b, heads], x, tol, (b, g, n))
    for a, b in zip(dev, want):
        assert torch.equal(a.cpu().nan_to_num(-1.0) if a.dtype == torch.float16 else a.cpu(), b.nan_to_num(-1.0) if b.dtype == torch.float16 else b)
    return out


@pytest.mark.parametrize("B,Hq,Hkv,d,max_len,lengths", [
    (1, 1, 1, 128, 1, [0]),                                            # nothing but the new token
    (1, 4, 1, 64, 3, [2]),
    (2, 32, 8, 128, 130, [63, 64]),                                    # a tile that the new token fills, one that it begins
    (3, 32, 32, 128, 400, [127, 300, 1]),
    (2, 28, 4, 128, 200, [199, 60]),                                   # seven queries per head; the last slot
    (4, 12, 4, 64, 333, [332, -1, 333, 100]),                          # two that take no part
    (2, 40, 2, 128, 150, [149, 3]),                                    # twenty queries per head: two blocks
    (2, 64, 1, 64, 90, [89, 70]),                                      # sixty-four
    (1, 8, 8, 128, 9000, [8765]),
    (1, 8, 1, 64, 70000, [65536]),                                     # many tiles of one head
    (70, 4, 2, 64, 140, [(37 * i) % 150 - 5 for i in range(70)])])     # more sequences than lanes, some out of range
def test_decode(ops, B, Hq, Hkv, d, max_len, lengths):
    check_decode(ops, decode_case(torch.Generator().manual_seed(B + max_len), B, Hq, Hkv, d, max_len, lengths))


@pytest.mark.parametrize("qscale,scale,spread", [(30.0, None, 1.0), (1e-3, None, 1.0), (2.0, 1.5, 1.0), (0.0, None, 1.0), (2.0, None, 10.0), (200.0, 1e-4, 1.0)])
def test_decode_magnitudes(ops, qscale, scale, spread):
    """Sharp and flat probabilities, queries of zeros, value scales that differ."""
    check_decode(ops, decode_case(torch.Generator().manual_seed(5), 2, 16, 4, 128, 700, [699, 350], qscale, spread), scale)


@pytest.mark.parametrize("scale", [2.0 ** -24, 1e-6, 9000.0])
def test_decode_value_scales(ops, scale):
    """Values that are tiny or huge throughout keep their precision."""
    case = decode_case(torch.Generator().manual_seed(6), 1, 8, 2, 128, 300, [255])
    case[6][3][:, :, :255] = scale
    case[2].mul_(0).add_(scale * 7 if scale < 1 else 6000.0)
    check_decode(ops, case)


def test_decode_step_by_step(ops):
    """Twenty tokens one after another, across a tile's border: every step sees what the steps before have written."""
    gen = torch.Generator().manual_seed(11)
    B, Hq, Hkv, d, max_len = 2, 8, 2, 128, 96
    lengths = [50, 60]
    cache = decode_case(gen, B, Hq, Hkv, d, max_len, lengths)[6]
    for _ in range(20):
        q, k, v = normal(gen, B, Hq, d, scale=2.0), normal(gen, B, Hkv, d), normal(gen, B, Hkv, d)
        cos, sin = rotary(gen, B, d)
        check_decode(ops, (q, k, v, cos, sin, torch.tensor(lengths), cache))
        (kc, ks), (vc, vs) = quantised(turned(k, cos, sin)), quantised(v.float())
        for b, n in enumerate(lengths):
            for at, new in zip(cache, (packed(kc[b]), ks[b], packed(vc[b]), vs[b])):
                at[b, :, n] = new
        lengths = [n + 1 for n in lengths]


# ------------------------------------------------------------------------------------------------ attention of a block
def check_prefill(ops, q, lengths, cache, scale=None, **more):
    B, T, Hq, d = q.shape
    Hkv, max_len = cache[0].size(1), cache[0].size(2)
    dev = [t.cuda() for t in cache]
    out = ops.prefill_attention_i4(q.cuda(), torch.tensor(lengths).cuda(), *dev, **({} if scale is None else {"scale": scale}), **more)
    assert out.shape == (B, T, Hq * d)
    got = out.view(B, T, Hq, d)
    rep = Hq // Hkv
    for b, n in enumerate(lengths):
        if not 0 <= n <= max_len - T:
            assert (got[b] == 0).all()
            continue
        for g in range(Hkv):
            kc, ks, vc, vs = unpacked(cache[0][b, g, :n + T]), cache[1][b, g, :n + T], unpacked(cache[2][b, g, :n + T]), cache[3][b, g, :n + T]
            limits = torch.arange(n + 1, n + T + 1).repeat_interleave(rep)
            x, tol = attend64(q[b, :, g * rep:(g + 1) * rep].reshape(T * rep, d), kc, ks, vc, vs, limits, d ** -0.5 if scale is None else scale)
            close(got[b, :, g * rep:(g + 1) * rep].reshape(T * rep, d), x, tol, (b, g, n))
    return out


def prefill_case(gen, B, T, Hq, Hkv, d, max_len, lengths, qscale=2.0):
    cache = random_cache(gen, B, Hkv, max_len, d)
    for b, n in enumerate(lengths):
        if 0 <= n + T < max_len:
            cache[1][b, :, n + T:], cache[3][b, :, n + T:] = float("inf"), float("nan")
    return normal(gen, B, T, Hq, d, scale=qscale), cache


@pytest.mark.parametrize("B,T,Hq,Hkv,d,max_len,lengths", [
    (1, 1, 1, 1, 128, 1, [0]),
    (1, 1, 32, 8, 64, 200, [130]),
    (2, 5, 32, 8, 128, 300, [63, 200]),
    (1, 64, 4, 4, 128, 64, [0]),
    (2, 65, 6, 2, 128, 200, [0, 127]),                                 # three queries per head: rows of a block that end inside a token
    (3, 33, 28, 4, 64, 150, [117, -1, 118]),                           # the last two take no part
    (1, 300, 8, 8, 64, 400, [77]),
    (1, 257, 16, 2, 128, 700, [301]),
    (2, 40, 40, 2, 128, 100, [60, 0]),                                 # twenty queries per head
    (1, 3, 4, 1, 128, 9000, [8990]),                                   # few rows, many tiles
    (1, 1100, 2, 1, 64, 1100, [0]),
    (1, 700, 64, 32, 128, 700, [0])])
def test_prefill(ops, B, T, Hq, Hkv, d, max_len, lengths):
    gen = torch.Generator().manual_seed(T + max_len)
    q, cache = prefill_case(gen, B, T, Hq, Hkv, d, max_len, lengths)
    check_prefill(ops, q, lengths, cache)


@pytest.mark.parametrize("T", [9, 600])                                # split over workgroups, and not
@pytest.mark.parametrize("qscale,scale", [(30.0, None), (1e-3, None), (2.0, 1.5), (0.0, None), (300.0, 1e-4)])
def test_prefill_magnitudes(ops, T, qscale, scale):
    gen = torch.Generator().manual_seed(T)
    q, cache = prefill_case(gen, 1, T, 16 if T < 100 else 64, 4 if T < 100 else 32, 128, 700, [100], qscale)
    check_prefill(ops, q, [100], cache, scale)


@pytest.mark.parametrize("T,Hq,Hkv", [(40, 4, 2), (400, 64, 32)])
def test_prefill_non_finite(ops, T, Hq, Hkv):
    """A key or a value that is NaN spoils the queries that see it, and no others; a query that is NaN spoils itself."""
    gen = torch.Generator().manual_seed(2)
    d, n = 128, 30
    q, cache = prefill_case(gen, 1, T, Hq, Hkv, d, 512, [n])
    bad = n + 20                                                       # (inside the first tile: queries in front of it share the tile)
    cache[1][0, 0, bad] = float("nan")
    cache[3][0, 1, bad + 3] = float("nan")
    q[0, 2, 0, 5] = float("inf")
    got = ops.prefill_attention_i4(q.cuda(), torch.tensor([n]).cuda(), *(t.cuda() for t in cache)).cpu().view(T, Hq, d)
    clean = [t.clone() for t in cache]
    clean[1][0, 0, bad], clean[3][0, 1, bad + 3] = 0.25, 0.25
    q[0, 2, 0, 5] = 0.5
    fine = ops.prefill_attention_i4(q.cuda(), torch.tensor([n]).cuda(), *(t.cuda() for t in clean)).cpu().view(T, Hq, d)
    rep = Hq // Hkv
    for h in range(Hq):
        first = {0: 20, 1: 23}.get(h // rep, T)
        for t in range(T):
            if t >= first or (t == 2 and h == 0):
                assert torch.isnan(got[t, h]).all(), (t, h)
            else:
                close(got[t, h], fine[t, h].double(), 4 * H16 * fine[t, h].double().abs() + 8 * H16, (t, h))


def test_decode_non_finite(ops):
    gen = torch.Generator().manual_seed(9)
    q, k, v, cos, sin, lengths, cache = decode_case(gen, 3, 4, 2, 128, 200, [100, 150, 199])
    k[0, 1, 4] = float("nan")                                          # the new key of a head
    cache[3][1, 0, 20] = float("nan")                                  # a value of another sequence
    out = ops.decode_attention_rope_i4(*(t.cuda() for t in (q, k, v, cos, sin, lengths)), *(t.cuda() for t in cache)).cpu()
    nan = torch.isnan(out).all(-1)
    assert nan.tolist() == [[False, False, True, True], [True, True, False, False], [False] * 4]
    assert torch.isfinite(out[~nan]).all()


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("d,Hq,Hkv", [(128, 16, 4), (64, 8, 8)])
def test_together(ops, d, Hq, Hkv):
    """A prompt in two blocks, then tokens one by one; every output is the attention over what the cache holds, and a block of tokens that
    were decoded one by one gives the decode steps' outputs."""
    gen = torch.Generator().manual_seed(d)
    B, max_len = 2, 260
    cache = [t.cuda() for t in random_cache(gen, B, Hkv, max_len, d)]
    lengths = torch.tensor([0, 40]).cuda()

    def block(T):
        q, k, v = normal(gen, B, T, Hq, d, scale=2.0), normal(gen, B, T, Hkv, d), normal(gen, B, T, Hkv, d)
        return [t.cuda() for t in (q, k, v, *rotary(gen, B, T, d))]

    for T in (100, 37):
        x = block(T)
        q = ops.rope_quantize_kv_cache_(*x, lengths, *cache)
        out = ops.prefill_attention_i4(q, lengths, *cache)
        again = check_prefill(ops, q.cpu(), lengths.tolist(), [t.cpu() for t in cache])
        assert torch.equal(out, again)
        lengths = lengths + T
    x = block(6)
    held = [t.clone() for t in cache]
    q = ops.rope_quantize_kv_cache_(*x, lengths, *held)
    whole = ops.prefill_attention_i4(q, lengths, *held).view(B, 6, Hq, d)
    for t in range(6):
        out = ops.decode_attention_rope_i4(*(y[:, t].contiguous() for y in x), lengths + t, *cache)
        # (the block's queries are rounded to fp16 between the two calls: 2^-11 of a score's terms, twice)
        spread = 3 * H16 + 2 * H16 * d ** -0.5 * q.double().abs().sum(-1).max().item() * 1.0
        assert (out.double() - whole[:, t].double()).abs().max().item() <= spread * 3
    for a, b in zip(cache, held):
        assert torch.equal(a, b)


def test_same_bits(ops):
    """The same call gives the same bits, whatever the workspace held."""
    gen = torch.Generator().manual_seed(4)
    q, k, v, cos, sin, lengths, cache = decode_case(gen, 5, 32, 8, 128, 3000, [2999, 100, 1777, 0, 640])
    x, dev = [t.cuda() for t in (q, k, v, cos, sin, lengths)], [t.cuda() for t in cache]
    first = ops.decode_attention_rope_i4(*x, *dev)
    ws = torch.full((64 << 20,), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(ops.decode_attention_rope_i4(*x, *dev, workspace=ws), first)
    q = normal(gen, 5, 7, 32, 128).cuda()
    lengths = torch.tensor([2900, 100, 1777, 0, 640]).cuda()
    dev = [t.cuda() for t in random_cache(gen, 5, 8, 3000, 128)]
    first = ops.prefill_attention_i4(q, lengths, *dev)
    ws.fill_(255)
    assert torch.equal(ops.prefill_attention_i4(q, lengths, *dev, workspace=ws), first)

"""The operators on a key / value cache held in 4 bits, as they are measured:

  write    rotary embedding and Hadamard rotation of a block of new queries and keys, keys and values quantised into the cache
           behind what it holds, ``rope_quantize_kv_cache_``; what was written is read back, ``dequantize_kv_cache``
  read     a range of every sequence's slots as fp16 keys and values, ``dequantize_kv_cache``
  decode   one new token per sequence: the same rotation and write, and its attention over the cache, ``decode_attention_rope_i4``
  prefill  causal attention of a block of new tokens over the cache that holds them, ``prefill_attention_i4``

A layer's cache is codes uint8 [batch, key / value heads, slots, channels / 2] (element 2 j in the low, 2 j + 1 in the high nibble of
byte j, two's complement) and scales fp16 [batch, key / value heads, slots], for keys (held rotated by the Hadamard matrix of a head) and
for values; ``lengths`` holds how many slots of each sequence are taken.  Cases have the heads of Llama-3-8B (32 query and 8 key / value heads
of 128 channels), of Llama-2-7B (32 of each), or heads of 64 channels.  `own` chooses between the library's operators and their plain form
in torch operations.
"""
import math

import torch

own = False

DEVICE = "cuda"


def listed():
    return [
        # a short question in a long chat, three sequences, heads of 64 channels
        {"name": "write_3x7_after_500_d64", "kind": "write", "batch": 3, "tokens": 7, "length": 500, "heads": 32, "kv_heads": 8,
         "channels": 64, "ragged": True},
        # a long prompt
        {"name": "write_1x8192", "kind": "write", "batch": 1, "tokens": 8192, "length": 0, "heads": 32, "kv_heads": 8, "channels": 128,
         "ragged": False},
        # one sequence's cache for an operator that takes fp16
        {"name": "read_1x900", "kind": "read", "batch": 1, "length": 900, "kv_heads": 8, "channels": 128, "ragged": False},
        # ... a batch's, one key / value head per query head, from slots of their own on
        {"name": "read_4x3000_ragged", "kind": "read", "batch": 4, "length": 3000, "kv_heads": 32, "channels": 128, "ragged": True},
        # the smallest step: the beginning of a chat
        {"name": "decode_1x300", "kind": "decode", "batch": 1, "length": 300, "heads": 32, "kv_heads": 8, "channels": 128,
         "ragged": False},
        # a few chats, one key / value head per query head
        {"name": "decode_5x777_mha", "kind": "decode", "batch": 5, "length": 777, "heads": 32, "kv_heads": 32, "channels": 128,
         "ragged": False},
        # one very long document
        {"name": "decode_1x60000", "kind": "decode", "batch": 1, "length": 60000, "heads": 32, "kv_heads": 8, "channels": 128,
         "ragged": False},
        # a ragged batch as a server has it
        {"name": "decode_32x8000_ragged", "kind": "decode", "batch": 32, "length": 8000, "heads": 32, "kv_heads": 8, "channels": 128,
         "ragged": True},
        # the second piece of a short prompt
        {"name": "prefill_1x300_after_77", "kind": "prefill", "batch": 1, "tokens": 300, "length": 77, "heads": 32, "kv_heads": 32,
         "channels": 128, "ragged": False},
        # a short turn of each of a few long chats
        {"name": "prefill_4x17_after_16000", "kind": "prefill", "batch": 4, "tokens": 17, "length": 16000, "heads": 32, "kv_heads": 8,
         "channels": 128, "ragged": True},
        # documents behind instructions, heads of 64 channels
        {"name": "prefill_2x1111_after_600_d64", "kind": "prefill", "batch": 2, "tokens": 1111, "length": 600, "heads": 16,
         "kv_heads": 16, "channels": 64, "ragged": True},
        # a long prompt
        {"name": "prefill_1x4096", "kind": "prefill", "batch": 1, "tokens": 4096, "length": 0, "heads": 32, "kv_heads": 8,
         "channels": 128, "ragged": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(("write", "read", "decode", "decode", "decode", "prefill", "prefill", "prefill"))
    heads, kv_heads, channels = rng.choice(((32, 8, 128), (32, 32, 128), (32, 8, 64), (16, 16, 64), (64, 8, 128), (12, 4, 128), (28, 4, 128)))
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "channels": channels, "ragged": rng.random() < 0.5}
    if kind == "write":
        tokens = _log_int(rng, 1, 4000)
        return {**case, "batch": _log_int(rng, 1, min(16, 4000 // tokens)), "tokens": tokens, "length": rng.choice((0, _log_int(rng, 1, 3000)))}
    if kind == "read":
        del case["heads"]
        length = _log_int(rng, 1, 8000)
        return {**case, "batch": _log_int(rng, 1, max(1, min(16, 96000 // (length * kv_heads)))), "length": length}
    if kind == "decode":
        length = _log_int(rng, 1, 60000)
        return {**case, "batch": _log_int(rng, 1, max(1, min(64, 900000 // (length * kv_heads)))), "length": length}
    tokens, most = _log_int(rng, 1, 2500), 2.6e8 / heads               # (pairs of a query and a slot that a head may have)
    length = rng.choice((0, _log_int(rng, 1, max(1, min(16000, int(most / tokens - tokens / 2))))))
    return {**case, "batch": _log_int(rng, 1, max(1, min(8, int(most / (tokens * (tokens / 2 + length)))))), "tokens": tokens, "length": length}


# ---------------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """Slots taken of each sequence: all `length`, or from there down to half of it."""
    n, b = case["length"], case["batch"]
    return [n - (n * i // (2 * b) if case["ragged"] else 0) for i in range(b)]


def _new(case):
    return 1 if case["kind"] == "decode" else case.get("tokens", 0)


def _rows(case):
    """Slots that a read takes of each sequence, and from where on."""
    lengths = _lengths(case)
    return min(lengths), [n - min(lengths) for n in lengths]


def _normal(gen, *shape, scale=1.0):
    return torch.empty(shape, device=DEVICE, dtype=torch.float16).normal_(0.0, scale, generator=gen)


def _pack(codes):
    """Codes [..., d] -> bytes [..., d / 2]"""
    low, high = codes[..., 0::2].to(torch.int32) & 15, codes[..., 1::2].to(torch.int32) & 15
    return (low | (high << 4)).to(torch.uint8)


def _filled(gen, batch, heads, slots, d, loud=False):
    """A cache of quantised normal rows; `loud`: a few positions that most queries look at."""
    codes = torch.empty(batch, heads, slots, d // 2, device=DEVICE, dtype=torch.uint8)
    scales = torch.empty(batch, heads, slots, device=DEVICE, dtype=torch.float16)
    for i in range(batch):                                             # (one sequence's values at a time)
        x = torch.empty(heads, slots, d, device=DEVICE).normal_(generator=gen)
        s = (x.abs().amax(-1) / 7).half()
        codes[i] = _pack(torch.round(x / s.float()[..., None]).clamp_(-8, 7))
        scales[i] = s
    if loud:
        scales[:, :, :: max(2, slots // 16)] *= 2.0
    return codes, scales


def _rotary(positions, d):
    angles = positions.double()[..., None] / 10000.0 ** (torch.arange(0, d, 2, device=DEVICE, dtype=torch.float64) / d)
    angles = torch.cat((angles, angles), -1)
    return angles.cos().half(), angles.sin().half()


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    b, g, d, t = case["batch"], case["kv_heads"], case["channels"], _new(case)
    slots = -(-(case["length"] + t) // 256) * 256                      # rounded up as a server allocates them
    state = {"case": case, "lengths": torch.tensor(_lengths(case), device=DEVICE)}
    state["k_codes"], state["k_scales"] = _filled(gen, b, g, slots, d, loud=case["kind"] != "write")
    state["v_codes"], state["v_scales"] = _filled(gen, b, g, slots, d)
    if case["kind"] == "read":
        state["first"] = torch.tensor(_rows(case)[1], device=DEVICE)
    elif case["kind"] == "prefill":
        state["q"] = _normal(gen, b, t, case["heads"], d, scale=2.0)
    else:
        state["q"] = _normal(gen, b, t, case["heads"], d, scale=2.0)
        state["k"], state["v"] = _normal(gen, b, t, g, d), _normal(gen, b, t, g, d)
        # channels of keys that are much larger than the others, as models have them
        state["k"][..., 5::37] *= 8.0
        state["cos"], state["sin"] = _rotary(state["lengths"][:, None] + torch.arange(t, device=DEVICE), d)
        if case["kind"] == "decode":
            for name in ("q", "k", "v", "cos", "sin"):
                state[name] = state[name][:, 0].contiguous()
    return state


# ---------------------------------------------------------------------------------------------------- the plain forms
def _rotate(x, cos, sin):
    """x [..., heads, d] with cos / sin [..., d] -> float32"""
    half = x.size(-1) // 2
    x = x.float()
    turned = torch.cat((-x[..., half:], x[..., :half]), -1)
    return x * cos.float()[..., None, :] + turned * sin.float()[..., None, :]


def _hadamard(x):
    """x H / sqrt(d) for the Hadamard matrix of the last axis, by butterflies over strides 1, 2, 4, ..."""
    d, shape, stride = x.size(-1), x.shape, 1
    while stride < d:
        pair = x.reshape(*shape[:-1], d // (2 * stride), 2, stride)
        x = torch.stack((pair[..., 0, :] + pair[..., 1, :], pair[..., 0, :] - pair[..., 1, :]), -2)
        stride *= 2
    return x.reshape(shape) * d ** -0.5


def _quantize(y):
    """float32 rows -> packed codes, fp16 scales"""
    s = (y.abs().amax(-1) * (1 / 7)).half()
    s = torch.where(s == 0, 1.0, s)
    return _pack(torch.round(y / s.float()[..., None]).clamp(-8, 7)), s


def _values(codes, scales):
    """Packed codes and scales -> what they stand for, float32"""
    low, high = codes & 15, codes >> 4
    c = torch.stack((low, high), -1).reshape(*codes.shape[:-1], -1).to(torch.int32)
    return (((c + 8) & 15) - 8).float() * scales.float()[..., None]


def _write_plain(s, k, v, cos, sin):
    """k, v [b, t, g, d] into the slots behind the sequences' lengths"""
    rows = torch.arange(k.size(0), device=DEVICE)[:, None]
    places = s["lengths"][:, None] + torch.arange(k.size(1), device=DEVICE)
    codes, scales = _quantize(_hadamard(_rotate(k, cos, sin)))
    s["k_codes"][rows, :, places], s["k_scales"][rows, :, places] = codes, scales
    codes, scales = _quantize(v.float())
    s["v_codes"][rows, :, places], s["v_scales"][rows, :, places] = codes, scales


def _read_plain(s, first, n):
    rows = torch.arange(first.numel(), device=DEVICE)[:, None]
    places = first[:, None] + torch.arange(n, device=DEVICE)
    at = [s[name][rows, :, places].transpose(1, 2) for name in ("k_codes", "k_scales", "v_codes", "v_scales")]
    return {"keys": _hadamard(_values(*at[:2])).half().contiguous(), "values": _values(*at[2:]).half().contiguous()}


def _attention_plain(s, q, n, seen):
    """q [b, t, heads, d] float32 over the first n slots of the caches, seen [b, t, n]"""
    b, t, heads, d = q.shape
    g = s["k_codes"].size(1)
    q = q.view(b, t, g, heads // g, d).permute(0, 2, 1, 3, 4).reshape(b * g, -1, d)
    k = _values(s["k_codes"][:, :, :n], s["k_scales"][:, :, :n]).transpose(2, 3).reshape(b * g, d, n)
    scores = (torch.bmm(q, k) * d ** -0.5).view(b, g, t, heads // g, n)
    scores.masked_fill_(~seen[:, None, :, None], -math.inf)
    p = torch.exp_(scores.sub_(scores.amax(-1, keepdim=True)))
    total = p.sum(-1, keepdim=True)
    v = _values(s["v_codes"][:, :, :n], s["v_scales"][:, :, :n]).reshape(b * g, n, d)
    out = torch.bmm(p.view(b * g, -1, n), v).view(b, g, t, heads // g, d) / total
    return out.permute(0, 2, 1, 3, 4).reshape(b, t, heads * d).half()


def _plain(s):
    case = s["case"]
    kind, t = case["kind"], _new(case)
    if kind == "read":
        return _read_plain(s, s["first"], _rows(case)[0])
    if kind == "write":
        _write_plain(s, s["k"], s["v"], s["cos"], s["sin"])
        return {"q": _hadamard(_rotate(s["q"], s["cos"], s["sin"])).half(), **_read_plain(s, s["lengths"], t)}
    n = case["length"] + t
    seen = torch.arange(n, device=DEVICE) <= s["lengths"][:, None, None] + torch.arange(t, device=DEVICE)[:, None]
    if kind == "prefill":
        return {"out": _attention_plain(s, s["q"].float(), n, seen)}
    cos, sin = s["cos"][:, None], s["sin"][:, None]
    _write_plain(s, s["k"][:, None], s["v"][:, None], cos, sin)
    out = _attention_plain(s, _hadamard(_rotate(s["q"][:, None], cos, sin)), n, seen)
    return {"out": out.view(s["q"].shape), **_read_plain(s, s["lengths"], 1)}


# ---------------------------------------------------------------------------------------------------- the library's operators
def _library(s):
    import flh_amd
    ops = flh_amd._CUDA
    case, cache = s["case"], (s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"])
    kind = case["kind"]
    if kind == "read":
        keys, values = ops.dequantize_kv_cache(*cache, s["first"], _rows(case)[0])
        return {"keys": keys, "values": values}
    if kind == "prefill":
        return {"out": ops.prefill_attention_i4(s["q"], s["lengths"], *cache)}
    if kind == "write":
        q = ops.rope_quantize_kv_cache_(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["lengths"], *cache)
        keys, values = ops.dequantize_kv_cache(*cache, s["lengths"], case["tokens"])
        return {"q": q, "keys": keys, "values": values}
    out = ops.decode_attention_rope_i4(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["lengths"], *cache)
    keys, values = ops.dequantize_kv_cache(*cache, s["lengths"], 1)
    return {"out": out, "keys": keys, "values": values}


def run(state):
    with torch.no_grad():
        return _library(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------- what it cannot do without
def work(case):
    kind, b, g, d, t = case["kind"], case["batch"], case["kv_heads"], case["channels"], _new(case)
    row, whole = g * (d + 4), g * 4 * d                                # a position's keys and values in 4 bits, and in fp16
    if kind == "read":
        return {"bytes": b * _rows(case)[0] * (row + whole), "flops": 0}
    heads, lengths = case["heads"], _lengths(case)
    if kind == "prefill":
        pairs = sum(t * n + t * (t + 1) // 2 for n in lengths)
        return {"bytes": sum((n + t) * row for n in lengths) + b * 4 * t * heads * d, "flops": 4 * d * heads * pairs}
    # queries in and out, keys and values in, their codes out, rotary rows; what was written comes back in fp16
    new = b * t * (4 * heads * d + 2 * whole + 2 * row + 4 * d)
    if kind == "write":
        return {"bytes": new, "flops": 0}
    return {"bytes": new + sum(lengths) * row, "flops": 4 * d * heads * sum(n + 1 for n in lengths)}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def _exact_matrix(d):
    m = torch.ones(1, 1, dtype=torch.float64, device=DEVICE)
    while m.size(0) < d:
        m = torch.kron(torch.tensor([[1.0, 1.0], [1.0, -1.0]], dtype=torch.float64, device=DEVICE), m)
    return m / math.sqrt(d)


def _exact_turned(x, cos, sin):
    """x [t, heads, d], cos / sin [t, d]"""
    first, second = x.double().chunk(2, -1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    h = first.size(-1)
    return torch.cat((first * c[..., :h] - second * s[..., :h], second * c[..., h:] + first * s[..., h:]), -1) @ _exact_matrix(x.size(-1))


def _exact_held(y):
    """What a row of 4-bit codes stands for"""
    s = (y.abs().amax(-1, keepdim=True) / 7).half().double()
    s = s.masked_fill(s == 0, 1.0)
    return (y / s).round().clamp(-8, 7) * s


def _exact_rows(codes, scales):
    c = codes.to(torch.int64)
    c = torch.stack((c % 16, c // 16), -1).flatten(-2)
    return torch.where(c > 7, c - 16, c).double() * scales.double()[..., None]


def exact(case, seed):
    s = prepare(case, seed)
    kind, b, t, d = case["kind"], case["batch"], _new(case), case["channels"]
    lengths = _lengths(case)
    if kind == "read":
        n, first = _rows(case)
        found = [(_exact_rows(s["k_codes"][i, :, f:f + n], s["k_scales"][i, :, f:f + n]) @ _exact_matrix(d),
                  _exact_rows(s["v_codes"][i, :, f:f + n], s["v_scales"][i, :, f:f + n])) for i, f in enumerate(first)]
        return {"keys": torch.stack([k for k, _ in found]), "values": torch.stack([v for _, v in found])}
    if kind == "decode":
        for name in ("q", "k", "v", "cos", "sin"):
            s[name] = s[name][:, None]
    out = []
    for i, n in enumerate(lengths):
        if kind == "prefill":
            q, n_cache = s["q"][i].double(), n + t
        else:
            q, n_cache = _exact_turned(s["q"][i], s["cos"][i], s["sin"][i]), n
            held = [_exact_held(x).transpose(0, 1) for x in (_exact_turned(s["k"][i], s["cos"][i], s["sin"][i]), s["v"][i].double())]
            back = {"keys": held[0] @ _exact_matrix(d), "values": held[1]}
            if kind == "write":
                out.append({"q": q, **back})
                continue
        keys = _exact_rows(s["k_codes"][i, :, :n_cache], s["k_scales"][i, :, :n_cache])
        values = _exact_rows(s["v_codes"][i, :, :n_cache], s["v_scales"][i, :, :n_cache])
        if kind == "decode":
            keys, values = torch.cat((keys, held[0]), 1), torch.cat((values, held[1]), 1)
        hidden = torch.ones(t, n + t, dtype=torch.bool, device=DEVICE).triu(n + 1)
        rep = q.size(1) // keys.size(0)
        heads = [torch.softmax((q[:, h] @ keys[h // rep].t() / math.sqrt(d)).masked_fill_(hidden, -math.inf), -1) @ values[h // rep]
                 for h in range(q.size(1))]
        o = torch.stack(heads, 1)
        out.append({"out": o.reshape(t, -1)} if kind == "prefill" else {"out": o[0], **back})
    return {name: torch.stack([o[name] for o in out]) for name in out[0]}

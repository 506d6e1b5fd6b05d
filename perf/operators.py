"""The operators on a key / value cache that serve drafted tokens and bounded caches, as they are measured:

  tree      attention of a tree of drafted tokens over the cache and the tree itself: rotary embedding, cache write,
            attention, ``tree_attention``
  commit    the drafted tokens that the model agrees with, and their rows moved behind the sequence in every layer's
            cache, ``tree_commit_``
  prefill   causal attention of a prompt that adds every cached position's attention weight to its running sum,
            ``prefill_attention_weights``
  decode    the same for one new token per sequence, ``decode_attention_weights``
  evict     the positions with the largest sums (and the latest ones) kept, the caches compacted, ``evict_kv_cache_``

Cases have the heads of Llama-3-8B (32 query and 8 key / value heads of 128 channels), of Llama-2-7B (32 of each), or heads of
64 channels.  Caches are fp16 [batch, key / value heads, slots, channels], one per layer; ``lengths`` holds how many slots of
each sequence are taken.  `own` chooses between the library's operators and their plain form in torch operations.
"""
import math

import torch

own = False

DEVICE = "cuda"


def listed():
    return [
        # the smallest call: a short chat with a small draft
        {"name": "tree_1x8_after_120", "kind": "tree", "batch": 1, "nodes": 8, "length": 120, "heads": 32, "kv_heads": 8,
         "channels": 128, "ragged": False, "per_sequence": False},
        # a batch of ordinary chats, ragged, one key / value head per query head, a fixed tree
        {"name": "tree_4x26_after_1500", "kind": "tree", "batch": 4, "nodes": 26, "length": 1500, "heads": 32, "kv_heads": 32,
         "channels": 128, "ragged": True, "per_sequence": False},
        # heads of 64 channels, an odd number of nodes, a tree of its own per sequence
        {"name": "tree_2x63_after_5001_d64", "kind": "tree", "batch": 2, "nodes": 63, "length": 5001, "heads": 32, "kv_heads": 8,
         "channels": 64, "ragged": True, "per_sequence": True},
        # long documents, a large tree
        {"name": "tree_8x64_after_8192", "kind": "tree", "batch": 8, "nodes": 64, "length": 8192, "heads": 32, "kv_heads": 8,
         "channels": 128, "ragged": False, "per_sequence": False},
        # the end of a speculative step of one sequence, all layers of the model
        {"name": "commit_1x8", "kind": "commit", "batch": 1, "nodes": 8, "length": 500, "layers": 32, "kv_heads": 8, "channels": 128},
        # ... of a large batch with large trees
        {"name": "commit_16x64", "kind": "commit", "batch": 16, "nodes": 64, "length": 777, "layers": 32, "kv_heads": 8,
         "channels": 128},
        # the second piece of a short prompt
        {"name": "prefill_1x300_after_77", "kind": "prefill", "batch": 1, "tokens": 300, "past": 77, "heads": 32, "kv_heads": 32},
        # a long prompt before its cache is cut
        {"name": "prefill_1x4096", "kind": "prefill", "batch": 1, "tokens": 4096, "past": 0, "heads": 32, "kv_heads": 8},
        # a decode step of one sequence
        {"name": "decode_1x2048", "kind": "decode", "batch": 1, "length": 2048, "heads": 32, "kv_heads": 8, "channels": 128,
         "ragged": False},
        # ... of a ragged batch on long caches
        {"name": "decode_16x4000_ragged", "kind": "decode", "batch": 16, "length": 4000, "heads": 32, "kv_heads": 8, "channels": 128,
         "ragged": True},
        # one sequence cut to half its cache, a few layers at once
        {"name": "evict_1x1100_to_512", "kind": "evict", "batch": 1, "length": 1100, "budget": 512, "recent": 64, "layers": 4,
         "kv_heads": 8, "channels": 128, "ragged": False},
        # a batch of long sequences, all layers of the model
        {"name": "evict_4x4000_to_2048", "kind": "evict", "batch": 4, "length": 4000, "budget": 2048, "recent": 256, "layers": 32,
         "kv_heads": 8, "channels": 128, "ragged": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("tree", "tree", "tree", "commit", "prefill", "decode", "decode", "evict"))
    heads, kv_heads, channels = rng.choice(((32, 8, 128), (32, 32, 128), (32, 8, 64), (16, 16, 64), (64, 8, 128), (12, 4, 128)))
    if kind == "tree":
        length = _log_int(rng, 1, 8192)
        batch = _log_int(rng, 1, max(1, min(32, 65536 // (length * kv_heads // 8 or 1))))
        return {"kind": kind, "batch": batch, "nodes": _log_int(rng, 1, 64), "length": length, "heads": heads,
                "kv_heads": kv_heads, "channels": channels, "ragged": rng.random() < 0.5, "per_sequence": rng.random() < 0.5}
    if kind == "commit":
        return {"kind": kind, "batch": _log_int(rng, 1, 16), "nodes": _log_int(rng, 1, 64), "length": _log_int(rng, 16, 900),
                "layers": rng.randint(1, 32), "kv_heads": min(kv_heads, 16), "channels": channels}
    if kind == "prefill":
        tokens, past = _log_int(rng, 2, 4096), rng.choice((0, _log_int(rng, 1, 2048)))
        heads, kv_heads = rng.choice(((32, 8), (32, 32), (12, 4)))
        batch = _log_int(rng, 1, max(1, min(8, 4096 * 4096 // (tokens * (tokens + 2 * past)))))
        return {"kind": kind, "batch": batch, "tokens": tokens, "past": past, "heads": heads, "kv_heads": kv_heads}
    if kind == "decode":
        length = _log_int(rng, 1, 8192)
        batch = _log_int(rng, 1, max(1, min(32, 65536 // (length * kv_heads // 8 or 1))))
        return {"kind": kind, "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads, "channels": channels,
                "ragged": rng.random() < 0.5}
    length = _log_int(rng, 64, 4096)
    budget = max(2, int(length * rng.uniform(0.25, 0.9)))
    kv_heads = min(kv_heads, 8)
    return {"kind": kind, "batch": _log_int(rng, 1, 4), "length": length, "budget": budget, "recent": rng.randint(0, budget // 2),
            "layers": rng.randint(1, 32), "kv_heads": kv_heads, "channels": channels, "ragged": rng.random() < 0.5}


# ---------------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """Slots taken of each sequence: all `length`, or from there down to half of it."""
    n, b = case["length"], case["batch"]
    return [n - (n * i // (2 * b) if case.get("ragged", True) else 0) for i in range(b)]


def _normal(gen, *shape, scale=1.0):
    return torch.empty(shape, device=DEVICE, dtype=torch.float16).normal_(0.0, scale, generator=gen)


def _slots(case):
    """Slots of a cache: what the case needs, rounded up as a server allocates them."""
    need = case["past"] + case["tokens"] if case["kind"] == "prefill" else case["length"] + case.get("nodes", 0)
    return -(-need // 256) * 256


def _weights(gen, *shape, scale=1.0):
    """Running sums of attention weights: a few positions have most of it."""
    return torch.empty(shape, device=DEVICE).log_normal_(math.log(scale), 1.5, generator=gen)


def _random_trees(gen, trees, nodes):
    """Parents of `trees` random trees: node 0 is the root, a node's parent has a lower index."""
    u = torch.rand(trees, nodes, device=DEVICE, generator=gen)
    index = torch.arange(nodes, device=DEVICE)
    parents = (u * index).long()
    parents[:, 0] = -1
    return parents


def _ancestors(parents):
    """[..., T, T] bool: whether node j is node i or above it."""
    t = parents.size(-1)
    index = torch.arange(t, device=DEVICE)
    child = (parents[..., :, None] == index) & (index < index[:, None])
    step = child.double() + torch.eye(t, device=DEVICE, dtype=torch.float64)
    return torch.linalg.matrix_power(step, t) > 0


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, b, g = case["kind"], case["batch"], case["kv_heads"]
    d, slots = case.get("channels", 128), _slots(case)
    state = {"case": case}
    if kind in ("commit", "evict"):
        state["keys"] = _normal(gen, case["layers"], b, g, slots, d)
        state["values"] = _normal(gen, case["layers"], b, g, slots, d)
        state["layers"] = list(state["keys"]), list(state["values"])   # the caches as a model holds them
    else:
        state["keys"], state["values"] = _normal(gen, b, g, slots, d), _normal(gen, b, g, slots, d)
        # a few positions that most queries look at
        state["keys"][:, :, :: max(2, slots // 16)] *= 2.0
    if kind != "prefill":
        state["lengths"] = torch.tensor(_lengths(case), device=DEVICE)
    if kind == "tree":
        t = case["nodes"]
        state["q"] = _normal(gen, b, t, case["heads"], d, scale=2.0)
        state["k"], state["v"] = _normal(gen, b, t, g, d), _normal(gen, b, t, g, d)
        parents = _random_trees(gen, b if case["per_sequence"] else 1, t)
        seen = _ancestors(parents)
        state["mask"] = (seen if case["per_sequence"] else seen[0]).contiguous()
        depth = seen.sum(-1) - 1
        positions = (state["lengths"][:, None] + depth).double()
        angles = positions[..., None] / 10000.0 ** (torch.arange(0, d, 2, device=DEVICE, dtype=torch.float64) / d)
        angles = torch.cat((angles, angles), -1)
        state["cos"], state["sin"] = angles.cos().half(), angles.sin().half()
    elif kind == "commit":
        t = case["nodes"]
        # a binary tree level by level; the model agrees with a random branch of it down to some level
        parents = (torch.arange(t, device=DEVICE) - 1) // 2
        parents[0] = -1
        state["parents"] = parents.expand(b, t).contiguous()
        state["tokens"] = torch.arange(t, device=DEVICE) + 1000 * torch.randint(1, 100, (b, 1), device=DEVICE, generator=gen)
        state["chosen"] = torch.randint(200000, 300000, (b, t), device=DEVICE, generator=gen)
        leaf = torch.tensor([2 ** (n - 1) - 1 for n in _accepted(case)], device=DEVICE)
        leaf = leaf + (torch.rand(b, device=DEVICE, generator=gen) * torch.minimum(leaf + 1, t - leaf)).long()
        seen = _ancestors(parents)[leaf]                               # the branch of each sequence
        agreed = seen & (torch.arange(t, device=DEVICE) > 0)
        at = parents.clamp(min=0).expand(b, t)
        spare = torch.cat((state["chosen"], torch.zeros(b, 1, dtype=torch.int64, device=DEVICE)), 1)
        spare.scatter_(1, torch.where(agreed, at, t), state["tokens"])
        state["chosen"] = spare[:, :t].contiguous()
    elif kind == "prefill":
        state["q"] = _normal(gen, b, case["tokens"], case["heads"], d, scale=2.0)
        state["weights"] = _weights(gen, b, g, slots)
    elif kind == "decode":
        state["q"] = _normal(gen, b, case["heads"], d, scale=2.0)
        state["weights"] = _weights(gen, b, g, slots, scale=1e-3)     # (few steps so far)
    else:
        state["weights"] = _weights(gen, case["layers"], b, g, slots)
    return state


def _accepted(case):
    """How many nodes of each sequence's tree the model agrees with: from the root alone to the deepest full level."""
    levels = (case["nodes"] + 1).bit_length() - 1
    return [1 + (5 * i + levels - 1) % levels for i in range(case["batch"])]


# ---------------------------------------------------------------------------------------------------- the plain forms
def _rotate(x, cos, sin):
    half = x.size(-1) // 2
    turned = torch.cat((-x[..., half:], x[..., :half]), -1)
    return x * cos.float()[:, :, None] + turned * sin.float()[:, :, None]


def _softmax(scores, seen):
    """Probabilities over the last axis where `seen`; rows that see nothing are zero."""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    return e / e.sum(-1, keepdim=True).clamp(min=1e-30)


def _tree_plain(s):
    case, keys, values = s["case"], s["keys"], s["values"]
    b, t, heads, d = s["q"].shape
    g, n = keys.size(1), case["length"] + case["nodes"]
    rows = torch.arange(b, device=DEVICE)[:, None]
    places = s["lengths"][:, None] + torch.arange(t, device=DEVICE)
    keys[rows, :, places] = _rotate(s["k"].float(), s["cos"], s["sin"]).half()
    values[rows, :, places] = s["v"]
    q = _rotate(s["q"].float(), s["cos"], s["sin"]).view(b, t, g, heads // g, d).permute(0, 2, 1, 3, 4).reshape(b * g, -1, d)
    k = keys[:, :, :n].float().transpose(2, 3).reshape(b * g, d, n)
    scores = (torch.bmm(q, k) * d ** -0.5).view(b, g, t, heads // g, n)
    slot = torch.arange(n, device=DEVICE)
    node = slot - s["lengths"][:, None]                                # [b, n]: the node in a slot
    mask = s["mask"].expand(b, t, t)
    in_tree = torch.gather(mask, 2, node.clamp(0, t - 1)[:, None].expand(b, t, n))
    seen = (node < 0)[:, None] | (in_tree & ((node >= 0) & (node < t))[:, None])
    p = _softmax(scores, seen[:, None, :, None])
    out = torch.bmm(p.view(b * g, -1, n), values[:, :, :n].float().reshape(b * g, n, d))
    out = out.view(b, g, t, heads // g, d).permute(0, 2, 1, 3, 4).reshape(b, t, heads * d)
    return {"out": out.half(), "keys": keys, "values": values}


def _commit_plain(s):
    tokens, parents, chosen = s["tokens"], s["parents"], s["chosen"]
    keys, values = s["keys"], s["values"]
    b, t = tokens.shape
    index = torch.arange(t, device=DEVICE)
    up = parents.clamp(min=0)
    agrees = (tokens == torch.gather(chosen, 1, up)) | (index == 0)
    # of children with one parent and one token, the first counts
    twin = (parents[:, :, None] == parents[:, None]) & (tokens[:, :, None] == tokens[:, None]) & (index < index[:, None])
    agrees = agrees & ~twin.any(-1)
    on_path = (agrees[:, None] | ~_ancestors(parents)).all(-1)
    accepted = on_path.sum(1)
    path = torch.sort(torch.where(on_path, index, t), 1).values
    taken = index < accepted[:, None]
    last = torch.gather(path, 1, accepted[:, None] - 1)
    rows = torch.arange(b, device=DEVICE)[:, None]
    to = s["lengths"][:, None] + index
    source = s["lengths"][:, None] + torch.where(taken, path, index)
    keys[:, rows, :, to] = keys[:, rows, :, source]
    values[:, rows, :, to] = values[:, rows, :, source]
    return {"path": torch.where(taken, path, -1), "accepted": accepted, "next": torch.gather(chosen, 1, last)[:, 0],
            "lengths": s["lengths"] + accepted, "keys": keys, "values": values}


def _attention_plain(s, seen):
    """Attention of q [b, t, heads, d] over the first slots of the caches, and the sums of each slot's probabilities."""
    q, keys, values, n = s["q"], s["keys"], s["values"], seen.size(-1)
    q = q if q.dim() == 4 else q[:, None]
    b, t, heads, d = q.shape
    g = keys.size(1)
    q = q.float().view(b, t, g, heads // g, d).permute(0, 2, 1, 3, 4).reshape(b * g, -1, d)
    k = keys[:, :, :n].float().transpose(2, 3).reshape(b * g, d, n)
    p = _softmax((torch.bmm(q, k) * d ** -0.5).view(b, g, t, heads // g, n), seen[:, None, :, None])
    out = torch.bmm(p.view(b * g, -1, n), values[:, :, :n].float().reshape(b * g, n, d))
    out = out.view(b, g, t, heads // g, d).permute(0, 2, 1, 3, 4).reshape(b, t, heads * d)
    s["weights"][:, :, :n] += p.sum((2, 3))
    return out.half()


def _prefill_plain(s):
    t, past = s["case"]["tokens"], s["case"]["past"]
    seen = torch.arange(past + t, device=DEVICE) <= past + torch.arange(t, device=DEVICE)[:, None]
    return {"out": _attention_plain(s, seen[None]), "weights": s["weights"]}


def _decode_plain(s):
    seen = torch.arange(s["case"]["length"], device=DEVICE) < s["lengths"][:, None]
    return {"out": _attention_plain(s, seen[:, None]).view(s["q"].shape), "weights": s["weights"]}


def _evict_plain(s):
    case, keys, values, weights, lengths = s["case"], s["keys"], s["values"], s["weights"], s["lengths"]
    budget, n = case["budget"], case["length"]
    slot = torch.arange(n, device=DEVICE)
    latest = (slot >= lengths[:, None] - case["recent"])[:, None]
    taken = (slot < lengths[:, None])[:, None]
    order = torch.where(latest, math.inf, weights[..., :n])
    order = torch.where(taken, order, -math.inf)
    best = torch.sort(order, dim=-1, descending=True, stable=True).indices[..., :budget]
    best = torch.where(lengths[:, None, None] > budget, torch.sort(best, -1).values, slot[:budget])
    held = slot[:budget] < lengths[:, None, None]
    at = best[..., None].expand(*best.shape, keys.size(-1))
    keys[..., :budget, :] = torch.gather(keys, 3, at)
    values[..., :budget, :] = torch.gather(values, 3, at)
    left = torch.zeros_like(weights)
    left[..., :budget] = torch.where(held, torch.gather(weights, 3, best), 0.0)
    return {"kept": torch.where(held, best, -1), "weights": left, "lengths": lengths.clamp(max=budget), "keys": keys, "values": values}


_PLAIN = {"tree": _tree_plain, "commit": _commit_plain, "prefill": _prefill_plain, "decode": _decode_plain, "evict": _evict_plain}


# ---------------------------------------------------------------------------------------------------- the library's operators
def _library(s):
    import flh_amd
    ops = flh_amd._CUDA
    case, keys, values = s["case"], s["keys"], s["values"]
    kind = case["kind"]
    if kind == "tree":
        out = ops.tree_attention(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["lengths"], s["mask"], keys, values)
        return {"out": out, "keys": keys, "values": values}
    if kind == "commit":
        path, accepted, token, lengths = ops.tree_commit_(s["tokens"], s["parents"], s["chosen"], s["lengths"], *s["layers"])
        return {"path": path, "accepted": accepted, "next": token, "lengths": lengths, "keys": keys, "values": values}
    if kind == "prefill":
        return {"out": ops.prefill_attention_weights(s["q"], keys, values, case["past"], s["weights"]), "weights": s["weights"]}
    if kind == "decode":
        return {"out": ops.decode_attention_weights(s["q"], keys, values, s["lengths"], s["weights"]), "weights": s["weights"]}
    kept, weights, lengths = ops.evict_kv_cache_(*s["layers"], s["weights"], s["lengths"], case["budget"], case["recent"])
    return {"kept": kept, "weights": weights, "lengths": lengths, "keys": keys, "values": values}


def run(state):
    with torch.no_grad():
        return _library(state) if own else _PLAIN[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------------------- what it cannot do without
def work(case):
    kind, b, g, d = case["kind"], case["batch"], case["kv_heads"], case.get("channels", 128)
    if kind == "prefill":
        t, past, heads = case["tokens"], case["past"], case["heads"]
        pairs = t * past + t * (t + 1) / 2
        # queries and output, every cached row once, the sums read and written; two products and one to find the weights again
        return {"bytes": b * (4 * t * heads * d + (past + t) * g * (4 * d + 8)), "flops": b * 6 * d * heads * pairs}
    lengths = _lengths(case)
    if kind == "decode":
        return {"bytes": sum(lengths) * g * (4 * d + 8) + 4 * b * case["heads"] * d, "flops": 4 * d * case["heads"] * sum(lengths)}
    if kind == "tree":
        t, heads = case["nodes"], case["heads"]
        # cached rows and new ones read, new ones written; queries and output; the rotary rows and the mask
        moved = 4 * d * g * (sum(lengths) + 2 * b * t) + 4 * b * t * heads * d + 4 * b * t * d + t * t
        return {"bytes": moved, "flops": 4 * d * heads * t * sum(n + t for n in lengths)}
    row = 2 * 2 * case["layers"] * g * d                               # a position's keys and values in all layers
    if kind == "commit":
        return {"bytes": sum(2 * row * (n - 1) + 8 * 4 * case["nodes"] + 24 for n in _accepted(case)), "flops": 0}
    cut = [n for n in lengths if n > case["budget"]]
    sums = 4 * case["layers"] * g
    return {"bytes": sum(2 * row * case["budget"] + sums * n for n in cut) + sums * b * _slots(case)
            + 8 * case["layers"] * b * g * case["budget"], "flops": 0}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def _exact_attention(q, k, v, seen):
    """softmax(q k^T / sqrt(d)) v of one key / value head: q [r, d], k / v [n, d], seen [r, n] -> (out, probabilities)."""
    scores = (q @ k.t()) / math.sqrt(q.size(-1))
    scores.masked_fill_(~seen, -math.inf)
    p = torch.softmax(scores, -1).nan_to_num(0.0)
    return p @ v, p


def _exact_rotate(x, cos, sin):
    first, second = x.double().chunk(2, -1)
    c, s = cos.double(), sin.double()
    h = first.size(-1)
    return torch.cat((first * c[..., :h] - second * s[..., :h], second * c[..., h:] + first * s[..., h:]), -1)


def exact(case, seed):
    s = prepare(case, seed)
    kind, keys, values = case["kind"], s["keys"], s["values"]
    if kind == "tree":
        b, t, heads, d = s["q"].shape
        rep = heads // keys.size(1)
        out = torch.zeros(b, t, heads, d, dtype=torch.float64, device=DEVICE)
        for i, n in enumerate(_lengths(case)):
            cos, sin = s["cos"][i][:, None], s["sin"][i][:, None]
            keys[i, :, n:n + t] = _exact_rotate(s["k"][i], cos, sin).half().transpose(0, 1)
            values[i, :, n:n + t] = s["v"][i].transpose(0, 1)
            q = _exact_rotate(s["q"][i], cos, sin)
            tree = s["mask"][i] if case["per_sequence"] else s["mask"]
            seen = torch.cat((torch.ones(t, n, dtype=torch.bool, device=DEVICE), tree), 1)
            for h in range(heads):
                k, v = keys[i, h // rep, :n + t].double(), values[i, h // rep, :n + t].double()
                out[i, :, h] = _exact_attention(q[:, h], k, v, seen)[0]
        return {"out": out.view(b, t, heads * d), "keys": keys, "values": values}
    if kind == "commit":
        tokens, parents, chosen = (s[x].tolist() for x in ("tokens", "parents", "chosen"))
        t = case["nodes"]
        paths, last = [], []
        for i in range(case["batch"]):
            path = [0]
            while True:
                found = [c for c in range(path[-1] + 1, t) if parents[i][c] == path[-1] and tokens[i][c] == chosen[i][path[-1]]]
                if not found:
                    break
                path.append(found[0])
            start = _lengths(case)[i]
            at = [start + x for x in path]
            for cache in (keys, values):
                cache[:, i, :, start:start + len(path)] = cache[:, i][:, :, at].clone()
            paths.append(path + [-1] * (t - len(path)))
            last.append(chosen[i][path[-1]])
        accepted = [sum(x >= 0 for x in p) for p in paths]
        whole = [torch.tensor(x, device=DEVICE) for x in (paths, accepted, last, [n + a for n, a in zip(_lengths(case), accepted)])]
        return dict(zip(("path", "accepted", "next", "lengths"), whole), keys=keys, values=values)
    if kind in ("prefill", "decode"):
        q = s["q"] if kind == "prefill" else s["q"][:, None]
        b, t, heads, d = q.shape
        rep = heads // keys.size(1)
        lengths = [case["past"] + t] * b if kind == "prefill" else _lengths(case)
        out = torch.zeros(b, t, heads, d, dtype=torch.float64, device=DEVICE)
        weights = s["weights"].double()
        for i, n in enumerate(lengths):
            seen = torch.ones(t, n, dtype=torch.bool, device=DEVICE).tril(n - t)
            for h in range(heads):
                k, v = keys[i, h // rep, :n].double(), values[i, h // rep, :n].double()
                out[i, :, h], p = _exact_attention(q[i, :, h].double(), k, v, seen)
                weights[i, h // rep, :n] += p.sum(0)
        return {"out": out.reshape(b, t, heads * d) if kind == "prefill" else out[:, 0], "weights": weights}
    budget, recent = case["budget"], case["recent"]
    kept = torch.full((case["layers"], case["batch"], case["kv_heads"], budget), -1, device=DEVICE)
    weights = torch.zeros_like(s["weights"], dtype=torch.float64)
    for i, n in enumerate(_lengths(case)):
        m = min(n, budget)
        if n > budget:
            old = s["weights"][:, i, :, :n - recent].double()
            best = torch.argsort(-old, dim=-1, stable=True)[..., :budget - recent]
            best = torch.cat((best.sort(-1).values, torch.arange(n - recent, n, device=DEVICE).expand(*best.shape[:-1], recent)), -1)
        else:
            best = torch.arange(n, device=DEVICE).expand(case["layers"], case["kv_heads"], n)
        kept[:, i, :, :m] = best
        weights[:, i, :, :m] = s["weights"][:, i].double().gather(-1, best)
        at = best[..., None].expand(*best.shape, keys.size(-1))
        for cache in (keys, values):
            cache[:, i, :, :m] = cache[:, i].gather(2, at)
    return {"kept": kept, "weights": weights, "lengths": s["lengths"].clamp(max=budget), "keys": keys, "values": values}

"""Measured cases of the cache operators: attention of a tree of drafted tokens over a cache, the accepted path and its
commit, attention that accumulates each cached row's weight, and eviction of the rows with the least of it.

``run`` computes a case in its plain form (elementary torch operations in 32 bits, rounded once at the end), or, where
``own`` is true, by the framework's operators. ``exact`` restates each from its definition in 64 bits, sequence by
sequence."""

import math

import torch

own = False

VOCAB = 151936  # the vocabulary of the decoder that the framework runs


def listed():
    return [
        # One user's decoder (16 query heads over 8 key-value heads of 128, a cache of 640 rows) verifying 8 drafted
        # tokens: the smallest call, where latency counts.
        {"name": "tree_one_user", "op": "tree_attention", "batch": 1, "nodes": 8, "q_heads": 16, "kv_heads": 8,
         "head_dim": 128, "length": 600, "capacity": 640, "ragged": False, "packed": False},
        # A served batch of the same decoder: ragged lengths, an odd number of nodes, K and V halves of one tensor.
        {"name": "tree_served_batch", "op": "tree_attention", "batch": 8, "nodes": 33, "q_heads": 16, "kv_heads": 8,
         "head_dim": 128, "length": 4000, "capacity": 4099, "ragged": True, "packed": True},
        # Wide trees over long contexts with eight query heads to a key-value head: 512 rows a head, matrix bound.
        {"name": "tree_wide_long", "op": "tree_attention", "batch": 4, "nodes": 64, "q_heads": 32, "kv_heads": 4,
         "head_dim": 128, "length": 32000, "capacity": 32768, "ragged": True, "packed": False},
        # Verification of one user's drafts: the walk alone.
        {"name": "accept_one_user", "op": "tree_accept", "batch": 1, "nodes": 8, "ragged": False},
        # Verification for a large served batch with wide trees.
        {"name": "accept_large_batch", "op": "tree_accept", "batch": 256, "nodes": 256, "ragged": True},
        # One layer's cache rows of one user's accepted path moved behind the committed ones.
        {"name": "commit_one_user", "op": "tree_commit", "batch": 1, "nodes": 8, "kv_heads": 8, "head_dim": 128,
         "length": 600, "capacity": 640, "ragged": False, "packed": False},
        # The same for a large served batch, long accepted paths.
        {"name": "commit_large_batch", "op": "tree_commit", "batch": 64, "nodes": 64, "kv_heads": 8, "head_dim": 128,
         "length": 500, "capacity": 700, "ragged": True, "packed": True},
        # One decode step of one user with the weights accumulated: a single token, latency.
        {"name": "weights_one_token", "op": "attention_weights", "batch": 1, "tokens": 1, "q_heads": 16, "kv_heads": 8,
         "head_dim": 128, "length": 600, "capacity": 640, "ragged": False, "packed": False},
        # One decode step of a served batch over long ragged caches: bound by reading K and V once.
        {"name": "weights_decode_batch", "op": "attention_weights", "batch": 16, "tokens": 1, "q_heads": 16,
         "kv_heads": 8, "head_dim": 128, "length": 16384, "capacity": 16400, "ragged": True, "packed": False},
        # A prompt of 2000 tokens from an empty cache, whose weights decide what an eviction keeps: matrix bound.
        {"name": "weights_prompt", "op": "attention_weights", "batch": 2, "tokens": 2000, "q_heads": 16,
         "kv_heads": 8, "head_dim": 128, "length": 0, "capacity": 2048, "ragged": True, "packed": False},
        # One user's cache cut from 2000 rows to 512 after the prompt.
        {"name": "evict_one_user", "op": "cache_evict", "batch": 1, "kv_heads": 8, "head_dim": 128, "length": 2000,
         "capacity": 2048, "keep": 512, "recent": 64, "sinks": 4, "ragged": False, "packed": False},
        # A served batch of long caches cut to 2048 rows each.
        {"name": "evict_served_batch", "op": "cache_evict", "batch": 16, "kv_heads": 8, "head_dim": 128,
         "length": 16384, "capacity": 16400, "keep": 2048, "recent": 256, "sinks": 4, "ragged": True, "packed": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["tree_attention", "tree_attention", "tree_accept", "tree_commit", "attention_weights",
                     "attention_weights", "cache_evict", "cache_evict"])
    ragged, packed = rng.random() < 0.6, rng.random() < 0.4
    if op == "tree_accept":
        return {"op": op, "batch": _log_int(rng, 1, 256), "nodes": _log_int(rng, 2, 256), "ragged": ragged}
    q_heads, kv_heads = rng.choice([(16, 8), (16, 8), (8, 8), (32, 8), (12, 4), (14, 2), (16, 1), (6, 2)])
    head_dim = rng.choice([64, 128, 128, 256])
    row = kv_heads * head_dim  # elements of one cached row; the largest listed cases hold 2^28 of them
    if op == "tree_attention":
        nodes = _log_int(rng, 1, 200)
        rows = _log_int(rng, 16, 32000)
        batch = _log_int(rng, 1, max(1, min(32, (1 << 25) // (row * rows), (1 << 19) // (q_heads * nodes),
                                            (1 << 27) // (nodes * q_heads * rows))))
        return {"op": op, "batch": batch, "nodes": nodes, "q_heads": q_heads, "kv_heads": kv_heads,
                "head_dim": head_dim, "length": rows, "capacity": rows + nodes + rng.randrange(0, 64),
                "ragged": ragged, "packed": packed}
    if op == "tree_commit":
        nodes, rows = _log_int(rng, 2, 200), _log_int(rng, 16, 1000)
        batch = _log_int(rng, 1, max(1, min(64, (1 << 25) // (row * (rows + nodes)))))
        return {"op": op, "batch": batch, "nodes": nodes, "kv_heads": kv_heads, "head_dim": head_dim, "length": rows,
                "capacity": rows + nodes + rng.randrange(0, 64), "ragged": ragged, "packed": packed}
    if op == "attention_weights":
        tokens = rng.choice([1, 1, _log_int(rng, 2, 64), _log_int(rng, 64, 1500)])
        rows = _log_int(rng, 16, 16000) if tokens < 64 else _log_int(rng, 1, 500)
        batch = _log_int(rng, 1, max(1, min(32, (1 << 25) // (row * rows),
                                            (1 << 26) // (tokens * q_heads * (rows + tokens)))))
        return {"op": op, "batch": batch, "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads,
                "head_dim": head_dim, "length": rows, "capacity": rows + tokens + rng.randrange(0, 64),
                "ragged": ragged, "packed": packed}
    rows = _log_int(rng, 64, 16000)
    batch = _log_int(rng, 1, max(1, min(32, (1 << 25) // (row * rows))))
    keep = max(8, int(rows * rng.uniform(0.1, 0.6)))
    recent = rng.randrange(0, keep // 2)
    return {"op": op, "batch": batch, "kv_heads": kv_heads, "head_dim": head_dim, "length": rows,
            "capacity": rows + rng.randrange(0, 64), "keep": keep, "recent": recent, "sinks": rng.randrange(0, 5),
            "ragged": ragged, "packed": packed}


# ---- inputs --------------------------------------------------------------------------------------------------------


def _lengths(case, g, longest, shortest=0):
    """Row counts of the batch: all the longest, or spread from a third of it up to it, the first the longest."""
    b = case["batch"]
    if not case["ragged"] or b == 1:
        return torch.full((b,), longest, dtype=torch.int64, device="cuda")
    low = max(shortest, longest // 3)
    n = torch.randint(low, longest + 1, (b,), generator=g, device="cuda")
    n[0] = longest
    return n


def _caches(case, g, topic):
    """K and V [batch, capacity, kv_heads, head_dim] in bf16, every row written once (rows past a sequence's end are
    what an earlier one left). One row in 32 and the first follow the topic that the queries share, so that attention
    has rows of heavy weight, as a trained model's has."""
    b, n, h, d = case["batch"], case["capacity"], case["kv_heads"], case["head_dim"]
    both = torch.empty((b, n, 2, h, d) if case["packed"] else (2, b, n, h, d), dtype=torch.bfloat16, device="cuda")
    k, v = (both[:, :, 0], both[:, :, 1]) if case["packed"] else (both[0], both[1])
    k.normal_(generator=g)
    v.normal_(generator=g)
    heavy = torch.rand((b, n, 1, 1), generator=g, device="cuda") < 1 / 32
    heavy[:, 0] = True
    k.add_(heavy * topic.to(torch.bfloat16))
    return k, v


def _queries(case, g, topic, tokens):
    h, d = case["q_heads"], case["head_dim"]
    q = torch.randn((case["batch"], tokens, h, d), generator=g, device="cuda")
    return (q + 2.0 * topic.repeat_interleave(h // case["kv_heads"], 0)).to(torch.bfloat16)


def _topic(case, g):
    return torch.randn((case["kv_heads"], case["head_dim"]), generator=g, device="cuda")


def _parents(case, g):
    """A drafted tree each: node 0 is its root, most nodes continue a recent node, some branch off anywhere."""
    b, t = case["batch"], case["nodes"]
    index = torch.arange(t, device="cuda").expand(b, t)
    near = index - 1 - torch.randint(0, 3, (b, t), generator=g, device="cuda")
    far = (torch.rand((b, t), generator=g, device="cuda") * index).long()
    p = torch.where(torch.rand((b, t), generator=g, device="cuda") < 0.8, near.clamp(min=0), far)
    p = torch.minimum(p, (index - 1).clamp(min=0))
    p[:, 0] = -1
    return p


def _ancestors(parents):
    """[batch, t, t], true where the second node is the first one or above it."""
    b, t = parents.shape
    see = torch.eye(t, dtype=torch.bool, device=parents.device).expand(b, t, t).clone()
    for i in range(1, t):
        see[:, i] |= torch.gather(see, 1, parents[:, i].view(b, 1, 1).expand(b, 1, t))[:, 0]
    return see


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op = case["op"]
    state = {"case": case}
    if op == "tree_attention":
        topic = _topic(case, g)
        state["k"], state["v"] = _caches(case, g, topic)
        state["q"] = _queries(case, g, topic, case["nodes"])
        state["lengths"] = _lengths(case, g, case["length"])
        state["mask"] = _ancestors(_parents(case, g))
        state["nodes"] = _lengths(case, g, case["nodes"], 1)
    elif op == "tree_accept":
        b, t = case["batch"], case["nodes"]
        parents = _parents(case, g)
        predicted = torch.randint(0, VOCAB, (b, t), generator=g, device="cuda")
        drafted = torch.randint(0, VOCAB, (b, t), generator=g, device="cuda")
        right = torch.gather(predicted, 1, parents.clamp(min=0))
        hit = torch.rand((b, t), generator=g, device="cuda") < 0.7
        state |= {"tokens": torch.where(hit, right, drafted), "parents": parents, "predicted": predicted,
                  "nodes": _lengths(case, g, t, 1)}
    elif op == "tree_commit":
        topic = _topic(case, g)
        state["k"], state["v"] = _caches(case, g, topic)
        state["lengths"] = _lengths(case, g, case["length"])
        b, t = case["batch"], case["nodes"]
        pick = torch.rand((b, t), generator=g, device="cuda") < 0.25
        pick[:, 0] = True
        index = torch.arange(t, device="cuda").expand(b, t)
        path = torch.where(pick, index, t).sort(1).values
        state["path"] = torch.where(path < t, path, -1)
        state["counts"] = pick.sum(1)
    elif op == "attention_weights":
        topic = _topic(case, g)
        state["k"], state["v"] = _caches(case, g, topic)
        state["q"] = _queries(case, g, topic, case["tokens"])
        state["lengths"] = _lengths(case, g, case["length"])
        state["counts"] = _lengths(case, g, case["tokens"], 1)
        state["weights"] = torch.rand((case["batch"], case["kv_heads"], case["capacity"]), generator=g, device="cuda")
    else:
        state["k"], state["v"] = _caches(case, g, _topic(case, g))
        state["lengths"] = _lengths(case, g, case["length"])
        w = torch.rand((case["batch"], case["kv_heads"], case["capacity"]), generator=g, device="cuda").log_().neg_()
        state["weights"] = torch.where(w < 0.02, 0.0, w * w)  # a long tail, and rows that nothing attended to
    return state


# ---- the operators ---------------------------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from cppinf_b200 import ops

        if op == "tree_attention":
            return ops.tree_attention(state["q"], state["k"], state["v"], state["lengths"], state["mask"],
                                      state["nodes"])
        if op == "tree_accept":
            return ops.tree_accept(state["tokens"], state["parents"], state["predicted"], state["nodes"])
        if op == "tree_commit":
            ops.tree_commit(state["k"], state["v"], state["lengths"], state["path"], state["counts"])
            return state["k"], state["v"]
        if op == "attention_weights":
            ctx = ops.decoder_attention_weights(state["q"], state["k"], state["v"], state["lengths"],
                                                state["weights"], state["counts"])
            return ctx, state["weights"]
        return ops.cache_evict(state["k"], state["v"], state["weights"], state["lengths"], case["keep"],
                               case["recent"], case["sinks"])
    if op == "tree_attention":
        return _tree_attention(**{n: state[n] for n in ("q", "k", "v", "lengths", "mask", "nodes")})
    if op == "tree_accept":
        return _tree_accept(state["tokens"], state["parents"], state["predicted"], state["nodes"])
    if op == "tree_commit":
        _tree_commit(state["k"], state["v"], state["lengths"], state["path"], state["counts"])
        return state["k"], state["v"]
    if op == "attention_weights":
        ctx = _attention_weights(state["q"], state["k"], state["v"], state["lengths"], state["weights"],
                                 state["counts"])
        return ctx, state["weights"]
    return _cache_evict(state["k"], state["v"], state["weights"], state["lengths"], case["keep"], case["recent"],
                        case["sinks"])


def _attention(q, k, v, see, used):
    """Probabilities [b, kv_heads, t, group, rows] and the context in 32 bits. see [b, t, rows]: the rows that a query
    sees; used [b, rows]: rows that hold anything."""
    b, t, hq, d = q.shape
    n, h = k.shape[1], k.shape[2]
    g = hq // h
    qf = q.float().view(b, t, h, g, d).permute(0, 2, 1, 3, 4).reshape(b, h, t * g, d)
    s = torch.matmul(qf, k.float().permute(0, 2, 3, 1)).view(b, h, t, g, n) * (1.0 / math.sqrt(d))
    s = torch.where(see[:, None, :, None, :], s, -torch.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -torch.inf, 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-38)
    vf = torch.where(used[:, :, None, None], v.float(), 0.0).permute(0, 2, 1, 3)
    ctx = torch.matmul(p.view(b, h, t * g, n), vf).view(b, h, t, g, d)
    return p, ctx.permute(0, 2, 1, 3, 4).reshape(b, t, hq, d)


def _tree_attention(q, k, v, lengths, mask, nodes):
    b, t = q.shape[:2]
    at = torch.arange(k.shape[1], device=q.device) - lengths[:, None]  # node that a row holds, or below 0
    drafted = torch.gather(mask, 2, at.clamp(0, t - 1)[:, None, :].expand(b, t, -1))
    inside = torch.arange(t, device=q.device) < nodes[:, None]
    see = ((at < 0)[:, None, :] | (drafted & ((at >= 0) & (at < nodes[:, None]))[:, None, :])) & inside[:, :, None]
    return _attention(q, k, v, see, at < nodes[:, None])[1].to(torch.bfloat16)


def _attention_weights(q, k, v, lengths, weights, counts):
    t = q.shape[1]
    at = torch.arange(k.shape[1], device=q.device) - lengths[:, None]
    token = torch.arange(t, device=q.device)
    see = (at[:, None, :] <= token[:, None]) & (token < counts[:, None])[:, :, None]
    p, ctx = _attention(q, k, v, see, at < counts[:, None])
    weights.add_(p.sum((2, 3)))
    return ctx.to(torch.bfloat16)


def _tree_accept(tokens, parents, predicted, nodes):
    b, t = tokens.shape
    index = torch.arange(t, device=tokens.device).expand(b, t)
    above = parents.clamp(0, t - 1)
    fits = (tokens == torch.gather(predicted, 1, above)) & (parents >= 0) & (parents < index) & (index < nodes[:, None])
    lowest = torch.full((b, t), t, dtype=torch.int64, device=tokens.device).scatter_reduce(
        1, above, torch.where(fits, index, t), "amin")
    taken = (fits & (torch.gather(lowest, 1, above) == index)) | ((index == 0) & (nodes[:, None] > 0))
    above = torch.where(index == 0, 0, above)
    for _ in range(max(1, (t - 1).bit_length())):  # every node's ancestors, twice as far up each time
        taken = taken & torch.gather(taken, 1, above)
        above = torch.gather(above, 1, above)
    path = torch.where(taken, index, t).sort(1).values
    path = torch.where(path < t, path, -1)
    counts = taken.sum(1)
    last = torch.gather(path, 1, (counts - 1).clamp(min=0)[:, None])
    following = torch.where(counts > 0, torch.gather(predicted, 1, last.clamp(min=0))[:, 0], -1)
    return path, counts, following


def _tree_commit(k, v, lengths, path, counts):
    b, t = path.shape
    index = torch.arange(t, device=path.device)
    to = lengths[:, None] + index
    source = torch.where(index < counts[:, None], lengths[:, None] + path, to)
    one = torch.arange(b, device=path.device)[:, None]
    k[one, to] = k[one, source]
    v[one, to] = v[one, source]


def _cache_evict(k, v, weights, lengths, keep, recent, sinks):
    b, n, h, d = k.shape
    row = torch.arange(n, device=k.device)
    inside = (row < lengths[:, None])[:, None, :]
    fixed = ((row < sinks) | (row >= lengths[:, None] - recent))[:, None, :]
    rank = torch.where(inside, torch.where(fixed, torch.inf, weights), -torch.inf)
    kept = rank.sort(dim=-1, descending=True, stable=True).indices[:, :, :keep].sort(-1).values
    left = lengths.clamp(max=keep)
    valid = (torch.arange(keep, device=k.device) < left[:, None])[:, None, :].expand(b, h, keep)
    at = kept.permute(0, 2, 1)[..., None].expand(b, keep, h, d)
    there = valid.permute(0, 2, 1)[..., None]
    k_out = torch.where(there, torch.gather(k, 1, at), 0.0)
    v_out = torch.where(there, torch.gather(v, 1, at), 0.0)
    return (k_out, v_out, torch.where(valid, torch.gather(weights, 2, kept), 0.0), left,
            torch.where(valid, kept, -1))


# ---- 64 bits ---------------------------------------------------------------------------------------------------------


def _exact_sequence(q, k, v, allowed):
    """One sequence: q [t, hq, d], k and v [rows, h, d], allowed [t, rows]; its context and each head's weights."""
    t, hq, d = q.shape
    h = k.shape[1]
    ctx = torch.zeros((t, hq, d), dtype=torch.float64, device=q.device)
    weights = torch.zeros((h, k.shape[0]), dtype=torch.float64, device=q.device)
    for head in range(hq):
        of = head // (hq // h)
        s = q[:, head].double() @ k[:, of].double().T / math.sqrt(d)
        e = torch.softmax(s.masked_fill(~allowed, -math.inf), 1)
        e = e.masked_fill(~allowed.any(1, keepdim=True), 0.0)
        ctx[:, head] = e @ v[:, of].double()
        weights[of] += e.sum(0)
    return ctx, weights


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "tree_attention":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for i, (n, m) in enumerate(zip(s["lengths"].tolist(), s["nodes"].tolist())):
            allowed = torch.cat([torch.ones((m, n), dtype=torch.bool, device="cuda"), s["mask"][i, :m, :m]], 1)
            out[i, :m] = _exact_sequence(s["q"][i, :m], s["k"][i, :n + m], s["v"][i, :n + m], allowed)[0]
        return out
    if op == "attention_weights":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        weights = s["weights"].double()
        for i, (n, m) in enumerate(zip(s["lengths"].tolist(), s["counts"].tolist())):
            allowed = torch.ones((m, n + m), dtype=torch.bool, device="cuda").tril(n)
            out[i, :m], w = _exact_sequence(s["q"][i, :m], s["k"][i, :n + m], s["v"][i, :n + m], allowed)
            weights[i, :, :n + m] += w
        return out, weights
    if op == "tree_accept":
        t = case["nodes"]
        paths, counts, following = [], [], []
        for tokens, parents, predicted, n in zip(*(s[x].tolist() for x in ("tokens", "parents", "predicted", "nodes"))):
            at, path = 0, [0]
            while True:
                fit = [c for c in range(at + 1, n) if parents[c] == at and tokens[c] == predicted[at]]
                if not fit:
                    break
                at = fit[0]
                path.append(at)
            paths.append(path + [-1] * (t - len(path)))
            counts.append(len(path))
            following.append(predicted[at])
        return torch.tensor(paths), torch.tensor(counts), torch.tensor(following)
    if op == "tree_commit":
        k, v = s["k"].double(), s["v"].double()
        for i, (n, m) in enumerate(zip(s["lengths"].tolist(), s["counts"].tolist())):
            rows = [n + p for p in s["path"][i, :m].tolist()]
            k[i, n:n + m], v[i, n:n + m] = k[i, rows], v[i, rows]
        return k, v
    keep, recent, sinks = case["keep"], case["recent"], case["sinks"]
    b, _, h, d = s["k"].shape
    k, v = (torch.zeros((b, keep, h, d), dtype=torch.float64, device="cuda") for _ in "kv")
    weights = torch.zeros((b, h, keep), dtype=torch.float64, device="cuda")
    index = torch.full((b, h, keep), -1, dtype=torch.int64, device="cuda")
    for i, n in enumerate(s["lengths"].tolist()):
        for head in range(h):
            w = s["weights"][i, head, :n]
            if n <= keep:
                rows = torch.arange(n, device="cuda")
            else:
                order = torch.sort(w[sinks:n - recent].double(), descending=True, stable=True).indices
                rows = torch.cat([torch.arange(sinks, device="cuda"), sinks + order[:keep - sinks - recent],
                                  torch.arange(n - recent, n, device="cuda")]).sort().values
            m = len(rows)
            index[i, head, :m] = rows
            weights[i, head, :m] = w[rows].double()
            k[i, :m, head], v[i, :m, head] = s["k"][i, rows, head].double(), s["v"][i, rows, head].double()
    return k, v, weights, s["lengths"].clamp(max=keep), index


def work(case):
    """Ragged lengths count with their mean, two thirds of the longest."""
    op, b = case["op"], case["batch"]
    share = 2 / 3 if case["ragged"] and b > 1 else 1.0
    if op == "tree_accept":
        return {"bytes": b * case["nodes"] * 8 * 4, "flops": 0}
    h, d = case["kv_heads"], case["head_dim"]
    if op == "tree_commit":
        return {"bytes": b * (case["nodes"] * 8 + 2 * 2 * (0.25 * case["nodes"] + 0.75) * h * d * 2), "flops": 0}
    if op == "cache_evict":
        rows, kept = share * case["length"], min(case["keep"], share * case["length"])
        return {"bytes": b * h * (4 * rows + kept * (2 * 2 * 2 * d + 4 + 8)), "flops": 0}
    t, hq = case["nodes" if op == "tree_attention" else "tokens"], case["q_heads"]
    n, m = share * case["length"], share * t if t > 1 else 1
    bytes_ = b * (2 * 2 * h * d * (n + m) + 2 * 2 * t * hq * d)
    if op == "tree_attention":
        return {"bytes": bytes_ + b * t * t, "flops": 4 * b * m * hq * d * n}
    return {"bytes": bytes_ + b * 2 * 4 * h * (n + m), "flops": 4 * b * hq * d * m * (n + (m + 1) / 2)}

"""The cache operators on the device (tree attention, accept, commit, attention weights, eviction) against a plain
restatement in 64 bits.

Tolerances, with u = 2^-24. A score is an f32 sum of D products times a factor: it is off by at most
e = (D + 3) u sum|q_i k_i| / sqrt(D) for any order of the sum, twice that where the adder truncates, which is what is
granted. A probability p_j then is off by a factor within exp(2 * 2e) (numerator and sum move apart), and by a few u for
the exponential and the sum: |dp_j| <= p_j (4.5 e + 2^-18), while 4e stays below 0.1.
- A weight is the sum of its probabilities, added up in f32 to what was there: off by at most
  sum p_j (4.5 e + 2^-18) + (rows + 2) u (w0 + sum p_j).
- A context may be formed from probabilities rounded to bf16 (half a step, 2^-8 each) and is rounded to bf16 itself:
  off by at most A (4.5 e + 2^-18 + 2^-8) + 2^-8 |ctx| (with the products of the two), A = sum_j p_j |v_j|.
"""

from __future__ import annotations

import math
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def ops(cuda):
    from cppinf_b200 import ops as _ops

    return _ops


def reference(q, k, v, lengths, counts, see, capacity):
    """Context, its bound, weights and their bound. see(b) -> bool [n, n] over a sequence's new tokens."""
    batch, tokens, hq, d = q.shape
    h = k.shape[2]
    ctx = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(ctx)
    weights = torch.zeros((batch, h, capacity), dtype=torch.float64, device=q.device)
    w_bound = torch.zeros_like(weights)
    for b in range(batch):
        n, m = lengths[b], counts[b]
        if m == 0:
            continue
        allowed = torch.cat([torch.ones((m, n), dtype=torch.bool, device=q.device), see(b)[:m, :m]], 1)
        for head in range(hq):
            of = head // (hq // h)
            kk, vv = k[b, :n + m, of].double(), v[b, :n + m, of].double()
            qq = q[b, :m, head].double()
            s = qq @ torch.nan_to_num(kk, 0, 0, 0).T / math.sqrt(d)
            size = qq.abs() @ torch.nan_to_num(kk, 0, 0, 0).abs().T / math.sqrt(d)
            e = 2 * (d + 3) * U * torch.where(allowed, size, 0.0).amax(1, keepdim=True)
            assert float(e.max()) < 0.025, "scores too large for the bound to hold"
            p = torch.softmax(s.masked_fill(~allowed, -math.inf), 1).masked_fill(~allowed, 0.0)
            p = p.masked_fill(~allowed.any(1, keepdim=True), 0.0)
            vz = torch.nan_to_num(vv, 0, 0, 0)
            ctx[b, :m, head] = p @ vz
            a = p @ vz.abs()
            rel = 4.5 * e + 2.0 ** -18
            off = a * (rel + 2.0 ** -8 * (1 + rel))
            bound[b, :m, head] = off + 2.0 ** -8 * (ctx[b, :m, head].abs() + off) + 2.0 ** -126
            weights[b, of, :n + m] += p.sum(0)
            w_bound[b, of, :n + m] += (p * rel).sum(0)
    return ctx, bound, weights, w_bound


def caches(g, batch, capacity, heads, d, layout, dtype=torch.bfloat16):
    """K and V, in one of the memory orders that the operators read in place (or copy: 'shifted')."""
    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    if layout == "packed":
        both = rand(batch, capacity, 2, heads, d)
        return both[:, :, 0], both[:, :, 1]
    if layout == "heads_first":
        return rand(batch, heads, capacity, d).transpose(1, 2), rand(batch, heads, capacity, d).transpose(1, 2)
    if layout == "layer":
        both = rand(2, 3, batch, capacity, heads, d)
        return both[0, 1], both[1, 2]
    if layout == "shifted":
        return rand(batch, capacity, heads, d + 4)[..., :d], rand(batch, capacity, heads, d + 4)[..., 4:]
    return rand(batch, capacity, heads, d), rand(batch, capacity, heads, d)


def spoil(cache, lengths, counts):
    """Fills the rows that no query sees with NaN and infinities."""
    for b in range(cache.shape[0]):
        end = lengths[b] + counts[b]
        cache[b, end:] = math.nan
        cache[b, end::2] = math.inf


def tree_masks(batch, tokens, g):
    parents = [[-1] + [int(torch.randint(max(0, i - 4), i, (1,), generator=g)) for i in range(1, tokens)]
               for _ in range(batch)]
    mask = torch.zeros((batch, tokens, tokens), dtype=torch.bool)
    for b in range(batch):
        for i in range(tokens):
            j = i
            while j >= 0:
                mask[b, i, j] = True
                j = parents[b][j]
    return mask.cuda()


# batch, tokens, query heads, kv heads, head dim, committed rows, valid nodes (None: all), layout
TREES = [
    (1, 1, 16, 8, 128, [0], None, "dense"),
    (1, 1, 16, 8, 128, [600], None, "dense"),
    (1, 8, 16, 8, 128, [127], None, "dense"),
    (2, 9, 16, 8, 128, [128, 119], [9, 4], "packed"),
    (3, 5, 8, 8, 64, [0, 1, 300], [5, 0, 1], "dense"),
    (2, 33, 14, 2, 64, [500, 33], [33, 20], "heads_first"),
    (2, 17, 6, 2, 256, [255, 90], [17, 17], "packed"),
    (1, 64, 12, 4, 256, [1000], None, "layer"),
    (1, 128, 16, 8, 128, [1025], [100], "dense"),
    (2, 100, 16, 1, 128, [700, 20], [100, 37], "dense"),
    (1, 256, 32, 4, 128, [300], None, "dense"),
    (1, 256, 2, 2, 64, [63], [255], "shifted"),
    (2, 3, 128, 1, 128, [2000, 129], None, "dense"),
    (3, 7, 5, 5, 64, [3000, 10, 1537], [7, 6, 2], "layer"),
    (1, 2, 10, 2, 256, [5000], None, "heads_first"),
    (1, 1, 32, 1, 128, [30000], None, "dense"),
    (1, 2, 8, 1, 64, [20000], None, "dense"),
    (1, 3, 4, 1, 256, [9000], [2], "dense"),
]


@pytest.mark.parametrize("batch,tokens,hq,h,d,lengths,nodes,layout", TREES)
def test_tree_attention(ops, batch, tokens, hq, h, d, lengths, nodes, layout):
    g = torch.Generator(device="cuda").manual_seed(tokens * 131 + d)
    host = torch.Generator().manual_seed(tokens)
    counts = nodes or [tokens] * batch
    capacity = max(lengths) + tokens + 3
    k, v = caches(g, batch, capacity, h, d, layout)
    spoil(k, lengths, counts)
    spoil(v, lengths, counts)
    q = torch.randn((batch, tokens, hq, d), generator=g, device="cuda").bfloat16()
    mask = tree_masks(batch, tokens, host)
    n = torch.tensor(lengths, device="cuda")
    m = None if nodes is None else torch.tensor(nodes, device="cuda")
    got = ops.tree_attention(q, k, v, n, mask, m)
    ctx, bound, _, _ = reference(q, k, v, lengths, counts, lambda b: mask[b], capacity)
    assert got.dtype == torch.bfloat16 and torch.isfinite(got).all()
    assert ((got.double() - ctx).abs() <= bound).all()
    for b in range(batch):
        assert (got[b, counts[b]:] == 0).all()
    assert torch.equal(got, ops.tree_attention(q, k, v, n, mask, m)), "two calls give the same bits"


def test_tree_attention_shared_mask_and_rows_that_see_nothing(ops):
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn((3, 6, 8, 128), generator=g, device="cuda").bfloat16()
    k, v = caches(g, 3, 200, 2, 128, "dense")
    mask = torch.rand((6, 6), generator=g, device="cuda") < 0.5
    mask[2] = False
    lengths = [0, 150, 0]
    n = torch.tensor(lengths, device="cuda")
    got = ops.tree_attention(q, k, v, n, mask)
    ctx, bound, _, _ = reference(q, k, v, lengths, [6, 6, 6], lambda b: mask, 200)
    assert ((got.double() - ctx).abs() <= bound).all()
    assert (got[0, 2] == 0).all() and (got[2, 2] == 0).all()
    each = mask.expand(3, 6, 6).contiguous()
    assert torch.equal(got, ops.tree_attention(q, k, v, n, each))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("tokens", [6, 140])
def test_tree_attention_keeps_masked_nodes_values_out(ops, tokens, d):
    """A drafted row of NaN or infinities reaches the nodes that see it and no other."""
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn((1, tokens, 4, d), generator=g, device="cuda").bfloat16()
    k, v = caches(g, 1, 512, 2, d, "dense")
    n = torch.tensor([250], device="cuda")
    mask = torch.eye(tokens, dtype=torch.bool, device="cuda")
    mask[:, 0] = True
    clean = ops.tree_attention(q, k, v, n, mask)
    k[0, 250 + 3], v[0, 250 + 3] = math.nan, math.nan
    v[0, 250 + 4, 1, 5] = math.inf
    got = ops.tree_attention(q, k, v, n, mask)
    others = [t for t in range(tokens) if t not in (3, 4)]
    assert torch.equal(got[:, others], clean[:, others])
    assert torch.isnan(got[0, 3]).all()
    assert torch.equal(got[0, 4, :2], clean[0, 4, :2])  # the other key-value head
    assert (got[0, 4, 2:, 5] == math.inf).all()
    keep = [i for i in range(d) if i != 5]
    assert torch.equal(got[0, 4, 2:][:, keep], clean[0, 4, 2:][:, keep])


def test_tree_attention_nan_in_a_seen_row_and_in_a_query(ops):
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randn((1, 3, 4, 128), generator=g, device="cuda").bfloat16()
    k, v = caches(g, 1, 512, 2, 128, "dense")
    n = torch.tensor([400], device="cuda")
    mask = torch.ones((3, 3), dtype=torch.bool, device="cuda")
    clean = ops.tree_attention(q, k, v, n, mask)
    q[0, 1, 2, 7] = math.nan
    got = ops.tree_attention(q, k, v, n, mask)
    assert torch.isnan(got[0, 1, 2]).all()
    got[0, 1, 2] = clean[0, 1, 2]
    assert torch.equal(got, clean)
    v[0, 10, 0, 3] = math.inf
    got = ops.tree_attention(q, k, v, n, mask)
    assert not torch.isfinite(got[0, [0, 2], :2, 3]).any()
    assert torch.equal(got[0, :, 3], clean[0, :, 3])


@pytest.mark.parametrize("tokens,rows", [(2, 3000), (150, 3000)])
def test_a_nan_query_stays_nan_through_the_join(ops, tokens, rows):
    """Rows whose key tiles several CTAs take: a NaN query gives NaN, an infinite score too, and no other row does."""
    g = torch.Generator(device="cuda").manual_seed(16)
    q = torch.randn((1, tokens, 4, 128), generator=g, device="cuda").bfloat16()
    k, v = caches(g, 1, rows + tokens, 2, 128, "dense")
    n = torch.tensor([rows], device="cuda")
    w = torch.zeros((1, 2, rows + tokens), device="cuda")
    clean = ops.decoder_attention_weights(q, k, v, n, w)
    q[0, 0, 1] = math.nan
    got = ops.decoder_attention_weights(q, k, v, n, w.zero_())
    assert torch.isnan(got[0, 0, 1]).all() and torch.isnan(w[0, 0, :rows + 1]).all() and torch.isfinite(w[0, 1]).all()
    got[0, 0, 1] = clean[0, 0, 1]
    assert torch.equal(got, clean)
    q[0, 0, 1] = 1.0
    k[0, rows // 2, 0] = math.inf
    got = ops.decoder_attention_weights(q, k, v, n, w.zero_())
    assert torch.isnan(got[0, 0, 1]).all()


def test_new_rows_past_the_capacity_are_padding(ops):
    g = torch.Generator(device="cuda").manual_seed(6)
    q = torch.randn((3, 8, 4, 64), generator=g, device="cuda").bfloat16()
    k, v = caches(g, 3, 100, 2, 64, "dense")
    mask = torch.ones((8, 8), dtype=torch.bool, device="cuda").tril()
    got = ops.tree_attention(q, k, v, torch.tensor([97, 1 << 40, -5], device="cuda"), mask)
    same = ops.tree_attention(q, k, v, torch.tensor([97, 100, 0], device="cuda"), mask,
                              torch.tensor([3, 0, 8], device="cuda"))
    assert torch.equal(got, same)
    assert (got[0, 3:] == 0).all() and (got[1] == 0).all() and (got[0, :3] != 0).any()
    w = torch.zeros((3, 2, 100), device="cuda")
    ctx = ops.decoder_attention_weights(q, k, v, torch.tensor([97, 1 << 40, -5], device="cuda"), w)
    assert torch.equal(ctx, got)
    assert torch.allclose(w.sum(2).cpu(), torch.tensor([6.0, 0.0, 16.0])[:, None].expand(3, 2), rtol=1e-5)


# batch, tokens, query heads, kv heads, head dim, committed rows, valid queries (None: all), layout
WEIGHTS = [
    (1, 1, 16, 8, 128, [0], None, "dense"),
    (1, 1, 16, 8, 128, [639], None, "dense"),
    (3, 1, 8, 8, 64, [127, 128, 5], [1, 1, 0], "packed"),
    (2, 1, 14, 2, 256, [4000, 777], None, "layer"),
    (2, 1, 64, 1, 128, [1500, 3], None, "dense"),
    (2, 7, 16, 8, 128, [121, 122], [7, 3], "heads_first"),
    (1, 64, 12, 4, 128, [65], None, "dense"),
    (1, 65, 16, 1, 64, [1], None, "dense"),
    (2, 200, 16, 8, 128, [0, 57], [200, 131], "packed"),
    (1, 513, 6, 2, 256, [10], None, "shifted"),
    (1, 1100, 4, 2, 128, [0], [1099], "dense"),
    (2, 700, 5, 5, 64, [300, 0], None, "dense"),
]


@pytest.mark.parametrize("batch,tokens,hq,h,d,lengths,counts,layout", WEIGHTS)
def test_decoder_attention_weights(ops, batch, tokens, hq, h, d, lengths, counts, layout):
    g = torch.Generator(device="cuda").manual_seed(tokens * 31 + d)
    valid = counts or [tokens] * batch
    capacity = max(lengths) + tokens + 2
    k, v = caches(g, batch, capacity, h, d, layout)
    spoil(k, lengths, valid)
    spoil(v, lengths, valid)
    q = torch.randn((batch, tokens, hq, d), generator=g, device="cuda").bfloat16()
    n = torch.tensor(lengths, device="cuda")
    m = None if counts is None else torch.tensor(counts, device="cuda")
    w0 = torch.rand((batch, h, capacity), generator=g, device="cuda")
    w = w0.clone()
    got = ops.decoder_attention_weights(q, k, v, n, w, m)
    causal = torch.ones((tokens, tokens), dtype=torch.bool, device="cuda").tril()
    ctx, bound, weights, w_bound = reference(q, k, v, lengths, valid, lambda b: causal, capacity)
    assert torch.isfinite(got).all() and torch.isfinite(w).all()
    assert ((got.double() - ctx).abs() <= bound).all()
    rows = tokens * (hq // h)
    assert ((w.double() - w0.double() - weights).abs() <= w_bound + (rows + 2) * U * (w0 + weights)).all()
    for b in range(batch):
        assert torch.equal(w[b, :, lengths[b] + valid[b]:], w0[b, :, lengths[b] + valid[b]:])
        assert (got[b, valid[b]:] == 0).all()
    again = w0.clone()
    assert torch.equal(got, ops.decoder_attention_weights(q, k, v, n, again, m))
    assert torch.equal(w, again), "two calls add the same bits"


@pytest.mark.parametrize("tokens", [4, 150])
def test_weights_keep_later_tokens_values_out(ops, tokens):
    """A NaN in the last token's key and value reaches the last query alone."""
    g = torch.Generator(device="cuda").manual_seed(8)
    q = torch.randn((1, tokens, 4, 128), generator=g, device="cuda").bfloat16()
    k, v = caches(g, 1, 400, 2, 128, "dense")
    n = torch.tensor([100], device="cuda")
    clean = ops.decoder_attention_weights(q, k, v, n, torch.zeros((1, 2, 400), device="cuda"))
    k[0, 100 + tokens - 1, 0] = math.nan
    v[0, 100 + tokens - 1] = math.nan
    w = torch.zeros((1, 2, 400), device="cuda")
    got = ops.decoder_attention_weights(q, k, v, n, w)
    assert torch.equal(got[:, :-1], clean[:, :-1])
    assert torch.isnan(got[:, -1]).all()
    assert torch.isnan(w[0, 0, :100 + tokens]).all() and torch.isfinite(w[0, 1]).all()
    assert (w[0, :, 100 + tokens:] == 0).all()


def test_weights_of_one_token_equal_those_of_the_batch(ops):
    """Token by token and all at once: the same context and the same weights within their bounds."""
    g = torch.Generator(device="cuda").manual_seed(9)
    tokens, d = 12, 128
    q = torch.randn((2, tokens, 8, d), generator=g, device="cuda").bfloat16()
    k, v = caches(g, 2, 64, 4, d, "dense")
    n = torch.tensor([20, 31], device="cuda")
    w = torch.zeros((2, 4, 64), device="cuda")
    whole = ops.decoder_attention_weights(q, k, v, n, w)
    w1 = torch.zeros_like(w)
    parts = [ops.decoder_attention_weights(q[:, t:t + 1].contiguous(), k, v, n + t, w1) for t in range(tokens)]
    causal = torch.ones((tokens, tokens), dtype=torch.bool, device="cuda").tril()
    _, bound, weights, w_bound = reference(q, k, v, [20, 31], [tokens, tokens], lambda b: causal, 64)
    assert ((whole.double() - torch.cat(parts, 1).double()).abs() <= 2 * bound).all()
    assert ((w.double() - w1.double()).abs() <= 2 * w_bound + 2 * (tokens * 2 + tokens + 2) * U * weights).all()


# ---- accept and commit ----------------------------------------------------------------------------------------------


def walk(tokens, parents, predicted, n):
    path = [0] if n > 0 else []
    while path:
        fit = [c for c in range(path[-1] + 1, n) if parents[c] == path[-1] and tokens[c] == predicted[path[-1]]]
        if not fit:
            break
        path.append(fit[0])
    return path, predicted[path[-1]] if path else -1


@pytest.mark.parametrize("batch,tokens,nodes", [(1, 1, None), (1, 8, None), (5, 33, [33, 0, 1, 20, 33]),
                                                (4, 256, [256, 255, 200, 3]), (300, 65, None), (2, 32, [99, -4])])
def test_tree_accept(ops, batch, tokens, nodes):
    g = torch.Generator().manual_seed(batch + tokens)
    parents = torch.stack([torch.tensor([-1] + [int(torch.randint(max(0, i - 3), i, (1,), generator=g))
                                                for i in range(1, tokens)]) for _ in range(batch)])
    predicted = torch.randint(0, 3, (batch, tokens), generator=g)
    ids = torch.randint(0, 3, (batch, tokens), generator=g)  # few tokens: repeated drafts and long paths
    if tokens > 4:
        parents[0, 4] = 4  # its own parent
        parents[0, 2] = 4  # a parent after its child
        parents[0, 3] = 1 << 40
    m = None if nodes is None else torch.tensor(nodes).cuda()
    path, counts, following = ops.tree_accept(ids.cuda(), parents.cuda(), predicted.cuda(), m)
    for b in range(batch):
        n = tokens if nodes is None else min(max(nodes[b], 0), tokens)
        want, token = walk(ids[b].tolist(), parents[b].tolist(), predicted[b].tolist(), n)
        assert path[b].tolist() == want + [-1] * (tokens - len(want))
        assert int(counts[b]) == len(want) and int(following[b]) == token


def test_tree_accept_without_nodes(ops):
    none = torch.empty((3, 0), dtype=torch.int64, device="cuda")
    path, counts, following = ops.tree_accept(none, none, none)
    assert path.shape == (3, 0) and counts.tolist() == [0, 0, 0] and following.tolist() == [-1, -1, -1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,tokens,h,d,layout", [(1, 8, 8, 128, "dense"), (3, 33, 2, 64, "packed"),
                                                     (2, 256, 1, 8, "heads_first"), (2, 100, 5, 256, "layer")])
def test_tree_commit(ops, batch, tokens, h, d, layout, dtype):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    lengths = [11 * b for b in range(batch)]
    k, v = caches(g, batch, tokens + 40, h, d, layout, dtype)
    index = torch.arange(tokens)
    path = torch.full((batch, tokens), -1)
    counts = torch.zeros(batch, dtype=torch.int64)
    for b in range(batch):
        pick = index[(torch.rand(tokens, generator=torch.Generator().manual_seed(b)) < 0.4) | (index == 0)]
        path[b, :len(pick)], counts[b] = pick, len(pick)
    counts[0] = 0 if batch > 1 else counts[0]
    want = []
    for cache in (k, v):
        w = cache.clone()
        for b in range(batch):
            n = int(counts[b])
            w[b, lengths[b]:lengths[b] + n] = cache[b, lengths[b] + path[b, :n].cuda()]
        want.append(w)
    ops.tree_commit(k, v, torch.tensor(lengths).cuda(), path.cuda(), counts.cuda())
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_tree_commit_skips_what_lies_outside(ops):
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = caches(g, 3, 20, 2, 64, "dense")
    before = k.clone()
    path = torch.tensor([[0, 3, 9, 5], [2, -7, 1, 3], [1, 2, 3, 1 << 40]]).cuda()
    ops.tree_commit(k, v, torch.tensor([2, 5, 18]).cuda(), path, torch.tensor([9, 3, 4]).cuda())
    want = before.clone()
    want[0, 3] = before[0, 5]    # row 1 takes node 3; 9 and 5 are no nodes
    want[1, 5] = before[1, 7]    # row 0 takes node 2; -7 and 1 break the order
    want[2, 18] = before[2, 19]  # rows 18 and 19 alone lie inside the cache
    assert torch.equal(k, want)


# ---- eviction --------------------------------------------------------------------------------------------------------


def kept_rows(w, n, keep, recent, sinks):
    if n <= keep:
        return list(range(n))
    middle = range(sinks, n - recent)
    order = sorted(middle, key=lambda i: (w[i] != w[i], -w[i] if w[i] == w[i] else 0.0, i))
    return sorted(list(range(sinks)) + order[:keep - sinks - recent] + list(range(n - recent, n)))


# batch, heads, head dim, capacity, lengths, keep, recent, sinks, output capacity, layout
EVICTIONS = [
    (1, 8, 128, 640, [640], 64, 16, 4, 64, "dense"),
    (3, 2, 64, 300, [300, 100, 101], 100, 30, 2, 120, "packed"),
    (2, 3, 64, 1500, [1025, 0], 1, 0, 0, 1, "dense"),
    (2, 3, 64, 1500, [1500, 1], 1, 1, 0, 3, "layer"),
    (2, 2, 256, 2100, [2049, 1024], 1024, 0, 0, 1024, "heads_first"),
    (1, 2, 8, 40000, [39999], 20000, 100, 4, 20001, "dense"),
    (4, 1, 64, 50, [50, 49, 1 << 40, -3], 10, 6, 4, 10, "shifted"),
    (1, 1, 64, 5000, [5000], 4999, 10, 10, 5000, "dense"),
    (1, 4, 128, 9000, [9000], 3000, 100, 4, 3000, "dense"),
]


@pytest.mark.parametrize("kind", ["smooth", "ties", "special"])
@pytest.mark.parametrize("batch,h,d,capacity,lengths,keep,recent,sinks,out,layout", EVICTIONS)
def test_cache_evict(ops, batch, h, d, capacity, lengths, keep, recent, sinks, out, layout, kind):
    g = torch.Generator(device="cuda").manual_seed(capacity + keep)
    dtype = torch.float32 if layout == "heads_first" else torch.bfloat16
    k, v = caches(g, batch, capacity, h, d, layout, dtype)
    w = torch.rand((batch, h, capacity), generator=g, device="cuda") ** 8
    if kind == "ties":
        w = (w * 6).round()
    elif kind == "special":
        some = torch.randint(0, 8, w.shape, generator=g, device="cuda")
        for i, x in enumerate([0.0, -0.0, math.inf, -math.inf, math.nan, -1.0]):
            w[some == i] = x
    k2, v2, w2, left, index = ops.cache_evict(k, v, w, torch.tensor(lengths).cuda(), keep, recent, sinks, out)
    assert k2.shape == v2.shape == (batch, out, h, d) and w2.shape == (batch, h, out)
    for b in range(batch):
        n = min(max(lengths[b], 0), capacity)
        m = min(n, keep)
        assert int(left[b]) == m
        for head in range(h):
            rows = torch.tensor(kept_rows(w[b, head].tolist(), n, keep, recent, sinks), dtype=torch.int64).cuda()
            assert torch.equal(index[b, head, :m], rows) and (index[b, head, m:] == -1).all()
            assert torch.equal(k2[b, :m, head], k[b, rows, head]) and torch.equal(v2[b, :m, head], v[b, rows, head])
            assert torch.equal(w2[b, head, :m].view(torch.int32), w[b, head, rows].view(torch.int32))
        assert not k2[b, m:].any() and not v2[b, m:].any() and not w2[b, :, m:].any()


# ---- together --------------------------------------------------------------------------------------------------------


def test_prompt_eviction_and_drafted_steps_together(ops):
    """A prompt with weights, an eviction to a budget, then two rounds of drafted tokens: attention, accept, commit.
    Every context equals the plain one over the rows that were kept and committed."""
    g = torch.Generator(device="cuda").manual_seed(11)
    host = torch.Generator().manual_seed(11)
    batch, hq, h, d, prompt, keep, drafts = 2, 8, 4, 128, 300, 96, 12
    k, v = caches(g, batch, prompt, h, d, "dense")
    counts = [300, 211]
    w = torch.zeros((batch, h, prompt), device="cuda")
    q = torch.randn((batch, prompt, hq, d), generator=g, device="cuda").bfloat16()
    zero = torch.zeros(batch, dtype=torch.int64, device="cuda")
    n = torch.tensor(counts, device="cuda")
    ops.decoder_attention_weights(q, k, v, zero, w, n)
    assert torch.allclose(w.sum(2), (n * (hq // h))[:, None].float().expand(batch, h), rtol=1e-4)
    k2, v2, w2, n2, index = ops.cache_evict(k, v, w, n, keep, 32, 4, keep + 40)
    kept_k = [torch.stack([k[b, index[b, i], i] for i in range(h)], 1) for b in range(batch)]
    kept_v = [torch.stack([v[b, index[b, i], i] for i in range(h)], 1) for b in range(batch)]
    for step in range(2):
        mask = tree_masks(batch, drafts, host)
        new_k = torch.randn((batch, drafts, h, d), generator=g, device="cuda").bfloat16()
        new_v = torch.randn((batch, drafts, h, d), generator=g, device="cuda").bfloat16()
        for b in range(batch):
            k2[b, int(n2[b]):int(n2[b]) + drafts], v2[b, int(n2[b]):int(n2[b]) + drafts] = new_k[b], new_v[b]
        q = torch.randn((batch, drafts, hq, d), generator=g, device="cuda").bfloat16()
        got = ops.tree_attention(q, k2, v2, n2, mask)
        lengths = [len(x) for x in kept_k]
        assert lengths == n2.tolist()
        size = max(lengths) + drafts
        full_k, full_v = (torch.zeros((batch, size, h, d), dtype=torch.bfloat16, device="cuda") for _ in "kv")
        for b in range(batch):
            full_k[b, :lengths[b] + drafts] = torch.cat([kept_k[b], new_k[b]])
            full_v[b, :lengths[b] + drafts] = torch.cat([kept_v[b], new_v[b]])
        ctx, bound, _, _ = reference(q, full_k, full_v, lengths, [drafts] * batch, lambda b: mask[b], size)
        assert ((got.double() - ctx).abs() <= bound).all()
        parents = torch.full((batch, drafts), -1)
        for b in range(batch):
            for i in range(1, drafts):
                parents[b, i] = max(j for j in range(i) if mask[b, i, j])
        predicted = torch.randint(0, 2, (batch, drafts), generator=host)
        ids = torch.randint(0, 2, (batch, drafts), generator=host)
        path, accepted, _ = ops.tree_accept(ids.cuda(), parents.cuda(), predicted.cuda())
        ops.tree_commit(k2, v2, n2, path, accepted)
        n2 = n2 + accepted
        for b in range(batch):
            rows = path[b, :int(accepted[b])]
            assert rows.tolist() == walk(ids[b].tolist(), parents[b].tolist(), predicted[b].tolist(), drafts)[0]
            kept_k[b], kept_v[b] = torch.cat([kept_k[b], new_k[b, rows]]), torch.cat([kept_v[b], new_v[b, rows]])
            assert torch.equal(k2[b, :int(n2[b])], kept_k[b]) and torch.equal(v2[b, :int(n2[b])], kept_v[b])


def test_rotary_positions_of_a_tree_from_a_gathered_table(ops):
    """Nodes at one depth share a position: q/k norm + RoPE on a gathered table equals a call for each node."""
    from cppinf_b200 import capi

    g = torch.Generator(device="cuda").manual_seed(18)
    hq, h, d, length = 16, 8, 128, 77
    depth = torch.tensor([0, 1, 1, 2, 2, 3], device="cuda")
    n = len(depth)
    q = torch.randn((n, hq, d), generator=g, device="cuda").bfloat16()
    k = torch.randn((n, h, d), generator=g, device="cuda").bfloat16()
    wq, wk = (torch.randn(d, generator=g, device="cuda").bfloat16() for _ in "qk")
    table = ops.rope_table(1e6, d, length + 4)[length + depth].contiguous()
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    capi.call("cppinf_qk_norm_rope", capi.DTYPE_BF16, q.data_ptr(), k.data_ptr(), wq.data_ptr(), wk.data_ptr(),
              q_out.data_ptr(), k_out.data_ptr(), n, hq, h, d, 0, 1e-6, table.data_ptr(), n,
              torch.cuda.current_stream().cuda_stream)
    for t in range(n):
        want = ops.qk_norm_rope(q[t:t + 1], k[t:t + 1], wq, wk, 1e-6, length + int(depth[t]))
        assert torch.equal(q_out[t:t + 1], want[0]) and torch.equal(k_out[t:t + 1], want[1])


@pytest.mark.parametrize("capacity,tokens", [(700, 10), (5000, 10), (3000, 200)])
def test_captured_calls_follow_the_lengths(ops, capacity, tokens):
    """One graph of attention, accept, commit, weights and eviction, replayed for lengths and inputs that change."""
    g = torch.Generator(device="cuda").manual_seed(12)
    batch, hq, h, d = 2, 8, 2, 128
    k, v = caches(g, batch, capacity, h, d, "dense")
    q = torch.randn((batch, tokens, hq, d), generator=g, device="cuda").bfloat16()
    n = torch.tensor([600, 100], device="cuda")
    host = torch.Generator().manual_seed(12)
    mask = tree_masks(batch, tokens, host)
    ids = torch.randint(0, 2, (batch, tokens), generator=host).cuda()
    parents = torch.arange(-1, tokens - 1).expand(batch, tokens).contiguous().cuda()
    predicted = torch.randint(0, 2, (batch, tokens), generator=host).cuda()
    w = torch.zeros((batch, h, capacity), device="cuda")

    def step(kk, vv, ww):
        ctx = ops.tree_attention(q, kk, vv, n, mask)
        path, counts, following = ops.tree_accept(ids, parents, predicted)
        ops.tree_commit(kk, vv, n, path, counts)
        ctx2 = ops.decoder_attention_weights(q, kk, vv, n, ww)
        return (ctx, path, counts, following, ctx2, *ops.cache_evict(kk, vv, ww, n, 64, 16, 4))

    step(k.clone(), v.clone(), w.clone())  # everything loaded before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(k, v, w)
    for lengths in ([600, 100], [3, 0], [capacity - tokens, 333]):
        n.copy_(torch.tensor(lengths))
        q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
        w.zero_()
        want = step(k.clone(), v.clone(), w.clone())
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            assert torch.equal(x, y)


def test_empty_calls(ops):
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    cache = torch.zeros((0, 8, 2, 64), dtype=torch.bfloat16, device="cuda")
    q = torch.zeros((0, 3, 4, 64), dtype=torch.bfloat16, device="cuda")
    mask = torch.ones((3, 3), dtype=torch.bool, device="cuda")
    assert ops.tree_attention(q, cache, cache, none, mask).shape == q.shape
    assert ops.decoder_attention_weights(q, cache, cache, none, torch.zeros((0, 2, 8), device="cuda")).shape == q.shape
    ops.tree_commit(cache, cache, none, none.view(0, 0), none)
    assert ops.cache_evict(cache, cache, torch.zeros((0, 2, 8), device="cuda"), none, 4, 2)[0].shape == (0, 4, 2, 64)
    # no rows at all: every query is padding, every eviction keeps nothing
    cache = torch.zeros((2, 0, 2, 64), dtype=torch.bfloat16, device="cuda")
    q = torch.ones((2, 3, 4, 64), dtype=torch.bfloat16, device="cuda")
    n = torch.zeros(2, dtype=torch.int64, device="cuda")
    w = torch.zeros((2, 2, 0), device="cuda")
    assert not ops.tree_attention(q, cache, cache, n, mask).any()
    assert not ops.decoder_attention_weights(q, cache, cache, n, w).any()
    k2, v2, w2, left, index = ops.cache_evict(cache, cache, w, n, 4, 2)
    assert not k2.any() and not v2.any() and not w2.any() and left.tolist() == [0, 0] and (index == -1).all()
    # and no tokens
    cache = torch.zeros((2, 8, 2, 64), dtype=torch.bfloat16, device="cuda")
    assert ops.tree_attention(q[:, :0], cache, cache, n, mask[:0, :0]).shape == (2, 0, 4, 64)


@pytest.mark.parametrize("batch,tokens", [(700, 1), (300, 40)])
def test_many_short_sequences(ops, batch, tokens):
    """More sequences than a warp has lanes, lengths of every kind: each equals the sequence alone within its bound."""
    g = torch.Generator(device="cuda").manual_seed(17)
    h, d, capacity = 2, 64, 400
    k, v = caches(g, batch, capacity, h, d, "dense")
    q = torch.randn((batch, tokens, 2 * h, d), generator=g, device="cuda").bfloat16()
    n = torch.randint(0, capacity - tokens + 1, (batch,), generator=g, device="cuda")
    m = torch.randint(0, tokens + 1, (batch,), generator=g, device="cuda")
    w = torch.zeros((batch, h, capacity), device="cuda")
    got = ops.decoder_attention_weights(q, k, v, n, w, m)
    causal = torch.ones((tokens, tokens), dtype=torch.bool, device="cuda").tril()
    assert torch.equal(got, ops.tree_attention(q, k, v, n, causal, m))
    some = list(range(0, batch, 37))
    ctx, bound, weights, w_bound = reference(q[some], k[some], v[some], n[some].tolist(), m[some].tolist(),
                                             lambda b: causal, capacity)
    assert ((got[some].double() - ctx).abs() <= bound).all()
    assert ((w[some].double() - weights).abs() <= w_bound + (2 * tokens + 2) * U * weights).all()


def test_calls_on_two_streams_do_not_share_anything(ops):
    g = torch.Generator(device="cuda").manual_seed(13)
    sets = []
    for i in range(2):
        k, v = caches(g, 4, 3000, 4, 128, "dense")
        q = torch.randn((4, 5, 8, 128), generator=g, device="cuda").bfloat16()
        sets.append((q, k, v, torch.tensor([2900 - 700 * i] * 4, device="cuda"), torch.zeros((4, 4, 3000), device="cuda")))
    want = [ops.decoder_attention_weights(q, k, v, n, w.clone()) for q, k, v, n, w in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                q, k, v, n, w = sets[i]
                got[i].append(ops.decoder_attention_weights(q, k, v, n, w))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


@pytest.mark.parametrize("tokens,capacity", [(3, 500), (3, 4000), (150, 700)])
def test_waits_that_run_out_are_reported(ops, tokens, capacity):
    """With a poll limit of 0 every first wait gives up at once: the error word is set, the copies still land and the
    results stand; with the default limit it stays clear."""
    from cppinf_b200 import capi

    g = torch.Generator(device="cuda").manual_seed(14)
    k, v = caches(g, 2, capacity, 4, 128, "dense")
    q = torch.randn((2, tokens, 8, 128), generator=g, device="cuda").bfloat16()
    n = torch.full((2,), capacity - tokens, device="cuda")
    mask = torch.ones((tokens, tokens), dtype=torch.bool, device="cuda").tril()
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    w = torch.zeros((2, 4, capacity), device="cuda")
    ctx = ops.tree_attention(q, k, v, n, mask, error=error)
    ctx2 = ops.decoder_attention_weights(q, k, v, n, w, error=error)
    assert error.item() == 0
    previous = capi.set_wait_poll_limit(0)
    try:
        w2 = torch.zeros_like(w)
        got = ops.tree_attention(q, k, v, n, mask, error=error)
        assert error.item() == 1
        error.zero_()
        got2 = ops.decoder_attention_weights(q, k, v, n, w2, error=error)
        assert error.item() == 1
        ops.tree_attention(q, k, v, n, mask)  # nobody asked: nothing to report to
    finally:
        capi.set_wait_poll_limit(previous)
    assert torch.equal(got, ctx) and torch.equal(got2, ctx2) and torch.equal(w2, w)


def test_rows_past_32_bit_offsets(ops):
    """Caches of more than 2^31 elements: the rows that count lie at the end."""
    g = torch.Generator(device="cuda").manual_seed(15)
    h, d, tail = 8, 256, 300
    capacity = (1 << 31) // (h * d) + 2000
    cache = torch.zeros((1, capacity, h, d), dtype=torch.bfloat16, device="cuda")
    cache[:, -tail:] = torch.randn((1, tail, h, d), generator=g, device="cuda").bfloat16()
    q = torch.randn((1, 4, 16, d), generator=g, device="cuda").bfloat16()
    n = torch.tensor([capacity - 4], device="cuda")
    mask = torch.ones((4, 4), dtype=torch.bool, device="cuda").tril()
    got = ops.tree_attention(q, cache, cache, n, mask)
    w = torch.zeros((1, h, capacity), device="cuda")
    got2 = ops.decoder_attention_weights(q, cache, cache, n, w)
    assert torch.equal(got, got2)
    for head in (0, 15):
        rows = cache[0, -tail:, head // 2].double()
        s = q[0, :, head].double() @ rows.T / math.sqrt(d)
        s.masked_fill_(~torch.ones_like(s, dtype=torch.bool).tril(tail - 4), -math.inf)
        e = torch.exp(s - s.max(1, keepdim=True).values)
        others = torch.exp(-s.max(1, keepdim=True).values) * (capacity - tail)  # zero keys: score 0
        p = e / (e.sum(1, keepdim=True) + others)
        ctx = p @ rows
        off = (p @ rows.abs()) * (2.0 ** -8 + 2.0 ** -10)
        assert ((got[0, :, head].double() - ctx).abs() <= off + 2.0 ** -8 * ctx.abs()).all()
    total = w.double().sum(2)
    assert ((total - 8).abs() < 8 * 2.0 ** -12).all()  # probabilities of 4 queries and 2 heads; f32 sums of 2^20 parts
    k2, v2, w2, left, index = ops.cache_evict(cache, cache, w, n + 4, 64, 32)
    assert int(left) == 64
    for head in range(h):
        rows = index[0, head]
        assert (rows[1:] > rows[:-1]).all() and rows[-32:].tolist() == list(range(capacity - 32, capacity))
        rest = w[0, head, :capacity - 32]
        assert torch.equal(w2[0, head, :32].sort().values, rest.topk(32).values.sort().values)
        assert torch.equal(k2[0, :, head], cache[0, rows, head]) and torch.equal(v2[0, :, head], cache[0, rows, head])
    before = cache[0, -12:].clone()
    n = torch.tensor([capacity - 12], device="cuda")
    path = torch.tensor([[0, 3, 5]], device="cuda")
    ops.tree_commit(cache, cache.clone(), n, path, torch.tensor([3], device="cuda"))
    assert torch.equal(cache[0, -12:], before)  # of three nodes: 3 and 5 are none
    path = torch.tensor([[0, 3, 5, -1, -1, -1]], device="cuda")
    ops.tree_commit(cache, cache.clone(), n, path, torch.tensor([3], device="cuda"))
    before[1], before[2] = before[3].clone(), before[5].clone()
    assert torch.equal(cache[0, -12:], before)
    del cache
    torch.cuda.empty_cache()


def test_refusals_on_the_device(ops):
    t = torch.zeros((1, 8, 2, 64), dtype=torch.bfloat16, device="cuda")
    q = torch.zeros((1, 2, 4, 64), dtype=torch.bfloat16, device="cuda")
    n = torch.zeros(1, dtype=torch.int64, device="cuda")
    mask = torch.ones((2, 2), dtype=torch.bool, device="cuda")
    with pytest.raises(ValueError, match="int64 lengths"):
        ops.tree_attention(q, t, t, n.int(), mask)
    with pytest.raises(ValueError, match="int64 counts"):
        ops.tree_attention(q, t, t, n, mask, torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.tree_attention(q, t, t, n.cpu(), mask)
    with pytest.raises(ValueError, match="contiguous f32 weights"):
        ops.decoder_attention_weights(q, t, t, n, torch.zeros((1, 2, 9), device="cuda"))
    with pytest.raises(ValueError, match="divide by key/value heads"):
        ops.tree_attention(q[:, :, :3].contiguous(), t, t, n, mask)
    with pytest.raises(NotImplementedError, match="256 drafted"):
        big = torch.zeros((1, 257, 4, 64), dtype=torch.bfloat16, device="cuda")
        ops.tree_attention(big, t, t, n, torch.ones((257, 257), dtype=torch.bool, device="cuda"))
    with pytest.raises(ValueError, match="dense 16-byte aligned rows"):
        odd = torch.zeros((1, 8, 2, 68), dtype=torch.bfloat16, device="cuda")[..., :64]
        ops.tree_commit(odd, odd, n, torch.zeros((1, 2), dtype=torch.int64, device="cuda"), n)


@pytest.mark.parametrize("capacity", [8192, 10174, 10175, 10240, 12288])
def test_cache_evict_around_the_default_shared_memory(ops, capacity):
    """In a process of its own, whose first eviction it is: an earlier one of a longer cache raises the kernel's limit."""
    code = (
        "import torch\n"
        "from cppinf_b200 import ops\n"
        f"n = {capacity}\n"
        "g = torch.Generator(device='cuda').manual_seed(5)\n"
        "k = torch.randn(1, n, 1, 64, device='cuda', generator=g).bfloat16()\n"
        "w = torch.rand(1, 1, n, device='cuda', generator=g)\n"
        "out = ops.cache_evict(k, k, w, torch.tensor([n], device='cuda'), 64, 16)\n"
        "rows = w[0, 0, :n - 16].sort(descending=True, stable=True).indices[:48].sort().values\n"
        "assert torch.equal(out[4][0, 0, :48], rows)\n"
        "assert torch.equal(out[0][0, :48], k[0, rows])\n"
    )
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr


def test_commit_of_an_empty_cache(ops):
    k = torch.zeros(1, 0, 2, 64, dtype=torch.bfloat16, device="cuda")
    n = torch.zeros(1, dtype=torch.int64, device="cuda")
    ops.tree_commit(k, k.clone(), n, torch.zeros(1, 4, dtype=torch.int64, device="cuda"), n)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("tokens,group", [(10, 3), (150, 3), (150, 2), (90, 5)])
def test_weights_of_a_row_whose_scores_are_minus_infinity(ops, tokens, group, d):
    """Such a row counts for nothing, as does one of a very low score, in every query tile, those with unused rows too."""
    g = torch.Generator(device="cuda").manual_seed(tokens + d)
    q = torch.randn((1, tokens, 2 * group, d), generator=g, device="cuda").bfloat16()
    q[..., 0] = 1.0
    k, v = caches(g, 1, 300 + tokens, 2, d, "dense")
    n = torch.tensor([300], device="cuda")
    results = []
    for low in (-1e30, -math.inf):
        k[0, 20, :, 0] = low
        k[0, 300 + tokens // 2, :, 0] = low
        w = torch.ones((1, 2, 300 + tokens), device="cuda")
        results.append((ops.decoder_attention_weights(q, k, v, n, w), w))
    assert torch.isfinite(results[0][0]).all()
    assert torch.equal(results[0][0], results[1][0])
    assert torch.equal(results[0][1], results[1][1])
    assert (results[1][1][0, :, 20] == 1).all()


def check_weights_of_a_long_cache(ops, rows, group, tokens):
    """Weights of one key-value head over `rows` committed rows (K and V are one tensor) against the formula in 64 bits, a
    piece of the rows at a time. Besides the file's bounds, l is a long sum: a CTA adds two halves of each of its key
    tiles to it, 32 terms in a half's partial sums, and the parts of all CTAs are joined, with at least 100 CTAs at work and
    at most 160."""
    g = torch.Generator(device="cuda").manual_seed(19)
    d = 64
    cache = torch.empty((1, rows + tokens, 1, d), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    q = torch.randn((1, tokens, group, d), generator=g, device="cuda").bfloat16()
    w = torch.zeros((1, 1, rows + tokens), device="cuda")
    ops.decoder_attention_weights(q, cache, cache, torch.tensor([rows], device="cuda"), w)
    qq = q[0].double().reshape(tokens * group, d)
    see = rows + torch.arange(tokens, device="cuda").repeat_interleave(group)  # each row's last key

    def pieces():
        for i in range(0, rows + tokens, 1 << 18):
            keys = cache[0, i:i + (1 << 18), 0].double()
            at = torch.arange(i, i + len(keys), device="cuda")
            s = (qq @ keys.T / math.sqrt(d)).masked_fill_(at > see[:, None], -math.inf)
            yield i, s, float((qq.abs() @ keys.abs().T).max()) / math.sqrt(d)

    top = torch.full((tokens * group, 1), -math.inf, dtype=torch.float64, device="cuda")
    size = 0.0
    for _, s, largest in pieces():
        top, size = torch.maximum(top, s.amax(1, keepdim=True)), max(size, largest)
    total = sum(torch.exp(s - top).sum(1, keepdim=True) for _, s, _ in pieces())
    adds = 2 * math.ceil((rows + tokens) / 128 / 100) + 32 + 160
    rel = 4.5 * 2 * (d + 3) * U * size + 2.0 ** -18 + adds * U
    for i, s, _ in pieces():
        want = (torch.exp(s - top) / total).sum(0)
        off = (w[0, 0, i:i + len(want)].double() - want).abs()
        assert (off <= want * (rel + (tokens * group + 2) * U)).all(), f"rows from {i} on"


def test_weights_of_rows_far_before_the_queries(ops):
    """Committed rows times query heads pass 2^31, and the query tile has columns that no query fills."""
    check_weights_of_a_long_cache(ops, (1 << 31) // 120 + 5000, 120, 1)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("tokens", [6, 140])
@pytest.mark.parametrize("committed", [250, 3050])
@pytest.mark.parametrize("row", ["early", "last committed", "drafted"])
def test_an_infinite_value_of_no_probability(ops, row, committed, tokens, d):
    """Its product with the probability 0 is NaN wherever the row lies: in a tile of committed rows alone, in the tile where
    the drafted rows begin, among those. Scores of -6000 and less leave a probability of 0 in 64 bits too."""
    g = torch.Generator(device="cuda").manual_seed(20)
    q = torch.randn((1, tokens, 4, d), generator=g, device="cuda").bfloat16()
    q[..., 0] = 1.0
    k, v = caches(g, 1, committed + tokens + 60, 2, d, "dense")
    n = torch.tensor([committed], device="cuda")
    mask = torch.ones((tokens, tokens), dtype=torch.bool, device="cuda").tril()
    first = 3 if row == "drafted" else 0  # the first node that sees the row
    at = {"early": 10, "last committed": committed - 1, "drafted": committed + 3}[row]
    k[0, at, :, 0] = -1e5
    want = ops.tree_attention(q, k, v, n, mask)
    assert torch.isfinite(want).all()
    v[0, at, 1, 5] = math.inf
    want[0, first:, 2:, 5] = math.nan
    got = ops.tree_attention(q, k, v, n, mask)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    w = torch.zeros((1, 2, k.shape[1]), device="cuda")
    v[0, at, 1, 5] = 0.0
    want = ops.decoder_attention_weights(q, k, v, n, w)
    v[0, at, 1, 5] = math.inf
    want[0, first:, 2:, 5] = math.nan
    got = ops.decoder_attention_weights(q, k, v, n, w.zero_())
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    assert torch.isfinite(w).all() and w[0, 0, at] == 0


def test_queries_off_the_16_byte_grid(ops):
    """Dense queries at any address give what a copy of them gives, as caches do."""
    g = torch.Generator(device="cuda").manual_seed(21)
    q = torch.randn((2 * 3 * 4 * 64 + 1,), generator=g, device="cuda").bfloat16()[1:].view(2, 3, 4, 64)
    assert q.is_contiguous() and q.data_ptr() % 16 == 2
    k, v = caches(g, 2, 100, 2, 64, "dense")
    n = torch.tensor([90, 13], device="cuda")
    mask = torch.ones((3, 3), dtype=torch.bool, device="cuda").tril()
    w, w2 = torch.zeros((2, 2, 2, 100), device="cuda")
    assert torch.equal(ops.tree_attention(q, k, v, n, mask), ops.tree_attention(q.clone(), k, v, n, mask))
    assert torch.equal(ops.decoder_attention_weights(q, k, v, n, w),
                       ops.decoder_attention_weights(q.clone(), k, v, n, w2))
    assert torch.equal(w, w2)


@pytest.mark.parametrize("group,tokens", [(1, 2), (16, 2)])
def test_weights_of_a_cache_whose_scores_are_too_many_to_keep(ops, group, tokens):
    """8.5 million rows of a head of 64: 68 MB of scores with two rows a head, which are kept, and more than 1 GiB with 32,
    which are not."""
    check_weights_of_a_long_cache(ops, 8_500_000, group, tokens)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("tokens", [5, 150])
def test_weights_of_calls_on_two_streams(ops, tokens):
    """Twenty calls on each of two streams at once add the bits that they add one after the other: from kept scores, and in
    units that are cut between CTAs."""
    g = torch.Generator(device="cuda").manual_seed(22)
    sets = []
    for i in range(2):
        k, v = caches(g, 3, 3000, 4, 128, "dense")
        q = torch.randn((3, tokens, 8, 128), generator=g, device="cuda").bfloat16()
        n = torch.tensor([2800 - 700 * i, 100, 1500], device="cuda")
        sets.append((q, k, v, n, torch.zeros((3, 4, 3000), device="cuda")))
    want = []
    for q, k, v, n, w in sets:
        want.append(w.clone())
        for _ in range(20):
            ops.decoder_attention_weights(q, k, v, n, want[-1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(20):
        for s, (q, k, v, n, w) in zip(streams, sets):
            with torch.cuda.stream(s):
                ops.decoder_attention_weights(q, k, v, n, w)
    torch.cuda.synchronize()
    for (_, _, _, _, w), same in zip(sets, want):
        assert w.any() and torch.equal(w, same)


@pytest.mark.parametrize("kind", ["smooth", "ties", "special"])
@pytest.mark.parametrize("layout,dtype", [("dense", torch.float32), ("packed", torch.float32), ("layer", torch.bfloat16),
                                          ("shifted", torch.float32)])
def test_cache_evict_of_more_rows_than_shared_memory_holds(ops, layout, dtype, kind):
    """Keys of more than 49152 rows are made again in each pass; equal weights, zeros of both signs, infinities and NaN."""
    g = torch.Generator(device="cuda").manual_seed(23)
    batch, h, d, capacity, lengths, keep, recent, sinks, out = 2, 2, 16, 50003, [50003, 49151], 20000, 50, 4, 20007
    k, v = caches(g, batch, capacity, h, d, layout, dtype)
    w = torch.rand((batch, h, capacity), generator=g, device="cuda") ** 8
    if kind == "ties":
        w = (w * 6).round()
    elif kind == "special":
        some = torch.randint(0, 8, w.shape, generator=g, device="cuda")
        for i, x in enumerate([0.0, -0.0, math.inf, -math.inf, math.nan, -1.0]):
            w[some == i] = x
    k2, v2, w2, left, index = ops.cache_evict(k, v, w, torch.tensor(lengths).cuda(), keep, recent, sinks, out)
    assert left.tolist() == [keep, keep]
    for b in range(batch):
        for head in range(h):
            rows = torch.tensor(kept_rows(w[b, head].tolist(), lengths[b], keep, recent, sinks), dtype=torch.int64).cuda()
            assert torch.equal(index[b, head], rows)
            assert torch.equal(k2[b, :keep, head], k[b, rows, head]) and torch.equal(v2[b, :keep, head], v[b, rows, head])
            assert torch.equal(w2[b, head, :keep].view(torch.int32), w[b, head, rows].view(torch.int32))
    assert not k2[:, keep:].any() and not v2[:, keep:].any() and not w2[:, :, keep:].any()

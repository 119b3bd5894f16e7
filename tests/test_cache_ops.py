"""Refusals of the cache operators (tree attention, accept, commit, attention weights, eviction) without a GPU: the C
entry points' status and message before any CUDA call, and the Python wrappers' exceptions on host tensors."""

from __future__ import annotations

import pytest
import torch

from cppinf_b200 import capi, ops


@pytest.fixture(scope="module")
def lib():
    return capi.load()


P = 1 << 20  # an aligned address that no check reads


def strides(*values):
    return capi.i64_array(values)


def tree(lib, batch=1, tokens=4, q_heads=4, kv_heads=2, d=64, capacity=16, q=P, k=P, ks=(2048, 128, 64), v=P,
         vs=(2048, 128, 64), lengths=P, mask=P, mask_stride=0, ctx=P):
    return lib.cppinf_tree_attention(q, k, strides(*ks), v, strides(*vs), lengths, mask, mask_stride, None, ctx, batch,
                                     tokens, q_heads, kv_heads, d, capacity, None, 0, None, None)


def weights(lib, batch=1, tokens=4, q_heads=4, kv_heads=2, d=64, capacity=16, q=P, k=P, ks=(2048, 128, 64), lengths=P,
            w=P, scratch=P, scratch_bytes=1 << 40):
    return lib.cppinf_decoder_attention_weights(q, k, strides(*ks), P, strides(2048, 128, 64), lengths, None, P, w,
                                                batch, tokens, q_heads, kv_heads, d, capacity, scratch, scratch_bytes,
                                                None, None)


@pytest.mark.parametrize("call", [tree, weights])
@pytest.mark.parametrize("status,message,change", [
    (capi.ERR_INVALID_ARGUMENT, "non-negative sizes", {"batch": -1}),
    (capi.ERR_INVALID_ARGUMENT, "non-negative sizes", {"tokens": -1}),
    (capi.ERR_INVALID_ARGUMENT, "non-zero head", {"kv_heads": 0}),
    (capi.ERR_INVALID_ARGUMENT, "divide by key/value heads", {"q_heads": 5}),
    (capi.ERR_UNSUPPORTED, "head sizes 64, 128 and 256", {"d": 96}),
    (capi.ERR_UNSUPPORTED, "128 query heads", {"q_heads": 258, "kv_heads": 2}),
    (capi.ERR_OVERFLOW, "index range", {"capacity": 1 << 31}),
    (capi.ERR_OVERFLOW, "index range", {"batch": 1 << 20, "tokens": 200, "q_heads": 64, "kv_heads": 64}),
    (capi.ERR_INVALID_ARGUMENT, "null pointer", {"q": None}),
    (capi.ERR_INVALID_ARGUMENT, "null pointer", {"k": None}),
    (capi.ERR_INVALID_ARGUMENT, "null pointer", {"lengths": None}),
    (capi.ERR_UNSUPPORTED, "aligned", {"q": P + 8}),
    (capi.ERR_UNSUPPORTED, "aligned", {"k": P + 2}),
    (capi.ERR_UNSUPPORTED, "multiples of 8", {"ks": (2048, 132, 64)}),
    (capi.ERR_INVALID_ARGUMENT, "positive cache strides", {"ks": (2048, -128, 64)}),
])
def test_attention_refusals(lib, call, status, message, change):
    assert call(lib, **change) == status
    assert message in capi.last_error()


def test_tree_attention_refusals(lib):
    assert tree(lib, tokens=257, capacity=400) == capi.ERR_UNSUPPORTED
    assert "256 drafted tokens" in capi.last_error()
    assert tree(lib, mask=None) == capi.ERR_INVALID_ARGUMENT
    assert tree(lib, mask_stride=-1) == capi.ERR_INVALID_ARGUMENT
    assert tree(lib, vs=(2048, 128, 60)) == capi.ERR_UNSUPPORTED


def test_weights_refusals(lib):
    assert weights(lib, w=None) == capi.ERR_INVALID_ARGUMENT
    assert weights(lib, scratch_bytes=8) == capi.ERR_INVALID_ARGUMENT
    assert "scratch" in capi.last_error()
    assert weights(lib, scratch=None) == capi.ERR_INVALID_ARGUMENT


def test_empty_calls_need_no_device(lib):
    assert tree(lib, batch=0) == capi.OK and tree(lib, tokens=0) == capi.OK
    assert weights(lib, batch=0) == capi.OK and weights(lib, tokens=0) == capi.OK
    assert lib.cppinf_tree_accept(None, None, None, None, None, None, None, 0, 8, None) == capi.OK
    assert commit(lib, batch=0) == capi.OK and commit(lib, tokens=0) == capi.OK
    assert evict(lib, batch=0) == capi.OK


def test_scratch_bytes(lib):
    for flag in (0, 1):
        assert lib.cppinf_cache_attention_scratch_bytes(2, 4, 8, 2, 128, 640, flag) >= 0
        assert lib.cppinf_cache_attention_scratch_bytes(2, 4, 8, 3, 128, 640, flag) < 0


def commit(lib, dtype=0, batch=1, tokens=4, heads=2, d=64, capacity=16, k=P, ks=(2048, 128, 64), path=P):
    return lib.cppinf_tree_commit(dtype, k, strides(*ks), P, strides(2048, 128, 64), P, path, P, batch, tokens, heads,
                                  d, capacity, None)


def evict(lib, dtype=0, batch=1, heads=2, d=64, capacity=16, keep=8, recent=2, sinks=1, out=8, k=P,
          ks=(2048, 128, 64), w=P):
    return lib.cppinf_cache_evict(dtype, k, strides(*ks), P, strides(2048, 128, 64), w, P, P, P, P, P, P, batch, heads,
                                  d, capacity, keep, recent, sinks, out, None)


def test_accept_refusals(lib):
    args = (P, P, P, None, P, P, P)
    assert lib.cppinf_tree_accept(*args, -1, 4, None) == capi.ERR_INVALID_ARGUMENT
    assert lib.cppinf_tree_accept(*args, 1, 257, None) == capi.ERR_UNSUPPORTED
    assert lib.cppinf_tree_accept(*args, 1 << 31, 4, None) == capi.ERR_OVERFLOW
    assert lib.cppinf_tree_accept(None, P, P, None, P, P, P, 1, 4, None) == capi.ERR_INVALID_ARGUMENT
    assert lib.cppinf_tree_accept(P, P, P, None, P, None, P, 1, 4, None) == capi.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("call", [commit, evict])
@pytest.mark.parametrize("status,change", [
    (capi.ERR_INVALID_ARGUMENT, {"dtype": 7}),
    (capi.ERR_INVALID_ARGUMENT, {"batch": -1}),
    (capi.ERR_UNSUPPORTED, {"d": 60}),
    (capi.ERR_UNSUPPORTED, {"ks": (2048, 132, 64)}),
    (capi.ERR_INVALID_ARGUMENT, {"ks": (-2048, 128, 64)}),
    (capi.ERR_UNSUPPORTED, {"k": P + 8}),
    (capi.ERR_INVALID_ARGUMENT, {"k": None}),
    (capi.ERR_OVERFLOW, {"batch": 1 << 24}),
])
def test_commit_and_evict_refusals(lib, call, status, change):
    assert call(lib, **change) == status


@pytest.mark.parametrize("status,change", [
    (capi.ERR_INVALID_ARGUMENT, {"keep": 0, "recent": 0, "sinks": 0}),
    (capi.ERR_INVALID_ARGUMENT, {"recent": -1}),
    (capi.ERR_INVALID_ARGUMENT, {"sinks": -1}),
    (capi.ERR_INVALID_ARGUMENT, {"recent": 8, "sinks": 1}),
    (capi.ERR_INVALID_ARGUMENT, {"recent": (1 << 63) - 1, "sinks": 1}),
    (capi.ERR_OUT_OF_RANGE, {"out": 7}),
    (capi.ERR_INVALID_ARGUMENT, {"w": None}),
])
def test_evict_budget_refusals(lib, status, change):
    assert evict(lib, **change) == status


# ---- the Python wrappers on host tensors ---------------------------------------------------------------------------


def host(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def tree_args(**change):
    args = {"q": host(2, 3, 4, 64), "k_cache": host(2, 8, 2, 64), "v_cache": host(2, 8, 2, 64),
            "lengths": host(2, dtype=torch.int64), "mask": host(3, 3, dtype=torch.bool)}
    return args | change


@pytest.mark.parametrize("message,change", [
    ("CUDA tensors", {}),
    ("bool mask", {"mask": host(3, 3, dtype=torch.uint8)}),
    ("bool mask", {"mask": host(3, 4, dtype=torch.bool)}),
    ("bool mask", {"mask": host(1, 3, 3, dtype=torch.bool)}),
    ("bool mask", {"mask": host(3, 3, 3, dtype=torch.bool)}),
    ("bool mask", {"q": host(3, 4, 64)}),
    ("K and V caches", {"k_cache": host(2, 8, 2, 128)}),
    ("K and V caches", {"k_cache": host(8, 2, 64), "v_cache": host(8, 2, 64)}),
    ("matching tensor dtypes", {"k_cache": host(2, 8, 2, 64, dtype=torch.float32)}),
    ("bf16", {"q": host(2, 3, 4, 64, dtype=torch.float32)}),
    ("as many cached sequences", {"q": host(1, 3, 4, 64)}),
    ("matching query/key/value head sizes", {"q": host(2, 3, 4, 128)}),
    ("error word", {"error": host(1)}),
])
def test_tree_attention_wrapper_refusals(message, change):
    with pytest.raises(ValueError, match=message):
        ops.tree_attention(**tree_args(**change))


def test_other_wrapper_refusals():
    ids = host(2, 3, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.tree_accept(ids, ids, ids)
    with pytest.raises(ValueError, match="batch, nodes"):
        ops.tree_accept(ids, ids[:1], ids)
    with pytest.raises(ValueError, match="int64 tokens"):
        ops.tree_accept(ids, ids, ids.int())
    cache, n = host(2, 8, 2, 64), host(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="int64 path"):
        ops.tree_commit(cache, cache, n, ids.int(), n)
    with pytest.raises(ValueError, match="int64 path"):
        ops.tree_commit(cache, cache, n, ids[:1], n)
    with pytest.raises(ValueError, match="unsupported dtype"):
        ops.tree_commit(cache.half(), cache.half(), n, ids, n)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.tree_commit(cache, cache, n, ids, n)
    w = host(2, 2, 8, dtype=torch.float32)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.decoder_attention_weights(host(2, 3, 4, 64), cache, cache, n, w)
    with pytest.raises(ValueError, match="f32 weights"):
        ops.cache_evict(cache, cache, w[:, :, :7], n, 4, 2)
    with pytest.raises(ValueError, match="cover recent and sinks"):
        ops.cache_evict(cache, cache, w, n, 4, 4, 1)
    with pytest.raises(IndexError, match="too small"):
        ops.cache_evict(cache, cache, w, n, 4, 2, capacity=3)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.cache_evict(cache, cache, w, n, 4, 2)


def test_cache_strides_say_which_views_are_read_in_place():
    t = host(2, 8, 2, 64)
    assert ops._cache_strides(t) == (1024, 128, 64)
    both = host(2, 8, 2, 2, 64)
    assert ops._cache_strides(both[:, :, 1]) == (2048, 256, 64)
    assert ops._cache_strides(host(2, 2, 8, 64).transpose(1, 2)) == (1024, 64, 512)
    assert ops._cache_strides(host(1, 8, 2, 64).expand(2, 8, 2, 64)) is None  # sequences share their rows
    assert ops._cache_strides(host(2, 8, 2, 68)[..., :64]) is None  # rows off the 16-byte grid
    assert ops._cache_strides(host(2, 8, 64, 2).transpose(2, 3)) is None
    assert ops._cache_strides(host(1, 8, 1, 64)) == (512, 64, 64)


def test_cache_strides_of_empty_caches():
    assert ops._cache_strides(host(1, 0, 2, 64)) == (128, 128, 64)
    assert ops._cache_strides(host(1, 8, 2, 64)[:, :0]) == (128, 128, 64)


def test_commit_refuses_one_cache_for_both_and_broadcast_strides(lib):
    assert commit(lib) == capi.ERR_INVALID_ARGUMENT
    assert b"of their own" in lib.cppinf_last_error()
    assert commit(lib, k=P + 4096, ks=(0, 128, 64)) == capi.ERR_INVALID_ARGUMENT
    assert evict(lib, ks=(0, 128, 64)) == capi.ERR_INVALID_ARGUMENT


def test_attention_sizes_that_pass_the_index_range(lib):
    args = (8, 2, 64, 1024)
    assert lib.cppinf_cache_attention_scratch_bytes(1, 1 << 60, *args, 1) == -1  # tokens * q_heads wraps round
    assert lib.cppinf_cache_attention_scratch_bytes(1, 1 << 61, *args, 1) == -1
    # 2^16 * 2^13 heads of one tile each: 2^29 tiles, and with an item's set-up before each 2^31 pieces.
    assert lib.cppinf_cache_attention_scratch_bytes(1 << 16, 1, 1 << 13, 1 << 13, 64, 16, 0) == -1


def test_scratch_of_long_caches_is_bounded(lib):
    """Kept scores, 4 bytes a row of a head and a cached row, take 1 GiB or a sixteenth of K and V at most; beside them lie
    the parts of 148 CTAs (2 * 148 * 32 rows of 128) and the rows' statistics, below 2^26 bytes together."""
    def scratch(tokens):  # 32 sequences of 131072 rows, 16 over 8 heads of 128: K and V take 16 GiB
        return lib.cppinf_cache_attention_scratch_bytes(32, tokens, 16, 8, 128, 131072, 1)

    assert scratch(16) < (1 << 30) + (1 << 26)  # 4 GiB of scores
    assert scratch(8) < (1 << 30) + (1 << 26)   # 2 GiB
    assert scratch(4) <= (1 << 30) + (1 << 26)  # 1 GiB
    assert 1 << 28 <= scratch(1) < (1 << 28) + (1 << 26)
    assert lib.cppinf_cache_attention_scratch_bytes(64, 4, 16, 8, 128, 131072, 1) < (1 << 31) + (1 << 26)

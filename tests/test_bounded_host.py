"""Host side of the bounded cache: what the C entries and the Python calls refuse before any
launch, row selection, and the pool's bookkeeping of evictions over a CPU arena."""

import ctypes
import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from aster_amd import EvictedTokens, KeyWeights, PagedKVCache, UnsupportedAttentionBackend, _native
from aster_amd.offload import PagedStateArchive
from aster_amd.paged_pool import CacheCapacityError, PagedStatePool, StateError
from aster_amd.runner import PagedAttentionStep
from tests.fake_arena import FakeArena
from tests.test_gpu_evict import chosen

EINVAL, EUNSUPPORTED = _native.ASTR_EINVAL, _native.ASTR_EUNSUPPORTED


def desc(**kw):
    d = dict(k_codes=1 << 20, v_codes=1 << 20, k_scales=1 << 20, v_scales=1 << 20,
             code_block_stride=2 * 2 * 16 * 64, code_head_stride=16 * 64, scale_block_stride=64,
             scale_head_stride=16, num_blocks=4, block_size=16, num_kv_heads=2, head_dim=64,
             key_valid=None, code_format=0)
    return _native.PagedKVDesc(**{**d, **kw})


def sinks(cache=None, **kw):
    a = dict(query=1 << 20, dtype=2, qt=4 * 64, qh=64, out=1 << 20, ot=4 * 64, oh=64, start=None, tokens=0,
             most=0, tables=1 << 20, stride=4, lens=1 << 20, seqs=2, heads=4, ctx=64, scale=0.1,
             window=16, sinks=4, ws=None, ws_bytes=0, flag=1 << 20)
    a.update(kw)
    return _native.lib().astr_paged_attention_i8_sinks(cache if cache is not None else desc(), *a.values(), None)


def weights_desc(**kw):
    return _native.KeyWeightsDesc(**{**dict(values=1 << 20, row_stride=2 * 64, head_stride=64, rows=None,
                                            num_rows=4, capacity=64), **kw})


def key_weights(w="default", **kw):
    a = dict(query=1 << 20, dtype=2, qt=4 * 64, qh=64, out=1 << 20, ot=4 * 64, oh=64, start=None, tokens=0,
             most=0, tables=1 << 20, stride=4, lens=1 << 20, seqs=2, heads=4, ctx=64, scale=0.1,
             w=weights_desc() if w == "default" else w, ws=None, ws_bytes=0, flag=1 << 20)
    a.update(kw)
    return _native.lib().astr_paged_attention_i8_key_weights(desc(), *a.values(), None)


def evict(**kw):
    a = dict(cache=desc(), layers=2, cl=2 * 2 * 16 * 64, sl=64, w=weights_desc(), wl=128, to=None,
             tables=1 << 20, stride=4, dst=None, dst_stride=0, lens=1 << 20, seqs=2, ctx=64, keep=32,
             sinks=4, recent=8, kept=1 << 20, new=1 << 20, flag=1 << 20)
    a.update(kw)
    return _native.lib().astr_kv_evict(*a.values(), None)


def test_sinks_refuse_bad_arguments_without_a_device():
    assert sinks(seqs=0) == 0
    for bad in (dict(window=0), dict(sinks=0), dict(query=None), dict(out=None), dict(tables=None),
                dict(lens=None), dict(flag=None), dict(seqs=-1), dict(heads=0), dict(heads=3),
                dict(ctx=65), dict(ctx=-1), dict(scale=0.0), dict(scale=math.inf), dict(qt=3),
                dict(oh=1), dict(query=(1 << 20) + 8), dict(start=1 << 20, tokens=-1)):
        assert sinks(**bad) == EINVAL, bad
    assert sinks(start=1 << 20, tokens=0) == 0  # no query token
    for bad in (dict(dtype=7), dict(heads=6), dict(seqs=70000)):
        assert sinks(**bad) == EUNSUPPORTED, bad
    for bad, code in ((dict(block_size=32), EUNSUPPORTED), (dict(head_dim=96), EUNSUPPORTED),
                      (dict(code_format=3), EUNSUPPORTED), (dict(num_blocks=0), EINVAL),
                      (dict(k_codes=(1 << 20) + 4), EINVAL), (dict(key_valid=(1 << 20) + 1), EINVAL),
                      (dict(scale_head_stride=15), EINVAL)):
        assert sinks(desc(**bad)) == code, bad
    # a long row needs a workspace
    assert sinks(seqs=1, ctx=16000, stride=1000, window=15000) == EINVAL
    assert "workspace" in _native.last_error()


def test_key_weights_refuse_bad_arguments_without_a_device():
    assert key_weights(seqs=0) == 0
    for w in (None, weights_desc(values=None), weights_desc(num_rows=0), weights_desc(capacity=63),
              weights_desc(values=(1 << 20) + 4), weights_desc(head_stride=63),
              weights_desc(row_stride=129)):
        assert key_weights(w) == EINVAL
    assert key_weights() == EINVAL  # scores need a workspace
    assert "workspace" in _native.last_error()


def test_evictions_refuse_bad_arguments_without_a_device():
    assert evict(seqs=0) == 0
    for bad in (dict(keep=0), dict(keep=11), dict(sinks=-1), dict(recent=-1), dict(layers=0),
                dict(kept=None), dict(new=None), dict(tables=None), dict(lens=None), dict(flag=None),
                dict(ctx=65), dict(w=weights_desc(capacity=48)), dict(w=weights_desc(values=None)),
                dict(dst=1 << 20, dst_stride=1), dict(cl=8), dict(cache=desc(num_blocks=0))):
        assert evict(**bad) == EINVAL, bad
    for bad in (dict(cache=desc(head_dim=96)), dict(cache=desc(block_size=8)), dict(seqs=70000),
                dict(layers=70000)):
        assert evict(**bad) == EUNSUPPORTED, bad


def test_workspace_sizes_grow_with_the_call():
    def size(seqs=1, heads=4, kv=2, dim=64, dtype=2, tokens=0, most=0, ctx=4096, window=0, sinks=0, kw=0):
        return _native.lib().astr_paged_attention_i8_bounded_workspace_bytes(
            seqs, heads, kv, dim, dtype, tokens, most, ctx, window, sinks, kw)

    assert size(kw=1) >= 4 * 4096 * 4 and size(seqs=0) == 0 and size(heads=3) == 0
    assert size(kw=1, ctx=8192) > size(kw=1)
    assert size(seqs=300, window=64, sinks=4) == 0  # a piece per row: no partials
    assert size(tokens=100, most=100, kw=1) > 0


# ---- Python checks (tensors on the CPU stand in for the device's) ----------------------------


def cpu_cache(**kw):
    """A PagedKVCache whose arena is on the CPU: good for argument checks alone."""
    cache = PagedKVCache.__new__(PagedKVCache)
    arena = FakeArena(num_blocks=8, num_layers=2, num_kv_heads=2, head_dim=64, **kw)
    cache.__dict__.update(arena.__dict__, code_format=0, _workspace=None, _bounded_sizes={},
                          err_flag=torch.zeros(1, dtype=torch.int32))
    cache._descs = [desc()] * 2
    return cache


def call_args(cache, rows=2, tokens=40):
    return (0, torch.zeros((rows, 4, 64), dtype=torch.bfloat16), torch.zeros((rows, 4), dtype=torch.int32),
            torch.full((rows,), tokens, dtype=torch.int32))


def test_python_refuses_sinks_that_no_kernel_serves():
    cache = cpu_cache()
    args = call_args(cache)
    for bad in (dict(sinks=0, window=8), dict(sinks=2.0, window=8), dict(sinks=4), dict(sinks=True + 0.5, window=4),
                dict(sinks=4, window=8, causal=False), dict(sinks=4, window=8, partition_tokens=64),
                dict(sinks=4, window=8, prefix_packs=object()), dict(sinks=4, window=8, decode_plan=object()),
                dict(sinks=4, window=0)):
        with pytest.raises(ValueError):
            cache.paged_attention(*args, max_context_len=40, **bad)
    with pytest.raises(ValueError, match="capacity"):
        cache.paged_attention(*args, max_context_len=65, window=8, sinks=2)
    with pytest.raises(UnsupportedAttentionBackend, match="dtype"):
        cache.paged_attention(0, args[1].double(), *args[2:], max_context_len=40, window=8, sinks=2)
    with pytest.raises(ValueError, match="one query row"):
        cache.paged_attention(0, args[1][:1], *args[2:], max_context_len=40, window=8, sinks=2)
    with pytest.raises(ValueError, match="workspace"):
        cache.paged_attention(0, args[1][:1], torch.zeros((1, 400), dtype=torch.int32), args[3][:1],
                              max_context_len=6000, window=5000, sinks=2,
                              workspace=torch.zeros(1, dtype=torch.uint8))


def test_python_refuses_key_weights_of_another_batch():
    cache = cpu_cache()
    kw = KeyWeights(cache, rows=3, capacity=33)
    assert kw.capacity == 48 and kw.values.shape == (3, 2, 2, 48) and (kw.values == 0).all()
    for bad in ([0, 0], [0, 3], [-1], [0.0], [True]):
        with pytest.raises(ValueError):
            kw.select(bad)
    for bad in (dict(rows=0, capacity=4), dict(rows=1, capacity=0), dict(rows=1.0, capacity=4)):
        with pytest.raises(ValueError):
            KeyWeights(cache, **bad)
    args = call_args(cache)
    with pytest.raises(ValueError, match="selected"):
        cache.paged_attention_weights(*args, kw, max_context_len=40)
    with pytest.raises(ValueError, match="one row per sequence"):
        cache.paged_attention_weights(*args, kw.select([0]), max_context_len=40)
    with pytest.raises(ValueError, match="capacity"):
        cache.paged_attention_weights(*args, kw.select([0, 1]), max_context_len=49)
    other = KeyWeights(SimpleNamespace(num_layers=1, num_kv_heads=2, device=cache.device), rows=2, capacity=48)
    with pytest.raises(ValueError, match="another cache"):
        cache.paged_attention_weights(*args, other.select([0, 1]), max_context_len=40)


def test_python_refuses_evictions_that_would_collide():
    cache = cpu_cache()
    kw = KeyWeights(cache, rows=4, capacity=48)
    tables, lens = call_args(cache)[2:]
    rows = kw.select([0, 1])
    for bad in (dict(keep=0), dict(keep=4, recent=3, sinks=2), dict(keep=4.0), dict(keep=8, recent=-1)):
        with pytest.raises(ValueError, match="keep must"):
            cache.evict(tables, lens, rows, max_context_len=40, **bad)
    for into in ([1, 0], [1, 2], [3, 0]):  # another sequence's row
        with pytest.raises(ValueError, match="another sequence"):
            cache.evict(tables, lens, rows, keep=8, max_context_len=40, into=kw.select(into))
    with pytest.raises(ValueError, match="into must"):
        cache.evict(tables, lens, rows, keep=8, max_context_len=40,
                    into=KeyWeights(cache, rows=2, capacity=48).select([0, 1]))
    with pytest.raises(ValueError, match="dst_tables"):
        cache.evict(tables, lens, rows, keep=20, max_context_len=40,
                    dst_tables=torch.zeros((2, 1), dtype=torch.int32))
    with pytest.raises(ValueError, match="capacity"):
        cache.evict(tables, lens, rows, keep=20, max_context_len=64)


# ---- the pool ---------------------------------------------------------------------------


class EvictingArena(FakeArena):
    """FakeArena with the eviction of a device arena."""

    def __init__(self, **kw):
        super().__init__(**kw)
        self.calls = []

    def evict(self, tables, lens, rows, *, keep, recent, sinks, max_context_len, dst_tables=None):
        self.calls.append((tables.clone(), lens.clone(), None if dst_tables is None else dst_tables.clone()))
        dst = tables if dst_tables is None else dst_tables
        codes, scales, valid = self.codes.clone(), self.scales.clone(), self.key_valid.clone()
        lengths = []
        for r, n in enumerate(lens.tolist()):
            pos = np.arange(n)
            table = tables[r].numpy()
            real = valid.numpy()[table[pos // 16], pos % 16] != 0
            for layer in range(self.num_layers):
                for h in range(self.num_kv_heads):
                    w = rows.weights.values[rows.rows[r], layer, h]
                    stay = chosen(w[:n].numpy(), real, keep, sinks, recent)
                    at = np.arange(len(stay))
                    d = dst[r].numpy()[at // 16]
                    self.codes[d, layer, :, h, at % 16] = codes[table[stay // 16], layer, :, h, stay % 16]
                    self.scales[d, layer, :, h, at % 16] = scales[table[stay // 16], layer, :, h, stay % 16]
                    self.key_valid[d, at % 16] = 1
                    w[:len(stay)] = w[:n][stay].clone()
            lengths.append(len(stay))
        return EvictedTokens(None, torch.tensor(lengths, dtype=torch.int32))


def make(blocks=24, lens=(40,), seed=0, padding=None):
    pool = PagedStatePool(EvictingArena(num_blocks=blocks, num_layers=2, num_kv_heads=2, head_dim=8))
    kw = KeyWeights(pool.cache, rows=len(lens) + 2, capacity=96)
    gen = torch.Generator().manual_seed(seed)
    kw.values.copy_(torch.rand(kw.values.shape, generator=gen))
    seqs = []
    for n in lens:
        s = pool.create("tenant")
        state = [(torch.randn((n, 2, 8), generator=gen), torch.randn((n, 2, 8), generator=gen)) for _ in range(2)]
        if padding is not None:
            state.append((torch.arange(n) % padding != 0,))
        pool.append_delta(s, state)
        seqs.append(s)
    return pool, kw, seqs


def kept_state(pool, seq, weights, keep, recent, sinks):
    state = pool.materialize(seq)
    real = state[-1][0][0, 0, :, 0].numpy()
    out = []
    for layer, (k, v) in enumerate(state[:-1]):
        rows = []
        for x in (k, v):
            rows.append(torch.stack([x[0, h, chosen(weights[layer, h, :seq.length].numpy(), real, keep, sinks,
                                                     recent)] for h in range(2)]))
        out.append(rows)
    return out


def check_state(pool, seq, want):
    for (k, v), (wk, wv) in zip(pool.materialize(seq)[:-1], want):
        assert torch.equal(k[0], wk) and torch.equal(v[0], wv)


def test_pool_evicts_in_place():
    pool, kw, (a, b, c) = make(lens=(70, 20, 45))
    want = [kept_state(pool, s, kw.values[r], 32, 8, 4) for s, r in ((a, 1), (c, 0))]
    small = pool.materialize(b)
    assert pool.evict([a, b, c], kw.select([1, 3, 0]), keep=32, recent=8, sinks=4) == (32, 20, 32)
    assert (a.evicted, b.evicted, c.evicted) == (38, 0, 13) and (a.floor, b.floor) == (32, 0)
    assert pool.used_blocks == 2 + 2 + 2 and len(pool.cache.calls) == 1
    check_state(pool, a, want[0]), check_state(pool, c, want[1])
    assert all(torch.equal(x, y) for p, q in zip(pool.materialize(b), small) for x, y in zip(p, q))
    # it grows again, and cannot be cut into what stayed
    pool.append_delta(a, [(torch.ones((3, 2, 8)), torch.ones((3, 2, 8)))] * 2)
    assert a.length == 35 and a.evicted == 38
    pool.truncate(a, 33)
    with pytest.raises(ValueError, match="eviction"):
        pool.truncate(a, 31)
    pool.truncate(a, 0)
    assert (a.evicted, a.floor) == (0, 0)


def test_pool_evicts_shared_and_read_pages_into_fresh_ones():
    pool, kw, (a,) = make(lens=(64,))
    child = pool.fork(a)
    before = pool.materialize(child)
    want = kept_state(pool, a, kw.values[0], 20, 4, 0)
    assert pool.evict([a], kw.select([0]), keep=20, recent=4) == (20,)
    check_state(pool, a, want)
    assert all(torch.equal(x, y) for p, q in zip(pool.materialize(child), before) for x, y in zip(p, q))
    assert pool.used_blocks == 4 + 2 and (child.evicted, a.evicted) == (0, 44)
    with pool.borrow(a):  # readers of its own pages
        pages = list(a.pages)
        pool.evict([a], kw.select([0]), keep=10)
        assert not set(p.index for p in a.pages) & set(p.index for p in pages)
        assert pool.used_blocks == 4 + 2 + 1
    assert pool.used_blocks == 4 + 1
    twin = pool.fork(a)
    assert (twin.evicted, twin.floor) == (a.evicted, a.floor) == (54, 10)
    # both at once, sharing their pages
    pool.evict([a, twin], kw.select([0, 1]), keep=5)
    assert a.pages != twin.pages and a.length == twin.length == 5


def test_pool_eviction_drops_padding():
    pool, kw, (a,) = make(lens=(50,), padding=3)
    want = kept_state(pool, a, kw.values[0], 60, 0, 0)
    assert pool.evict([a], kw.select([0]), keep=60) == (33,)  # 17 of 50 are padding
    check_state(pool, a, want)
    assert pool.materialize(a)[-1][0].all() and a.evicted == 17


def test_pool_eviction_refusals_change_nothing():
    pool, kw, (a, b) = make(blocks=9, lens=(70, 60))
    child = pool.fork(a)
    state = pool.materialize(a)
    with pytest.raises(CacheCapacityError):
        pool.evict([a], kw.select([0]), keep=64)
    for call in (lambda: pool.evict([], kw.select([])), lambda: pool.evict([a, a], kw.select([0, 1]), keep=4),
                 lambda: pool.evict([a], kw.select([0, 1]), keep=4), lambda: pool.evict([a], kw, keep=4),
                 lambda: pool.evict([a], kw.select([0]), keep=4, recent=5)):
        with pytest.raises((ValueError, TypeError)):
            call()
    with pytest.raises(StateError):
        pool.evict([PagedStatePool(pool.cache).create("x")], kw.select([0]), keep=4)

    def failing(*args, **kwargs):
        raise RuntimeError("launch")

    pool.cache.evict = failing
    used = pool.used_blocks
    pool.release(b)
    with pytest.raises(RuntimeError, match="launch"):
        pool.evict([a], kw.select([0]), keep=16)
    assert pool.used_blocks == used - 4 and a.length == 70 and a.evicted == 0
    assert all(torch.equal(x, y) for p, q in zip(pool.materialize(a), state) for x, y in zip(p, q))
    pool.release(child)


def test_pool_evictions_are_refused_before_anything_moves():
    """A shared sequence is evicted ahead of the others: neither an error flagged earlier nor
    another sequence's refusal may leave its weights moved."""
    pool, kw, (a, b) = make(blocks=16, lens=(70, 60))
    pool.fork(a)
    weights, state = kw.values.clone(), [pool.materialize(s) for s in (a, b)]
    short = KeyWeights(pool.cache, rows=2, capacity=64)
    small = short.values.clone()
    with pytest.raises(ValueError, match="capacity"):
        pool.evict([b, a], short.select([0, 1]), keep=16)
    pool.fork(b)
    with pytest.raises(ValueError, match="capacity"):
        pool.evict([b, a], short.select([0, 1]), keep=16)

    def flagged():
        raise ValueError("Quantized KV requires finite floating input")

    real, pool.cache.raise_errors = pool.cache.raise_errors, flagged
    with pytest.raises(ValueError, match="finite"):
        pool.evict([a, b], kw.select([0, 1]), keep=16)
    pool.cache.raise_errors = real
    assert not pool.cache.calls and torch.equal(kw.values, weights) and torch.equal(short.values, small)
    for s, before in zip((a, b), state):
        assert s.evicted == s.floor == 0
        assert all(torch.equal(x, y) for p, q in zip(pool.materialize(s), before) for x, y in zip(p, q))


def test_an_eviction_that_drops_nothing_leaves_no_floor():
    pool, kw, (a, b) = make(blocks=16, lens=(30, 20), padding=5)
    c = pool.create("tenant")
    ones = [(torch.ones((25, 2, 8)), torch.ones((25, 2, 8)))] * 2 + [(torch.ones(25, dtype=torch.bool),)]
    pool.append_delta(c, ones)
    assert pool.evict([c], kw.select([2]), keep=64) == (25,)
    assert (c.evicted, c.floor) == (0, 0)
    pool.truncate(c, 3)


def test_archived_evictions_of_every_token_come_back():
    """All tokens were padding and left; what came after is archived with their count."""
    pool, kw, (seq,) = make(blocks=8, lens=(20,), padding=1)
    assert pool.evict([seq], kw.select([0]), keep=8) == (0,)
    assert (seq.evicted, seq.floor) == (20, 0)
    pool.append_delta(seq, [(torch.ones((3, 2, 8)), torch.ones((3, 2, 8)))] * 2 +
                      [(torch.ones(3, dtype=torch.bool),)])
    archive = PagedStateArchive(pool)
    archive._to_host = lambda s: (torch.zeros(1), torch.zeros(1), torch.zeros(1))
    archive._copy_stream = lambda: None
    got = {}
    pool.restore_pages = lambda payloads, **kw: got.update(kw)
    archive.restore(archive.put(seq), identity="tenant")
    assert (got["evicted"], got["floor"]) == (20, 0)


def test_archived_evictions_come_back():
    class Pool(PagedStatePool):
        def restore_pages(self, payloads, *, identity, length, stream=None, evicted=0, floor=0):
            sequence = self.create(identity)
            sequence.length, sequence.evicted, sequence.floor = length, evicted, floor
            return sequence

    pool = Pool(EvictingArena(num_blocks=8, num_layers=2, num_kv_heads=2, head_dim=8))
    seq = pool.create("tenant")
    pool.append_delta(seq, [(torch.ones((40, 2, 8)), torch.ones((40, 2, 8)))] * 2)
    kw = KeyWeights(pool.cache, rows=1, capacity=48)
    pool.evict([seq], kw.select([0]), keep=30)
    archive = PagedStateArchive(pool)
    archive._to_host = lambda s: (torch.zeros(1), torch.zeros(1), torch.zeros(1))
    archive._copy_stream = lambda: None
    handle = archive.put(seq)
    back = archive.restore(handle, identity="tenant")
    assert (back.length, back.evicted, back.floor) == (30, 10, 30)


def test_steps_refuse_windows_over_evicted_tokens():
    step = PagedAttentionStep.__new__(PagedAttentionStep)
    step.__dict__.update(_open=True, num_tokens=1, work=None, evicted=[3], key_weights=None,
                         pool=SimpleNamespace(cache=None))
    x = torch.zeros((1, 2, 8))
    with pytest.raises(UnsupportedAttentionBackend, match="windows"):
        step.attend(0, x, x, x, window=4)
    step.evicted, step.key_weights = [0], object()
    with pytest.raises(UnsupportedAttentionBackend, match="window"):
        step.attend(0, x, x, x, window=4)

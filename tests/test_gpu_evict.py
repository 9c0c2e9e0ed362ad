"""Eviction by gathered weight: which tokens stay, and where their codes, scales and weights
go, against a plain selection; all of it is exact."""

import numpy as np
import pytest
import torch

from aster_amd import KeyWeights
from tests.bounded_rows import make_arena, on

pytestmark = pytest.mark.gpu


def chosen(weights, real, keep, sinks, recent):
    """Positions that stay of one head: plain numpy, in 64 bits."""
    tokens = np.flatnonzero(real)
    n = len(tokens)
    if n <= keep:
        return tokens
    w = weights[tokens].astype(np.float64)
    rank = np.lexsort((np.arange(n), np.where(np.isnan(w), 0.0, -w), np.isnan(w)))  # NaN last
    fixed = np.zeros(n, bool)
    fixed[:sinks] = True
    fixed[n - recent:] = True
    others = [i for i in rank if not fixed[i]][:keep - sinks - recent]
    return np.sort(np.concatenate([tokens[fixed], tokens[others]])).astype(np.int64)


def check(cache, kw, tables, lens, rows, before, got, *, keep, sinks, recent, dst=None, to=None):
    codes0, scales0, weights0, valid0 = before
    dst = tables if dst is None else dst
    to = rows if to is None else to
    kept, lengths = got.kept.cpu().numpy(), got.lengths.cpu().numpy()
    codes, scales, weights = cache.codes.cpu(), cache.scales.cpu(), kw.values.cpu()
    want_codes, want_scales, want_weights = codes0.clone(), scales0.clone(), weights0.clone()
    want_valid = valid0.clone()
    for r, n in enumerate(lens):
        pos = np.arange(n)
        real = valid0.numpy()[tables[r][pos // 16], pos % 16] != 0
        for layer in range(cache.num_layers):
            for h in range(cache.num_kv_heads):
                stay = chosen(weights0[rows[r], layer, h, :n].numpy(), real, keep, sinks, recent)
                assert lengths[r] == len(stay)
                assert kept[r, layer, h, :len(stay)].tolist() == stay.tolist()
                assert (kept[r, layer, h, len(stay):] == -1).all()
                at = np.arange(len(stay))
                s, d = tables[r][stay // 16], dst[r][at // 16]
                want_codes[d, layer, :, h, at % 16] = codes0[s, layer, :, h, stay % 16]
                want_scales[d, layer, :, h, at % 16] = scales0[s, layer, :, h, stay % 16]
                want_weights[to[r], layer, h, at] = weights0[rows[r], layer, h, stay]
                want_valid[d, at % 16] = 1
    assert torch.equal(codes, want_codes)
    assert torch.equal(scales, want_scales)
    assert torch.equal(weights.view(torch.int32), want_weights.view(torch.int32))
    if cache.has_padding:
        assert torch.equal(cache.key_valid.cpu(), want_valid)


def setup(device, lens, *, kv_heads=2, dim=64, layers=2, fmt="int8", padding=0.0, seed=0, ties=False,
          spare=8):
    cache, tables, free = make_arena(device, lens, kv_heads=kv_heads, dim=dim, layers=layers, fmt=fmt,
                                     padding=padding, seed=seed, spare=spare)
    kw = KeyWeights(cache, rows=2 * len(lens) + 1, capacity=max(max(lens), 16))
    gen = torch.Generator(device=device).manual_seed(seed + 9)
    w = torch.rand(kw.values.shape, generator=gen, device=device).pow(6) * 30
    kw.values.copy_((w * 2).round() if ties else w)
    return cache, tables, free, kw


def state(cache, kw):
    return cache.codes.cpu(), cache.scales.cpu(), kw.values.cpu(), cache.key_valid.cpu()


def evict(cache, kw, tables, lens, rows, **extra):
    dev = cache.device
    return cache.evict(on(dev, tables), on(dev, np.asarray(lens, np.int32)), kw.select(rows),
                       max_context_len=int(max(lens)), check=True, **extra)


@pytest.mark.parametrize("padding", [0.0, 0.2])
@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (16, 4, 8), (33, 0, 33), (64, 1, 5),
                                               (100, 100, 0), (500, 4, 100), (2000, 3, 1)])
def test_in_place(device, padding, ties, keep, sinks, recent):
    lens = [1, 0, 16, 63, 101, 700, 1500]
    cache, tables, _, kw = setup(device, lens, padding=padding, ties=ties)
    rows = [5, 0, 3, 1, 2, 14, 9]
    before = state(cache, kw)
    got = evict(cache, kw, tables, lens, rows, keep=keep, sinks=sinks, recent=recent)
    check(cache, kw, tables, lens, rows, before, got, keep=keep, sinks=sinks, recent=recent)


@pytest.mark.parametrize("dim,fmt", [(64, "int8"), (128, "fp8_e4m3fn"), (256, "fp8_e5m2")])
@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("padding", [0.0, 0.1])
def test_into_other_pages(device, dim, fmt, into, padding):
    lens, keep = [40, 900, 0, 333], 200
    cache, tables, free, kw = setup(device, lens, dim=dim, fmt=fmt, layers=3, padding=padding, spare=60)
    dst = free[:4 * 13].reshape(4, 13)
    rows, to = [0, 1, 2, 3], [4, 1, 7, 8]
    before = state(cache, kw)
    got = evict(cache, kw, tables, lens, rows, keep=keep, recent=30, dst_tables=on(device, dst),
                into=kw.select(to) if into else None)
    check(cache, kw, tables, lens, rows, before, got, keep=keep, sinks=0, recent=30, dst=dst,
          to=to if into else rows)


def test_many_tokens_in_order(device):
    """Rows of many batches of the move, whose destinations overlap the sources."""
    lens = [6000, 5999]
    cache, tables, _, kw = setup(device, lens, kv_heads=1, dim=128, layers=1)
    before = state(cache, kw)
    got = evict(cache, kw, tables, lens, [0, 1], keep=5500, sinks=4, recent=64)
    check(cache, kw, tables, lens, [0, 1], before, got, keep=5500, sinks=4, recent=64)


def test_weights_of_every_kind(device):
    """Zeros of both signs, infinities, NaN, denormals and negative numbers."""
    lens = [160]
    cache, tables, _, kw = setup(device, lens, kv_heads=1, layers=1)
    kinds = torch.tensor([0.0, -0.0, float("inf"), float("nan"), 1e-42, -1e-42, -3.5, float("-inf"),
                          3e38, 1.0], device=device)
    kw.values[0, 0, 0, :160] = kinds.repeat(16)
    for keep in (1, 15, 16, 17, 40, 80, 95, 96, 120, 143, 144, 159):
        saved = (cache.codes.clone(), cache.scales.clone(), kw.values.clone())
        before = state(cache, kw)
        got = evict(cache, kw, tables, lens, [0], keep=keep)
        check(cache, kw, tables, lens, [0], before, got, keep=keep, sinks=0, recent=0)
        cache.codes.copy_(saved[0]), cache.scales.copy_(saved[1]), kw.values.copy_(saved[2])


def test_ids_out_of_range_move_nothing(device):
    lens = [100, 90]
    cache, tables, free, kw = setup(device, lens, kv_heads=1, layers=1)
    bad = tables.copy()
    bad[0, 3] = cache.num_blocks
    codes = cache.codes.cpu()
    dst = free[:8].reshape(2, 4)
    with pytest.raises(ValueError, match="outside the KV arena"):
        evict(cache, kw, bad, lens, [0, 1], keep=64, dst_tables=on(device, dst))
    changed = (cache.codes.cpu() != codes).flatten(1).any(1).nonzero().flatten().tolist()
    assert set(changed) <= set(dst.flatten().tolist())
    rows = kw.select([0, 1])
    rows.table.copy_(torch.tensor([0, 99], dtype=torch.int32))
    codes = cache.codes.cpu()
    with pytest.raises(ValueError, match="outside the KV arena"):
        cache.evict(on(device, tables), on(device, np.asarray(lens, np.int32)), rows, keep=96,
                    max_context_len=100, check=True)


def test_eviction_replays_in_a_graph(device):
    lens = [400, 90, 1000]
    cache, tables, free, kw = setup(device, lens, spare=40)
    dst = on(device, free[:24].reshape(3, 8))
    t, n = on(device, tables), on(device, np.asarray(lens, np.int32))
    rows, into = kw.select([0, 1, 2]), kw.select([3, 4, 5])

    def step():
        return cache.evict(t, n, rows, keep=128, recent=16, max_context_len=1000, dst_tables=dst,
                           into=into)

    want = step()
    torch.cuda.synchronize()
    after = state(cache, kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        cache.codes[dst.long()] = 0
        cache.scales[dst.long()] = 0
        kw.values[3:6] = -1
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got.kept, want.kept) and torch.equal(got.lengths, want.lengths)
        for r, length in enumerate(want.lengths.tolist()):  # what lies behind was cleared above
            at = np.arange(length)
            page, slot = dst.cpu().numpy()[r][at // 16], at % 16
            assert torch.equal(cache.codes.cpu()[page, :, :, :, slot], after[0][page, :, :, :, slot])
            assert torch.equal(cache.scales.cpu()[page, :, :, :, slot], after[1][page, :, :, :, slot])
            assert torch.equal(kw.values[3 + r, :, :, :length].cpu(), after[2][3 + r, :, :, :length])
    cache.raise_errors()


@pytest.mark.parametrize("apart", [False, True])
def test_pages_past_two_gigabytes(device, apart):
    """Codes that lie past 2^31 bytes of the arena, in place and into pages before them."""
    from aster_amd import PagedKVCache

    blocks = (1 << 31) // (2 * 8 * 16 * 128) + 70  # a block of one layer: 32 KB
    cache = PagedKVCache(num_blocks=blocks, num_layers=1, num_kv_heads=8, head_dim=128, device=device)
    gen = torch.Generator(device=device).manual_seed(3)
    cache.codes[-64:] = torch.randint(-127, 128, cache.codes[-64:].shape, generator=gen, device=device,
                                      dtype=torch.int8)
    cache.scales[-64:] = torch.rand(cache.scales[-64:].shape, generator=gen, device=device)
    kw = KeyWeights(cache, rows=1, capacity=1000)
    kw.values.copy_(torch.rand(kw.values.shape, generator=gen, device=device))
    high = np.arange(blocks - 64, blocks, dtype=np.int32)[None]
    low = np.arange(3, 11, dtype=np.int32)[None] if apart else high
    weights = kw.values[0, 0].cpu().numpy()
    codes, scales = cache.codes[-64:].clone(), cache.scales[-64:].clone()
    extra = {"dst_tables": on(device, low)} if apart else {}
    got = evict(cache, kw, high, [1000], [0], keep=100, recent=10, sinks=2, **extra)
    assert got.lengths.tolist() == [100]
    at = torch.arange(100, device=device)
    dst = torch.from_numpy(low[0].astype(np.int64)).to(device)[at // 16]
    for h in range(8):
        stay = chosen(weights[h, :1000], np.ones(1000, bool), 100, 2, 10)
        src = torch.from_numpy(stay).to(device)
        assert torch.equal(cache.codes[dst, 0, :, h, at % 16], codes[src // 16, 0, :, h, src % 16])
        assert torch.equal(cache.scales[dst, 0, :, h, at % 16], scales[src // 16, 0, :, h, src % 16])


def test_evictions_on_another_stream(device):
    lens = [300, 90]
    cache, tables, _, kw = setup(device, lens, padding=0.2)
    before = state(cache, kw)
    t, n, rows = on(device, tables), on(device, np.asarray(lens, np.int32)), kw.select([0, 1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cache.evict(t, n, rows, keep=64, recent=8, sinks=1, max_context_len=300)
    side.synchronize()
    check(cache, kw, tables, lens, [0, 1], before, got, keep=64, recent=8, sinks=1)

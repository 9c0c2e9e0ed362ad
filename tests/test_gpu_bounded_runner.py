"""The operators of a bounded cache as a serving loop runs them: steps that gather key weights,
evictions between them, forks and copy-on-write around those, and a decoder whose windows keep
sink tokens; each against plain 64-bit results over what the arena holds."""

import numpy as np
import pytest
import torch

from aster_amd import (KeyWeights, PagedAttentionRunner, PagedKVCache, PagedStateArchive,
                       UnsupportedAttentionBackend)
from aster_amd.paged_pool import PagedStatePool
from aster_amd.runner import PagedAttentionStep
from tests.bounded_rows import attend_row, check_out, check_weights
from tests.llama_like import LlamaLike
from tests.test_gpu_evict import chosen

pytestmark = pytest.mark.gpu

LAYERS, HEADS, KV, DIM = 2, 8, 2, 64


def make_pool(device, blocks=64):
    return PagedStatePool(PagedKVCache(num_blocks=blocks, num_layers=LAYERS, num_kv_heads=KV,
                                       head_dim=DIM, device=device))


class Loop:
    """A serving loop with random projections that checks every attention call and eviction."""

    def __init__(self, device, dtype, rows):
        self.device, self.dtype = device, dtype
        self.pool = make_pool(device)
        self.weights = KeyWeights(self.pool.cache, rows=rows, capacity=160)
        self.weights.values.fill_(float("nan"))  # nothing reads what was not gathered
        self.gathered = {}  # row -> [LAYERS, KV, tokens] in 64 bits
        self.gen = torch.Generator(device=device).manual_seed(7)
        self.unit, self.added = 0.0, 0

    def randn(self, *shape):
        return torch.randn(shape, generator=self.gen, device=self.device).to(self.dtype)

    def step(self, seqs, rows, counts):
        pool, total = self.pool, sum(counts)
        with PagedAttentionStep(pool, seqs, counts, key_weights=self.weights.select(rows)) as step:
            assert step.positions == [s.length + s.evicted for s in seqs]
            for layer in range(LAYERS):
                q, k, v = self.randn(total, HEADS, DIM), self.randn(total, KV, DIM), self.randn(total, KV, DIM)
                out = step.attend(layer, q, k, v)
                at = 0
                for r, (n, res) in enumerate(zip(counts, step.reservations)):
                    table = [p.index for p in res.pages]
                    want, absolute, unit, w = attend_row(pool.cache, np.array(table), res.length, q[at:at + n],
                                                         layer=layer)
                    check_out(out[at:at + n], want, absolute, unit, chunk=n > 1)
                    self.unit = max(self.unit, unit)
                    old = self.gathered.setdefault(rows[r], torch.zeros((LAYERS, KV, 0), dtype=torch.float64,
                                                                        device=self.device))
                    if layer == 0:
                        fresh = torch.zeros((LAYERS, KV, n), dtype=torch.float64, device=self.device)
                        self.gathered[rows[r]] = torch.cat([old[..., :res.start], fresh], -1)
                    self.gathered[rows[r]][layer] += w
                    at += n
        self.added += 1
        for row in rows:
            have = self.gathered[row]
            check_weights(self.weights.values[row][..., :have.shape[-1]], have, self.unit,
                          terms=64 * HEADS * self.added)

    def evict(self, seqs, rows, **budget):
        before = [self.pool.materialize(s) for s in seqs]
        lengths, evicted = [s.length for s in seqs], [s.evicted for s in seqs]
        held = self.weights.values.cpu().numpy()
        self.pool.evict(seqs, self.weights.select(rows), **budget)
        keep, recent, sinks = budget["keep"], budget.get("recent", 0), budget.get("sinks", 0)
        for s, row, state, n, gone in zip(seqs, rows, before, lengths, evicted):
            now = self.pool.materialize(s)
            assert s.length == min(n, keep) and s.evicted == gone + n - s.length
            kept = torch.zeros((LAYERS, KV, s.length), dtype=torch.float64, device=self.device)
            for layer in range(LAYERS):
                for h in range(KV):
                    stay = chosen(held[row, layer, h, :n], np.ones(n, bool), keep, sinks, recent)
                    for x, y in zip(now[layer], state[layer]):
                        assert torch.equal(x[0, h], y[0, h, stay])
                    kept[layer, h] = self.gathered[row][layer, h, stay]
            self.gathered[row] = kept


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_serving_loop_with_a_budget(device, dtype):
    loop = Loop(device, dtype, rows=5)
    pool = loop.pool
    a, b, c = (pool.create("tenant") for _ in range(3))
    loop.step([a, b, c], [3, 0, 4], [50, 3, 33])        # prompts
    for _ in range(3):
        loop.step([a, b, c], [3, 0, 4], [1, 1, 1])      # decode
    loop.evict([a, b, c], [3, 0, 4], keep=24, recent=8, sinks=2)
    loop.step([c, a], [4, 3], [1, 1])                   # another order, a row left out
    loop.step([a, b, c], [3, 0, 4], [20, 1, 1])         # a chunk beside decode rows
    # a fork shares pages; its weights go on apart
    child = pool.fork(a)
    loop.weights.values[1].copy_(loop.weights.values[3])
    loop.gathered[1] = loop.gathered[3].clone()
    loop.step([a, child], [3, 1], [1, 1])               # copy-on-write of the shared tail
    loop.evict([child], [1], keep=16, recent=4)         # shared pages: into fresh ones
    loop.evict([a, c], [3, 4], keep=16, recent=4, sinks=4)
    for _ in range(18):
        loop.step([a, child, c, b], [3, 1, 4, 0], [1, 1, 1, 1])
        if a.length > 24:
            loop.evict([a, child, c], [3, 1, 4], keep=20, recent=8, sinks=1)
    for s in (a, b, c, child):
        pool.release(s)
    assert pool.used_blocks == 0


def test_an_aborted_step_rolls_back_and_the_next_one_gathers_anew(device):
    loop = Loop(device, torch.bfloat16, rows=1)
    seq = loop.pool.create("tenant")
    loop.step([seq], [0], [20])
    kept = loop.weights.values.clone()
    x = loop.randn(1, HEADS, DIM)
    kv = loop.randn(1, KV, DIM)
    with pytest.raises(RuntimeError, match="stop"):
        with PagedAttentionStep(loop.pool, [seq], [1], key_weights=loop.weights.select([0])) as step:
            step.attend(0, x, kv, kv)
            raise RuntimeError("stop")
    assert seq.length == 20
    assert torch.equal(loop.weights.values[:, 1].contiguous().view(torch.int32),
                       kept[:, 1].contiguous().view(torch.int32))
    # the aborted token's place starts at 0 again
    loop.weights.values[..., :20].copy_(kept[..., :20])
    loop.step([seq], [0], [1])


def test_steps_check_their_key_weights(device):
    pool = make_pool(device)
    seq = pool.create("tenant")
    small = KeyWeights(pool.cache, rows=2, capacity=16)
    for bad in (small.select([0]), small.select([0, 1]), small):
        with pytest.raises(ValueError):
            PagedAttentionStep(pool, [seq], [20], key_weights=bad)
        assert pool.used_blocks == 0


def test_evicted_sequences_through_the_archive(device):
    loop = Loop(device, torch.bfloat16, rows=1)
    seq = loop.pool.create("tenant")
    loop.step([seq], [0], [60])
    loop.evict([seq], [0], keep=40, recent=4)
    archive = PagedStateArchive(loop.pool)
    handle = archive.put(seq)
    loop.pool.release(seq)
    back = archive.restore(handle, identity="tenant")
    assert (back.length, back.evicted, back.floor) == (40, 20, 40)
    loop.step([back], [0], [1])
    with pytest.raises(ValueError, match="eviction"):
        loop.pool.truncate(back, 39)


SINK_LAYERS = ((None, 0), (12, 3))


# ---- a decoder ---------------------------------------------------------------------------


def checked(monkeypatch, runner, layers):
    """Checks every attention call of ``runner`` against 64 bits over the arena's pages, and
    collects the positions its layers' rotary embeddings see. ``layers``: (window, sinks) each."""
    real, positions = PagedAttentionStep.attend, []

    def attend(step, layer, query, key, value, **kw):
        window, sinks = layers[layer]
        assert kw["window"] == window and (kw["sinks"] or 0) == sinks
        out = real(step, layer, query, key, value, **kw)
        if not sinks and step.key_weights is None:
            return out  # the calls that were there before have their own tests
        at = 0
        for n, res in zip(step.counts, step.reservations):
            table = np.array([p.index for p in res.pages])
            want, absolute, unit, _ = attend_row(step.pool.cache, table, res.length, query[at:at + n],
                                                 scale=kw["scale"], window=window, sinks=sinks, layer=layer)
            check_out(out[at:at + n], want, absolute, unit, chunk=n > 1)
            at += n
        return out

    monkeypatch.setattr(PagedAttentionStep, "attend", attend)
    for layer in runner.model.model.layers:
        layer.self_attn.rope.register_forward_pre_hook(
            lambda module, args: positions.append(args[1].cpu().tolist()))
    return positions


def make_runner(model, device):
    return PagedAttentionRunner(model.to(device), policy_artifact_id="test", backend="hip_int8_paged",
                                max_blocks=64)


def test_decoder_with_sink_tokens(device, monkeypatch):
    """Prompt, chunk and decode tokens of a decoder whose windowed layer keeps three sinks; the
    logits differ from those without."""
    model = LlamaLike(windows=(None, 12))
    rng = np.random.default_rng(3)
    ids = [rng.integers(0, 97, 40).tolist() for _ in range(2)]
    plain = make_runner(LlamaLike(windows=(None, 12)), device)
    apart = [plain.pool.create("t") for _ in ids]
    spans = ((0, 30), (30, 38), (38, 39), (39, 40))
    without = [plain.forward_batch(apart, [x[lo:hi] for x in ids]) for lo, hi in spans]
    model.model.layers[1].self_attn.sink_tokens = 3
    runner = make_runner(model, device)
    seqs = [runner.pool.create("t") for _ in ids]
    checked(monkeypatch, runner, SINK_LAYERS)
    for (lo, hi), other in zip(spans, without):
        got = runner.forward_batch(seqs, [x[lo:hi] for x in ids])
        assert all(torch.isfinite(x).all() for x in got)
        assert not np.allclose(other[0].numpy(), got[0].numpy(), atol=1e-2)


def test_decoder_goes_on_behind_its_evictions(device, monkeypatch):
    """After an eviction the next token's position counts the dropped ones, and each KV head
    attends to its own tokens."""
    rng = np.random.default_rng(4)
    ids = rng.integers(0, 97, 42).tolist()
    runner = make_runner(LlamaLike(windows=(None, None)), device)
    seq = runner.pool.create("t")
    runner.forward_batch([seq], [ids[:1]])
    weights = KeyWeights(runner.pool.cache, rows=1, capacity=64)
    row = weights.select([0])
    runner.pool.truncate(seq, 0)
    positions = checked(monkeypatch, runner, ((None, 0), (None, 0)))
    runner.forward_batch([seq], [ids[:40]], key_weights=row)
    assert all(p == [list(range(40))] for p in positions) and len(positions) == 4  # q and k, two layers
    runner.pool.evict([seq], row, keep=16, recent=6, sinks=1)
    del positions[:]
    runner.forward_batch([seq], [ids[40:]], key_weights=row)
    assert all(p == [[40, 41]] for p in positions) and seq.length == 18 and seq.evicted == 24
    monkeypatch.undo()
    windowed = make_runner(LlamaLike(windows=(None, 12)), device)
    other = windowed.pool.create("t")
    windowed.forward_batch([other], [ids[:20]])
    with pytest.raises(UnsupportedAttentionBackend, match="window"):
        windowed.forward_batch([other], [ids[20:21]], key_weights=KeyWeights(
            windowed.pool.cache, rows=1, capacity=64).select([0]))
    assert other.length == 20


def test_positions_past_the_model_are_refused_with_evictions_counted(device):
    model = LlamaLike(windows=(None,), max_positions=48)
    runner = make_runner(model, device)
    seq = runner.pool.create("t")
    runner.forward_batch([seq], [[1] * 4])
    weights = KeyWeights(runner.pool.cache, rows=1, capacity=64)
    runner.forward_batch([seq], [[1] * 36])
    weights.values.zero_()
    runner.pool.evict([seq], weights.select([0]), keep=16)
    assert seq.evicted == 24
    runner.forward_batch([seq], [[1] * 8])
    with pytest.raises(ValueError, match="position"):
        runner.forward_batch([seq], [[1]])

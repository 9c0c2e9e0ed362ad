"""Attention of a bounded cache against plain 64-bit results: windows beside which the first
tokens stay visible, and softmax weights gathered per key, for rows of one token and chunks."""

import ctypes

import numpy as np
import pytest
import torch

from aster_amd import KernelWork, KeyWeights, _native
from tests.bounded_rows import attend_row, check_out, check_weights, make_arena, on

pytestmark = pytest.mark.gpu

FORMATS = ("int8", "fp8_e4m3fn", "fp8_e5m2")
DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def queries(device, tokens, heads, dim, dtype, seed=1, scale=1.0):
    gen = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn((tokens, heads, dim), generator=gen, device=device) * scale).to(dtype)


def run_sinks(cache, tables, lens, q, window, sinks, counts=None, **kw):
    dev = cache.device
    if counts is not None:
        starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        kw.update(query_start_loc=on(dev, starts), max_query_len=int(max(counts)))
    return cache.paged_attention(0, q, on(dev, tables), on(dev, np.asarray(lens, np.int32)),
                                 max_context_len=int(max(max(lens), 1)), window=window, sinks=sinks,
                                 check=True, **kw)


def check_rows(cache, tables, lens, q, out, counts=None, weights=None, before=None, rows=None,
               chunk_kernel=None, **kw):
    counts = [1] * len(lens) if counts is None else counts
    at = 0
    for r, (n, ctx) in enumerate(zip(counts, lens)):
        if n == 0:
            continue
        if ctx == 0:
            assert (out[at:at + n] == 0).all()
            at += n
            continue
        want, absolute, unit, w64 = attend_row(cache, tables[r], ctx, q[at:at + n], **kw)
        chunk = n > 1 if chunk_kernel is None else chunk_kernel
        check_out(out[at:at + n], want, absolute, unit, chunk=chunk)
        if weights is not None:
            old = before[rows[r]].double()
            expect = old.clone()
            expect[:, ctx - n:ctx] = 0
            expect[:, :ctx] += w64
            check_weights(weights[rows[r]][:, :ctx], expect[:, :ctx], unit, terms=n * q.shape[1])
            assert torch.equal(weights[rows[r]][:, ctx:].view(torch.int32),
                               before[rows[r]][:, ctx:].view(torch.int32))
        at += n


LENS = [1, 0, 15, 16, 17, 31, 63, 64, 65, 130, 200, 257, 700]


@pytest.mark.parametrize("window,sinks", [(1, 1), (16, 4), (17, 1), (64, 16), (100, 5), (64, 33),
                                          (5, 700), (1000, 3), (48, 64)])
def test_windows_and_sinks(device, window, sinks):
    """Every meeting of window and sinks: apart, in one block, touching, overlapping, past the
    row; sinks and rows that end inside a block."""
    cache, tables, _ = make_arena(device, LENS, kv_heads=2, dim=64)
    q = queries(device, len(LENS), 8, 64, torch.float32)
    out = run_sinks(cache, tables, LENS, q, window, sinks)
    check_rows(cache, tables, LENS, q, out, window=window, sinks=sinks)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 4), (128, 8, 2), (256, 2, 1), (128, 16, 1),
                                                (256, 16, 1), (64, 16, 2)])
def test_decode_types_and_layouts(device, fmt, dtype, dim, heads, kv_heads):
    lens = [1, 40, 333, 1500, 2049]
    cache, tables, _ = make_arena(device, lens, kv_heads=kv_heads, dim=dim, fmt=fmt, padding=0.1)
    q = queries(device, len(lens), heads, dim, dtype)
    out = run_sinks(cache, tables, lens, q, 300, 7)
    check_rows(cache, tables, lens, q, out, window=300, sinks=7)


@pytest.mark.parametrize("rows", [1, 3, 70, 300])
@pytest.mark.parametrize("window", [512, 4096])
def test_decode_batches(device, rows, window):
    """Few rows (wide workgroups, rows cut into pieces) and many (one workgroup a row)."""
    rng = np.random.default_rng(rows)
    lens = rng.integers(1, 6000 if rows < 100 else 900, size=rows).tolist()
    lens[-1] = 5000 if rows < 100 else 900
    cache, tables, _ = make_arena(device, lens, kv_heads=4, dim=64)
    q = queries(device, rows, 8, 64, torch.bfloat16)
    out = run_sinks(cache, tables, lens, q, window, 20)
    check_rows(cache, tables, lens, q, out, window=window, sinks=20)


@pytest.mark.parametrize("v_scale,k_scale,q_scale", [(1e-30, 1.0, 1.0), (1e30, 1.0, 1.0),
                                                     (1.0, 40.0, 1.0), (1.0, 1e-6, 3e5),
                                                     (1.0, 1e6, 1e-6)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_decode_magnitudes(device, fmt, v_scale, k_scale, q_scale):
    lens = [5, 90, 400]
    cache, tables, _ = make_arena(device, lens, kv_heads=2, dim=128, fmt=fmt, v_scale=v_scale,
                                  k_scale=k_scale)
    q = queries(device, 3, 8, 128, torch.float32, scale=q_scale)
    out = run_sinks(cache, tables, lens, q, 64, 4)
    check_rows(cache, tables, lens, q, out, window=64, sinks=4)


def test_mixed_value_scales(device):
    """V scales that grow and shrink by powers of ten along a row."""
    lens = [600]
    cache, tables, _ = make_arena(device, lens, kv_heads=1, dim=64)
    factor = 10.0 ** torch.randint(-6, 7, (cache.num_blocks,), device=device).float()
    cache.scales[:, :, 1] *= factor[:, None, None, None]
    q = queries(device, 1, 4, 64, torch.float32)
    out = run_sinks(cache, tables, lens, q, 500, 32)
    check_rows(cache, tables, lens, q, out, window=500, sinks=32)


def test_rows_without_a_visible_key(device):
    lens = [40, 100, 0]
    cache, tables, _ = make_arena(device, lens, kv_heads=2, dim=64, padding=1e-9)
    pages = on(device, tables[0][:3].astype(np.int64))
    cache.key_valid[pages] = 0
    q = queries(device, 3, 4, 64, torch.bfloat16)
    out = run_sinks(cache, tables, lens, q, 16, 4)
    assert (out[0] == 0).all() and (out[2] == 0).all()
    check_rows(cache, tables, lens, q, out, window=16, sinks=4)
    kw = KeyWeights(cache, rows=3, capacity=112)
    kw.values.fill_(0.5)
    out = cache.paged_attention_weights(0, q, on(device, tables), on(device, np.asarray(lens, np.int32)),
                                        kw.select([2, 1, 0]), max_context_len=100, check=True)
    assert (out[0] == 0).all() and (out[2] == 0).all()
    assert (kw.values[0] == 0.5).all()                       # the row without a token
    assert (kw.values[2, 0, :, 39] == 0).all()               # its new token, unseen as padding
    assert (kw.values[2, 0, :, :39] == 0.5).all()


def test_pages_between_sinks_and_window_are_not_read(device):
    lens = [900, 450]
    cache, tables, _ = make_arena(device, lens, kv_heads=2, dim=64)
    q = queries(device, 2, 4, 64, torch.bfloat16)
    want = run_sinks(cache, tables, lens, q, 100, 20)
    holes = tables.copy()
    holes[0, 2:(900 - 100) // 16] = 1 << 30
    holes[1, 2:(450 - 100) // 16] = -7
    assert torch.equal(run_sinks(cache, holes, lens, q, 100, 20), want)
    chunk = queries(device, 60, 4, 64, torch.bfloat16)
    want = run_sinks(cache, tables, lens, chunk, 100, 20, counts=[40, 20])
    holes[0, 2:(860 - 100) // 16] = 1 << 30
    holes[0, (860 - 100) // 16:] = tables[0, (860 - 100) // 16:]
    holes[1] = tables[1]
    assert torch.equal(run_sinks(cache, holes, lens, chunk, 100, 20, counts=[40, 20]), want)


def test_strided_rows_and_outputs(device):
    lens = [30, 500, 77]
    cache, tables, _ = make_arena(device, lens, kv_heads=2, dim=128)
    wide = queries(device, 3, 24, 256, torch.float16)
    q = wide[:, 4:12, 64:192]
    buffer = torch.full((3, 3, 8, 128), 7.0, dtype=torch.float16, device=device)
    out = run_sinks(cache, tables, lens, q, 60, 2, out=buffer[:, 1])
    assert out.data_ptr() == buffer[:, 1].data_ptr()
    assert (buffer[:, 0] == 7).all() and (buffer[:, 2] == 7).all()
    check_rows(cache, tables, lens, q, out, window=60, sinks=2)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 4), (128, 8, 2), (256, 2, 1), (64, 16, 1)])
def test_chunks(device, fmt, dtype, dim, heads, kv_heads):
    counts = [3, 40, 130, 2]
    lens = [3, 300, 520, 700]
    cache, tables, _ = make_arena(device, lens, kv_heads=kv_heads, dim=dim, fmt=fmt, padding=0.05)
    q = queries(device, sum(counts), heads, dim, dtype)
    out = run_sinks(cache, tables, lens, q, 150, 6, counts=counts)
    check_rows(cache, tables, lens, q, out, counts, window=150, sinks=6)


@pytest.mark.parametrize("window,sinks", [(1, 1), (16, 4), (33, 70), (64, 64), (100, 257), (2000, 3),
                                          (5, 900), (40, 130)])
def test_chunk_windows_and_sinks(device, window, sinks):
    """Sinks of more than a key step, reaching into the window of some of a tile's tokens."""
    counts, lens = [200, 64, 2, 17], [200, 700, 900, 64]
    cache, tables, _ = make_arena(device, lens, kv_heads=2, dim=64)
    q = queries(device, sum(counts), 4, 64, torch.bfloat16)
    out = run_sinks(cache, tables, lens, q, window, sinks, counts=counts)
    check_rows(cache, tables, lens, q, out, counts, window=window, sinks=sinks)


def test_long_chunk_in_pieces(device):
    """A chunk whose units are cut into key ranges, the sinks in the first of them."""
    cache, tables, _ = make_arena(device, [6000], kv_heads=2, dim=128)
    q = queries(device, 64, 8, 128, torch.float16)
    out = run_sinks(cache, tables, [6000], q, 5000, 100, counts=[64])
    check_rows(cache, tables, [6000], q, out, [64], window=5000, sinks=100)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_mixed_step(device, dtype):
    counts = [1, 40, 1, 0, 1, 9]
    lens = [500, 40, 0, 33, 17, 300]
    cache, tables, _ = make_arena(device, lens, kv_heads=2, dim=128)
    q = queries(device, sum(counts), 8, 128, dtype)
    out = run_sinks(cache, tables, lens, q, 30, 3, counts=counts)
    check_rows(cache, tables, lens, q, out, counts, window=30, sinks=3)


# ---- key weights -----------------------------------------------------------------------


def run_weights(cache, tables, lens, q, kw, rows, counts=None, **extra):
    dev = cache.device
    if counts is not None:
        starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        extra.update(query_start_loc=on(dev, starts), max_query_len=int(max(counts)))
    return cache.paged_attention_weights(0, q, on(dev, tables), on(dev, np.asarray(lens, np.int32)),
                                         kw.select(rows), max_context_len=int(max(lens)), check=True,
                                         **extra)


def gathered(cache, lens, rows, seed=5, counts=None):
    """Key weights with some history; what the new tokens' places hold is NaN."""
    kw = KeyWeights(cache, rows=len(lens) + 2, capacity=max(lens) + 40)
    gen = torch.Generator(device=cache.device).manual_seed(seed)
    kw.values.copy_(torch.rand(kw.values.shape, generator=gen, device=cache.device))
    for r, ctx in enumerate(lens):
        kw.values[rows[r], :, :, ctx - (1 if counts is None else counts[r]):] = float("nan")
    return kw


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 4), (128, 8, 2), (256, 2, 1), (128, 16, 1)])
def test_decode_weights(device, fmt, dtype, dim, heads, kv_heads):
    lens = [1, 16, 33, 700, 2500]
    rows = [4, 0, 6, 1, 3]
    cache, tables, _ = make_arena(device, lens, kv_heads=kv_heads, dim=dim, fmt=fmt, padding=0.1)
    kw = gathered(cache, lens, rows)
    before = kw.values[:, 0].clone()
    q = queries(device, len(lens), heads, dim, dtype)
    out = run_weights(cache, tables, lens, q, kw, rows)
    check_rows(cache, tables, lens, q, out, weights=kw.values[:, 0], before=before, rows=rows)
    for other in set(range(kw.rows)) - set(rows):
        assert torch.equal(kw.values[other, 0], before[other])


@pytest.mark.parametrize("rows", [1, 70, 200])
def test_decode_weights_batches(device, rows):
    rng = np.random.default_rng(rows)
    lens = rng.integers(1, 3000, size=rows).tolist()
    lens[0] = 5001
    cache, tables, _ = make_arena(device, lens, kv_heads=2, dim=64)
    ids = rng.permutation(rows + 2)[:rows].tolist()
    kw = gathered(cache, lens, ids)
    before = kw.values[:, 0].clone()
    q = queries(device, rows, 8, 64, torch.bfloat16)
    out = run_weights(cache, tables, lens, q, kw, ids)
    check_rows(cache, tables, lens, q, out, weights=kw.values[:, 0], before=before, rows=ids)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 4), (128, 8, 2), (256, 2, 1), (64, 16, 1)])
def test_chunk_weights(device, fmt, dtype, dim, heads, kv_heads):
    counts = [2, 33, 130, 65]
    lens = [2, 300, 130, 700]
    rows = [1, 5, 0, 2]
    cache, tables, _ = make_arena(device, lens, kv_heads=kv_heads, dim=dim, fmt=fmt, padding=0.05)
    kw = gathered(cache, lens, rows, counts=counts)
    before = kw.values[:, 0].clone()
    q = queries(device, sum(counts), heads, dim, dtype)
    out = run_weights(cache, tables, lens, q, kw, rows, counts)
    check_rows(cache, tables, lens, q, out, counts, kw.values[:, 0], before, rows)


def test_chunk_weights_in_pieces_and_mixed(device):
    counts = [64, 1, 1, 20, 0]
    lens = [6000, 300, 1, 21, 50]
    rows = [0, 1, 2, 3, 4]
    cache, tables, _ = make_arena(device, lens, kv_heads=2, dim=128)
    kw = gathered(cache, lens, rows, counts=[max(c, 1) for c in counts])
    kw.values[4] = 0.25
    before = kw.values[:, 0].clone()
    q = queries(device, sum(counts), 8, 128, torch.bfloat16)
    out = run_weights(cache, tables, lens, q, kw, rows, counts)
    check_rows(cache, tables, lens, q, out, counts, kw.values[:, 0], before, rows)
    assert torch.equal(kw.values[4, 0], before[4])  # no query, nothing gathered


def test_weights_of_one_layer_leave_the_others(device):
    lens = [40, 90]
    cache, tables, _ = make_arena(device, lens, kv_heads=2, dim=64, layers=3)
    kw = KeyWeights(cache, rows=2, capacity=90)
    q = queries(device, 2, 4, 64, torch.bfloat16)
    work = KernelWork()
    cache.paged_attention_weights(1, q, on(device, tables), on(device, np.asarray(lens, np.int32)),
                                  kw.select([0, 1]), max_context_len=90, check=True, work=work)
    assert (kw.values[:, [0, 2]] == 0).all() and work.backend == "hip_int8_paged"
    # every query's weights sum to 1 per head
    assert torch.allclose(kw.values[:, 1].sum(-1), torch.full((2, 2), 2.0, device=device), atol=1e-5)


def test_weights_do_not_depend_on_the_run(device):
    counts, lens = [100, 1, 30], [400, 2000, 30]
    cache, tables, _ = make_arena(device, lens, kv_heads=2, dim=128)
    q = queries(device, sum(counts), 8, 128, torch.bfloat16)
    got = []
    for _ in range(3):
        kw = KeyWeights(cache, rows=3, capacity=2000)
        run_weights(cache, tables, lens, q, kw, [0, 1, 2], counts)
        got.append(kw.values)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_non_finite_scores_are_reported_and_add_nothing(device):
    for counts, lens in ((None, [50, 60]), ([20, 30], [50, 60])):
        cache, tables, _ = make_arena(device, lens, kv_heads=1, dim=64)
        total = 2 if counts is None else sum(counts)
        q = queries(device, total, 2, 64, torch.float32)
        q[0, 0, 3] = float("inf")
        kw = KeyWeights(cache, rows=2, capacity=64)
        with pytest.raises(ValueError, match="overflow"):
            run_weights(cache, tables, lens, q, kw, [0, 1], counts)
        assert torch.isfinite(kw.values).all()
        assert (kw.values[1, 0, :, :60].sum() > 0).all()


@pytest.mark.parametrize("v_scale,k_scale,q_scale", [(1e-30, 1.0, 1.0), (1e30, 1.0, 1.0),
                                                     (1.0, 40.0, 1.0), (1.0, 1e-6, 3e5),
                                                     (1.0, 1e6, 1e-6)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_chunk_magnitudes(device, dtype, v_scale, k_scale, q_scale):
    counts, lens = [70, 5, 40], [90, 5, 400]
    cache, tables, _ = make_arena(device, lens, kv_heads=2, dim=128, v_scale=v_scale, k_scale=k_scale)
    q = queries(device, sum(counts), 8, 128, dtype, scale=q_scale)
    out = run_sinks(cache, tables, lens, q, 64, 4, counts)
    check_rows(cache, tables, lens, q, out, counts, window=64, sinks=4)
    kw = gathered(cache, lens, [0, 1, 2], counts=counts)
    before = kw.values[:, 0].clone()
    out = run_weights(cache, tables, lens, q, kw, [0, 1, 2], counts)
    check_rows(cache, tables, lens, q, out, counts, kw.values[:, 0], before, [0, 1, 2])


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_non_finite_query_leaves_the_others_weights(device, dtype):
    cache, tables, _ = make_arena(device, [90], kv_heads=2, dim=64)
    q = queries(device, 40, 2, 64, dtype)
    plain = q.clone()
    plain[7] = 0
    q[7] = float("nan")
    kw = KeyWeights(cache, rows=1, capacity=96)
    with pytest.raises(ValueError, match="overflow"):
        run_weights(cache, tables, [90], q, kw, [0], [40])
    _, _, unit, every = attend_row(cache, tables[0], 90, plain)
    without = attend_row(cache, tables[0], 58, plain[7:8])[3]  # token 7 sees 58 keys
    every[:, :58] -= without
    check_weights(kw.values[0, 0, :, :90], every, unit, terms=40)


def test_chunks_past_the_host_bound_are_cut_and_reported(device):
    counts, lens = [30, 20], [50, 90]
    cache, tables, _ = make_arena(device, lens, kv_heads=1, dim=64)
    q = queries(device, sum(counts), 2, 64, torch.bfloat16)
    starts = on(device, np.array([0, 30, 50], np.int32))
    args = (0, q, on(device, tables), on(device, np.asarray(lens, np.int32)))
    with pytest.raises(ValueError, match="outside the KV arena"):
        cache.paged_attention(*args, max_context_len=60, window=16, sinks=2, query_start_loc=starts,
                              max_query_len=30, check=True)
    kw = KeyWeights(cache, rows=2, capacity=96)
    kw.values.fill_(0.5)
    before = kw.values[:, 0].clone()
    out = torch.empty_like(q)
    with pytest.raises(ValueError, match="outside the KV arena"):
        cache.paged_attention_weights(*args, kw.select([0, 1]), max_context_len=60, out=out,
                                      query_start_loc=starts, max_query_len=30, check=True)
    # the row within the bound as ever, the other one as if it ended there
    check_rows(cache, tables, [50, 60], q, out, counts, kw.values[:, 0], before, [0, 1])


def test_lengths_and_ids_out_of_range_are_reported(device):
    lens = [50, 60]
    cache, tables, _ = make_arena(device, lens, kv_heads=1, dim=64)
    q = queries(device, 2, 2, 64, torch.bfloat16)
    bad = tables.copy()
    bad[0, 1] = cache.num_blocks
    with pytest.raises(ValueError, match="outside the KV arena"):
        run_sinks(cache, bad, lens, q, 40, 2)
    kw = KeyWeights(cache, rows=2, capacity=64)
    with pytest.raises(ValueError, match="outside the KV arena"):
        run_weights(cache, bad, lens, q, kw, [0, 1])
    assert torch.isfinite(kw.values).all()
    with pytest.raises(ValueError, match="outside the KV arena"):  # longer than the host's bound
        cache.paged_attention_weights(0, q, on(device, tables), on(device, np.array([50, 61], np.int32)),
                                      kw.select([0, 1]), max_context_len=60, check=True)
    with pytest.raises(ValueError, match="outside the KV arena"):
        cache.paged_attention(0, q, on(device, tables), on(device, np.array([-1, 60], np.int32)),
                              max_context_len=60, window=8, sinks=2, check=True)
    # a row number past the weights' rows, through the C entry: nothing is gathered for it
    kw = KeyWeights(cache, rows=2, capacity=64)
    rows = kw.select([0, 1])
    rows.table.copy_(torch.tensor([0, 2], dtype=torch.int32))
    with pytest.raises(ValueError, match="outside the KV arena"):
        cache.paged_attention_weights(0, q, on(device, tables), on(device, np.asarray(lens, np.int32)),
                                      rows, max_context_len=60, check=True)
    assert (kw.values[1] == 0).all() and (kw.values[0] != 0).any()


def test_on_another_stream(device):
    lens = [3000, 77]
    cache, tables, _ = make_arena(device, lens, kv_heads=2, dim=128)
    q = queries(device, 2, 8, 128, torch.bfloat16)
    want = run_sinks(cache, tables, lens, q, 2000, 9)
    t, n = on(device, tables), on(device, np.asarray(lens, np.int32))
    side = torch.cuda.Stream()
    ws = torch.empty(max(256, cache.bounded_workspace_bytes(2, 8, 3000, q.dtype, window=2000, sinks=9)),
                     dtype=torch.uint8, device=device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = cache.paged_attention(0, q, t, n, max_context_len=3000, window=2000, sinks=9,
                                    workspace=ws)
    side.synchronize()
    assert torch.equal(out, want)


def test_graphs_replay(device):
    """A step of sink windows and one that gathers weights, each captured with a workspace of
    its own and replayed between eager work: every replay as the eager call."""
    counts, lens = [40, 1, 1], [300, 2500, 90]
    cache, tables, _ = make_arena(device, lens, kv_heads=2, dim=64)
    q = queries(device, sum(counts), 8, 64, torch.bfloat16)
    t, n = on(device, tables), on(device, np.asarray(lens, np.int32))
    starts = on(device, np.array([0, 40, 41, 42], np.int32))
    kw = KeyWeights(cache, rows=3, capacity=2500)
    rows = kw.select([2, 0, 1])
    common = dict(max_context_len=2500, query_start_loc=starts, max_query_len=40)
    sizes = [cache.bounded_workspace_bytes(3, 8, 2500, q.dtype, window=200, sinks=5,
                                           num_query_tokens=42, max_query_len=40),
             cache.bounded_workspace_bytes(3, 8, 2500, q.dtype, key_weights=True,
                                           num_query_tokens=42, max_query_len=40)]
    spaces = [torch.empty(max(s, 256), dtype=torch.uint8, device=device) for s in sizes]
    outs = [torch.empty_like(q), torch.empty_like(q)]

    def sink_step():
        cache.paged_attention(0, q, t, n, window=200, sinks=5, out=outs[0], workspace=spaces[0], **common)

    def weight_step():
        cache.paged_attention_weights(0, q, t, n, rows, out=outs[1], workspace=spaces[1], **common)

    sink_step(), weight_step()
    torch.cuda.synchronize()
    first, want = kw.values.clone(), [o.clone() for o in outs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sink_step(), weight_step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for step in (sink_step, weight_step):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append(graph)
    for _ in range(3):
        for o in outs:
            o.fill_(float("nan"))
        kw.values.zero_()
        run_sinks(cache, tables, lens, q, 30, 2, counts=counts)  # eager work between
        torch.cuda.synchronize()
        graphs[0].replay(), graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        assert torch.equal(kw.values, first)
    cache.raise_errors()


def test_positions_past_two_gigabytes(device):
    """Pages whose codes lie past 2^31 bytes of the arena."""
    from aster_amd import PagedKVCache

    blocks = (1 << 31) // (2 * 8 * 16 * 128) + 70  # a block of one layer: 32 KB
    cache = PagedKVCache(num_blocks=blocks, num_layers=1, num_kv_heads=8, head_dim=128, device=device)
    high = np.arange(blocks - 64, blocks, dtype=np.int32)[None]
    gen = torch.Generator(device=device).manual_seed(3)
    cache.codes[-64:] = torch.randint(-127, 128, cache.codes[-64:].shape, generator=gen,
                                      device=device, dtype=torch.int8)
    cache.scales[-64:] = 0.02
    q = queries(device, 1, 8, 128, torch.bfloat16)
    out = run_sinks(cache, high, [1000], q, 500, 40)
    check_rows(cache, high, [1000], q, out, window=500, sinks=40)
    chunk = queries(device, 30, 8, 128, torch.bfloat16)
    kw = KeyWeights(cache, rows=1, capacity=1000)
    before = kw.values[:, 0].clone()
    out = run_weights(cache, high, [1000], chunk, kw, [0], [30])
    check_rows(cache, high, [1000], chunk, out, [30], kw.values[:, 0], before, [0])


def test_streams_have_workspaces_of_their_own(device):
    lens = [6000, 77]
    cache, tables, _ = make_arena(device, lens, kv_heads=2, dim=128)
    q = queries(device, 2, 8, 128, torch.bfloat16)
    t, n = on(device, tables), on(device, np.asarray(lens, np.int32))
    calls = [dict(max_context_len=6000, window=5000, sinks=9),  # in pieces
             dict(max_context_len=6000, window=3500, sinks=3)]
    want = [cache.paged_attention(0, q, t, n, **c) for c in calls]
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for side, call in zip(sides, calls):
            with torch.cuda.stream(side):
                got.append(cache.paged_attention(0, q, t, n, **call))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i % 2]) for i, o in enumerate(got))


def test_a_captured_call_without_a_workspace_is_refused(device):
    lens = [6000]
    cache, tables, _ = make_arena(device, lens, kv_heads=2, dim=128)
    q = queries(device, 1, 8, 128, torch.bfloat16)
    t, n = on(device, tables), on(device, np.asarray(lens, np.int32))
    assert cache.bounded_workspace_bytes(1, 8, 6000, q.dtype, window=5000, sinks=9) > 0
    cell, graph = torch.zeros(4, device=device), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        cell.add_(1)
        with pytest.raises(ValueError, match="workspace of its own"):
            cache.paged_attention(0, q, t, n, max_context_len=6000, window=5000, sinks=9)
    graph.replay()
    torch.cuda.synchronize()
    assert (cell == 1).all()
    cache.raise_errors()


@pytest.mark.parametrize("counts", [[40, 1, 9], [20, 20, 20], [1, 1, 2]])
def test_rows_behind_the_last_sequence_stay(device, counts):
    lens = [300, 70, 20]
    cache, tables, _ = make_arena(device, lens, kv_heads=2, dim=128)
    q = queries(device, sum(counts) + 5, 8, 128, torch.bfloat16)
    out = torch.full_like(q, 3.0)
    run_sinks(cache, tables, lens, q, 50, 6, counts, out=out)
    check_rows(cache, tables, lens, q, out, counts, window=50, sinks=6)
    assert (out[sum(counts):] == 3).all()
    kw = gathered(cache, lens, [2, 0, 1], counts=counts)
    before = kw.values[:, 0].clone()
    run_weights(cache, tables, lens, q, kw, [2, 0, 1], counts, out=out.fill_(3))
    check_rows(cache, tables, lens, q, out, counts, kw.values[:, 0], before, [2, 0, 1])
    assert (out[sum(counts):] == 3).all()

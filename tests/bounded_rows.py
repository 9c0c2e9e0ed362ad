"""Plain 64-bit results of the operators of a bounded cache, with the errors that the kernels'
roundings allow, and arenas to run them on."""

import numpy as np
import torch

from aster_amd import KVQuantization, PagedKVCache

MAXIMUM = {"int8": 127.0, "fp8_e4m3fn": 448.0, "fp8_e5m2": 57344.0}


def make_arena(device, lens, *, kv_heads, dim, fmt="int8", layers=1, seed=0, spare=8, padding=0.0,
               v_scale=1.0, k_scale=1.0):
    """An arena of random codes and scales and shuffled tables for rows of ``lens`` tokens;
    table entries past a row's pages are -1."""
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=device).manual_seed(seed)
    pages = [-(-int(n) // 16) for n in lens]
    blocks = sum(pages) + spare
    cache = PagedKVCache(num_blocks=blocks, num_layers=layers, num_kv_heads=kv_heads, head_dim=dim,
                         device=device, quantization=KVQuantization(fmt))
    shape = cache.codes.shape
    x = torch.randn(shape, generator=gen, device=device)
    amax = x.abs().amax(-1)
    scales = amax / MAXIMUM[fmt]
    units = (x / scales[..., None]).clamp(-MAXIMUM[fmt], MAXIMUM[fmt])
    units = units.round() if fmt == "int8" else units
    cache.codes.copy_(units.to(cache.quantization.dtype).view(torch.int8))
    scales[:, :, 0] *= k_scale
    scales[:, :, 1] *= v_scale
    cache.scales.copy_(scales)
    if padding:
        valid = torch.rand((blocks * 16,), generator=gen, device=device) >= padding
        cache.write_key_valid(torch.arange(blocks * 16, device=device), valid)
    order = rng.permutation(blocks).astype(np.int32)
    tables = np.full((len(lens), max(1, max(pages))), -1, np.int32)
    at = 0
    for r, n in enumerate(pages):
        tables[r, :n] = order[at:at + n]
        at += n
    return cache, tables, order[at:]


def on(device, values):
    return torch.from_numpy(np.ascontiguousarray(values)).to(device)


def dequantized(cache, table, n, layer=0):
    """K, V ``[Hkv, n, D]`` in 64 bits and the real tokens of the first ``n`` of a row."""
    pages = torch.from_numpy(np.asarray(table[: -(-n // 16)], np.int64)).to(cache.device)
    x = cache.code_view(cache.codes[pages, layer]).double() * cache.scales[pages, layer].double()[..., None]
    x = x.permute(1, 2, 0, 3, 4).reshape(2, cache.num_kv_heads, -1, cache.head_dim)[:, :, :n]
    real = cache.key_valid[pages].reshape(-1)[:n].bool()
    return x[0], x[1], real


def attend_row(cache, table, ctx, q, *, scale=None, window=None, sinks=0, layer=0):
    """One row of ``n`` queries ``[n, Hq, D]``: (outputs, sum p|v|, a score's error in units of
    2^-21, key weights ``[Hkv, ctx]``), all in 64 bits."""
    n, heads, dim = q.shape
    group = heads // cache.num_kv_heads
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros((n, heads, dim), dtype=torch.float64, device=cache.device)
    absolute = torch.zeros_like(out)
    weights = torch.zeros((cache.num_kv_heads, ctx), dtype=torch.float64, device=cache.device)
    if ctx == 0:
        return out, absolute, 0.0, weights
    k, v, real = dequantized(cache, table, ctx, layer)
    keys = torch.arange(ctx, device=cache.device)
    pos = torch.arange(ctx - n, ctx, device=cache.device)[:, None]
    seen = (keys <= pos) & real
    if window is not None:
        seen &= (keys > pos - window) | (keys < sinks)
    q = q.double()
    for h in range(heads):
        kv = h // group
        s = (q[:, h] @ k[kv].t().contiguous()) * scale
        top = s.masked_fill(~seen, -torch.inf).amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top.isfinite(), top, 0.0)).masked_fill(~seen, 0.0)
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
        out[:, h] = p @ v[kv]
        absolute[:, h] = p @ v[kv].abs()
        weights[kv] += p.sum(0)
    unit = float(scale * q.abs().max() * k.abs().sum(-1).max()) if q.numel() else 0.0
    return out, absolute, unit, weights


def check_out(got, want, absolute, unit, *, chunk=False):
    """``got`` within its rounding to the query's type (half a step), the roundings of the
    softmax weights and a score's error: every score is within ``unit`` 2^-21 (22 bits of the
    query, fp32 sums), which moves a weight by e^(2 unit 2^-21) at most. bf16 queries: one f16
    rounding per weight (2^-11), others two f16 terms (2^-22); sums and the rest 2^-20. Rows of
    one token and chunks (``chunk``) alike."""
    eps = torch.finfo(got.dtype).eps / 2
    term = 2 ** -20 + (2 ** -11 if got.dtype == torch.bfloat16 else 0)
    error = absolute * (term + 3 * unit * 2 ** -21)
    # (below 2^-24 of the largest V scale's unit an f16 weight is a subnormal: 2^-25 absolute)
    error = error + absolute.amax() * 2 ** -20 * (1 if got.dtype != torch.float32 else 2 ** -4)
    limit = error + eps * (want.abs() + error) + torch.finfo(got.dtype).tiny
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= limit).all(), float((off / limit).max())


def check_weights(got, want, unit, *, terms):
    """fp32 sums of ``terms`` weights, each within its score's error and 2^-21."""
    limit = want * (3 * unit * 2 ** -21 + 2 ** -20 + terms ** 0.5 * 2 ** -22) + 1e-30
    off = (got.double() - want).abs()
    assert (off <= limit).all(), float((off / limit).max())

"""64-bit forms of the rotary and paged-cache operators on the CPU, and the bounds of their errors.

A rounding to a type is off by at most half a step: `unit(t)` = eps / 2 of the value."""
import math

import torch


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def rotate(x, positions, inv_freq, layout='interleaved', scale=1.0, inverse=False):
    """(float64 rotation of x [tokens, heads, dim], bound of the operator's error)."""
    x64, pairs = x.double().cpu(), inv_freq.numel()
    p = positions.double().cpu().reshape(x.shape[0], -1)
    angle = p.repeat_interleave(pairs // p.shape[1], 1) * inv_freq.cpu()
    cos, sin = (angle.cos() * scale)[:, None], (angle.sin() * scale)[:, None] * (-1 if inverse else 1)
    a, b = ((x64[..., :pairs], x64[..., pairs:2 * pairs]) if layout == 'half' else
            (x64[..., 0:2 * pairs:2], x64[..., 1:2 * pairs:2]))
    u, v = a * cos - b * sin, a * sin + b * cos
    # 32-bit sines and cosines (2 ulp each with the scale's rounding), two products and a sum: under 2^-21 of |a| + |b|
    size = (a.abs() + b.abs()) * scale
    y, loose = x64.clone(), torch.zeros_like(x64)
    if layout == 'half':
        y[..., :pairs], y[..., pairs:2 * pairs] = u, v
        loose[..., :pairs], loose[..., pairs:2 * pairs] = size, size
    else:
        y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = u, v
        loose[..., 0:2 * pairs:2], loose[..., 1:2 * pairs:2] = size, size
    bound = unit(x.dtype) * y.abs() + 2.0 ** -21 * loose + torch.finfo(x.dtype).smallest_normal * unit(x.dtype)
    return y, torch.where(loose > 0, bound, torch.zeros_like(bound))


def close(got, want, bound):
    got = got.double().cpu()
    bad = ~((got - want).abs() <= bound)
    bad &= ~(got.isnan() & want.isnan())
    assert not bad.any(), (int(bad.sum()), got[bad][:4].tolist(), want[bad][:4].tolist())


def sequence_keys(pages, table_row, length):
    """[kv_heads, length, dim] of one sequence."""
    page = pages.shape[2]
    rows = pages[table_row[:-(-length // page)].long()]
    return rows.transpose(0, 1).reshape(pages.shape[1], -1, pages.shape[3])[:, :length]


def attend(q, k, v, causal, scale, dtype):
    """One sequence: q [n, heads, dim], k and v [kv_heads, keys, dim] -> (out, its bound, lse, its bound) in float64.

    The bound, with w the softmax weights and S = sum w |v|: scores are fp32 sums of dim products (each weight then off by
    the relative e = 2 (dim + 2) 2^-24 scale sum |q k| and 2^-20 for the exponential); weights are rounded to the type
    (unit) and their sum to 32 bits; the products with v are summed in 32 bits (truncated at worst: 2^-23 a term); fp16
    weights have a least step of 2^-24 and are held 2^7 times larger (2^-32 each); the output is rounded (unit)."""
    n, heads, dim = q.shape
    group, keys = heads // k.shape[0], k.shape[1]
    q64, k64, v64 = q.double(), k.double().repeat_interleave(group, 0), v.double().repeat_interleave(group, 0)
    score = torch.einsum('nhd,hkd->hnk', q64, k64) * scale
    size = torch.einsum('nhd,hkd->hnk', q64.abs(), k64.abs()) * scale
    if causal:
        hidden = torch.arange(keys)[None] > keys - n + torch.arange(n)[:, None]
        score = score.masked_fill(hidden, -math.inf)
        size = size.masked_fill(hidden, 0.)
    if keys == 0:
        zero = torch.zeros((n, heads, dim), dtype=torch.float64)
        return zero, zero, torch.full((n, heads), -math.inf, dtype=torch.float64), zero[..., 0]
    lse = torch.logsumexp(score, -1)
    w = torch.where(lse[..., None].isinf(), 0., (score - lse[..., None]).exp())
    out = w @ v64
    spread = w @ v64.abs()
    e = 2 * (dim + 2) * 2.0 ** -24 * size.amax(-1) + 2.0 ** -20
    bound = spread * (unit(dtype) + 2 * e + keys * 2.0 ** -23)[..., None] + unit(dtype) * out.abs()
    if dtype == torch.float16:
        bound = bound + keys * 2.0 ** -31 * v64.abs().amax(1)[:, None] + 2.0 ** -25
    lse_bound = 2 * e + keys * 2.0 ** -24 + 2.0 ** -22 * lse.abs()
    swap = lambda t: t.transpose(0, 1)  # noqa: E731
    return swap(out), swap(bound), swap(lse), torch.where(swap(lse).isinf(), 0., swap(lse_bound))


def attention(q, k_pages, v_pages, table, lengths, offsets, causal, scale=None):
    """Per sequence `attend`, on CPU copies; rows outside of every sequence are None in `rows`."""
    q, k_pages, v_pages, table = q.cpu(), k_pages.cpu(), v_pages.cpu(), table.cpu()
    scale = q.shape[2] ** -0.5 if scale is None else scale
    tokens, heads, dim = q.shape
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    lse, lse_bound = (torch.zeros((tokens, heads), dtype=torch.float64) for _ in range(2))
    owned = torch.zeros(tokens, dtype=torch.bool)
    for s, length in enumerate(lengths.tolist()):
        rows = slice(int(offsets[s]), int(offsets[s + 1]))
        if rows.stop == rows.start:
            continue
        owned[rows] = True
        out[rows], bound[rows], lse[rows], lse_bound[rows] = attend(
            q[rows], sequence_keys(k_pages, table[s], length), sequence_keys(v_pages, table[s], length), causal, scale,
            q.dtype)
    return out, bound, lse, lse_bound, owned

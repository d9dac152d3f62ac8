"""Rotary positions and the paged cache without a GPU: frequencies, and every refusal, which comes before any launch."""
import math

import numpy as np
import pytest
import torch

from streamvoxel_b200 import _lib, build, model, ops


@pytest.fixture(scope='module', autouse=True)
def lib():
    build.build()
    return _lib.load()


def test_plain_frequencies_are_the_framework_s_axial_ones():
    freq, scale = ops.rope_frequencies(96, axes=3, device='cpu')
    want = model.rope_frequencies(96).double().repeat(3)
    assert scale == 1.0 and freq.dtype == torch.float64
    torch.testing.assert_close(freq, want, rtol=1e-6, atol=0)   # the framework's are fp32


@pytest.mark.parametrize('rot,factor', [(64, 8.0), (128, 4.0), (32, 1.0)])
def test_scalings(rot, factor):
    plain, _ = ops.rope_frequencies(rot, device='cpu')
    linear, scale = ops.rope_frequencies(rot, scaling='linear', factor=factor, device='cpu')
    assert scale == 1.0 and torch.equal(linear, plain / factor)
    base, scale = ops.rope_frequencies(rot, scaling='base', factor=factor, device='cpu')
    assert scale == 1.0 and base[0] == plain[0]
    assert math.isclose(base[-1], plain[-1] / factor, rel_tol=1e-12)
    parts, scale = ops.rope_frequencies(rot, scaling='by_parts', factor=factor, original=8192, device='cpu')
    turns = 8192 * plain / (2 * math.pi)
    assert math.isclose(scale, 0.1 * math.log(factor) + 1)
    assert torch.equal(parts[turns >= 32], plain[turns >= 32])
    torch.testing.assert_close(parts[turns <= 1], plain[turns <= 1] / factor, rtol=1e-15, atol=0)
    assert bool(((parts <= plain * (1 + 1e-12)) & (parts >= plain / factor * (1 - 1e-12))).all())


@pytest.mark.parametrize('args', [dict(rot=0), dict(rot=7), dict(rot=64, axes=3), dict(rot=64, scaling='other'),
                                  dict(rot=64, scaling='linear', factor=0.5), dict(rot=2, scaling='base', factor=2.0),
                                  dict(rot=64, base=-1.0)])
def test_frequencies_refuse(args):
    with pytest.raises(ValueError):
        ops.rope_frequencies(device='cpu', **args)


def _rope(**change):
    args = dict(x=torch.zeros(4, 2, 64), positions=torch.zeros(4, dtype=torch.int64),
                inv_freq=torch.ones(32, dtype=torch.float64))
    kwargs = {k: change.pop(k) for k in list(change) if k not in args}
    args.update(change)
    return ops.rope(args['x'], args['positions'], args['inv_freq'], **kwargs)


@pytest.mark.parametrize('change', [
    dict(x=torch.zeros(4, 128)), dict(x=torch.zeros(4, 2, 64, dtype=torch.float64)), dict(x=torch.zeros(4, 2, 32)),
    dict(x=torch.zeros(4, 64, 2).transpose(1, 2)), dict(positions=torch.zeros(3, dtype=torch.int64)),
    dict(positions=torch.zeros(4, dtype=torch.float64)), dict(positions=torch.zeros((4, 3))),
    dict(positions=torch.zeros(8, dtype=torch.int64)[::2]), dict(positions=None), dict(inv_freq=torch.ones(32)),
    dict(inv_freq=torch.ones(0, dtype=torch.float64)), dict(layout='other'), dict(scale=math.inf),
    dict(out=torch.zeros(4, 2, 32)), dict(out=torch.zeros(1, 2, 64).expand(4, 2, 64)),
    dict(out=torch.zeros(4, 2, 64, dtype=torch.bfloat16)),
    dict(x=torch.zeros((4, 2, 64), requires_grad=True), out=torch.zeros(4, 2, 64)),
    dict()])   # the last: operands on the CPU
def test_rope_refuses(change):
    with pytest.raises(ValueError):
        _rope(**change)


def _cache(pages=6, heads=2, page=16, dim=64, sequences=2, width=3, dtype=torch.bfloat16):
    return dict(k_pages=torch.zeros((pages, heads, page, dim), dtype=dtype),
                v_pages=torch.zeros((pages, heads, page, dim), dtype=dtype),
                table=torch.zeros((sequences, width), dtype=torch.int32),
                lengths=torch.ones(sequences, dtype=torch.int32),
                offsets=torch.arange(sequences + 1, dtype=torch.int32))


CACHE_FAULTS = [dict(k_pages=torch.zeros((6, 2, 32, 64), dtype=torch.bfloat16)), _cache(dtype=torch.float32),
                _cache(page=24), _cache(page=8), dict(table=torch.zeros((2, 3), dtype=torch.int64)),
                dict(table=torch.zeros(6, dtype=torch.int32)), dict(table=torch.zeros((2, 0), dtype=torch.int32)),
                dict(table=torch.zeros((3, 2), dtype=torch.int32).t()),
                dict(lengths=torch.ones(3, dtype=torch.int32)), dict(offsets=torch.zeros(2, dtype=torch.int32)),
                dict(status=torch.zeros(3, dtype=torch.int32)),
                dict(k_pages=torch.zeros((6, 16, 2, 64), dtype=torch.bfloat16).transpose(1, 2)),
                dict()]   # the last: operands on the CPU


@pytest.mark.parametrize('change', CACHE_FAULTS + [
    dict(k=torch.zeros(2, 3, 64, dtype=torch.bfloat16)), dict(v=torch.zeros(3, 2, 64, dtype=torch.bfloat16)),
    dict(k=torch.zeros(2, 2, 64)), dict(positions=torch.zeros(2, dtype=torch.int32)),
    dict(q=torch.zeros(2, 4, 64, dtype=torch.bfloat16)),
    dict(q_out=torch.zeros(2, 4, 64, dtype=torch.bfloat16)),
    dict(inv_freq=torch.ones(32, dtype=torch.float64), q=torch.zeros(3, 4, 64, dtype=torch.bfloat16)),
    dict(inv_freq=torch.ones(40, dtype=torch.float64)),
    dict(k=torch.zeros((2, 2, 64), dtype=torch.bfloat16, requires_grad=True))])
def test_append_refuses(change):
    args = dict(k=torch.zeros(2, 2, 64, dtype=torch.bfloat16), v=torch.zeros(2, 2, 64, dtype=torch.bfloat16), **_cache())
    args.update(change)
    with pytest.raises(ValueError):
        ops.paged_append(**args)


@pytest.mark.parametrize('change', CACHE_FAULTS + [
    _cache(dim=80) | dict(q=torch.zeros(2, 4, 80, dtype=torch.bfloat16)),
    dict(q=torch.zeros(2, 3, 64, dtype=torch.bfloat16)), dict(q=torch.zeros(2, 4, 64, dtype=torch.float16)),
    dict(q=torch.zeros(2, 0, 64, dtype=torch.bfloat16)), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan),
    dict(scale=math.inf), dict(out=torch.zeros(2, 4, 32, dtype=torch.bfloat16)),
    dict(lse=torch.zeros(2, 4, dtype=torch.bfloat16)), dict(lse=torch.zeros(4, 2)), dict(max_query=-1),
    dict(q=torch.zeros((2, 4, 64), dtype=torch.bfloat16, requires_grad=True))])
def test_attention_refuses(change):
    args = dict(q=torch.zeros(2, 4, 64, dtype=torch.bfloat16), **_cache())
    args.update(change)
    with pytest.raises(ValueError):
        ops.paged_attention(**args)


def test_library_refuses_before_any_launch(lib):
    """The C entries check what the Python surface checks before they launch."""
    import ctypes
    at = 4096   # never read: every call below is refused
    good = dict(k=at, v=at, dtype=_lib.BF16, pages=4, kv_heads=2, page=16, dim=64, sequences=2, table_width=3, table=at,
                lengths=at, offsets=at, status=None)
    make = lambda **c: ctypes.byref(_lib.PagedCache(**{**good, **c}))  # noqa: E731
    rotary = lambda **c: ctypes.byref(_lib.Rotary(**{**dict(inv_freq=at, rot=64, layout=0, axes=1, scale=1.0,  # noqa: E731
                                                            positions=at, position_type=_lib.I64), **c}))
    append = lambda cache, rot=None, q=None, heads=0: lib.svx_paged_append(  # noqa: E731
        cache, at, 128, 64, at, 128, 64, 2, rot, q, 128, 64, heads, q, None)
    attend = lambda cache, q=at, token=128, tokens=2, heads=4, scale=0.1, out=at, ws=at: lib.svx_paged_attention(  # noqa: E731
        cache, q, token, 64, tokens, heads, 1, scale, out, None, 1, ws, None)
    faults = [dict(dtype=_lib.F32), dict(pages=0), dict(kv_heads=0), dict(page=24), dict(page=8), dict(page=2048),
              dict(dim=60), dict(dim=0), dict(sequences=-1), dict(table_width=0), dict(table_width=1 << 27),
              dict(k=None), dict(k=at + 8), dict(table=None), dict(offsets=None)]
    calls = [lambda f=f: append(make(**f)) for f in faults] + [lambda f=f: attend(make(**f)) for f in faults]
    calls += [lambda: append(None), lambda: attend(None),
              lambda: append(make(), rotary(rot=66)), lambda: append(make(), rotary(rot=63)),
              lambda: append(make(), rotary(axes=3)), lambda: append(make(), rotary(layout=2)),
              lambda: append(make(), rotary(positions=None, axes=2)), lambda: append(make(), rotary(inv_freq=None)),
              lambda: append(make(), rotary(position_type=_lib.BF16)), lambda: append(make(), None, at, 4),
              lambda: append(make(), rotary(), at, 0),
              lambda: attend(make(dim=80)), lambda: attend(make(), heads=3), lambda: attend(make(), heads=0),
              lambda: attend(make(), tokens=-1), lambda: attend(make(), scale=0.0), lambda: attend(make(), scale=math.inf),
              lambda: attend(make(), scale=math.nan), lambda: attend(make(), token=132), lambda: attend(make(), q=at + 2),
              lambda: attend(make(), out=None), lambda: attend(make(), ws=None),
              lambda: lib.svx_rope(at, _lib.I32, 64, 64, at, 64, 64, 2, 1, 64, rotary(), 0, None),
              lambda: lib.svx_rope(at, _lib.F32, 64, 64, at, 64, 64, -1, 1, 64, rotary(), 0, None),
              lambda: lib.svx_rope(at, _lib.F32, 64, 64, None, 64, 64, 2, 1, 64, rotary(), 0, None),
              lambda: lib.svx_rope(at, _lib.F32, 64, 64, at, 64, 64, 2, 1, 64, rotary(positions=None), 0, None),
              lambda: lib.svx_rope(at, _lib.F32, 64, 64, at, 64, 64, 2, 1, 64, None, 0, None)]
    for i, call in enumerate(calls):
        assert call() == _lib.SVX_ERR_INVALID, i
    assert lib.svx_paged_attention_workspace_bytes(2, 1, 3, 2, 64, 0) == 0
    assert lib.svx_rope(None, _lib.F32, 64, 64, None, 64, 64, 0, 1, 64, rotary(), 0, None) == _lib.SVX_OK


def _line(lengths, news, heads, unit_tokens, causal):
    """The line of key tiles: (sequence, token tile, head) -> its tiles, in order."""
    units = []
    for s, (length, n) in enumerate(zip(lengths, news)):
        for j in range(-(-n // unit_tokens)):
            seen = max(0, min(length, length - n + min((j + 1) * unit_tokens, n))) if causal else length
            units += [((s, j, h), max(1, -(-seen // 64))) for h in range(heads)]
    return units


def test_closed_form_of_the_tile_count():
    """The kernels find their place on the line of tiles by a closed form (a floor sum): the same, restated, against
    counting."""
    def floor_sum(n, a, b):
        g = a & -a if a % 64 else 64
        period = 64 // g
        periods = n // period
        residues = periods * (period * (b % g) + g * period * (period - 1) // 2)
        residues += sum((a * i + b) % 64 for i in range(n - periods * period))
        return (a * (n * (n - 1) // 2) + b * n - residues) // 64

    def tiles_before(length, n, unit, causal, count):
        if not count:
            return 0
        one = lambda keys: max(1, -(-keys // 64))  # noqa: E731
        if not causal:
            return count * one(length)
        seen = lambda j: max(0, min(length, length - n + min((j + 1) * unit, n)))  # noqa: E731
        if count == 1:
            return one(seen(0))
        full, base = min(count, n // unit), length - n
        ones = 0 if base >= 64 else min(full, (64 - base) // unit)
        total = ones
        if full > ones:
            total += floor_sum(full - ones, unit, base + (ones + 1) * unit + 63)
        return total + (one(seen(full)) if count > full else 0)

    rng = np.random.default_rng(0)
    for _ in range(3000):
        n, unit = int(rng.integers(1, 400)), int(rng.choice([1, 2, 3, 5, 8, 16, 21, 36, 42, 64, 128, 256]))
        length = int(rng.integers(0, 700)) if rng.random() < 0.3 else n + int(rng.integers(0, 700))
        causal = bool(rng.random() < 0.8)
        counts = [t for (_, _, _), t in _line([length], [n], 1, unit, causal)]
        for count in {0, 1, len(counts), int(rng.integers(0, len(counts) + 1))}:
            assert tiles_before(length, n, unit, causal, count) == sum(counts[:count]), (n, unit, length, causal, count)

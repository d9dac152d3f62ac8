"""How paged attention is divided among CTAs: the kernels' own arithmetic, compiled for the host, against counting.

A batch is a line of units (sequence, head, token tile) of 64-key tiles. Some units are dealt out whole, the rest of the
line is cut into runs; a unit that several CTAs share leaves partials, which its last CTA names for the joining kernel."""
import collections
import ctypes
import os
import subprocess

import numpy as np
import pytest

from streamvoxel_b200 import build

SMS = 148


@pytest.fixture(scope='module')
def division(tmp_path_factory):
    target = str(tmp_path_factory.mktemp('division') / 'division.so')
    source = os.path.join(os.path.dirname(os.path.abspath(__file__)), 'paged_division.cu')
    command = [build.nvcc(), *build.ARCH, *build.FLAGS, '-I' + build.CSRC, '-shared', source, '-o', target]
    result = subprocess.run(command, capture_output=True, text=True)
    assert result.returncode == 0, result.stderr
    call = ctypes.CDLL(target).paged_division

    def run(news, lengths, kv_heads, unit_tokens, causal, *, ctas=SMS, two_tiles=True, min_tiles=4, blocks=1, threads=16):
        offsets = np.concatenate(([0], np.cumsum(news))).astype(np.int32)
        lengths = np.asarray(lengths, np.int32)
        width = max(1, -(-int(lengths.max()) // 16))
        shape = np.array([offsets[-1], len(news), kv_heads, causal, unit_tokens, blocks, min_tiles, ctas, two_tiles, 4,
                          width, threads], np.int32)
        units = sum(-(-int(n) // unit_tokens) for n in news) * kv_heads * blocks
        segments, joins = np.zeros((units + 2 * ctas, 8), np.int32), np.zeros(16 * ctas + 64, np.int32)
        counts = np.zeros(2, np.int32)
        at = lambda a: a.ctypes.data_as(ctypes.c_void_p)  # noqa: E731
        rows = call(at(shape), at(lengths), at(offsets), at(segments), len(segments), at(joins), joins.size, at(counts))
        assert rows >= 0
        named, i = [], 0
        while i < counts[0]:
            parts = int(joins[i + 1])
            named.append((int(joins[i]), tuple(joins[i + 2:i + 5].tolist()), joins[i + 5:i + 5 + parts].tolist()))
            i += 5 + parts
        return segments[:rows].tolist(), named, int(counts[1])

    return run


def check_cover(segments, news, lengths, kv_heads, unit_tokens, causal, ctas=SMS, min_tiles=4, blocks=1):
    """Every tile of every unit is taken once, in as many tiles a CTA as an equal share (one more at most)."""
    units = {}
    for s, (n, length) in enumerate(zip(news, lengths)):
        for j in range(-(-n // unit_tokens)):
            seen = max(0, min(length, length - n + min((j + 1) * unit_tokens, n))) if causal else length
            units.update({(s, h, j): max(1, -(-seen // 64)) for h in range(kv_heads * blocks)})
    taken, load = collections.defaultdict(list), collections.Counter()
    for cta, s, h, j, t0, t1, tiles, slot in segments:
        assert tiles == units[s, h, j] and t0 < t1 <= tiles
        assert (slot < 0) == (t0 == 0 and t1 == tiles)
        taken[s, h, j].append((t0, t1))
        load[cta] += t1 - t0
    assert taken.keys() == units.keys()
    for unit, runs in taken.items():
        runs.sort()
        assert runs[0][0] == 0 and runs[-1][1] == units[unit]
        assert all(a[1] == b[0] for a, b in zip(runs, runs[1:])), (unit, runs)
    assert max(load.values(), default=0) <= max(min_tiles, -(-sum(units.values()) // ctas)) + 1


def batches(count, seed):
    rng = np.random.default_rng(seed)
    for _ in range(count):
        sequences = int(rng.choice([1, 2, 3, 4, 6, 16, 40]))
        causal = bool(rng.random() < 0.6)
        if rng.random() < 0.4:   # equal sequences, sizes that divide evenly
            news = [int(rng.choice([64, 128, 256, 512, 700]))] * sequences
            older = [int(rng.choice([0, 64, 1024, 1000]))] * sequences
        else:
            news = [int(np.exp(rng.uniform(0, np.log(3000)))) for _ in range(sequences)]
            older = [int(rng.integers(0, 3000)) for _ in range(sequences)]
        lengths = [n + o for n, o in zip(news, older)] if causal or rng.random() < 0.5 else [o for o in older]
        yield dict(news=news, lengths=lengths, kv_heads=int(rng.choice([1, 2, 4, 8, 16])),
                   unit_tokens=2 * (128 // int(rng.choice([1, 2, 3, 4, 6, 8, 16]))), causal=causal)


def test_every_tile_is_taken_once(division):
    dealt = 0
    for batch in batches(1500, 0):
        segments, _, waves = division(**batch)
        check_cover(segments, **batch)
        dealt += waves > 0
    assert dealt > 100


@pytest.mark.parametrize('ctas', [592, 444, 296])
def test_every_tile_is_taken_once_in_equal_runs(division, ctas):
    """The few-rows form and the one-tile form: no unit is dealt out, the heads of a group may be in several blocks."""
    rng = np.random.default_rng(1)
    for batch in batches(200, ctas):
        batch['unit_tokens'] = int(rng.choice([1, 2, 4, 16]))
        batch['news'] = [min(n, 200) for n in batch['news']]
        batch['lengths'] = [max(n, m) if batch['causal'] else m for n, m in zip(batch['news'], batch['lengths'])]
        blocks = int(rng.choice([1, 2]))
        segments, named, waves = division(**batch, ctas=ctas, two_tiles=False, min_tiles=2, blocks=blocks)
        assert waves == 0
        check_cover(segments, **batch, ctas=ctas, min_tiles=2, blocks=blocks)
        check_joins(segments, named)


def check_joins(segments, named):
    """Every unit in several parts is joined once, from the partials that its own segments left, in order."""
    left, parts = {}, collections.defaultdict(list)
    for cta, s, h, j, t0, t1, tiles, slot in segments:
        if slot >= 0:
            assert slot not in left and slot // 2 == cta
            left[slot] = s, h, j
            parts[s, h, j].append((t0, slot))
    joined = set()
    for cta, unit, slots in named:
        assert unit not in joined
        joined.add(unit)
        assert [left.get(slot) for slot in slots] == [unit] * len(slots), (unit, slots)
        assert slots == [slot for _, slot in sorted(parts[unit])]
    assert joined == set(parts)


# An empty run between two CTAs that share a unit: the dealt units of a CTA in the middle fill its share exactly.
FULL_SHARES = [dict(news=[512] * 16, lengths=[512] * 16, kv_heads=8, unit_tokens=64, causal=True),
               dict(news=[753, 1163, 511], lengths=[820, 3847, 679], kv_heads=4, unit_tokens=32, causal=True),
               dict(news=[784, 768, 3184], lengths=[128, 320, 128], kv_heads=1, unit_tokens=16, causal=False)]


@pytest.mark.parametrize('batch', FULL_SHARES)
def test_joins_of_full_shares(division, batch):
    segments, named, waves = division(**batch)
    assert waves > 0 and named
    check_cover(segments, **batch)
    check_joins(segments, named)


def test_joins_read_what_their_units_left(division):
    dealt = 0
    for batch in batches(3000, 2):
        segments, named, waves = division(**batch)
        dealt += waves > 0
        check_joins(segments, named)
    assert dealt > 200

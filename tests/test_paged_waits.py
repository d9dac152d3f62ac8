"""Waits of the tcgen05 form of paged attention, without a GPU.

A lane that gives a wait up by itself leaves its warp's .sync.aligned instructions and full-mask votes to the others, which
is undefined and can hang, so the lanes agree on the outcome of every wait."""
import os
import random
import re

import pytest

import paged_barriers
from streamvoxel_b200 import build


def _code():
    text = open(os.path.join(build.CSRC, 'paged_tc.cu')).read()
    return re.sub(r'//[^\n]*', '', text)


def test_lanes_agree_on_every_wait():
    code = _code()
    calls = [code[code.rindex('\n', 0, m.start()) + 1:code.index('\n', m.start())].strip()
             for m in re.finditer(r'(?<![\w:])(?:tc::)?wait\(', code)]
    # the definition, and the one call, under the warp's vote
    assert len(calls) == 2 and calls[0].startswith('__device__') and 'return __all_sync(0xffffffffu, wait(' in calls[1]
    assert 'mbar_try_wait' not in code[code.index('chunk_kernel('):]


def test_teardown_waits_are_followed_by_a_convergence():
    """The waits without a vote are the bounded ones of the teardown, whose warps meet again before they go on."""
    code = _code()
    for m in re.finditer(r'(?<![\w:])mbar_wait\(', code):
        rest = code[m.end():]
        assert '__syncwarp();' in rest[:rest.index('asm volatile("barrier') if 'drained' not in rest[:20] else
                                       rest.index('tc::tmem_dealloc')]


@pytest.mark.parametrize('chains,stages', [(1, 2), (1, 4), (2, 4), (2, 8)])   # 128- and 96-wide heads, 64-wide ones
def test_barriers_under_random_schedules(chains, stages):
    """No deadlock, no mistaken phase, no buffer overwritten in use: whole units and runs of any length, in any order, with
    second query tiles that have no tokens and sequences that end inside a tile."""
    rng = random.Random(100 * chains + stages)
    for _ in range(400):
        units = [(chains == 2 and rng.random() < 0.4, rng.choice([1, 1, 2, 3, 4, 5, 7, 11, 23]), rng.random() < 0.5)
                 for _ in range(rng.randint(1, 8))]
        paged_barriers.Kernel(units, stages, chains, rng).run()


def test_model_has_the_kernel_s_barriers():
    """Rings, arrival counts and the waits' phases of the model are those of the source."""
    code = _code()
    for text in ('stages = kChains == 2 ? (atoms == 2 ? 4 : 8) : (atoms == 2 ? 2 : 4)', 'mbar_init(q_full, 1)',
                 'mbar_init(q_empty, kChains)', 'mbar_init(k_full + i, 1)', 'mbar_init(k_empty + i, kChains)',
                 'mbar_init(v_full + i, 1)', 'mbar_init(v_empty + i, kChains)', 'mbar_init(v_end, 1)',
                 'mbar_init(s_full + i, 1)', 'mbar_init(p_full + i, 4)', 'mbar_init(pv_done + i, 1)',
                 'mbar_init(drained, 2 * kChains)', 'bars + 2 * i + (n & 1), (n >> 1) & 1',
                 'wait_w(q_full, w.units & 1', 'wait_w(k_full + s, (g / C::stages) & 1',
                 'wait_w(v_full + s, (g / C::stages) & 1', 'wait_w(empty + s, (g / C::stages - 1) & 1',
                 'wait_w(q_empty, (w.units - 1) & 1', 'buffer_wait(pv_done, i, n - 2)', 'buffer_wait(p_full, i, n)',
                 'buffer_wait(s_full, i, n)', 'buffer_wait(pv_done, i, n - 1)',
                 'buffer_wait(pv_done, i, n0 + count - 1)'):
        assert text in code, text


def test_the_model_sees_mistakes():
    """Planted in the model: products with V that skip a wait, a loader of K that does not wait for its stage, and one set of
    barriers for both S buffers."""
    class Always:
        def arrive(self):
            pass

        def passed(self, k):
            return True

    class NoP(paged_barriers.Kernel):
        def values(self, i):
            yield from (f if j % 3 != 1 else (lambda: True) for j, f in enumerate(super().values(i)))

    class EarlyLoad(paged_barriers.Kernel):
        def loader(self, is_v):
            self.k_empty = [Always() for _ in self.k_empty]
            yield from super().loader(is_v)

    class OneSBuffer(paged_barriers.Kernel):
        def __init__(self, *args):
            super().__init__(*args)
            for s, p, d in zip(self.s_full, self.p_full, self.pv_done):
                s[1], p[1], d[1] = s[0], p[0], d[0]

    for kind in (NoP, EarlyLoad, OneSBuffer):
        rng, caught = random.Random(1), 0
        for _ in range(30):
            try:
                kind([(False, 7, False), (False, 5, True)], 4, 2, rng).run()
            except AssertionError:
                caught += 1
        assert caught > 15, kind

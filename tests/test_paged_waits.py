"""Waits of the tcgen05 form of paged attention, without a GPU.

A lane that gives a wait up by itself leaves its warp's .sync.aligned instructions and full-mask votes to the others, which
is undefined and can hang, so the lanes agree on the outcome of every wait."""
import os
import re

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

"""Rotary positions, the append to a paged cache and the attention over it on the GPU, against 64-bit forms.

Bounds are derived in `paged_reference` (half a step of each rounding, fp32 sums term by term); what is copied or not
touched has to be equal."""
import math

import numpy as np
import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


@pytest.fixture(scope='module')
def ops():
    from streamvoxel_b200 import _lib, ops
    _lib.require_device()
    return ops


@pytest.fixture(autouse=True)
def no_grad():
    with torch.no_grad():
        yield


# ------------------------------------------------------------------------------------------------------ rope

ROPE_SHAPES = [(96, 96, 3), (128, 64, 1), (80, 40, 1), (64, 64, 2), (6, 6, 3), (70, 2, 1), (512, 512, 1), (33, 32, 4)]


@pytest.mark.parametrize('dtype', list(TYPES))
@pytest.mark.parametrize('layout', ['interleaved', 'half'])
@pytest.mark.parametrize('dim,rot,axes', ROPE_SHAPES)
def test_rope(ops, dtype, layout, dim, rot, axes):
    g = torch.Generator().manual_seed(dim + rot)
    freq, _ = ops.rope_frequencies(rot, axes=axes)
    for tokens, heads in ((1, 1), (37, 3), (700, 5)):
        x = torch.randn((tokens, heads, dim), generator=g).to(TYPES[dtype]).cuda()
        positions = (torch.randint(-4000, 4000, (tokens, axes), generator=g).float() / 2).cuda()
        positions = positions[:, 0].contiguous() if axes == 1 else positions
        for inverse in (False, True):
            got = ops.rope(x, positions, freq, layout=layout, scale=1.25, inverse=inverse)
            want, bound = ref.rotate(x, positions, freq, layout, 1.25, inverse)
            assert got.dtype == x.dtype and got.is_contiguous()
            ref.close(got, want, bound)


@pytest.mark.parametrize('kind', [torch.int32, torch.int64])
def test_rope_far_positions(ops, kind):
    """Angles of positions past a million, and past what 32 bits hold exactly, keep 32-bit accuracy."""
    freq, _ = ops.rope_frequencies(128)
    positions = torch.tensor([0, 1, 999_983, 2 ** 24 + 1, 2 ** 31 - 1, -5], dtype=kind, device='cuda')
    x = torch.randn((6, 2, 128), generator=torch.Generator().manual_seed(1)).cuda()
    ref.close(ops.rope(x, positions, freq), *ref.rotate(x, positions, freq))


@pytest.mark.parametrize('dtype', list(TYPES))
def test_rope_strides_and_in_place(ops, dtype):
    """Queries inside a packed [tokens, 3 heads, dim] tensor, rows at odd offsets, and the input as the output."""
    g = torch.Generator().manual_seed(3)
    freq, _ = ops.rope_frequencies(64)
    positions = torch.arange(50, device='cuda')
    packed = torch.randn((50, 12, 64), generator=g).to(TYPES[dtype]).cuda()
    want, bound = ref.rotate(packed[:, 4:8], positions, freq, 'half')
    ref.close(ops.rope(packed[:, 4:8], positions, freq, layout='half'), want, bound)
    before = packed.clone()
    got = ops.rope(packed[:, 4:8], positions, freq, layout='half', out=packed[:, 4:8])
    assert got.data_ptr() == packed[:, 4:8].data_ptr()
    ref.close(packed[:, 4:8], want, bound)
    assert torch.equal(packed[:, :4], before[:, :4]) and torch.equal(packed[:, 8:], before[:, 8:])
    wide = torch.randn((50, 2, 77), generator=g).to(TYPES[dtype]).cuda()
    odd = wide[:, :, 3:73]
    ref.close(ops.rope(odd, positions, freq), *ref.rotate(odd, positions, freq))
    turned = torch.randn((3, 50, 64), generator=g).to(TYPES[dtype]).cuda().transpose(0, 1)
    ref.close(ops.rope(turned, positions, freq), *ref.rotate(turned, positions, freq))
    one = torch.randn((1, 2, 64), generator=g).to(TYPES[dtype]).cuda().expand(50, 2, 64)   # a broadcast input
    ref.close(ops.rope(one, positions, freq), *ref.rotate(one, positions, freq))
    assert ops.rope(packed[:0], positions[:0], freq).shape == (0, 12, 64)


def test_rope_is_the_framework_s_axial_rotation(ops):
    from streamvoxel_b200 import model
    positions = model.patch_centers_xyz((64, 16, 16), 4).cuda() / 4
    x = torch.randn((len(positions), 8, 96), generator=torch.Generator().manual_seed(4)).cuda()
    freq, _ = ops.rope_frequencies(96, axes=3)
    want = model._rope(x.transpose(0, 1), positions, model.rope_frequencies(96).cuda()).transpose(0, 1)
    # the framework's frequencies are fp32: 2^-24 of angles up to 64, on top of both sides' own 2^-21
    torch.testing.assert_close(ops.rope(x, positions, freq), want, rtol=0, atol=6 * (64 * 2 ** -24 + 2 ** -20))


@pytest.mark.parametrize('layout', ['interleaved', 'half'])
def test_rope_gradient(ops, layout):
    """The gradient equals the formula's (the transposed rotation) and differences of the rotation, which is linear."""
    g = torch.Generator().manual_seed(5)
    freq, scale = ops.rope_frequencies(64, scaling='by_parts', factor=4.0)
    positions = torch.randint(0, 100_000, (40,), generator=g).cuda()
    x = torch.randn((40, 3, 96), generator=g).cuda()
    y = torch.randn((40, 3, 96), generator=g).cuda()
    with torch.enable_grad():
        leaf = x.clone().requires_grad_()
        out = ops.rope(leaf, positions, freq, layout=layout, scale=scale)
        y.requires_grad_()
        grad, = torch.autograd.grad(out, leaf, y, create_graph=True)
        twice, = torch.autograd.grad(grad, y, x)
    y, grad = y.detach(), grad.detach()
    ref.close(twice, *ref.rotate(x, positions, freq, layout, scale))
    ref.close(grad, *ref.rotate(y, positions, freq, layout, scale, inverse=True))
    # <R(x + h) - R(x - h), y> = 2 <h, R^T y>
    h = torch.randn((40, 3, 96), generator=g).cuda()
    args = dict(layout=layout, scale=scale)
    left = ((ops.rope(x + h, positions, freq, **args).double() - ops.rope(x - h, positions, freq, **args).double())
            * y.double()).sum()
    right = 2 * (h.double() * grad.double()).sum()
    # every value's error is under 2^-20 of its pair's size (about 3), times |y|: n independent ones, ten deviations
    assert abs(float(left - right)) < 10 * math.sqrt(x.numel()) * 2 ** -20 * 6 * 3
    with torch.enable_grad():   # a gradient broadcast over heads has stride 0
        out = ops.rope(leaf, positions, freq, **args)
        broadcast, = torch.autograd.grad(out.sum(), leaf)
    ref.close(broadcast, *ref.rotate(torch.ones_like(x), positions, freq, layout, scale, inverse=True))


# ---------------------------------------------------------------------------------------------------- the cache


def _cache(rng, lengths, heads, page, dim, dtype, fill=math.nan, spare=3, width=None):
    """Pools full of `fill` and a table of pages in random order; unused entries hold ids outside the pool."""
    per = [-(-n // page) for n in lengths]
    pages = sum(per) + spare
    ids = rng.permutation(pages)
    table = np.full((len(per), max(1, max(per, default=1)) if width is None else width), -7, np.int32)
    at = 0
    for s, n in enumerate(per):
        table[s, :n] = ids[at:at + n]
        at += n
    pools = [torch.full((pages, heads, page, dim), fill, dtype=dtype, device='cuda') for _ in range(2)]
    return (*pools, torch.from_numpy(table).cuda(), torch.tensor(lengths, dtype=torch.int32, device='cuda'))


def _fill(pools, table, lengths, g):
    """Random keys and values in the sequences' places, the rest of the pools left as it is."""
    for s, n in enumerate(lengths.tolist()):
        for p in range(-(-n // pools[0].shape[2])):
            rows = min(pools[0].shape[2], n - p * pools[0].shape[2])
            for pool in pools:
                pool[int(table[s, p]), :, :rows] = torch.randn((pool.shape[1], rows, pool.shape[3]), generator=g).to(pool)


def _offsets(news, first=0):
    return torch.tensor(np.concatenate(([first], first + np.cumsum(news))), dtype=torch.int32, device='cuda')


APPEND_SHAPES = [('bf16', 8, 96, 64, 96, 3, 'interleaved'), ('fp16', 2, 128, 16, 64, 1, 'half'),
                 ('bf16', 1, 64, 32, 64, 1, 'interleaved'), ('bf16', 3, 40, 16, 20, 1, 'half'),
                 ('fp16', 5, 24, 256, 8, 2, 'interleaved')]


@pytest.mark.parametrize('dtype,heads,dim,page,rot,axes,layout', APPEND_SHAPES)
def test_append(ops, dtype, heads, dim, page, rot, axes, layout):
    """Sequences of no, one and many new tokens, pages that end among them, rows before and behind the sequences."""
    rng, g, dtype = np.random.default_rng(dim), torch.Generator().manual_seed(dim), TYPES[dtype]
    news = [1, 0, 17, 3, 64, 1, 200, 0]
    old = [0, 5, 15, page - 1, 2 * page, 300, 1, 0]
    k_pages, v_pages, table, lengths = _cache(rng, [a + b for a, b in zip(news, old)], heads, page, dim, dtype)
    offsets, tokens = _offsets(news, first=2), sum(news) + 7
    k, v = (torch.randn((tokens, heads, dim), generator=g).to(dtype).cuda() for _ in range(2))
    q = torch.randn((tokens, 2 * heads, dim), generator=g).to(dtype).cuda()
    freq, _ = ops.rope_frequencies(rot, axes=axes)
    places = [torch.arange(b, a + b) for a, b in zip(news, old)]
    at = torch.cat([torch.zeros(2, dtype=torch.long), *places, torch.zeros(5, dtype=torch.long)])
    positions = None if axes == 1 else (torch.randint(-99, 99, (tokens, axes), generator=g).float() / 2).cuda()
    status = torch.zeros(len(news), dtype=torch.int32, device='cuda')
    q_out = torch.full_like(q, 3.0)
    got = ops.paged_append(k, v, k_pages, v_pages, table, lengths, offsets, inv_freq=freq, positions=positions,
                           layout=layout, rope_scale=0.75, q=q, q_out=q_out, status=status)
    assert got is q_out and not status.any()
    position = at.cuda() if positions is None else positions
    want_k, bound_k = ref.rotate(k, position, freq, layout, 0.75)
    want_q, bound_q = ref.rotate(q, position, freq, layout, 0.75)
    live = slice(2, 2 + sum(news))
    ref.close(q_out[live], want_q[live], bound_q[live])
    assert bool((q_out[:2] == 3).all()) and bool((q_out[live.stop:] == 3).all())
    written = torch.zeros(k_pages.shape[:3], dtype=torch.bool)
    for s, rows in enumerate(places):
        for i, place in enumerate(rows.tolist()):
            row, spot = int(offsets[s]) + i, (int(table[s, place // page]), slice(None), place % page)
            assert not written[spot].any()
            written[spot] = True
            assert torch.equal(v_pages[spot], v[row])
            ref.close(k_pages[spot], want_k[row], bound_k[row])
    assert bool(k_pages.isnan().all(-1)[~written].all()) and bool(v_pages.isnan().all(-1)[~written].all())


def test_append_without_rotation_copies(ops):
    rng, g = np.random.default_rng(0), torch.Generator().manual_seed(0)
    k_pages, v_pages, table, lengths = _cache(rng, [40, 7], 2, 16, 72, torch.float16)
    packed = torch.randn((47, 3, 2, 72), generator=g).half().cuda()   # k and v inside a wider tensor
    ops.paged_append(packed[:, 1], packed[:, 2], k_pages, v_pages, table, lengths, _offsets([40, 7]))
    for s, rows in enumerate((slice(0, 40), slice(40, 47))):
        n = rows.stop - rows.start
        assert torch.equal(ref.sequence_keys(k_pages, table[s], n).transpose(0, 1), packed[rows, 1])
        assert torch.equal(ref.sequence_keys(v_pages, table[s], n).transpose(0, 1), packed[rows, 2])


def test_append_bad_places(ops):
    """Page ids outside the pool and places outside the table are not stored and say so; the others are."""
    from streamvoxel_b200 import _lib
    rng, g = np.random.default_rng(1), torch.Generator().manual_seed(1)
    k_pages, v_pages, table, lengths = _cache(rng, [20, 20, 20, 20, 20], 2, 16, 64, torch.bfloat16)
    table[1, 1] = 1 << 30          # keys 16-19 of sequence 1
    table[2, 0] = -1               # keys 0-15 of sequence 2
    lengths[3] = 2 * 16 + 5        # ends past its table of two pages: its last five
    lengths[4] = 3                 # fewer keys than new tokens: the first two have no place
    news = [20, 20, 20, 20, 5]
    k, v = (torch.randn((85, 2, 64), generator=g).bfloat16().cuda() for _ in range(2))
    status = torch.zeros(5, dtype=torch.int32, device='cuda')
    ops.paged_append(k, v, k_pages, v_pages, table, lengths, _offsets(news), status=status)
    bad = _lib.STATUS_BAD_PAGE
    assert status.tolist() == [0, bad, bad, bad, bad]
    stored = ~k_pages.isnan().all(-1)
    assert int(stored.sum()) == 2 * (20 + 16 + 4 + 15 + 3)
    assert torch.equal(k_pages[int(table[1, 0])].transpose(0, 1), k[20:36])
    assert torch.equal(v_pages[int(table[2, 1]), :, :4].transpose(0, 1), v[56:60])
    assert torch.equal(k_pages[int(table[4, 0]), :, :3].transpose(0, 1), k[82:85])


# ---------------------------------------------------------------------------------------------------- attention


def _check(ops, g, q, k_pages, v_pages, table, lengths, offsets, causal, scale=None, max_query=None):
    tokens, heads = q.shape[:2]
    out = torch.full((tokens, heads, q.shape[2]), 5.0, dtype=q.dtype, device='cuda')
    lse = torch.full((tokens, heads), 5.0, device='cuda')
    status = torch.zeros(len(lengths), dtype=torch.int32, device='cuda')
    got = ops.paged_attention(q, k_pages, v_pages, table, lengths, offsets, causal=causal, scale=scale, out=out, lse=lse,
                              max_query=max_query, status=status)
    want, bound, want_lse, lse_bound, owned = ref.attention(q, k_pages, v_pages, table, lengths, offsets.cpu(), causal,
                                                            scale)
    assert got is out and not status.any()
    ref.close(out[owned.cuda()], want[owned], bound[owned])
    rows = want_lse[owned]
    assert torch.equal(lse[owned.cuda()].cpu().isinf(), rows.isinf())
    ref.close(lse[owned.cuda()].cpu()[~rows.isinf()], rows[~rows.isinf()], lse_bound[owned][~rows.isinf()])
    assert bool((out[~owned.cuda()] == 5).all()) and bool((lse[~owned.cuda()] == 5).all())
    return out, lse


NEWS = [1, 0, 1, 5, 1, 33, 2, 1, 130, 17]
KEYS = [1, 9, 0, 5, 64, 33, 65, 577, 200, 3]   # a sequence without keys, and one with fewer keys than new tokens
ATTENTION = [('bf16', 96, 8, 1, 64), ('bf16', 128, 2, 4, 16), ('fp16', 64, 1, 6, 32), ('fp16', 128, 1, 8, 128),
             ('bf16', 64, 3, 3, 16), ('bf16', 64, 1, 16, 256), ('fp16', 96, 2, 7, 16), ('bf16', 128, 1, 20, 32)]


@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('dtype,dim,heads,group,page', ATTENTION)
def test_attention(ops, dtype, dim, heads, group, page, causal):
    """One token, chunks, ends inside tiles and pages, rows without keys, rows outside of the sequences, stale NaN in
    every place of the pool that no sequence owns."""
    rng, g, dtype = np.random.default_rng(dim), torch.Generator().manual_seed(group), TYPES[dtype]
    k_pages, v_pages, table, lengths = _cache(rng, KEYS, heads, page, dim, dtype)
    _fill((k_pages, v_pages), table, lengths, g)
    offsets = _offsets(NEWS, first=3)
    q = (1.5 * torch.randn((3 + sum(NEWS) + 4, heads * group, dim), generator=g)).to(dtype).cuda()
    _check(ops, g, q, k_pages, v_pages, table, lengths, offsets, causal, max_query=max(NEWS))
    single = _offsets([1] * len(KEYS))
    _check(ops, g, q[:len(KEYS) + 2], k_pages, v_pages, table, lengths, single, causal, max_query=1)


@pytest.mark.parametrize('hint', [None, 1, 4, 100000])
@pytest.mark.parametrize('news', [[1, 1, 1], [9, 1, 300], [700, 0, 0]])
def test_attention_hint_changes_nothing(ops, hint, news):
    rng, g = np.random.default_rng(2), torch.Generator().manual_seed(2)
    k_pages, v_pages, table, lengths = _cache(rng, [1500, 90, 801], 2, 32, 128, torch.bfloat16)
    _fill((k_pages, v_pages), table, lengths, g)
    q = torch.randn((sum(news), 6, 128), generator=g).bfloat16().cuda()
    _check(ops, g, q, k_pages, v_pages, table, lengths, _offsets(news), True, max_query=hint)


@pytest.mark.parametrize('heads,group,dim,news', [(1, 1, 64, 1), (1, 8, 128, 1), (2, 4, 128, 3), (1, 1, 96, 40),
                                                  (1, 4, 128, 300), (1, 4, 96, 20), (1, 2, 96, 300)])
def test_attention_one_long_sequence(ops, heads, group, dim, news):
    """The keys of one sequence are divided over the whole card and joined."""
    rng, g = np.random.default_rng(3), torch.Generator().manual_seed(3)
    k_pages, v_pages, table, lengths = _cache(rng, [40_001], heads, 16, dim, torch.bfloat16)
    _fill((k_pages[:], v_pages[:]), table, lengths, g)
    q = torch.randn((news, heads * group, dim), generator=g).bfloat16().cuda()
    _check(ops, g, q, k_pages, v_pages, table, lengths, _offsets([news]), True, max_query=news)


@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('news', [1, 150])
def test_attention_extreme_scores(ops, dtype, news):
    """One dominant key late, scores of thousands, scores all alike, a base that keeps growing along the keys."""
    dtype, keys, dim = TYPES[dtype], 1000, 64
    rng, g = np.random.default_rng(4), torch.Generator().manual_seed(4)
    k_pages, v_pages, table, lengths = _cache(rng, [keys] * 4, 1, 16, dim, dtype)
    _fill((k_pages, v_pages), table, lengths, g)
    unit = torch.zeros(dim)
    unit[0] = 1
    ramps = [torch.where(torch.arange(keys) == keys - 200, 500., 0.), torch.linspace(-900, 900, keys).round(),
             torch.zeros(keys), torch.linspace(0, 60, keys)]
    for s, ramp in enumerate(ramps):
        for place in range(keys):
            k_pages[int(table[s, place // 16]), 0, place % 16] = (ramp[place] * unit).to(dtype)
    q = unit.expand(4 * news, 2, dim).to(dtype).cuda().contiguous()
    _check(ops, g, q, k_pages, v_pages, table, lengths, _offsets([news] * 4), True, scale=1.0, max_query=news)


@pytest.mark.parametrize('news', [1, 200])
def test_attention_not_a_number_stays_in_its_rows(ops, news):
    """A NaN or an infinity in a row of q, or in a key of one sequence, reaches that row or that sequence alone."""
    rng, g = np.random.default_rng(5), torch.Generator().manual_seed(5)
    k_pages, v_pages, table, lengths = _cache(rng, [300, 300], 2, 16, 64, torch.bfloat16)
    _fill((k_pages, v_pages), table, lengths, g)
    q = torch.randn((2 * news, 4, 64), generator=g).bfloat16().cuda()
    args = (table, lengths, _offsets([news, news]))
    clean = ops.paged_attention(q, k_pages, v_pages, *args, causal=False, max_query=news)
    dirty = q.clone()
    dirty[0, 1] = math.nan
    got = ops.paged_attention(dirty, k_pages, v_pages, *args, causal=False, max_query=news)
    assert bool(got[0, 1].isnan().all())
    got[0, 1] = clean[0, 1]
    assert torch.equal(got, clean)
    v_pages[int(table[1, 2]), 0, 3, 5] = math.inf
    got = ops.paged_attention(q, k_pages, v_pages, *args, causal=False, max_query=news)
    assert torch.equal(got[:news], clean[:news]) and torch.equal(got[:, 2:], clean[:, 2:])
    assert bool((got[news:, :2, 5] == math.inf).all())
    k_pages[int(table[1, 2]), 1, 3, 5] = math.nan
    got = ops.paged_attention(q, k_pages, v_pages, *args, causal=False, max_query=news)
    assert torch.equal(got[:news], clean[:news]) and bool(got[news:, 2:].isnan().all())


@pytest.mark.parametrize('news', [1, 90])
def test_attention_bad_pages(ops, news):
    """Page ids outside the pool read as zeros, lengths outside the table are clamped; both say so, and other sequences
    are as before."""
    from streamvoxel_b200 import _lib
    rng, g = np.random.default_rng(6), torch.Generator().manual_seed(6)
    k_pages, v_pages, table, lengths = _cache(rng, [100] * 4, 1, 16, 64, torch.float16, fill=0.0)
    _fill((k_pages, v_pages), table, lengths, g)
    q = torch.randn((4 * news, 2, 64), generator=g).half().cuda()
    offsets = _offsets([news] * 4)
    clean = ops.paged_attention(q, k_pages, v_pages, table, lengths, offsets, causal=False, max_query=news)
    table[1, 3], table[2, 0] = k_pages.shape[0], -1
    lengths[3] = 7 * 16 + 60
    status = torch.zeros(4, dtype=torch.int32, device='cuda')
    got = ops.paged_attention(q, k_pages, v_pages, table, lengths, offsets, causal=False, max_query=news, status=status)
    assert status.tolist() == [0] + [_lib.STATUS_BAD_PAGE] * 3
    assert torch.equal(got[:news], clean[:news]) and bool(got.isfinite().all())
    k_cpu, v_cpu = k_pages.cpu(), v_pages.cpu()
    for s, p in ((1, 3), (2, 0)):
        k, v = (ref.sequence_keys(t, table[s].clamp(0, k_cpu.shape[0] - 1).cpu(), 100).clone() for t in (k_cpu, v_cpu))
        k[:, p * 16:p * 16 + 16], v[:, p * 16:p * 16 + 16] = 0, 0
        rows = slice(s * news, (s + 1) * news)
        ref.close(got[rows], *ref.attend(q[rows].cpu(), k, v, False, 64 ** -0.5, torch.float16)[:2])


@pytest.mark.parametrize('news', [1, 70])
def test_attention_strided_queries(ops, news):
    rng, g = np.random.default_rng(7), torch.Generator().manual_seed(7)
    k_pages, v_pages, table, lengths = _cache(rng, [200, 131], 2, 64, 96, torch.bfloat16)
    _fill((k_pages, v_pages), table, lengths, g)
    packed = torch.randn((2 * news, 8, 96), generator=g).bfloat16().cuda()
    wide = torch.randn((4, 2 * news, 96), generator=g).bfloat16().cuda()
    for q in (packed[:, 2:6], wide.transpose(0, 1)):
        _check(ops, g, q, k_pages, v_pages, table, lengths, _offsets([news, news]), True, max_query=news)
    with pytest.raises(ValueError):
        ops.paged_attention(torch.zeros((2, 4, 100), device='cuda', dtype=torch.bfloat16)[:, :, :96], k_pages, v_pages,
                            table, lengths, _offsets([1, 1]))


def test_attention_many_sequences(ops):
    """More sequences than a block has threads, many of them empty."""
    rng, g = np.random.default_rng(8), torch.Generator().manual_seed(8)
    keys = rng.integers(0, 90, 700).tolist()
    news = [int(min(n, rng.choice([0, 1, 1, 2]))) for n in keys]
    k_pages, v_pages, table, lengths = _cache(rng, keys, 1, 16, 64, torch.bfloat16, fill=0.25)
    k_pages.copy_(torch.randn(k_pages.shape, generator=g))
    v_pages.copy_(torch.randn(v_pages.shape, generator=g))
    q = torch.randn((sum(news) + 3, 2, 64), generator=g).bfloat16().cuda()
    _check(ops, g, q, k_pages, v_pages, table, lengths, _offsets(news), True, max_query=2)
    news = [n if n else 0 for n in keys]
    q = torch.randn((sum(news), 2, 64), generator=g).bfloat16().cuda()
    _check(ops, g, q, k_pages, v_pages, table, lengths, _offsets(news), True, max_query=90)


@pytest.mark.parametrize('news,keys', [([600, 500, 700, 20, 650], [900, 500, 700, 3000, 651]),
                                       ([700, 1, 1, 700, 700, 700], [700, 9000, 5, 800, 2000, 710]),
                                       ([1400, 1100], [1400, 7000])])
def test_attention_many_units(ops, news, keys):
    """Enough token tiles to deal whole ones out to the CTAs before the rest is divided; lengths that make the dealt ones
    unequal."""
    rng, g = np.random.default_rng(11), torch.Generator().manual_seed(11)
    k_pages, v_pages, table, lengths = _cache(rng, keys, 8, 64, 64, torch.bfloat16)
    _fill((k_pages, v_pages), table, lengths, g)
    q = torch.randn((sum(news), 32, 64), generator=g).bfloat16().cuda()
    _check(ops, g, q, k_pages, v_pages, table, lengths, _offsets(news), True, max_query=max(news))


def test_attention_shared_pages(ops):
    """Sequences whose tables begin with the same pages (a shared prefix)."""
    rng, g = np.random.default_rng(9), torch.Generator().manual_seed(9)
    k_pages, v_pages, table, lengths = _cache(rng, [200, 200, 200], 2, 16, 64, torch.bfloat16)
    table[1:, :8] = table[0, :8]
    _fill((k_pages, v_pages), table, lengths, g)
    for news in (1, 40):
        q = torch.randn((3 * news, 4, 64), generator=g).bfloat16().cuda()
        _check(ops, g, q, k_pages, v_pages, table, lengths, _offsets([news] * 3), True, max_query=news)


def test_places_past_32_bits(ops):
    """Pools of more than 2^32 bytes and 2^31 values: pages at their end are stored and read."""
    pages, heads, page, dim = 140_000, 8, 16, 128
    assert pages * heads * page * dim > 2 ** 31
    pools = [torch.empty((pages, heads, page, dim), dtype=torch.bfloat16, device='cuda') for _ in range(2)]
    g = torch.Generator().manual_seed(10)
    table = torch.tensor([[pages - 1, 0, pages - 2, 65_537, 131_073]], dtype=torch.int32, device='cuda')
    lengths, offsets = torch.tensor([77], dtype=torch.int32, device='cuda'), _offsets([77])
    k, v = (torch.randn((77, heads, dim), generator=g).bfloat16().cuda() for _ in range(2))
    ops.paged_append(k, v, *pools, table, lengths, offsets)
    kept = [pool[table[0].long()].cpu() for pool in pools]
    for pool, rows in zip(kept, (k, v)):
        assert torch.equal(pool.transpose(1, 2).reshape(-1, heads, dim)[:77], rows.cpu())
    for news in (1, 77):
        q = torch.randn((news, 2 * heads, dim), generator=g).bfloat16().cuda()
        got = ops.paged_attention(q, *pools, table, lengths, _offsets([news]), max_query=news)
        want = ref.attend(q.cpu(), k.cpu().transpose(0, 1), v.cpu().transpose(0, 1), True, dim ** -0.5, q.dtype)
        ref.close(got, *want[:2])


# -------------------------------------------------------------------------------------------- streams and graphs


def _step(ops, s):
    q = ops.paged_append(s['k'], s['v'], s['k_pages'], s['v_pages'], s['table'], s['lengths'], s['offsets'],
                         inv_freq=s['freq'], q=s['q'])
    return ops.paged_attention(q, s['k_pages'], s['v_pages'], s['table'], s['lengths'], s['offsets'],
                               max_query=s['max_query'], workspace=s.get('workspace'))


def _state(ops, seed, news, keys, heads=2, group=4, dim=128, page=16):
    rng, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    k_pages, v_pages, table, lengths = _cache(rng, keys, heads, page, dim, torch.bfloat16, fill=0.0)
    _fill((k_pages, v_pages), table, lengths, g)
    tokens = sum(news)
    s = dict(k_pages=k_pages, v_pages=v_pages, table=table, lengths=lengths, offsets=_offsets(news),
             freq=ops.rope_frequencies(dim)[0], max_query=max(news))
    for name, n in (('k', heads), ('v', heads), ('q', heads * group)):
        s[name] = torch.randn((tokens, n, dim), generator=g).bfloat16().cuda()
    return s


@pytest.mark.parametrize('news', [[1, 1, 1], [200, 1, 60]])
def test_capture_and_replay(ops, news):
    """A captured step follows the lengths, tables and rows that its tensors hold at each replay; two graphs with
    workspaces of their own run side by side; eager calls give the same bits."""
    states = [_state(ops, 20 + i, news, [900, 300, 2000]) for i in range(2)]
    for s in states:
        s['workspace'] = ops.paged_attention_workspace(sum(news), 3, 8, 2, 128, 'cuda', max(news))
    graphs, outs = [], []
    for s in states:
        _step(ops, s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(ops, s))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for round_ in range(3):
        for s in states:
            s['lengths'].copy_(torch.tensor([900 - 200 * round_, 300, 2000 - 7 * round_]))
            s['q'].mul_(0.9)
        want = [_step(ops, s).clone() for s in states]
        for out in outs:
            out.fill_(9)
        torch.cuda.synchronize()
        for _ in range(20):
            for stream, graph in zip(streams, graphs):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert torch.equal(out, w)


def test_other_stream(ops):
    """Work on a side stream is ordered with that stream's other work."""
    s = _state(ops, 30, [1, 1], [500, 3000])
    want = _step(ops, s)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        s['q'].mul_(2)
        s['q'].mul_(0.5)
        got = _step(ops, s)
    stream.synchronize()
    assert torch.equal(got, want)


def test_repeated_calls_give_the_same_bits(ops):
    s = _state(ops, 31, [1, 1, 30, 1], [9000, 17, 4000, 800])
    first = _step(ops, s)
    for _ in range(5):
        assert torch.equal(_step(ops, s), first)


# ------------------------------------------------------------------------------------------------- runs of them


@pytest.mark.parametrize('dtype,dim,heads,group,layout', [('bf16', 128, 2, 4, 'half'), ('fp16', 64, 4, 1, 'interleaved')])
def test_prompt_in_chunks_then_single_tokens(ops, dtype, dim, heads, group, layout):
    """Two conversations: prompts in chunks, then token by token, pages handed out as they grow. Every step's rows equal
    the attention of the whole history, the keys rotated in 64 bits and rounded once."""
    dtype, page, totals = TYPES[dtype], 16, (230, 90)
    g = torch.Generator().manual_seed(40)
    freq, scale = ops.rope_frequencies(dim, scaling='by_parts', factor=4.0, original=512)
    pools = [torch.full((40, heads, page, dim), math.nan, dtype=dtype, device='cuda') for _ in range(2)]
    free, table = list(range(39, -1, -1)), torch.zeros((2, 16), dtype=torch.int32)
    rows = [{n: torch.randn((t, h, dim), generator=g).to(dtype) for n, h in (('k', heads), ('v', heads),
                                                                             ('q', heads * group))} for t in totals]
    done, held = [0, 0], [0, 0]
    for news in [(100, 64), (97, 0), (30, 23)] + [(1, 1)] * 3:
        for s in range(2):
            while held[s] * page < done[s] + news[s]:
                table[s, held[s]] = free.pop()
                held[s] += 1
        step = {n: torch.cat([r[n][d:d + k] for r, d, k in zip(rows, done, news)]).cuda() for n in 'kvq'}
        lengths = torch.tensor([d + k for d, k in zip(done, news)], dtype=torch.int32, device='cuda')
        args = (*pools, table.cuda(), lengths, _offsets(news))
        q = ops.paged_append(step['k'], step['v'], *args, inv_freq=freq, layout=layout, rope_scale=scale, q=step['q'])
        out = ops.paged_attention(q, *args, max_query=max(news))
        at = 0
        for s in range(2):
            n, length = news[s], done[s] + news[s]
            k = ref.sequence_keys(pools[0], args[2][s], length).cpu()
            want_k, bound_k = ref.rotate(rows[s]['k'][:length], torch.arange(length), freq, layout, scale)
            ref.close(k.transpose(0, 1), want_k, bound_k)
            if n:
                want = ref.attend(q[at:at + n].cpu(), k, rows[s]['v'][:length].transpose(0, 1), True, dim ** -0.5, dtype)
                ref.close(out[at:at + n], *want[:2])
            at += n
            done[s] = length


def test_windows_cross_attention_over_pages(ops):
    """The condition keys of two windows as the engine's encoder makes them, stored in pages instead of slot buffers: the
    cross-attention over them agrees with `ops.attention` over the slot buffers."""
    from streamvoxel_b200 import model as sm
    cfg = sm.small_test_config()
    prepared = sm.PreparedModel(cfg, sm.synthetic_state_dict(cfg, seed=2, std=0.05), 'cuda')
    g = torch.Generator().manual_seed(41)
    counts, heads, page = (333, 200), cfg.heads, 64
    rng = np.random.default_rng(41)
    k_pages, v_pages, table, lengths = _cache(rng, counts, heads, page, 96, torch.bfloat16)
    slot_k, slot_v = (torch.zeros((2, heads, 384, 96), dtype=torch.bfloat16, device='cuda') for _ in range(2))
    keys, values = [], []
    for s, n in enumerate(counts):
        tokens = torch.randn((n, cfg.d), generator=g).cuda()
        positions = (torch.randint(-60, 60, (n, 3), generator=g).float() / 2).cuda()
        k, v = prepared.key_values(tokens, positions)[0]      # [heads, n, 96], keys rotated
        slot_k[s, :, :n], slot_v[s, :, :n] = k, v
        keys.append(k.transpose(0, 1))
        values.append(v.transpose(0, 1))
    offsets = _offsets(counts)
    ops.paged_append(torch.cat(keys), torch.cat(values), k_pages, v_pages, table, lengths, offsets)
    for s, n in enumerate(counts):
        assert torch.equal(ref.sequence_keys(k_pages, table[s], n), slot_k[s, :, :n])
    queries = cfg.patches
    q = torch.randn((2 * queries, heads, 96), generator=g).bfloat16().cuda()
    got = ops.paged_attention(q, k_pages, v_pages, table, lengths, _offsets([queries] * 2), causal=False,
                              max_query=queries)
    slots = ops.attention(q, slot_k, slot_v, 2, heads, queries, 384, q_row_stride=heads * 96,
                          kv_slot_stride=heads * 384 * 96, kv_head_stride=384 * 96, kv_row_stride=96, lengths=lengths)
    for s, n in enumerate(counts):
        rows = slice(s * queries, (s + 1) * queries)
        want, bound = ref.attend(q[rows].cpu(), slot_k[s, :, :n].cpu(), slot_v[s, :, :n].cpu(), False, 96 ** -0.5,
                                 torch.bfloat16)[:2]
        ref.close(got[rows], want, bound)
        # the slot form has the same roundings, and a quarter of its exponentials 2.7e-6 off
        ref.close(slots[rows].view(queries, heads, 96), want, bound * 1.01)

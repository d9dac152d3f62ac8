"""Edges of the rotary and paged-cache operators on the GPU: calls that their documentation allows and that once went wrong."""
import math

import numpy as np
import pytest
import torch

import paged_reference as ref
from test_gpu_paged import TYPES, _cache, _check, _fill, _offsets

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ops():
    from streamvoxel_b200 import _lib, ops
    _lib.require_device()
    return ops


@pytest.fixture(autouse=True)
def no_grad():
    with torch.no_grad():
        yield


@pytest.mark.parametrize('news,lengths,heads,group,page,causal', [
    ([512] * 16, [512] * 16, 8, 4, 64, True), ([753, 1163, 511], [820, 3847, 679], 4, 8, 64, True),
    ([784, 768, 3184], [128, 320, 128], 1, 16, 16, False)])
def test_whole_units_that_fill_a_share(ops, news, lengths, heads, group, page, causal):
    """Batches in which the units that a CTA takes whole are its share exactly: nothing is joined that this call did not
    write, whatever the workspace held before."""
    rng, g = np.random.default_rng(23), torch.Generator().manual_seed(23)
    k_pages, v_pages, table, lengths = _cache(rng, lengths, heads, page, 64, torch.bfloat16)
    _fill((k_pages, v_pages), table, lengths, g)
    offsets = _offsets(news)
    q = torch.randn((sum(news), heads * group, 64), generator=g).bfloat16().cuda()
    workspace = ops.paged_attention_workspace(sum(news), len(news), heads * group, heads, 64, 'cuda', max(news))
    lse = torch.empty((sum(news), heads * group), device='cuda')
    want, bound, want_lse, lse_bound, _ = ref.attention(q, k_pages, v_pages, table, lengths, offsets.cpu(), causal)
    for fill in (255, 0, 0x7f):   # NaN, zeros, 3.4e38
        workspace.fill_(fill)
        got = ops.paged_attention(q, k_pages, v_pages, table, lengths, offsets, causal=causal, lse=lse,
                                  max_query=max(news), workspace=workspace)
        ref.close(got, want, bound)
        ref.close(lse, want_lse, lse_bound)


@pytest.mark.parametrize('news', [5, 60, 200])   # one form of the kernel each
@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('kind', ['hidden', 'far below'])
def test_values_without_weight_count_nothing(ops, dtype, news, kind):
    """Values near the type's largest behind keys that the mask hides, or whose weight is under 2^-200, add nothing."""
    rng, g, dtype = np.random.default_rng(20), torch.Generator().manual_seed(20), TYPES[dtype]
    keys, dim, last = 300, 64, 20 if news > 20 else 2
    k_pages, v_pages, table, lengths = _cache(rng, [keys], 2, 16, dim, dtype)
    _fill((k_pages, v_pages), table, lengths, g)
    largest = 2.0 ** 127 if dtype == torch.bfloat16 else 2.0 ** 15
    q = torch.randn((news, 2, dim), generator=g).to(dtype).cuda()
    q[..., 0] = 1
    for place in range(keys - last, keys):
        v_pages[int(table[0, place // 16]), :, place % 16] = largest
        if kind != 'hidden':
            k_pages[int(table[0, place // 16]), :, place % 16, 0] = -1200   # scores of -150
    args = q, k_pages, v_pages, table, lengths, _offsets([news])
    got = ops.paged_attention(*args, causal=kind == 'hidden', max_query=news)
    want, bound = ref.attention(*args[:5], args[5].cpu(), kind == 'hidden')[:2]
    rows = news - last if kind == 'hidden' else news   # the last rows see those values
    ref.close(got[:rows], want[:rows], bound[:rows])


@pytest.mark.parametrize('news,length,hint', [(5, 2, 5), (16, 3, 16), (40, 7, 40), (40, 7, 1), (300, 30, 300)])
def test_rows_without_keys_take_nothing_from_their_neighbours(ops, news, length, hint):
    """Fewer keys than new tokens: the first rows see none and give 0, whatever the values of the others' keys are."""
    rng, g = np.random.default_rng(21), torch.Generator().manual_seed(21)
    k_pages, v_pages, table, lengths = _cache(rng, [length], 1, 16, 64, torch.bfloat16)
    _fill((k_pages, v_pages), table, lengths, g)
    v_pages[int(table[0, 0]), :, :length] = math.nan
    v_pages[int(table[0, 0]), :, 0] = math.inf
    q = torch.randn((news, 1, 64), generator=g).bfloat16().cuda()
    lse = torch.zeros((news, 1), device='cuda')
    out = ops.paged_attention(q, k_pages, v_pages, table, lengths, _offsets([news]), lse=lse, max_query=hint)
    none = news - length
    assert bool((out[:none] == 0).all()) and bool((lse[:none] == -math.inf).all())
    assert not bool(out[none:].isfinite().any()) and bool(lse[none:].isfinite().all())


@pytest.mark.parametrize('layout', ['interleaved', 'half'])
@pytest.mark.parametrize('positions', [torch.tensor([2 ** 50, 2 ** 54 + 4, -2 ** 62 + 512, 2 ** 63 - 1]),
                                       torch.tensor([1e17, -3e20, 1e30, 3e38])])
def test_rope_of_any_position_is_a_rotation(ops, positions, layout):
    """Positions past what float64 angles resolve still turn every pair without changing its length."""
    freq, _ = ops.rope_frequencies(64)
    x = torch.randn((4, 3, 64), generator=torch.Generator().manual_seed(22)).cuda()
    y = ops.rope(x, positions.cuda(), freq, layout=layout).double()
    pair = (lambda t: t.unflatten(-1, (2, 32)).movedim(-2, -1)) if layout == 'half' else \
        (lambda t: t.unflatten(-1, (32, 2)))
    before, after = pair(x.double()).norm(dim=-1), pair(y).norm(dim=-1)
    # cosine and sine within 2^-22 each, two products and a sum: 2^-21 of |a| + |b| a value, two values, |a| + |b| <= 1.5 r
    assert bool(((after - before).abs() <= 2.0 ** -19 * before).all())


def _saved(tensor):
    """A product whose backward pass needs `tensor` as it is now."""
    with torch.enable_grad():
        leaf = torch.ones_like(tensor, requires_grad=True)
        return (leaf * tensor).sum()


def _spoilt(product):
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        product.backward()


def test_written_tensors_spoil_backward_passes_that_saved_them(ops):
    """Outputs that the caller hands in, and the pools, are in-place writes for autograd."""
    rng, g = np.random.default_rng(24), torch.Generator().manual_seed(24)
    freq, _ = ops.rope_frequencies(64)
    x, positions = torch.randn((4, 2, 64), generator=g).cuda(), torch.arange(4, device='cuda')
    untouched, packed = _saved(x), torch.randn((4, 6, 64), generator=g).cuda()
    product = _saved(packed)
    ops.rope(x, positions, freq, out=packed[:, 2:4])   # a view of the saved tensor
    _spoilt(product)
    product = _saved(x)
    ops.rope(x, positions, freq)
    untouched.backward()
    product.backward()
    k_pages, v_pages, table, lengths = _cache(rng, [4], 2, 16, 64, torch.bfloat16, fill=0.0)
    k, v = (torch.randn((4, 2, 64), generator=g).bfloat16().cuda() for _ in range(2))
    q_out, args = torch.zeros_like(k), (k_pages, v_pages, table, lengths, _offsets([4]))
    products = [_saved(t) for t in (k_pages, v_pages, q_out)]
    ops.paged_append(k, v, *args, inv_freq=freq, q=k, q_out=q_out)
    for product in products:
        _spoilt(product)
    out, lse = torch.zeros_like(k), torch.zeros((4, 2), device='cuda')
    products = [_saved(t) for t in (out, lse)]
    kept = _saved(k_pages)
    ops.paged_attention(k, *args, out=out, lse=lse)
    for product in products:
        _spoilt(product)
    kept.backward()   # the pools were only read


def test_tensors_of_inference_mode(ops):
    """Pools and outputs made under inference mode, which have no version, are written in and outside of it."""
    rng, g = np.random.default_rng(25), torch.Generator().manual_seed(25)
    freq, _ = ops.rope_frequencies(64)
    with torch.inference_mode():
        k_pages, v_pages, table, lengths = _cache(rng, [4], 2, 16, 64, torch.bfloat16, fill=0.0)
        k = torch.randn((4, 2, 64), generator=g).bfloat16().cuda()
        args = (k_pages, v_pages, table, lengths, _offsets([4]))
        out = torch.zeros_like(k)
    for mode in (torch.inference_mode, torch.no_grad):
        with mode():
            q = ops.paged_append(k, k, *args, inv_freq=freq, q=k)
            assert ops.paged_attention(q, *args, out=out) is out
            assert ops.rope(out, torch.arange(4, device='cuda'), freq, out=out) is out

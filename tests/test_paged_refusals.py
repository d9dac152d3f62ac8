"""More refusals of the rotary and paged-cache operators, each by its reason; they come before any launch."""
import pytest
import torch
from torch.autograd import forward_ad

from streamvoxel_b200 import build, ops


@pytest.fixture(scope='module', autouse=True)
def lib():
    build.build()


def _rope_args():
    return dict(x=torch.zeros(4, 2, 64), positions=torch.zeros(4), inv_freq=torch.ones(32, dtype=torch.float64), out=None)


def _append_args():
    half = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16)  # noqa: E731
    return dict(k=half(2, 2, 64), v=half(2, 2, 64), k_pages=half(6, 2, 16, 64), v_pages=half(6, 2, 16, 64),
                table=torch.zeros((2, 3), dtype=torch.int32), lengths=torch.ones(2, dtype=torch.int32),
                offsets=torch.arange(3, dtype=torch.int32), q=half(2, 4, 64), q_out=half(2, 4, 64),
                inv_freq=torch.ones(32, dtype=torch.float64), positions=torch.zeros(2))


def _attention_args():
    args = {n: t for n, t in _append_args().items() if n not in ('k', 'v', 'q_out', 'inv_freq', 'positions')}
    return dict(args, out=torch.zeros_like(args['q']), lse=torch.zeros(2, 4))


CALLS = [(ops.rope, _rope_args, 'positions'), (ops.rope, _rope_args, 'inv_freq'), (ops.rope, _rope_args, 'out')]
CALLS += [(ops.paged_append, _append_args, n) for n in
          ('k', 'v', 'k_pages', 'v_pages', 'q', 'q_out', 'inv_freq', 'positions')]
CALLS += [(ops.paged_attention, _attention_args, n) for n in ('q', 'k_pages', 'v_pages', 'out', 'lse')]


@pytest.mark.parametrize('call,make,name', CALLS)
def test_gradients_are_not_lost(call, make, name):
    """An operand that requires grad, or has a forward-mode tangent, and that the operator has no derivative for."""
    args = make()
    if args[name] is None:
        args[name] = torch.zeros(4, 2, 64)
    args[name].requires_grad_()
    with pytest.raises(ValueError, match='gradient|autograd'):
        call(**args)
    with torch.no_grad(), pytest.raises(ValueError, match='one CUDA device'):   # a constant there: the next check
        call(**args)
    args[name] = args[name].detach()
    with forward_ad.dual_level():
        args[name] = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(ValueError, match='gradient|autograd'):
            call(**args)


def test_rope_refuses_forward_mode():
    args = _rope_args()
    with forward_ad.dual_level():
        args['x'] = forward_ad.make_dual(args['x'], torch.ones_like(args['x']))
        with pytest.raises(ValueError, match='forward-mode'):
            ops.rope(**args)


def _far(shape, like):
    """A tensor of that shape without memory behind it (strides 0)."""
    return torch.zeros([1] * len(shape), dtype=like.dtype).expand(shape)


@pytest.mark.parametrize('shape', [(2 ** 31, 2, 64), (2 ** 32 + 4, 2, 64), (4, 2 ** 32 + 2, 64)])
def test_rope_refuses_sizes_past_32_bits(shape):
    args = _rope_args()
    args['x'] = _far(shape, args['x'])
    with pytest.raises(ValueError, match='past 32 bits'):
        ops.rope(**args)


def test_append_refuses_sizes_past_32_bits():
    args = _append_args()
    args['k'] = args['v'] = _far((2 ** 32 + 2, 2, 64), args['k'])
    with pytest.raises(ValueError, match='past 32 bits'):
        ops.paged_append(**args)


def test_attention_refuses_sizes_past_32_bits():
    args = _attention_args()
    args['q'] = _far((2 ** 32 + 2, 4, 64), args['q'])
    with pytest.raises(ValueError, match='past 32 bits'):
        ops.paged_attention(**args)


@pytest.mark.parametrize('call,make', [(ops.paged_append, _append_args), (ops.paged_attention, _attention_args)])
@pytest.mark.parametrize('change,reason', [
    (dict(table=(2 ** 20 + 1, 3), lengths=(2 ** 20 + 1,), offsets=(2 ** 20 + 2,)), 'sequences'),
    (dict(table=(2, 2 ** 32 + 3)), 'keys a sequence'), (dict(table=(2, 2 ** 26 + 1)), 'keys a sequence'),
    (dict(k_pages=(6, 0, 16, 64), v_pages=(6, 0, 16, 64)), 'heads'),
    (dict(k_pages=(6, 1025, 16, 64), v_pages=(6, 1025, 16, 64)), 'heads'),
    (dict(k_pages=(0, 2, 16, 64), v_pages=(0, 2, 16, 64)), 'pages')])
def test_caches_refuse_sizes(call, make, change, reason):
    args = make()
    for name, shape in change.items():
        args[name] = _far(shape, args[name])
    with pytest.raises(ValueError, match=reason):
        call(**args)


@pytest.mark.parametrize('scale', [1e39, -1e39, float('inf'), float('nan')])
def test_rotary_scales_are_finite_in_32_bits(scale):
    with pytest.raises(ValueError, match='finite'):
        ops.rope(**_rope_args(), scale=scale)
    with pytest.raises(ValueError, match='finite'):
        ops.paged_append(**_append_args(), rope_scale=scale)

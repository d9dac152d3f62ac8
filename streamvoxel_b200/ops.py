"""Torch-tensor wrappers over the libsvx entry points (device tensors in, device tensors out, current stream).

Each wrapper validates dtypes/shapes on the host and calls exactly one C-ABI function; there is no CPU path.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from streamvoxel_b200 import _lib
from streamvoxel_b200._lib import check, ptr, stream_ptr

STEP_DTYPE = np.dtype([('k', '<i4'), ('step', '<i4'), ('committed', '<i8'), ('frac', '<f8'), ('seed', '<u8')])
assert STEP_DTYPE.itemsize == ctypes.sizeof(_lib.StepParams)


def _dtype_code(t):
    if t.dtype == torch.bfloat16:
        return _lib.BF16
    if t.dtype == torch.float32:
        return _lib.F32
    raise ValueError(f'logits must be bf16 or fp32, got {t.dtype}')


def step_params(rows, device=None, out=None):
    """Pack per-slot step scalars [(k, step, committed, frac, seed)] into an `svx_step_params` array.

    Returns a uint8 tensor on `device` (or copies into `out`, a pinned/device uint8 tensor of the right size)."""
    arr = np.zeros(len(rows), STEP_DTYPE)
    for i, (k, step, committed, frac, seed) in enumerate(rows):
        arr[i] = (int(k), int(step), int(committed), float(frac), int(seed) & 0xFFFFFFFFFFFFFFFF)
    host = torch.from_numpy(arr.view(np.uint8).copy())
    if out is not None:
        out.copy_(host, non_blocking=False)
        return out
    return host.to(device)


def _slots_view(logits):
    """[S, C, ...] contiguous -> (S, C, voxels, slot stride)."""
    if not logits.is_contiguous():
        raise ValueError('logits must be contiguous [slots, classes, Y, Z, X]')
    s, c = logits.shape[0], logits.shape[1]
    voxels = logits[0, 0].numel()
    return s, c, voxels, c * voxels


def ease_scores(logits, status=None, out=None):
    """Negative entropy per voxel of class-major logits [S, C, Y, Z, X] -> fp32 [S, Y, Z, X]."""
    s, c, voxels, stride = _slots_view(logits)
    scores = out if out is not None else torch.empty((s, *logits.shape[2:]), device=logits.device, dtype=torch.float32)
    check(_lib.load().svx_ease_scores(ptr(logits), _dtype_code(logits), s, c, voxels, stride, ptr(scores), ptr(status),
                                      stream_ptr()), 'svx_ease_scores')
    return scores


def ease_mark(logits, air_ids, last_eps, last=None, last_count=None):
    """Marking forward: per-column top run of voxels with P(air) > 1 - eps. Returns (last uint8, last_count int32).
    air_ids: a sequence of ids, or an int32 device tensor of them (no host-to-device copy per call)."""
    s, c, voxels, stride = _slots_view(logits)
    height, depth, width = logits.shape[2:]
    dev = logits.device
    if last is None:
        last = torch.empty((s, height, depth, width), device=dev, dtype=torch.uint8)
    if last_count is None:
        last_count = torch.empty(s, device=dev, dtype=torch.int32)
    if isinstance(air_ids, torch.Tensor) and air_ids.is_cuda:
        air = air_ids
        assert air.dtype == torch.int32 and air.is_contiguous()
    else:
        air = torch.as_tensor(list(air_ids), dtype=torch.int32, device=dev)
    check(_lib.load().svx_ease_mark(ptr(logits), _dtype_code(logits), s, c, height, depth, width, stride, ptr(air),
                                    len(air), float(last_eps), ptr(last), ptr(last_count), stream_ptr()),
          'svx_ease_mark')
    return last, last_count


def select_workspace(slots, voxels, device):
    n = _lib.load().svx_ease_select_workspace_bytes(slots, voxels)
    return torch.empty(n, dtype=torch.uint8, device=device)


def ease_select(scores, tokens, last, pos, params, mask_id, index_capacity, *, chosen=None, index=None, count=None,
                status=None, workspace=None, block=4):
    """Block-quota selection. Returns (chosen uint8 [S,Y,Z,X], index int32 [S, capacity], count int32 [S])."""
    s, height, depth, width = tokens.shape
    dev = tokens.device
    assert tokens.dtype == torch.int16 and last.dtype == torch.uint8 and scores.dtype == torch.float32
    assert pos.dtype == torch.int32 and params.dtype == torch.uint8
    if chosen is None:
        chosen = torch.empty((s, height, depth, width), device=dev, dtype=torch.uint8)
    if index is None:
        index = torch.empty((s, index_capacity), device=dev, dtype=torch.int32)
    if count is None:
        count = torch.empty(s, device=dev, dtype=torch.int32)
    if workspace is None:
        workspace = select_workspace(s, height * depth * width, dev)
    check(_lib.load().svx_ease_select(ptr(scores), ptr(tokens), ptr(last), ptr(pos), ptr(params), s, height, depth,
                                      width, block, mask_id, ptr(chosen), ptr(index), index_capacity, ptr(count),
                                      ptr(status), ptr(workspace), stream_ptr()), 'svx_ease_select')
    return chosen, index, count


EVAL_MODES = dict(random=0, entropy=1, mixed=2, block=3, threshold=4)


def eval_params(rows, device):
    """Pack per-slot evaluation-step scalars [(mode, k, candidates, committed, threshold, step)] (`svx_eval_params`)
    into a device uint8 tensor."""
    arr = (_lib.EvalParams * len(rows))(*[_lib.EvalParams(EVAL_MODES[m] if isinstance(m, str) else int(m), int(k),
                                                          int(c), int(done), float(th), int(st))
                                          for m, k, c, done, th, st in rows])
    host = torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8)
    return host.to(device)


def eval_select(scores, draw, tokens, pos, params, mask_id, *, chosen, index, count, commit_step=None,
                quota_range=None, status=None):
    """Selections of the evaluation decoders (random / entropy / mixed / block / threshold) over the masked voxels
    of each slot: fills chosen [S, Y, Z, X] uint8, index [S, capacity] (ascending, -1 padded), count [S] and, when
    given, commit_step [S, Y, Z, X] int32 and quota_range [S, 2] int32."""
    s, height, depth, width = tokens.shape
    check(_lib.load().svx_eval_select(ptr(scores), ptr(draw), ptr(tokens), ptr(pos), ptr(params), s, height, depth,
                                      width, mask_id, ptr(chosen), ptr(index), index.shape[1], ptr(count),
                                      ptr(commit_step), ptr(quota_range), ptr(status), stream_ptr()),
          'svx_eval_select')
    return chosen, index, count


def ease_sample(logits, index, params, tokens, noise=None, values=None, status=None):
    """Categorical draw for the chosen voxels; writes tokens in place. noise [S, capacity, C] fp32 or None (native)."""
    s, c, voxels, stride = _slots_view(logits)
    capacity = index.shape[1]
    if values is None:
        values = torch.empty((s, capacity), device=logits.device, dtype=torch.int16)
    noise_stride = 0
    if noise is not None:
        assert noise.dtype == torch.float32 and noise.is_contiguous() and noise.shape[-1] == c
        noise_stride = noise[0].numel() if noise.dim() == 3 else 0
    check(_lib.load().svx_ease_sample(ptr(logits), _dtype_code(logits), s, c, voxels, stride, ptr(index), ptr(params),
                                      ptr(noise), noise_stride, capacity, ptr(tokens), ptr(values), ptr(status),
                                      stream_ptr()), 'svx_ease_sample')
    return values


def softmax_rows(x):
    out = torch.empty_like(x)
    check(_lib.load().svx_softmax_rows(ptr(x), x.shape[0], x.shape[1], ptr(out), stream_ptr()), 'svx_softmax_rows')
    return out


def ease_finish(tokens, last, finish, air_token):
    s = tokens.shape[0]
    check(_lib.load().svx_ease_finish(ptr(tokens), ptr(last), ptr(finish), s, tokens[0].numel(), int(air_token),
                                      stream_ptr()), 'svx_ease_finish')


def patch_embed(tokens, classes, table_b, bias_b, add_b, table_c=None, bias_c=None, add_c=None, out_b=None,
                out_c=None, stats_b=None, stats_c=None):
    """Patch-4 token embed of both branches; stats_b / stats_c (optional fp32 [d/32, rows, 2]) receive each output
    row's 32-column chunk statistics (mean, M2), chunk-major, for the LayerNorm fold of the next linear."""
    s, height, depth, width = tokens.shape
    d = table_b.shape[1]
    patches = (height // 4) * (depth // 4) * (width // 4)
    if out_b is None:
        out_b = torch.empty((s * patches, d), device=tokens.device, dtype=torch.bfloat16)
    if table_c is not None and out_c is None:
        out_c = torch.empty((s * patches, d), device=tokens.device, dtype=torch.bfloat16)
    check(_lib.load().svx_patch_embed(ptr(tokens), s, height, depth, width, 4, classes, d, ptr(table_b), ptr(bias_b),
                                      ptr(add_b), ptr(out_b), ptr(table_c), ptr(bias_c), ptr(add_c), ptr(out_c),
                                      ptr(stats_b), ptr(stats_c), stream_ptr()), 'svx_patch_embed')
    return out_b, out_c


def layernorm_modulate(x, eps=1e-6, one_plus_scale=None, shift=None, out=None):
    rows, d = x.shape
    if out is None:
        out = torch.empty_like(x)
    check(_lib.load().svx_layernorm_modulate(ptr(x), rows, d, float(eps), ptr(one_plus_scale), ptr(shift), ptr(out),
                                             stream_ptr()), 'svx_layernorm_modulate')
    return out


def layernorm_affine(x, eps, pre=None, weight=None, bias=None, gelu=False, out=None):
    """bf16(g(LN(x + pre) * weight + bias)) in fp32 (the condition encoder's LayerNorms; g = GELU(erf) with gelu).
    x [rows, d] bf16; pre, weight, bias [d] fp32 or None."""
    rows, d = x.shape
    if out is None:
        out = torch.empty_like(x)
    check(_lib.load().svx_layernorm_affine(ptr(x), rows, d, float(eps), ptr(pre), ptr(weight), ptr(bias), int(gelu),
                                           ptr(out), stream_ptr()), 'svx_layernorm_affine')
    return out


def gemm(a, w, bias, epilogue=_lib.EPI_BIAS, out=None, gate=None, residual=None, rope=None, rope_cols=0,
         rows_per_slot=0, head_dim=96, classes=0, geometry=(0, 0, 0), ln=None, stats_out=None):
    """out = epilogue(a @ w.T + bias) on the tcgen05 GEMM. a [M,K], w [N,K], bias [N] bf16.
    ln = (stats [K/32, M, 2] fp32, u [N], v [N] fp32, eps): the LayerNorm folded in, out = epilogue(r (acc - mu u) + v)
    with w the modulated weights; stats_out: fp32 [N/32, M, 2] chunk statistics of the bf16 output rows."""
    m, k = a.shape
    n = w.shape[0]
    for t in (a, w, bias):
        assert t.dtype == torch.bfloat16 and t.is_contiguous()
    if out is None:
        if epilogue == _lib.EPI_CLASS_MAJOR:
            out = torch.empty((m // rows_per_slot, classes, *geometry), device=a.device, dtype=torch.bfloat16)
        else:
            out = torch.empty((m, n), device=a.device, dtype=torch.bfloat16)
    args = _lib.EpilogueArgs(epilogue=epilogue, bias=bias.data_ptr(), gate=ptr(gate).value, residual=ptr(residual).value,
                             rope_sin=ptr(rope[0] if rope else None).value, rope_cos=ptr(rope[1] if rope else None).value,
                             rope_cols=rope_cols, rows_per_slot=rows_per_slot, head_dim=head_dim, classes=classes,
                             height=geometry[0], depth=geometry[1], width=geometry[2], patch=4)
    if ln is not None:
        stats, u, v, eps = ln
        assert stats.dtype == u.dtype == v.dtype == torch.float32
        args.ln_stats_in, args.ln_u, args.ln_v, args.ln_eps = ptr(stats).value, ptr(u).value, ptr(v).value, eps
    if stats_out is not None:
        assert stats_out.dtype == torch.float32
        args.ln_stats_out = ptr(stats_out).value
    check(_lib.load().svx_gemm(ptr(a), ptr(w), ptr(out), m, n, k, ctypes.byref(args), stream_ptr()), 'svx_gemm')
    return out


def gemm_group(problems):
    """Two gated-residual GEMMs with row statistics in one launch (`svx_gemm_group`): problems = two dicts with a, w,
    bias, gate, residual, stats_out (and optional out); out_i = bf16(res_i + bf16(gate_i bf16(a_i w_i^T + bias_i))).
    Returns the two outputs."""
    outs, args = [], []
    for p in problems:
        m, k = p['a'].shape
        n = p['w'].shape[0]
        for t in (p['a'], p['w'], p['bias'], p['gate'], p['residual']):
            assert t.dtype == torch.bfloat16 and t.is_contiguous()
        assert p['stats_out'].dtype == torch.float32
        out = p.get('out')
        if out is None:
            out = torch.empty((m, n), device=p['a'].device, dtype=torch.bfloat16)
        outs.append(out)
        args.append(_lib.EpilogueArgs(epilogue=_lib.EPI_GATE_RESIDUAL, bias=p['bias'].data_ptr(),
                                      gate=p['gate'].data_ptr(), residual=p['residual'].data_ptr(),
                                      ln_stats_out=p['stats_out'].data_ptr(), patch=4))
    (m, k), n = problems[0]['a'].shape, problems[0]['w'].shape[0]
    assert problems[1]['a'].shape == (m, k) and problems[1]['w'].shape == (n, k)
    check(_lib.load().svx_gemm_group(ptr(problems[0]['a']), ptr(problems[0]['w']), ptr(outs[0]), ctypes.byref(args[0]),
                                     ptr(problems[1]['a']), ptr(problems[1]['w']), ptr(outs[1]), ctypes.byref(args[1]),
                                     m, n, k, stream_ptr()), 'svx_gemm_group')
    return outs


def attention_plan(lengths, slots, heads, queries, keys, ctas, device=None):
    """Work-unit plan of `svx_attention_plan` for host key lengths (sequence or None) on `ctas` CTAs. Returns the
    int32 plan (on `device`, or a host tensor) and the CTA count the launch must use."""
    lib = _lib.load()
    size = lib.svx_attention_plan_ints(slots, heads, queries, ctas)
    if size <= 0:
        raise ValueError('attention_plan: bad shape')
    plan = torch.empty(size, dtype=torch.int32)
    host = None if lengths is None else torch.as_tensor(list(lengths), dtype=torch.int32)
    check(lib.svx_attention_plan(ptr(host), slots, heads, queries, keys, ctas, ptr(plan), size),
          'svx_attention_plan')
    units = slots * heads * ((queries // 128 + 1) // 2)
    return (plan if device is None else plan.to(device)), min(ctas, units)


def attention_multi_plan(problems, slots, heads, queries, ctas, device=None):
    """Joint work plan of `svx_attention_multi_plan` for one or two problems, each given as (host key lengths or
    None, keys). Returns the int32 plan (on `device`, or a host tensor) and the CTA count the launch must use."""
    lib = _lib.load()
    count = len(problems)
    size = lib.svx_attention_multi_plan_ints(count, slots, heads, queries, ctas)
    if size <= 0:
        raise ValueError('attention_multi_plan: bad shape')
    hosts = [None if lengths is None else torch.as_tensor(list(lengths), dtype=torch.int32)
             for lengths, _ in problems]
    lens = (ctypes.c_void_p * count)(*[None if h is None else h.data_ptr() for h in hosts])
    keys = (ctypes.c_int * count)(*[int(k) for _, k in problems])
    plan = torch.empty(size, dtype=torch.int32)
    check(lib.svx_attention_multi_plan(lens, keys, count, slots, heads, queries, ctas, ptr(plan), size),
          'svx_attention_multi_plan')
    units = count * slots * heads * ((queries // 128 + 1) // 2)
    return (plan if device is None else plan.to(device)), min(ctas, units)


def attention_multi(problems, slots, heads, queries, plan):
    """One launch over one or two attention problems (dicts of `attention`'s arguments: q, k, v, keys, the four
    strides, lengths, out), with a plan from `attention_multi_plan`. Returns the outputs."""
    raw = _lib.raw_ptr
    table, ctas = plan
    structs = []
    for pr in problems:
        structs.append(_lib.AttentionProblem(raw(pr['q']), raw(pr['k']), raw(pr['v']), pr['q_row_stride'],
                                             pr['kv_slot_stride'], pr['kv_head_stride'], pr['kv_row_stride'],
                                             ptr(pr.get('lengths')), pr['keys'], ptr(pr['out'])))
    arr = (_lib.AttentionProblem * len(structs))(*structs)
    check(_lib.load().svx_attention_multi(arr, len(structs), slots, heads, queries, ptr(table), ctas, stream_ptr()),
          'svx_attention_multi')
    return [pr['out'] for pr in problems]


def attention(q, k, v, slots, heads, queries, keys, *, q_row_stride, kv_slot_stride, kv_head_stride, kv_row_stride,
              lengths=None, out=None, plan=None):
    """Non-causal head_dim-96 attention over per-slot key lengths; out [slots*queries, heads*96] bf16.
    `plan`: an `attention_plan` result (device plan, CTA count) or None."""
    if out is None:
        out = torch.empty((slots * queries, heads * 96), device=q.device, dtype=torch.bfloat16)
    raw = _lib.raw_ptr
    table, ctas = plan if plan is not None else (None, 0)
    check(_lib.load().svx_attention(raw(q), q_row_stride, raw(k), raw(v), kv_slot_stride, kv_head_stride,
                                    kv_row_stride, ptr(lengths), slots, heads, queries, keys, ptr(out), ptr(table),
                                    ctas, stream_ptr()),
          'svx_attention')
    return out


# ------------------------------------------------------------------------- rotary positions and the paged cache

_ROW_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_F32_MAX = torch.finfo(torch.float32).max
_POSITION_DTYPES = {torch.int32: _lib.I32, torch.int64: _lib.I64, torch.float32: _lib.F32}


_INT_MAX = 2 ** 31 - 1   # the library's sizes; ctypes cuts larger ones without a word


def _need(ok, text):
    if not ok:
        raise ValueError(text)


# The wrappers below are called once or twice a layer for a handful of tokens, where the time of a call is the host's: they
# read each attribute once, build their messages only when they raise, and pass plain addresses.

def _launch_on(index, function, *args):
    """function(*args, stream) on the current stream of CUDA device `index`, with that device current."""
    if index == torch.cuda.current_device():
        return function(*args, _raw_stream(index))
    with torch.cuda.device(index):
        return function(*args, _raw_stream(index))


def _raw_stream(index):
    return torch.cuda.current_stream(index).cuda_stream


_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', _raw_stream)


def _index_of(first, *others):
    """The one CUDA device of the tensors (None entries apart)."""
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            index = -1
    if index < 0:
        raise ValueError('operands must be on one CUDA device')
    return index


def _rows(name, t, tokens, heads, dim, dtype):
    """(token stride, head stride) of a [tokens, heads, dim] operand with contiguous rows."""
    shape = t.shape
    if len(shape) != 3:
        raise ValueError(f'{name} must be [tokens, heads, dim]')
    if tokens > _INT_MAX or heads > _INT_MAX:
        raise ValueError(f'{name} has sizes past 32 bits: {tuple(shape)}')
    if shape[0] != tokens or shape[1] != heads or shape[2] != dim:
        raise ValueError(f'{name} is {tuple(shape)}, expected {(tokens, heads, dim)}')
    if t.dtype != dtype:
        raise ValueError(f'{name} must be {dtype}, got {t.dtype}')
    strides = t.stride()
    if strides[2] != 1 and dim != 1:
        raise ValueError(f'{name} must have contiguous rows (stride 1 in dim)')
    return strides[0], strides[1]


def _rotary(inv_freq, positions, tokens, dim, layout, scale):
    if inv_freq.dtype != torch.float64 or inv_freq.ndim != 1 or not inv_freq.is_contiguous():
        raise ValueError('inv_freq must be a contiguous float64 vector, one entry per pair')
    pairs = inv_freq.numel()
    if not 0 < 2 * pairs <= dim:
        raise ValueError(f'{pairs} pairs do not fit heads of {dim}')
    if layout not in _lib.ROPE_LAYOUTS:
        raise ValueError(f'layout must be one of {sorted(_lib.ROPE_LAYOUTS)}')
    scale = float(scale)
    if not abs(scale) <= _F32_MAX:
        raise ValueError('the rotary scale must be finite in 32 bits')
    if positions is None:
        return _lib.Rotary(inv_freq.data_ptr(), 2 * pairs, _lib.ROPE_LAYOUTS[layout], 1, scale, None, _lib.I64)
    shape = positions.shape
    if positions.dtype not in _POSITION_DTYPES:
        raise ValueError('positions must be int32, int64 or float32')
    if len(shape) not in (1, 2) or shape[0] != tokens or not positions.is_contiguous():
        raise ValueError(f'positions must be a contiguous [{tokens}] or [{tokens}, axes] tensor')
    axes = shape[1] if len(shape) == 2 else 1
    if axes < 1 or pairs % axes:
        raise ValueError(f'{axes} axes do not share {pairs} pairs evenly')
    return _lib.Rotary(inv_freq.data_ptr(), 2 * pairs, _lib.ROPE_LAYOUTS[layout], axes, scale, positions.data_ptr(),
                       _POSITION_DTYPES[positions.dtype])


def rope_frequencies(rot, base=10000.0, *, axes=1, scaling=None, factor=1.0, original=8192, device='cuda'):
    """(inv_freq [rot / 2] float64, scale) of `rope` and `paged_append`: base^(-2j / width) with width = rot / axes,
    repeated for every axis. `scaling` stretches the positions a model was trained on (`original` of them) by `factor`:
    'linear' divides every frequency by it; 'base' enlarges the base so that the slowest pair is divided by it and the
    fastest keeps its angle; 'by_parts' keeps the pairs that turn at least 32 times within `original` positions, divides
    those that turn at most once, blends between, and gives scale = 0.1 ln(factor) + 1. Otherwise scale is 1."""
    _need(rot > 0 and axes > 0 and rot % (2 * axes) == 0, f'rot ({rot}) must be a positive multiple of 2 x {axes} axes')
    _need(scaling in (None, 'linear', 'base', 'by_parts'), f'unknown scaling {scaling!r}')
    _need(base > 0 and factor >= 1 and original > 0, 'base and original must be positive, factor at least 1')
    width, scale = rot // axes, 1.0
    if scaling == 'base':
        _need(width > 2, "scaling 'base' needs more than one pair an axis")
        base = base * factor ** (width / (width - 2))
    freq = float(base) ** (-np.arange(0, width, 2, dtype=np.float64) / width)
    if scaling == 'linear':
        freq = freq / factor
    elif scaling == 'by_parts':
        keep = np.clip((original * freq / (2 * math.pi) - 1) / 31, 0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
        scale = 0.1 * math.log(factor) + 1
    return torch.from_numpy(np.tile(freq, axes)).to(device), scale


class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, inv_freq, layout, scale, inverse):
        ctx.save_for_backward(positions, inv_freq)
        ctx.args = layout, scale, inverse
        return rope(x, positions, inv_freq, layout=layout, scale=scale, inverse=inverse)

    @staticmethod
    def backward(ctx, grad):
        layout, scale, inverse = ctx.args
        grad = grad if grad.stride(-1) == 1 else grad.contiguous()   # one broadcast over the values of a head
        return rope(grad, *ctx.saved_tensors, layout=layout, scale=scale, inverse=not inverse), *[None] * 5


def rope(x, positions, inv_freq, *, layout='interleaved', scale=1.0, inverse=False, out=None):
    """Rotary positions: the first 2 * len(inv_freq) values of each head of x [tokens, heads, dim] (fp32, bf16, fp16;
    token and head strides free) turned by positions * inv_freq and multiplied by scale, the others copied.

    positions: [tokens], or [tokens, axes] with the pairs split evenly among the axes (int32, int64 or float32). inv_freq:
    float64, from `rope_frequencies`. Angles are formed in float64: an angle a is off by up to 2^-51 |a|. Pairs are (2j, 2j + 1) ('interleaved') or (j, j + rot / 2) ('half'). inverse: the
    transposed rotation, the gradient's way back; x that requires grad takes it by itself (positions and inv_freq have no
    gradient, x no forward-mode derivative: refused). out: a [tokens, heads, dim]
    tensor of x's type, x itself or one that does not overlap it."""
    if x.ndim != 3:
        raise ValueError('x must be [tokens, heads, dim]')
    tokens, heads, dim = x.shape
    dtype = x.dtype
    if dtype not in _ROW_DTYPES:
        raise ValueError(f'x must be fp32, bf16 or fp16, got {dtype}')
    if heads < 1 or dim < 1:
        raise ValueError('x has no heads or values')
    if positions is None:
        raise ValueError('rope needs positions')
    strides = _rows('x', x, tokens, heads, dim, dtype)
    rotary = _rotary(inv_freq, positions, tokens, dim, layout, scale)
    _constant('rope has no gradient for positions, inv_freq or out', positions, inv_freq, out)
    if _forward_mode() and _has_tangent(x):
        raise ValueError('rope has no forward-mode derivative; rotate the tangent by a call of its own')
    if x.requires_grad and torch.is_grad_enabled():
        if out is not None:
            raise ValueError('out is not available for x that requires grad')
        return _Rope.apply(x, positions, inv_freq, layout, scale, inverse)
    given = out
    if out is None:
        index = _index_of(x, positions, inv_freq)
        out = x.new_empty((tokens, heads, dim))
        out_strides = heads * dim, dim
    else:
        out_strides = _rows('out', out, tokens, heads, dim, dtype)
        if (out_strides[0] == 0 and tokens > 1) or (out_strides[1] == 0 and heads > 1):
            raise ValueError('out must not repeat memory')
        index = _index_of(x, positions, inv_freq, out)
    status = _launch_on(index, _lib.load().svx_rope, x.data_ptr(), _ROW_DTYPES[dtype], *strides, out.data_ptr(),
                        *out_strides, tokens, heads, dim, ctypes.byref(rotary), bool(inverse))
    if status:
        check(status, 'svx_rope')
    if given is not None:
        increment_version(given)
    return out


def _forward_mode():
    """Whether tensors may carry forward-mode tangents at present."""
    return getattr(forward_ad, '_current_level', 0) >= 0


def _has_tangent(t):
    return forward_ad.unpack_dual(t).tangent is not None


def _constant(what, *tensors):
    """Refuse tensors whose derivative would be lost: those that require grad, or carry a forward-mode tangent."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(what)
    if _forward_mode():
        for t in tensors:
            if t is not None and _has_tangent(t):
                raise ValueError(what)


def _written(*tensors):
    """Tell autograd that these were written, so that a backward pass that saved one of them says so."""
    increment_version([t for t in tensors if t is not None])


def _paged_cache(k_pages, v_pages, table, lengths, offsets, status):
    shape, dtype = k_pages.shape, k_pages.dtype
    if len(shape) != 4 or shape != v_pages.shape or dtype != v_pages.dtype:
        raise ValueError('k_pages and v_pages must be [pages, kv_heads, page, dim] pools of one shape and type')
    if dtype != torch.bfloat16 and dtype != torch.float16:
        raise ValueError(f'the cache must be bf16 or fp16, got {dtype}')
    pages, heads, page, dim = shape
    if not (0 < pages <= _INT_MAX and 0 < heads <= 1024):
        raise ValueError(f'the pools need pages and 1 to 1024 heads, got {tuple(shape)}')
    if page not in (16, 32, 64, 128, 256, 512, 1024):
        raise ValueError(f'a page must hold 16, 32, .. 1024 keys, got {page}')
    shape = table.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError('table must be [sequences, pages of a sequence]')
    sequences, width = shape
    if sequences > 1 << 20 or width * page > 1 << 30:
        raise ValueError(f'table {tuple(shape)} is past 2^20 sequences or 2^30 keys a sequence')
    if lengths.ndim != 1 or len(lengths) != sequences or offsets.ndim != 1 or len(offsets) != sequences + 1:
        raise ValueError(f'lengths must be [{sequences}] and offsets [{sequences + 1}]')
    if not table.dtype == lengths.dtype == offsets.dtype == torch.int32:
        raise ValueError('table, lengths and offsets must be int32')
    if not (k_pages.is_contiguous() and v_pages.is_contiguous() and table.is_contiguous() and lengths.is_contiguous()
            and offsets.is_contiguous()):
        raise ValueError('the pools, table, lengths and offsets must be contiguous')
    if status is not None:
        if tuple(status.shape) != (sequences,) or status.dtype != torch.int32 or not status.is_contiguous():
            raise ValueError(f'status must be a contiguous int32 [{sequences}] tensor')
        status = status.data_ptr()
    return _lib.PagedCache(k_pages.data_ptr(), v_pages.data_ptr(), _ROW_DTYPES[dtype], pages, heads, page, dim,
                           sequences, width, table.data_ptr(), lengths.data_ptr(), offsets.data_ptr(), status)


_CACHE_GRAD = 'the paged cache takes no part in autograd: detach its operands or call under torch.no_grad()'


def paged_append(k, v, k_pages, v_pages, table, lengths, offsets, *, inv_freq=None, positions=None,
                 layout='interleaved', rope_scale=1.0, q=None, q_out=None, status=None):
    """Store new keys and values [tokens, kv_heads, dim] in a paged cache, the keys rotated on the way.

    k_pages, v_pages: pools [pages, kv_heads, page, dim] (bf16 or fp16; a page holds 16, 32, .. 1024 keys), written in
    place. table [sequences, n] int32: page ids in order. Sequence s owns the new rows offsets[s] .. offsets[s + 1] - 1 and
    has lengths[s] keys with them (int32, read on the device only). Rows outside of every sequence are left alone.
    inv_freq, layout, rope_scale and positions as in `rope`; without positions a key's place in the cache is its
    position. q [tokens, q_heads, dim] (optional) is rotated in the same launch and returned (into q_out where given:
    contiguous). A key whose place lies outside the table, or whose page id lies outside the pool, is not stored; status
    [sequences] int32 (optional) gets STATUS_BAD_PAGE for its sequence. Two tokens given the same place race."""
    cache = _paged_cache(k_pages, v_pages, table, lengths, offsets, status)
    dtype, heads, dim, tokens = k_pages.dtype, cache.kv_heads, cache.dim, len(k)
    k_strides = _rows('k', k, tokens, heads, dim, dtype)
    v_strides = _rows('v', v, tokens, heads, dim, dtype)
    _constant(_CACHE_GRAD, k, v, k_pages, v_pages, inv_freq, positions, q, q_out)
    rotary = None
    if inv_freq is not None:
        rotary = ctypes.byref(_rotary(inv_freq, positions, tokens, dim, layout, rope_scale))
    elif q is not None or positions is not None:
        raise ValueError('q and positions need inv_freq')
    index = _index_of(k_pages, v_pages, table, lengths, offsets, k, v, inv_freq, positions, q, q_out, status)
    if q is None:
        if q_out is not None:
            raise ValueError('q_out needs q')
        queries = None, 0, 0, 0, None
    else:
        q_heads = q.shape[1] if q.ndim == 3 else 0
        q_strides = _rows('q', q, tokens, q_heads, dim, dtype)
        if not 0 < q_heads <= 4096:
            raise ValueError('q must have 1 to 4096 heads')
        if q_out is None:
            q_out = q.new_empty((tokens, q_heads, dim))
        else:
            _rows('q_out', q_out, tokens, q_heads, dim, dtype)
            if not q_out.is_contiguous():
                raise ValueError('q_out must be contiguous')
        queries = q.data_ptr(), *q_strides, q_heads, q_out.data_ptr()
    code = _launch_on(index, _lib.load().svx_paged_append, ctypes.byref(cache), k.data_ptr(), *k_strides, v.data_ptr(),
                      *v_strides, tokens, rotary, *queries)
    if code:
        check(code, 'svx_paged_append')
    _written(k_pages, v_pages, q_out, status)
    return q_out


def paged_attention_workspace(tokens, sequences, q_heads, kv_heads, dim, device, max_query=0):
    """Scratch of one `paged_attention` call of these sizes (for one call at a time)."""
    with torch.cuda.device(device):
        size = _lib.load().svx_paged_attention_workspace_bytes(tokens, sequences, q_heads, kv_heads, dim,
                                                               int(max_query))
    _need(size > 0, f'paged_attention does not take {q_heads} query heads over {kv_heads} of dim {dim}')
    return torch.empty(size, dtype=torch.uint8, device=device)


def paged_attention(q, k_pages, v_pages, table, lengths, offsets, *, causal=True, scale=None, out=None, lse=None,
                    max_query=None, workspace=None, status=None):
    """Attention of new tokens over the keys of their sequences in a paged cache (`paged_append`'s arguments).

    q [tokens, q_heads, dim] (token and head strides multiples of 8), dim 64, 96 or 128, query head h reading kv head
    h // (q_heads / kv_heads). Sequence s's rows are its last tokens: causal, row i of n sees lengths[s] - n + i + 1 keys;
    else all lengths[s]. A row that sees none gives 0; hidden keys weigh 0, so an infinite or NaN value among them is NaN in the
    row. scale: 1 / sqrt(dim) unless given. Returns out [tokens, q_heads,
    dim] (contiguous, not overlapping q); rows outside of every sequence are left as they were. lse [tokens, q_heads]
    float32 (optional): the natural logarithm of the row's sum of exponentials, -inf for a row without keys.
    max_query: the most new tokens of a sequence in the batch, where the caller knows it; it picks the kernel's form, never
    the result's meaning. Without it the mean decides, and a long chunk among single tokens may take the form for few rows
    (2000 tokens and 199 single ones, 8 heads of 128: 382 us against 235). workspace: from `paged_attention_workspace`, not shared by calls that may overlap; allocated
    here unless given. status [sequences] int32 (optional) gets STATUS_BAD_PAGE where a page id lies outside the pool (read
    as zeros) or a length outside the table (clamped)."""
    cache = _paged_cache(k_pages, v_pages, table, lengths, offsets, status)
    dim, kv_heads = cache.dim, cache.kv_heads
    tokens, heads = q.shape[:2] if q.ndim == 3 else (0, 0)
    strides = _rows('q', q, tokens, heads, dim, k_pages.dtype)
    if dim not in (64, 96, 128):
        raise ValueError(f'dim must be 64, 96 or 128, got {dim}')
    if heads < 1 or heads % kv_heads:
        raise ValueError(f'{heads} query heads are not a multiple of the {kv_heads} heads of the cache')
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0 < scale <= 1e30:
        raise ValueError('scale must be positive and finite')
    if max_query is None:
        max_query = 0
    elif max_query < 0:
        raise ValueError('max_query must not be negative')
    _constant(_CACHE_GRAD, q, k_pages, v_pages, out, lse)
    index = _index_of(q, k_pages, v_pages, table, lengths, offsets, out, lse, workspace, status)
    given = out
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _rows('out', out, tokens, heads, dim, q.dtype)
        if not out.is_contiguous():
            raise ValueError('out must be contiguous')
    if lse is not None and (lse.shape != (tokens, heads) or lse.dtype != torch.float32 or not lse.is_contiguous()):
        raise ValueError(f'lse must be a contiguous float32 [{tokens}, {heads}] tensor')
    lib, max_query = _lib.load(), min(int(max_query), tokens)
    sizes = tokens, cache.sequences, heads, kv_heads, dim, max_query
    if index == torch.cuda.current_device():
        size = lib.svx_paged_attention_workspace_bytes(*sizes)
    else:
        with torch.cuda.device(index):
            size = lib.svx_paged_attention_workspace_bytes(*sizes)
    if workspace is None:
        workspace = q.new_empty((size,), dtype=torch.uint8)
    elif workspace.dtype != torch.uint8 or workspace.numel() < size or not workspace.is_contiguous():
        raise ValueError(f'workspace must be a contiguous uint8 tensor of at least {size} bytes')
    code = _launch_on(index, lib.svx_paged_attention, ctypes.byref(cache), q.data_ptr(), *strides, tokens, heads, bool(causal),
                      scale, out.data_ptr(), None if lse is None else lse.data_ptr(), max_query, workspace.data_ptr())
    if code:
        check(code, 'svx_paged_attention')
    if given is not None or lse is not None or status is not None:
        _written(given, lse, status)
    return out

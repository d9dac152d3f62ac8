"""Torch-tensor wrappers over the libsvx entry points (device tensors in, device tensors out, current stream).

Each wrapper validates dtypes/shapes on the host and calls exactly one C-ABI function; there is no CPU path.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

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
_POSITION_DTYPES = {torch.int32: _lib.I32, torch.int64: _lib.I64, torch.float32: _lib.F32}


def _need(ok, text):
    if not ok:
        raise ValueError(text)


def _device_of(*tensors):
    """The one CUDA device of the tensors (None entries apart)."""
    devices = {t.device for t in tensors if t is not None}
    _need(len(devices) == 1 and next(iter(devices)).type == 'cuda', 'operands must be on one CUDA device')
    return devices.pop()


def _rows(name, t, tokens=None, heads=None, dim=None, dtype=None):
    """A [tokens, heads, dim] operand with contiguous rows; the token and head strides are free."""
    _need(t.ndim == 3, f'{name} must be [tokens, heads, dim]')
    for size, want, what in zip(t.shape, (tokens, heads, dim), ('tokens', 'heads', 'dim')):
        _need(want is None or size == want, f'{name} has {size} {what}, expected {want}')
    _need(dtype is None or t.dtype == dtype, f'{name} must be {dtype}')
    _need(t.stride(2) == 1 or t.shape[2] == 1, f'{name} must have contiguous rows (stride 1 in dim)')


def _rotary(inv_freq, positions, tokens, dim, layout, scale):
    _need(inv_freq.dtype == torch.float64 and inv_freq.ndim == 1 and inv_freq.is_contiguous(),
          'inv_freq must be a contiguous float64 vector, one entry per pair')
    pairs = inv_freq.numel()
    _need(0 < 2 * pairs <= dim, f'{pairs} pairs do not fit heads of {dim}')
    _need(layout in _lib.ROPE_LAYOUTS, f'layout must be one of {sorted(_lib.ROPE_LAYOUTS)}')
    axes, kind = 1, _lib.I64
    if positions is not None:
        _need(positions.dtype in _POSITION_DTYPES, 'positions must be int32, int64 or float32')
        _need(positions.ndim in (1, 2) and positions.shape[0] == tokens and positions.is_contiguous(),
              f'positions must be a contiguous [{tokens}] or [{tokens}, axes] tensor')
        axes = positions.shape[1] if positions.ndim == 2 else 1
        kind = _POSITION_DTYPES[positions.dtype]
        _need(axes > 0 and pairs % axes == 0, f'{axes} axes do not share {pairs} pairs evenly')
    _need(math.isfinite(scale), 'the rotary scale must be finite')
    return _lib.Rotary(inv_freq.data_ptr(), 2 * pairs, _lib.ROPE_LAYOUTS[layout], axes, float(scale),
                       ptr(positions), kind)


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
        grad = grad if grad.stride(-1) == 1 else grad.contiguous()
        return rope(grad, *ctx.saved_tensors, layout=layout, scale=scale, inverse=not inverse), *[None] * 5


def rope(x, positions, inv_freq, *, layout='interleaved', scale=1.0, inverse=False, out=None):
    """Rotary positions: the first 2 * len(inv_freq) values of each head of x [tokens, heads, dim] (fp32, bf16, fp16;
    token and head strides free) turned by positions * inv_freq and multiplied by scale, the others copied.

    positions: [tokens], or [tokens, axes] with the pairs split evenly among the axes (int32, int64 or float32). inv_freq:
    float64, from `rope_frequencies`. Pairs are (2j, 2j + 1) ('interleaved') or (j, j + rot / 2) ('half'). inverse: the
    transposed rotation, the gradient's way back; x that requires grad takes it by itself. out: a [tokens, heads, dim]
    tensor of x's type, x itself or one that does not overlap it."""
    _rows('x', x)
    _need(x.dtype in _ROW_DTYPES, f'x must be fp32, bf16 or fp16, got {x.dtype}')
    tokens, heads, dim = x.shape
    _need(heads > 0 and dim > 0, 'x has no heads or values')
    _need(positions is not None, 'rope needs positions')
    rotary = _rotary(inv_freq, positions, tokens, dim, layout, scale)
    if torch.is_grad_enabled() and x.requires_grad:
        _need(out is None, 'out is not available for x that requires grad')
        return _Rope.apply(x, positions, inv_freq, layout, scale, inverse)
    if out is None:
        out = torch.empty((tokens, heads, dim), device=x.device, dtype=x.dtype)
    else:
        _rows('out', out, tokens, heads, dim, x.dtype)
        _need(all(n == 1 or s != 0 for n, s in zip(out.shape, out.stride())), 'out must not repeat memory')
    with torch.cuda.device(_device_of(x, positions, inv_freq, out)):
        check(_lib.load().svx_rope(_lib.raw_ptr(x), _ROW_DTYPES[x.dtype], x.stride(0), x.stride(1), _lib.raw_ptr(out),
                                   out.stride(0), out.stride(1), tokens, heads, dim, ctypes.byref(rotary), int(inverse),
                                   stream_ptr()), 'svx_rope')
    return out


def _paged_cache(k_pages, v_pages, table, lengths, offsets, status):
    _need(k_pages.ndim == 4 and k_pages.shape == v_pages.shape and k_pages.dtype == v_pages.dtype,
          'k_pages and v_pages must be [pages, kv_heads, page, dim] pools of one shape and type')
    _need(k_pages.dtype in (torch.bfloat16, torch.float16), f'the cache must be bf16 or fp16, got {k_pages.dtype}')
    pages, heads, page, dim = k_pages.shape
    _need(page in (16, 32, 64, 128, 256, 512, 1024), f'a page must hold 16, 32, .. 1024 keys, got {page}')
    for name, t in (('table', table), ('lengths', lengths), ('offsets', offsets), ('status', status)):
        _need(t is None or t.dtype == torch.int32, f'{name} must be int32')
    _need(table.ndim == 2 and table.shape[1] > 0, 'table must be [sequences, pages of a sequence]')
    sequences = table.shape[0]
    _need(tuple(lengths.shape) == (sequences,), f'lengths must be [{sequences}]')
    _need(tuple(offsets.shape) == (sequences + 1,), f'offsets must be [{sequences + 1}]')
    _need(status is None or tuple(status.shape) == (sequences,), f'status must be [{sequences}]')
    return _lib.PagedCache(ptr(k_pages), ptr(v_pages), _ROW_DTYPES[k_pages.dtype], pages, heads, page, dim, sequences,
                           table.shape[1], ptr(table), ptr(lengths), ptr(offsets), ptr(status))


def _no_grad(*tensors):
    _need(not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)),
          'the paged cache takes no part in autograd: call under torch.no_grad()')


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
    _rows('k', k, None, cache.kv_heads, cache.dim, k_pages.dtype)
    _rows('v', v, k.shape[0], cache.kv_heads, cache.dim, k_pages.dtype)
    tokens = k.shape[0]
    _need(inv_freq is not None or (q is None and positions is None), 'q and positions need inv_freq')
    _need(q is not None or q_out is None, 'q_out needs q')
    rotary = None if inv_freq is None else _rotary(inv_freq, positions, tokens, cache.dim, layout, rope_scale)
    if q is not None:
        _rows('q', q, tokens, None, cache.dim, k_pages.dtype)
        _need(0 < q.shape[1] <= 4096, 'q must have 1 to 4096 heads')
        if q_out is None:
            q_out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
        else:
            _rows('q_out', q_out, tokens, q.shape[1], cache.dim, q.dtype)
    _no_grad(k, v, k_pages, v_pages, q)
    strides = (0, 0, 0) if q is None else (q.stride(0), q.stride(1), q.shape[1])
    with torch.cuda.device(_device_of(k, v, k_pages, v_pages, table, lengths, offsets, inv_freq, positions, q, q_out,
                                      status)):
        check(_lib.load().svx_paged_append(ctypes.byref(cache), _lib.raw_ptr(k), k.stride(0), k.stride(1),
                                           _lib.raw_ptr(v), v.stride(0), v.stride(1), tokens,
                                           None if rotary is None else ctypes.byref(rotary), _lib.raw_ptr(q), *strides,
                                           ptr(q_out), stream_ptr()), 'svx_paged_append')
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
    else all lengths[s]. A row that sees none gives 0. scale: 1 / sqrt(dim) unless given. Returns out [tokens, q_heads,
    dim] (contiguous, not overlapping q); rows outside of every sequence are left as they were. lse [tokens, q_heads]
    float32 (optional): the natural logarithm of the row's sum of exponentials, -inf for a row without keys.
    max_query: the most new tokens of a sequence in the batch, where the caller knows it; it picks the kernel's form, never
    the result's meaning. workspace: from `paged_attention_workspace`, not shared by calls that may overlap; allocated
    here unless given. status [sequences] int32 (optional) gets STATUS_BAD_PAGE where a page id lies outside the pool (read
    as zeros) or a length outside the table (clamped)."""
    cache = _paged_cache(k_pages, v_pages, table, lengths, offsets, status)
    _rows('q', q, None, None, cache.dim, k_pages.dtype)
    tokens, heads = q.shape[:2]
    _need(cache.dim in (64, 96, 128), f'dim must be 64, 96 or 128, got {cache.dim}')
    _need(heads > 0 and heads % cache.kv_heads == 0,
          f'{heads} query heads are not a multiple of the {cache.kv_heads} heads of the cache')
    scale = cache.dim ** -0.5 if scale is None else float(scale)
    _need(0 < scale <= 1e30, 'scale must be positive and finite')
    if out is None:
        out = torch.empty((tokens, heads, cache.dim), device=q.device, dtype=q.dtype)
    else:
        _rows('out', out, tokens, heads, cache.dim, q.dtype)
    _need(lse is None or (tuple(lse.shape) == (tokens, heads) and lse.dtype == torch.float32),
          f'lse must be a float32 [{tokens}, {heads}] tensor')
    _need(max_query is None or max_query >= 0, 'max_query must not be negative')
    _no_grad(q, k_pages, v_pages)
    limit = 0 if max_query is None else min(int(max_query), 2 ** 31 - 1)
    device = _device_of(q, k_pages, v_pages, table, lengths, offsets, out, lse, workspace, status)
    with torch.cuda.device(device):
        lib = _lib.load()
        size = lib.svx_paged_attention_workspace_bytes(tokens, cache.sequences, heads, cache.kv_heads, cache.dim, limit)
        if workspace is None:
            workspace = torch.empty(size, dtype=torch.uint8, device=device)
        _need(workspace.dtype == torch.uint8 and workspace.numel() >= size,
              f'workspace must be a uint8 tensor of at least {size} bytes')
        check(lib.svx_paged_attention(ctypes.byref(cache), _lib.raw_ptr(q), q.stride(0), q.stride(1), tokens, heads,
                                      int(causal), scale, ptr(out), ptr(lse), limit, ptr(workspace), stream_ptr()),
              'svx_paged_attention')
    return out

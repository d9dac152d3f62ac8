"""Cases of the rotary and paged-cache operators: rope, paged_append and paged_attention.

With `own` false, `run` computes a case with elementary torch operations (32 bits, angles in 64); with `own` true it
calls the operators of `streamvoxel_b200.ops`. `exact` gives the definition's result in 64 bits.

A paged cache is two pools [pages][kv heads][page][dim] (keys, values) and a table [sequences][pages per sequence] of
page ids. `offsets` [sequences + 1] bounds each sequence's rows among the new tokens, `lengths` [sequences] counts each
sequence's keys, the new ones among them.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def listed():
    return [
        # the rotation of a few tokens' queries between two other launches: latency
        dict(name='rope-token', op='rope', tokens=33, heads=8, dim=96, rot=96, axes=3, layout='interleaved',
             scaling='none', far=256, dtype='bf16', inverse=False),
        # queries and keys (8 + 8 heads of 96) of 8 slots of 1024 patches at their three-axis positions
        dict(name='rope-patches', op='rope', tokens=8192, heads=16, dim=96, rot=96, axes=3, layout='interleaved',
             scaling='none', far=256, dtype='bf16', inverse=False),
        # gradient of the rotation over long text: half of each head, positions to a million, scaled by parts
        dict(name='rope-far-back', op='rope', tokens=16384, heads=32, dim=128, rot=64, axes=1, layout='half',
             scaling='by_parts', far=1000000, dtype='fp16', inverse=True),
        # one decoding step of 64 sequences: queries rotated, keys rotated and stored, values stored
        dict(name='append-token', op='append', sequences=64, new_low=1, new_high=1, low=17, high=4096, kv_heads=8,
             group=4, dim=128, page=16, rot=128, axes=1, layout='half', with_q=True, dtype='bf16', spread=1),
        # the condition keys of 8 windows of unequal length, stored whole at their three-axis positions
        dict(name='append-windows', op='append', sequences=8, new_low=2368, new_high=9536, low=0, high=0, kv_heads=8,
             group=1, dim=96, page=64, rot=96, axes=3, layout='interleaved', with_q=False, dtype='bf16', spread=2),
        # one new token of one conversation: latency, the keys split over the whole card
        dict(name='attn-token-single', op='attention', sequences=1, new_low=1, new_high=1, low=4001, high=4001,
             kv_heads=8, group=4, dim=128, page=16, causal=True, lse=False, dtype='bf16', spread=3),
        # a serving batch of 128 sequences of very unequal length, one token each
        dict(name='attn-token-batch', op='attention', sequences=128, new_low=1, new_high=1, low=40, high=16384,
             kv_heads=8, group=4, dim=128, page=16, causal=True, lse=False, dtype='bf16', spread=4),
        # few sequences of far context, every query head with keys of its own
        dict(name='attn-token-far', op='attention', sequences=3, new_low=1, new_high=1, low=90000, high=131072,
             kv_heads=16, group=1, dim=64, page=128, causal=True, lse=True, dtype='fp16', spread=5),
        # five drafted tokens a sequence, checked at once
        dict(name='attn-verify', op='attention', sequences=32, new_low=5, new_high=5, low=300, high=12000, kv_heads=4,
             group=8, dim=128, page=32, causal=True, lse=False, dtype='bf16', spread=6),
        # cross-attention of 8 slots of 1024 patches to their windows' condition keys
        dict(name='attn-windows', op='attention', sequences=8, new_low=1024, new_high=1024, low=2368, high=9536,
             kv_heads=8, group=1, dim=96, page=64, causal=False, lse=False, dtype='bf16', spread=7),
        # single tokens and prompt chunks in one batch
        dict(name='attn-mixed', op='attention', sequences=24, new_low=1, new_high=700, low=700, high=6000, kv_heads=4,
             group=6, dim=64, page=16, causal=True, lse=True, dtype='fp16', spread=8),
        # long prompts taken in chunks of about 2,000 tokens over a far context
        dict(name='attn-chunk', op='attention', sequences=4, new_low=1500, new_high=2048, low=9000, high=32768,
             kv_heads=8, group=4, dim=128, page=64, causal=True, lse=False, dtype='bf16', spread=9),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(['rope', 'append', 'attention', 'attention', 'attention'])
    dim = rng.choice([64, 96, 128])
    layout = rng.choice(['interleaved', 'half'])
    axes = rng.choice([1, 1, 2, 3]) if dim == 96 else rng.choice([1, 1, 2])
    if op == 'rope':
        case = dict(op=op, tokens=_log_int(rng, 1, 16384), heads=rng.randint(1, 40), dim=dim,
                    rot=dim if rng.random() < 0.6 else dim // 2, axes=axes, layout=layout,
                    scaling=rng.choice(['none', 'linear', 'base', 'by_parts']) if axes == 1 else 'none',
                    far=_log_int(rng, 64, 1000000), dtype=rng.choice(['bf16', 'fp16', 'fp32']),
                    inverse=rng.random() < 0.4)
        room = 16384 * 32 * 128 * 2
        case['tokens'] = min(case['tokens'], room // (case['heads'] * dim * DTYPES[case['dtype']].itemsize))
        return case
    case = dict(op=op, sequences=_log_int(rng, 1, 200), kv_heads=rng.choice([1, 2, 4, 8, 16]),
                group=rng.choice([1, 1, 2, 3, 4, 4, 5, 6, 7, 8, 16]), dim=dim, page=rng.choice([16, 32, 64, 128, 256]),
                dtype=rng.choice(['bf16', 'bf16', 'fp16']), spread=rng.randrange(10 ** 6))
    if op == 'append':
        high = _log_int(rng, 1, 9536)
        case.update(new_low=_log_int(rng, 1, high), new_high=high, low=0, high=_log_int(rng, 1, 8192), rot=dim,
                    axes=axes, layout=layout, with_q=rng.random() < 0.5)
    else:
        kind = rng.choice(['token', 'token', 'few', 'chunk', 'mixed'])
        new_low, new_high = {'token': (1, 1), 'few': (1, rng.randint(2, 16)), 'mixed': (1, _log_int(rng, 17, 1024)),
                             'chunk': (_log_int(rng, 16, 1024), 2048)}[kind]
        high = _log_int(rng, 16, 131072)
        case.update(new_low=new_low, new_high=new_high, low=_log_int(rng, 1, high), high=high,
                    causal=rng.random() < 0.75, lse=rng.random() < 0.4)
    largest = [work(c) for c in listed()]
    most_bytes = max(w['bytes'] for w in largest) if op == 'attention' else 1.2e8
    most_flops = max(w['flops'] for w in largest)
    while work(case)['bytes'] > most_bytes or work(case)['flops'] > most_flops:
        if case['sequences'] > 1:
            case['sequences'] = case['sequences'] * 2 // 3
        else:
            for name in ('new_low', 'new_high', 'low', 'high'):
                case[name] = max(min(1, case[name]), case[name] * 2 // 3)
    return case


def _sequences(case):
    """(new tokens, keys with the new ones) of every sequence: spread over the logarithm, the same for every seed."""
    rng = np.random.RandomState(case['spread'])
    n = case['sequences']

    def between(low, high):
        if low == high:
            return np.full(n, low, np.int64)
        v = np.exp(rng.uniform(math.log(max(low, 1)), math.log(high), n))
        return np.clip(np.rint(v).astype(np.int64), low, high)
    new, old = between(case['new_low'], case['new_high']), between(case['low'], case['high'])
    if case['op'] == 'append':
        return new, old + new
    return new, np.maximum(old, new) if case['causal'] else old


def _frequencies(case):
    """Angle per position and pair, float64 [rot / 2], and the factor on the rotated part."""
    rot = case['rot']
    width = rot // case['axes']
    exponent = np.arange(0, width, 2, dtype=np.float64) / width
    scaling, factor, original, base = case.get('scaling', 'none'), 8.0, 8192, 10000.0
    scale = 1.0
    if scaling == 'base':
        base = base * factor ** (width / (width - 2))
    freq = base ** -exponent
    if scaling == 'linear':
        freq = freq / factor
    if scaling == 'by_parts':
        # pairs that turn over 32 times within the original length keep their angle, those under once are slowed
        turns = original * freq / (2 * math.pi)
        keep = np.clip((turns - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        freq = freq * keep + freq / factor * (1 - keep)
        scale = 0.1 * math.log(factor) + 1.0
    return np.tile(freq, case['axes']), scale


def _random(shape, dtype, g, gain=1.0):
    return (torch.randn(shape, generator=g, device='cuda', dtype=torch.float32) * gain).to(dtype) \
        if math.prod(shape) < 1 << 27 else \
        torch.empty(shape, device='cuda', dtype=dtype).normal_(0.0, gain, generator=g)


def _positions(tokens, axes, far, rng):
    if axes == 1:
        start = int(rng.integers(0, max(1, far - tokens) + 1))
        return torch.from_numpy((start + np.arange(tokens)).astype(np.int64)).cuda()
    # centres of patches on a grid: halves of whole numbers
    return torch.from_numpy((rng.integers(-far, far, (tokens, axes)) / 2).astype(np.float32)).cuda()


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    rng = np.random.default_rng(seed)
    dtype, dim = DTYPES[case['dtype']], case['dim']
    state = dict(case=case)
    if case['op'] != 'attention':
        freq, state['rope_scale'] = _frequencies(case)
        state['freq'] = torch.from_numpy(freq).cuda()
    if case['op'] == 'rope':
        state['x'] = _random((case['tokens'], case['heads'], dim), dtype, g)
        state['positions'] = _positions(case['tokens'], case['axes'], case['far'], rng)
        state['out'] = torch.empty_like(state['x'])
        return state
    new, keys = _sequences(case)
    page = case['page']
    per = [int(-(-k // page)) for k in keys]
    pages, width = sum(per) + 3, max(per)
    ids = rng.permutation(pages).astype(np.int32)
    table = np.zeros((len(per), max(1, width)), np.int32)
    at = 0
    for s, n in enumerate(per):
        table[s, :n] = ids[at:at + n]
        at += n
    state['table'] = torch.from_numpy(table).cuda()
    state['lengths'] = torch.from_numpy(keys.astype(np.int32)).cuda()
    state['offsets'] = torch.from_numpy(np.concatenate(([0], np.cumsum(new))).astype(np.int32)).cuda()
    # a program's scheduler knows these on the host too
    state['new'], state['keys'] = [int(v) for v in new], [int(v) for v in keys]
    tokens, heads = int(new.sum()), case['kv_heads'] * case['group']
    pool = (pages, case['kv_heads'], page, dim)
    if case['op'] == 'append':
        state['k'] = _random((tokens, case['kv_heads'], dim), dtype, g)
        state['v'] = _random((tokens, case['kv_heads'], dim), dtype, g)
        state['k_pages'], state['v_pages'] = torch.zeros(pool, device='cuda', dtype=dtype), \
            torch.zeros(pool, device='cuda', dtype=dtype)
        state['positions'] = None if case['axes'] == 1 else _positions(tokens, case['axes'], 512, rng)
        state['q'] = _random((tokens, heads, dim), dtype, g) if case['with_q'] else None
        return state
    # scores of standard deviation 1.5; the pools' rows past a sequence's length hold values of earlier use
    state['q'] = _random((tokens, heads, dim), dtype, g, 1.5)
    state['k_pages'] = _random(pool, dtype, g)
    state['v_pages'] = _random(pool, dtype, g)
    state['lse'] = torch.empty((tokens, heads), device='cuda', dtype=torch.float32) if case['lse'] else None
    return state


# ------------------------------------------------------------------------------------------------- plain forms


def _angles(positions, freq):
    """[tokens, rot / 2] float64: the pairs are split evenly among the axes of the positions."""
    p = positions.double()
    p = p[:, None] if p.ndim == 1 else p
    return p.repeat_interleave(freq.numel() // p.shape[1], 1) * freq


def _rotate(x, angle, scale, layout):
    """[tokens, heads, dim] in 32 bits, its first 2 * angle.shape[1] dims turned by the angles."""
    cos, sin = (angle.cos() * scale).float()[:, None], (angle.sin() * scale).float()[:, None]
    y = x.float()
    half = angle.shape[1]
    part = y[..., :2 * half]
    if layout == 'half':
        a, b = part[..., :half], part[..., half:]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((turned, y[..., 2 * half:]), -1)


def _plain_append(state):
    case = state['case']
    new = state['offsets'].diff()
    sequence = torch.repeat_interleave(torch.arange(len(new), device='cuda'), new, output_size=len(state['k']))
    row = torch.arange(len(state['k']), device='cuda') - state['offsets'][sequence]
    at = (state['lengths'] - new)[sequence] + row
    angle = _angles(at if state['positions'] is None else state['positions'], state['freq'])
    page = state['table'][sequence, at // case['page']].long()
    dtype = state['k'].dtype
    state['k_pages'][page, :, at % case['page']] = \
        _rotate(state['k'], angle, state['rope_scale'], case['layout']).to(dtype)
    state['v_pages'][page, :, at % case['page']] = state['v']
    out = dict(k_pages=state['k_pages'], v_pages=state['v_pages'])
    if state['q'] is not None:
        out['q'] = _rotate(state['q'], angle, state['rope_scale'], case['layout']).to(dtype)
    return out


def _plain_attention(state):
    case = state['case']
    heads, group, dim = case['kv_heads'], case['group'], case['dim']
    outs, sums = [], []
    for s, (q, keys) in enumerate(zip(state['q'].split(state['new']), state['keys'])):
        pages = state['table'][s, :-(-keys // case['page'])].long()
        k = state['k_pages'][pages].transpose(0, 1).reshape(heads, -1, dim)[:, :keys].float()
        v = state['v_pages'][pages].transpose(0, 1).reshape(heads, -1, dim)[:, :keys].float()
        rows = q.float().view(-1, heads, group, dim).permute(1, 2, 0, 3).reshape(heads, -1, dim)
        score = rows @ k.transpose(1, 2) * dim ** -0.5
        if case['causal']:
            last = keys - len(q) + torch.arange(len(q), device='cuda')
            hidden = torch.arange(keys, device='cuda') > last[:, None]
            score.view(heads, group, len(q), keys).masked_fill_(hidden, -math.inf)
        top = score.amax(-1, keepdim=True)
        weight = score.sub_(top).exp_()
        total = weight.sum(-1, keepdim=True)
        out = weight @ v / total
        outs.append(out.view(heads, group, len(q), dim).permute(2, 0, 1, 3).reshape(len(q), heads * group, dim))
        sums.append((top + total.log()).view(heads, group, len(q)).permute(2, 0, 1).reshape(len(q), heads * group))
    out = dict(out=torch.cat(outs).to(state['q'].dtype))
    if case['lse']:
        out['lse'] = torch.cat(sums)
    return out


def run(state):
    case = state['case']
    if own:
        from streamvoxel_b200 import ops
        if case['op'] == 'rope':
            return ops.rope(state['x'], state['positions'], state['freq'], layout=case['layout'],
                            scale=state['rope_scale'], inverse=case['inverse'], out=state['out'])
        if case['op'] == 'append':
            q = ops.paged_append(state['k'], state['v'], state['k_pages'], state['v_pages'], state['table'],
                                 state['lengths'], state['offsets'], inv_freq=state['freq'],
                                 positions=state['positions'], layout=case['layout'], rope_scale=state['rope_scale'],
                                 q=state['q'])
            out = dict(k_pages=state['k_pages'], v_pages=state['v_pages'])
            return out if q is None else dict(out, q=q)
        out = ops.paged_attention(state['q'], state['k_pages'], state['v_pages'], state['table'], state['lengths'],
                                  state['offsets'], causal=case['causal'], lse=state['lse'],
                                  max_query=max(state['new']))
        return dict(out=out) if state['lse'] is None else dict(out=out, lse=state['lse'])
    if case['op'] == 'rope':
        angle = _angles(state['positions'], state['freq'])
        return _rotate(state['x'], -angle if case['inverse'] else angle, state['rope_scale'],
                       case['layout']).to(state['x'].dtype)
    return _plain_append(state) if case['op'] == 'append' else _plain_attention(state)


def work(case):
    size = DTYPES[case['dtype']].itemsize
    if case['op'] == 'rope':
        values = case['tokens'] * case['heads'] * case['dim']
        position = 8 if case['axes'] == 1 else 4 * case['axes']
        return dict(bytes=2 * values * size + case['tokens'] * position, flops=6 * values * case['rot'] // case['dim'] // 2)
    new, keys = _sequences(case)
    tokens, heads, dim = int(new.sum()), case['kv_heads'], case['dim']
    table = int((-(-keys // case['page'])).sum()) * 4 + len(new) * 8
    if case['op'] == 'append':
        rotated = tokens * heads * dim * (1 + (case['group'] if case['with_q'] else 0))
        moved = rotated + tokens * heads * dim
        positions = 0 if case['axes'] == 1 else 4 * case['axes'] * tokens
        return dict(bytes=2 * moved * size + positions + table, flops=3 * rotated)
    pairs = new * keys - (new * (new - 1) // 2 if case['causal'] else 0)
    queries = tokens * heads * case['group']
    return dict(bytes=(2 * int(keys.sum()) * heads * dim + 2 * queries * dim) * size + table
                + (4 * queries if case['lse'] else 0),
                flops=4 * int(pairs.sum()) * heads * case['group'] * dim)


# --------------------------------------------------------------------------------------------- 64-bit results


def _turn64(x, position, freq, scale, layout, sign=1):
    """Rotation as a product of complex numbers: pair (a, b) is a + ib."""
    tokens, heads, dim = x.shape
    pairs = freq.numel()
    position = position.to(torch.float64).reshape(tokens, -1)
    angle = torch.cat([position[:, a:a + 1] * part for a, part in enumerate(freq.chunk(position.shape[1]))], 1)
    spin = torch.polar(torch.full_like(angle, scale), sign * angle)[:, None, :]
    z = x.double()
    y = z.clone()
    if layout == 'interleaved':
        first, second = slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)
    else:
        first, second = slice(0, pairs), slice(pairs, 2 * pairs)
    turned = torch.complex(z[..., first], z[..., second]) * spin
    y[..., first], y[..., second] = turned.real, turned.imag
    return y


def exact(case, seed):
    state = prepare(case, seed)
    if case['op'] == 'rope':
        return _turn64(state['x'], state['positions'], state['freq'], state['rope_scale'], case['layout'],
                       -1 if case['inverse'] else 1)
    if case['op'] == 'append':
        new, keys, page = state['new'], state['keys'], case['page']
        at = torch.cat([torch.arange(k - n, k) for n, k in zip(new, keys)]).cuda()
        position = at if state['positions'] is None else state['positions']
        out = {}
        turned = _turn64(state['k'], position, state['freq'], state['rope_scale'], case['layout'])
        for name, rows in (('k_pages', turned), ('v_pages', state['v'].double())):
            pool = state[name].double()
            begin = 0
            for s, n in enumerate(new):
                for p in range((keys[s] - n) // page, -(-keys[s] // page)):
                    low, high = max(p * page, keys[s] - n), min((p + 1) * page, keys[s])
                    part = rows[begin + low - (keys[s] - n):begin + high - (keys[s] - n)]
                    pool[int(state['table'][s, p]), :, low - p * page:high - p * page] = part.transpose(0, 1)
                begin += n
            out[name] = pool
        if state['q'] is not None:
            out['q'] = _turn64(state['q'], position, state['freq'], state['rope_scale'], case['layout'])
        return out
    if work(case)['flops'] > 2e13:
        return None
    out = torch.zeros(state['q'].shape, device='cuda', dtype=torch.float64)
    lse = torch.zeros(state['q'].shape[:2], device='cuda', dtype=torch.float64)
    group, begin = case['group'], 0
    for s, (n, keys) in enumerate(zip(state['new'], state['keys'])):
        index = torch.arange(keys, device='cuda')
        page, row = state['table'][s].long()[index // case['page']], index % case['page']
        for h in range(case['kv_heads']):
            k, v = state['k_pages'][page, h, row].double(), state['v_pages'][page, h, row].double()
            q = state['q'][begin:begin + n, h * group:(h + 1) * group].double()
            score = torch.einsum('ngd,kd->ngk', q, k) / math.sqrt(case['dim'])
            if case['causal']:
                ahead = index[None] - (keys - n) > torch.arange(n, device='cuda')[:, None]
                score = torch.where(ahead[:, None], -math.inf, score)
            total = torch.logsumexp(score, -1)
            lse[begin:begin + n, h * group:(h + 1) * group] = total
            out[begin:begin + n, h * group:(h + 1) * group] = \
                torch.einsum('ngk,kd->ngd', torch.exp(score - total[..., None]), v)
        begin += n
    return dict(out=out, lse=lse) if case['lse'] else dict(out=out)

"""Workloads of the sequence operators: rotary positions, attention over packed sequences, the paged key / value cache
(plain or in 8 bits) and attention of new tokens over it.

A case is a dict of plain values; `prepare` makes what a program has in hand before the call, `run` makes one pass through
an operator - through the framework's entry points where `own` is true, in elementary torch operations otherwise - and
`exact` gives the same outputs from the definition in 64 bits.  Lengths are texts of numbers ("900 412 1"), one a sequence."""
import math
import random

import numpy as np
import torch

own = False

TYPES = {'bf16': torch.bfloat16, 'f32': torch.float32, 'e4m3': torch.float8_e4m3fn}
BYTES = {'bf16': 2, 'f32': 4, 'e4m3': 1}


def _ints(text):
    return [int(n) for n in text.split()]


def _text(ns):
    return ' '.join(str(n) for n in ns)


def _ragged(seed, n, low, high):
    r = random.Random(seed)
    return _text([high] + [r.randint(low, high) for _ in range(n - 1)])


# --------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one step of incremental synthesis for a batch of 16 at this framework's benchmark width (4 heads of 64): the
        # smallest call there is, bound by latency.  Half of each head is rotated, adjacent pairs.
        dict(name='rotary step', op='rotary', tokens=16, heads=4, kv_heads=4, dh=64, rot=32, interleaved=True,
             scaling='linear', factor=4.0, far=4096, type='f32', train=False),
        # a training step's queries and keys, grouped heads, frequencies stretched by bands for positions far beyond the
        # trained length: bound by memory
        dict(name='rotary train', op='rotary', tokens=16384, heads=32, kv_heads=8, dh=128, rot=128, interleaved=False,
             scaling='bands', factor=16.0, far=131072, type='bf16', train=True),
        # one short utterance through a layer of the reference's shipped width (2 heads of 192): latency
        dict(name='packed one utterance', op='packed', lens='61', heads=2, kv_heads=2, dh=192, causal=True, type='bf16', train=False),
        # the benchmark's batch of 32 utterances of up to 900 frames without its padding, every key seen (the decoder's
        # attention blocks), forward and backward
        dict(name='packed utterances train', op='packed', lens=_ragged(1, 32, 200, 900), heads=4, kv_heads=4, dh=64, causal=False,
             type='bf16', train=True),
        # the exact precision: a smaller causal batch in fp32, two query heads to a key head
        dict(name='packed f32 train', op='packed', lens=_ragged(2, 8, 60, 700), heads=4, kv_heads=2, dh=64, causal=True,
             type='f32', train=True),
        # whole prompts of very different lengths in one call, grouped heads, before a cache is read
        dict(name='packed prompts', op='packed', lens='8192 3001 513 1', heads=16, kv_heads=8, dh=128, causal=True, type='bf16', train=False),
        # a long causal training batch, eight query heads to a key head
        dict(name='packed long train', op='packed', lens='6000 1999 193', heads=16, kv_heads=2, dh=128, causal=True, type='bf16', train=True),
        # the keys and values of one decoding step of 64 sequences go into their pages: latency
        dict(name='cache append', op='cache', new=_text([1] * 64), lens=_ragged(3, 64, 1, 1536), page=16, kv_heads=8, dh=128,
             type='bf16', cache='bf16'),
        # whole prompts quantised to 8 bits as they are written, and read back: memory
        dict(name='cache prompts e4m3', op='cache', new='8191 4096 333', lens='8191 4096 333', page=64, kv_heads=8, dh=128,
             type='bf16', cache='e4m3'),
        # one decoding step of 32 sequences over caches of up to 8192 tokens in small pages
        dict(name='paged decode', op='paged', new=_text([1] * 32), lens=_ragged(4, 32, 100, 8192), page=16, heads=16, kv_heads=4,
             dh=128, type='bf16', cache='bf16'),
        # one decoding step of two long sequences over 8-bit caches: few rows and a long axis
        dict(name='paged decode long e4m3', op='paged', new='1 1', lens='131072 70001', page=64, heads=32, kv_heads=8, dh=128,
             type='bf16', cache='e4m3'),
        # chunks of prompts behind what is cached already, together with a single token
        dict(name='paged chunks', op='paged', new='512 384 97 1', lens='16384 9000 97 4001', page=32, heads=16, kv_heads=4, dh=128,
             type='bf16', cache='bf16'),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    kv = rng.choice([1, 2, 2, 4, 4, 8, 3])
    return kv * rng.choice([1, 1, 2, 4, 8] if kv < 8 else [1, 2, 4]), kv


def _split(rng, total, parts):
    """`total` in at most `parts` lengths, very uneven ones among them (a length of zero too)."""
    w = [rng.random() ** 3 + 1e-3 for _ in range(parts)]
    return [int(total * x / sum(w)) for x in w]


def draw(rng):
    op = rng.choice(['rotary', 'packed', 'packed', 'cache', 'paged', 'paged'])
    heads, kv = _heads(rng)
    dh = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192])
    kind = rng.choice(['bf16', 'bf16', 'f32'])
    if op == 'rotary':
        rot = rng.choice([dh, dh, dh // 2, dh // 4])
        tokens = min(_log(rng, 1, 16384), 16384 * 40 * 128 // ((heads + kv) * dh * BYTES[kind]))
        return dict(op=op, tokens=tokens, heads=heads, kv_heads=kv, dh=dh, rot=rot, interleaved=rng.random() < 0.5,
                    scaling=rng.choice(['none', 'linear', 'base', 'bands']), factor=rng.choice([2.0, 8.0, 32.0]),
                    far=_log(rng, 1024, 1048576), type=kind, train=rng.random() < 0.5)
    if op == 'packed':
        train = rng.random() < 0.6
        lens = _split(rng, _log(rng, 1, 9000 if kind == 'bf16' else 3000), rng.choice([1, 2, 5, 16, 40]))
        case = dict(op=op, heads=heads, kv_heads=kv, dh=dh, causal=rng.random() < 0.7, type=kind, train=train)
        # the plain form's padded scores fit, and no more work than the largest case above
        while len(lens) * heads * max(lens) ** 2 > 2e9 or work(dict(case, lens=_text(lens)))['flops'] > (5.5e11 if kind == 'bf16' else 6e10):
            lens = [n * 3 // 4 for n in lens]
        if max(lens) < (2 if train else 1):                  # (of one key alone the scores' gradients are nothing but rounding)
            lens[0] = 2
        return dict(case, lens=_text(lens))
    page = rng.choice([8, 16, 32, 64, 128])
    cache = rng.choice([kind, kind, 'e4m3'])
    kv = min(kv, 4) if kind == 'f32' else kv
    heads = heads // kv * kv
    if op == 'cache':
        n = rng.choice([1, 3, 16, 64])
        new = [1] * n if rng.random() < 0.4 else [max(1, x) for x in _split(rng, _log(rng, n, 12000), n)]
        lens = [x + rng.choice([0, rng.randrange(512)]) for x in new]
        return dict(op=op, new=_text(new), lens=_text(lens), page=page, kv_heads=kv, dh=dh, type=kind, cache=cache)
    n = rng.choice([1, 2, 4, 8, 32])
    new = [1] * n if rng.random() < 0.5 else [max(1, x) for x in _split(rng, _log(rng, n, 900), n)]
    most = min(131072, 200000 * 8 // (n * kv), 2 ** 29 // (n * heads * max(new)))
    lens = [x + _log(rng, 1, max(2, most)) - 1 for x in new]
    return dict(op=op, new=_text(new), lens=_text(lens), page=page, heads=heads, kv_heads=kv, dh=dh, type=kind, cache=cache)


# -------------------------------------------------------------------------------------------------------------- inputs
def frequencies(case):
    """Radians per position of each rotated pair, in 64 bits."""
    n, base, s = case['rot'], 10000.0, case['factor']
    i = np.arange(n // 2, dtype=np.float64)
    if case['scaling'] == 'base' and n > 2:
        base *= s ** (n / (n - 2))
    f = base ** (-2.0 * i / n)
    if case['scaling'] == 'linear':
        f = f / s
    if case['scaling'] == 'bands':                     # fast pairs kept, slow ones divided, a ramp of turns in between
        turns = 4096 * f / (2 * math.pi)
        keep = np.clip((turns - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        f = f * keep + f / s * (1 - keep)
    return f


def _randn(gen, shape, kind):
    return torch.randn(shape, generator=gen, device='cuda', dtype=torch.float32).to(TYPES[kind])


def _starts(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device='cuda')


def _split_projection(gen, rows, widths, dh, kind):
    """Views [rows, heads, dh] of one fused projection's output, as a layer has them; the first one (the queries) and the
    second (the keys) a little wider than normal, so that the softmax has rows that are flat and rows with a peak."""
    x = _randn(gen, (rows, sum(widths), dh), kind)
    x[:, :sum(widths[:2])] *= 1.25
    return list(torch.split(x, widths, dim=1))


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    state = {'case': case}
    dh, kind, kv = case['dh'], case['type'], case['kv_heads']
    if case['op'] == 'rotary':
        n = case['tokens']
        q, k = _split_projection(gen, n, [case['heads'], kv], dh, kind)
        state.update(q=q, k=k, freqs=torch.from_numpy(frequencies(case)).cuda(), scale=1.0 + 0.1 * math.log(case['factor']),
                     positions=torch.randint(0, case['far'], (n,), generator=gen, device='cuda', dtype=torch.int32))
        if case['train']:
            state.update(dq=_randn(gen, q.shape, kind), dk=_randn(gen, k.shape, kind))
        return state
    if case['op'] == 'packed':
        lens = _ints(case['lens'])
        q, k, v = _split_projection(gen, sum(lens), [case['heads'], kv, kv], dh, kind)
        state.update(q=q, k=k, v=v, starts=_starts(lens), longest=max(lens))
        if case['train']:
            state.update(dout=_randn(gen, q.shape, kind))
        return state
    new, lens, page = _ints(case['new']), _ints(case['lens']), case['page']
    counts = [-(-n // page) for n in lens]
    width, total = max(counts), sum(counts)
    pages = total + total // 4 + 1                                   # some free pages, the used ones in no order
    order = torch.randperm(pages, generator=gen, device='cuda', dtype=torch.int64)[:total].to(torch.int32)
    table = torch.full((len(new), width), -1, dtype=torch.int32, device='cuda')
    table[torch.arange(width, device='cuda')[None] < torch.tensor(counts, device='cuda')[:, None]] = order
    shape = (pages, kv, page, dh)
    for name in 'kv':
        x = torch.randn(shape, generator=gen, device='cuda', dtype=torch.float32)
        if name == 'k':
            x[..., ::17] *= 4.0                                      # a few wide channels, as keys have
        if case['cache'] == 'e4m3':
            state[name + '_pages'], state[name + '_exp'] = _quantise(x)
        else:
            state[name + '_pages'], state[name + '_exp'] = x.to(TYPES[case['cache']]), None
    state.update(table=table, starts=_starts(new), lens=torch.tensor(lens, dtype=torch.int32, device='cuda'), most_new=max(new),
                 longest=max(lens), total=sum(lens), ends=_starts(lens))
    if case['op'] == 'cache':
        state['k'], state['v'] = _split_projection(gen, sum(new), [kv, kv], dh, kind)
    else:
        state['q'] = _split_projection(gen, sum(new), [case['heads']], dh, kind)[0]
    return state


# --------------------------------------------------------------------------------------------------------- plain forms
def _power(e):
    """2^e of whole numbers, built from its bits: nothing is rounded."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x):
    """fp32 rows -> (e4m3 values, biased exponent of the row's power-of-two scale): the smallest scale that brings the
    row's largest finite magnitude to 448 at most."""
    top = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).abs().amax(-1)
    m, e = torch.frexp(top)
    e = torch.where(top > 0, torch.clamp(e - 8 - (m <= 0.875).to(e.dtype), -126, 127), torch.zeros_like(e))
    y = x * _power(-e[..., None])
    return y.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _values(pages, exp):
    x = pages.to(torch.float32)
    return x if exp is None else x * _power(exp.to(torch.int32)[..., None] - 127)


def _rotate(x, cos, sin, rot, interleaved):
    y = x.float()
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:rot])
    c, d = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1)
    return torch.cat((turned, y[..., rot:]), -1).to(x.dtype)


def _plain_rotary(s):
    c = s['case']
    angle = s['positions'].double()[:, None] * s['freqs'][None]
    cos, sin = ((s['scale'] * t).float()[:, None] for t in (torch.cos(angle), torch.sin(angle)))
    out = [_rotate(s[n], cos, sin, c['rot'], c['interleaved']) for n in 'qk']
    if c['train']:                                       # the gradient turns back
        out += [_rotate(s[n], cos, -sin, c['rot'], c['interleaved']) for n in ('dq', 'dk')]
    return out


def _rows(starts, longest, n):
    """Row numbers [sequences, longest] of packed sequences, and which of them are there."""
    at = torch.arange(longest, device=starts.device)
    rows = starts[:-1, None].long() + at
    there = at < (starts[1:] - starts[:-1])[:, None]
    return torch.where(there, rows, 0).clamp(max=max(n - 1, 0)), there


def _softmax(s, seen):
    s = s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = s.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    return e / e.sum(-1, keepdim=True).clamp_min(1e-30)


def _grouped(x, kv):
    """[B, L, H, dh] -> [B, kv, G * L, dh] in 32 bits."""
    b, n, h, dh = x.shape
    return x.float().view(b, n, kv, h // kv, dh).permute(0, 2, 3, 1, 4).reshape(b, kv, h // kv * n, dh)


def _ungrouped(x, n):
    b, kv, gn, dh = x.shape
    return x.view(b, kv, gn // n, n, dh).permute(0, 3, 1, 2, 4).reshape(b, n, kv * gn // n, dh)


def _plain_packed(s):
    c, q, k, v, kv = s['case'], s['q'], s['k'], s['v'], s['case']['kv_heads']
    rows, there = _rows(s['starts'], s['longest'], len(q))
    n, scale, group = s['longest'], 1.0 / math.sqrt(c['dh']), c['heads'] // kv
    pad = lambda x: _grouped(torch.where(there[..., None, None], x[rows], torch.zeros_like(x[:1])), kv)
    back = lambda x, like: _ungrouped(x, n)[there].to(like.dtype)
    seen = there[:, None, :].expand(-1, n, -1)
    if c['causal']:
        seen = seen & torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
    seen = seen[:, None, None]
    Q, K, V = pad(q), pad(k), pad(v)
    p = _softmax(((Q @ K.transpose(-1, -2)) * scale).view(-1, kv, group, n, n), seen).view(-1, kv, group * n, n)
    o = p @ V
    if not c['train']:
        return [back(o, q)]
    D = pad(s['dout'])
    dv = p.transpose(-1, -2) @ D
    ds = (D @ V.transpose(-1, -2)).sub_((D * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    return [back(o, q), back(ds @ K, q), back(ds.transpose(-1, -2) @ Q, k), back(dv, v)]


def _slots(s, which):
    """Flat page slots [tokens] of the new tokens (which = 'new') or of every token (which = 'all') in packed order."""
    starts = s['starts'] if which == 'new' else s['ends']
    n = len(s['k']) if which == 'new' else s['total']
    at = torch.arange(n, device=starts.device)
    b = torch.searchsorted(starts, at.to(torch.int32), right=True) - 1
    pos = s['lens'][b] - (starts[b + 1] - at)
    page = s['case']['page']
    return s['table'][b, pos // page].long(), pos.long() % page


def _plain_cache(s):
    p, r = _slots(s, 'new')
    for n in 'kv':
        if s[n + '_exp'] is None:
            s[n + '_pages'][p, :, r] = s[n].to(s[n + '_pages'].dtype)
        else:
            x, e = _quantise(s[n].float())
            s[n + '_pages'].view(torch.uint8)[p, :, r] = x.view(torch.uint8)
            s[n + '_exp'][p, :, r] = e
    if s['k_exp'] is None:
        return [s['k_pages'], s['v_pages']]
    p, r = _slots(s, 'all')
    return [_values(s[n + '_pages'].view(torch.uint8)[p, :, r].view(torch.float8_e4m3fn), s[n + '_exp'][p, :, r]).to(s[n].dtype) for n in 'kv']


def _plain_paged(s):
    c, q, kv = s['case'], s['q'], s['case']['kv_heads']
    rows, there = _rows(s['starts'], s['most_new'], len(q))
    n, table = s['most_new'], s['table'].clamp(min=0).long()
    b, width = table.shape

    def dense(name):
        e = s[name + '_exp']
        raw = s[name + '_pages'] if e is None else s[name + '_pages'].view(torch.uint8)
        x = raw[table] if e is None else raw[table].view(torch.float8_e4m3fn)
        return _values(x, None if e is None else e[table]).permute(0, 2, 1, 3, 4).reshape(b, kv, width * c['page'], c['dh'])

    Q = _grouped(torch.where(there[..., None, None], q[rows], torch.zeros_like(q[:1])), kv)
    group = c['heads'] // kv
    key = torch.arange(width * c['page'], device=q.device)
    pos = (s['lens'] - (s['starts'][1:] - s['starts'][:-1]))[:, None] + torch.arange(n, device=q.device)
    seen = ((key <= pos[..., None]) & (key < s['lens'][:, None, None]) & there[..., None])[:, None, None]
    w = (Q @ dense('k').transpose(-1, -2)).mul_(1.0 / math.sqrt(c['dh'])).view(b, kv, group, n, -1)
    o = _softmax(w, seen).view(b, kv, group * n, -1) @ dense('v')
    return [_ungrouped(o, n)[there].to(q.dtype)]


def run(state):
    if own:
        return _own(state)
    return {'rotary': _plain_rotary, 'packed': _plain_packed, 'cache': _plain_cache, 'paged': _plain_paged}[state['case']['op']](state)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    from transformertts_amd import ops
    c = s['case']
    if c['op'] == 'rotary':
        q, k = s['q'], s['k']
        if not c['train']:
            return list(ops.rotary(q, k, s['positions'], s['freqs'], interleaved=c['interleaved'], scale=s['scale']))
        q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
        out = ops.rotary(q, k, s['positions'], s['freqs'], interleaved=c['interleaved'], scale=s['scale'])
        return list(out) + list(torch.autograd.grad(out, [q, k], [s['dq'], s['dk']]))
    if c['op'] == 'packed':
        qkv = [s[n] for n in 'qkv']
        if not c['train']:
            return [ops.packed_attention(*qkv, s['starts'], causal=c['causal'])]
        qkv = [t.detach().requires_grad_() for t in qkv]
        out = ops.packed_attention(*qkv, s['starts'], causal=c['causal'])
        return [out] + list(torch.autograd.grad(out, qkv, s['dout']))
    cache = ops.KVCache(s['k_pages'], s['v_pages'], s['k_exp'], s['v_exp'])
    if c['op'] == 'cache':
        ops.kv_cache_write(cache, s['k'], s['v'], s['table'], s['starts'], s['lens'])
        if s['k_exp'] is None:
            return [cache.k, cache.v]
        return list(ops.kv_cache_read(cache, s['table'], s['lens'], s['ends'], s['total'], dtype=s['k'].dtype))
    return [ops.paged_attention(s['q'], cache, s['table'], s['starts'], s['lens'])]


# ---------------------------------------------------------------------------------------------------------------- cost
def work(case):
    dh, kv, size = case['dh'], case['kv_heads'], BYTES[case['type']]
    if case['op'] == 'rotary':
        n = case['tokens'] * (case['heads'] + kv)
        passes = 2 if case['train'] else 1
        return {'bytes': passes * (2 * n * dh * size + 4 * case['tokens']), 'flops': passes * 3 * n * case['rot']}
    if case['op'] == 'packed':
        lens, h = _ints(case['lens']), case['heads']
        pairs = sum(n * (n + 1) // 2 if case['causal'] else n * n for n in lens)
        rows = sum(lens) * dh * size                         # q, k, v -> out; the step also reads dout and writes three gradients
        return {'bytes': rows * (2 * h + 2 * kv) + (rows * (2 * h + 2 * kv) if case['train'] else 0),
                'flops': (14 if case['train'] else 4) * dh * h * pairs}
    new, lens, stored = _ints(case['new']), _ints(case['lens']), BYTES[case['cache']] * dh + (1 if case['cache'] == 'e4m3' else 0)
    if case['op'] == 'cache':
        b = 2 * kv * sum(new) * (dh * size + stored)
        return {'bytes': b + (2 * kv * sum(lens) * (dh * size + stored) if case['cache'] == 'e4m3' else 0),
                'flops': 2 * kv * dh * (sum(new) + sum(lens)) if case['cache'] == 'e4m3' else 0}
    h = case['heads']
    pairs = sum(n * (2 * t - n + 1) // 2 for n, t in zip(new, lens))
    return {'bytes': 2 * kv * sum(lens) * stored + 2 * sum(new) * h * dh * size, 'flops': 4 * dh * h * pairs}


# --------------------------------------------------------------------------------------------------------------- exact
def _exact_rotary(s):
    c = s['case']
    n = c['rot']
    turn = torch.polar(torch.full_like(s['freqs'], s['scale'])[None], s['positions'].double()[:, None] * s['freqs'])[:, None]
    pick = torch.arange(n).view(n // 2, 2).T if c['interleaved'] else torch.arange(n).view(2, n // 2)

    def turned(x, w):
        y = x.double().clone()
        z = torch.complex(y[..., pick[0]], y[..., pick[1]]) * w
        y[..., pick[0]], y[..., pick[1]] = z.real, z.imag
        return y
    out = [turned(s['q'], turn), turned(s['k'], turn)]
    return out + ([turned(s['dq'], turn.conj()), turned(s['dk'], turn.conj())] if c['train'] else [])


def _exact_attention(q, k, v, first, causal=True):
    """q [n, H, dh] at positions first, first + 1, ... over k, v [t, kv, dh], head by head in 64 bits."""
    group, out = q.shape[1] // k.shape[1], []
    hidden = torch.arange(k.shape[0], device=q.device) > (first + torch.arange(q.shape[0], device=q.device))[:, None]
    for h in range(q.shape[1]):
        w = q[:, h].double() @ k[:, h // group].double().T / math.sqrt(q.shape[2])
        w = torch.softmax(w.masked_fill(hidden, -math.inf) if causal else w, -1)
        out.append(w @ v[:, h // group].double())
    return torch.stack(out, 1)


def _exact_packed(s):
    c = s['case']
    parts, at = [], 0
    for n in _ints(c['lens']):
        if n == 0:
            continue
        x = [s[name][at:at + n].double().detach().requires_grad_(c['train']) for name in 'qkv']
        o, grads = [], [torch.zeros_like(t) for t in x]
        group = c['heads'] // c['kv_heads']
        for h in range(c['heads']):                          # one head's graph at a time
            one = _exact_attention(x[0][:, h:h + 1], x[1][:, h // group:h // group + 1], x[2][:, h // group:h // group + 1], 0, c['causal'])
            if c['train']:
                for total, g in zip(grads, torch.autograd.grad(one, x, s['dout'][at:at + n, h:h + 1].double())):
                    total += g
            o.append(one.detach())
        parts.append([torch.cat(o, 1)] + (grads if c['train'] else []))
        at += n
    return [torch.cat(p) for p in zip(*parts)]


def _two_to(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _grid(x):
    """The nearest e4m3 value of a 64-bit number (ties to even), under the row's smallest power-of-two scale."""
    top = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)
    scale = _two_to(torch.where(top > 0, (e - 9 + (m > 0.875)).clamp(-126, 127), torch.zeros_like(e)))
    y = x / scale
    step = _two_to(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -20))).clamp_min(-6) - 3)
    return torch.round(y / step) * step * scale


def _exact_cache(s):
    c, new, lens, outs = s['case'], _ints(s['case']['new']), _ints(s['case']['lens']), []
    for name in 'kv':
        plain = s[name + '_exp'] is None
        pages = s[name + '_pages'].double().clone() if plain else s[name + '_pages'].double() * _two_to(s[name + '_exp'].long() - 127)[..., None]
        fresh = s[name].double() if plain else _grid(s[name].double())
        back, at = [], 0
        for b, (n, t) in enumerate(zip(new, lens)):
            used = s['table'][b, :-(-t // c['page'])].long()
            seq = pages[used].transpose(1, 2).reshape(-1, c['kv_heads'], c['dh'])
            seq[t - n:t] = fresh[at:at + n]
            pages[used] = seq.view(len(used), c['page'], c['kv_heads'], c['dh']).transpose(1, 2)
            back.append(seq[:t])
            at += n
        outs.append(pages if plain else torch.cat(back))
    return outs


def _exact_paged(s):
    c, outs, at = s['case'], [], 0
    for b, (n, t) in enumerate(zip(_ints(c['new']), _ints(c['lens']))):
        used = s['table'][b, :-(-t // c['page'])].long()
        x = []
        for name in 'kv':
            y = s[name + '_pages'].view(torch.uint8)[used].view(torch.float8_e4m3fn).double() if c['cache'] == 'e4m3' else s[name + '_pages'][used].double()
            y = y if s[name + '_exp'] is None else y * _two_to(s[name + '_exp'][used].long() - 127)[..., None]
            x.append(y.transpose(1, 2).reshape(-1, c['kv_heads'], c['dh'])[:t])
        outs.append(_exact_attention(s['q'][at:at + n], *x, t - n))
        at += n
    return [torch.cat(outs)]


def exact(case, seed):
    s = prepare(case, seed)
    return {'rotary': _exact_rotary, 'packed': _exact_packed, 'cache': _exact_cache, 'paged': _exact_paged}[case['op']](s)

"""-m gpu tests of how exact the bf16 attention operators are on batches of short sequences and on single tokens: a product's rounded
operand (a probability, a score gradient) goes in as two bf16 parts there, so that the outputs are off by their own rounding and
little more.

In sequences of a few keys nothing averages an operand's rounding: with one part the gradients of two keys were up to 2.1 times as
far from the formula as their own rounding puts them.  Bounds, element by element, from the sizes of the terms in 64 bits: HALF =
2^-8 for the output's rounding, TWO = 2^-16 for an operand of two parts (half a step of half a step), U = 2^-23 for fp32 operations."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
U, HALF, TWO = 2.0 ** -23, 2.0 ** -8, 2.0 ** -16
BF, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def _ops():
    from transformertts_amd import ops
    return ops


def _randn(shape, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(BF)


def _starts(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=DEV)


def exact_attention(q, k, v, first, causal, scale, d=None):
    """One sequence in 64 bits: ([out, dq, dk, dv], [bound of each])."""
    (n, H, dh), (t, Hkv, _) = q.shape, k.shape
    G = H // Hkv
    q, k, v = (x.double().transpose(0, 1) for x in (q, k, v))
    q = q.reshape(Hkv, G * n, dh)                                                            # the rows of a group's heads, one after the other
    seen = torch.ones(n, t, dtype=torch.bool)
    if causal:
        seen = torch.arange(t) <= first + torch.arange(n)[:, None]
    seen = seen.repeat(G, 1)
    s = (q @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1)
    mag = (q.abs() @ k.abs().transpose(1, 2) * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    ep = 2 * (dh + 8) * U * mag + (t + 16) * U                                              # a probability's, relative
    out = p @ v
    e_out = (ep + TWO) * (p @ v.abs())                                                       # before its rounding
    res, bounds = [out], [e_out + HALF * (out.abs() + e_out)]
    if d is not None:
        d = d.double().transpose(0, 1).reshape(Hkv, G * n, dh)
        dp, delta = d @ v.transpose(1, 2), (d * out).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        e_delta = (d.abs() * (e_out + TWO * out.abs())).sum(-1, keepdim=True) + (dh + 8) * U * (d.abs() * out.abs()).sum(-1, keepdim=True)
        e_ds = p * ((ep + 4 * U) * (dp - delta).abs() + (dh + 8) * U * (d.abs() @ v.abs().transpose(1, 2)) + e_delta)
        e_ds = e_ds + TWO * (ds.abs() + e_ds)
        rows = G * n
        res += [scale * ds @ k, scale * ds.transpose(1, 2) @ q, p.transpose(1, 2) @ d]
        raw = [scale * (e_ds + (t + 8) * U * ds.abs()) @ k.abs(), scale * (e_ds + (rows + 8) * U * ds.abs()).transpose(1, 2) @ q.abs(),
               ((ep + TWO + (rows + 8) * U) * p).transpose(1, 2) @ d.abs()]
        bounds += [b + HALF * (x.abs() + b) for x, b in zip(res[1:], raw)]
    back = lambda x: (x.reshape(Hkv, G, n, dh).reshape(H, n, dh) if x.shape[1] == G * n and x.shape[0] == Hkv else x)
    heads = [back(x) if i < 2 else x for i, x in enumerate(res)]
    limits = [back(x) if i < 2 else x for i, x in enumerate(bounds)]
    return [x.transpose(0, 1) for x in heads], [x.transpose(0, 1) + 1e-30 for x in limits]


def _within(got, want, bound, what):
    got = got.detach().double().cpu()
    bad = ~((got - want).abs() <= bound)
    off = int(bad.sum())
    assert off == 0, f'{what}: {off} of {bad.numel()} off, {float(((got - want).abs() / bound).max()):.2f} times the bound'


@pytest.mark.parametrize('lens,H,Hkv,dh,causal', [
    ([2], 4, 4, 128, True), ([2], 8, 2, 192, False), ([12], 4, 2, 192, True), ([2, 1, 0, 5], 8, 2, 64, False), ([6, 29], 2, 2, 32, True), ([61], 2, 2, 192, True),
    ([9, 70, 33], 4, 1, 80, True), ([200, 57], 4, 4, 128, False), ([250], 8, 2, 64, True), ([255, 250], 2, 2, 96, True), ([3] * 40, 4, 2, 64, True), ([130], 3, 3, 184, False),
    ([170, 255], 4, 2, 128, True)])
def test_packed_attention_of_few_rows(lens, H, Hkv, dh, causal):
    from transformertts_amd import _lib
    M = sum(lens)
    q, k, v, d = (_randn((M, h, dh), 30 + i, 1.25 if i < 2 else 1.0) for i, h in enumerate((H, Hkv, Hkv, H)))
    x = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    out = _ops().packed_attention(*x, _starts(lens), causal=causal)
    assert _lib.lib().ttsmi_last_kernel() == b'seq_attn_fwd_kernel, keys in two'
    got = [out] + list(torch.autograd.grad(out, x, d.to(DEV)))
    at = 0
    for n in lens:
        if n:
            want, bound = exact_attention(*(t[at:at + n] for t in (q, k, v)), 0, causal, dh ** -0.5, d[at:at + n])
            for name, g, w, b in zip(('out', 'dq', 'dk', 'dv'), got, want, bound):
                _within(g[at:at + n], w, b, f'{name} of the sequence of {n}')
        at += n


@pytest.mark.parametrize('stored', [BF, E4M3])
@pytest.mark.parametrize('new,lens,page,H,Hkv,dh', [([1], [2], 16, 4, 4, 128), ([1, 1], [700, 33], 8, 16, 2, 128), ([2, 1, 1], [9, 70, 1], 16, 8, 4, 64), ([1], [2500], 64, 8, 1, 192),
                                                    ([1] * 20, [1 + 13 * i for i in range(20)], 32, 4, 2, 32)])
def test_single_tokens_over_the_cache(new, lens, page, H, Hkv, dh, stored):
    from transformertts_amd import _lib
    ops = _ops()
    counts = [-(-n // page) for n in lens]
    cache = ops.KVCache.zeros(sum(counts), page, Hkv, dh, stored, DEV)
    table, at = torch.full((len(lens), max(counts)), -1, dtype=torch.int32), 0
    for b, c in enumerate(counts):
        table[b, :c] = torch.arange(at, at + c)
        at += c
    table, ln, total = table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), sum(lens)
    ops.kv_cache_write(cache, _randn((total, Hkv, dh), 1, 1.25).to(DEV), _randn((total, Hkv, dh), 2).to(DEV), table, _starts(lens), ln)
    k, v = (t.cpu() for t in ops.kv_cache_read(cache, table, ln, _starts(lens), total, dtype=BF))
    q = _randn((sum(new), H, dh), 3, 1.25)
    got = ops.paged_attention(q.to(DEV), cache, table, _starts(new), ln)
    assert _lib.lib().ttsmi_last_kernel() == b'paged_rows_kernel'
    at = base = 0
    for m, n in zip(new, lens):
        want, bound = exact_attention(q[at:at + m], k[base:base + n], v[base:base + n], n - m, True, dh ** -0.5)
        _within(got[at:at + m], want[0], bound[0], f'{m} over {n}')
        at, base = at + m, base + n

"""-m gpu tests that every key and every row counts once in the attention operators, whatever the tiles, waves, pages and splits
between them.

With all scores equal a probability is one over the number of keys seen, and each sum is marked so that every (key, row) pair has a
place of its own in the result: a key lost is a 0 there, one taken twice is twice the value, and a count off by one is off by 1 / n.
Tolerances: HALF (half a step of the type) for every rounding to bf16 - the probability or score gradient where it becomes an
operand, and the output - and U = 2^-23 for each fp32 operation; the normaliser n and its logarithm, where the backward passes take
n from it, are off by a few U, the logarithm times at most log2(n) < 16 more."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
U = 2.0 ** -23
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
BF, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _ops():
    from transformertts_amd import ops
    return ops


def _kernel():
    from transformertts_amd import _lib
    return _lib.lib().ttsmi_last_kernel()


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(lens):
    return _ints([0] + torch.tensor(lens).cumsum(0).tolist())


def _near(got, want, bound, what):
    off = (got.double() - want).abs() - bound
    assert bool((off <= 0).all()), f'{what}: {int((off > 0).sum())} of {off.numel()} off, first at {(off > 0).nonzero()[0].tolist()}'


def _marks(total, heads, dh, nth):
    """[total, heads, dh] fp32 with element (head, c) of index nth heads dh + head dh + c set to 1: every index has a place in one of
    the ceil(total / (heads dh)) marks."""
    x = torch.zeros(total, heads, dh, device=DEV)
    at = nth * heads * dh + torch.arange(heads * dh, device=DEV)
    there = at < total
    x.view(total, heads * dh)[at[there], torch.arange(heads * dh, device=DEV)[there]] = 1
    return x


PAGED = [([1, 1, 1, 1], [5003, 64, 1, 129], 16, 128, 8, 128, b'paged_rows_kernel'), ([1], [20011], 64, 64, 4, 192, b'paged_rows_kernel'),
         ([2, 1], [3001, 4097], 8, 32, 4, 64, b'paged_rows_kernel'), ([1], [3001], 2, 64, 4, 64, b'paged_rows_kernel'),
         ([40], [5003], 16, 64, 8, 128, b'seq_attn_fwd_kernel'), ([130, 70, 66], [9001, 70, 67], 64, 16, 4, 64, b'seq_attn_fwd_kernel'),
         ([70], [2050], 4, 16, 4, 128, b'seq_attn_fwd_kernel'), ([70], [2050], 8, 8, 2, 192, b'seq_attn_fwd_kernel'),
         ([300] * 9, [300 + 67 * i for i in range(9)], 32, 32, 8, 64, b'seq_attn_fwd_kernel')]
TYPES = [(BF, BF), (BF, E4M3), (F32, F32), (F32, E4M3)]


class _Cached:
    def __init__(self, lens, page, Hkv, dh, stored):
        counts = [-(-n // page) for n in lens]
        self.cache = _ops().KVCache.zeros(sum(counts) + 1, page, Hkv, dh, stored, DEV)
        order = torch.randperm(sum(counts) + 1, generator=torch.Generator().manual_seed(3)).to(torch.int32)
        table, at = torch.full((len(lens), max(counts)), -1, dtype=torch.int32), 0
        for b, c in enumerate(counts):
            table[b, :c] = order[at:at + c]
            at += c
        self.table, self.lens, self.all = table.to(DEV), _ints(lens), _starts(lens)

    def write(self, k, v):
        _ops().kv_cache_write(self.cache, k, v, self.table, self.all, self.lens)


@pytest.mark.parametrize('dtype,stored', TYPES)
@pytest.mark.parametrize('new,lens,page,H,Hkv,dh,form', PAGED)
def test_every_cached_key_counts_once(new, lens, page, H, Hkv, dh, form, dtype, stored):
    world, total = _Cached(lens, page, Hkv, dh, stored), sum(lens)
    q, st = torch.zeros(sum(new), H, dh, dtype=dtype, device=DEV), _starts(new)
    keys = torch.randn((total, Hkv, dh), generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    seen = torch.cat([torch.arange(n - m + 1, n + 1) for m, n in zip(new, lens)]).to(DEV).double()
    for nth in range(-(-max(lens) // (Hkv * dh))):
        world.write(keys, torch.cat([_marks(n, Hkv, dh, nth) for n in lens]).to(dtype))
        got = _ops().paged_attention(q, world.cache, world.table, st, world.lens)
        at = (nth * Hkv * dh + torch.arange(Hkv * dh, device=DEV)).view(1, Hkv, 1, dh)
        want = ((at < seen.view(-1, 1, 1, 1)).double() / seen.view(-1, 1, 1, 1)).expand(-1, -1, H // Hkv, -1).reshape(-1, H, dh)
        _near(got, want, (HALF[dtype] + 8 * U) * want, f'keys from {nth * Hkv * dh}')
    assert _kernel() == form


@pytest.mark.parametrize('dtype,stored', TYPES)
@pytest.mark.parametrize('new,lens,page,H,Hkv,dh,form', PAGED)
def test_every_cached_key_is_found(new, lens, page, H, Hkv, dh, form, dtype, stored):
    """Every key in turn is the one that a query asks for: keys are random signs, the query is the key's own signs, and all other
    scores stay more than 30 below (6.3 deviations of the largest of 10^9 products: 104 below for heads of 192, 57 for 128 and for 64,
    whose scale is 4), so that they add less than 20011 e^-30 < 2^-28: the output is that key's value, with the roundings of its
    probability and of the output."""
    world, total = _Cached(lens, page, Hkv, dh, stored), sum(lens)
    gen = torch.Generator().manual_seed(5)
    k, v = (torch.randint(0, 2, (total, Hkv, dh), generator=gen).to(DEV) * 2.0 - 1 for _ in 'kv')
    world.write(k.to(dtype), v.to(dtype))
    st, scale, G = _starts(new), 4.0 if dh == 64 else 1.0, H // Hkv
    seen = torch.cat([torch.arange(n - m + 1, n + 1) for m, n in zip(new, lens)]).to(DEV)
    first = torch.repeat_interleave(torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist()[:-1]), torch.tensor(new)).to(DEV)
    step = min(m for m in new) * G                        # keys of each sequence asked for by one call, at least
    for nth in range(-(-max(lens) // step)):
        want_key = torch.empty((sum(new), H), dtype=torch.int64, device=DEV)
        at = 0
        for m, n in zip(new, lens):                        # token t, query head g of the group: key nth step + (t G + g), the latest seen if it is past that
            r = (torch.arange(m, device=DEV).view(-1, 1) * G + torch.arange(G, device=DEV)).repeat(1, Hkv)
            want_key[at:at + m] = torch.minimum(nth * step + r, seen[at:at + m].view(-1, 1) - 1)
            at += m
        index = first.view(-1, 1) + want_key
        head = torch.arange(H, device=DEV) // G
        q = k[index, head].to(dtype)
        got = _ops().paged_attention(q, world.cache, world.table, st, world.lens, scale=scale)
        _near(got, v[index, head].double(), torch.tensor((1 + HALF[dtype]) ** 2 * (1 + 16 * U) - 1, device=DEV), f'keys from {nth * step}')


PACKED = [([515], 4, 2, 64), ([700, 3, 0, 1100], 8, 8, 64), ([130, 64, 1], 2, 1, 128), ([900], 12, 4, 192), ([2050, 31], 8, 4, 128), ([300] * 40, 8, 8, 64), ([600] * 5, 32, 8, 128),
          ([37] * 70 + [200], 8, 2, 64)]


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('lens,H,Hkv,dh', PACKED)
def test_every_pair_of_a_sequence_counts_once(lens, H, Hkv, dh, causal, dtype):
    """Forward: every key in every row.  dV and dK: every row of every head in every key.  dQ: every key in every row."""
    ops, M, G, st, scale = _ops(), sum(lens), H // Hkv, _starts(lens), dh ** -0.5
    place = torch.cat([torch.arange(n) for n in lens]).to(DEV)                               # of a token in its sequence
    length = torch.repeat_interleave(torch.tensor(lens), torch.tensor(lens)).to(DEV)
    seen = (place + 1 if causal else length).double()
    twice = (1 + HALF[dtype]) * (1 + (HALF[dtype] if dtype == BF else 0.0)) * (1 + 64 * U) - 1       # an operand's rounding and the output's
    rest = 2.0 ** -16 + 16 * U                                                                    # delta: of an output known to two bf16 parts
    keys = torch.randn((M, Hkv, dh), generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    zeros = lambda h: torch.zeros(M, h, dh, dtype=dtype, device=DEV)
    sign = (1.0 - 2.0 * (place % 2)).double()                                              # a value's sign: + - + - ...
    mean = torch.where(seen % 2 == 1, 1 / seen, torch.zeros_like(seen))                       # of the signs seen: delta
    flat, gate = zeros(Hkv), zeros(H)
    flat[:, :, 0], gate[:, :, 0] = sign.to(dtype).view(-1, 1), 1.0

    def step(q, k, v, d):
        x = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ops.packed_attention(*x, st, causal=causal)
        return [out.detach()] + list(torch.autograd.grad(out, x, d))
    longest = max(lens)
    for nth in range(-(-longest // (Hkv * dh))):
        marks = torch.cat([_marks(n, Hkv, dh, nth) for n in lens]).to(dtype)
        key = (nth * Hkv * dh + torch.arange(Hkv * dh, device=DEV)).view(1, Hkv, 1, dh)
        there = (key < (place + 1 if causal else length).view(-1, 1, 1, 1)).double()
        pair = (there / seen.view(-1, 1, 1, 1)).expand(-1, -1, G, -1).reshape(M, H, dh)
        got = step(zeros(H), keys, marks, zeros(H))[0]
        _near(got, pair, (HALF[dtype] + 8 * U) * pair, f'out, keys from {nth * Hkv * dh}')
        # q = 0: the marked keys stand in dQ with the score gradients of their pairs, p_ij (+-1 - mean)
        ds = (there * (1.0 - 2.0 * (key % 2)) - there * mean.view(-1, 1, 1, 1)) / seen.view(-1, 1, 1, 1) * scale
        ds = ds.expand(-1, -1, G, -1).reshape(M, H, dh)
        got = step(zeros(H), marks, flat, gate)[1]
        _near(got, ds, twice * ds.abs() + rest * pair * scale, f'dq, keys from {nth * Hkv * dh}')
    rows = longest * G
    for nth in range(-(-rows // dh)):
        # row r of a sequence (token r / G, head r % G of each group) marks column r - nth dh of every key head
        r = nth * dh + torch.arange(dh, device=DEV)
        tok = r // G
        marks = zeros(H)
        ok = tok.view(1, -1) < length.view(-1, 1)
        own = (place.view(-1, 1) == tok.view(1, -1)) & ok                                   # [M, dh]
        t, c = own.nonzero(as_tuple=True)
        for hk in range(Hkv):
            marks[t, hk * G + r[c] % G, c] = 1
        met = ok & ((place.view(-1, 1) <= tok.view(1, -1)) if causal else torch.ones_like(ok))        # key (row of the array) meets row r
        n = (tok + 1).view(1, -1).double().expand(M, -1) if causal else length.view(-1, 1).double().expand(-1, dh)
        pair = (met.double() / n).view(M, 1, dh).expand(-1, Hkv, -1)
        dv = step(zeros(H), zeros(Hkv), zeros(Hkv), marks)[3]
        _near(dv, pair, twice * pair, f'dv, rows from {nth * dh}')
        mean_r = torch.where(n % 2 == 1, 1 / n, torch.zeros_like(n))
        ds = ((met.double() * (sign.view(-1, 1) - mean_r)) / n * scale).view(M, 1, dh).expand(-1, Hkv, -1)
        dk = step(marks, zeros(Hkv), flat, gate)[2]
        _near(dk, ds, twice * ds.abs() + rest * pair * scale, f'dk, rows from {nth * dh}')

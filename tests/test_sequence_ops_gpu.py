"""-m gpu tests of the sequence operators (rotary positions, attention over packed sequences, the paged key / value cache and
attention over it) against plain 64-bit CPU restatements.

Tolerances are bounds, element by element, from the sizes of the terms of each sum (in 64 bits) and the roundings that the
operators make: U = 2^-23 for an fp32 operation (twice the half step, for the matrix unit's accumulation), H = 2^-8 (bf16) for
each rounding of a probability, a score gradient or an output, 0 for fp32 tensors."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
U = 2.0 ** -23
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def _ops():
    from transformertts_amd import ops
    return ops


def _randn(shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _starts(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist() if lens else [0], dtype=torch.int32)


def _within(got, want, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), f'{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - want).abs()[bad].max())} where {float(bound[bad].min())} is allowed'


# ------------------------------------------------------------------------------------------------------------------ oracle
def attention_oracle(q, k, v, first, causal, scale, dtype, dout=None):
    """q [n, H, dh] at positions first .. over k, v [t, Hkv, dh] in 64 bits: ([out, dq, dk, dv], [bound of each])."""
    n, H, dh = q.shape
    t, Hkv = k.shape[:2]
    q, k, v = q.double(), k.double(), v.double()
    Hb = HALF[dtype] if dtype == torch.bfloat16 else 0.0
    seen = torch.ones(n, t, dtype=torch.bool)
    if causal:
        seen = torch.arange(t)[None] <= first + torch.arange(n)[:, None]
    out, bout = torch.zeros(n, H, dh).double(), torch.zeros(n, H, dh).double()
    grads = [torch.zeros_like(x) for x in (q, k, v)]
    bounds = [torch.zeros_like(x) for x in (q, k, v)]
    for h in range(H):
        g = h // (H // Hkv)
        s = (q[:, h] @ k[:, g].T * scale).masked_fill(~seen, -math.inf)
        some = seen.any(1, keepdim=True)
        p = torch.where(seen, torch.softmax(torch.where(some, s, torch.zeros_like(s)), -1), torch.zeros_like(s))
        # relative error of a probability: twice the score's (its own and the normaliser's), exp2 and the sums
        mag = (q[:, h].abs() @ k[:, g].abs().T * scale)
        es = (dh + 8) * U * (mag * seen).amax(1, keepdim=True) if t else torch.zeros(n, 1).double()
        ep = 2 * es + (t + 16) * U
        o = p @ v[:, g]
        out[:, h] = o
        bo = (ep + Hb) * (p @ v[:, g].abs())
        bout[:, h] = bo + HALF[dtype] * (o.abs() + bo) + 1e-30
        if dout is None:
            continue
        d = dout[:, h].double()
        dp, delta = d @ v[:, g].T, (d * o).sum(1, keepdim=True)
        ds = p * (dp - delta)
        e_dp = (dh + 8) * U * (d.abs() @ v[:, g].abs().T)
        e_delta = (d.abs() * bout[:, h]).sum(1, keepdim=True) + (dh + 8) * U * (d.abs() * o.abs()).sum(1, keepdim=True)
        e_ds = p * ((ep + 4 * U) * (dp - delta).abs() + e_dp + e_delta)
        e_ds = e_ds + Hb * (ds.abs() + e_ds)
        rows = n * (H // Hkv)
        grads[0][:, h] = scale * ds @ k[:, g]
        bounds[0][:, h] += scale * (e_ds + (t + 8) * U * ds.abs()) @ k[:, g].abs()
        grads[1][:, g] += scale * ds.T @ q[:, h]
        bounds[1][:, g] += scale * (e_ds + (rows + 8) * U * ds.abs()).T @ q[:, h].abs()
        grads[2][:, g] += p.T @ d
        bounds[2][:, g] += ((ep + Hb + (rows + 8) * U) * p).T @ d.abs()
    bounds = [b + HALF[dtype] * (x.abs() + b) + 1e-30 for x, b in zip(grads, bounds)]
    return [out] + grads, [bout] + bounds


def packed_oracle(q, k, v, lens, causal, scale, dout=None):
    parts, at = [], 0
    for n in lens:
        x = [None if y is None else y[at:at + n] for y in (q, k, v, dout)]
        parts.append(attention_oracle(x[0], x[1], x[2], 0, causal, scale, q.dtype, x[3]))
        at += n
    return [[torch.cat(c) for c in zip(*(p[i] for p in parts))] for i in (0, 1)]


def _grads(out, xs, d):
    return [out] + list(torch.autograd.grad(out, xs, d))


# --------------------------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('lens,H,Hkv,dh,causal', [
    ([1], 1, 1, 8, True), ([2], 4, 2, 64, True), ([61], 2, 2, 192, True), ([33], 3, 1, 40, False), ([5, 0, 130, 1, 64], 4, 2, 64, True),
    ([5, 0, 130, 1, 64], 4, 4, 64, False), ([0, 0, 7], 2, 1, 128, True), ([257, 128, 31], 8, 2, 128, True), ([200, 90], 6, 3, 96, False),
    ([300], 4, 1, 192, True), ([129, 127], 16, 2, 80, True), ([3] * 70 + [0, 65], 2, 2, 32, True), ([515], 12, 4, 16, True)])
def test_packed_attention(lens, H, Hkv, dh, causal, dtype):
    ops = _ops()
    M = sum(lens)
    q, k, v, d = (_randn((M, h, dh), i, dtype, s) for i, (h, s) in enumerate([(H, 1.5), (Hkv, 1.5), (Hkv, 1.0), (H, 1.0)]))
    want, bound = packed_oracle(q, k, v, lens, causal, dh ** -0.5, d)
    xs = [x.to(DEV).requires_grad_() for x in (q, k, v)]
    got = _grads(ops.packed_attention(*xs, _starts(lens).to(DEV), causal=causal), xs, d.to(DEV))
    for name, g, w, b in zip(('out', 'dq', 'dk', 'dv'), got, want, bound):
        assert g.dtype == dtype
        _within(g, w, b, name)
    with torch.no_grad():                                               # the form without lse: the same bits
        assert torch.equal(ops.packed_attention(*xs, _starts(lens).to(DEV), causal=causal), got[0])


@pytest.mark.parametrize('dtype,lens,H,Hkv,dh,causal', [
    (torch.bfloat16, [1100, 0, 3, 1001], 16, 16, 64, True), (torch.bfloat16, [650, 490], 32, 32, 128, True), (torch.bfloat16, [1030, 65], 32, 32, 192, False),
    (torch.float32, [900, 350], 32, 32, 64, True), (torch.float32, [700, 450], 32, 32, 128, False), (torch.float32, [600], 64, 64, 184, True),
    (torch.bfloat16, [1100], 64, 64, 8, False), (torch.float32, [900, 700], 128, 128, 8, True), (torch.bfloat16, [700, 33], 96, 12, 72, True)])
def test_packed_attention_many_tiles(dtype, lens, H, Hkv, dh, causal):
    """Batches that fill the card: a wave meets every key of its tiles, and key tiles enough for the dK / dV pass not to split rows."""
    from transformertts_amd import _lib
    ops = _ops()
    M = sum(lens)
    q, k, v, d = (_randn((M, h, dh), 50 + i, dtype) for i, h in enumerate((H, Hkv, Hkv, H)))
    want, bound = packed_oracle(q, k, v, lens, causal, dh ** -0.5, d)
    xs = [x.to(DEV).requires_grad_() for x in (q, k, v)]
    out = ops.packed_attention(*xs, _starts(lens).to(DEV), causal=causal)
    assert _lib.lib().ttsmi_last_kernel() == b'seq_attn_fwd_kernel'
    for name, g, w, b in zip(('out', 'dq', 'dk', 'dv'), _grads(out, xs, d.to(DEV)), want, bound):
        _within(g, w, b, name)


@pytest.mark.parametrize('dtype,causal', [(torch.bfloat16, True), (torch.bfloat16, False), (torch.float32, True)])
def test_packed_attention_more_sequences_than_lanes(dtype, causal):
    """Seventy and more sequences, several rounds of workgroups: tiles start in the order of their work, 64 sequences at a time, and
    every one of them starts once."""
    ops = _ops()
    lens, H, Hkv, dh = [37] * 40 + [500, 0, 1, 129] + [37] * 30 + [900, 0, 130, 64], 8, 8, 64
    M = sum(lens)
    q, k, v, d = (_randn((M, h, dh), 80 + i, dtype) for i, h in enumerate((H, Hkv, Hkv, H)))
    want, bound = packed_oracle(q, k, v, lens, causal, dh ** -0.5, d)
    xs = [x.to(DEV).requires_grad_() for x in (q, k, v)]
    for name, g, w, b in zip(('out', 'dq', 'dk', 'dv'), _grads(ops.packed_attention(*xs, _starts(lens).to(DEV), causal=causal), xs, d.to(DEV)), want, bound):
        _within(g, w, b, name)


@pytest.mark.parametrize('dtype,lens,H,Hkv,dh,causal,parts', [
    (torch.bfloat16, [1000, 333], 4, 2, 128, True, 'four'), (torch.bfloat16, [700, 90, 400], 8, 8, 64, False, 'four'), (torch.bfloat16, [1999], 6, 2, 40, True, 'four'),
    (torch.float32, [515, 300], 2, 1, 64, True, 'four'), (torch.float32, [129, 600], 3, 3, 24, False, 'four'), (torch.bfloat16, [900, 7], 8, 8, 128, True, 'four'), (torch.bfloat16, [1500], 8, 8, 128, True, 'two'),
    (torch.float32, [450, 450], 4, 4, 128, False, 'two'), (torch.bfloat16, [333, 500], 4, 2, 192, True, 'two'), (torch.float32, [60] * 20, 4, 4, 64, True, 'two')])
def test_packed_attention_keys_in_parts(dtype, lens, H, Hkv, dh, causal, parts):
    """Few tiles: two or four waves share a row block, the keys between them - parts that have none, or end inside a run, among them."""
    from transformertts_amd import _lib
    ops = _ops()
    M = sum(lens)
    q, k, v, d = (_randn((M, h, dh), 60 + i, dtype) for i, h in enumerate((H, Hkv, Hkv, H)))
    want, bound = packed_oracle(q, k, v, lens, causal, dh ** -0.5, d)
    xs = [x.to(DEV).requires_grad_() for x in (q, k, v)]
    out = ops.packed_attention(*xs, _starts(lens).to(DEV), causal=causal)
    assert _lib.lib().ttsmi_last_kernel() == b'seq_attn_fwd_kernel, keys in ' + parts.encode()
    for name, g, w, b in zip(('out', 'dq', 'dk', 'dv'), _grads(out, xs, d.to(DEV)), want, bound):
        _within(g, w, b, name)


def test_packed_attention_scale_and_peaked_scores():
    """Scores of some hundreds: the running maximum carries them, forward and backward stay finite and right."""
    ops = _ops()
    lens, H, dh = [190, 66], 2, 64
    q, k, v, d = (_randn((256, H, dh), i, torch.float32, 4.0) for i in range(4))
    want, bound = packed_oracle(q, k, v, lens, True, 0.7, d)
    xs = [x.to(DEV).requires_grad_() for x in (q, k, v)]
    got = _grads(ops.packed_attention(*xs, _starts(lens).to(DEV), scale=0.7), xs, d.to(DEV))
    for name, g, w, b in zip(('out', 'dq', 'dk', 'dv'), got, want, bound):
        _within(g, w, b, name)


def test_packed_attention_gradient_against_differences():
    """Directional derivatives of the 64-bit definition, by central differences (their own error: h^2 and 2^-52 / h)."""
    ops = _ops()
    lens, H, Hkv, dh = [37, 1, 20], 4, 2, 24
    M = sum(lens)
    x = [_randn((M, h, dh), i) for i, h in enumerate((H, Hkv, Hkv))]
    d, dirs = _randn((M, H, dh), 7), [_randn(t.shape, 10 + i).double() for i, t in enumerate(x)]
    xs = [t.to(DEV).requires_grad_() for t in x]
    got = _grads(ops.packed_attention(*xs, _starts(lens).to(DEV)), xs, d.to(DEV))[1:]
    bounds = packed_oracle(*x, lens, True, dh ** -0.5, d)[1][1:]
    for i in range(3):
        f = []
        for h in (1e-4, -1e-4):
            y = [t.double() + (h * dirs[i] if j == i else 0) for j, t in enumerate(x)]
            outs, at = [], 0
            for n in lens:
                a, b, c = (t[at:at + n].transpose(0, 1) for t in y)
                b, c = (t.repeat_interleave(H // Hkv, 0) for t in (b, c))
                w = (a @ b.transpose(1, 2) * dh ** -0.5).masked_fill(~torch.ones(n, n, dtype=torch.bool).tril(), -math.inf)
                outs.append((torch.softmax(w, -1) @ c).transpose(0, 1))
                at += n
            f.append(float((torch.cat(outs) * d.double()).sum()))
        slope = (f[0] - f[1]) / 2e-4
        mine = float((got[i].double().cpu() * dirs[i]).sum())
        assert abs(mine - slope) <= float((bounds[i] * dirs[i].abs()).sum()) + 1e-5 * abs(slope) + 1e-5, (i, mine, slope)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_packed_attention_views_and_orders(dtype):
    """The parts of one fused projection, rows off 16-byte boundaries, a transposed layout, an expanded gradient: the same
    bits as contiguous copies."""
    ops = _ops()
    lens, H, Hkv, dh = [70, 130], 4, 2, 64
    M, st = 200, _starts([70, 130]).to(DEV)
    x = _randn((M, H + 2 * Hkv, dh), 1, dtype).to(DEV)
    q, k, v = torch.split(x, [H, Hkv, Hkv], dim=1)
    want = None
    odd = torch.empty(M * Hkv * dh + 1, dtype=dtype, device=DEV)[1:].view(M, Hkv, dh)
    odd.copy_(k)
    across = torch.empty((H, M, dh), dtype=dtype, device=DEV).transpose(0, 1)
    across.copy_(q)
    deep = torch.empty((M, Hkv, dh, 2), dtype=dtype, device=DEV)[..., 0]
    deep.copy_(v)
    ones = torch.ones((), dtype=dtype, device=DEV).expand(M, H, dh)
    for a, b, c, d in ((q.contiguous(), k.contiguous(), v.contiguous(), ones.contiguous()), (q, k, v, ones), (across, odd, deep, ones)):
        a, b, c = (t.detach().requires_grad_() for t in (a, b, c))
        got = _grads(ops.packed_attention(a, b, c, st), (a, b, c), d)
        want = want or got
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_packed_attention_rows_behind_the_last_sequence():
    """Zero outputs and gradients behind starts[-1], whatever stands there; the C entry leaves them as they were unless told."""
    from transformertts_amd import _lib
    ops = _ops()
    H, Hkv, dh, M, used = 4, 2, 64, 700, 133
    st = torch.tensor([0, 100, used], dtype=torch.int32, device=DEV)
    q, k, v, d = (_randn((M, h, dh), i).to(DEV) for i, h in enumerate((H, Hkv, Hkv, H)))
    clean = [t.clone().requires_grad_() for t in (q, k, v)]       # (as many tokens: their number decides how the keys are shared out)
    want = [t[:used] for t in _grads(ops.packed_attention(*clean, st), clean, d.clone())]
    for t in (q, k, v, d):
        t[used:] = float('nan')
    xs = [t.requires_grad_() for t in (q, k, v)]
    got = _grads(ops.packed_attention(*xs, st), xs, d)
    for g, w in zip(got, want):
        assert torch.equal(g[:used], w) and not g[used:].any()
    out = torch.full((M, H, dh), 7.0, device=DEV)
    args = [a for t in (q, k, v) for a in (t.data_ptr(), t.stride(0), t.stride(1))]
    assert _lib.lib().ttsmi_packed_attention_fwd(*args, st.data_ptr(), 2, M, H, Hkv, dh, dh ** -0.5, 1, out.data_ptr(), H * dh, dh, None, None, 0,
                                                 _lib.TTSMI_F32, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out[:used], want[0]) and bool((out[used:] == 7).all())
    none = ops.packed_attention(*(t.detach() for t in xs), torch.zeros(1, dtype=torch.int32, device=DEV))
    assert none.shape == (M, H, dh) and not none.any()
    empty = [t.detach()[:0].requires_grad_() for t in xs]
    got = _grads(ops.packed_attention(*empty, torch.zeros(3, dtype=torch.int32, device=DEV)), empty, d[:0])
    assert [tuple(g.shape) for g in got] == [(0, H, dh), (0, H, dh), (0, Hkv, dh), (0, Hkv, dh)]


def test_packed_attention_nan_stays_in_its_sequence():
    ops = _ops()
    lens, H, dh = [50, 64, 90], 2, 64
    st = _starts(lens).to(DEV)
    x = [_randn((204, H, dh), i, torch.bfloat16).to(DEV) for i in range(4)]
    clean = [t.clone().requires_grad_() for t in x[:3]]
    want = _grads(ops.packed_attention(*clean, st), clean, x[3])
    for t in x[:3]:
        t[60:100] = float('nan')
        t[101] = float('inf')
    bad = [t.requires_grad_() for t in x[:3]]
    got = _grads(ops.packed_attention(*bad, st), bad, x[3])
    for g, w in zip(got, want):
        assert torch.equal(g[:50], w[:50]) and torch.equal(g[114:], w[114:])
    # a NaN key that a causal query does not see does not reach it either
    k = clean[1].detach().clone()
    k[40:50] = float('nan')
    assert torch.equal(ops.packed_attention(clean[0].detach(), k, clean[2].detach(), st)[:40], want[0][:40])


def test_packed_attention_graph_replays_on_other_lengths():
    """Forward and backward captured once, replayed with other lengths and inputs, eager work in between; two captured graphs
    side by side keep their own workspaces."""
    ops = _ops()
    H, Hkv, dh, M = 4, 2, 64, 384
    def eager(x, d, st):
        y = [t.detach().clone().requires_grad_() for t in x]
        return [g.clone() for g in _grads(ops.packed_attention(*y, st), y, d)]
    graphs = []
    for n in range(2):
        x = [_randn((M, h, dh), 5 * n + i, torch.bfloat16).to(DEV).requires_grad_() for i, h in enumerate((H, Hkv, Hkv))]
        d, st = _randn((M, H, dh), 9 + n, torch.bfloat16).to(DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            st.copy_(_starts([100, 200, 84]))
            g0 = _grads(ops.packed_attention(*x, st), x, d)
        torch.cuda.synchronize()
        del g0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            res = _grads(ops.packed_attention(*x, st), x, d)
        graphs.append((graph, x, d, st, res))
    for lens in ([100, 200, 84], [1, 0, 383], [384, 0, 0], [10, 20, 30]):
        for n, (graph, x, d, st, res) in enumerate(graphs):
            with torch.no_grad():
                for i, t in enumerate(x):
                    t.copy_(_randn(t.shape, sum(lens) + 3 * i + n, torch.bfloat16))
            st.copy_(_starts(lens))
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, x, d, st, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, eager(x, d, st))), lens


def test_packed_attention_on_another_stream_and_twice():
    ops = _ops()
    st = _starts([300, 212]).to(DEV)
    x = [_randn((512, 4, 128), i, torch.bfloat16).to(DEV) for i in range(4)]
    def go():
        y = [t.clone().requires_grad_() for t in x[:3]]
        return _grads(ops.packed_attention(*y, st), y, x[3])
    want = go()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = go()
    again = go()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, again))


def test_packed_attention_keeps_what_the_rounding_left():
    """The forward's second output is at most half a step of the first, and dq is closer to the formula's with it than without
    (peaked scores: delta is then half of a small difference; 9 % here by arithmetic, the rounding of the score gradients and of
    dq itself stay)."""
    from transformertts_amd import _lib
    ops = _ops()
    n, H, dh = 1500, 2, 128
    q, k, v, d = (_randn((n, H, dh), 70 + i, torch.bfloat16, 1.25 if i < 2 else 1.0) for i in range(4))
    want, _ = packed_oracle(q, k, v, [n], True, dh ** -0.5, d)
    q, k, v, d, st = (t.to(DEV) for t in (q, k, v, d, _starts([n])))
    out, lse, rest = ops._packed_fwd(q, k, v, st, dh ** -0.5, True, True)
    assert rest.any() and bool((rest.float().abs() <= 2.0 ** -8 * out.float().abs() + 2.0 ** -126).all())
    off = []
    for r in (rest.data_ptr(), None):
        g = [torch.zeros_like(t) for t in (q, k, v)]
        args = lambda *ts: [a for t in ts for a in (t.data_ptr(), t.stride(0), t.stride(1))]
        ws = torch.empty(_lib.lib().ttsmi_packed_attention_bwd_ws_bytes(1, n, H, H, dh, 1) + 256, dtype=torch.uint8, device=DEV)
        assert _lib.lib().ttsmi_packed_attention_bwd(*args(q, k, v, out), r, *args(d), lse.data_ptr(), st.data_ptr(), 1, n, H, H, dh, dh ** -0.5, 1, *args(*g), 1,
                                                     ws.data_ptr(), ws.numel(), _lib.TTSMI_BF16_IO, torch.cuda.current_stream().cuda_stream) == 0
        off.append(float((g[0].double().cpu() - want[1]).norm() / want[1].norm()))
    assert off[0] < 0.98 * off[1] and off[0] < 0.003, off


def test_training_steps_of_two_threads_at_once():
    """Each on its own stream, forward and backward interleaved as they come."""
    import threading
    ops = _ops()
    freqs = torch.rand(32, dtype=torch.float64, device=DEV)
    jobs = []
    for i, lens in enumerate(([300, 212, 700], [1024, 33])):
        M = sum(lens)
        x = [_randn((M, h, 64), 10 * i + j, torch.bfloat16).to(DEV) for j, h in enumerate((8, 2, 2, 8))]
        jobs.append((x, _starts(lens).to(DEV), torch.arange(M, dtype=torch.int32, device=DEV)))
    def step(x, st, pos):
        y = [t.clone().requires_grad_() for t in x[:3]]
        q, k = ops.rotary(y[0], y[1], pos, freqs)
        return _grads(ops.packed_attention(q, k, y[2], st), y, x[3])
    want = [step(*j) for j in jobs]
    torch.cuda.synchronize()
    bad = []
    def work(n):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(15):
                got = step(*jobs[n])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[n])):
                    bad.append(n)
    threads = [threading.Thread(target=work, args=(n,)) for n in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


# ------------------------------------------------------------------------------------------------------------------ rotary
def rotary_oracle(x, positions, freqs, interleaved, scale, sign=1):
    n = 2 * len(freqs)
    y = x.double().clone()
    ang = positions.double()[:, None, None] * freqs.double()
    c, s = torch.cos(ang) * scale, torch.sin(ang) * scale * sign
    ia, ib = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    a, b = x[..., ia].double(), x[..., ib].double()
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag = torch.zeros_like(y)
    mag[..., ia], mag[..., ib] = (a.abs() + b.abs()) * scale, (a.abs() + b.abs()) * scale
    # the cosine and the sine of an angle reduced in 64 bits, each off by a few fp32 steps of 1; the two products and the sum
    return y, 12 * U * mag + HALF[x.dtype] * (y.abs() + 12 * U * mag)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('M,H,Hkv,dh,pairs', [(1, 1, 1, 2, 1), (16, 4, 4, 64, 16), (37, 6, 2, 80, 10), (5, 32, 8, 128, 64), (9, 3, 1, 192, 96),
                                              (3, 2, 1, 26, 5), (130, 5, 5, 66, 33), (4, 1, 1, 512, 256), (6, 2, 2, 64, 0)])
def test_rotary(M, H, Hkv, dh, pairs, interleaved, dtype):
    from transformertts_amd.model.transformer_utils import rotary_frequencies
    ops = _ops()
    f = torch.from_numpy(rotary_frequencies(2 * pairs)) if pairs else torch.zeros(0, dtype=torch.float64)
    pos = torch.randint(0, 1 << 20, (M,), generator=torch.Generator().manual_seed(M), dtype=torch.int32)
    pos[0] = 2 ** 31 - 1
    q, k, dq, dk = (_randn((M, h, dh), i, dtype) for i, h in enumerate((H, Hkv, H, Hkv)))
    xs = [t.to(DEV).requires_grad_() for t in (q, k)]
    out = ops.rotary(*xs, pos.to(DEV), f.to(DEV), interleaved=interleaved, scale=1.25)
    got = list(out) + list(torch.autograd.grad(out, xs, [dq.to(DEV), dk.to(DEV)]))
    for g, x, sign in zip(got, (q, k, dq, dk), (1, 1, -1, -1)):
        _within(g, *rotary_oracle(x, pos, f, interleaved, 1.25, sign), 'rotary')
    if pairs == 0:
        assert torch.equal(got[0].cpu(), q)
    with torch.no_grad():
        alone = ops.rotary(xs[0], None, pos.to(DEV), f.to(DEV), interleaved=interleaved, scale=1.25)
        assert torch.equal(alone[0], out[0]) and alone[1] is None
        here = [x.detach().clone() for x in xs]
        back = ops.rotary(*here, pos.to(DEV), f.to(DEV), interleaved=interleaved, scale=1.25, inplace=True)
        assert back[0] is here[0] and all(torch.equal(a, b) for a, b in zip(here, out))


def test_rotary_views_and_one_sided_gradient():
    ops = _ops()
    x = _randn((50, 10, 64), 3).to(DEV)
    q, k = x[:, :6], x[:, 6:8]
    f, pos = torch.rand(32, dtype=torch.float64, device=DEV), torch.arange(50, dtype=torch.int32, device=DEV)
    want = ops.rotary(q.contiguous(), k.contiguous(), pos, f)
    assert all(torch.equal(a, b) for a, b in zip(want, ops.rotary(q, k, pos, f)))
    flat = torch.empty(50 * 6 * 64 + 1, device=DEV)[1:].view(50, 6, 64).copy_(q)                  # off every wide boundary
    assert torch.equal(ops.rotary(flat, None, pos, f)[0], want[0])
    other = x.clone()
    ops.rotary(other[:, :6], other[:, 6:8], pos, f, inplace=True)
    assert torch.equal(other[:, :6], want[0]) and torch.equal(other[:, 6:8], want[1]) and torch.equal(other[:, 8:], x[:, 8:])
    kk = k.detach().clone().requires_grad_()
    d = _randn((50, 2, 64), 4).to(DEV)
    g, = torch.autograd.grad(ops.rotary(q, kk, pos, f)[1], kk, d)
    _within(g, *rotary_oracle(d.cpu(), pos.cpu(), f.cpu(), False, 1.0, -1), 'dk')


# ------------------------------------------------------------------------------------------------------------------- cache
class Paged:
    """A cache and its table on the CPU (64-bit values of what it stands for) and on the GPU."""

    def __init__(self, lens, page, heads, dh, dtype, stored, seed=0, spare=3, fill=float('nan')):
        ops = _ops()
        counts = [-(-n // page) for n in lens]
        pages = sum(counts) + spare
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        self.table = torch.full((len(lens), max(counts + [1]) + 1), -1, dtype=torch.int32)
        at = 0
        for b, c in enumerate(counts):
            self.table[b, :c] = order[at:at + c]
            at += c
        self.cache = ops.KVCache.zeros(pages, page, heads, dh, stored, DEV)
        if stored == torch.float8_e4m3fn:                               # rows that nobody wrote: NaN
            self.cache.k.view(torch.uint8).fill_(0x7f)
            self.cache.v.view(torch.uint8).fill_(0x7f)
        else:
            self.cache.k.fill_(fill)
            self.cache.v.fill_(fill)
        self.lens, self.k, self.v = lens, [], []
        starts = _starts(lens).to(DEV)
        k, v = (_randn((sum(lens), heads, dh), seed + i, dtype) for i in (1, 2))
        ops.kv_cache_write(self.cache, k.to(DEV), v.to(DEV), self.table.to(DEV), starts, torch.tensor(lens, dtype=torch.int32).to(DEV))
        if stored == torch.float8_e4m3fn:
            k, v = (quantised_oracle(x)[0] for x in (k, v))
        self.k, self.v = torch.split(k, lens), torch.split(v, lens)
        self.args = (self.table.to(DEV), None, torch.tensor(lens, dtype=torch.int32).to(DEV))


def quantised_oracle(x):
    """(values that the e4m3 rows stand for, biased exponents): the smallest power-of-two scale with |row| <= 448 scale, every
    value to the nearest multiple of its step (2^-3 of its power of two, at least 2^-9), ties to even."""
    x = x.double()
    top = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)
    e = torch.where(top > 0, (e - 9 + (m > 0.875)).clamp(min=-126), torch.zeros_like(e))
    y = torch.ldexp(x, -e)
    _, ye = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (ye - 1).clamp(min=-6) - 3)
    return torch.where(torch.isfinite(x), torch.round(y / step) * step * torch.ldexp(torch.ones_like(top), e), torch.full_like(x, float('nan'))), (e + 127).squeeze(-1)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('quantise', [False, True])
@pytest.mark.parametrize('lens,page,heads,dh', [([1], 1, 1, 8), ([5, 0, 70], 16, 2, 64), ([129, 1, 64], 64, 3, 128), ([40], 8, 4, 192), ([33, 2], 1024, 1, 24),
                                                ([2] * 130, 2, 1, 32)])
def test_cache_write_and_read(lens, page, heads, dh, quantise, dtype):
    ops = _ops()
    stored = torch.float8_e4m3fn if quantise else dtype
    p = Paged(lens, page, heads, dh, dtype, stored)
    table, _, ln = p.args
    for out_type in {dtype, torch.float32} if quantise else {dtype}:
        k, v = ops.kv_cache_read(p.cache, table, ln, _starts(lens).to(DEV), sum(lens), dtype=out_type)
        for g, w in ((k, p.k), (v, p.v)):
            assert torch.equal(g.double().cpu(), torch.cat(w).double())             # exact: one rounding, and none on the way back
    # only the rows written differ from what was there
    if not quantise:
        assert int(torch.isfinite(p.cache.k).sum()) == sum(lens) * heads * dh
    # the last tokens only, into a longer tensor whose rest stays
    n = [min(x, 3) for x in lens]
    out = [torch.full((sum(n) + 5, heads, dh), 9.0, dtype=dtype, device=DEV) for _ in 'kv']
    ops.kv_cache_read(p.cache, table, ln, _starts(n).to(DEV), sum(n) + 5, out=tuple(out))
    for g, w in zip(out, (p.k, p.v)):
        assert torch.equal(g[:sum(n)].double().cpu(), torch.cat([x[len(x) - m:] for x, m in zip(w, n)]).double()) and bool((g[sum(n):] == 9).all())
    fresh = ops.kv_cache_read(p.cache, table, ln, _starts(n).to(DEV), sum(n) + 5, dtype=dtype)[0]
    assert torch.equal(fresh[:sum(n)], out[0][:sum(n)]) and not fresh[sum(n):].any()


def test_cache_quantised_rows_at_their_borders():
    """Zeros, one value, values at and next to 448 2^e, halfway cases, tiny and huge rows, NaN and infinity."""
    ops = _ops()
    rows = [[0.0] * 8, [448.0] + [1.0] * 7, [449.0, 17.0, 18.0, 19.0, 0.5, -0.5, 464.0, 3.0], [3.5, 0.001, -0.002, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 0.0, -0.0],
            [1e-38] * 8, [2.0 ** -126, 2.0 ** -130, 0, 0, 0, 0, 0, 1e-40], [3.4e38, -1e37, 1.0, 0, 0, 0, 0, 0], [float('nan'), 2.0, 1.0, 0, 0, 0, 0, 0],
            [float('inf'), -float('inf'), 5.0, 100.0, 0, 0, 0, 0], [1.0625, 1.1875, 1.3125, -1.0625, 448.0, 432.0, 440.0, 424.0]]
    x = torch.tensor(rows).view(-1, 1, 8)
    n = len(rows)
    cache = ops.KVCache.zeros(1, 16, 1, 8, torch.float8_e4m3fn, DEV)
    table, st, ln = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([[0]], [0, n], [n]))
    ops.kv_cache_write(cache, x.to(DEV), -x.to(DEV), table, st, ln)
    want, e = quantised_oracle(x)
    k, v = ops.kv_cache_read(cache, table, ln, st, n, dtype=torch.float32)
    assert torch.equal(torch.nan_to_num(k.cpu().double(), nan=1e300), torch.nan_to_num(want.float().double(), nan=1e300))
    assert torch.equal(torch.nan_to_num(v.cpu().double(), nan=1e300), torch.nan_to_num((-want).float().double(), nan=1e300))
    assert torch.equal(cache.k_exp[0, 0, :n].cpu().long(), e.view(-1).long())


def test_cache_bad_pages_and_positions():
    """Page numbers outside the cache and tokens without a position: nothing is written, zeros are read, no row of another page
    changes."""
    ops = _ops()
    for dtype in (torch.bfloat16, torch.float8_e4m3fn):
        cache = ops.KVCache.zeros(4, 8, 2, 32, dtype, DEV)
        raw = lambda t: t.view(torch.uint8) if dtype == torch.float8_e4m3fn else t
        raw(cache.k).fill_(1)
        before = raw(cache.k).clone()
        table = torch.tensor([[4, 1], [-1, 2 ** 31 - 1], [-2 ** 31, 3]], dtype=torch.int32, device=DEV)
        st, ln = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([0, 10, 20, 24], [10, 40, 2]))
        k = _randn((24, 2, 32), 1, torch.bfloat16).to(DEV)
        ops.kv_cache_write(cache, k, k, table, st, ln)
        # sequence 0: positions 8, 9 lie in page 1; sequence 1: positions 30 .. 39 past the table; sequence 2: 2 tokens too many
        changed = (raw(cache.k) != before).flatten(2).any(-1).any(-1) if False else (raw(cache.k) != before).view(4, 2, 8, 32).any(-1).any(1)
        assert changed.nonzero().tolist() == [[1, 0], [1, 1]]
        back = ops.kv_cache_read(cache, table, ln, st, 24, dtype=torch.bfloat16)[0]
        assert not back[:8].any() and not back[10:].any() and bool(back[8:10].any())


def test_cache_offsets_past_32_bits():
    """More than 2^32 bytes of pages: the last page is written, read and attended to."""
    ops = _ops()
    page, heads, dh = 64, 8, 128
    pages = (1 << 32) // (page * heads * dh) + 40
    cache = ops.KVCache(*(torch.empty((pages, heads, page, dh), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in 'kv'),
                        *(torch.full((pages, heads, page), 127, dtype=torch.uint8, device=DEV) for _ in 'kv'))
    n = 100
    table, st, ln = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([[pages - 1, pages - 30]], [0, n], [n]))
    k, v, q = (_randn((n, h, dh), i, torch.bfloat16) for i, h in enumerate((heads, heads, 16)))
    ops.kv_cache_write(cache, k.to(DEV), v.to(DEV), table, st, ln)
    back = ops.kv_cache_read(cache, table, ln, st, n)
    kq, vq = quantised_oracle(k)[0], quantised_oracle(v)[0]
    assert torch.equal(back[0].double().cpu(), kq) and torch.equal(back[1].double().cpu(), vq)
    want, bound = attention_oracle(q, kq, vq, 0, True, dh ** -0.5, torch.bfloat16)
    _within(ops.paged_attention(q.to(DEV), cache, table, st, ln), want[0], bound[0], 'out')


# --------------------------------------------------------------------------------------------------------- paged attention
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('quantise', [False, True])
@pytest.mark.parametrize('new,lens,page,H,Hkv,dh', [
    ([1], [1], 16, 1, 1, 8), ([1] * 5, [1, 700, 64, 65, 1023], 16, 8, 2, 128), ([1, 1], [5000, 3], 64, 4, 4, 64), ([1, 1, 1], [300, 17, 90], 8, 32, 2, 64),
    ([70, 1, 200], [300, 513, 200], 32, 4, 2, 64), ([129], [129], 1, 2, 1, 192), ([3, 0, 40], [1000, 20, 1040], 128, 6, 3, 80), ([17] * 9, [17 + 31 * i for i in range(9)], 16, 16, 2, 128),
    ([2, 3, 1, 4], [2000, 999, 640, 641], 64, 8, 1, 192), ([1] * 150, [1 + 7 * i for i in range(150)], 8, 4, 2, 32), ([1], [20000], 64, 2, 1, 64),
    ([300], [310], 16, 512, 32, 8), ([40, 90], [700, 90], 32, 4, 2, 24)])
def test_paged_attention(new, lens, page, H, Hkv, dh, quantise, dtype):
    from transformertts_amd import _lib
    ops = _ops()
    p = Paged(lens, page, Hkv, dh, dtype, torch.float8_e4m3fn if quantise else dtype)
    q = _randn((sum(new), H, dh), 9, dtype, 1.5)
    table, _, ln = p.args
    st = _starts(new).to(DEV)
    got = ops.paged_attention(q.to(DEV), p.cache, table, st, ln)
    at = 0
    want, bound = [], []
    for b, n in enumerate(new):
        w, e = attention_oracle(q[at:at + n], p.k[b], p.v[b], lens[b] - n, True, dh ** -0.5, dtype)
        want.append(w[0])
        bound.append(e[0])
        at += n
    want, bound = torch.cat(want), torch.cat(bound)
    _within(got, want, bound, 'out')
    assert torch.equal(got, ops.paged_attention(q.to(DEV), p.cache, table, st, ln))
    rows = sum(new) * (H // Hkv) <= (16 if p.cache.k.element_size() == 2 else 64) * len(new) and dh * p.cache.k.element_size() % 16 == 0
    assert _lib.lib().ttsmi_last_kernel() == (b'paged_rows_kernel' if rows else b'seq_attn_fwd_kernel')


def test_paged_attention_rows_that_see_nothing_and_bad_pages():
    ops = _ops()
    p = Paged([40, 6], 8, 2, 64, torch.float32, torch.float32)
    table, _, _ = p.args
    q = _randn((9, 4, 64), 1).to(DEV)
    st, ln = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([0, 5, 7], [3, 0]))
    for H in (4, 64):                                          # few rows a sequence, and many
        q = _randn((9, H, 64), 1).to(DEV)
        got = ops.paged_attention(q, p.cache, table, st, ln)
        # sequence 0 has 3 cached tokens and 5 queries: the first two stand before position 0; sequence 1 is empty; two rows behind
        assert not got[:2].any() and not got[5:].any()
        want, bound = attention_oracle(q[2:5].cpu(), p.k[0][:3], p.v[0][:3], 0, True, 0.125, torch.float32)
        _within(got[2:5], want[0], bound[0], 'out')
        out = torch.full_like(q, 5.0)
        back = ops.paged_attention(q, p.cache, table, st, ln, out=out)
        assert back is out and torch.equal(out[:7], got[:7]) and bool((out[7:] == 5).all())
    bad = table.clone()
    bad[0, 1] = 10 ** 6                                        # positions 8 .. 15 read as zeros
    st, ln = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([0, 1, 2], [40, 6]))
    k, v = p.k[0].clone(), p.v[0].clone()
    k[8:16], v[8:16] = 0, 0
    want, bound = attention_oracle(q[:1].cpu(), k, v, 39, True, 0.125, torch.float32)
    _within(ops.paged_attention(q[:2].contiguous(), p.cache, bad, st, ln)[:1], want[0], bound[0], 'out')
    # lens past what the table holds: those positions hold no key, however far they reach
    want, bound = attention_oracle(q[:1].cpu(), p.k[0][:16], p.v[0][:16], 39, True, 0.125, torch.float32)
    for length in (40, 2 ** 31 - 1):
        ln[0] = length
        _within(ops.paged_attention(q[:2].contiguous(), p.cache, table[:, :2].contiguous(), st, ln)[:1], want[0], bound[0], 'out')
        wide = q[:1].expand(64, 64, 64).contiguous()           # the form for many rows: 64 new tokens, the last one here
        many = torch.tensor([0, 64], dtype=torch.int32, device=DEV)
        got = ops.paged_attention(wide, p.cache, table[:1, :2].contiguous(), many, ln[:1] + (24 if length == 40 else 0))[-1:]
        _within(got, want[0], bound[0], 'out')


@pytest.mark.parametrize('H', [4, 64])
def test_cache_without_pages_or_table(H):
    """A cache of no pages, and a table of no columns: nothing is written, zeros are read, and attention gives zeros."""
    ops = _ops()
    st, ln = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([0, 3, 40], [9, 37]))
    for dtype in (torch.bfloat16, torch.float8_e4m3fn):
        for pages, width in ((0, 3), (2, 0)):
            cache = ops.KVCache.zeros(pages, 8, 2, 64, dtype, DEV)
            table = torch.zeros((2, width), dtype=torch.int32, device=DEV)
            k = _randn((40, 2, 64), 1, torch.bfloat16).to(DEV)
            ops.kv_cache_write(cache, k, k, table, st, ln)
            assert not any(t.any() for t in ops.kv_cache_read(cache, table, ln, st, 40, dtype=torch.bfloat16))
            assert not ops.paged_attention(_randn((40, H, 64), 2, torch.bfloat16).to(DEV), cache, table, st, ln).any()


def test_paged_attention_missing_page_beside_any_exponents():
    """A page that is not there reads as zeros, whatever the bytes of the page that stands in for it."""
    ops = _ops()
    for H in (4, 64):
        q = _randn((1, H, 64), 3, torch.bfloat16)
        p = Paged([40], 8, 2, 64, torch.bfloat16, torch.float8_e4m3fn)
        table = p.args[0]
        st, ln = torch.tensor([0, 1], dtype=torch.int32, device=DEV), torch.tensor([40], dtype=torch.int32, device=DEV)
        table = table.clone()
        first = table == 0
        spare = torch.cat([p.cache.k.view(torch.uint8), p.cache.k.view(torch.uint8)[:1]]), torch.cat([p.cache.v.view(torch.uint8), p.cache.v.view(torch.uint8)[:1]])
        exps = [torch.cat([e, e[:1]]) for e in (p.cache.k_exp, p.cache.v_exp)]
        table[first] = len(spare[0]) - 1                         # page 0 moves behind the last, and nobody names it any more
        for e in exps:
            e[0] = 255
        cache = ops.KVCache(*(t.view(torch.float8_e4m3fn) for t in spare), *exps)
        table[0, 1] = -1
        k, v = p.k[0].clone(), p.v[0].clone()
        k[8:16], v[8:16] = 0, 0
        want, bound = attention_oracle(q, k, v, 39, True, 0.125, torch.bfloat16)
        _within(ops.paged_attention(q.to(DEV), cache, table, st, ln), want[0], bound[0], 'out')


def test_tokens_in_front_of_the_first_sequence():
    """They belong to no sequence: zeros out, zero gradients, nothing of them in the others; in a given output they stay."""
    ops = _ops()
    front, lens, M, dh = 150, [40, 133], 400, 64
    st = _starts(lens).to(DEV) + front
    for dtype, H, Hkv in ((torch.bfloat16, 4, 2), (torch.float32, 6, 1)):
        x = [_randn((M, h, dh), i, dtype).to(DEV) for i, h in enumerate((H, Hkv, Hkv, H))]
        own = slice(front, front + 173)
        clean = [t[own].clone().requires_grad_() for t in x[:3]]
        want = _grads(ops.packed_attention(*clean, st - front), clean, x[3][own].clone())
        for t in x:
            t[:front], t[front + 173:] = float('nan'), float('nan')
        xs = [t.requires_grad_() for t in x[:3]]
        for g, w in zip(_grads(ops.packed_attention(*xs, st), xs, x[3]), want):
            assert torch.equal(g[own], w) and not g[:front].any() and not g[front + 173:].any()
    p = Paged([40, 133], 16, 2, 64, torch.bfloat16, torch.bfloat16)
    table, _, ln = p.args
    st0 = st - front
    for t, w in zip(ops.kv_cache_read(p.cache, table, ln, st, M), ops.kv_cache_read(p.cache, table, ln, st0, 173)):
        assert torch.equal(t[own], w) and not t[:front].any() and not t[front + 173:].any()
    for H in (4, 64):
        q = _randn((M, H, 64), 5, torch.bfloat16).to(DEV)
        got, want = ops.paged_attention(q, p.cache, table, st, ln), ops.paged_attention(q[own].contiguous(), p.cache, table, st0, ln)
        assert not got[:front].any() and not got[front + 173:].any()
        # (the keys may be split elsewhere: fp32 sums in another order, then one rounding to bf16, a step at most between them)
        assert bool(((got[own].float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 2.0 ** -16).all())


def test_starts_that_overlap_stay_in_range():
    """Not a valid call - but every access is bounded by the token count and the workspace, and it ends: the rows are whatever
    they are, memory on both sides of the outputs stays as it was."""
    ops = _ops()
    M, H, Hkv, dh, B = 300, 8, 2, 64, 65
    st = torch.tensor([(0 if b % 2 == 0 else M) for b in range(B + 1)], dtype=torch.int32, device=DEV)
    x = [_randn((M, h, dh), i, torch.bfloat16).to(DEV) for i, h in enumerate((H, Hkv, Hkv, H))]
    _grads(ops.packed_attention(*[t.requires_grad_() for t in x[:3]], st), x[:3], x[3])
    p = Paged([700] * B, 64, Hkv, dh, torch.bfloat16, torch.bfloat16)
    table, _, ln = p.args
    guarded = torch.full((M + 200, H, dh), 3.0, dtype=torch.bfloat16, device=DEV)
    for new in (40, M):
        ops.paged_attention(x[0][:new].detach().contiguous(), p.cache, table, st.clamp(max=new), ln, out=guarded[100:100 + new])
        assert bool((guarded[:100] == 3).all()) and bool((guarded[100 + new:] == 3).all())
    torch.cuda.synchronize()


def test_rows_too_far_apart_and_broadcast_destinations():
    from transformertts_amd import _lib
    ops = _ops()
    st = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    q, k, v = (_randn((3, h, 64), i, torch.bfloat16).to(DEV) for i, h in enumerate((4, 2, 2)))
    far = torch.zeros(2 * (1 << 25) + 256, dtype=torch.bfloat16, device=DEV).as_strided((3, 4, 64), (1 << 25, 64, 1))
    far.copy_(q)
    assert torch.equal(ops.packed_attention(far, k, v, st), ops.packed_attention(q, k, v, st))
    one = q[:1].expand(3, 4, 64)
    pos, freqs = torch.arange(3, dtype=torch.int32, device=DEV), torch.ones(32, dtype=torch.float64, device=DEV)
    cache = ops.KVCache.zeros(2, 8, 2, 64, torch.bfloat16, DEV)
    table, ln = torch.zeros((1, 1), dtype=torch.int32, device=DEV), torch.tensor([3], dtype=torch.int32, device=DEV)
    for call in (lambda: ops.rotary(one, k, pos, freqs, inplace=True), lambda: ops.rotary(q, k[:, :1].expand(3, 2, 64), pos, freqs, inplace=True),
                 lambda: ops.paged_attention(q, cache, table, st, ln, out=one), lambda: ops.kv_cache_read(cache, table, ln, st, 3, out=(k, one[:, :2])),
                 lambda: ops.KVCache(cache.k, cache.k)):
        with pytest.raises(_lib.TtsmiError):
            call()
    w = torch.ones((64, 8), device=DEV, requires_grad=True)
    x = _randn((3, 2, 64), 7).to(DEV)
    y = (x @ w).sum()
    ops.rotary(x, None, pos, freqs, inplace=True)               # what the product saved has changed: its gradient is refused, not wrong
    with pytest.raises(RuntimeError):
        y.backward()


def test_paged_attention_graph_replay_decodes_on():
    """One captured decoding step - rotary, cache write, attention - replayed as the sequences grow, against the eager calls."""
    ops = _ops()
    H, Hkv, dh, B = 8, 2, 64, 3
    f = torch.rand(32, dtype=torch.float64, device=DEV)
    def world():
        p = Paged([30, 1, 77], 16, Hkv, dh, torch.bfloat16, torch.float8_e4m3fn, spare=30)
        table = torch.arange(B * 10, dtype=torch.int32, device=DEV).view(B, 10)
        fresh = ops.KVCache.zeros(B * 10, 16, Hkv, dh, torch.float8_e4m3fn, DEV)
        k, v = ops.kv_cache_read(p.cache, p.args[0], p.args[2], _starts(p.lens).to(DEV), 108)
        ops.kv_cache_write(fresh, k, v, table, _starts(p.lens).to(DEV), p.args[2])
        return fresh, table, p.args[2].clone(), _starts([1] * B).to(DEV)
    x = [torch.zeros((B, h, dh), dtype=torch.bfloat16, device=DEV) for h in (H, Hkv, Hkv)]
    def step(cache, table, ln, st):
        ln += 1
        q, k = ops.rotary(x[0], x[1], ln - 1, f)
        ops.kv_cache_write(cache, k, x[2], table, st, ln)
        return ops.paged_attention(q, cache, table, st, ln)
    a, b = world(), world()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(*world())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        res = step(*a)
    for i in range(6):
        for j, t in enumerate(x):
            t.copy_(_randn(t.shape, 40 + 3 * i + j, torch.bfloat16))
        graph.replay()
        want = step(*b)
        torch.cuda.synchronize()
        assert torch.equal(res, want) and torch.equal(a[0].k_exp, b[0].k_exp), i


# ----------------------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize('stored', [torch.bfloat16, torch.float8_e4m3fn])
def test_prompt_then_chunks_then_single_tokens(stored):
    """The operators as they are used together: rotary positions, the prompts through packed attention while their keys and
    values go into the cache, then a chunk, then single tokens over the cache - against the 64-bit definition on the whole
    sequences (from the turned and stored values that the operators return)."""
    from transformertts_amd.model.transformer_utils import rotary_frequencies
    ops = _ops()
    H, Hkv, dh, page, dtype = 8, 2, 64, 16, torch.bfloat16
    f = torch.from_numpy(rotary_frequencies(dh, scaling='bands', factor=8.0)).to(DEV)
    B, steps = 3, [[50, 7, 129], [40, 1, 3], [1, 1, 1], [1, 1, 1]]
    cache = ops.KVCache.zeros(60, page, Hkv, dh, stored, DEV)
    table = torch.randperm(60, generator=torch.Generator().manual_seed(1)).to(torch.int32)[:B * 20].view(B, 20).to(DEV)
    lens = [0] * B
    seen_q = [[] for _ in range(B)]
    for i, new in enumerate(steps):
        M, st = sum(new), _starts(new).to(DEV)
        lens = [a + b for a, b in zip(lens, new)]
        ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
        q, k, v = (t.to(DEV) for t in torch.split(_randn((M, H + 2 * Hkv, dh), 20 + i, dtype), [H, Hkv, Hkv], 1))
        pos = torch.cat([torch.arange(a - n, a) for a, n in zip(lens, new)]).to(torch.int32).to(DEV)
        q, k = ops.rotary(q, k, pos, f)
        ops.kv_cache_write(cache, k, v, table, st, ln)
        out = ops.packed_attention(q, k, v, st) if i == 0 else ops.paged_attention(q, cache, table, st, ln)
        kk, vv = ops.kv_cache_read(cache, table, ln, _starts(lens).to(DEV), sum(lens), dtype=dtype)
        at, base = 0, 0
        for b, n in enumerate(new):
            # (the prompt is attended to as it is, before it is quantised)
            K, V = (t[base:base + lens[b]].cpu() for t in (kk, vv)) if i else (t[at:at + n].cpu() for t in (k, v))
            want, bound = attention_oracle(q[at:at + n].cpu(), K, V, lens[b] - n, True, dh ** -0.5, dtype)
            _within(out[at:at + n], want[0], bound[0], f'step {i}, sequence {b}')
            at, base = at + n, base + lens[b]

"""-m gpu tests of the sequence operators' calls beside other work of the process: steps of other threads, autograd, caches whose
tensors change."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def _ops():
    from transformertts_amd import ops
    return ops


def _randn(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _calls(ops, x):
    """Every entry point on x = (q, k, v, dout), results in one list."""
    q, k, v, d = x
    n = len(q)
    st, ln, table, pos = _ints([0, n]), _ints([n]), _ints([[1, 0]]), torch.arange(n, dtype=torch.int32, device=DEV)
    freqs = torch.linspace(1.0, 0.1, 32, dtype=torch.float64).to(DEV)
    cache = ops.KVCache.zeros(2, 64, k.shape[1], 64, torch.bfloat16, DEV)

    def run():
        y = [t.detach().requires_grad_() for t in (q, k, v)]
        a, b = ops.rotary(y[0], y[1], pos, freqs)
        out = ops.packed_attention(a, b, y[2], st)
        grads = torch.autograd.grad(out, y, d)
        with torch.no_grad():
            ops.kv_cache_write(cache, b, v, table, st, ln)
            return [a, b, out, *grads, ops.paged_attention(a, cache, table, st, ln), *ops.kv_cache_read(cache, table, ln, st, n)]
    return run


def test_a_pinned_step_of_another_thread_beside_a_graph():
    """While another thread pins a stream of its own, a capture here holds every launch of the calls made here: its replays
    give what new inputs ask for."""
    ops = _ops()
    x = [_randn((100, h, 64), i, torch.bfloat16) for i, h in enumerate((4, 2, 2, 4))]
    run = _calls(ops, x)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    inside, leave = threading.Event(), threading.Event()

    def step():
        with torch.cuda.stream(other), ops.pinned_stream():
            inside.set()
            leave.wait(60)
    thread = threading.Thread(target=step)
    thread.start()
    try:
        assert inside.wait(60)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            res = run()
    finally:
        leave.set()
        thread.join()
    for seed in (10, 20, 30):
        for i, t in enumerate(x):
            t.copy_(_randn(t.shape, seed + i, torch.bfloat16))
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, want))


def test_calls_on_a_device_that_is_not_the_current_one(monkeypatch):
    """The way through a change of the device (to the same one here: that is all a test machine has), forward and backward."""
    ops = _ops()
    run = _calls(ops, [_randn((100, h, 64), i, torch.bfloat16) for i, h in enumerate((4, 2, 2, 4))])
    want, asked = run(), []

    def current():
        asked.append(1)
        return -1 if len(asked) % 2 else 0
    monkeypatch.setattr(ops, '_current_device', current)
    got = run()
    assert len(asked) == 10 and all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_saved_tensor_that_was_written_is_refused_not_used():
    """A tensor that a product keeps for its gradient, then handed to an operator as its output: the gradient is refused."""
    ops = _ops()
    cache = ops.KVCache.zeros(2, 16, 2, 64, torch.float32, DEV)
    st, ln, table = _ints([0, 3]), _ints([3]), _ints([[0]])
    q, k = _randn((3, 4, 64), 1), _randn((3, 2, 64), 2)
    w = torch.ones((64, 8), device=DEV, requires_grad=True)
    for out, write in ((torch.zeros_like(q), lambda t: ops.paged_attention(q, cache, table, st, ln, out=t)),
                       (torch.zeros_like(k), lambda t: ops.kv_cache_read(cache, table, ln, st, 3, out=(t, torch.zeros_like(k)))),
                       (torch.zeros_like(k), lambda t: ops.kv_cache_read(cache, table, ln, st, 3, out=(torch.zeros_like(k), t))),
                       (cache.k, lambda t: ops.kv_cache_write(cache, k, k, table, st, ln)), (cache.v, lambda t: ops.kv_cache_write(cache, k, k, table, st, ln))):
        y = (out @ w).sum()
        write(out)
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            y.backward()


def test_rotary_differentiated_twice():
    """The gradient is linear in the incoming one: its own gradient is the turn itself, to the same bits."""
    ops = _ops()
    q, k, dq, dk, wq, wk = (_randn((37, h, 64), i, torch.bfloat16) for i, h in enumerate((4, 2) * 3))
    pos, freqs = torch.arange(37, dtype=torch.int32, device=DEV), torch.linspace(1.0, 0.1, 16, dtype=torch.float64).to(DEV)
    for t in (q, k, dq, dk):
        t.requires_grad_()
    out = ops.rotary(q, k, pos, freqs, scale=1.5)
    grads = torch.autograd.grad(out, (q, k), (dq, dk), create_graph=True)
    once = torch.autograd.grad(out, (q, k), (dq, dk), retain_graph=True)
    again = torch.autograd.grad(grads, (dq, dk), (wq, wk), retain_graph=True)
    want = ops.rotary(wq, wk, pos, freqs, scale=1.5)
    assert all(torch.equal(a, b) for a, b in zip([*grads, *again], [*once, *want]))
    only, = torch.autograd.grad(grads[1], dk, wk)
    assert torch.equal(only, want[1])


def test_attention_differentiated_twice_is_refused():
    from transformertts_amd import _lib
    ops = _ops()
    x = [_randn((37, h, 64), i, torch.bfloat16).requires_grad_() for i, h in enumerate((4, 2, 2))]
    out = ops.packed_attention(*x, _ints([0, 30, 37]))
    grads = torch.autograd.grad(out.sum(), x, create_graph=True)
    once = torch.autograd.grad(out.sum(), x)
    assert all(torch.equal(a, b) for a, b in zip(grads, once))
    with pytest.raises(_lib.TtsmiError, match='second derivatives'):
        torch.autograd.grad(sum((g.float() ** 2).sum() for g in grads), x)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float8_e4m3fn])
def test_growing_a_cache(dtype):
    """Larger pages are a new cache: the old rows copied, both read as before; the tensors of a cache are not exchanged."""
    ops = _ops()
    old = ops.KVCache.zeros(2, 16, 2, 64, dtype, DEV)
    st, ln, table = _ints([0, 20]), _ints([20]), _ints([[1, 0]])
    q, k, v = (_randn((20, h, 64), i, torch.bfloat16) for i, h in enumerate((4, 2, 2)))
    ops.kv_cache_write(old, k, v, table, st, ln)
    want = ops.paged_attention(q, old, table, st, ln)
    with pytest.raises(AttributeError):
        old.k = torch.zeros_like(old.k)
    grown = ops.KVCache.zeros(5, 16, 2, 64, dtype, DEV)
    for name in ('k', 'v', 'k_exp', 'v_exp'):
        a, b = getattr(old, name), getattr(grown, name)
        if a is not None:
            b.view(torch.uint8)[:2].copy_(a.view(torch.uint8))
    import copy
    twin = copy.deepcopy(old)
    assert twin.k.data_ptr() != old.k.data_ptr() == old.args[0]
    for cache in (grown, old, twin):
        assert torch.equal(ops.paged_attention(q, cache, table, st, ln), want)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('lens,H,Hkv', [([61], 2, 2), ([193], 1, 1), ([200], 2, 1), ([61], 16, 1), ([130, 0, 400, 1], 8, 2), ([129] * 7, 16, 4), ([1500], 4, 1), ([5, 700, 3], 32, 2)])
def test_backward_stays_in_its_workspace(lens, H, Hkv, causal, dtype):
    """No byte behind the size asked for, with splits and without; the gradients are the ones that a far larger batch's workspace
    gives (which division of the rows is made goes by the tokens, not by the workspace)."""
    from transformertts_amd import _lib
    ops, dh = _ops(), 64
    M, B = sum(lens), len(lens)
    q, k, v, d = (_randn((M, h, dh), i, dtype) for i, h in enumerate((H, Hkv, Hkv, H)))
    st = _ints([0] + torch.tensor(lens).cumsum(0).tolist())
    out, lse, rest = ops._packed_fwd(q, k, v, st, 0.125, causal, True)
    need = _lib.lib().ttsmi_packed_attention_bwd_ws_bytes(B, M, H, Hkv, dh, int(causal))
    args = lambda *ts: [a for t in ts for a in (t.data_ptr(), t.stride(0), t.stride(1))]
    want = None
    for ws_bytes, fill in ((need, 0x7f), (need, 0xff), (need + (1 << 20), 0x55)):
        ws = torch.full((ws_bytes + 4096,), fill, dtype=torch.uint8, device=DEV)
        g = [torch.full_like(t, float('nan')) for t in (q, k, v)]
        assert _lib.lib().ttsmi_packed_attention_bwd(*args(q, k, v, out), None if rest is None else rest.data_ptr(), *args(d), lse.data_ptr(), st.data_ptr(), B, M, H, Hkv,
                                                     dh, 0.125, int(causal), *args(*g), 1, ws.data_ptr(), ws_bytes, ops._SEQ_DTYPES[dtype],
                                                     torch.cuda.current_stream().cuda_stream) == 0
        assert bool((ws[need:] == fill).all()) and all(bool(torch.isfinite(t).all()) for t in g)
        want = want or g
        assert all(torch.equal(a, b) for a, b in zip(g, want))


@pytest.mark.parametrize('new,lens,H,Hkv,page', [([1] * 3, [900, 33, 4000], 8, 2, 16), ([200, 5], [2000, 5], 16, 2, 8), ([70], [70], 4, 4, 64), ([300], [3000], 8, 1, 4)])
@pytest.mark.parametrize('dtype,stored', [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float8_e4m3fn), (torch.float32, torch.float32)])
def test_attention_into_its_own_queries(new, lens, H, Hkv, page, dtype, stored):
    """out = q, split keys and whole ones: the same bits as into a tensor of its own, rows of no sequence left as they were."""
    ops, dh = _ops(), 64
    counts = [-(-n // page) for n in lens]
    cache = ops.KVCache.zeros(sum(counts), page, Hkv, dh, stored, DEV)
    order = torch.randperm(sum(counts), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    table, at = torch.full((len(lens), max(counts)), -1, dtype=torch.int32), 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    table, ln, total = table.to(DEV), _ints(lens), sum(lens)
    ops.kv_cache_write(cache, *(_randn((total, Hkv, dh), i, dtype) for i in (1, 2)), table, _ints([0] + torch.tensor(lens).cumsum(0).tolist()), ln)
    st = _ints([0] + torch.tensor(new).cumsum(0).tolist())
    fused = _randn((sum(new) + 3, H + 2, dh), 3, dtype)
    q = fused[:, 1:H + 1]
    before, want = fused.clone(), ops.paged_attention(q, cache, table, st, ln)
    assert ops.paged_attention(q, cache, table, st, ln, out=q) is q
    assert torch.equal(q[:sum(new)], want[:sum(new)]) and torch.equal(q[sum(new):], before[sum(new):, 1:H + 1])
    assert torch.equal(fused[:, 0], before[:, 0]) and torch.equal(fused[:, -1], before[:, -1])

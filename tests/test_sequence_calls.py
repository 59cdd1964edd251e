"""CPU-side checks of what the host mirror of the sequence operators does around its launches: the stream that they go to, what
autograd is told, and which calls it refuses.  A recorder stands in for the library, and CPU tensors say that they are on a GPU:
nothing is launched."""
import threading

import pytest
import torch


class OnGpu(torch.Tensor):
    is_cuda = True

    def get_device(self):
        return 0


def _t(*shape, dtype=torch.float32, fill=1.0, grad=False):
    return torch.full(shape, fill, dtype=dtype).as_subclass(OnGpu).requires_grad_(grad)


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32).as_subclass(OnGpu)


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if name.endswith('_ws_bytes'):
            return lambda *a: 256

        def call(*a):
            self.calls.append((name, a))
            return 0
        return call


@pytest.fixture
def world(monkeypatch):
    """(ops, the recorder): the current device is 0, and every thread's current stream is its own number."""
    from transformertts_amd import _lib, ops
    rec = Recorder()
    monkeypatch.setattr(_lib, 'lib', lambda: rec)
    monkeypatch.setattr(ops, '_current_device', lambda: 0)
    monkeypatch.setattr(ops, '_raw_stream', lambda index: threading.get_ident())
    yield ops, rec
    ops._packed_bwd_ws.cache_clear()                       # (the recorder's sizes)
    ops._paged_ws.cache_clear()


def _every_call(ops):
    """One call of each entry point, by name."""
    q, k, v, cache = _t(3, 2, 8), _t(3, 1, 8), _t(3, 1, 8), _cache(ops)
    st, ln, table, pos, freqs = _ints(0, 3), _ints(3), _ints(0).view(1, 1), _ints(0, 1, 2), _t(4, dtype=torch.float64)

    def training_step():
        x = [t.detach().requires_grad_() for t in (q, k, v)]
        a, b = (t.as_subclass(OnGpu) for t in ops.rotary(x[0], x[1], pos, freqs))
        torch.autograd.grad(ops.packed_attention(a, b, x[2], st), x, torch.ones(3, 2, 8))
    return {'rotary': lambda: ops.rotary(q, k, pos, freqs), 'rotary in place': lambda: ops.rotary(q, k, pos, freqs, inplace=True),
            'packed_attention': lambda: ops.packed_attention(q, k, v, st), 'training step': training_step,
            'kv_cache_write': lambda: ops.kv_cache_write(cache, k, v, table, st, ln),
            'kv_cache_read': lambda: ops.kv_cache_read(cache, table, ln, st, 3, out=(_t(3, 1, 8), _t(3, 1, 8))),
            'paged_attention': lambda: ops.paged_attention(q, cache, table, st, ln)}


def _cache(ops, dtype=torch.float32):
    exp = () if dtype != torch.float8_e4m3fn else (_t(2, 1, 4, dtype=torch.uint8), _t(2, 1, 4, dtype=torch.uint8))
    pages = [torch.zeros(2, 1, 4, 8, dtype=torch.uint8).view(dtype) if exp else torch.zeros(2, 1, 4, 8, dtype=dtype) for _ in 'kv']
    return ops.KVCache(*(t.as_subclass(OnGpu) for t in pages), *exp)


class _InAnotherThread:
    """`with _InAnotherThread(context):` - the context is entered by another thread and left by it at the end."""

    def __init__(self, context):
        self.context, self.inside, self.leave = context, threading.Event(), threading.Event()

    def _run(self):
        with self.context:
            self.inside.set()
            self.leave.wait(60)

    def __enter__(self):
        self.thread = threading.Thread(target=self._run)
        self.thread.start()
        assert self.inside.wait(60)
        return self

    def __exit__(self, *exc):
        self.leave.set()
        self.thread.join()
        return False


NAMES = ['rotary', 'rotary in place', 'packed_attention', 'training step', 'kv_cache_write', 'kv_cache_read', 'paged_attention']


@pytest.mark.parametrize('name', NAMES)
def test_launches_go_to_the_calling_threads_stream(world, name):
    """A training step of another thread pins ITS stream for as long as it takes; a call made meanwhile stays on its own."""
    ops, rec = world
    with _InAnotherThread(ops.pin_stream(99)):
        _every_call(ops)[name]()
    assert len(rec.calls) == (4 if name == 'training step' else 1) and all(a[-1] == threading.get_ident() for _, a in rec.calls)


@pytest.mark.parametrize('name', NAMES)
def test_a_call_on_another_device_leaves_another_threads_pin_alone(world, monkeypatch, name):
    """The step of the other thread keeps its pinned stream during the call, and no stream of an ended step is put back after it."""
    ops, rec = world
    import contextlib
    step = _InAnotherThread(ops.pin_stream(99))
    here, seen = [1], []

    @contextlib.contextmanager
    def device(d):
        here[0] = 0
        seen.append(ops._PINNED_STREAM)
        yield
        if step.thread.is_alive():                         # the step ends while the call runs
            step.__exit__()
        here[0] = 1
    monkeypatch.setattr(torch.cuda, 'device', device)
    monkeypatch.setattr(ops, '_current_device', lambda: here[0])
    launch = rec.__class__.__getattr__

    def watched(self, n):
        f = launch(self, n)

        def call(*a):
            seen.append(ops._PINNED_STREAM)
            return f(*a)
        return call
    monkeypatch.setattr(Recorder, '__getattr__', watched)
    with step:
        _every_call(ops)[name]()
    assert rec.calls and seen[0] == 99 and (name == 'training step' or set(seen) == {99})
    assert ops._PINNED_STREAM is None


def _versions(*ts):
    return [t._version for t in ts]


@pytest.mark.parametrize('dtype', [torch.float32, torch.float8_e4m3fn])
def test_autograd_is_told_of_every_tensor_written(world, dtype):
    ops, _ = world
    cache = _cache(ops, dtype)
    q, k, v = _t(3, 2, 8), _t(3, 1, 8), _t(3, 1, 8)
    st, ln, table = _ints(0, 3), _ints(3), _ints(0).view(1, 1)
    written = [t for t in (cache.k, cache.v, cache.k_exp, cache.v_exp) if t is not None]
    before = _versions(*written)
    ops.kv_cache_write(cache, k, v, table, st, ln)
    assert all(a < b for a, b in zip(before, _versions(*written)))
    before, outs = _versions(*written), (_t(3, 1, 8), _t(3, 1, 8), _t(3, 2, 8))
    ops.kv_cache_read(cache, table, ln, st, 3, out=outs[:2])
    ops.paged_attention(q, cache, table, st, ln, out=outs[2])
    assert all(n > 0 for n in _versions(*outs)) and _versions(*written) == before and _versions(q, k, v) == [0, 0, 0]
    with torch.inference_mode():                           # (tensors of no version take the same way)
        ops.paged_attention(q, cache, table, st, ln, out=_t(3, 2, 8))


def test_gradients_that_would_be_dropped_are_refused(world):
    """Keys, pages, outputs and frequencies that want a gradient no operator gives; without grad mode the calls go through."""
    from transformertts_amd import _lib
    ops, rec = world
    q, k, v = _t(3, 2, 8), _t(3, 1, 8), _t(3, 1, 8)
    st, ln, table, pos, freqs = _ints(0, 3), _ints(3), _ints(0).view(1, 1), _ints(0, 1, 2), _t(4, dtype=torch.float64)
    cache, learned = _cache(ops), ops.KVCache(*(torch.zeros(2, 1, 4, 8).as_subclass(OnGpu).requires_grad_() for _ in 'kv'))
    g = dict(q=_t(3, 2, 8, grad=True), k=_t(3, 1, 8, grad=True), freqs=_t(4, dtype=torch.float64, grad=True))
    calls = [lambda: ops.kv_cache_write(cache, g['k'], v, table, st, ln), lambda: ops.kv_cache_write(cache, k, g['k'], table, st, ln),
             lambda: ops.kv_cache_write(learned, k, v, table, st, ln), lambda: ops.kv_cache_read(learned, table, ln, st, 3, out=(_t(3, 1, 8), _t(3, 1, 8))),
             lambda: ops.kv_cache_read(cache, table, ln, st, 3, out=(g['k'], _t(3, 1, 8))), lambda: ops.kv_cache_read(cache, table, ln, st, 3, out=(_t(3, 1, 8), g['k'])),
             lambda: ops.paged_attention(g['q'], cache, table, st, ln), lambda: ops.paged_attention(q, learned, table, st, ln),
             lambda: ops.paged_attention(q, cache, table, st, ln, out=g['q']), lambda: ops.rotary(q, k, pos, g['freqs']),
             lambda: ops.rotary(q, k, pos, g['freqs'], inplace=True), lambda: ops.rotary(g['q'], k, pos, g['freqs'])]
    for call in calls:
        with pytest.raises(_lib.TtsmiError, match='gradient'):
            call()
    assert not rec.calls
    with torch.no_grad():
        for call in calls:
            call()
    assert len(rec.calls) == len(calls)


def test_second_derivatives_of_attention_are_refused(world):
    """A penalty on a gradient is refused, not given without a term - however the gradient is asked for, and also where the loss is
    linear in the output; create_graph alone is not."""
    from transformertts_amd import _lib
    ops, _ = world
    for power in (1, 2):
        for grad in (lambda loss, x: torch.autograd.grad(loss, x), lambda loss, x: loss.backward()):
            x = [_t(3, h, 8, grad=True) for h in (2, 1, 1)]
            loss = (ops.packed_attention(*x, _ints(0, 3)) ** power).sum()
            grads = torch.autograd.grad(loss, x, create_graph=True)
            torch.autograd.grad(loss, x, retain_graph=True)
            with pytest.raises(_lib.TtsmiError, match='second derivatives'):
                grad(loss + sum((g ** 2).sum() for g in grads), x)


def test_second_derivatives_of_rotary_are_turns(world):
    """The gradient's own gradient is asked of the kernel, turned the other way again."""
    ops, rec = world
    q, k, dq, dk = (_t(3, h, 8, grad=True) for h in (2, 1, 2, 1))
    out = ops.rotary(q, k, _ints(0, 1, 2), _t(4, dtype=torch.float64), scale=0.5)
    grads = torch.autograd.grad(out, (q, k), (dq, dk), create_graph=True)
    again = torch.autograd.grad(grads, (dq, dk), (torch.ones(3, 2, 8), torch.ones(3, 1, 8)))
    assert [tuple(g.shape) for g in again] == [(3, 2, 8), (3, 1, 8)]
    assert [a[-3] for _, a in rec.calls] == [0, 1, 0] and [a[-4] for _, a in rec.calls] == [0.5] * 3


def test_forward_mode_tangents_are_refused(world):
    """A dual tensor wants no gradient and has a pointer: its tangent would be dropped."""
    from transformertts_amd import _lib
    import torch.autograd.forward_ad as fwd
    ops, rec = world
    q, k, v, freqs = _t(3, 2, 8), _t(3, 1, 8), _t(3, 1, 8), _t(4, dtype=torch.float64)
    st, ln, table, pos, cache = _ints(0, 3), _ints(3), _ints(0).view(1, 1), _ints(0, 1, 2), _cache(ops)
    with fwd.dual_level():
        def dual(t):
            return fwd.make_dual(t, torch.ones(t.shape, dtype=t.dtype)).as_subclass(OnGpu)
        a, b, f = dual(q), dual(k), dual(freqs)
        learned = ops.KVCache(dual(torch.zeros(2, 1, 4, 8)), torch.zeros(2, 1, 4, 8).as_subclass(OnGpu))
        for call in (lambda: ops.rotary(a, k, pos, freqs), lambda: ops.rotary(q, b, pos, freqs), lambda: ops.rotary(a, None, pos, freqs, inplace=True),
                     lambda: ops.rotary(q, k, pos, f), lambda: ops.packed_attention(a, k, v, st), lambda: ops.packed_attention(q, b, v, st),
                     lambda: ops.packed_attention(q, k, b, st), lambda: ops.packed_attention(a.detach().requires_grad_(), b, v, st),
                     lambda: ops.kv_cache_write(cache, b, v, table, st, ln), lambda: ops.kv_cache_write(cache, k, b, table, st, ln),
                     lambda: ops.kv_cache_read(learned, table, ln, st, 3, out=(_t(3, 1, 8), _t(3, 1, 8))), lambda: ops.paged_attention(a, cache, table, st, ln),
                     lambda: ops.paged_attention(q, learned, table, st, ln), lambda: ops.paged_attention(q, cache, table, st, ln, out=dual(_t(3, 2, 8)))):
            with pytest.raises(_lib.TtsmiError, match='tangent'):
                call()
        assert not rec.calls
        ops.packed_attention(q, k, v, st)                  # tensors of no tangent go through
        ops.paged_attention(q, cache, table, st, ln)
    assert len(rec.calls) == 2


@pytest.mark.parametrize('dtype', [torch.float32, torch.float8_e4m3fn])
def test_a_cache_holds_the_tensors_it_was_made_of(world, dtype):
    """Its tensors cannot be exchanged under the pointers that the calls use: assigning is an error, and a tensor whose memory has
    moved is noticed before anything is launched."""
    from transformertts_amd import _lib
    ops, rec = world
    q, k, v = _t(3, 2, 8), _t(3, 1, 8), _t(3, 1, 8)
    st, ln, table = _ints(0, 3), _ints(3), _ints(0).view(1, 1)
    cache = _cache(ops, dtype)
    names = ['k', 'v'] + ['k_exp', 'v_exp'] * (cache.k_exp is not None)
    for name in names + ['args', 'heads', 'dh', 'page_size', 'dtype', 'code', 'index']:
        old = getattr(cache, name)
        with pytest.raises(AttributeError):
            setattr(cache, name, old)
        with pytest.raises(AttributeError):
            delattr(cache, name)
        assert getattr(cache, name) is old
    for name in names:
        cache = _cache(ops, dtype)
        t = getattr(cache, name)
        kept = t.data                                      # (the old memory stays where it is)
        t.data = torch.zeros((64,) + t.shape[1:], dtype=torch.uint8).view(t.dtype) if t.element_size() == 1 else torch.zeros((64,) + t.shape[1:])
        for call in (lambda: ops.kv_cache_write(cache, k, v, table, st, ln), lambda: ops.paged_attention(q, cache, table, st, ln),
                     lambda: ops.kv_cache_read(cache, table, ln, st, 3, out=(_t(3, 1, 8), _t(3, 1, 8)))):
            with pytest.raises(_lib.TtsmiError, match='moved'):
                call()
        t.data = kept
        ops.kv_cache_write(cache, k, v, table, st, ln)
    assert len(rec.calls) == len(names)
    import copy
    other = copy.copy(cache)
    assert other.args == cache.args and other.k is cache.k and other.heads == cache.heads


def test_the_overlap_of_views_is_found(world):
    """ops._share against the elements' own addresses, over views of one buffer in every order that a layer makes."""
    import random
    ops, _ = world
    rng, found = random.Random(3), [0, 0]
    base = torch.zeros(6000)

    def addresses(t):
        return {t.storage_offset() + i * t.stride(0) + j * t.stride(1) + c for i in range(t.shape[0]) for j in range(t.shape[1]) for c in range(t.shape[2])}
    for n in range(4000):
        M, dh = rng.choice([1, 2, 3, 7]), rng.choice([2, 4, 8])
        views = []
        layout, W = rng.choice(['rows', 'heads', 'parts', 'blocks']), rng.choice([2, 3, 6])
        for _ in 'ab':
            if layout == 'rows':                           # parts of a fused projection
                x, lo = base[:M * W * dh].view(M, W, dh), rng.randrange(W)
                views.append(x[:, lo:lo + rng.randint(1, W)] if rng.random() < 0.8 else x[:, lo::2])
            elif layout == 'heads':                        # [heads, tokens, dh]
                x, lo = base[:W * M * dh].view(W, M, dh), rng.randrange(W)
                views.append(x[lo:lo + rng.randint(1, W)].transpose(0, 1))
            elif layout == 'blocks':                       # [heads, parts, tokens, dh]
                x, lo = base[:M * W * 3 * dh].view(W, 3, M, dh), rng.randrange(W)
                views.append(x[lo:lo + rng.randint(1, W), rng.randrange(3)].transpose(0, 1))
            else:                                          # [tokens, heads, parts, dh]
                x = base[:M * W * 3 * dh].view(M, W, 3, dh)
                views.append(x[:, :, rng.randrange(3)])
        if rng.random() < 0.3:
            shift = rng.randrange(1, 3 * dh)
            views[1] = torch.as_strided(base, views[1].shape, views[1].stride(), views[1].storage_offset() + shift)
        common = bool(addresses(views[0]) & addresses(views[1]))
        found[common] += 1
        assert ops._share(*views) == common, (n, layout, [(tuple(v.shape), v.stride(), v.storage_offset()) for v in views])
    assert min(found) > 500
    assert not ops._share(base[:0].view(0, 1, 2), base[:2].view(1, 1, 2)) and not ops._share(base[:4].view(2, 1, 2), torch.zeros(2, 1, 2))


def test_destinations_that_share_memory_are_refused(world):
    """Keys and queries turned in place, rows read back and attention's output would be written over each other or while they are
    read; an output that is the queries themselves is not among them."""
    from transformertts_amd import _lib
    ops, rec = world
    x = torch.ones(3, 6, 8).as_subclass(OnGpu)
    st, ln, table, pos, freqs, cache = _ints(0, 3), _ints(3), _ints(0).view(1, 1), _ints(0, 1, 2), _t(4, dtype=torch.float64), _cache(ops)
    pages = torch.zeros(3, 1, 4, 8).as_subclass(OnGpu)
    bytes_ = torch.zeros(256, dtype=torch.uint8)
    e4m3 = [bytes_[n:n + 64].view(torch.float8_e4m3fn).view(2, 1, 4, 8).as_subclass(OnGpu) for n in (0, 64)]
    exps = [bytes_[n:n + 8].view(2, 1, 4).as_subclass(OnGpu) for n in (128, 136, 132, 60)]
    for call in (lambda: ops.rotary(x[:, :4], x[:, :4], pos, freqs, inplace=True), lambda: ops.rotary(x[:, :4], x[:, 3:5], pos, freqs, inplace=True),
                 lambda: ops.kv_cache_read(cache, table, ln, st, 3, out=(x[:, :1], x[:, :1])),
                 lambda: ops.paged_attention(x[:, :4], cache, table, st, ln, out=x[:, 1:5]),
                 lambda: ops.KVCache(pages[:2], pages[1:]), lambda: ops.KVCache(*e4m3, exps[0], exps[2]), lambda: ops.KVCache(*e4m3, exps[0], exps[0]),
                 lambda: ops.KVCache(*e4m3, exps[3], exps[1])):
        with pytest.raises(_lib.TtsmiError, match='memory'):
            call()
    assert not rec.calls
    ops.rotary(x[:, :4], x[:, 4:6], pos, freqs, inplace=True)
    ops.rotary(x[:, :4], x[:, 3:5], pos, freqs)
    ops.kv_cache_read(cache, table, ln, st, 3, out=(x[:, :1], x[:, 1:2]))
    ops.paged_attention(x[:, :4], cache, table, st, ln, out=x[:, :4])
    ops.KVCache(pages[:1], pages[1:2])
    ops.KVCache(*e4m3, exps[0], exps[1])
    assert len(rec.calls) == 4

"""CPU-side checks of the sequence operators: what the C entries refuse before any launch, workspace sizes, what the host
mirror refuses, and the rotary frequencies."""
import ctypes

import numpy as np
import pytest
import torch


@pytest.fixture(scope='module')
def lib():
    from transformertts_amd import _lib
    return _lib.lib()


ONE, ODD = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 4)         # never dereferenced: every call is refused, or has no tokens
F32, BF16, E4M3 = 0, 2, 4


def _packed(lib, bwd=False, **over):
    a = dict(q=ONE, q_row=256, q_head=64, k=ONE, k_row=128, k_head=64, v=ONE, v_row=128, v_head=64, out=ONE, o_row=256, o_head=64, dout=ONE,
             d_row=256, d_head=64, lse=ONE, rest=ONE, starts=ONE, B=2, tokens=10, H=4, Hkv=2, dh=64, scale=0.125, causal=1, dq=ONE, dq_row=256, dq_head=64,
             dk=ONE, dk_row=128, dk_head=64, dv=ONE, dv_row=128, dv_head=64, zero_rest=1, ws=ONE, ws_bytes=1 << 30, dtype=BF16)
    a.update(over)
    fwd = 'q q_row q_head k k_row k_head v v_row v_head starts B tokens H Hkv dh scale causal out o_row o_head lse rest zero_rest dtype'
    back = ('q q_row q_head k k_row k_head v v_row v_head out o_row o_head rest dout d_row d_head lse starts B tokens H Hkv dh scale causal dq dq_row '
            'dq_head dk dk_row dk_head dv dv_row dv_head zero_rest ws ws_bytes dtype')
    f = lib.ttsmi_packed_attention_bwd if bwd else lib.ttsmi_packed_attention_fwd
    return f(*[a[n] for n in (back if bwd else fwd).split()], None), lib.ttsmi_last_error()


@pytest.mark.parametrize('over,code,word', [
    (dict(dtype=1), -1, b'dtype'), (dict(dtype=E4M3), -1, b'dtype'), (dict(H=5), -1, b'heads'), (dict(Hkv=0), -1, b'heads'), (dict(H=0), -1, b'heads'),
    (dict(dh=60), -1, b'head size'), (dict(dh=200), -1, b'head size'), (dict(dh=0), -1, b'head size'), (dict(scale=0.0), -1, b'scale'),
    (dict(scale=-1.0), -1, b'scale'), (dict(scale=float('nan')), -1, b'scale'), (dict(scale=float('inf')), -1, b'scale'), (dict(tokens=-1), -1, b'tokens'),
    (dict(B=-1), -1, b'sequences'), (dict(tokens=1 << 30), -1, b'too large'), (dict(starts=None), -1, b'starts'), (dict(q=None), -1, b'null'),
    (dict(k=ODD), -1, b'aligned'), (dict(v_row=132), -1, b'aligned'), (dict(q_head=60), -1, b'aligned'), (dict(out=None), -1, b'null'), (dict(rest=ODD), -1, b'aligned'), (dict(k_row=-128), -1, b'aligned'),
    (dict(k_row=1 << 24), -1, b'too far apart'), (dict(q_head=1 << 30), -1, b'too far apart'), (dict(q_row=1 << 40), -1, b'too far apart')])
@pytest.mark.parametrize('bwd', [False, True])
def test_packed_attention_refuses(lib, over, code, word, bwd):
    rc, err = _packed(lib, bwd, **over)
    assert rc == code and word in err, (rc, err)


def test_packed_attention_bwd_refuses_and_empty_calls_pass(lib):
    for over, code, word in ((dict(lse=None), -1, b'lse'), (dict(dq=ODD), -1, b'aligned'), (dict(dk=None), -1, b'null'), (dict(dv_row=4), -1, b'aligned'),
                             (dict(ws=None), -4, b'workspace'), (dict(ws_bytes=10 * 4 * 4 - 1), -4, b'workspace'), (dict(ws=ODD), -4, b'workspace')):
        rc, err = _packed(lib, True, **over)
        assert rc == code and word in err, (over, rc, err)
    assert _packed(lib, tokens=0, q=None)[0] == 0 and _packed(lib, True, tokens=0, ws=None)[0] == 0
    assert lib.ttsmi_packed_attention_bwd_ws_bytes(2, 10, 4, 2, 64, 1) >= 160 and lib.ttsmi_packed_attention_bwd_ws_bytes(2, 0, 4, 2, 64, 1) == 0


def _cache_args(order, **over):
    a = dict(k=ONE, k_row=128, k_head=64, v=ONE, v_row=128, v_head=64, q=ONE, q_row=256, q_head=64, out=ONE, o_row=256, o_head=64, kp=ONE, vp=ONE, ke=ONE, ve=ONE,
             cache=E4M3, pages=8, page=16, table=ONE, width=4, starts=ONE, lens=ONE, B=2, tokens=10, H=4, Hkv=2, dh=64, scale=0.125, zero_rest=1,
             ws=ONE, ws_bytes=1 << 30, dtype=BF16)
    a.update(over)
    return [a[n] for n in order.split()] + [None]


_ORDERS = {
    'ttsmi_kv_cache_write': 'k k_row k_head v v_row v_head kp vp ke ve cache pages page table width starts lens B tokens Hkv dh dtype',
    'ttsmi_kv_cache_read': 'kp vp ke ve cache pages page table width starts lens B tokens Hkv dh k k_row k_head v v_row v_head zero_rest dtype',
    'ttsmi_paged_attention': 'q q_row q_head kp vp ke ve cache pages page table width starts lens B tokens H Hkv dh scale out o_row o_head zero_rest ws ws_bytes dtype'}


@pytest.mark.parametrize('name', sorted(_ORDERS))
@pytest.mark.parametrize('over,word', [
    (dict(dtype=1), b'dtype'), (dict(cache=F32), b'cache dtype'), (dict(cache=7), b'cache dtype'), (dict(page=0), b'pages of'), (dict(page=24), b'pages of'),
    (dict(page=2048), b'pages of'), (dict(pages=-1), b'pages of'), (dict(width=-1), b'pages of'), (dict(dh=12), b'head size'), (dict(tokens=-3), b'tokens'),
    (dict(Hkv=0), b'heads'), (dict(starts=None), b'starts'), (dict(lens=None), b'lens'), (dict(table=None), b'table'), (dict(kp=ODD), b'aligned'),
    (dict(vp=None), b'pages null'), (dict(ke=None), b'exponents'), (dict(ve=None), b'exponents'), (dict(k=ODD, q=ODD), b'aligned'),
    (dict(v_head=4, o_head=4), b'aligned')])
def test_cache_entries_refuse(lib, name, over, word):
    rc = getattr(lib, name)(*_cache_args(_ORDERS[name], **over))
    err = lib.ttsmi_last_error()
    if name == 'ttsmi_kv_cache_write' or name == 'ttsmi_kv_cache_read':
        word = b'key heads' if over == dict(Hkv=0) else word
    assert rc == -1 and word in err, (rc, err)
    assert getattr(lib, name)(*_cache_args(_ORDERS[name], tokens=0)) == 0


def test_paged_attention_workspace(lib):
    need = lib.ttsmi_paged_attention_ws_bytes(2, 10, 4, 2, 64, E4M3, BF16)
    assert need >= 2 * 10 * 4 * 66 * 4                                       # a few rows over a long cache are split
    order = _ORDERS['ttsmi_paged_attention']
    for over in (dict(ws=None), dict(ws_bytes=need - 1), dict(ws=ODD)):
        assert lib.ttsmi_paged_attention(*_cache_args(order, **over)) == -4 and b'workspace' in lib.ttsmi_last_error()
    assert lib.ttsmi_paged_attention_ws_bytes(1, 1 << 16, 32, 8, 128, BF16, BF16) == 0          # tiles that fill the card are not
    assert lib.ttsmi_paged_attention_ws_bytes(0, 0, 4, 2, 64, BF16, BF16) == 0 and lib.ttsmi_paged_attention_ws_bytes(1, 1, 4, 0, 64, BF16, BF16) == 0
    for over in (dict(scale=0.0), dict(H=3), dict(out=None)):
        assert lib.ttsmi_paged_attention(*_cache_args(order, **over)) == -1


@pytest.mark.parametrize('over,word', [
    (dict(dtype=4), b'dtype'), (dict(dh=63), b'even'), (dict(rot=3), b'even'), (dict(rot=66), b'even'), (dict(dh=1200, rot=514), b'turned'), (dict(tokens=-1), b'tokens'),
    (dict(H=-1), b'heads'), (dict(pos=None), b'positions'), (dict(freqs=None), b'frequencies'), (dict(q=None), b'null'), (dict(ko=None), b'null'),
    (dict(k=ctypes.c_void_p((1 << 20) + 1)), b'aligned')])
def test_rotary_refuses(lib, over, word):
    a = dict(q=ONE, q_row=256, q_head=64, qo=ONE, qo_row=256, qo_head=64, H=4, k=ONE, k_row=128, k_head=64, ko=ONE, ko_row=128, ko_head=64, Hkv=2, pos=ONE, freqs=ONE,
             tokens=5, dh=64, rot=64, inter=0, scale=1.0, inverse=0, dtype=BF16)
    call = lambda **o: lib.ttsmi_rotary(*{**a, **o}.values(), None)
    assert call(**over) == -1 and word in lib.ttsmi_last_error(), lib.ttsmi_last_error()
    assert call(tokens=0) == 0


def test_the_host_mirror_refuses_cpu_tensors_and_bad_shapes():
    from transformertts_amd import _lib, ops
    q, st = torch.zeros(4, 2, 8), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.packed_attention(q, q, q, st), lambda: ops.rotary(q, q, st, torch.zeros(4, dtype=torch.float64)),
                 lambda: ops.packed_attention(q[0], q, q, st), lambda: ops.paged_attention(q, None, st, st, st),
                 lambda: ops.KVCache(torch.zeros(1, 1, 8, 8), torch.zeros(1, 1, 8, 8)),
                 lambda: ops.KVCache(torch.zeros(1, 1, 9, 8), torch.zeros(1, 1, 9, 8)), lambda: ops.KVCache(torch.zeros(1, 1, 8, 9), torch.zeros(1, 1, 8, 9)),
                 lambda: ops.KVCache(*[torch.zeros(1, 1, 8, 8, dtype=torch.uint8).view(torch.float8_e4m3fn)] * 2),
                 lambda: ops.KVCache(torch.zeros(1, 1, 8, 8), torch.zeros(1, 2, 8, 8)), lambda: ops.KVCache(*[torch.zeros(1, 1, 8, 8, dtype=torch.float16)] * 2)):
        with pytest.raises(_lib.TtsmiError):
            call()


def test_rotary_frequencies():
    from transformertts_amd.model.transformer_utils import rotary_frequencies
    f = rotary_frequencies(8, base=100.0)
    assert f.dtype == np.float64 and np.allclose(f, [1.0, 100 ** -0.25, 100 ** -0.5, 100 ** -0.75], rtol=1e-15)
    assert np.array_equal(rotary_frequencies(8, scaling='linear', factor=4.0), rotary_frequencies(8) / 4.0)
    s = rotary_frequencies(64, scaling='base', factor=8.0)
    assert s[0] == 1.0 and np.isclose(s[-1], rotary_frequencies(64)[-1] / 8.0, rtol=1e-12)
    n, b = rotary_frequencies(128), rotary_frequencies(128, scaling='bands', factor=16.0, original_length=4096)
    turns = 4096 * n / (2 * np.pi)
    assert np.array_equal(b[turns >= 32], n[turns >= 32]) and np.allclose(b[turns <= 1], n[turns <= 1] / 16.0, rtol=1e-15)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and np.all(b[mid] < n[mid]) and np.all(b[mid] > n[mid] / 16.0) and np.all(np.diff(b) < 0)
    for bad in (dict(dim=7), dict(dim=0), dict(dim=8, scaling='ntk'), dict(dim=8, factor=0.0), dict(dim=8, scaling='bands', slow_turns=4.0, fast_turns=4.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def test_packed_attention_bwd_workspace_follows_the_tokens(lib):
    """delta and lse2, and partial sums for no more row splits than the tokens allow: a split has 192 rows at least, a sequence of
    no more than that (61 tokens, one or two heads a key head) none."""
    need = lib.ttsmi_packed_attention_bwd_ws_bytes
    for B, tokens, H, Hkv, dh in ((1, 61, 2, 2, 192), (1, 61, 4, 2, 64), (3, 190, 8, 8, 128), (0, 96, 4, 2, 64), (40, 96, 32, 16, 192)):
        for causal in (0, 1):
            assert need(B, tokens, H, Hkv, dh, causal) == (2 * tokens * H * 4 + 255) // 256 * 256
    tile = 2 * 128 * 64 * 4                                              # dK and dV of 128 keys of 64
    assert need(1, 61, 16, 1, 64, 1) == (2 * 61 * 16 * 4 + 255) // 256 * 256 + (1 + 1 + 5) * tile                 # 976 rows, one key tile: 5 splits behind the first
    for causal, slots in ((0, 512), (1, 1536)):                          # long ones: what the card holds, as before
        assert need(1, 6000, 16, 2, 128, causal) == 2 * 6000 * 16 * 4 + (6000 // 128 + 2 + slots // 2) * 2 * 2 * tile
        assert need(1, 6000, 2, 1, 64, causal) == 2 * 6000 * 2 * 4 + (6000 // 128 + 2 + slots) * tile

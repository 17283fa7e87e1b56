"""CPU: the sequence operators are registered, refuse CPU tensors, and their C entry points refuse bad calls before any launch;
the float64 forms they are tested against agree with each other."""
import ctypes

import pytest
import torch

from helpers import ROOT  # noqa: F401
from oracle import sequence_oracle as ref

from tempenslearnagg_qcnet_amd import _lib, ops

INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3
FAKE = 1 << 20      # an address that is never read: every call below is refused, or has nothing to do, on the host


def test_registered_and_refusing_cpu_tensors():
    assert ops.SEQUENCE_OP_NAMES == ['rotary_embed', 'attn_window', 'window_cache_append', 'attn_window_step']
    for name in ops.SEQUENCE_OP_NAMES:
        assert str(getattr(torch.ops.qcnet_hip, name).default._schema).startswith('qcnet_hip::%s(' % name)
    x, n = torch.zeros(4, 2, 16), torch.zeros(4, dtype=torch.int64)
    c = torch.zeros(4, 2, 6, 16)
    for call in (lambda: ops.rotary_embed(x, None, torch.zeros(4, 1), torch.zeros(8), [8]),
                 lambda: ops.attn_window(x, x, x, torch.tensor([0, 4]), 3),
                 lambda: ops.window_cache_append(x, x, torch.arange(5), n, c, c.clone(), 1),
                 lambda: ops.attn_window_step(x, x, x, n, c, c.clone(), 1)):
        with pytest.raises(_lib.QcnError, match='no CPU fallback'):
            call()
    for bad in (float('nan'), float('inf'), -0.5):
        with pytest.raises(ValueError):
            ops.attn_window(x, x, x, torch.tensor([0, 4]), 3, scale=bad)


def _window(lib, q=FAKE, k=FAKE, v=FAKE, tok=32, head=16, cu=FAKE, n_seq=1, nq=4, nk=4, hq=2, hk=2, dim=16, dtype=0, win=3, sinks=0,
            scale=1.0, out=FAKE):
    return lib.qcn_attn_window(q, tok, head, k, tok, head, v, tok, head, cu, cu, None, n_seq, nq, nk, hq, hk, dim, dtype, win, sinks,
                               ctypes.c_float(scale), out, None)


def test_window_entry_point_refusals():
    lib = _lib.lib()
    for bad in (dict(hq=3), dict(hq=0), dict(hk=0), dict(n_seq=-1), dict(nq=-1), dict(nk=-1), dict(win=0), dict(sinks=-1), dict(dtype=3),
                dict(scale=-1.0), dict(scale=float('nan')), dict(scale=float('inf')), dict(q=None), dict(k=None), dict(cu=None),
                dict(out=None), dict(q=FAKE + 4), dict(k=FAKE + 8), dict(tok=33), dict(head=2), dict(out=FAKE + 4)):
        assert _window(lib, **bad) == INVALID, bad
    for bad in (dict(dim=20), dict(dim=136), dict(dim=0), dict(nq=1 << 41)):
        assert _window(lib, **bad) == UNSUPPORTED, bad
    assert _window(lib, nq=0) == 0


def _step(lib, q=FAKE, k=FAKE, v=FAKE, lengths=FAKE, key_mask=None, batch=2, hq=4, hk=2, dim=64, dtype=2, win=4, sinks=1, kc=FAKE, vc=FAKE,
          mc=None, out=FAKE, ws=None, ws_bytes=0, tok=512, head=64):
    return lib.qcn_attn_window_step(q, tok, head, k, tok, head, v, tok, head, lengths, key_mask, batch, hq, hk, dim, dtype, win, sinks,
                                    ctypes.c_float(1.0), kc, vc, mc, out, ws, ws_bytes, None)


def test_step_and_append_entry_point_refusals():
    lib = _lib.lib()
    for bad in (dict(hq=3), dict(hk=0), dict(batch=-1), dict(win=0), dict(sinks=-1), dict(dtype=-1), dict(q=None), dict(lengths=None),
                dict(kc=None), dict(vc=FAKE + 2), dict(out=None), dict(key_mask=FAKE), dict(head=60), dict(win=1 << 41)):
        assert _step(lib, **bad) == INVALID, bad
    assert _step(lib, dim=12) == UNSUPPORTED
    assert _step(lib, batch=0) == 0
    app = lambda k=FAKE, n_seq=1, n=4, hk=2, dim=16, dtype=0, win=3, sinks=0, kc=FAKE, km=None, mc=None, tok=32: \
        lib.qcn_window_cache_append(k, tok, 16, FAKE, 32, 16, FAKE, FAKE, km, n_seq, n, hk, dim, dtype, win, sinks, kc, FAKE, mc, None)
    for bad in (dict(k=None), dict(n_seq=-1), dict(n=-1), dict(hk=0), dict(dtype=9), dict(win=0), dict(sinks=-2), dict(kc=None),
                dict(km=FAKE), dict(tok=31)):
        assert app(**bad) == INVALID, bad
    assert app(dim=18) == UNSUPPORTED
    assert app(n=0) == 0 and app(n_seq=0) == 0


def test_rotary_entry_point_refusals():
    lib = _lib.lib()

    def call(sections=(8,), n=4, hq=2, hk=0, k=None, dim=16, dtype=0, pos=FAKE, pos_type=0, q=FAKE, out=FAKE, interleaved=0, tok=32):
        arr = (ctypes.c_int32 * max(1, len(sections)))(*sections)
        return lib.qcn_rotary_embed(q, tok, 16, hq, k, tok, 16, hk, n, dim, dtype, pos, pos_type, len(sections), FAKE, arr, interleaved, 0,
                                    out, out, None)
    for bad in (dict(sections=()), dict(sections=(1,) * 9), dict(sections=(9,)), dict(sections=(0,)), dict(sections=(-1, 4)), dict(dim=15),
                dict(dtype=5), dict(pos_type=3), dict(pos=None), dict(q=None), dict(hk=1), dict(k=FAKE), dict(n=-1),
                dict(interleaved=1, tok=33)):
        assert call(**bad) == INVALID, bad
    assert call(dim=258) == UNSUPPORTED and call(n=1 << 31) == UNSUPPORTED
    assert call(n=0) == 0


def test_the_cache_holds_what_a_position_sees():
    """step() over the cache equals window() over the whole sequence, for every position (float64, no kernel)."""
    g = torch.Generator().manual_seed(0)
    for win, sinks in ((1, 0), (4, 0), (3, 2), (5, 7), (40, 3)):
        n, b = 23, 2
        q, k, v = torch.randn(b * n, 2, 8, generator=g), torch.randn(b * n, 1, 8, generator=g), torch.randn(b * n, 1, 8, generator=g)
        mask = torch.rand(b * n, generator=g) < 0.7
        want = ref.window(q, k, v, [0, n, 2 * n], win, sinks, key_mask=mask)[0]
        kc, vc = torch.zeros(b, 1, win + sinks, 8), torch.zeros(b, 1, win + sinks, 8)
        mc = torch.zeros(b, win + sinks, dtype=torch.bool)
        for t in range(n):
            at = torch.tensor([t, n + t])
            got = ref.step(q[at], k[at], v[at], torch.tensor([t, t]), kc, vc, sinks, mask[at], mc)[0]
            assert torch.allclose(got, want[at], atol=1e-12)


def test_rotary_form_keeps_lengths_and_turns_back():
    g = torch.Generator().manual_seed(1)
    x, pos, freqs = torch.randn(9, 2, 20, generator=g), torch.randn(9, 2, generator=g) * 50, torch.rand(8, generator=g)
    for interleaved in (False, True):
        y = ref.rotary(x, pos, freqs, [5, 3], interleaved)
        assert torch.allclose(y.norm(dim=-1), x.double().norm(dim=-1))
        assert torch.allclose(ref.rotary(y, pos, freqs, [5, 3], interleaved, inverse=True), x.double())

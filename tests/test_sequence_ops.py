"""CPU: the sequence operators are registered, refuse CPU tensors, and their C entry points refuse bad calls before any launch;
the float64 forms they are tested against agree with each other."""
import struct

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


def _call(lib, name, fmt, fields, **over):
    """The entry point on its argument struct: ``fields`` in the header's order, with some of them replaced."""
    values = dict(fields, **over)
    assert list(values) == list(fields)
    return getattr(lib, name)(struct.pack('=' + fmt, *[x for v in values.values() for x in (v if isinstance(v, tuple) else (v,))]), None)


def test_window_entry_point_refusals():
    lib = _lib.lib()
    fields = dict(q=FAKE, qs=(32, 16), k=FAKE, ks=(32, 16), v=FAKE, vs=(32, 16), cu_q=FAKE, cu_k=FAKE, mask=0, n_seq=1, nq=4, nk=4, hq=2,
                  hk=2, dim=16, dtype=0, window=3, sinks=0, scale=1.0, out=FAKE, ws=0, ws_bytes=0)
    call = lambda **over: _call(lib, 'qcn_attn_window', '21qd3q', fields, **over)
    for bad in (dict(hq=3), dict(hq=0), dict(hk=0), dict(n_seq=-1), dict(nq=-1), dict(nk=-1), dict(window=0), dict(sinks=-1), dict(dtype=3),
                dict(scale=-1.0), dict(scale=float('nan')), dict(scale=float('inf')), dict(q=0), dict(k=0), dict(v=0), dict(cu_q=0),
                dict(cu_k=0), dict(out=0), dict(q=FAKE + 4), dict(k=FAKE + 8), dict(qs=(33, 16)), dict(vs=(32, 2)), dict(out=FAKE + 4)):
        assert call(**bad) == INVALID, bad
    for bad in (dict(dim=20), dict(dim=136), dict(dim=0), dict(nq=1 << 31), dict(nk=1 << 31), dict(n_seq=1 << 31), dict(hq=1 << 16),
                dict(ks=(1 << 24, 16))):
        assert call(**bad) == UNSUPPORTED, bad
    assert call(nq=0) == 0
    # 32 queries behind 8192 keys: split over blocks, which takes a workspace
    assert call(dtype=2, dim=64, qs=(128, 64), ks=(128, 64), vs=(128, 64), nq=32, nk=8192, window=4096) == WORKSPACE
    assert lib.qcn_attn_window(None, None) == INVALID


def test_step_and_append_entry_point_refusals():
    lib = _lib.lib()
    fields = dict(q=FAKE, qs=(512, 64), k=FAKE, ks=(512, 64), v=FAKE, vs=(512, 64), lengths=FAKE, key_mask=0, batch=2, hq=4, hk=2, dim=64,
                  dtype=2, window=4, sinks=1, scale=1.0, kc=FAKE, vc=FAKE, mc=0, out=FAKE, ws=0, ws_bytes=0)
    step = lambda **over: _call(lib, 'qcn_attn_window_step', '18qd6q', fields, **over)
    for bad in (dict(hq=3), dict(hk=0), dict(batch=-1), dict(window=0), dict(sinks=-1), dict(dtype=-1), dict(q=0), dict(lengths=0), dict(kc=0),
                dict(vc=FAKE + 2), dict(out=0), dict(key_mask=FAKE), dict(qs=(512, 60)), dict(window=1 << 41), dict(scale=-1.0)):
        assert step(**bad) == INVALID, bad
    assert step(dim=12) == UNSUPPORTED and step(batch=1 << 31) == UNSUPPORTED
    assert step(batch=0) == 0
    need = lib.qcn_attn_window_step_workspace_bytes(2, 4, 2, 64, 4096, 1)
    assert need > 0 and lib.qcn_attn_window_step_workspace_bytes(2, 4, 2, 64, 50, 1) == 0
    assert step(window=4096) == WORKSPACE and step(window=4096, ws=FAKE, ws_bytes=need - 1) == WORKSPACE
    assert lib.qcn_attn_window_step(None, None) == INVALID
    fields2 = dict(k=FAKE, ks=(32, 16), v=FAKE, vs=(32, 16), cu=FAKE, lengths=FAKE, key_mask=0, n_seq=1, n=4, hk=2, dim=16, dtype=0, window=3,
                   sinks=0, kc=FAKE, vc=FAKE, mc=0)
    app = lambda **over: _call(lib, 'qcn_window_cache_append', '19q', fields2, **over)
    for bad in (dict(k=0), dict(n_seq=-1), dict(n=-1), dict(hk=0), dict(dtype=9), dict(window=0), dict(sinks=-2), dict(kc=0),
                dict(key_mask=FAKE), dict(ks=(31, 16)), dict(cu=0), dict(lengths=0)):
        assert app(**bad) == INVALID, bad
    assert app(dim=18) == UNSUPPORTED
    assert app(n=0) == 0 and app(n_seq=0) == 0
    assert lib.qcn_window_cache_append(None, None) == INVALID


def test_rotary_entry_point_refusals():
    lib = _lib.lib()
    fields = dict(q=FAKE, qs=(32, 16), hq=2, k=0, ks=(0, 0), hk=0, n=4, dim=16, dtype=0, pos=FAKE, pos_type=0, axes=1,
                  sections=(8,) + (0,) * 7, freqs=FAKE, interleaved=0, inverse=0, q_out=FAKE, k_out=0)
    call = lambda **over: _call(lib, 'qcn_rotary_embed', '27q', fields, **over)
    for bad in (dict(axes=0), dict(axes=9), dict(sections=(9,) + (0,) * 7), dict(sections=(0,) * 8), dict(sections=(-1, 4) + (0,) * 6, axes=2),
                dict(dim=15), dict(dtype=5), dict(pos_type=3), dict(pos=0), dict(freqs=0), dict(q=0), dict(q_out=0), dict(hk=1), dict(k=FAKE),
                dict(n=-1), dict(interleaved=1, qs=(33, 16)), dict(q=FAKE + 2)):
        assert call(**bad) == INVALID, bad
    assert call(dim=258) == UNSUPPORTED and call(n=1 << 31) == UNSUPPORTED and call(hq=1 << 16) == UNSUPPORTED
    assert call(n=0) == 0
    assert lib.qcn_rotary_embed(None, None) == INVALID


def test_strides_that_point_backwards_and_sizes_past_32_bits_are_refused():
    lib = _lib.lib()
    window = dict(q=FAKE, qs=(32, 16), k=FAKE, ks=(32, 16), v=FAKE, vs=(32, 16), cu_q=FAKE, cu_k=FAKE, mask=0, n_seq=1, nq=4, nk=4, hq=2,
                  hk=2, dim=16, dtype=0, window=3, sinks=0, scale=1.0, out=FAKE, ws=0, ws_bytes=0)
    for bad in (dict(qs=(-32, 16)), dict(ks=(32, -16)), dict(vs=(-32, -16))):
        assert _call(lib, 'qcn_attn_window', '21qd3q', window, **bad) == INVALID, bad
    for bad in (dict(nq=(1 << 31) - 1), dict(nk=(1 << 31) - 200)):
        assert _call(lib, 'qcn_attn_window', '21qd3q', window, **bad) == UNSUPPORTED, bad
    step = dict(q=FAKE, qs=(512, 64), k=FAKE, ks=(512, 64), v=FAKE, vs=(512, 64), lengths=FAKE, key_mask=0, batch=2, hq=4, hk=2, dim=64,
                dtype=2, window=4, sinks=1, scale=1.0, kc=FAKE, vc=FAKE, mc=0, out=FAKE, ws=0, ws_bytes=0)
    append = dict(k=FAKE, ks=(32, 16), v=FAKE, vs=(32, 16), cu=FAKE, lengths=FAKE, key_mask=0, n_seq=1, n=4, hk=2, dim=16, dtype=0, window=3,
                  sinks=0, kc=FAKE, vc=FAKE, mc=0)
    rotary = dict(q=FAKE, qs=(-32, 16), hq=2, k=0, ks=(0, 0), hk=0, n=4, dim=16, dtype=0, pos=FAKE, pos_type=0, axes=1,
                  sections=(8,) + (0,) * 7, freqs=FAKE, interleaved=0, inverse=0, q_out=FAKE, k_out=0)
    assert _call(lib, 'qcn_attn_window_step', '18qd6q', step, ks=(-512, 64)) == INVALID
    assert _call(lib, 'qcn_window_cache_append', '19q', append, vs=(32, -16)) == INVALID
    assert _call(lib, 'qcn_rotary_embed', '27q', rotary) == INVALID


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


def test_calls_go_past_the_dispatcher_only_where_nothing_has_to_see_them():
    """Plain eager tensors may; under a tracer, a function transform, a dual level or a dispatch mode, and with something to
    differentiate, the call has to be an operator."""
    from torch.utils._python_dispatch import TorchDispatchMode
    from tempenslearnagg_qcnet_amd import sequence_ops
    seen = []

    def f(t):
        seen.append(sequence_ops._plain(t, None))
        return t * 2

    class Watching(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x = torch.ones(3, 2)
    f(x)
    with torch.no_grad():
        f(x.clone().requires_grad_())
    assert seen == [True, False] or seen == [True, True]       # no_grad: nothing to differentiate, either way is right
    seen.clear()
    torch.jit.trace(f, (x,), check_trace=False)
    torch.vmap(f)(x)
    torch.func.jvp(f, (x,), (x,))
    torch.func.grad(lambda t: f(t).sum())(x)
    torch.func.functionalize(f)(x)
    with torch.autograd.forward_ad.dual_level():
        f(torch.autograd.forward_ad.make_dual(x, x))
    with Watching():
        f(x)
    f(x.clone().requires_grad_())
    assert len(seen) == 8 and not any(seen), seen
    seen.clear()
    f(x)
    assert seen == [True]


def test_scales_whose_base_2_form_is_no_float_are_refused():
    """scale * log2(e) overflows float32 above 2.358e38, and an infinite factor makes NaN of a score of 0."""
    lib = _lib.lib()
    window = dict(q=FAKE, qs=(32, 16), k=FAKE, ks=(32, 16), v=FAKE, vs=(32, 16), cu_q=FAKE, cu_k=FAKE, mask=0, n_seq=1, nq=0, nk=4, hq=2,
                  hk=2, dim=16, dtype=0, window=3, sinks=0, scale=1.0, out=FAKE, ws=0, ws_bytes=0)
    step = dict(q=FAKE, qs=(512, 64), k=FAKE, ks=(512, 64), v=FAKE, vs=(512, 64), lengths=FAKE, key_mask=0, batch=0, hq=4, hk=2, dim=64,
                dtype=2, window=4, sinks=1, scale=1.0, kc=FAKE, vc=FAKE, mc=0, out=FAKE, ws=0, ws_bytes=0)
    for name, fmt, fields in (('qcn_attn_window', '21qd3q', window), ('qcn_attn_window_step', '18qd6q', step)):
        assert _call(lib, name, fmt, fields, scale=2.35e38) == 0                # no tokens: nothing to do
        for bad in (2.4e38, 2.9e38, 3.0e38):
            assert _call(lib, name, fmt, fields, scale=bad) == INVALID, (name, bad)
    x, n, c = torch.zeros(4, 2, 16), torch.zeros(4, dtype=torch.int64), torch.zeros(4, 2, 6, 16)
    with pytest.raises(ValueError, match='scale'):
        ops.attn_window(x, x, x, torch.tensor([0, 4]), 3, scale=2.4e38)
    with pytest.raises(ValueError, match='scale'):
        ops.attn_window_step(x, x, x, n, c, c.clone(), 1, scale=2.9e38)


def test_sizes_past_what_a_launch_can_count_are_refused():
    """2^24 blocks of 256 threads are 2^32 threads, one more than a launch counts.  The sizes are refused before any launch, with the
    status that other sizes which are not supported have."""
    lib = _lib.lib()
    window = dict(q=FAKE, qs=(16, 16), k=FAKE, ks=(16, 16), v=FAKE, vs=(16, 16), cu_q=FAKE, cu_k=FAKE, mask=0, n_seq=1, nq=1 << 30, nk=1 << 30,
                  hq=1, hk=1, dim=16, dtype=0, window=3, sinks=0, scale=1.0, out=FAKE, ws=0, ws_bytes=0)
    assert _call(lib, 'qcn_attn_window', '21qd3q', window) == UNSUPPORTED
    assert _call(lib, 'qcn_attn_window', '21qd3q', window, hk=2, hq=4, dim=64, dtype=2) == UNSUPPORTED
    assert _call(lib, 'qcn_attn_window', '21qd3q', window, nq=4, n_seq=1 << 24) == UNSUPPORTED
    step = dict(q=FAKE, qs=(16, 16), k=FAKE, ks=(16, 16), v=FAKE, vs=(16, 16), lengths=FAKE, key_mask=0, batch=1 << 26, hq=1, hk=1, dim=16,
                dtype=2, window=1, sinks=0, scale=1.0, kc=FAKE, vc=FAKE, mc=0, out=FAKE, ws=0, ws_bytes=0)
    assert _call(lib, 'qcn_attn_window_step', '18qd6q', step) == UNSUPPORTED
    assert _call(lib, 'qcn_attn_window_step', '18qd6q', step, batch=1 << 24, window=300) == UNSUPPORTED
    append = dict(k=FAKE, ks=(16, 16), v=FAKE, vs=(16, 16), cu=FAKE, lengths=FAKE, key_mask=0, n_seq=1, n=1 << 28, hk=1, dim=16, dtype=0,
                  window=3, sinks=0, kc=FAKE, vc=FAKE, mc=0)
    assert _call(lib, 'qcn_window_cache_append', '19q', append) == UNSUPPORTED
    rotary = dict(q=FAKE, qs=(8192, 256), hq=32, k=0, ks=(0, 0), hk=0, n=1 << 30, dim=256, dtype=0, pos=FAKE, pos_type=0, axes=1,
                  sections=(8,) + (0,) * 7, freqs=FAKE, interleaved=0, inverse=0, q_out=FAKE, k_out=0)
    assert _call(lib, 'qcn_rotary_embed', '27q', rotary) == UNSUPPORTED


def test_arguments_that_are_no_tensors_are_type_errors():
    from tempenslearnagg_qcnet_amd import sequence_ops
    x, n, c, cu = torch.zeros(4, 2, 16), torch.zeros(4, dtype=torch.int64), torch.zeros(4, 2, 6, 16), torch.tensor([0, 4])
    for call in (lambda: ops.attn_window(None, x, x, cu, 3), lambda: ops.attn_window([1.0], x, x, cu, 3),
                 lambda: ops.attn_window_step(None, x, x, n, c, c.clone(), 1), lambda: ops.attn_window(x, None, x, cu, 3, scale=1.0),
                 lambda: ops.window_cache_append(None, x, cu, n, c, c.clone(), 1),
                 lambda: ops.rotary_embed(None, None, torch.zeros(4, 1), torch.zeros(8), [8]),
                 lambda: sequence_ops._mask_bytes([True] * 4, 'key_mask', 0, torch.device('cuda', 0), 4)):
        with pytest.raises(TypeError, match='must be a tensor'):
            call()
    with pytest.raises(_lib.QcnError, match='no CPU fallback'):
        ops.attn_window(torch.tensor(1.0), x, x, cu, 3)


def test_windows_of_any_size_are_taken_by_the_operator_too(monkeypatch):
    """A window past 64 bits is one that holds everything, whether the call goes through the dispatcher or past it."""
    from tempenslearnagg_qcnet_amd import sequence_ops
    x = torch.zeros(4, 2, 16)
    for direct in (True, False):
        monkeypatch.setattr(sequence_ops, '_plain', lambda *a: direct)
        with pytest.raises(_lib.QcnError, match='no CPU fallback'):
            ops.attn_window(x, x, x, torch.tensor([0, 4]), 1 << 70, 1 << 64)


def test_a_launch_for_a_device_that_is_not_current(monkeypatch):
    """The launch happens with the tensors' device current and on that device's current stream, and so does the question for a
    workspace; where it is current already, nothing is switched."""
    from tempenslearnagg_qcnet_amd import sequence_ops
    now, log = [0], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            now.append(self.index)

        def __exit__(self, *exc):
            now.pop()

    class Library:
        def qcn_attn_window_step(self, args, stream):
            log.append((now[-1], args, stream))
            return 0

        def qcn_attn_window_workspace_bytes(self, args):
            log.append((now[-1], len(args)))
            return 64

        def qcn_status_string(self, status):
            return b'refused'

    library = Library()
    monkeypatch.setattr(_lib, 'lib', lambda: library)
    monkeypatch.setattr(torch._C, '_cuda_getDevice', lambda: now[-1], raising=False)
    monkeypatch.setattr(torch._C, '_cuda_getCurrentRawStream', lambda index: 70 + index, raising=False)
    monkeypatch.setattr(torch.cuda, 'device', Device)
    sequence_ops._launch(0, 'qcn_attn_window_step', b'a')
    sequence_ops._launch(3, 'qcn_attn_window_step', b'b')
    assert log == [(0, b'a', 70), (3, b'b', 73)] and now == [0]
    log.clear()
    sequence_ops._window_workspace.cache_clear()
    assert sequence_ops._window_workspace(2, 1, 1, 4, 4, 2, 2, 64, 9, 0) == 64 and log == [(2, 25 * 8)] and now == [0]
    sequence_ops._window_workspace.cache_clear()
    library.qcn_attn_window_step = lambda args, stream: INVALID
    with pytest.raises(_lib.QcnError, match='refused'):
        sequence_ops._launch(3, 'qcn_attn_window_step', b'c')
    assert now == [0]

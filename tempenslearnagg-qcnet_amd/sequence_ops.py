"""Token-sequence operators over the C ABI: rotary positions over several axes, attention with a sliding window and a few first
tokens that stay visible, and its bounded cache with the single-token form.

They are a family of their own for token sequences; the models' layers do not run on them.  The temporal attention of an agent
(modules/qcnet_agent_encoder.py:129-140) is a causal band over an edge list: 1 .. ``time_span`` steps back, the own step left out, with
a 512-byte positional row per edge added to k and v.  Here the band is a window over a ragged sequence that holds the own position
(``window=10``: that and the 9 before it), positions are rotations of q and k, and a new step costs one token
(:func:`attn_window_step`).  Forward only, like every operator of this package; the gradient of a rotation is the rotation with
``inverse=True``.

Row tensors are ``[tokens, heads, dim]`` in float32, float16 or bfloat16 and may be views (of a fused projection, for one): rows
whose features are contiguous and 16-byte aligned are read in place, anything else is copied first.  Scores, sums and softmax
statistics are float32 and every output is rounded once.  Softmax weights meet v unrounded, but for :func:`attn_window` in 16-bit types
with heads above 32 features (above 16 if window + sinks is above 17): the matrix units take them rounded to the type there, and
the error against 64 bits is 1.4 times that of rounding the output alone.  All of them launch on torch's current stream of the
tensors' device, allocate their outputs with torch, never synchronise, and can be captured into graphs.
"""
import functools
import struct
from typing import List, Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from .ops import _as_u8, _op, _register, _require

SEQUENCE_OP_NAMES: List[str] = []

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}          # QCN_DTYPE_*
_POS_TYPES = {torch.float32: 0, torch.int32: 1, torch.int64: 2}            # QCN_POS_*
MAX_HEAD_DIM = 128
_MOST = (1 << 62) - 1      # windows and sinks above it mean the same, and operators take 64 bits
_MOST_TOK = 1 << 24      # token stride in elements
_MAX_SCALE = 2.35e38      # times log2(e) it is still a float32
_NO_SECTIONS = (0,) * 8

# the argument structs of include/qcnet_hip.h (8-byte fields: no padding)
_ROTARY_ARGS = struct.Struct('=27q').pack
_WINDOW_ARGS = struct.Struct('=21qd3q').pack
_APPEND_ARGS = struct.Struct('=19q').pack
_STEP_ARGS = struct.Struct('=18qd6q').pack


# (names of this module: an attribute of a torch module costs as much as the question itself)
_Tensor = torch.Tensor
_compiling = torch.compiler.is_compiling
_grad_enabled = torch.is_grad_enabled
_dispatch_modes = torch._C._len_torch_dispatch_stack
_recording = torch._C._is_tracing
_transform = torch._C._functorch.peek_interpreter_stack


def _plain(*tensors) -> bool:
    """Whether the call can go to the implementation directly: plain tensors, nothing tracing, no function transform (its wrappers
    are of the plain type), nothing to differentiate in either direction.  The dispatcher costs 5 us a call, as much as everything
    else the host does for a decoding step; all of the above have to see the operator, and a launch past it is nothing to them."""
    if _compiling() or _dispatch_modes() or _recording() or _transform() is not None or forward_ad._current_level >= 0:
        return False
    grad = _grad_enabled()
    for t in tensors:
        if t is not None and (type(t) is not _Tensor or (grad and t.requires_grad)):
            return False
    return True


def _is(t, dtype: torch.dtype, index: int, shape) -> bool:
    return isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == index and t.shape == shape and t.is_contiguous()


def _rows(t: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device) -> None:
    """[tokens, heads, dim] of the wanted type and device, or the error."""
    if not torch.is_tensor(t):
        raise TypeError('%s must be a tensor' % name)
    if not t.is_cuda:
        raise _lib.QcnError('%s is on %s: the QCNet hot path runs on the GPU only (no CPU fallback)' % (name, t.device))
    if t.device != device:
        raise ValueError('%s is on %s, expected %s' % (name, t.device, device))
    if t.dtype != dtype:
        raise TypeError('%s has dtype %s, expected %s' % (name, t.dtype, dtype))
    if t.dim() != 3:
        raise ValueError('%s must be [tokens, heads, dim], got %s' % (name, tuple(t.shape)))


def _in_place(t: torch.Tensor):
    """(t, its strides) when its rows can be read in 16-byte pieces, else of a contiguous copy."""
    tok, head, feat = strides = t.stride()
    if feat == 1 and (tok | head) % (16 // t.element_size()) == 0 and tok < _MOST_TOK and t.data_ptr() % 16 == 0:
        return t, strides
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride()


# a contiguous tensor of the same shape and type (two thirds of new_empty's time, and a call for few tokens is the host's time)
_out_like = functools.partial(torch.empty_like, memory_format=torch.contiguous_format)


def _dtype_code(t: torch.Tensor, name: str) -> int:
    if not isinstance(t, torch.Tensor):
        raise TypeError('%s must be a tensor' % name)
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError('%s has dtype %s, expected float32, float16 or bfloat16' % (name, t.dtype))
    return code


def _on_device(index: int, fn, *args):
    """One C ABI call with the tensors' own device current."""
    if torch._C._cuda_getDevice() == index:
        return fn(*args)
    with torch.cuda.device(index):
        return fn(*args)


def _launch(index: int, what: str, args: bytes) -> None:
    """A launch on the tensors' own device and its current stream."""
    fn = getattr(_lib.lib(), what)
    if torch._C._cuda_getDevice() == index:
        status = fn(args, torch._C._cuda_getCurrentRawStream(index))
    else:
        status = _on_device(index, fn, args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status, what)


@functools.lru_cache(maxsize=1024)
def _step_workspace(index, batch, hq, hk, dim, window, sinks) -> int:
    """Bytes that a step of these sizes needs on this device; a serving loop asks for the same sizes every time."""
    return _on_device(index, _lib.lib().qcn_attn_window_step_workspace_bytes, batch, hq, hk, dim, window, sinks)


@functools.lru_cache(maxsize=1024)
def _window_workspace(index, code, n_seq, nq, nk, hq, hk, dim, window, sinks) -> int:
    args = _WINDOW_ARGS(*[0] * 12, n_seq, nq, nk, hq, hk, dim, code, window, sinks, 0.0, 0, 0, 0)
    return _on_device(index, _lib.lib().qcn_attn_window_workspace_bytes, args)


def _scale(scale: Optional[float], q: torch.Tensor) -> float:
    if scale is None:
        if not isinstance(q, torch.Tensor):
            raise TypeError('q must be a tensor')
        return max(q.size(-1) if q.dim() else 1, 1) ** -0.5
    scale = float(scale)
    if not 0 <= scale <= _MAX_SCALE:                          # (NaN is neither)
        raise ValueError('scale must be 0 .. %g, got %r' % (_MAX_SCALE, scale))
    return scale


# ------------------------------------------------------------------------------------------------
# rotary positions
# ------------------------------------------------------------------------------------------------
def rotary_embed(q: torch.Tensor, k: Optional[torch.Tensor], pos: torch.Tensor, freqs: torch.Tensor, sections: Sequence[int],
                 interleaved: bool = False, inverse: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """qcn_rotary_embed: q [N, Hq, D] and k [N, Hk, D] (or None) turned by their tokens' positions, as new contiguous tensors.

    ``pos`` [N, n_axes] (float32, int32 or int64): a position per axis — time, x, y of an agent, or time, height, width.
    ``sections``: how many feature pairs each axis turns, in order; ``freqs`` [sum(sections)] float32: radians per unit of
    position and pair.  Pair i is features (i, i + pairs), ``interleaved``: (2 i, 2 i + 1); features behind the pairs stay as
    they are.  Angles are formed in float64 (far positions keep their fraction of a turn).  ``inverse`` turns back."""
    sections = [int(s) for s in sections]
    call = _rotary_embed if _plain(q, k, pos, freqs) else _op('rotary_embed')
    out = call(q, k, pos, freqs, sections, bool(interleaved), bool(inverse))
    return out[0], (out[1] if k is not None else None)


def _rotary_embed_fake(q, k, pos, freqs, sections, interleaved, inverse):
    return [q.new_empty(q.shape)] + ([k.new_empty(k.shape)] if k is not None else [])


def _even_rows(t):
    """(t, its strides): any strides will do as long as a row's features are contiguous and no pair straddles its alignment."""
    tok, head, feat = strides = t.stride()
    if feat == 1 and not (tok | head) & 1 and t.data_ptr() % (2 * t.element_size()) == 0:
        return t, strides
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride()


@_register('rotary_embed', '(Tensor q, Tensor? k, Tensor pos, Tensor freqs, int[] sections, bool interleaved, bool inverse) -> Tensor[]',
           _rotary_embed_fake, SEQUENCE_OP_NAMES)
def _rotary_embed(q, k, pos, freqs, sections, interleaved, inverse):
    code = _dtype_code(q, 'q')
    dtype, index, shape = q.dtype, q.get_device(), q.shape
    if index < 0 or len(shape) != 3:
        _rows(q, 'q', dtype, q.device)
    n, hq, dim = shape
    if dim % 2 or not 2 <= dim <= 256:
        raise _lib.QcnError('head dim %d is not supported (even, 2 .. 256)' % dim)
    pairs, axes = sum(sections), len(sections)
    if not 1 <= axes <= 8 or min(sections) < 0 or pairs < 1 or 2 * pairs > dim:
        raise ValueError('sections %s: one to eight axes, at least one pair, at most dim / 2 = %d pairs' % (list(sections), dim // 2))
    pos_type = _POS_TYPES.get(pos.dtype) if isinstance(pos, torch.Tensor) else None
    if pos_type is None:
        raise TypeError('pos must be a float32, int32 or int64 tensor')
    if not _is(pos, pos.dtype, index, (n, axes)):
        _require(pos, 'pos', pos.dtype, q.device, (n, axes))
    if not _is(freqs, torch.float32, index, (pairs,)):
        _require(freqs, 'freqs', torch.float32, q.device, (pairs,))
    q, qs = _even_rows(q)
    q_out = _out_like(q)
    hk = kp = ks0 = ks1 = k_out_ptr = 0
    outs = [q_out]
    if k is not None:
        if not (isinstance(k, torch.Tensor) and k.dtype is dtype and k.get_device() == index and k.dim() == 3):
            _rows(k, 'k', dtype, q.device)
        nk, hk, dk = k.shape
        if nk != n or dk != dim:
            raise ValueError('k has shape %s, expected (%d, heads, %d)' % (tuple(k.shape), n, dim))
        if hk == 0:
            raise ValueError('k has no heads: pass None')
        k, (ks0, ks1, _) = _even_rows(k)
        kp = k.data_ptr()
        k_out = _out_like(k)
        k_out_ptr = k_out.data_ptr()
        outs.append(k_out)
    if n and (hq or hk):
        _launch(index, 'qcn_rotary_embed', _ROTARY_ARGS(
            q.data_ptr(), qs[0], qs[1], hq, kp, ks0, ks1, hk, n, dim, code, pos.data_ptr(), pos_type, axes,
            *sections, *_NO_SECTIONS[axes:], freqs.data_ptr(), interleaved, inverse, q_out.data_ptr(), k_out_ptr))
    return outs


# ------------------------------------------------------------------------------------------------
# attention over ragged sequences
# ------------------------------------------------------------------------------------------------
def _check_kv(k, v) -> int:
    """The type code of matching keys and values, or the error."""
    code = _dtype_code(k, 'k')
    dtype, index = k.dtype, k.get_device()
    ks = k.shape
    if not (index >= 0 and len(ks) == 3 and isinstance(v, torch.Tensor) and v.dtype is dtype and v.get_device() == index and v.shape == ks):
        _rows(k, 'k', dtype, k.device)
        _rows(v, 'v', dtype, k.device)
        raise ValueError('k and v differ in shape: %s and %s' % (tuple(ks), tuple(v.shape)))
    _, hk, dim = ks
    if dim % 8 or not 8 <= dim <= MAX_HEAD_DIM:
        raise _lib.QcnError('head dim %d is not supported (a multiple of 8, 8 .. %d)' % (dim, MAX_HEAD_DIM))
    if hk < 1:
        raise ValueError('k has no heads')
    return code


def _check_qkv(q, k, v) -> int:
    code = _check_kv(k, v)
    _, hk, dim = k.shape
    if not (isinstance(q, torch.Tensor) and q.dtype is k.dtype and q.get_device() == k.get_device() and q.dim() == 3):
        _rows(q, 'q', k.dtype, k.device)
    if q.size(2) != dim or q.size(1) < 1 or q.size(1) % hk:
        raise ValueError('q has shape %s: its dim must be %d and its heads a multiple of %d' % (tuple(q.shape), dim, hk))
    return code


def _mask_bytes(mask, name: str, index: int, device: torch.device, n: int):
    """A mask of n as bytes in memory: bool as it is, anything else as ops.py's masks are taken."""
    if _is(mask, torch.bool, index, (n,)):
        return mask
    if not isinstance(mask, torch.Tensor):
        raise TypeError('%s must be a tensor' % name)
    return _as_u8(mask, name, device, (n,))


def attn_window(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, window: int, sinks: int = 0,
                cu_k: Optional[torch.Tensor] = None, key_mask: Optional[torch.Tensor] = None,
                scale: Optional[float] = None) -> torch.Tensor:
    """qcn_attn_window: causal attention of ragged sequences, each position seeing the last ``window`` positions (itself among
    them) and the first ``sinks``; returns [Nq, Hq, D].

    q [Nq, Hq, D], k / v [Nk, Hkv, D] with Hq a multiple of Hkv; ``cu_q`` int64 [B + 1]: boundaries of the sequences in q
    (ascending from 0); ``cu_k``: those in k and v, if a sequence has keys in front of its queries (a chunk behind a prefix: the
    queries are its last positions).  ``key_mask`` bool [Nk]: false keys are seen by nobody, whatever k and v hold there.  A row
    that sees nothing is zero, and so are rows behind ``cu_q[-1]``.  ``scale`` defaults to D ** -0.5."""
    call = _attn_window if _plain(q, k, v, cu_q, cu_k, key_mask) else _op('attn_window')
    return call(q, k, v, cu_q, min(int(window), _MOST), min(int(sinks), _MOST), cu_k, key_mask, _scale(scale, q))


@_register('attn_window', '(Tensor q, Tensor k, Tensor v, Tensor cu_q, int window, int sinks, Tensor? cu_k, Tensor? key_mask, '
           'float scale) -> Tensor', lambda q, k, v, cu_q, window, sinks, cu_k, key_mask, scale: q.new_empty(q.shape),
           SEQUENCE_OP_NAMES)
def _attn_window(q, k, v, cu_q, window, sinks, cu_k, key_mask, scale):
    code = _check_qkv(q, k, v)
    index = k.get_device()
    nq, hq, dim = q.shape
    nk, hk, _ = k.shape
    if window < 1 or sinks < 0:
        raise ValueError('window must be at least 1 and sinks at least 0, got %d and %d' % (window, sinks))
    if not torch.is_tensor(cu_q) or cu_q.dim() != 1 or cu_q.numel() < 1:
        raise ValueError('cu_q must hold B + 1 boundaries')
    n_cu = cu_q.size(0)
    if not _is(cu_q, torch.int64, index, (n_cu,)):
        _require(cu_q, 'cu_q', torch.int64, k.device, (n_cu,))
    cu_k_ptr = cu_q.data_ptr()
    if cu_k is None:
        if nk != nq:
            raise ValueError('k has %d tokens and q %d: pass cu_k' % (nk, nq))
    else:
        if not _is(cu_k, torch.int64, index, (n_cu,)):
            _require(cu_k, 'cu_k', torch.int64, k.device, (n_cu,))
        cu_k_ptr = cu_k.data_ptr()
    mask_ptr = 0
    if key_mask is not None:
        key_mask = _mask_bytes(key_mask, 'key_mask', index, k.device, nk)
        mask_ptr = key_mask.data_ptr()
    scale = _scale(scale, q)
    q, qs = _in_place(q)
    k, ks = _in_place(k)
    v, vs = _in_place(v)
    out = _out_like(q)
    if nq:
        args = (q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], cu_q.data_ptr(), cu_k_ptr, mask_ptr,
                n_cu - 1, nq, nk, hq, hk, dim, code, window, sinks, scale, out.data_ptr())
        ws_ptr = ws_bytes = 0
        if code:                                            # 16-bit types: keys split over blocks when query tokens are few
            ws_bytes = _window_workspace(index, code, n_cu - 1, nq, nk, hq, hk, dim, window, sinks)
            if ws_bytes:
                ws = q.new_empty((ws_bytes,), dtype=torch.uint8)
                ws_ptr = ws.data_ptr()
        _launch(index, 'qcn_attn_window', _WINDOW_ARGS(*args, ws_ptr, ws_bytes))
    return out


# ------------------------------------------------------------------------------------------------
# the bounded cache
# ------------------------------------------------------------------------------------------------
def _written(k_cache, v_cache, mask_cache) -> None:
    """The caches have new contents: what autograd has saved of them is no longer what it was, and says so."""
    torch._C._increment_version((k_cache, v_cache) if mask_cache is None else (k_cache, v_cache, mask_cache))


def _check_cache(k, lengths, k_cache, v_cache, sinks, mask_cache, key_mask, batch):
    """(window, pointer of the mask cache) of a matching cache, or the error.  Caches are written in place: no copy stands in."""
    _, hk, dim = k.shape
    dtype, index = k.dtype, k.get_device()
    if sinks < 0:
        raise ValueError('sinks must be at least 0, got %d' % sinks)
    slots = k_cache.size(2) if torch.is_tensor(k_cache) and k_cache.dim() == 4 else -1
    shape = (batch, hk, slots, dim)
    if not (_is(k_cache, dtype, index, shape) and _is(v_cache, dtype, index, shape)):
        _require(k_cache, 'k_cache', dtype, k.device, (batch, hk, None, dim))
        _require(v_cache, 'v_cache', dtype, k.device, shape)
    if slots <= sinks:
        raise ValueError('the cache has %d slots: sinks + window, with a window of at least 1 behind %d sinks' % (slots, sinks))
    kp, vp = k_cache.data_ptr(), v_cache.data_ptr()
    if (kp | vp) % 16:
        raise ValueError('the caches must start on 16-byte boundaries')
    if abs(kp - vp) < k_cache.numel() * k_cache.element_size():
        raise ValueError('k_cache and v_cache share memory')
    if not _is(lengths, torch.int64, index, (batch,)):
        _require(lengths, 'lengths', torch.int64, k.device, (batch,))
    if mask_cache is not None:
        if not _is(mask_cache, torch.bool, index, (batch, slots)):
            if torch.is_tensor(mask_cache) and mask_cache.dtype == torch.bool:
                mask_cache = mask_cache.view(torch.uint8)
            _require(mask_cache, 'mask_cache', torch.uint8, k.device, (batch, slots))
        return slots - sinks, mask_cache.data_ptr()
    if key_mask is not None:
        raise ValueError('key_mask needs a mask_cache to keep it in')
    return slots - sinks, 0


def window_cache_append(k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, lengths: torch.Tensor, k_cache: torch.Tensor,
                        v_cache: torch.Tensor, sinks: int = 0, key_mask: Optional[torch.Tensor] = None,
                        mask_cache: Optional[torch.Tensor] = None) -> None:
    """qcn_window_cache_append: the tokens of B ragged sequences (k / v [N, Hkv, D], boundaries ``cu`` int64 [B + 1]) go into
    their caches [B, Hkv, sinks + window, D] (contiguous) behind the ``lengths`` [B] (int64) tokens each has seen.

    Position p lies in slot p (p < sinks) or sinks + (p - sinks) % window.  ``lengths`` is left as it is, so that the layers of a
    model share it: advance it once per call of the model.  Sequences with a negative length and rows behind ``cu[-1]`` are left
    alone.  ``mask_cache`` bool [B, sinks + window] takes ``key_mask`` [N] (true where that is None).  k and v may be views of other
    rows of the caches, but not of slots that the call writes."""
    call = _window_cache_append if _plain(k, v, cu, lengths, k_cache, v_cache, key_mask, mask_cache) else _op('window_cache_append')
    call(k, v, cu, lengths, k_cache, v_cache, int(sinks), key_mask, mask_cache)


@_register('window_cache_append', '(Tensor k, Tensor v, Tensor cu, Tensor lengths, Tensor(a!) k_cache, Tensor(b!) v_cache, int sinks, '
           'Tensor? key_mask, Tensor(c!)? mask_cache) -> ()',
           lambda k, v, cu, lengths, k_cache, v_cache, sinks, key_mask, mask_cache: None, SEQUENCE_OP_NAMES)
def _window_cache_append(k, v, cu, lengths, k_cache, v_cache, sinks, key_mask, mask_cache):
    code = _check_kv(k, v)
    index = k.get_device()
    n, hk, dim = k.shape
    if not torch.is_tensor(cu) or cu.dim() != 1 or cu.numel() < 1:
        raise ValueError('cu must hold B + 1 boundaries')
    batch = cu.size(0) - 1
    if not _is(cu, torch.int64, index, (batch + 1,)):
        _require(cu, 'cu', torch.int64, k.device, (batch + 1,))
    window, mask_cache_ptr = _check_cache(k, lengths, k_cache, v_cache, sinks, mask_cache, key_mask, batch)
    mask_ptr = 0
    if key_mask is not None:
        key_mask = _mask_bytes(key_mask, 'key_mask', index, k.device, n)
        mask_ptr = key_mask.data_ptr()
    k, ks = _in_place(k)
    v, vs = _in_place(v)
    if n and batch:
        _launch(index, 'qcn_window_cache_append', _APPEND_ARGS(
            k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], cu.data_ptr(), lengths.data_ptr(), mask_ptr, batch, n, hk, dim,
            code, window, sinks, k_cache.data_ptr(), v_cache.data_ptr(), mask_cache_ptr))
        _written(k_cache, v_cache, mask_cache)


def attn_window_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor, k_cache: torch.Tensor,
                     v_cache: torch.Tensor, sinks: int = 0, key_mask: Optional[torch.Tensor] = None,
                     mask_cache: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """qcn_attn_window_step: one new token per sequence.  k / v [B, Hkv, D] go into the caches at position ``lengths[b]`` and q
    [B, Hq, D] attends to what that position sees (:func:`attn_window`'s rule, out of the cache); returns [B, Hq, D].

    ``lengths`` is left as it is (see :func:`window_cache_append`).  A negative length marks a row that is not in use: its output
    is zero and its cache untouched.  ``key_mask`` bool [B]: whether the new token is visible, kept in ``mask_cache``.  q, k
    and v may not lie in slots that the call writes."""
    call = _attn_window_step if _plain(q, k, v, lengths, k_cache, v_cache, key_mask, mask_cache) else _op('attn_window_step')
    return call(q, k, v, lengths, k_cache, v_cache, int(sinks), key_mask, mask_cache, _scale(scale, q))


@_register('attn_window_step', '(Tensor q, Tensor k, Tensor v, Tensor lengths, Tensor(a!) k_cache, Tensor(b!) v_cache, int sinks, '
           'Tensor? key_mask, Tensor(c!)? mask_cache, float scale) -> Tensor',
           lambda q, k, v, lengths, k_cache, v_cache, sinks, key_mask, mask_cache, scale: q.new_empty(q.shape), SEQUENCE_OP_NAMES)
def _attn_window_step(q, k, v, lengths, k_cache, v_cache, sinks, key_mask, mask_cache, scale):
    code = _check_qkv(q, k, v)
    index = k.get_device()
    batch, hq, dim = q.shape
    hk = k.size(1)
    if k.size(0) != batch:
        raise ValueError('k has %d rows, expected %d' % (k.size(0), batch))
    window, mask_cache_ptr = _check_cache(k, lengths, k_cache, v_cache, sinks, mask_cache, key_mask, batch)
    mask_ptr = 0
    if key_mask is not None:
        key_mask = _mask_bytes(key_mask, 'key_mask', index, k.device, batch)
        mask_ptr = key_mask.data_ptr()
    scale = _scale(scale, q)
    q, qs = _in_place(q)
    k, ks = _in_place(k)
    v, vs = _in_place(v)
    out = _out_like(q)
    if batch:
        ws_bytes = _step_workspace(index, batch, hq, hk, dim, window, sinks)
        ws = q.new_empty((ws_bytes,), dtype=torch.uint8) if ws_bytes else None
        _launch(index, 'qcn_attn_window_step', _STEP_ARGS(
            q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], lengths.data_ptr(), mask_ptr, batch, hq,
            hk, dim, code, window, sinks, scale, k_cache.data_ptr(), v_cache.data_ptr(), mask_cache_ptr, out.data_ptr(),
            ws.data_ptr() if ws_bytes else 0, ws_bytes))
        _written(k_cache, v_cache, mask_cache)
    return out

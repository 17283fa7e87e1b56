"""Token-sequence operators over the C ABI: rotary positions over several axes, attention with a sliding window and a few first
tokens that stay visible, and its bounded cache with the single-token form.

They are the dense form of what the encoders do with edge lists: the temporal attention of an agent is a causal band of
``time_span`` steps (modules/qcnet_agent_encoder.py:129-140) whose positions enter through a 512-byte row per edge; here the
band is a window over a ragged token sequence, positions are rotations of q and k, and a new time step costs one token
(:func:`attn_window_step`) instead of a frame.  Forward only, like every operator of this package; the gradient of a rotation is
the rotation with ``inverse=True``.

Row tensors are ``[tokens, heads, dim]`` in float32, float16 or bfloat16 and may be views (of a fused projection, for one): rows
whose features are contiguous and 16-byte aligned are read in place, anything else is copied first.  Sums and softmax statistics
are float32 and every output is rounded once.  All of them launch on torch's current stream of the tensors' device, allocate
their outputs with torch, never synchronise, and can be captured into graphs.
"""
import ctypes
import math
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib
from .ops import _as_u8, _op, _ptr, _register, _require, _stream

SEQUENCE_OP_NAMES: List[str] = []

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}          # QCN_DTYPE_*
_POS_TYPES = {torch.float32: 0, torch.int32: 1, torch.int64: 2}            # QCN_POS_*
MAX_HEAD_DIM = 128


def _rows(t: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """[tokens, heads, dim] of the wanted type and device."""
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
    return t


def _in_place(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself when its rows can be read in 16-byte pieces, else a contiguous copy."""
    tok, head, feat = t.stride()
    piece = 16 // t.element_size()
    if feat == 1 and tok % piece == 0 and head % piece == 0 and t.data_ptr() % 16 == 0:
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _dtype_code(t: torch.Tensor, name: str) -> int:
    if t.dtype not in _DTYPES:
        raise TypeError('%s has dtype %s, expected float32, float16 or bfloat16' % (name, t.dtype))
    return _DTYPES[t.dtype]


def _head_dim(dim: int) -> None:
    if dim % 8 or not 8 <= dim <= MAX_HEAD_DIM:
        raise _lib.QcnError('head dim %d is not supported (a multiple of 8, 8 .. %d)' % (dim, MAX_HEAD_DIM))


def _launch(device: torch.device, what: str, *args) -> None:
    """One C ABI call on the tensors' own device."""
    fn = getattr(_lib.lib(), what)
    if torch.cuda.current_device() == device.index:
        _lib.check(fn(*args, _stream(device)), what)
    else:
        with torch.cuda.device(device):
            _lib.check(fn(*args, _stream(device)), what)


def _scale(scale: Optional[float], dim: int) -> float:
    scale = max(dim, 1) ** -0.5 if scale is None else float(scale)
    if not (math.isfinite(scale) and 0 <= scale <= 3e38):
        raise ValueError('scale must be finite and not negative, got %r' % scale)
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
    out = _op('rotary_embed')(q, k, pos, freqs, [int(s) for s in sections], bool(interleaved), bool(inverse))
    return out[0], (out[1] if k is not None else None)


def _rotary_embed_fake(q, k, pos, freqs, sections, interleaved, inverse):
    return [q.new_empty(q.shape)] + ([k.new_empty(k.shape)] if k is not None else [])


@_register('rotary_embed', '(Tensor q, Tensor? k, Tensor pos, Tensor freqs, int[] sections, bool interleaved, bool inverse) -> Tensor[]',
           _rotary_embed_fake, SEQUENCE_OP_NAMES)
def _rotary_embed(q, k, pos, freqs, sections, interleaved, inverse):
    dev = q.device
    code = _dtype_code(q, 'q')
    _rows(q, 'q', q.dtype, dev)
    n, hq, dim = q.shape
    if dim % 2 or not 2 <= dim <= 256:
        raise _lib.QcnError('head dim %d is not supported (even, 2 .. 256)' % dim)
    pairs, axes = sum(sections), len(sections)
    if not 1 <= axes <= 8 or any(s < 0 for s in sections) or pairs < 1 or 2 * pairs > dim:
        raise ValueError('sections %s: one to eight axes, at least one pair, at most dim / 2 = %d pairs' % (list(sections), dim // 2))
    if pos.dtype not in _POS_TYPES:
        raise TypeError('pos has dtype %s, expected float32, int32 or int64' % pos.dtype)
    _require(pos, 'pos', pos.dtype, dev, (n, axes))
    _require(freqs, 'freqs', torch.float32, dev, (pairs,))
    hk = 0
    if k is not None:
        _rows(k, 'k', q.dtype, dev)
        hk = k.size(1)
        if k.size(0) != n or k.size(2) != dim:
            raise ValueError('k has shape %s, expected (%d, heads, %d)' % (tuple(k.shape), n, dim))
        if hk == 0:
            raise ValueError('k has no heads: pass None')
    # any stride is fine as long as a row's features are contiguous and no pair straddles its alignment
    ok = lambda t: t.stride(2) == 1 and t.stride(0) % 2 == 0 and t.stride(1) % 2 == 0 and t.data_ptr() % (2 * t.element_size()) == 0
    q = q if ok(q) else q.clone(memory_format=torch.contiguous_format)
    q_out = torch.empty(n, hq, dim, dtype=q.dtype, device=dev)
    k_out = None
    if k is not None:
        k = k if ok(k) else k.clone(memory_format=torch.contiguous_format)
        k_out = torch.empty(n, hk, dim, dtype=q.dtype, device=dev)
    _launch(dev, 'qcn_rotary_embed', q.data_ptr(), q.stride(0), q.stride(1), hq, k.data_ptr() if hk else None,
            k.stride(0) if hk else 0, k.stride(1) if hk else 0, hk, n, dim, code, pos.data_ptr(), _POS_TYPES[pos.dtype], axes,
            freqs.data_ptr(), (ctypes.c_int32 * axes)(*sections), int(interleaved), int(inverse), q_out.data_ptr(),
            k_out.data_ptr() if hk else None)
    return [q_out] + ([k_out] if hk else [])


# ------------------------------------------------------------------------------------------------
# attention over ragged sequences
# ------------------------------------------------------------------------------------------------
def _check_kv(q, k, v):
    code = _dtype_code(k, 'k')
    dev = k.device
    _rows(k, 'k', k.dtype, dev)
    _rows(v, 'v', k.dtype, dev)
    if k.shape != v.shape:
        raise ValueError('k and v differ in shape: %s and %s' % (tuple(k.shape), tuple(v.shape)))
    _head_dim(k.size(2))
    if k.size(1) < 1:
        raise ValueError('k has no heads')
    if q is not None:
        _rows(q, 'q', k.dtype, dev)
        if q.size(2) != k.size(2) or q.size(1) < 1 or q.size(1) % k.size(1):
            raise ValueError('q has shape %s: its dim must be %d and its heads a multiple of %d' % (tuple(q.shape), k.size(2), k.size(1)))
    return code, dev


def attn_window(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, window: int, sinks: int = 0,
                cu_k: Optional[torch.Tensor] = None, key_mask: Optional[torch.Tensor] = None,
                scale: Optional[float] = None) -> torch.Tensor:
    """qcn_attn_window: causal attention of ragged sequences, each position seeing the last ``window`` positions (itself among
    them) and the first ``sinks``; returns [Nq, Hq, D].

    q [Nq, Hq, D], k / v [Nk, Hkv, D] with Hq a multiple of Hkv; ``cu_q`` int64 [B + 1]: boundaries of the sequences in q
    (ascending from 0); ``cu_k``: those in k and v, if a sequence has keys in front of its queries (a chunk behind a prefix: the
    queries are its last positions).  ``key_mask`` bool [Nk]: false keys are seen by nobody, whatever k and v hold there.  A row
    that sees nothing is zero, and so are rows behind ``cu_q[-1]``.  ``scale`` defaults to D ** -0.5."""
    return _op('attn_window')(q, k, v, cu_q, int(window), int(sinks), cu_k, key_mask, _scale(scale, q.size(-1)))


@_register('attn_window', '(Tensor q, Tensor k, Tensor v, Tensor cu_q, int window, int sinks, Tensor? cu_k, Tensor? key_mask, '
           'float scale) -> Tensor', lambda q, k, v, cu_q, window, sinks, cu_k, key_mask, scale: q.new_empty(q.shape),
           SEQUENCE_OP_NAMES)
def _attn_window(q, k, v, cu_q, window, sinks, cu_k, key_mask, scale):
    code, dev = _check_kv(q, k, v)
    nq, hq, dim = q.shape
    nk, hk = k.size(0), k.size(1)
    if window < 1 or sinks < 0:
        raise ValueError('window must be at least 1 and sinks at least 0, got %d and %d' % (window, sinks))
    _require(cu_q, 'cu_q', torch.int64, dev, (None,))
    if cu_q.numel() < 1:
        raise ValueError('cu_q must hold B + 1 boundaries')
    if cu_k is None:
        if nk != nq:
            raise ValueError('k has %d tokens and q %d: pass cu_k' % (nk, nq))
        cu_k = cu_q
    else:
        _require(cu_k, 'cu_k', torch.int64, dev, (cu_q.numel(),))
    if key_mask is not None:
        key_mask = _as_u8(key_mask, 'key_mask', dev, (nk,))
    scale = _scale(scale, dim)
    q, k, v = _in_place(q), _in_place(k), _in_place(v)
    out = torch.empty(nq, hq, dim, dtype=q.dtype, device=dev)
    _launch(dev, 'qcn_attn_window', q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
            v.stride(0), v.stride(1), cu_q.data_ptr(), cu_k.data_ptr(), key_mask.data_ptr() if key_mask is not None else None,
            cu_q.numel() - 1, nq, nk, hq, hk, dim, code, min(window, 1 << 62), min(sinks, 1 << 62), scale, out.data_ptr())
    return out


# ------------------------------------------------------------------------------------------------
# the bounded cache
# ------------------------------------------------------------------------------------------------
def _check_cache(k, lengths, k_cache, v_cache, sinks, mask_cache, key_mask, batch, dev):
    hk, dim = k.size(1), k.size(2)
    if sinks < 0:
        raise ValueError('sinks must be at least 0, got %d' % sinks)
    _require(k_cache, 'k_cache', k.dtype, dev, (batch, hk, None, dim))
    slots = k_cache.size(2)
    _require(v_cache, 'v_cache', k.dtype, dev, (batch, hk, slots, dim))
    if slots <= sinks:
        raise ValueError('the cache has %d slots: sinks + window, with a window of at least 1 behind %d sinks' % (slots, sinks))
    if k_cache.data_ptr() % 16 or v_cache.data_ptr() % 16:
        raise ValueError('the caches must start on 16-byte boundaries')
    if batch and k_cache.data_ptr() == v_cache.data_ptr():
        raise ValueError('k_cache and v_cache are the same memory')
    _require(lengths, 'lengths', torch.int64, dev, (batch,))
    if mask_cache is not None:
        if mask_cache.dtype == torch.bool:
            mask_cache = mask_cache.view(torch.uint8)
        _require(mask_cache, 'mask_cache', torch.uint8, dev, (batch, slots))      # written in place: no copy may stand in for it
    elif key_mask is not None:
        raise ValueError('key_mask needs a mask_cache to keep it in')
    return slots - sinks, mask_cache


def window_cache_append(k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, lengths: torch.Tensor, k_cache: torch.Tensor,
                        v_cache: torch.Tensor, sinks: int = 0, key_mask: Optional[torch.Tensor] = None,
                        mask_cache: Optional[torch.Tensor] = None) -> None:
    """qcn_window_cache_append: the tokens of B ragged sequences (k / v [N, Hkv, D], boundaries ``cu`` int64 [B + 1]) go into
    their caches [B, Hkv, sinks + window, D] (contiguous) behind the ``lengths`` [B] (int64) tokens each has seen.

    Position p lies in slot p (p < sinks) or sinks + (p - sinks) % window.  ``lengths`` is left as it is, so that the layers of a
    model share it: advance it once per call of the model.  Sequences with a negative length and rows behind ``cu[-1]`` are left
    alone.  ``mask_cache`` bool [B, sinks + window] takes ``key_mask`` [N] (true where that is None)."""
    _op('window_cache_append')(k, v, cu, lengths, k_cache, v_cache, int(sinks), key_mask, mask_cache)


@_register('window_cache_append', '(Tensor k, Tensor v, Tensor cu, Tensor lengths, Tensor(a!) k_cache, Tensor(b!) v_cache, int sinks, '
           'Tensor? key_mask, Tensor(c!)? mask_cache) -> ()',
           lambda k, v, cu, lengths, k_cache, v_cache, sinks, key_mask, mask_cache: None, SEQUENCE_OP_NAMES)
def _window_cache_append(k, v, cu, lengths, k_cache, v_cache, sinks, key_mask, mask_cache):
    code, dev = _check_kv(None, k, v)
    n, hk, dim = k.shape
    _require(cu, 'cu', torch.int64, dev, (None,))
    batch = cu.numel() - 1
    if batch < 0:
        raise ValueError('cu must hold B + 1 boundaries')
    window, mask_cache = _check_cache(k, lengths, k_cache, v_cache, sinks, mask_cache, key_mask, batch, dev)
    if key_mask is not None:
        key_mask = _as_u8(key_mask, 'key_mask', dev, (n,))
    k, v = _in_place(k), _in_place(v)
    _launch(dev, 'qcn_window_cache_append', k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
            cu.data_ptr(), lengths.data_ptr(), key_mask.data_ptr() if key_mask is not None else None, batch, n, hk, dim, code,
            window, sinks, k_cache.data_ptr(), v_cache.data_ptr(), mask_cache.data_ptr() if mask_cache is not None else None)


def attn_window_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor, k_cache: torch.Tensor,
                     v_cache: torch.Tensor, sinks: int = 0, key_mask: Optional[torch.Tensor] = None,
                     mask_cache: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """qcn_attn_window_step: one new token per sequence.  k / v [B, Hkv, D] go into the caches at position ``lengths[b]`` and q
    [B, Hq, D] attends to what that position sees (:func:`attn_window`'s rule, out of the cache); returns [B, Hq, D].

    ``lengths`` is left as it is (see :func:`window_cache_append`).  A negative length marks a row that is not in use: its output
    is zero and its cache untouched.  ``key_mask`` bool [B]: whether the new token is visible, kept in ``mask_cache``."""
    return _op('attn_window_step')(q, k, v, lengths, k_cache, v_cache, int(sinks), key_mask, mask_cache, _scale(scale, q.size(-1)))


@_register('attn_window_step', '(Tensor q, Tensor k, Tensor v, Tensor lengths, Tensor(a!) k_cache, Tensor(b!) v_cache, int sinks, '
           'Tensor? key_mask, Tensor(c!)? mask_cache, float scale) -> Tensor',
           lambda q, k, v, lengths, k_cache, v_cache, sinks, key_mask, mask_cache, scale: q.new_empty(q.shape), SEQUENCE_OP_NAMES)
def _attn_window_step(q, k, v, lengths, k_cache, v_cache, sinks, key_mask, mask_cache, scale):
    code, dev = _check_kv(q, k, v)
    batch, hq, dim = q.shape
    hk = k.size(1)
    if k.size(0) != batch:
        raise ValueError('k has %d rows, expected %d' % (k.size(0), batch))
    window, mask_cache = _check_cache(k, lengths, k_cache, v_cache, sinks, mask_cache, key_mask, batch, dev)
    if key_mask is not None:
        key_mask = _as_u8(key_mask, 'key_mask', dev, (batch,))
    scale = _scale(scale, dim)
    q, k, v = _in_place(q), _in_place(k), _in_place(v)
    out = torch.empty(batch, hq, dim, dtype=q.dtype, device=dev)
    ws_bytes = _lib.lib().qcn_attn_window_step_workspace_bytes(batch, hq, hk, dim, window, sinks)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    _launch(dev, 'qcn_attn_window_step', q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
            v.stride(0), v.stride(1), lengths.data_ptr(), key_mask.data_ptr() if key_mask is not None else None, batch, hq, hk, dim,
            code, window, sinks, scale, k_cache.data_ptr(), v_cache.data_ptr(),
            mask_cache.data_ptr() if mask_cache is not None else None, out.data_ptr(), ws.data_ptr() if ws is not None else None,
            ws_bytes)
    return out

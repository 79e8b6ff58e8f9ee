"""The cache operators (include/st_runtime.h) on torch tensors: what a model's attention does between its
Q/K/V projection and its output projection.

``KvCache`` holds keys and values with a sliding window and sinks, ``qk_norm_rope_append`` norms and
rotates the heads of new tokens and appends their keys and values, ``window_attention`` attends over the
cache. The calls launch on torch's current stream of the tensors' device, do not synchronize, and can be
captured into a graph. They have no gradients, and refuse tensors that ask for one where torch records
them. Bad arguments raise ValueError, a failing library RuntimeError; there is no fallback. torch is imported by the first use, and has to be the HIP runtime that the library is
loaded with: import torch before the first call into the library.
"""
from __future__ import annotations

import ctypes
import math

from . import runtime as _runtime

__all__ = ['KvCache', 'qk_norm_rope_append', 'window_attention']

_MOST = 1 << 30  # rows, slots: far below what 32-bit fields hold
GROUP = 32  # values that share a (scale, minimum) pair in a 4-bit cache
_F32, _F16, _BF16, _INT4 = range(4)


class _Cache(ctypes.Structure):
    _fields_ = [('streams', ctypes.c_int32), ('kv_heads', ctypes.c_int32), ('head_dim', ctypes.c_int32),
                ('window', ctypes.c_int32), ('sinks', ctypes.c_int32), ('ring', ctypes.c_int32),
                ('dtype', ctypes.c_int32), ('stream_stride', ctypes.c_int64), ('head_stride', ctypes.c_int64),
                ('slot_stride', ctypes.c_int64), ('keys', ctypes.c_void_p), ('values', ctypes.c_void_p),
                ('key_params', ctypes.c_void_p), ('value_params', ctypes.c_void_p), ('positions', ctypes.c_void_p)]


class _Rows(ctypes.Structure):
    _fields_ = [('tokens', ctypes.c_int32), ('max_tokens', ctypes.c_int32), ('offsets', ctypes.c_void_p)]


class _Append(ctypes.Structure):
    _fields_ = [('dtype', ctypes.c_int32), ('q_heads', ctypes.c_int32), ('q', ctypes.c_void_p), ('k', ctypes.c_void_p),
                ('v', ctypes.c_void_p), ('q_out', ctypes.c_void_p), ('q_strides', ctypes.c_int64 * 2),
                ('k_strides', ctypes.c_int64 * 2), ('v_strides', ctypes.c_int64 * 2), ('out_strides', ctypes.c_int64 * 2),
                ('q_gain', ctypes.c_void_p), ('k_gain', ctypes.c_void_p), ('epsilon', ctypes.c_float),
                ('rope_dims', ctypes.c_int32), ('rope_halves', ctypes.c_int32), ('inv_freq', ctypes.c_void_p),
                ('rope', ctypes.c_void_p)]


class _Attention(ctypes.Structure):
    _fields_ = [('dtype', ctypes.c_int32), ('q_heads', ctypes.c_int32), ('q', ctypes.c_void_p), ('out', ctypes.c_void_p),
                ('q_strides', ctypes.c_int64 * 2), ('out_strides', ctypes.c_int64 * 2), ('scale', ctypes.c_float),
                ('workspace', ctypes.c_void_p), ('workspace_bytes', ctypes.c_size_t)]


_torch = None
_types = {}
_stream = None  # device index -> torch's current stream, a hipStream_t


def _load():
    """torch and the library, sharing one HIP runtime."""
    global _torch, _stream
    if _torch is None:
        import torch
        lib = _runtime.library()
        with open('/proc/self/maps') as maps:
            loaded = {line.split()[-1] for line in maps if 'libamdhip64' in line}
        if len(loaded) > 1:
            raise RuntimeError('two HIP runtimes are loaded (' + ', '.join(sorted(loaded)) +
                               '): import torch before the first call into the library')
        _types.update({torch.float32: _F32, torch.float16: _F16, torch.bfloat16: _BF16})
        _stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
        _torch = torch
        return torch, lib
    return _torch, _runtime._lib


def _need(ok, message):
    if not ok:
        raise ValueError(message)


def _no_gradients(*tensors):
    if _torch.is_grad_enabled():
        _need(not any(t is not None and t.requires_grad for t in tensors),
              'the cache operators have no gradients: call them under torch.no_grad()')


def _sig(t):
    """All that the checks ask of a tensor argument but its address."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device(), t.requires_grad)


class KvCache:
    """Keys and values of `streams` streams with a sliding window: for each stream and key/value head
    `sinks` rows for the first positions, which stay visible, and a ring of window + max_tokens - 1 rows
    for those after them, max_tokens being the most new tokens that one call brings a stream. Position p
    lives in slot p where p < sinks, else in slot sinks + (p - sinks) mod ring.

    dtype: torch.float32, float16, bfloat16, or 'int4' (codes of 0..15 with an FP16 scale and minimum
    for each 32 values; head_dim a multiple of 32). `keys` and `values` are
    [streams, kv_heads, slots, head_dim] tensors; of a 4-bit cache uint8 [.., head_dim / 2], beside
    `key_params` and `value_params`, float16 [.., head_dim / 32, 2].

    `positions` (int64, [streams], on the device) counts the tokens that each stream has; -1 leaves a stream
    out of a call. The operators read it; :meth:`advance` adds a call's tokens once every layer has them (the
    layers of a model may share one tensor of positions). A cache keeps its tensors: write into them, none can
    be replaced."""

    def __init__(self, streams, kv_heads, head_dim, window, sinks=0, max_tokens=1, dtype=None, device=None, positions=None):
        torch, _ = _load()
        dtype = torch.float32 if dtype is None else dtype
        _need(dtype == 'int4' or dtype in _types, "dtype must be torch.float32, float16, bfloat16 or 'int4'")
        _need(min(streams, kv_heads, head_dim, window, max_tokens) >= 1 and sinks >= 0, 'sizes must be positive')
        device = torch.device('cuda' if device is None else device)
        shape = (streams, kv_heads, sinks + window + max_tokens - 1)
        params = [None, None]
        if dtype == 'int4':
            _need(head_dim % GROUP == 0, 'a 4-bit cache needs a head dimension that is a multiple of 32')
            rows = [torch.zeros((*shape, head_dim // 2), dtype=torch.uint8, device=device) for _ in range(2)]
            params = [torch.zeros((*shape, head_dim // GROUP, 2), dtype=torch.float16, device=device) for _ in range(2)]
        else:
            rows = [torch.zeros((*shape, head_dim), dtype=dtype, device=device) for _ in range(2)]
        if positions is None:
            positions = torch.zeros(streams, dtype=torch.int64, device=device)
        self._adopt(*rows, positions, window, sinks, *params)

    @classmethod
    def from_tensors(cls, keys, values, positions, *, window, sinks=0, key_params=None, value_params=None):
        """A cache over the caller's tensors, shaped as above. keys and values need the same strides, with
        rows of adjacent elements that start at multiples of 16 bytes; the params the same in rows."""
        _load()
        self = cls.__new__(cls)
        self._adopt(keys, values, positions, window, sinks, key_params, value_params)
        return self

    def _adopt(self, keys, values, positions, window, sinks, key_params, value_params):
        torch, _ = _load()
        _no_gradients(keys, values, key_params, value_params)
        int4 = key_params is not None or value_params is not None
        _need(keys.dim() == 4 and keys.shape == values.shape and keys.dtype == values.dtype,
              'keys and values must be tensors of one shape [streams, kv_heads, slots, row] and type')
        _need(keys.device.type == 'cuda' and values.device == keys.device, 'the cache must be on a GPU')
        streams, kv_heads, slots, row = keys.shape
        dim = row * 2 if int4 else row
        if int4:
            _need(keys.dtype == torch.uint8, 'a 4-bit cache holds its codes as uint8')
            for t in (key_params, value_params):
                _need(t is not None and t.dtype == torch.float16 and t.shape == (streams, kv_heads, slots, dim // GROUP, 2)
                      and t.device == keys.device and dim % GROUP == 0,
                      'a 4-bit cache needs key_params and value_params, float16 [streams, kv_heads, slots, head_dim / 32, 2]')
        else:
            _need(keys.dtype in _types, 'the cache must be float32, float16, bfloat16, or 4-bit with its params')
        _need(positions.dtype == torch.int64 and positions.shape == (streams,) and positions.is_contiguous()
              and positions.device == keys.device, 'positions must be int64 [streams] on the cache\'s device')
        window, sinks = int(window), int(sinks)
        ring = slots - sinks
        _need(window >= 1 and sinks >= 0 and ring >= window, 'a cache needs sinks + window slots at least')
        _need(slots <= _MOST, 'a cache has at most 2^30 slots')
        strides = self._row_strides(keys, row)
        _need(strides is not None and self._row_strides(values, row) == strides,
              'keys and values must have the same strides, in whole rows')
        for t in (key_params, value_params):
            _need(t is None or (t.stride(-1) == 1 and t.stride(-2) == 2 and
                                self._row_strides(t.flatten(-2), dim // GROUP * 2) == strides),
                  'the params must have the strides of the codes, in rows')
        self.keys, self.values, self.key_params, self.value_params = keys, values, key_params, value_params
        self.positions = positions
        self.streams, self.kv_heads, self.head_dim, self.slots = streams, kv_heads, dim, slots
        self.window, self.sinks, self.ring = window, sinks, ring
        self.max_tokens = ring - window + 1
        self.dtype = 'int4' if int4 else keys.dtype
        self.device = keys.device
        self._int4 = int4
        self._struct = _Cache(streams, kv_heads, dim, window, sinks, ring, _INT4 if int4 else _types[keys.dtype], *strides,
                              keys.data_ptr(), values.data_ptr(), key_params.data_ptr() if int4 else None,
                              value_params.data_ptr() if int4 else None, positions.data_ptr())
        self._address = ctypes.addressof(self._struct)
        self._plans = {}  # checked argument structs by the arguments' shapes, strides and types
        self._fixed = True

    def __setattr__(self, name, value):
        # The struct holds the tensors' addresses: one put in a tensor's place would never be read. (x += y on an
        # attribute assigns the tensor that is there, which is fine.)
        if getattr(self, '_fixed', False) and value is not getattr(self, name, None):
            raise AttributeError(f'{name} of a cache is fixed: write into its tensors')
        object.__setattr__(self, name, value)

    @staticmethod
    def _row_strides(t, row):
        """Strides of streams, heads and slots in rows, or None. Sizes of one have no stride of their own."""
        if t.stride(3) != 1 and row != 1:
            return None
        shape, out = t.shape, []
        for i, usual in ((0, shape[1] * shape[2]), (1, shape[2]), (2, 1)):
            s = t.stride(i) if shape[i] > 1 else usual * row
            if s % row or s <= 0:
                return None
            out.append(s // row)
        return tuple(out)

    def advance(self, tokens) -> None:
        """Add a call's tokens: a number for every stream, or an int64 tensor [streams]. Streams that are left
        out (negative positions) stay so."""
        self.positions.add_(_torch.where(self.positions < 0, 0, tokens))

    def reset(self, stream=None) -> None:
        """Forget one stream (all when None)."""
        if stream is None:
            self.positions.zero_()
        else:
            self.positions[stream] = 0

    def dequantized(self):
        """(keys, values) of every slot as float32, what the stored rows stand for."""
        if not self._int4:
            return self.keys.float(), self.values.float()
        torch = _torch
        out = []
        for codes, params in ((self.keys, self.key_params), (self.values, self.value_params)):
            b = codes.unflatten(-1, (-1, 4))
            lo, hi = b & 15, b >> 4
            c = torch.stack((lo[..., 0], lo[..., 2], hi[..., 0], hi[..., 2], lo[..., 1], lo[..., 3], hi[..., 1], hi[..., 3]), -1)
            c = c.flatten(-2).unflatten(-1, (-1, GROUP)).float()
            out.append((params[..., 1:].float() + params[..., :1].float() * c).flatten(-2))
        return tuple(out)

    def _rows(self, q, offsets, max_tokens):
        """(tokens, tokens per stream, row struct) of a call whose queries are q."""
        torch = _torch
        if offsets is None:
            _need(q.dim() == 4 and q.shape[0] == self.streams, 'without offsets q is [streams, tokens, heads, head_dim]')
            n = q.shape[1]
            _need(max_tokens is None or max_tokens == n, 'max_tokens goes with offsets')
            if n == 0:
                return 0, None
            _need(self.streams * n <= _MOST, 'a call has at most 2^30 tokens')
            return self.streams * n, _Rows(self.streams * n, n, None)
        _need(q.dim() == 3, 'with offsets q is [tokens, heads, head_dim]')
        _need(offsets.dtype == torch.int32 and offsets.shape == (self.streams + 1,) and offsets.is_contiguous()
              and offsets.device == self.device, 'offsets must be int32 [streams + 1] on the cache\'s device')
        _need(max_tokens is not None, 'offsets need max_tokens, the most tokens of one stream')
        _need(q.shape[0] <= _MOST and 1 <= max_tokens <= self.max_tokens,
              f'a call has at most 2^30 tokens, and this cache takes 1 to {self.max_tokens} of one stream')
        return q.shape[0], _Rows(q.shape[0], max_tokens, offsets.data_ptr())

    def _heads(self, t, like, heads, name, dtype):
        """Token and head strides of a [.., heads, head_dim] tensor whose leading sizes are `like`'s."""
        _need(t.dtype == dtype and t.device == self.device, f'{name} must be {dtype} on the cache\'s device')
        shape = t.shape
        _need(shape[:-2] == like.shape[:-2] and shape[-2] == heads and shape[-1] == self.head_dim,
              f'{name} must be [.., {heads}, {self.head_dim}] beside q')
        s = t.stride()
        _need(s[-1] == 1, f'{name} needs adjacent elements')
        if len(shape) == 4 and shape[0] > 1 and shape[1] > 1:
            _need(s[0] == s[1] * shape[1], f'the tokens of {name} must be evenly spaced over the streams')
            return s[1], s[2]
        return (s[0] if len(shape) == 4 and shape[0] > 1 else s[-3]), s[-2]

    def _plan(self, key, make):
        """The checked structs of a call; the same shapes, strides and types are checked once."""
        plan = self._plans.get(key)
        if plan is None:
            plan = make()
            if len(self._plans) >= 256:
                self._plans.clear()
            self._plans[key] = plan
        return plan


def _launch(device, call, *args):
    torch = _torch
    index = device.index
    if torch.cuda.current_device() == index:
        status = call(*args, _stream(index))
    else:
        with torch.cuda.device(device):
            status = call(*args, _stream(index))
    if status:
        message = _runtime._lib.st_last_error().decode() or f'libstamd error {status}'
        raise (ValueError if status == 1 else RuntimeError)(message)


def _plan_append(cache, q, k, v, q_gain, k_gain, inv_freq, rope, rope_dims, pairs, offsets, max_tokens, out):
    torch = _torch
    _no_gradients(q, k, v, q_gain, k_gain, inv_freq, rope, out)
    tokens, rows = cache._rows(q, offsets, max_tokens)
    dtype = q.dtype
    _need(dtype in _types, 'q must be float32, float16 or bfloat16')
    heads = q.shape[-2]
    _need(heads <= 65535, 'at most 65535 query heads')
    args = _Append()
    args.dtype, args.q_heads = _types[dtype], heads
    args.q_strides = cache._heads(q, q, heads, 'q', dtype)
    args.k_strides = cache._heads(k, q, cache.kv_heads, 'k', dtype)
    args.v_strides = cache._heads(v, q, cache.kv_heads, 'v', dtype)
    args.out_strides = cache._heads(out, q, heads, 'out', dtype)
    _need(pairs in ('adjacent', 'halves'), "pairs must be 'adjacent' or 'halves'")
    _need(inv_freq is None or rope is None, 'give inv_freq or rope, not both')
    if inv_freq is not None:
        _need(inv_freq.dtype == torch.float64 and inv_freq.dim() == 1 and inv_freq.is_contiguous()
              and inv_freq.device == cache.device, 'inv_freq must be float64 [rope_dims / 2] on the cache\'s device')
        half = inv_freq.shape[0]
    elif rope is not None:
        _need(rope.dtype == torch.float32 and rope.dim() == 3 and rope.shape[0] == tokens and rope.shape[2] == 2
              and rope.is_contiguous() and rope.device == cache.device,
              'rope must be float32 [rows, rope_dims / 2, 2] on the cache\'s device')
        half = rope.shape[1]
    else:
        half = 0
    _need(rope_dims is None or rope_dims == 2 * half, 'rope_dims must be twice the frequencies\' number')
    args.rope_dims, args.rope_halves = 2 * half, int(pairs == 'halves')
    for name, gain in (('q_gain', q_gain), ('k_gain', k_gain)):
        _need(gain is None or (gain.dtype == torch.float32 and gain.shape == (cache.head_dim,) and gain.is_contiguous()
                               and gain.device == cache.device), f'{name} must be float32 [head_dim] on the cache\'s device')
    return tokens, rows, args


def qk_norm_rope_append(cache, q, k, v, *, q_gain=None, k_gain=None, epsilon=1e-6, inv_freq=None, rope=None,
                        rope_dims=None, pairs='adjacent', offsets=None, max_tokens=None, out=None):
    """Norm, rotate and append new tokens in one pass; returns the rotated queries (into `out` if given,
    which may be q).

    q [streams, tokens, q_heads, head_dim], k and v [streams, tokens, kv_heads, head_dim], any even
    spacing of the tokens and heads (views of one projection's output, for instance); or, for unequal
    numbers of tokens, [rows, heads, head_dim] with `offsets` (int32 [streams + 1]: stream b has the rows
    offsets[b] .. offsets[b + 1] - 1) and `max_tokens`, the most of one stream.
    q_gain, k_gain: float32 [head_dim], the gains of each query's and key's RMS norm; None: no norm.
    The first rope_dims elements of each query and key are rotated by position * inv_freq (float64
    [rope_dims / 2]) or by the given rotations, `rope` (float32 [rows, rope_dims / 2, 2]: cos, sin);
    rope_dims follows from either, and neither means no rotation. pairs: 'adjacent' elements (2i, 2i + 1) or
    'halves' (i, i + rope_dims / 2)."""
    torch, lib = _load()
    _need(isinstance(cache, KvCache), 'cache must be a KvCache')
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    key = (_sig(q), _sig(k), _sig(v), _sig(q_gain), _sig(k_gain), _sig(inv_freq), _sig(rope), rope_dims, pairs, _sig(offsets),
           max_tokens, _sig(out), torch.is_grad_enabled())
    tokens, rows, args = cache._plan(key, lambda: _plan_append(cache, q, k, v, q_gain, k_gain, inv_freq, rope, rope_dims, pairs,
                                                               offsets, max_tokens, out))
    if not tokens:
        return out
    args = _Append.from_buffer_copy(args)
    args.q, args.k, args.v, args.q_out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    if q_gain is not None:
        args.q_gain = q_gain.data_ptr()
    if k_gain is not None:
        args.k_gain = k_gain.data_ptr()
    args.epsilon = epsilon
    if inv_freq is not None:
        args.inv_freq = inv_freq.data_ptr()
    elif rope is not None:
        args.rope = rope.data_ptr()
    if offsets is not None:
        rows = _Rows(rows.tokens, rows.max_tokens, offsets.data_ptr())
    _launch(cache.device, lib.st_qk_norm_rope_append, cache._address, ctypes.addressof(rows), ctypes.addressof(args))
    return out


def _plan_attention(cache, q, offsets, max_tokens, out):
    _no_gradients(q, out)
    tokens, rows = cache._rows(q, offsets, max_tokens)
    dtype = q.dtype
    _need(dtype in _types, 'q must be float32, float16 or bfloat16')
    heads = q.shape[-2]
    _need(heads <= 65535, 'at most 65535 query heads')
    args = _Attention()
    args.dtype, args.q_heads = _types[dtype], heads
    args.q_strides = cache._heads(q, q, heads, 'q', dtype)
    args.out_strides = cache._heads(out, q, heads, 'out', dtype)
    if tokens:
        size = ctypes.c_size_t(0)
        _launch(cache.device, lambda *a: _runtime._lib.st_window_attention_workspace(*a[:-1]), cache._address,
                ctypes.addressof(rows), heads, _types[dtype], ctypes.byref(size))
        args.workspace_bytes = size.value
    return tokens, rows, args


def window_attention(cache, q, *, scale=None, offsets=None, max_tokens=None, out=None):
    """Attention of new tokens' queries over the cache, which holds their keys and values already
    (:func:`qk_norm_rope_append`): each query sees the sinks and the last `window` positions up to its own.
    q, offsets, max_tokens and out as there, and q_heads a multiple of the cache's heads: query head h reads
    cache head h // (q_heads // kv_heads). scale: 1 / sqrt(head_dim) if None, positive. Float32 queries go with
    every cache, 16-bit ones with a cache of their own type or a 4-bit one."""
    torch, lib = _load()
    _need(isinstance(cache, KvCache), 'cache must be a KvCache')
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    key = (_sig(q), _sig(offsets), max_tokens, _sig(out), torch.is_grad_enabled())
    tokens, rows, args = cache._plan(key, lambda: _plan_attention(cache, q, offsets, max_tokens, out))
    if not tokens:
        return out
    args = _Attention.from_buffer_copy(args)
    args.q, args.out = q.data_ptr(), out.data_ptr()
    args.scale = 1.0 / math.sqrt(cache.head_dim) if scale is None else scale
    if args.workspace_bytes:
        workspace = torch.empty(args.workspace_bytes, dtype=torch.uint8, device=cache.device)
        args.workspace = workspace.data_ptr()
    if offsets is not None:
        rows = _Rows(rows.tokens, rows.max_tokens, offsets.data_ptr())
    _launch(cache.device, lib.st_window_attention, cache._address, ctypes.addressof(rows), ctypes.addressof(args))
    return out

"""Helpers of the cache operators' tests: device memory, streams and graphs of the HIP runtime that the
library is linked to, calls of the C ABI on numpy data, and the operators in 64 bits."""
import ctypes
import math

import numpy as np

from streamtx import library
from streamtx.cache import _Append, _Attention, _Cache, _Rows

F32, F16, BF16, INT4 = range(4)
# Half a step of each type, relative to the value.
STEP = {F32: 2.0**-24, F16: 2.0**-11, BF16: 2.0**-8}
NAMES = {F32: 'f32', F16: 'f16', BF16: 'bf16', INT4: 'int4'}
GROUP = 32


class Hip:
    """The few HIP calls that the tests make, each checked."""

    def __init__(self):
        library()
        self.lib = ctypes.CDLL('/opt/rocm/lib/libamdhip64.so')

    def __getattr__(self, name):
        fn = getattr(self.lib, name)

        def call(*args):
            status = fn(*args)
            assert status == 0, f'{name}: {status}'
        return call


_hip = None


def hip():
    global _hip
    if _hip is None:
        _hip = Hip()
    return _hip


def sync():
    hip().hipDeviceSynchronize()


class Device:
    """A numpy array's copy in device memory."""

    def __init__(self, data):
        data = np.ascontiguousarray(data)
        self.shape, self.dtype, self.nbytes = data.shape, data.dtype, data.nbytes
        p = ctypes.c_void_p()
        hip().hipMalloc(ctypes.byref(p), ctypes.c_size_t(max(data.nbytes, 256)))
        self.ptr = p.value
        self.put(data)

    def put(self, data):
        data = np.ascontiguousarray(data, dtype=self.dtype)
        assert data.nbytes == self.nbytes
        hip().hipMemcpy(ctypes.c_void_p(self.ptr), data.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(self.nbytes), 1)

    def get(self):
        out = np.empty(self.shape, self.dtype)
        sync()
        hip().hipMemcpy(out.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(self.ptr), ctypes.c_size_t(self.nbytes), 2)
        return out

    def __del__(self):
        if getattr(self, 'ptr', None):
            hip().lib.hipFree(ctypes.c_void_p(self.ptr))
            self.ptr = None


def encode(x, dtype):
    """float values rounded (nearest even) to a type's array."""
    x = np.asarray(x)
    if dtype == F32:
        return x.astype(np.float32)
    if dtype == F16:
        with np.errstate(over='ignore'):
            return x.astype(np.float16)
    u = x.astype(np.float32).view(np.uint32).astype(np.uint64)
    nan = ((u & 0x7f800000) == 0x7f800000) & ((u & 0x7fffff) != 0)
    r = (u + 0x7fff + ((u >> 16) & 1)) >> 16
    return np.where(nan, (u >> 16) | 0x40, r).astype(np.uint16)


def decode(a, dtype):
    if dtype == BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def pack(codes):
    c = codes.reshape(*codes.shape[:-1], -1, 4, 2).astype(np.uint8)
    e, o = c[..., 0], c[..., 1]
    return np.stack((e[..., 0] | e[..., 1] << 4, e[..., 2] | e[..., 3] << 4, o[..., 0] | o[..., 1] << 4,
                     o[..., 2] | o[..., 3] << 4), -1).reshape(*codes.shape[:-1], -1)


def unpack(packed):
    p = packed.reshape(*packed.shape[:-1], -1, 4)
    lo, hi = p & 15, p >> 4
    return np.stack((lo[..., 0], lo[..., 2], hi[..., 0], hi[..., 2], lo[..., 1], lo[..., 3], hi[..., 1], hi[..., 3]),
                    -1).reshape(*packed.shape[:-1], -1)


def quantise(x):
    """(codes, params) of rows of float32 values, in float32 as the format defines them."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, GROUP)
    low, high = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
    bad = ~np.isfinite(g).all(-1, keepdims=True)
    with np.errstate(all='ignore'):
        scale = ((high - low) / np.float32(15)).astype(np.float16)
        zero = low.astype(np.float16)
        s, z = scale.astype(np.float32), zero.astype(np.float32)
        code = np.where(s > 0, np.clip(np.rint((g - z) / s), 0, 15), 0)
    code = np.where(bad, 0, code).astype(np.uint8).reshape(x.shape)
    params = np.concatenate((np.where(bad, np.float16(np.nan), scale), np.where(bad, np.float16(np.nan), zero)), -1)
    return code, params


def dequantise(codes, params):
    c = codes.astype(np.float64).reshape(*codes.shape[:-1], -1, GROUP)
    p = params.astype(np.float64)
    return (p[..., 1:] + p[..., :1] * c).reshape(codes.shape)


def pointer(a):
    return a.ptr if a is not None else None


class Cache:
    """A cache in device memory. order: the axes of the allocation, outermost first, of (stream, head, slot)."""

    def __init__(self, streams, kv_heads, dim, window, sinks, dtype, max_tokens=1, fill=None, order=(0, 1, 2), positions=None):
        self.dims = (streams, kv_heads, sinks + window + max_tokens - 1)
        self.dim, self.window, self.sinks, self.ring, self.dtype = dim, window, sinks, window + max_tokens - 1, dtype
        self.order = order
        sizes = [self.dims[i] for i in order]
        strides = [0, 0, 0]
        for place, axis in enumerate(order):
            strides[axis] = int(np.prod(sizes[place + 1:], dtype=np.int64))
        rng = np.random.default_rng(0 if fill is None else fill)
        self.params = [None, None]
        if dtype == INT4:
            rows = [Device(self.stored(np.zeros((*self.dims, dim // 2), np.uint8))) for _ in range(2)]
            self.params = [Device(self.stored(np.zeros((*self.dims, dim // GROUP, 2), np.float16))) for _ in range(2)]
        else:
            rows = [Device(self.stored(encode(np.zeros((*self.dims, dim)), dtype))) for _ in range(2)]
        self.rows = rows
        self.positions = Device(np.zeros(streams, np.int64) if positions is None else np.asarray(positions, np.int64))
        if fill is not None:
            self.write(rng.standard_normal((*self.dims, dim)), rng.standard_normal((*self.dims, dim)) + 0.3)
        self.struct = _Cache(streams, kv_heads, dim, window, sinks, self.ring, dtype, *strides, rows[0].ptr, rows[1].ptr,
                             pointer(self.params[0]), pointer(self.params[1]), self.positions.ptr)

    def stored(self, a):
        """[stream, head, slot, ...] in the order of the allocation."""
        return np.ascontiguousarray(np.transpose(a, (*self.order, *range(3, a.ndim))))

    def seen(self, a):
        """The reverse."""
        return np.transpose(a, (*np.argsort(self.order), *range(3, a.ndim)))

    def write(self, keys, values):
        for i, x in enumerate((keys, values)):
            if self.dtype == INT4:
                codes, params = quantise(np.asarray(x, np.float32))
                self.rows[i].put(self.stored(pack(codes)))
                self.params[i].put(self.stored(params))
            else:
                self.rows[i].put(self.stored(encode(x, self.dtype)))

    def raw(self):
        """The stored arrays, [stream, head, slot, ...]."""
        out = [self.seen(r.get()) for r in self.rows]
        return out + [self.seen(p.get()) for p in self.params if p is not None]

    def values(self):
        """(keys, values) that the rows stand for, float64 [stream, head, slot, dim]."""
        out = []
        for i in range(2):
            a = self.seen(self.rows[i].get())
            out.append(dequantise(unpack(a), self.seen(self.params[i].get())) if self.dtype == INT4 else decode(a, self.dtype))
        return out

    def slot(self, p):
        return np.where(p < self.sinks, p, self.sinks + (p - self.sinks) % self.ring)


class Heads:
    """[rows, heads, dim] in device memory, possibly inside wider rows (pad: elements between heads and rows)."""

    def __init__(self, x, dtype, pad=0):
        self.data, self.dtype, self.pad = encode(x, dtype), dtype, pad
        n, h, d = self.data.shape
        wide = np.full((n, h + (1 if pad else 0), d + pad), 7 if dtype != BF16 else 0x40e0, self.data.dtype)
        wide[:, :h, :d] = self.data
        self.strides = (wide.shape[1] * wide.shape[2], wide.shape[2])
        self.n, self.h, self.d = n, h, d
        self.dev = Device(wide)
        self.ptr = self.dev.ptr

    def float(self):
        return decode(self.data, self.dtype)

    def get(self):
        """(values, whether everything around the rows is as it was)."""
        a = self.dev.get()
        around = a.copy()
        around[:, :self.h, :self.d] = 0
        mark = 7 if self.dtype != BF16 else 0x40e0
        keep = np.full_like(a, mark)
        keep[:, :self.h, :self.d] = 0
        return decode(a[:, :self.h, :self.d], self.dtype), bool((around == keep).all())


def rows_struct(cache, counts=None, n=None, offsets=None):
    """(struct, first row of each stream, total). counts: tokens of each stream (ragged), else n each."""
    streams = cache.dims[0]
    if counts is None:
        return _Rows(streams * n, n, None), [b * n for b in range(streams)], streams * n
    ends = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    return _Rows(int(ends[-1]), n, offsets.ptr), list(ends[:-1]), int(ends[-1])


def check(status):
    if status:
        raise RuntimeError(f'{status}: ' + library().st_last_error().decode())


def append(cache, rows, q, k, v, out, q_gain=None, k_gain=None, epsilon=1e-6, inv_freq=None, rope=None, rope_dims=0,
           halves=0, stream=None):
    a = _Append(q.dtype, q.h, q.ptr, k.ptr, v.ptr, out.ptr, q.strides, k.strides, v.strides, out.strides, pointer(q_gain),
                pointer(k_gain), epsilon, rope_dims, halves, pointer(inv_freq), pointer(rope))
    check(library().st_qk_norm_rope_append(ctypes.addressof(cache.struct), ctypes.addressof(rows), ctypes.addressof(a), stream))


def workspace_bytes(cache, rows, heads, dtype):
    need = ctypes.c_size_t(0)
    check(library().st_window_attention_workspace(ctypes.addressof(cache.struct), ctypes.addressof(rows), heads, dtype,
                                                  ctypes.byref(need)))
    return need.value


def attend(cache, rows, q, out, scale=None, stream=None, workspace=None):
    """Runs the attention; returns its workspace, which has to live until the work is done."""
    need = workspace_bytes(cache, rows, q.h, q.dtype)
    if workspace is None and need:
        workspace = Device(np.full(need, 0xff, np.uint8))  # NaN, wherever it is read before it is written
    scale = 1 / math.sqrt(cache.dim) if scale is None else scale
    a = _Attention(q.dtype, q.h, q.ptr, out.ptr, q.strides, out.strides, scale, pointer(workspace),
                   workspace.nbytes if workspace else 0)
    check(library().st_window_attention(ctypes.addressof(cache.struct), ctypes.addressof(rows), ctypes.addressof(a), stream))
    return workspace


def turned(x, gain, epsilon, angles, rope_dims, halves):
    """Norm and rotation in 64 bits: x [rows, heads, dim], angles [rows, rope_dims / 2]. Also the length of
    each element's pair, which errors of the rotation are relative to."""
    x = np.asarray(x, np.float64)
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + epsilon) * gain
    y, size = x.copy(), np.abs(x)
    h = rope_dims // 2
    if h:
        i, j = (np.arange(h), np.arange(h) + h) if halves else (2 * np.arange(h), 2 * np.arange(h) + 1)
        c, s = np.cos(angles)[:, None], np.sin(angles)[:, None]
        y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., i] * s + x[..., j] * c
        size[..., i] = size[..., j] = np.hypot(x[..., i], x[..., j])
    return y, size


def attention(cache_values, cache, q, starts, firsts, counts, scale):
    """softmax(scale q . K) V in 64 bits over what each query sees, row by row, and the bound's two
    ingredients: sum p |v| and the largest sum |q k| scale of a row."""
    keys, values = cache_values
    heads = q.shape[1]
    group = heads // cache.dims[1]
    out = np.full(q.shape, np.nan)
    mass = np.full(q.shape, np.nan)
    size = np.full(q.shape[:2], np.nan)
    for b, (start, first, n) in enumerate(zip(starts, firsts, counts)):
        if start < 0:
            continue
        for i in range(n):
            t = start + i
            low = max(t - cache.window + 1, 0)
            p = np.concatenate((np.arange(0, min(cache.sinks, low)), np.arange(low, t + 1)))
            at = cache.slot(p)
            for kv in range(cache.dims[1]):
                rows = q[first + i, kv * group:(kv + 1) * group]
                k, v = keys[b, kv, at], values[b, kv, at]
                x = rows @ k.T * scale
                w = np.exp(x - x.max(-1, keepdims=True))
                w /= w.sum(-1, keepdims=True)
                out[first + i, kv * group:(kv + 1) * group] = w @ v
                mass[first + i, kv * group:(kv + 1) * group] = w @ np.abs(v)
                size[first + i, kv * group:(kv + 1) * group] = (np.abs(rows) @ np.abs(k).T * abs(scale)).max(-1)
    return out, mass, size


def attention_bound(out, mass, size, keys, cache, dtype):
    """How far the kernel may be from the exact output of `keys` keys. Logits are sums of dim products in FP32
    accumulators, up to `size`, with six more roundings to scale and subtract them: dim + 6 roundings. A
    weight's relative error is its logit's error plus the exponential's (2^-22). The output is a quotient of
    two sums of `keys` such terms, numerator and denominator off alike: twice. 16-bit products round each
    weight once (half a step; FP16 also up to 2^-25 of the largest weight below its smallest normal number)
    and the output once. 4-bit rows that go to 16-bit products are rounded to FP16: keys within the
    logits, values within the sum. (Where a kernel takes weights or keys in two terms it is closer than that.)"""
    u = 2.0**-24
    top = max(np.abs(cache.values()[1]).max(), 1e-30)
    logit = (cache.dim + 6) * u * size[..., None]
    if dtype != F32 and cache.dtype == INT4:
        logit = logit + STEP[F16] * size[..., None]
    err = 2 * (logit + 2.0**-22 + (keys + 8) * u) * mass
    if dtype != F32:
        p = BF16 if dtype == BF16 and cache.dtype != INT4 else F16
        err = err + STEP[p] * mass + (keys * 2.0**-25 * top if p == F16 else 0)
        if cache.dtype == INT4:
            err = err + STEP[F16] * mass
    return err + STEP[dtype] * np.abs(out) + 1e-30

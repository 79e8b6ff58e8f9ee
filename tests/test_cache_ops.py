"""CPU checks of the cache operators' entry points: what they refuse, before any device work, and that they
never let a bad call through to the GPU."""
import ctypes
import subprocess
import sys
from pathlib import Path

import pytest

from streamtx import library
from streamtx.cache import _Append, _Attention, _Cache, _Rows

ROOT = Path(__file__).resolve().parent.parent
INVALID = 1
A = 1 << 20  # an aligned address that nothing reads
F32, F16, BF16, INT4 = range(4)
MOST = 2**31 - 1


def cache(**more):
    c = _Cache(2, 2, 64, 16, 1, 20, F32, 0, 0, 0, A, A, None, None, A)
    for k, v in more.items():
        setattr(c, k, v)
    return c


def rows(**more):
    r = _Rows(4, 2, None)
    for k, v in more.items():
        setattr(r, k, v)
    return r


def append_args(**more):
    a = _Append(F32, 4, A, A, A, A, (512, 64), (512, 64), (512, 64), (256, 64), None, None, 1e-6, 64, 0, A, None)
    for k, v in more.items():
        setattr(a, k, v)
    return a


def attention_args(**more):
    a = _Attention(F32, 4, A, A, (256, 64), (256, 64), 0.125, None, 0)
    for k, v in more.items():
        setattr(a, k, v)
    return a


def refused(c, r, a, match):
    lib = library()
    call = lib.st_qk_norm_rope_append if isinstance(a, _Append) else lib.st_window_attention
    pointers = [ctypes.addressof(x) if x is not None else None for x in (c, r, a)]
    assert call(*pointers, None) == INVALID, match
    assert match in lib.st_last_error().decode()


CACHES = [
    (dict(streams=0), 'streams and heads'), (dict(streams=65536), 'streams and heads'), (dict(kv_heads=0), 'streams and heads'),
    (dict(head_dim=0), 'head dimension'), (dict(head_dim=60), 'head dimension'), (dict(head_dim=264), 'head dimension'),
    (dict(dtype=4), 'cache type'), (dict(dtype=-1), 'cache type'),
    (dict(window=0), 'window'), (dict(window=21), 'window'), (dict(sinks=-1), 'window'), (dict(ring=MOST), 'window'),
    (dict(ring=2**30, window=2**30, sinks=1), 'window'),
    (dict(keys=None), 'Null'), (dict(values=None), 'Null'), (dict(positions=None), 'Null'),
    (dict(keys=A + 8), 'Misaligned'), (dict(values=A + 2), 'Misaligned'), (dict(positions=A + 4), 'Misaligned'),
    (dict(dtype=INT4), 'scales'), (dict(dtype=INT4, key_params=A, value_params=A + 2), 'scales'),
    (dict(dtype=INT4, key_params=A, value_params=A, head_dim=80), 'multiple of 32'),
    (dict(stream_stride=1), 'strides'), (dict(slot_stride=-1), 'strides'), (dict(slot_stride=1, stream_stride=21), 'strides'),
    (dict(slot_stride=2**24, head_stride=1, stream_stride=1), 'strides'),
    (dict(slot_stride=1, head_stride=-1, stream_stride=1), 'strides'),
    (dict(slot_stride=1, head_stride=1, stream_stride=2**40), 'strides'),
]
ROWS = [
    (dict(tokens=-1), 'tokens'), (dict(tokens=MOST, offsets=A), 'tokens'), (dict(max_tokens=0), 'tokens'), (dict(max_tokens=-5), 'tokens'),
    (dict(tokens=3), 'Without offsets'), (dict(tokens=12, max_tokens=6), 'beside the window'),
    (dict(max_tokens=MOST), 'beside the window'), (dict(offsets=A + 2), 'offsets'),
]


@pytest.mark.parametrize('change,match', CACHES, ids=str)
def test_caches_refused(change, match):
    refused(cache(**change), rows(), append_args(), match)
    refused(cache(**change), rows(), attention_args(), match)
    need = ctypes.c_size_t(7)
    c, r = cache(**change), rows()
    assert library().st_window_attention_workspace(ctypes.addressof(c), ctypes.addressof(r), 4, F32, ctypes.byref(need)) == INVALID
    assert need.value == 7


@pytest.mark.parametrize('change,match', ROWS, ids=str)
def test_rows_refused(change, match):
    refused(cache(), rows(**change), append_args(), match)
    refused(cache(), rows(**change), attention_args(), match)


@pytest.mark.parametrize('change,match', [
    (dict(dtype=3), 'element type'), (dict(dtype=F16), 'own type'), (dict(dtype=BF16), 'own type'),
    (dict(q_heads=0), 'multiple'), (dict(q_heads=3), 'multiple'), (dict(q_heads=65536), 'multiple'),
    (dict(q=None), 'Null'), (dict(k=None), 'Null'), (dict(v=None), 'Null'), (dict(q_out=None), 'Null'),
    (dict(q=A + 4), 'multiples of 16'), (dict(k=A + 8), 'multiples of 16'), (dict(q_out=A + 8), 'multiples of 16'),
    (dict(q_strides=(510, 64)), 'multiples of 16'), (dict(v_strides=(512, 66)), 'multiples of 16'),
    (dict(k_strides=(2**40, 64)), 'Stride'), (dict(out_strides=(0, 64)), 'overlap'), (dict(out_strides=(256, 0)), 'overlap'),
    (dict(q_gain=A, epsilon=0.0), 'epsilon'), (dict(k_gain=A, epsilon=-1.0), 'epsilon'), (dict(k_gain=A, epsilon=1e-40), 'epsilon'),
    (dict(k_gain=A, epsilon=float('nan')), 'epsilon'), (dict(q_gain=A, epsilon=float('inf')), 'epsilon'),
    (dict(rope_dims=66), 'Rotated'), (dict(rope_dims=31), 'Rotated'), (dict(rope_dims=-2), 'Rotated'),
    (dict(rope_halves=2), 'rope_halves'), (dict(inv_freq=None), 'frequencies'), (dict(rope=A), 'frequencies'),
], ids=str)
def test_append_arguments_refused(change, match):
    refused(cache(), rows(), append_args(**change), match)


@pytest.mark.parametrize('change,match', [
    (dict(dtype=3), 'element type'), (dict(dtype=F16), 'own type'), (dict(q_heads=5), 'multiple'),
    (dict(q=None), 'Null'), (dict(out=None), 'Null'), (dict(q=A + 8), 'multiples of 16'), (dict(out=A + 4), 'multiples of 16'),
    (dict(out_strides=(256, 3)), 'multiples of 16'), (dict(out_strides=(0, 64)), 'overlap'),
    (dict(scale=float('nan')), 'scale'), (dict(scale=float('inf')), 'scale'),
    (dict(scale=0.0), 'scale'), (dict(scale=-0.125), 'scale'),
], ids=str)
def test_attention_arguments_refused(change, match):
    refused(cache(), rows(), attention_args(**change), match)


def test_null_structs_and_workspaces_refused():
    for missing in range(3):
        for a in (append_args(), attention_args()):
            items = [cache(), rows(), a]
            keep, items[missing] = items[missing], None
            lib = library()
            call = lib.st_qk_norm_rope_append if isinstance(a, _Append) else lib.st_window_attention
            assert call(*[ctypes.addressof(x) if x is not None else None for x in items], None) == INVALID
            assert 'Null' in lib.st_last_error().decode()
            del keep
    # One stream with a long window is split: it needs a workspace.
    c, r = cache(streams=1, kv_heads=1, window=100000, ring=100000), rows(tokens=1, max_tokens=1)
    need = ctypes.c_size_t(0)
    assert library().st_window_attention_workspace(ctypes.addressof(c), ctypes.addressof(r), 1, F32, ctypes.byref(need)) == 0
    assert need.value > 0
    a = dict(q_heads=1, q_strides=(64, 64), out_strides=(64, 64))
    refused(c, r, attention_args(**a), 'Workspace')
    refused(c, r, attention_args(**a, workspace=A, workspace_bytes=need.value - 1), 'Workspace')
    refused(c, r, attention_args(**a, workspace=A + 8, workspace_bytes=need.value), 'Workspace')
    refused(cache(ring=2**29, window=16), rows(tokens=2**30 - 30, max_tokens=2**29 - 15), attention_args(q_heads=16), 'Too many rows')


def test_no_tokens_is_no_work():
    c, r = cache(), rows(tokens=0, offsets=A)
    a, b = append_args(q=None, k=None, v=None, q_out=None), attention_args(q=None, out=None)
    lib = library()
    assert lib.st_qk_norm_rope_append(ctypes.addressof(c), ctypes.addressof(r), ctypes.addressof(a), None) == 0
    assert lib.st_window_attention(ctypes.addressof(c), ctypes.addressof(r), ctypes.addressof(b), None) == 0


TORCH = '''
import torch
from streamtx import KvCache, qk_norm_rope_append, window_attention

def refused(call, match):
    try:
        call()
    except ValueError as e:
        assert match in str(e), (match, e)
    else:
        raise AssertionError(match)

z = torch.zeros
refused(lambda: KvCache.from_tensors(z(1, 1, 8, 64), z(1, 1, 8, 64), z(1, dtype=torch.int64), window=8), 'GPU')
refused(lambda: KvCache.from_tensors(z(1, 8, 64), z(1, 8, 64), z(1, dtype=torch.int64), window=8), 'shape')
refused(lambda: KvCache.from_tensors(z(1, 1, 8, 64), z(1, 1, 9, 64), z(1, dtype=torch.int64), window=8), 'shape')
refused(lambda: KvCache(1, 1, 64, 0, device='cpu'), 'positive')
refused(lambda: KvCache(1, 1, 64, 4, sinks=-1, device='cpu'), 'positive')
refused(lambda: KvCache(1, 1, 64, 4, dtype=torch.float64, device='cpu'), 'dtype')
refused(lambda: KvCache(1, 1, 80, 4, dtype='int4', device='cpu'), 'multiple of 32')
refused(lambda: KvCache(1, 1, 64, 4, device='cpu'), 'GPU')
refused(lambda: qk_norm_rope_append(None, z(1), z(1), z(1)), 'KvCache')
refused(lambda: window_attention(z(1), z(1)), 'KvCache')
print('ok')
'''


def test_torch_binding_refuses_without_a_gpu():
    """In a process of its own: torch brings its HIP runtime, which has to be the library's."""
    out = subprocess.run([sys.executable, '-c', TORCH], capture_output=True, text=True, timeout=300,
                         cwd=ROOT / 'streaming-transformer_amd')
    assert out.returncode == 0 and out.stdout.strip() == 'ok', out.stderr[-2000:]


def test_two_hip_runtimes_refused():
    code = ('from streamtx import library, KvCache\nlibrary()\ntry:\n    KvCache(1, 1, 64, 4)\n'
            "except RuntimeError as e:\n    assert 'two HIP runtimes' in str(e)\n    print('ok')\n")
    out = subprocess.run([sys.executable, '-c', code], capture_output=True, text=True, timeout=300,
                         cwd=ROOT / 'streaming-transformer_amd')
    assert out.returncode == 0 and out.stdout.strip() == 'ok', out.stderr[-2000:]

"""CPU checks of st_batch_create_with: what it refuses, before any device work, and checkpoints with head norms."""
import ctypes

import numpy as np
import pytest

from streamtx import (BatchOptions, BatchRuntime, ModelConfig, WeightStorage, library, load_checkpoint, synthetic_checkpoint,
                      tensor_names, write_checkpoint)
from streamtx.runtime import _BatchOptions

CONFIG = ModelConfig(1, 64, 2, 128, 16, 32)


def refused(match, config=CONFIG, mixed=False, tensors=None, streams=2, **options):
    w = synthetic_checkpoint(config, seed=0, mixed=mixed) if tensors is None else tensors
    with pytest.raises(RuntimeError, match=match):
        BatchRuntime((config, w, mixed), streams, options=BatchOptions(**options))


@pytest.mark.parametrize('options,match', [
    (dict(sinks=-1), 'Sinks'), (dict(sinks=4097), 'Sinks'), (dict(head_norm=2), 'head_norm'),
    (dict(kv_dtype=4), 'K/V storage'), (dict(kv_dtype=-2), 'K/V storage'), (dict(weight_dtype=7), 'weight storage'),
])
def test_options_refused(options, match):
    refused(match, **options)


def test_combinations_refused():
    refused('FP32 checkpoints', mixed=True, sinks=1)
    refused('FP32 checkpoints', mixed=True, kv_dtype=1)
    refused('multiple of 8', ModelConfig(1, 48, 4, 64, 16, 32), sinks=1)
    refused('multiple of 8', ModelConfig(1, 1024, 2, 64, 16, 32), sinks=1)
    refused('multiple of 32', ModelConfig(1, 96, 2, 128, 16, 32), kv_dtype=3)
    refused('between 1 and 256', streams=0, sinks=1)
    with_norms = dict(synthetic_checkpoint(CONFIG, seed=0), **{'layers.0.q_norm': np.ones(32, np.float32)})
    refused('head norms', tensors=with_norms)
    w = synthetic_checkpoint(CONFIG, seed=0)
    for more in (dict(resident=True), dict(weight_dtype=WeightStorage.BF16)):
        with pytest.raises(ValueError, match='options'):
            BatchRuntime((CONFIG, w, False), 2, options=BatchOptions(), **more)


def test_head_norms_refuse_an_epsilon_below_normal_numbers():
    w = dict(synthetic_checkpoint(CONFIG, seed=0), **{f'layers.0.{n}': np.ones(32, np.float32) for n in ('q_norm', 'k_norm')})
    refused('epsilon', ModelConfig(1, 64, 2, 128, 16, 32, epsilon=1e-38), tensors=w, head_norm=1)


def test_default_options():
    o = _BatchOptions(9, 9, 9, 9)
    library().st_batch_options_default(ctypes.byref(o))
    assert (o.weight_dtype, o.sinks, o.head_norm, o.kv_dtype) == (0, 0, 0, -1)
    library().st_batch_options_default(None)


def test_checkpoint_with_head_norms(tmp_path):
    w = synthetic_checkpoint(CONFIG, seed=0)
    plain = write_checkpoint(tmp_path / 'plain', CONFIG, w)
    assert [n for n, _ in tensor_names(CONFIG)] == list(load_checkpoint(plain).tensors)
    for n in ('q_norm', 'k_norm'):
        w[f'layers.0.{n}'] = np.linspace(0.5, 1.5, 32, dtype=np.float32)
    ck = load_checkpoint(write_checkpoint(tmp_path / 'norms', CONFIG, w))
    np.testing.assert_array_equal(ck.tensors['layers.0.k_norm'], w['layers.0.k_norm'])
    w['layers.0.k_norm'] = np.ones(16, np.float32)
    with pytest.raises(ValueError, match='k_norm'):
        load_checkpoint(write_checkpoint(tmp_path / 'bad', CONFIG, w))

"""Host side of the MI355X streaming-step backend (libstamd.so).

streamtx.model    checkpoint format, config validation, synthetic checkpoints
streamtx.runtime  ctypes binding of the C ABI (include/st_runtime.h), mirroring Stream::Runtime
streamtx.cache    cache operators on torch tensors: norm, rotation and append; windowed attention
streamtx.numerical acceptance metrics of the reference (include/Numerical.hpp, reference/numerical.py)
streamtx.build    hipcc build of libstamd.so for gfx950
"""
from .cache import KvCache, qk_norm_rope_append, window_attention
from .model import (Checkpoint, ModelConfig, load_checkpoint, round_bf16, round_half, synthetic_checkpoint,
                    tensor_names, write_checkpoint)
from .runtime import Backend, BatchOptions, BatchRuntime, KvStorage, Runtime, RuntimeOptions, WeightStorage, library, probe, transport_bench

__all__ = ['Backend', 'BatchOptions', 'BatchRuntime', 'Checkpoint', 'KvCache', 'KvStorage', 'ModelConfig', 'Runtime', 'RuntimeOptions', 'WeightStorage', 'library',
           'load_checkpoint', 'probe', 'qk_norm_rope_append', 'transport_bench', 'window_attention', 'round_bf16', 'round_half', 'synthetic_checkpoint', 'tensor_names',
           'write_checkpoint']

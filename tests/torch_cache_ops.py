"""The torch binding of the cache operators, run in a process of its own (torch brings its HIP runtime):
prints 'ok' when everything holds. Run by test_cache_ops_torch_gpu.py."""
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / 'streaming-transformer_amd'))

from streamtx import KvCache, qk_norm_rope_append, window_attention  # noqa: E402

DEV = torch.device('cuda', 0)
STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def exact(cache, q, starts, scale):
    """q [streams, n, heads, dim] over the cache as it stands, in 64 bits."""
    keys, values = (t.double() for t in cache.dequantized())
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    group = q.shape[2] // cache.kv_heads
    for b, s in enumerate(starts):
        for i in range(q.shape[1]):
            t = s + i
            low = max(t - cache.window + 1, 0)
            p = torch.tensor([*range(min(cache.sinks, low)), *range(low, t + 1)], device=DEV)
            at = torch.where(p < cache.sinks, p, cache.sinks + (p - cache.sinks) % cache.ring)
            for h in range(q.shape[2]):
                k, v = keys[b, h // group, at], values[b, h // group, at]
                out[b, i, h] = torch.softmax(k @ q[b, i, h].double() * scale, 0) @ v
    return out


def close(got, want, dtype, what):
    # Weights and the output rounded once each, 4-bit rows once more, FP32 sums beside them; values up to 5.
    bound = (4 * STEP[dtype] + 2.0**-18) * 5
    err = (got.double() - want).abs().max().item()
    assert err <= bound, (what, err, bound)


def generation(dtype, stored, shared_positions):
    """Two layers over a prompt, then steps: views of one projection as inputs, advance between calls."""
    torch.manual_seed(1)
    streams, heads, kv, dim, window, sinks, n = 3, 6, 2, 64, 20, 2, 11
    positions = torch.zeros(streams, dtype=torch.int64, device=DEV)
    caches = [KvCache(streams, kv, dim, window, sinks, n, stored, DEV, positions) for _ in range(2)]
    assert caches[0].positions is caches[1].positions and caches[0].max_tokens == n
    gains = [torch.randn(dim, device=DEV) * 0.1 + 1 for _ in range(2)]
    freq = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEV) / dim)
    start = 0
    for tokens in (n, 1, 1, 5, 1, n, n, 1):
        for c in caches:
            x = torch.randn(streams, tokens, heads + 2 * kv, dim, device=DEV).to(dtype)
            q, k, v = x.split((heads, kv, kv), 2)
            rot = qk_norm_rope_append(c, q, k, v, q_gain=gains[0], k_gain=gains[1], inv_freq=freq, pairs='halves')
            out = window_attention(c, rot)
            close(out, exact(c, rot, [start] * streams, 1 / math.sqrt(dim)), dtype, (dtype, stored, start))
        start += tokens
        caches[0].advance(tokens)
    assert positions.tolist() == [start] * streams
    caches[0].reset(1)
    assert positions.tolist() == [start, 0, start]
    positions[2] = -1
    caches[0].advance(torch.tensor([1, 2, 3], device=DEV))
    assert positions.tolist() == [start + 1, 2, -1]


def other_stream():
    """The work goes to torch's current stream, where it waits for what that stream does before."""
    torch.manual_seed(2)
    c = KvCache(2, 2, 128, 5000, 4, dtype=torch.bfloat16, device=DEV)
    for t in (c.keys, c.values):
        t.copy_(torch.randn(t.shape, device=DEV))
    c.positions.fill_(9000)
    q = torch.randn(2, 1, 8, 128, device=DEV).bfloat16()
    want = window_attention(c, q)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(5):
        late = torch.zeros_like(q)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            torch.cuda._sleep(20_000_000)
            late.copy_(q)
            got = window_attention(c, late)
        s.synchronize()
        assert torch.equal(got, want)


def captured():
    """A decoding step in a graph: positions advance inside it; eager work of the same cache between."""
    torch.manual_seed(3)
    dim, heads, kv = 64, 4, 2
    freq = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEV) / dim)
    caches = [KvCache(2, kv, dim, 4096, 2, dtype='int4', device=DEV) for _ in range(2)]
    x = torch.randn(2, 1, heads + 2 * kv, dim, device=DEV).half()

    def step(c):
        q, k, v = x.split((heads, kv, kv), 2)
        out = window_attention(c, qk_norm_rope_append(c, q, k, v, inv_freq=freq))
        c.advance(1)
        return out

    for c in caches:
        for _ in range(3):
            step(c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0])
    for i in range(8):
        x.copy_(torch.randn(x.shape, device=DEV))
        graph.replay()
        want = step(caches[1])
        assert torch.equal(out, want), i
        if i == 4:  # a step of the captured cache outside of its graph
            x.copy_(torch.randn(x.shape, device=DEV))
            assert torch.equal(step(caches[0]), step(caches[1]))
    assert caches[0].positions.tolist() == caches[1].positions.tolist() == [12, 12]
    for a, b in ((caches[0].keys, caches[1].keys), (caches[0].value_params, caches[1].value_params)):
        assert torch.equal(a, b)


def refusals():
    c = KvCache(2, 2, 64, 8, 1, 3, torch.float16, DEV)
    z = lambda *s, d=torch.float16: torch.zeros(s, dtype=d, device=DEV)  # noqa: E731
    f = torch.ones(32, dtype=torch.float64, device=DEV)
    q, k = z(2, 1, 4, 64), z(2, 1, 2, 64)
    bad = [
        (lambda: window_attention(c, q.bfloat16()), 'own type'),
        (lambda: window_attention(c, z(2, 4, 4, 64)), 'beside the window'),
        (lambda: window_attention(c, z(3, 1, 4, 64)), 'streams'),
        (lambda: window_attention(c, z(2, 1, 3, 64)), 'multiple'),
        (lambda: window_attention(c, z(2, 1, 4, 32)), 'beside q'),
        (lambda: window_attention(c, q.cpu()), 'device'),
        (lambda: window_attention(c, z(2, 1, 4, 128)[..., ::2]), 'adjacent'),
        (lambda: window_attention(c, z(2, 1, 4, 68)[..., 2:66]), 'multiples of 16'),
        (lambda: window_attention(c, q, out=q.float()), 'float16'),
        (lambda: window_attention(c, q, max_tokens=2), 'goes with offsets'),
        (lambda: window_attention(c, q[:, 0], offsets=torch.tensor([0, 1, 2], device=DEV)), 'int32'),
        (lambda: window_attention(c, q[:, 0], offsets=torch.tensor([0, 1, 2], device=DEV).int()), 'max_tokens'),
        (lambda: window_attention(c, q, scale=float('nan')), 'scale'),
        (lambda: qk_norm_rope_append(c, q, k, k, inv_freq=f.float()), 'float64'),
        (lambda: qk_norm_rope_append(c, q, k, k, inv_freq=f, rope_dims=32), 'twice'),
        (lambda: qk_norm_rope_append(c, q, k, k, inv_freq=torch.ones(33, dtype=torch.float64, device=DEV)), 'Rotated'),
        (lambda: qk_norm_rope_append(c, q, k, k, rope=z(2, 32, 2)), 'float32'),
        (lambda: qk_norm_rope_append(c, q, k, k, inv_freq=f, rope=z(2, 32, 2, d=torch.float32)), 'not both'),
        (lambda: qk_norm_rope_append(c, q, k, k, pairs='other'), 'pairs'),
        (lambda: qk_norm_rope_append(c, q, k, k, q_gain=z(64)), 'float32'),
        (lambda: qk_norm_rope_append(c, q, k, k, q_gain=z(64, d=torch.float32), epsilon=0.0), 'epsilon'),
        (lambda: qk_norm_rope_append(c, q, z(2, 1, 4, 64), k), 'beside q'),
        (lambda: qk_norm_rope_append(c, q, k, k.float()), 'float16'),
        (lambda: qk_norm_rope_append(c, q, k, k, out=torch.zeros(1, 1, 4, 64, device=DEV).half().expand(2, 1, 4, 64)), 'overlap'),
        (lambda: KvCache.from_tensors(c.keys, c.values[:, :, :-1], c.positions, window=8), 'shape'),
        (lambda: KvCache.from_tensors(c.keys, c.values, c.positions.int(), window=8), 'int64'),
        (lambda: KvCache.from_tensors(c.keys, c.values, c.positions, window=12), 'slots'),
        (lambda: KvCache.from_tensors(c.keys, c.values.transpose(1, 2).contiguous().transpose(1, 2), c.positions, window=8), 'strides'),
        (lambda: KvCache.from_tensors(c.keys.transpose(2, 3), c.values.transpose(2, 3), c.positions, window=8), 'strides'),
    ]
    for i, (call, match) in enumerate(bad):
        try:
            call()
        except ValueError as e:
            assert match in str(e), (i, match, str(e))
        else:
            raise AssertionError((i, match))
    assert window_attention(c, z(2, 0, 4, 64)).shape == (2, 0, 4, 64)
    torch.cuda.synchronize()


def fixed():
    """A cache's tensors cannot be replaced (the library has their addresses), rows beyond 32 bits and tensors
    that ask for gradients are refused; writing in place, and the same calls without gradients, go through."""
    c = KvCache(2, 2, 64, 8, 1, 3, torch.float16, DEV)
    q, k = (torch.ones(2, 1, h, 64, dtype=torch.float16, device=DEV) for h in (4, 2))
    at = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    for name in ('positions', 'keys', 'values', 'window', 'sinks'):
        try:
            setattr(c, name, getattr(c, name) + 1)
        except AttributeError as e:
            assert 'fixed' in str(e), str(e)
        else:
            raise AssertionError(name)
    c.positions += 1
    assert c.positions.tolist() == [1, 1]
    wide = torch.empty(1, 1, 4, 64, dtype=torch.float16, device=DEV)
    grad = q.clone().requires_grad_()
    bad = [
        (lambda: window_attention(c, wide[0].expand(2**32 + 2, 4, 64), out=wide[0].expand(2**32 + 2, 4, 64), offsets=at,
                                  max_tokens=1), '2^30'),
        (lambda: window_attention(c, wide.expand(2, 2**31 + 1, 4, 64), out=wide.expand(2, 2**31 + 1, 4, 64)), '2^30'),
        (lambda: window_attention(c, q[:, 0], offsets=at, max_tokens=2**32 + 1), 'takes 1 to 3'),
        (lambda: window_attention(c, q[:, 0], offsets=at, max_tokens=0), 'takes 1 to 3'),
        (lambda: window_attention(c, grad), 'no_grad'),
        (lambda: qk_norm_rope_append(c, q, k, k, q_gain=torch.ones(64, device=DEV, requires_grad=True)), 'no_grad'),
        (lambda: qk_norm_rope_append(c, q, k.clone().requires_grad_(), k), 'no_grad'),
    ]
    for i, (call, match) in enumerate(bad):
        try:
            call()
        except ValueError as e:
            assert match in str(e), (i, match, str(e))
        else:
            raise AssertionError((i, match))
    with torch.no_grad():
        qk_norm_rope_append(c, grad, k, k)
        out = window_attention(c, grad)
    # Slot 0 holds zeros (nothing appended it), slot 1 ones: q . k = 0 and 64, over sqrt(64).
    want = math.exp(8) / (1 + math.exp(8))
    assert not out.requires_grad and (out.double() - want).abs().max().item() <= 4 * STEP[torch.float16] + 2.0**-18


if __name__ == '__main__':
    for dtype, stored in ((torch.float32, torch.float32), (torch.bfloat16, 'int4'), (torch.float32, torch.float16)):
        print('generation', dtype, stored, flush=True)
        generation(dtype, stored, True)
    for check in (other_stream, captured, refusals, fixed):
        print(check.__name__, flush=True)
        check()
    torch.cuda.synchronize()
    print('ok', flush=True)

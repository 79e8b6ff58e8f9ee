"""The cache operators' workloads, as plain cases: what a model's attention does between its Q/K/V
projection and its output projection.

Operators:
  rope    norms of the queries and keys of each head, the position rotation and the append of keys
          and values to a sliding-window cache, in one pass (qk_norm_rope_append)
  window  attention over that cache: a sliding window and a few first tokens that stay visible
          (window_attention)
  int4    the same attention over a cache held in 4 bits; with `append` the new token is normed,
          rotated, quantised and appended first, as one layer of a decoding step does

A cache keeps, per stream and key/value head, `sinks` rows for positions 0 .. sinks - 1 and a ring of
window + tokens - 1 rows for the positions after them (slot sinks + (p - sinks) mod ring). A query at
position t sees the positions p <= t with p < sinks or p > t - window.

With `own` false, `run` computes the operators in elementary torch operations; with `own` true it makes
the calls of the framework's operators.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = 'cuda' if torch.cuda.is_available() else 'cpu'
TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
EPSILON = 1e-6
THETA = 10000.0
GROUP = 32  # values that share a scale and a minimum in a 4-bit cache


def _framework():
    path = str(Path('streaming-transformer_amd').resolve())
    if path not in sys.path:
        sys.path.insert(0, path)
    import streamtx
    return streamtx


def _case(name, op, dtype, streams, tokens, heads, kv_heads, dim, window, sinks, context, ragged=False,
          pairs='halves', rotary=None, append=False):
    return dict(name=name, op=op, dtype=dtype, streams=streams, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                window=window, sinks=sinks, context=context, ragged=ragged, pairs=pairs,
                rotary=dim if rotary is None else rotary, append=append)


def listed():
    return [
        # One event of one stream in the main model's shape: the smallest call, launch latency only.
        _case('rope-step-f32-1', 'rope', 'f32', 1, 1, 8, 8, 64, 128, 0, 500, pairs='adjacent'),
        # A full serving batch, one token for each stream, grouped heads.
        _case('rope-step-bf16-256', 'rope', 'bf16', 256, 1, 32, 8, 128, 1024, 4, 3000),
        # Streams that bring histories of unequal lengths, an odd head dimension, rotated in part.
        _case('rope-ragged-f16-37', 'rope', 'f16', 37, 211, 12, 4, 80, 500, 3, 700, ragged=True, pairs='adjacent', rotary=48),
        # One long prompt read in one call.
        _case('rope-prompt-bf16-16384', 'rope', 'bf16', 1, 16384, 32, 8, 128, 2048, 4, 0),
        # A step of the large model's batch: FP32 all through, one query head per cache head.
        _case('window-step-f32-16', 'window', 'f32', 16, 1, 16, 16, 64, 512, 4, 1300),
        # Decoding for many streams with long windows: bound by reading the cache.
        _case('window-step-bf16-64', 'window', 'bf16', 64, 1, 32, 8, 128, 4096, 4, 9000),
        # One stream with a very long window: few rows, work split along the window.
        _case('window-step-f16-long', 'window', 'f16', 1, 1, 32, 8, 128, 131072, 4, 200000),
        # A long prompt through a window much shorter than itself: bound by matrix products.
        _case('window-prompt-bf16-8192', 'window', 'bf16', 1, 8192, 32, 8, 128, 2048, 4, 0),
        # Unequal pieces of prompts, an odd head dimension and odd group: tiles that end anywhere.
        _case('window-ragged-f16-19', 'window', 'f16', 19, 333, 15, 5, 80, 777, 5, 1000, ragged=True),
        # The large model's batch over a 4-bit cache with FP32 queries.
        _case('int4-step-f32-16', 'int4', 'f32', 16, 1, 16, 16, 64, 512, 4, 1300),
        # One layer of a decoding step over long 4-bit windows: append, then attend.
        _case('int4-step-bf16-64', 'int4', 'bf16', 64, 1, 32, 8, 128, 8191, 4, 17000, append=True),
        # Pieces of prompts continued over a 4-bit cache.
        _case('int4-prompt-f16-4', 'int4', 'f16', 4, 1024, 32, 8, 128, 4096, 4, 6000),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(['rope', 'window', 'window', 'int4', 'int4'])
    dtype = rng.choice(['f32', 'f16', 'bf16', 'bf16'])
    kind = rng.choice(['step', 'step', 'few', 'prompt', 'ragged'])
    dim = rng.choice([32, 64, 64, 96, 128, 128, 256]) if op == 'int4' else rng.choice([16, 40, 64, 64, 80, 96, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    streams = 1 if rng.random() < 0.2 else _log_int(rng, 1, 256)
    tokens = {'step': 1, 'few': rng.randint(2, 8), 'prompt': _log_int(rng, 16, 8192), 'ragged': _log_int(rng, 16, 2048)}[kind]
    window = _log_int(rng, 16, 65536 if kind == 'step' else 4096)
    case = _case('', op, dtype, streams, tokens, heads, kv_heads, dim, window, rng.choice([0, 0, 1, 4, 7, 64]),
                 rng.choice([0, _log_int(rng, 1, 4 * window)]), ragged=kind == 'ragged',
                 pairs=rng.choice(['adjacent', 'halves']), rotary=rng.choice([dim, dim, dim // 32 * 16]),
                 append=op == 'int4' and dtype == 'bf16' and kind == 'step' and rng.random() < 0.5)
    del case['name']
    # Fewer streams, then fewer tokens, then a shorter window where the case would cost more than
    # the largest listed one, or hold more than the largest listed cache.
    most = max(_cost(c) for c in listed())
    while _cost(case) > most or _slots(case) * case['streams'] * case['kv_heads'] * case['dim'] > 600_000_000:
        if case['streams'] > 1:
            case['streams'] = max(1, case['streams'] * 3 // 4)
        elif case['tokens'] > 64:
            case['tokens'] = case['tokens'] * 3 // 4
        else:
            case['window'] = case['window'] * 3 // 4
    return case


def _ring(case):
    return case['window'] + case['tokens'] - 1


def _slots(case):
    return case['sinks'] + _ring(case)


def _starts(case):
    """The position of each stream's first new token: around the context, spread over the streams."""
    return [int(case['context'] * (0.5 + b * 0.6180339887 % 1.0)) if b else case['context'] for b in range(case['streams'])]


def _counts(case):
    """New tokens of each stream: all the same, or spread from none to case['tokens']."""
    if not case['ragged']:
        return [case['tokens']] * case['streams']
    return [case['tokens'] if b == 0 else int((case['tokens'] + 1) * (b * 0.6180339887 % 1.0)) for b in range(case['streams'])]


def _pairs(case):
    """(query, visible position) pairs of one query head, and cache rows that any query sees, over all streams."""
    pairs = rows = 0
    w, s = case['window'], case['sinks']
    for start, n in zip(_starts(case), _counts(case)):
        for t in range(start, start + n):
            pairs += min(t + 1, min(s, max(t - w + 1, 0)) + w)
        if n:
            last, low = start + n - 1, max(start - w + 1, 0)
            rows += last + 1 - max(low, 0) + min(s, low)
    return pairs, rows


def _row_bytes(case):
    if case['op'] == 'int4':
        return case['dim'] // 2 + case['dim'] // GROUP * 4
    return case['dim'] * TYPES[case['dtype']].itemsize


def work(case):
    """rope: q, k and v read, q and the cache rows written, each once. Attention: q read, the output
    written, every cache row that some query sees read once; two products over the visible pairs."""
    size = TYPES[case['dtype']].itemsize
    tokens, dim = sum(_counts(case)), case['dim']
    q, kv = tokens * case['heads'] * dim, tokens * case['kv_heads'] * dim
    appended = (q + 2 * kv) * size + q * size + 2 * tokens * case['kv_heads'] * _row_bytes(case)
    flops = 8 * (q + kv)
    if case['op'] == 'rope':
        return {'bytes': appended + 16 * case['dim'], 'flops': flops}
    pairs, rows = _pairs(case)
    # With the append, the normed and rotated queries stay between the two calls.
    read = 2 * rows * case['kv_heads'] * _row_bytes(case) + 2 * q * size
    if case['append']:
        return {'bytes': read + (q + 2 * kv) * size + 2 * tokens * case['kv_heads'] * _row_bytes(case),
                'flops': flops + 4 * pairs * case['heads'] * dim}
    return {'bytes': read, 'flops': 4 * pairs * case['heads'] * dim}


def _cost(case):
    w = work(case)
    return w['bytes'] / 5e12 + w['flops'] / (1e14 if case['dtype'] == 'f32' else 1e15)


class _State:
    pass


def _inputs(case, seed):
    """The tensors of a case, made from the seed alone."""
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(1000003 * (seed + 1))

    def normal(*shape, dtype=torch.float32, scale=1.0):
        out = torch.empty(shape, dtype=dtype, device=DEVICE)
        flat = out.view(-1)
        for i in range(0, flat.numel(), 1 << 28):  # no FP32 copy of a whole cache
            part = flat[i:i + (1 << 28)]
            part.copy_(torch.randn(part.shape, generator=gen, device=DEVICE) * scale)
        return out

    s = _State()
    dtype, b, n, dim = TYPES[case['dtype']], case['streams'], case['tokens'], case['dim']
    heads, kv, slots = case['heads'], case['kv_heads'], _slots(case)
    counts = _counts(case)
    total = sum(counts)
    # Queries, keys and values as one projection leaves them: one row of all heads per token.
    s.projected = normal(total, heads + 2 * kv, dim, dtype=dtype, scale=1.0)
    s.q, s.k, s.v = s.projected[:, :heads], s.projected[:, heads:heads + kv], s.projected[:, heads + kv:]
    s.gain_q = 1.0 + 0.1 * normal(dim)
    s.gain_k = 1.0 + 0.1 * normal(dim)
    s.freq = THETA ** (-torch.arange(0, case['rotary'], 2, dtype=torch.float64) / max(case['rotary'], 1))
    s.freq = s.freq.to(DEVICE)
    s.positions = torch.tensor(_starts(case), dtype=torch.int64, device=DEVICE)
    ends = [0]
    for c in counts:
        ends.append(ends[-1] + c)
    s.offsets = torch.tensor(ends, dtype=torch.int32, device=DEVICE)
    # The cache, with every slot filled: slots that no query sees hold other numbers.
    if case['op'] == 'int4':
        s.keys, s.key_params = _packed(gen, b * kv * slots, dim, (b, kv, slots))
        s.values, s.value_params = _packed(gen, b * kv * slots, dim, (b, kv, slots))
    elif case['op'] == 'window':
        s.keys, s.values = normal(b, kv, slots, dim, dtype=dtype), normal(b, kv, slots, dim, dtype=dtype)
    else:
        s.keys = torch.zeros(b, kv, slots, dim, dtype=dtype, device=DEVICE)
        s.values = torch.zeros_like(s.keys)
    return s


def _packed(gen, rows, dim, shape):
    """Codes of bell-shaped values, packed, and FP16 (scale, minimum) pairs for each 32 of them."""
    codes = torch.empty((rows, dim // 2), dtype=torch.uint8, device=DEVICE)
    step = max(1, (1 << 27) // dim)
    for i in range(0, rows, step):
        x = torch.randn((min(step, rows - i), dim), generator=gen, device=DEVICE)
        codes[i:i + step] = _pack((x * 3.2 + 7.5).round().clamp(0, 15).to(torch.uint8))
    scale = (0.3 + 0.03 * torch.randn((rows, dim // GROUP, 1), generator=gen, device=DEVICE)).abs()
    params = torch.cat((scale, scale * -7.5 + 0.1 * torch.randn(scale.shape, generator=gen, device=DEVICE)), -1)
    return codes.view(*shape, dim // 2), params.half().view(*shape, dim // GROUP, 2)


# In each four bytes of a packed row, taken as one little-endian word of eight codes: element 2j in
# bits 4j, element 2j + 1 in bits 16 + 4j.
def _pack(codes):
    c = codes.unflatten(-1, (-1, 4, 2))  # [word, j, even or odd]
    even, odd = c[..., 0], c[..., 1]
    return torch.stack((even[..., 0] | even[..., 1] << 4, even[..., 2] | even[..., 3] << 4,
                        odd[..., 0] | odd[..., 1] << 4, odd[..., 2] | odd[..., 3] << 4), -1).flatten(-2)


def _unpack(packed):
    p = packed.unflatten(-1, (-1, 4))
    low, high = p & 15, p >> 4
    return torch.stack((low[..., 0], low[..., 2], high[..., 0], high[..., 2],
                        low[..., 1], low[..., 3], high[..., 1], high[..., 3]), -1).flatten(-2)


def prepare(case, seed):
    s = _inputs(case, seed)
    s.case = case
    s.scale = 1.0 / math.sqrt(case['dim'])
    if own:
        stx = _framework()
        s.stx = stx
        more = dict(key_params=s.key_params, value_params=s.value_params) if case['op'] == 'int4' else {}
        s.cache = stx.KvCache.from_tensors(s.keys, s.values, s.positions, window=case['window'], sinks=case['sinks'], **more)
    return s


def run(s):
    c = s.case
    if own:
        rows = dict(offsets=s.offsets, max_tokens=c['tokens']) if c['ragged'] else {}
        q, k, v = s.q, s.k, s.v
        if not rows:
            q, k, v = (t.unflatten(0, (c['streams'], c['tokens'])) for t in (q, k, v))
        if c['op'] == 'rope' or c['append']:
            q = s.stx.qk_norm_rope_append(s.cache, q, k, v, q_gain=s.gain_q, k_gain=s.gain_k, epsilon=EPSILON,
                                          inv_freq=s.freq, pairs=c['pairs'], **rows)
        if c['op'] == 'rope':
            return {'q': q, 'keys': s.keys, 'values': s.values}
        return {'out': s.stx.window_attention(s.cache, q, scale=s.scale, **rows)}
    q = s.q
    if c['op'] == 'rope' or c['append']:
        q = _plain_append(s)
    if c['op'] == 'rope':
        return {'q': q if c['ragged'] else q.unflatten(0, (c['streams'], c['tokens'])), 'keys': s.keys, 'values': s.values}
    out = _plain_attention(s, q)
    return {'out': out if c['ragged'] else out.unflatten(0, (c['streams'], c['tokens']))}


# The plain forms.

def _rows(s):
    """The stream and the position of each row of new tokens."""
    row = torch.arange(s.q.shape[0], device=DEVICE)
    stream = torch.searchsorted(s.offsets, row.to(torch.int32), right=True) - 1
    return stream, s.positions[stream] + row - s.offsets[stream]


def _plain_append(s):
    c = s.case
    stream, position = _rows(s)
    angle = position[:, None].double() * s.freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def normed(x, gain):
        x = x.float()
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPSILON) * gain

    def rotated(x):
        rot, rest = x[..., :c['rotary']], x[..., c['rotary']:]
        if c['pairs'] == 'adjacent':
            a, b = rot[..., 0::2], rot[..., 1::2]
            rot = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        else:
            a, b = rot.chunk(2, -1)
            rot = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
        return torch.cat((rot, rest), -1)

    q = rotated(normed(s.q, s.gain_q)).to(s.q.dtype)
    k, v = rotated(normed(s.k, s.gain_k)), s.v
    slot = torch.where(position < c['sinks'], position, c['sinks'] + (position - c['sinks']) % _ring(c))
    if c['op'] == 'int4':
        for x, codes, params in ((k, s.keys, s.key_params), (v, s.values, s.value_params)):
            x = x.float().unflatten(-1, (-1, GROUP))
            low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
            scale, low = ((high - low) / 15).half(), low.half()
            code = ((x - low.float()) / scale.float()).round().clamp(0, 15)
            code = torch.where(scale > 0, code, 0).to(torch.uint8).flatten(-2)
            codes[stream, :, slot] = _pack(code)
            params[stream, :, slot] = torch.cat((scale, low), -1)
    else:
        s.keys[stream, :, slot] = k.to(s.keys.dtype)
        s.values[stream, :, slot] = v
    return q


def _plain_attention(s, q):
    c = s.case
    b, n, kv, dim, slots = c['streams'], c['tokens'], c['kv_heads'], c['dim'], _slots(c)
    group = c['heads'] // kv
    counts = s.offsets[1:] - s.offsets[:-1]
    if c['ragged']:  # rows of each stream side by side, padded
        index = s.offsets[:-1, None] + torch.arange(n, device=DEVICE)
        index = index.clamp(max=q.shape[0] - 1)
        q = q[index.long()]
    else:
        q = q.unflatten(0, (b, n))
    q = q.float().view(b, n, kv, group, dim).permute(0, 2, 1, 3, 4)  # [b, kv, n, group, dim]
    # The position that each slot holds once the new tokens are in.
    last = s.positions + counts - 1
    slot = torch.arange(slots, device=DEVICE)
    held = torch.where(slot < c['sinks'], slot, last[:, None] - (last[:, None] - slot) % _ring(c))
    held = torch.where((slot >= c['sinks']) & (held < c['sinks']), -1, held)
    out = torch.empty((b, kv, n, group, dim), device=DEVICE)
    most = 1 << 29  # values of a cache in FP32, or of logits, at a time
    some = max(1, most // (kv * slots * max(dim, group * min(n, 256))))
    for i in range(0, b, some):
        part = slice(i, min(b, i + some))
        if c['op'] == 'int4':
            k, v = ((_unpack(codes[part]).float().unflatten(-1, (-1, GROUP)) * params[part][..., :1].float()
                      + params[part][..., 1:].float()).flatten(-2)
                    for codes, params in ((s.keys, s.key_params), (s.values, s.value_params)))
        else:
            k, v = s.keys[part].float(), s.values[part].float()
        kt = k.transpose(-1, -2).contiguous()
        rows = max(1, most // (kv * slots * group * k.shape[0]))
        for j in range(0, n, rows):
            t = s.positions[part, None] + torch.arange(j, min(n, j + rows), device=DEVICE)  # [b, rows]
            p = held[part, None, :]
            seen = (p >= 0) & (p <= t[:, :, None]) & ((p < c['sinks']) | (p > t[:, :, None] - c['window']))
            x = q[part, :, j:j + rows]
            logits = torch.matmul(x.flatten(2, 3), kt).unflatten(2, (x.shape[2], group)) * s.scale
            logits = logits.masked_fill(~seen[:, None, :, None, :], -math.inf)
            weight = (logits - logits.amax(-1, keepdim=True)).exp()
            total = weight.sum(-1, keepdim=True)
            out[part, :, j:j + rows] = torch.matmul(weight.flatten(2, 3), v).unflatten(2, (x.shape[2], group)) / total
    out = out.permute(0, 2, 1, 3, 4).reshape(b, n, c['heads'], dim).to(TYPES[c['dtype']])
    if not c['ragged']:
        return out.flatten(0, 1)
    stream, position = _rows(s)
    return out[stream, position - s.positions[stream]]


def exact(case, seed):
    """What `run` returns, one stream after the other in 64 bits: the norms and rotations as complex
    products, attention over the visible positions alone. For keys that are quantised after their norm
    and rotation the codes are those of the 64-bit values."""
    s = _inputs(case, seed)
    dim, sinks, window, ring = case['dim'], case['sinks'], case['window'], _ring(case)
    starts, counts = _starts(case), _counts(case)
    ends = s.offsets.tolist()
    dtype = TYPES[case['dtype']]

    def slots_of(p):
        return torch.where(p < sinks, p, (p - sinks) % ring + sinks)

    def turned(x, gain, position):
        x = x.double()
        x = x / (x.square().sum(-1, keepdim=True) / dim + EPSILON).sqrt() * gain.double()
        r = case['rotary']
        if not r:
            return x
        first, second = (slice(0, r, 2), slice(1, r, 2)) if case['pairs'] == 'adjacent' else (slice(0, r // 2), slice(r // 2, r))
        unit = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE), position[:, None, None].double() * s.freq)
        z = torch.complex(x[..., first], x[..., second]) * unit
        out = x.clone()
        out[..., first], out[..., second] = z.real, z.imag
        return out

    def stands_for(codes, params):
        v = _unpack(codes).double().unflatten(-1, (-1, GROUP))
        return (params[..., 1:].double() + params[..., :1].double() * v).flatten(-2)

    def quantised(x):
        g = x.unflatten(-1, (-1, GROUP))
        low, span = g.amin(-1, keepdim=True).float(), (g.amax(-1, keepdim=True) - g.amin(-1, keepdim=True)).float()
        scale, low = (span / 15).half().double(), low.half().double()
        code = torch.where(scale > 0, ((g - low) / scale).round().clamp(0, 15), 0.0)
        return (low + scale * code).flatten(-2)

    append = case['op'] == 'rope' or case['append']
    q_all = torch.zeros(s.q.shape, dtype=torch.float64, device=DEVICE)
    if case['op'] == 'rope':
        keys, values = (torch.zeros(s.keys.shape, dtype=torch.float64, device=DEVICE) for _ in range(2))
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEVICE)
    for b in range(case['streams']):
        n, first = counts[b], ends[b]
        if not n:
            continue
        rows = slice(first, first + n)
        t = torch.arange(starts[b], starts[b] + n, device=DEVICE)
        q = s.q[rows]
        if append:
            q, k = turned(q, s.gain_q, t), turned(s.k[rows], s.gain_k, t)
            if case['op'] == 'rope':
                q_all[rows] = q
                keys[b][:, slots_of(t)] = k.transpose(0, 1)
                values[b][:, slots_of(t)] = s.v[rows].double().transpose(0, 1)
                continue
            q = q.to(dtype)  # the queries go to the attention in their own type
        group = case['heads'] // case['kv_heads']
        for j in range(0, n, 512):
            tj = t[j:j + 512]
            low = max(0, int(tj[0]) - window + 1)
            p = torch.arange(low, int(tj[-1]) + 1, device=DEVICE)
            p = torch.cat((torch.arange(0, min(sinks, low), device=DEVICE), p))
            at = slots_of(p)
            if case['op'] == 'int4':
                kb = stands_for(s.keys[b][:, at], s.key_params[b][:, at])
                vb = stands_for(s.values[b][:, at], s.value_params[b][:, at])
                if append:  # the new token's rows, appended before
                    new = p.shape[0] - 1
                    kb[:, new], vb[:, new] = quantised(k[0]), quantised(s.v[rows][0].double())
            else:
                kb, vb = s.keys[b][:, at].double(), s.values[b][:, at].double()
            x = q[j:j + 512].double().unflatten(1, (case['kv_heads'], group)).permute(1, 2, 0, 3)  # [kv, group, n, dim]
            hidden = (p[None] > tj[:, None]) | ((p[None] >= sinks) & (p[None] <= tj[:, None] - window))
            for h in range(case['kv_heads']):
                logits = x[h].reshape(-1, dim) @ kb[h].T.contiguous() / math.sqrt(dim)
                logits = logits.view(group, -1, p.shape[0]).masked_fill(hidden, -math.inf)
                mixed = torch.softmax(logits, -1).view(-1, p.shape[0]) @ vb[h]
                out[rows][j:j + 512, h * group:(h + 1) * group] = mixed.view(group, -1, dim).transpose(0, 1)
    fold = (lambda x: x) if case['ragged'] else (lambda x: x.unflatten(0, (case['streams'], case['tokens'])))
    if case['op'] == 'rope':
        return {'q': fold(q_all), 'keys': keys, 'values': values}
    return {'out': fold(out)}

"""The cache operators (st_qk_norm_rope_append, st_window_attention) on the GPU against 64-bit results, over
types, head layouts, lengths, strides, windows and sinks, and the ways a serving program calls them."""
import ctypes

import numpy as np
import pytest

from cacheops import (BF16, F16, F32, INT4, NAMES, STEP, Cache, Device, Heads, append, attend, attention, attention_bound,
                      decode, encode, hip, quantise, rows_struct, sync, turned, unpack, workspace_bytes)

pytestmark = pytest.mark.gpu

PAIRS = [(F32, F32), (F32, F16), (F32, BF16), (F32, INT4), (F16, F16), (F16, INT4), (BF16, BF16), (BF16, INT4)]


def pair_id(p):
    return NAMES[p[0]] + '-' + NAMES[p[1]] if isinstance(p, tuple) else str(p)


def frequencies(rope_dims):
    return 10000.0 ** (-np.arange(0, rope_dims, 2) / max(rope_dims, 1))


def angles_of(starts, firsts, counts, total, freq):
    position = np.zeros(total)
    for s, f, n in zip(starts, firsts, counts):
        position[f:f + n] = s + np.arange(n)
    return position[:, None] * freq


def norm_bound(y, size, dtype):
    """FP32 arithmetic: the sum of squares 13 roundings deep (half of it in the root), the mean, the root, its
    reciprocal and two products five more, the rotation's angle (pi / 2^25 of a turn's half) and its
    cosine and sine 4, its products and sum 3: below 24 in all, relative to the pair; then one rounding to
    the type, FP16's below its smallest normal number."""
    return 24 * 2.0**-24 * size + STEP[dtype] * np.abs(y) * (dtype != F32) + (2.0**-25 if dtype == F16 else 0) + 1e-30


# ------------------------------------------------------------------------------------------------
# norm, rotation and append

APPEND = [  # dim, q heads, kv heads, rotated, halves, norm, pad
    (64, 8, 8, 64, 0, True, 0),
    (128, 8, 2, 128, 1, True, 0),
    (32, 3, 1, 16, 0, True, 32),
    (96, 5, 5, 48, 1, False, 32),
    (256, 4, 2, 256, 1, True, 0),
    (128, 33, 11, 0, 0, True, 64),
    (64, 4, 4, 30, 1, True, 0),
    (64, 4, 4, 62, 0, False, 0),
]


def run_append(types, shape, starts, n, counts=None):
    dtype, stored = types
    dim, heads, kv, rope_dims, halves, norm, pad = shape
    rng = np.random.default_rng(dim + heads)
    window, sinks = 9, 2
    cache = Cache(len(starts), kv, dim, window, sinks, stored, max_tokens=n, positions=starts)
    offsets = None
    if counts is not None:
        offsets = Device(np.concatenate(([0], np.cumsum(counts))).astype(np.int32))
    rows, firsts, total = rows_struct(cache, counts, n, offsets)
    counts = [n] * len(starts) if counts is None else counts
    q, k, v = (Heads(rng.standard_normal((total, h, dim)) * 2, dtype, pad) for h in (heads, kv, kv))
    out = Heads(np.zeros((total, heads, dim)), dtype, pad)
    gq, gk = (1 + 0.2 * rng.standard_normal(dim).astype(np.float32) for _ in range(2)) if norm else (None, None)
    freq = frequencies(rope_dims)
    dev = [Device(g) if g is not None else None for g in (gq, gk)]
    inv = Device(freq) if rope_dims else None
    append(cache, rows, q, k, v, out, *dev, inv_freq=inv, rope_dims=rope_dims, halves=halves)
    angles = angles_of(starts, firsts, counts, total, freq)
    got, clean = out.get()
    assert clean
    want, size = turned(q.float(), gq, 1e-6, angles, rope_dims, halves)
    for start, first, m in zip(starts, firsts, counts):
        if start < 0:
            want[first:first + m] = size[first:first + m] = 0
    assert (np.abs(got - want) <= norm_bound(want, size, dtype)).all()

    kw, size = turned(k.float(), gk, 1e-6, angles, rope_dims, halves)
    stored_rows = cache.values()
    untouched = np.ones(cache.dims, bool)
    raw = cache.raw()
    for b in range(len(starts)):
        if starts[b] < 0 or not counts[b]:
            continue
        at = cache.slot(starts[b] + np.arange(counts[b]))
        untouched[b][:, at] = False
        part = slice(firsts[b], firsts[b] + counts[b])
        keys, values = (x[b][:, at].transpose(1, 0, 2) for x in stored_rows)
        if stored == INT4:
            # Keys: the nearest code of a range that is itself rounded to FP16.
            codes, params = (x[b][:, at].transpose(1, 0, 2) if x.ndim == 4 else x[b][:, at].transpose(1, 0, 2, 3)
                             for x in raw[0:3:2])
            p = params.astype(np.float64)
            step = np.repeat(p[..., 0], 32, -1)
            ends = np.repeat(np.abs(p[..., 1]) + 15 * p[..., 0], 32, -1)
            assert (np.abs(keys - kw[part]) <= step / 2 + ends * 2 * STEP[F16] + norm_bound(kw, size, F32)[part]).all()
            # Values come as they are: the format's own arithmetic, bit for bit.
            want_codes, want_params = quantise(v.float()[part].astype(np.float32))
            assert (unpack(raw[1][b][:, at].transpose(1, 0, 2)) == want_codes).all()
            assert (raw[3][b][:, at].transpose(1, 0, 2, 3) == want_params).all()
        else:
            assert (np.abs(keys - kw[part]) <= norm_bound(kw, size, stored)[part]).all()
            assert (values == decode(encode(v.float()[part], stored), stored)).all()
    for x in raw:
        assert (x[untouched] == 0).all()


@pytest.mark.parametrize('types', PAIRS, ids=pair_id)
@pytest.mark.parametrize('shape', APPEND, ids=str)
def test_append(types, shape):
    run_append(types, shape, [0, 5, 1000003, 1], 3)


@pytest.mark.parametrize('types', PAIRS, ids=pair_id)
@pytest.mark.parametrize('shape', [
    (96, 3, 3, 48, 1, True, 0),   # 1300 tokens
    (64, 2, 1, 64, 1, True, 0),   # 4225 tokens of few heads
    (32, 3, 1, 16, 0, True, 32),
    (128, 2, 1, 90, 1, True, 0),
], ids=str)
def test_append_many_tokens(types, shape):
    """Unequal numbers of tokens, none among them, and a stream that is left out."""
    n = 400 if shape[0] == 96 else 1300
    run_append(types, shape, [0, 7, 12345, -5, 1], n, [n, 0, 3 * n // 4, n, n // 2])


def test_append_a_token_of_each_of_many_streams():
    run_append((BF16, INT4), (64, 1, 1, 64, 1, True, 0), [b * 7 if b % 5 else -1 for b in range(5003)], 1)


def test_append_a_long_prompt():
    run_append((BF16, BF16), (128, 8, 2, 128, 1, True, 0), [3], 16500)


def test_append_in_place_and_from_a_table():
    """q_out may be q; a table of rotations gives what its angles give, to the table's rounding."""
    rng = np.random.default_rng(3)
    cache = [Cache(3, 2, 64, 8, 0, F32, positions=[4, 0, 90]) for _ in range(2)]
    rows, firsts, total = rows_struct(cache[0], n=1)
    x = [rng.standard_normal((total, h, 64)) for h in (4, 2, 2)]
    freq = frequencies(64)
    angles = angles_of([4, 0, 90], firsts, [1] * 3, total, freq)
    table = np.stack((np.cos(angles), np.sin(angles)), -1).astype(np.float32)
    q, k, v = (Heads(a, F32) for a in x)
    append(cache[0], rows, q, k, v, q, inv_freq=Device(freq), rope_dims=64)
    q2, out = Heads(x[0], F32), Heads(np.zeros_like(x[0]), F32)
    t = Device(table)
    append(cache[1], rows, q2, k, v, out, rope=t, rope_dims=64)
    want, size = turned(q2.float(), None, 0, angles, 64, 0)
    for got in (q.get()[0], out.get()[0]):
        assert (np.abs(got - want) <= norm_bound(want, size, F32)).all()
    for a, b in zip(cache[0].values(), cache[1].values()):
        assert np.abs(a - b).max() <= 24 * 2.0**-24 * np.abs(b).max()


def test_append_far_positions():
    """Angles of positions that FP32 does not hold, on both sides of 2^31."""
    for start in (2**31 - 2, 2**40 + 1):
        cache = Cache(1, 1, 64, 16, 3, F32, max_tokens=4, positions=[start])
        rows, firsts, total = rows_struct(cache, n=4)
        rng = np.random.default_rng(7)
        q, k, v = (Heads(rng.standard_normal((4, 1, 64)), F32) for _ in range(3))
        out = Heads(np.zeros((4, 1, 64)), F32)
        freq = frequencies(64)
        append(cache, rows, q, k, v, out, inv_freq=Device(freq), rope_dims=64)
        # cos and sin of the exact product: 64-bit long double arithmetic, reduced before it is rounded.
        turns = np.longdouble(start + np.arange(4))[:, None] * np.longdouble(freq) / (2 * np.longdouble('3.14159265358979323846'))
        angles = ((turns - np.rint(turns)) * 2 * np.pi).astype(np.float64)
        want, size = turned(q.float(), None, 0, angles, 64, 0)
        # The kernel's product and its division by a turn round to 64 bits: 2 half steps of the turns.
        slack = float(start) / (2 * np.pi) * 2.0**-52 * 2 * np.pi
        assert (np.abs(out.get()[0] - want) <= norm_bound(want, size, F32) + slack * size).all()
        at = cache.slot(start + np.arange(4))
        assert (cache.values()[1][0, 0, at] == v.float()[:, 0]).all()


def test_append_rows_of_zeros_and_not_finite():
    cache = Cache(1, 1, 64, 8, 0, INT4, max_tokens=3)
    rows, _, total = rows_struct(cache, n=3)
    x = np.random.default_rng(1).standard_normal((3, 1, 64))
    x[0] = 0
    x[1, 0, 5], x[1, 0, 40] = np.inf, np.nan
    x[2] = 2.5
    q = Heads(x, F32)
    out = Heads(np.ones_like(x), F32)
    gain = Device(np.ones(64, np.float32))
    append(cache, rows, q, q, q, out, gain, None)
    got = out.get()[0]
    assert (got[0] == 0).all() and np.isnan(got[1]).any()
    keys, values = cache.values()
    assert (values[0, 0, 0] == 0).all() and (values[0, 0, 2] == 2.5).all()
    assert np.isnan(values[0, 0, 1]).all()  # both groups hold a value that is not finite
    assert (keys[0, 0, 0] == 0).all()


# ------------------------------------------------------------------------------------------------
# attention

ATTEND = [  # dim, q heads, kv heads, window, sinks, tokens, starts
    (64, 4, 4, 128, 0, 1, [0, 1, 127, 128, 500]),
    (64, 8, 8, 100, 4, 1, [2, 3, 4, 103, 104, 1000]),
    (128, 8, 2, 500, 4, 1, [0, 499, 503, 504, 3000]),
    (128, 32, 2, 1, 0, 1, [0, 5]),
    (128, 24, 1, 33, 70, 1, [10, 69, 70, 102, 103, 150]),
    (256, 6, 2, 77, 1, 1, [0, 76, 400]),
    (32, 5, 5, 64, 2, 1, [63, 64, 65]),
    (96, 6, 3, 200, 3, 2, [0, 198, 199, 203, 700]),
    (64, 6, 2, 40, 4, 17, [0, 3, 36, 44, 333]),
    (128, 8, 2, 16, 2, 70, [0, 1, 2, 100]),
    (128, 4, 4, 300, 0, 130, [0, 250]),
    (256, 2, 1, 90, 5, 65, [0, 1000]),
    (64, 3, 3, 1000, 100, 33, [50, 90, 2000]),
    (128, 4, 1, 1, 0, 40, [0, 9]),
    (128, 12, 4, 64, 7, 200, [0, 6, 500]),
]


def run_attention(dtype, stored, dim, heads, kv, window, sinks, n, starts, counts=None, order=(0, 1, 2), pad=0, spread=1.0,
                  seed=1):
    rng = np.random.default_rng(seed)
    streams = len(starts)
    cache = Cache(streams, kv, dim, window, sinks, stored, max_tokens=n, fill=seed, order=order, positions=starts)
    ends = Device(np.concatenate(([0], np.cumsum(counts))).astype(np.int32)) if counts is not None else None
    rows, firsts, total = rows_struct(cache, counts, n, ends)
    q = Heads(rng.standard_normal((total, heads, dim)) * spread, dtype, pad)
    out = Heads(np.full((total, heads, dim), 9.0), dtype, pad)
    keep = attend(cache, rows, q, out)
    got, clean = out.get()
    assert clean
    values = cache.values()
    counts = [n] * streams if counts is None else counts
    want, mass, size = attention(values, cache, q.float(), starts, firsts, counts, 1 / np.sqrt(dim))
    live = ~np.isnan(mass)
    assert (got[~live] == 9.0).all()
    keys = sinks + window
    bound = attention_bound(np.nan_to_num(want), np.nan_to_num(mass), np.nan_to_num(size), keys, cache, dtype)
    err = np.abs(got - want)
    assert (err <= bound)[live].all(), float((err / bound)[live].max())
    del keep
    return got


@pytest.mark.parametrize('types', PAIRS, ids=pair_id)
@pytest.mark.parametrize('shape', ATTEND, ids=str)
def test_attention(types, shape):
    if types[1] == INT4 and shape[0] % 32:
        pytest.skip('4-bit rows hold whole groups of 32')
    run_attention(*types, *shape)


@pytest.mark.parametrize('dim', [8, 16, 40, 72, 80, 136, 248])
@pytest.mark.parametrize('types', [(F32, F32), (F16, F16), (BF16, BF16), (F32, BF16)], ids=pair_id)
def test_attention_odd_head_dims(types, dim):
    run_attention(*types, dim, 6, 3, 50, 3, 1, [0, 20, 200])
    run_attention(*types, dim, 6, 3, 50, 3, 37, [0, 20, 200])


@pytest.mark.parametrize('order', [(0, 2, 1), (1, 0, 2), (2, 0, 1)], ids=str)
@pytest.mark.parametrize('types', [(F32, F32), (BF16, BF16), (F16, INT4)], ids=pair_id)
def test_attention_strides(types, order):
    """Caches of other orders than [stream, head, slot], heads inside wider rows."""
    run_attention(*types, 64, 6, 2, 60, 3, 1, [0, 70, 200], order=order, pad=32)
    run_attention(*types, 128, 6, 2, 60, 3, 20, [0, 70, 200], order=order, pad=32)


@pytest.mark.parametrize('types', PAIRS, ids=pair_id)
def test_attention_ragged(types):
    """Unequal numbers of new tokens, none and all among them, and a stream that is left out."""
    run_attention(*types, 64, 6, 3, 30, 2, 40, [0, 5, 100, -1, 7, 31], counts=[40, 0, 13, 6, 1, 33])
    run_attention(*types, 128, 3, 3, 30, 2, 5, [0, -3, 12], counts=[5, 2, 0])


@pytest.mark.parametrize('dtype,stored', [(F32, F32), (F16, F16), (BF16, INT4)])
def test_attention_long_window_is_split(dtype, stored):
    """One stream with a long window: the keys are split over workgroups and merged."""
    run_attention(dtype, stored, 64, 2, 1, 20000, 4, 1, [30000])
    run_attention(dtype, stored, 128, 4, 1, 9000, 4, 3, [8000])


@pytest.mark.parametrize('dtype,stored', [(BF16, BF16), (F16, INT4), (F32, F32)])
def test_attention_many_rows_are_split(dtype, stored):
    """Few streams, many rows and long windows: row tiles, each split over workgroups along the keys."""
    run_attention(dtype, stored, 64, 32, 4, 8192, 4, 34, [9000, 100, 8190, -1], counts=[34, 34, 30, 0])


def test_attention_cache_past_the_infinity_cache():
    """A 16-bit cache of more than 256 MB, whose rows are read with non-temporal loads: values at both ends of the
    window and at its start, all keys zero but one."""
    dim, slots = 128, 700_000
    rows = []
    for _ in range(2):
        p = ctypes.c_void_p()
        hip().hipMalloc(ctypes.byref(p), ctypes.c_size_t(slots * dim * 2))
        hip().hipMemset(p, 0, ctypes.c_size_t(slots * dim * 2))
        rows.append(p)
    from streamtx.cache import _Cache
    cache = Cache.__new__(Cache)
    cache.dims, cache.dim, cache.window, cache.sinks, cache.ring, cache.dtype = (1, 1, slots), dim, slots, 0, slots, BF16
    cache.positions = Device(np.asarray([slots + 5], np.int64))
    cache.struct = _Cache(1, 1, dim, slots, 0, slots, BF16, 0, 0, 0, rows[0].value, rows[1].value, None, None,
                          cache.positions.ptr)
    mark = encode(np.random.default_rng(4).standard_normal((3, dim)), BF16)
    for m, at in zip(mark, (0, 399_999, slots - 1)):
        hip().hipMemcpy(ctypes.c_void_p(rows[1].value + at * dim * 2), m.ctypes.data_as(ctypes.c_void_p), dim * 2, 1)
    r, _, _ = rows_struct(cache, n=1)
    q, k, v = (Heads(np.ones((1, n, dim)), BF16) for n in (4, 1, 1))
    out = Heads(np.zeros((1, 4, dim)), BF16)
    append(cache, r, q, k, v, out)
    keep = attend(cache, r, q, out, scale=0.125)
    e = np.exp(-16.0)
    want = (1 + e * decode(mark, BF16).sum(0)) / (1 + e * (slots - 1))
    # The weights' sums in FP32 (some 2000 roundings deep where a wave walks its share), then the output's rounding.
    assert np.abs(out.get()[0] - want).max() <= (STEP[BF16] + 4096 * 2.0**-24) * np.abs(want).max()
    for p in rows:
        hip().hipFree(p)
    del keep


@pytest.mark.parametrize('dtype,stored', [(F32, F32), (F16, F16), (BF16, BF16), (F16, INT4), (BF16, INT4)])
def test_attention_large_logits(dtype, stored):
    """Logits of a hundred and more: the running maximum carries the exponentials."""
    run_attention(dtype, stored, 64, 4, 2, 200, 2, 1, [150, 1000], spread=30.0)
    run_attention(dtype, stored, 64, 4, 2, 200, 2, 50, [0, 1000], spread=30.0)


@pytest.mark.parametrize('n', [1, 21])
@pytest.mark.parametrize('types', [(F32, F32), (F32, BF16), (F16, F16), (BF16, BF16)], ids=pair_id)
def test_values_that_no_query_sees_do_not_matter(types, n):
    """Infinities and NaN in slots outside every window, and in keys and values that some queries of a call
    see and others do not: each query's result is its own."""
    dtype, stored = types
    dim, heads, kv, window, sinks = 64, 4, 2, 40, 3
    starts = [0, 30, 500]
    cache = Cache(3, kv, dim, window, sinks, stored, max_tokens=n, fill=5, positions=starts)
    k, v = (x.copy() for x in cache.values())
    free = np.ones(cache.dims[::2], bool)
    for b, s in enumerate(starts):
        for t in range(s, s + n):
            low = max(t - window + 1, 0)
            free[b, cache.slot(np.concatenate((np.arange(min(sinks, low)), np.arange(low, t + 1))))] = False
    k[free.nonzero()[0], :, free.nonzero()[1]] = np.nan
    v[free.nonzero()[0], :, free.nonzero()[1]] = np.inf
    # The last new token of stream 1 holds values that are not finite: earlier queries do not see it.
    last = cache.slot(starts[1] + n - 1)
    v[1, 0, last, 3], v[1, 0, last, 9], v[1, 1, last, 60] = np.nan, -np.inf, np.inf
    cache.write(k, v)
    rows, firsts, total = rows_struct(cache, n=n)
    q = Heads(np.random.default_rng(2).standard_normal((total, heads, dim)), dtype)
    out = Heads(np.zeros((total, heads, dim)), dtype)
    keep = attend(cache, rows, q, out)
    got = out.get()[0]
    with np.errstate(invalid='ignore'):
        values = cache.values()
        want, mass, size = attention(values, cache, q.float(), starts, firsts, [n] * 3, 1 / 8)
    assert np.isfinite(got[:n]).all() and np.isfinite(got[2 * n:]).all()
    finite = np.isfinite(want)
    assert finite.sum() == want.size - 2 * 3  # the last query of stream 1: two heads each of 2 + 1 dims
    assert (np.isnan(got) == np.isnan(want)).all() and (got[np.isinf(want)] == want[np.isinf(want)]).all()
    assert np.abs(got - want)[finite].max() <= 4 * STEP[dtype] * 5 + 1e-5
    del keep


def test_logits_that_are_not_finite():
    """A NaN in a visible key makes its queries NaN and no others; a key at minus infinity weighs nothing;
    with nothing but minus infinity the softmax is 0 / 0."""
    dim, n = 64, 5
    cache = Cache(1, 1, dim, 3, 0, F32, max_tokens=n, fill=1, positions=[10])
    k, v = (x.copy() for x in cache.values())
    k[0, 0, cache.slot(11), 0] = np.nan
    cache.write(k, v)
    rows, firsts, total = rows_struct(cache, n=n)
    q = np.abs(np.random.default_rng(2).standard_normal((n, 1, dim)))
    qd, out = Heads(q, F32), Heads(np.zeros((n, 1, dim)), F32)
    attend(cache, rows, qd, out)
    got = out.get()[0]
    assert np.isnan(got[1:4]).all() and np.isfinite(got[[0, 4]]).all()
    k[0, 0, cache.slot(11)] = -np.inf
    cache.write(k, v)
    attend(cache, rows, qd, out)
    want, mass, size = attention(cache.values(), cache, qd.float(), [10], firsts, [n], 1 / 8)
    assert np.abs(out.get()[0] - want).max() < 1e-5
    cache.write(np.full_like(k, -np.inf), v)
    attend(cache, rows, qd, out)
    assert np.isnan(out.get()[0]).all()


def test_offsets_past_32_bits():
    """Rows of one cache more than 4 GiB apart, within a stream and between streams."""
    dim, slots = 256, 5_000_000
    for order in ((0, 1, 2), (1, 0, 2)):
        cache = Cache.__new__(Cache)
        cache.dims, cache.dim, cache.window, cache.sinks, cache.ring, cache.dtype = (2, 1, slots), dim, slots, 0, slots, F32
        rows = []
        for _ in range(2):
            p = ctypes.c_void_p()
            hip().hipMalloc(ctypes.byref(p), ctypes.c_size_t(2 * slots * dim * 4))
            hip().hipMemset(p, 0, ctypes.c_size_t(2 * slots * dim * 4))
            rows.append(p)
        starts = [slots + 7, 3]
        cache.positions = Device(np.asarray(starts, np.int64))
        from streamtx.cache import _Cache
        cache.struct = _Cache(2, 1, dim, slots, 0, slots, F32, slots, slots, 1, rows[0].value, rows[1].value, None, None,
                              cache.positions.ptr)
        mark = np.random.default_rng(4).standard_normal((3, dim)).astype(np.float32)
        places = [slots - 1, 4_500_000, 2 * slots - 1]  # of stream 0, 0, and 1 (outside its window)
        for m, at in zip(mark, places):
            hip().hipMemcpy(ctypes.c_void_p(rows[1].value + at * dim * 4), m.ctypes.data_as(ctypes.c_void_p), dim * 4, 1)
        r, firsts, total = rows_struct(cache, n=1)
        q, k, v = (Heads(np.ones((2, 1, dim)), F32) for _ in range(3))
        out = Heads(np.zeros((2, 1, dim)), F32)
        append(cache, r, q, k, v, out)  # position slots + 7 lands in slot 7, position 3 in slot 3
        keep = attend(cache, r, q, out)
        got = out.get()[0]
        # Stream 0: keys are zero but the new one, whose logit is 256 / 16; stream 1 sees three zeros and it.
        e = np.exp(-16.0)
        want0 = (1 + e * (mark[0].astype(float) + mark[1])) / (1 + e * (slots - 1))
        want1 = 1 / (1 + 3 * e) * np.ones(dim)
        assert np.abs(got[0, 0] - want0).max() < 1e-4 and np.abs(got[1, 0] - want1).max() < 1e-6
        for p in rows:
            hip().hipFree(p)
        del keep


# ------------------------------------------------------------------------------------------------
# as a serving program uses them

class Model:
    """One attention layer of a small model over a cache: norm, rotation, append, attention."""

    def __init__(self, dtype, stored, streams, max_tokens, heads=4, kv=2, dim=64, window=24, sinks=3):
        self.dtype, self.heads, self.kv, self.dim = dtype, heads, kv, dim
        rng = np.random.default_rng(11)
        self.gains = [Device((1 + 0.1 * rng.standard_normal(dim)).astype(np.float32)) for _ in range(2)]
        self.freq = Device(frequencies(dim))
        self.cache = Cache(streams, kv, dim, window, sinks, stored, max_tokens=max_tokens)
        self.at = np.zeros(streams, np.int64)

    def call(self, x, counts, n):
        """x [rows, heads + 2 kv, dim] of unequal numbers of tokens; returns the outputs."""
        ends = Device(np.concatenate(([0], np.cumsum(counts))).astype(np.int32))
        rows, _, total = rows_struct(self.cache, counts, n, ends)
        h, kv = self.heads, self.kv
        q, k, v = (Heads(x[:, a:b], self.dtype) for a, b in ((0, h), (h, h + kv), (h + kv, h + 2 * kv)))
        out = Heads(np.zeros((total, h, self.dim)), self.dtype)
        self.cache.positions.put(self.at)
        append(self.cache, rows, q, k, v, out, *self.gains, inv_freq=self.freq, rope_dims=self.dim, halves=1)
        keep = attend(self.cache, rows, out, out)  # in place, as a layer may
        got = out.get()[0]
        self.at = self.at + np.asarray(counts)
        del keep, ends
        return got


@pytest.mark.parametrize('types', PAIRS, ids=pair_id)
def test_a_prompt_in_pieces(types):
    """Whatever pieces a prompt comes in, the cache holds the same bits and the outputs agree."""
    total = 90
    x = np.random.default_rng(5).standard_normal((total, 8, 64))
    results = []
    for pieces in ([90], [1] * 90, [40, 1, 1, 30, 18]):
        model = Model(*types, streams=1, max_tokens=90)
        got = []
        for n in pieces:
            got.append(model.call(x[int(model.at[0]):int(model.at[0]) + n], [n], max(n, 1)))
        results.append((np.concatenate(got), model.cache.raw()))
    for got, raw in results[1:]:
        for a, b in zip(raw, results[0][1]):
            assert a.tobytes() == b.tobytes()
        # Two orders of the same sums: each within the bound of the exact result.
        assert np.abs(got - results[0][0]).max() <= 4 * max(STEP[types[0]], 2.0**-20) * 6


@pytest.mark.parametrize('types', PAIRS, ids=pair_id)
def test_streams_do_not_depend_on_their_neighbours(types):
    """A stream's bits are the same alone and in a batch with others, and from run to run."""
    x = np.random.default_rng(6).standard_normal((5, 60, 8, 64))
    batch = Model(*types, streams=5, max_tokens=30)
    first = batch.call(np.concatenate([x[b, :n] for b, n in enumerate((30, 7, 0, 1, 16))]), [30, 7, 0, 1, 16], 30)
    step = batch.call(np.concatenate([x[b, 30:31] for b in range(5)]), [1] * 5, 1)
    for b, n in enumerate((30, 7, 0, 1, 16)):
        for _ in range(2):
            alone = Model(*types, streams=1, max_tokens=30)
            ends = np.cumsum((0, 30, 7, 0, 1, 16))
            if n:
                assert alone.call(x[b, :n], [n], 30).tobytes() == first[ends[b]:ends[b + 1]].tobytes()
            assert alone.call(x[b, 30:31], [1], 1).tobytes() == step[b:b + 1].tobytes()


@pytest.mark.parametrize('window', [24, 4000])
def test_captured_graph(window):
    """A step captured into a graph and replayed, with new inputs and positions between the replays and the
    program's own eager work on the same cache in between: every replay gives what the eager calls give."""
    streams, heads, kv, dim, sinks = 3, 4, 2, 64, 2
    h = hip()
    caches = [Cache(streams, kv, dim, window, sinks, F16, fill=9, positions=[0, 100, 7]) for _ in range(2)]
    rng = np.random.default_rng(8)
    gains = [Device((1 + 0.1 * rng.standard_normal(dim)).astype(np.float32)) for _ in range(2)]
    freq = Device(frequencies(dim))
    sets = []
    for c in caches:
        rows, _, total = rows_struct(c, n=1)
        q, k, v = (Heads(np.zeros((total, n, dim)), F16) for n in (heads, kv, kv))
        rotated, out = Heads(np.zeros((total, heads, dim)), F16), Heads(np.zeros((total, heads, dim)), F16)
        need = workspace_bytes(c, rows, heads, F16)
        sets.append((c, rows, q, k, v, rotated, out, Device(np.zeros(max(need, 1), np.uint8)) if need else None))
    assert (window == 4000) == (sets[0][-1] is not None)  # the long window is split

    def calls(s, stream):
        c, rows, q, k, v, rotated, out, ws = s
        append(c, rows, q, k, v, rotated, *gains, inv_freq=freq, rope_dims=dim, stream=stream)
        attend(c, rows, rotated, out, stream=stream, workspace=ws)

    stream = ctypes.c_void_p()
    h.hipStreamCreateWithFlags(ctypes.byref(stream), 1)
    graph, execution = ctypes.c_void_p(), ctypes.c_void_p()
    h.hipStreamBeginCapture(stream, 1)
    calls(sets[0], stream)
    h.hipStreamEndCapture(stream, ctypes.byref(graph))
    h.hipGraphInstantiate(ctypes.byref(execution), graph, None, None, ctypes.c_size_t(0))
    at = np.array([0, 100, 7], np.int64)
    for step in range(6):
        x = rng.standard_normal((streams, heads + 2 * kv, dim))
        for s in sets:
            s[0].positions.put(at)
            for t, part in zip(s[2:5], (x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:])):
                t.dev.put(encode(part, F16))
        sync()
        h.hipGraphLaunch(execution, stream)
        sync()
        calls(sets[1], None)
        sync()
        assert sets[0][6].get()[0].tobytes() == sets[1][6].get()[0].tobytes(), step
        for a, b in zip(caches[0].raw(), caches[1].raw()):
            assert a.tobytes() == b.tobytes()
        at += 1
    h.hipGraphExecDestroy(execution)
    h.hipGraphDestroy(graph)
    h.hipStreamDestroy(stream)


def test_calls_on_two_streams():
    """Two caches, workspaces and streams at once."""
    h = hip()
    sets = []
    for seed in range(2):
        c = Cache(1, 2, 64, 6000, 4, BF16, fill=seed, positions=[9000])
        rows, firsts, _ = rows_struct(c, n=1)
        q = Heads(np.random.default_rng(seed).standard_normal((1, 4, 64)), BF16)
        out = Heads(np.zeros((1, 4, 64)), BF16)
        s = ctypes.c_void_p()
        h.hipStreamCreateWithFlags(ctypes.byref(s), 1)
        sets.append((c, rows, q, out, s))
    alone = []
    for c, rows, q, out, s in sets:
        attend(c, rows, q, out, stream=s)
        alone.append(out.get()[0])
    keep = []
    for _ in range(10):
        for c, rows, q, out, s in sets:
            keep.append(attend(c, rows, q, out, stream=s))
    for (c, rows, q, out, s), want in zip(sets, alone):
        assert out.get()[0].tobytes() == want.tobytes()
        h.hipStreamDestroy(s)


def test_rows_past_the_limits_are_left_out():
    """Offsets that name more rows than max_tokens or than the call has: the rest stays as it is."""
    cache = Cache(2, 1, 64, 10, 0, F32, max_tokens=4, fill=2, positions=[0, 50])
    before = cache.raw()
    ends = Device(np.array([0, 6, 40], np.int32))
    from streamtx.cache import _Rows
    rows = _Rows(8, 4, ends.ptr)
    x = Heads(np.random.default_rng(1).standard_normal((8, 1, 64)), F32)
    out = Heads(np.full((8, 1, 64), 5.0), F32)
    append(cache, rows, x, x, x, out)
    got = out.get()[0]
    assert (got[4:6] == 5).all() and (got[:4] == x.float()[:4]).all() and (got[6:] == x.float()[6:]).all()
    after = cache.raw()
    assert (after[0][0, 0, :4] == x.data[:4, 0]).all() and (after[0][0, 0, 4:] == before[0][0, 0, 4:]).all()
    out = Heads(np.full((8, 1, 64), 5.0), F32)
    keep = attend(cache, rows, x, out)
    got = out.get()[0]
    assert (got[4:6] == 5).all() and (got[:4] != 5).all() and (got[6:] != 5).all()
    del keep

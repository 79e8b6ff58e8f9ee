"""Batches with sinks, head norms and other K/V storage (st_batch_create_with) on the GPU: the QKV projection, the
cache operators and the rest of the step together, against the model in 64 bits."""
import numpy as np
import pytest

from streamtx import BatchOptions, BatchRuntime, KvStorage, ModelConfig, WeightStorage, round_bf16, synthetic_checkpoint

pytestmark = pytest.mark.gpu

STORED = {KvStorage.F16: 2.0**-11, KvStorage.BF16: 2.0**-8}

SHAPES = {
    'small': ModelConfig(2, 256, 4, 512, 24, 64),
    'dh32': ModelConfig(3, 128, 4, 256, 16, 32),
    'dh128': ModelConfig(2, 256, 2, 512, 20, 29),
    'long': ModelConfig(1, 128, 2, 128, 1500, 32),
}


def checkpoint(c, seed, head_norm):
    w = synthetic_checkpoint(c, seed=seed, std=0.08)
    if head_norm:
        rng = np.random.default_rng(seed + 1)
        for l in range(c.layers):
            for n in ('q_norm', 'k_norm'):
                w[f'layers.{l}.{n}'] = (1 + 0.2 * rng.standard_normal(c.dim)).astype(np.float32)
    return w


U = 2.0**-24  # half a step of FP32


class Model:
    """The step in 64 bits, one stream, and beside each value a bound of how far FP32 arithmetic may be from it:
    a sum of n products is off by at most (n + 2) U times the sum of their sizes, whatever its order, and by
    its operands' errors through the partial derivatives; functions (root, exponential, cosine) by 4 U.
    `cache`: keys and values come from there instead of from its own projections (what a quantised cache
    holds; they carry no error then)."""

    def __init__(self, c, w, sinks, head_norm):
        self.c, self.sinks, self.head_norm = c, sinks, head_norm
        self.w = {k: v.astype(np.float64) for k, v in w.items()}
        self.freq = np.array([np.float32(10000.0) ** np.float32(-(2 * j) / c.dim) for j in range(c.dim // 2)], np.float32)
        self.reset()

    def reset(self):
        self.t, self.rows = 0, [([], []) for _ in range(self.c.layers)]

    def product(self, name, x):
        """W x and its error, x a pair (value, error)."""
        m = self.w[name]
        return m @ x[0], np.abs(m) @ x[1] + (m.shape[1] + 2) * U * (np.abs(m) @ np.abs(x[0]))

    def norm(self, x, name):
        v, e = x
        g, n = self.w[name], v.shape[-1]
        square = (v * v).mean(-1, keepdims=True) + self.c.epsilon
        relative = (np.abs(v) * e).mean(-1, keepdims=True) / square + (n / 2 + 8) * U
        y = v / np.sqrt(square) * g
        return y, np.abs(g) / np.sqrt(square) * e + np.abs(y) * relative

    def rotate(self, x):
        angle = (np.float32(self.t) * self.freq).astype(np.float64)
        co, si = np.cos(angle), np.sin(angle)
        (v, e), y, f = x, x[0].copy(), x[1].copy()
        a, b, ea, eb = v[:, 0::2], v[:, 1::2], e[:, 0::2], e[:, 1::2]
        y[:, 0::2], y[:, 1::2] = a * co - b * si, a * si + b * co
        f[:, 0::2] = np.abs(co) * ea + np.abs(si) * eb + 7 * U * (np.abs(a) + np.abs(b))
        f[:, 1::2] = np.abs(si) * ea + np.abs(co) * eb + 7 * U * (np.abs(a) + np.abs(b))
        return y, f

    def new_rows(self, l, x):
        """Query, key and value of a layer's input."""
        c, p = self.c, f'layers.{l}.'
        z = self.norm(x, p + 'norm1')
        q, k, v = (tuple(a.reshape(c.heads, c.dim) for a in self.product(p + n, z)) for n in 'qkv')
        if self.head_norm:
            q, k = self.norm(q, p + 'q_norm'), self.norm(k, p + 'k_norm')
        return self.rotate(q), self.rotate(k), v

    def embed(self, event):
        return self.product('input', (event.astype(np.float64), np.zeros(event.shape)))

    def step(self, event, cache=None):
        """(score, its error), (hidden, its error)."""
        c, t = self.c, self.t
        x = self.embed(event)
        low = max(t - c.window + 1, 0)
        seen = np.concatenate((np.arange(min(self.sinks, low)), np.arange(low, t + 1)))
        hidden = []
        self.new = []
        for l in range(c.layers):
            p = f'layers.{l}.'
            q, k, v = self.new_rows(l, x)
            self.new.append((k, v))
            self.rows[l][0].append(k)
            self.rows[l][1].append(v)
            if cache is None:  # [head, seen, dim]
                (keys, ek), (values, ev) = (tuple(np.stack([r[i] for r in rows])[seen].transpose(1, 0, 2) for i in range(2))
                                            for rows in self.rows[l])
            else:
                at = np.where(seen < self.sinks, seen, self.sinks + (seen - self.sinks) % c.window)
                keys, values = cache[0][l][:, at].astype(np.float64), cache[1][l][:, at].astype(np.float64)
                ek, ev = np.zeros(keys.shape), np.zeros(keys.shape)
            dot = lambda a, b: np.einsum('hd,hnd->hn', a, b) / np.sqrt(c.dim)  # noqa: E731
            s = dot(q[0], keys)
            es = dot(q[1], np.abs(keys)) + dot(np.abs(q[0]), ek) + (c.dim + 8) * U * dot(np.abs(q[0]), np.abs(keys))
            weight = np.exp(s - s.max(-1, keepdims=True))
            weight /= weight.sum(-1, keepdims=True)
            # A weight's relative error: twice the largest logit error, the exponential's, the sum's.
            relative = 2 * es.max(-1, keepdims=True) + 4 * 2.0**-22 + (len(seen) + 8) * 2 * U
            a = np.einsum('hn,hnd->hd', weight, values)
            ea = np.einsum('hn,hnd->hd', weight, ev + np.abs(values) * relative[..., None])
            y = self.product(p + 'out', (a.reshape(-1), ea.reshape(-1)))
            x = (x[0] + y[0], x[1] + y[1] + U * np.abs(x[0] + y[0]))
            z = self.norm(x, p + 'norm2')
            (g, eg), (u, eu) = self.product(p + 'gate', z), self.product(p + 'up', z)
            silu = g / (1 + np.exp(-g))  # its derivative is below 1.1
            act = silu * u
            y = self.product(p + 'down', (act, 1.1 * eg * np.abs(u) + np.abs(silu) * eu + 10 * U * np.abs(act)))
            x = (x[0] + y[0], x[1] + y[1] + U * np.abs(x[0] + y[0]))
            hidden.append(x)
        self.t += 1
        score = self.product('score', self.norm(x, 'final_norm'))
        return (score[0][0], score[1][0]), tuple(np.array([h[i] for h in hidden]) for i in range(2))

    def ring(self):
        """Keys and values as a snapshot has them, each (value, error)."""
        c = self.c
        out = [[np.zeros((c.layers, c.heads, self.sinks + c.window, c.dim)) for _ in range(2)] for _ in range(2)]
        for l in range(c.layers):
            for i in range(2):
                for p in range(self.t):
                    at = p if p < self.sinks else self.sinks + (p - self.sinks) % c.window
                    for e in range(2):
                        out[i][e][l][:, at] = self.rows[l][i][p][e]
        return out


def within(got, want):
    value, error = want
    ratio = float((np.abs(np.asarray(got, np.float64) - value) / (error + 1e-30)).max())
    assert ratio <= 1, ratio


def events(c, seed, steps, streams):
    return np.random.default_rng(seed).standard_normal((steps, streams, c.features)).astype(np.float32)


@pytest.mark.parametrize('name,streams,sinks,head_norm,weights', [
    ('small', 3, 4, False, WeightStorage.AS_MODEL),
    ('small', 17, 0, True, WeightStorage.AS_MODEL),
    ('dh32', 5, 3, True, WeightStorage.BF16),
    ('dh128', 2, 1, True, WeightStorage.AS_MODEL),
    ('dh128', 34, 7, False, WeightStorage.BF16),
    ('long', 1, 5, True, WeightStorage.AS_MODEL),
])
def test_sinks_and_head_norms(name, streams, sinks, head_norm, weights):
    """Scores and state of every stream, through the window's first turns, with resets."""
    c = SHAPES[name]
    w = checkpoint(c, 5, head_norm)
    used = {k: round_bf16(v) if weights == WeightStorage.BF16 and not k.endswith(('q_norm', 'k_norm')) else v
            for k, v in w.items()}
    steps = 60 if name != 'long' else 1530
    x = events(c, 6, steps, streams)
    models = [Model(c, used, sinks, head_norm) for _ in range(streams)]
    checked = range(steps) if name != 'long' else {0, 3, 700, 1504, 1505, 1529}
    with BatchRuntime((c, w, False), streams, options=BatchOptions(weights, sinks, head_norm)) as rt:
        for i in range(steps):
            if i == 33 and name != 'long':
                rt.reset(streams - 1)
                models[-1].reset()
            got = rt.step(x[i])
            for b, m in enumerate(models):
                if name == 'long' and i not in checked:  # keys and values of one layer do not depend on attention
                    _, k, v = m.new_rows(0, m.embed(x[i, b]))
                    m.rows[0][0].append(k)
                    m.rows[0][1].append(v)
                    m.t += 1
                    continue
                want, hidden = m.step(x[i, b])
                within(got[b], want)
        for b in (0, streams - 1):
            state = rt.snapshot(b)
            assert state[0] == models[b].t
            for a, o in zip(state[1:3], models[b].ring()):
                within(a, o)
            if b == streams - 1:
                within(state[3], hidden)


@pytest.mark.parametrize('kv', [KvStorage.F16, KvStorage.BF16, KvStorage.INT4], ids=lambda k: k.name)
@pytest.mark.parametrize('streams,sinks', [(2, 0), (19, 3)])
def test_kv_storage(kv, streams, sinks):
    """One layer, whose keys and values follow from the event alone: the stored rows are the exact ones rounded
    to their type, and the step is exact over what the rows stand for."""
    c = ModelConfig(1, 128, 2, 256, 12, 32)
    w = checkpoint(c, 8, True)
    steps = 40
    x = events(c, 9, steps, streams)
    models = [Model(c, w, sinks, True) for _ in range(streams)]
    with BatchRuntime((c, w, False), streams, options=BatchOptions(sinks=sinks, head_norm=True, kv_dtype=kv)) as rt:
        for i in range(steps):
            got = rt.step(x[i])
            for b in {0, streams - 1}:
                m = models[b]
                state = rt.snapshot(b)
                want, hidden = m.step(x[i, b], cache=state[1:3])
                within(got[b], want)
                within(state[3], hidden)
                at = i if i < sinks else sinks + (i - sinks) % c.window
                for stored, (exact, error) in zip(state[1:3], m.new[0]):
                    row = stored[0][:, at].astype(np.float64)
                    if kv == KvStorage.INT4:
                        g = exact.reshape(c.heads, -1, 32)
                        step = (g.max(-1) - g.min(-1))[..., None] / 15 * (1 + 2.0**-10)
                        # The range's ends are rounded to FP16, and all of it computed in FP32.
                        slack = 2.0**-10 * np.abs(g).max(-1, keepdims=True) + 2 * error.max()
                        assert (np.abs(row.reshape(g.shape) - g) <= step / 2 + slack).all()
                    else:
                        assert (np.abs(row - exact) <= STORED[kv] * np.abs(exact) + 2 * error).all()


def test_default_options_are_the_plain_batch():
    """st_batch_create's own batch, bit for bit; sinks that the window still covers change nothing but the
    order of sums."""
    c = SHAPES['small']
    w = checkpoint(c, 3, False)
    x = events(c, 4, 30, 5)
    with BatchRuntime((c, w, False), 5) as a, BatchRuntime((c, w, False), 5, options=BatchOptions()) as b, \
            BatchRuntime((c, w, False), 5, options=BatchOptions(sinks=6)) as s:
        models = [Model(c, w, 0, False) for _ in range(5)]
        for i in range(30):
            plain = a.step(x[i])
            np.testing.assert_array_equal(plain, b.step(x[i]))
            sunk = s.step(x[i])
            for j, m in enumerate(models):
                want, _ = m.step(x[i, j])
                within(plain[j], want)
                if i < c.window:
                    within(sunk[j], want)
        for p, q in zip(a.snapshot(2), b.snapshot(2)):
            np.testing.assert_array_equal(p, q)


@pytest.mark.parametrize('kv', [KvStorage.AS_MODEL, KvStorage.INT4], ids=lambda k: k.name)
def test_eager_device_run_and_resets(kv):
    """The captured step, eager launches and a preloaded run give the same bits, after resets too."""
    c = SHAPES['dh32']
    w = checkpoint(c, 2, True)
    x = events(c, 1, 24, 4)
    options = BatchOptions(sinks=2, head_norm=True, kv_dtype=kv)
    with BatchRuntime((c, w, False), 4, options=options) as a, BatchRuntime((c, w, False), 4, options=options) as b, \
            BatchRuntime((c, w, False), 4, options=options) as d:
        b.set_eager(True)
        for i in range(24):
            if i == 9:
                for rt in (a, b):
                    rt.reset(2)
            np.testing.assert_array_equal(a.step(x[i]), b.step(x[i]))
        for rt in (a, d):
            rt.reset()
            for p in rt.snapshot(1):
                assert not np.any(p)
            rt.device_run(x)
        b.reset()
        for i in range(24):
            b.step(x[i])
        for s in range(4):
            for p, q, r in zip(a.snapshot(s), b.snapshot(s), d.snapshot(s)):
                np.testing.assert_array_equal(p, q)
                np.testing.assert_array_equal(p, r)

"""The formulas of csrc/adamw.hip restated with numpy, one array operation per operation: in float32 (`step32`: what the kernel has to
give bit for bit) and in float64.  Test infrastructure."""
import numpy as np

BLOCK = 256
M32 = np.uint64(0xFFFFFFFF)


def bf16_to_f32(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def key(seed, step):
    z = (seed + step * 0x9E3779B97F4A7C15) & (1 << 64) - 1
    z = ((z ^ z >> 30) * 0xBF58476D1CE4E5B9) & (1 << 64) - 1
    z = ((z ^ z >> 27) * 0x94D049BB133111EB) & (1 << 64) - 1
    z ^= z >> 31
    return z & 0xFFFFFFFF, z >> 32


def random_bits(index, n, seed, step):
    """32 bits for elements index .. index + n - 1 of a step."""
    k0, k1 = key(seed, step)
    i = np.arange(n, dtype=np.uint64) + np.uint64(index)
    x = ((i & M32) ^ np.uint64(k0)) + (i >> np.uint64(32)) * np.uint64(0x9E3779B1) & M32
    x = (x ^ x >> np.uint64(16)) * np.uint64(0x7FEB352D) + np.uint64(k1) & M32
    x = (x ^ x >> np.uint64(15)) * np.uint64(0x846CA68B) & M32
    return x ^ x >> np.uint64(16)


def scalars(hp, step):
    f, b1, b2 = np.float32, hp['betas'][0], hp['betas'][1]
    return dict(b1=f(b1), c1=f(1 - b1), b2=f(b2), c2=f(1 - b2), decay=f(1 - hp['lr'] * hp['weight_decay']), step=f(hp['lr'] / (1 - b1 ** step)),
                rbc2=f((1 - b2 ** step) ** -0.5), eps=f(hp['eps']), d=f(hp.get('ema') or 0), cd=f(1 - (hp.get('ema') or 0)))


def step32(p, g, m, v, hp, step, factor=1.0, ema=None):
    """float32 arrays -> (p, m, v, ema), every operation rounded once."""
    s = scalars(hp, step)
    with np.errstate(all='ignore'):
        g = g * np.float32(factor)
        m = m * s['b1'] + g * s['c1']
        v = v * s['b2'] + (g * g) * s['c2']
        p = p * s['decay'] - (m / (np.sqrt(v) * s['rbc2'] + s['eps'])) * s['step']
        if ema is not None:
            ema = ema * s['d'] + p * s['cd']
    for x in (p, m, v):
        assert x.dtype == np.float32
    return p, m, v, ema


def step64(p, g, m, v, hp, step, factor=1.0):
    b1, b2 = hp['betas']
    p, g, m, v = (x.astype(np.float64) for x in (p, g, m, v))
    g = g * factor
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - hp['lr'] * hp['weight_decay']) - hp['lr'] / (1 - b1 ** step) * m / (np.sqrt(v / (1 - b2 ** step)) + hp['eps'])
    return p, m, v


def _blocks(x):
    return [x[i:i + BLOCK] for i in range(0, len(x), BLOCK)]


def to_8_bits(x, noise, second):
    """x rounded to what 8 bits hold (float32 -> float32), by arithmetic in float64: noise: 16 random bits per element."""
    low = 30 if second else 14      # exponents below the block's that are still normal
    out = []
    for b, r in zip(_blocks(x), _blocks(noise)):
        top = np.max(np.abs(b)) if len(b) else 0.0
        if not np.isfinite(top):
            out.append(np.full(len(b), np.nan, np.float32))
            continue
        frac, e = np.frexp(np.float64(top))         # top = frac * 2^e, frac in [0.5, 1)
        e = max(int(e) + (1 if frac > 0.9375 else 0), -125) if top > 0 else -125
        a = np.abs(b.astype(np.float64))
        q = np.ldexp(1.0, np.maximum(np.frexp(a)[1], e - low) - 4)
        # the kernel forms a * 2^k as a float32 first: values below 2^-149 * 2^-k are rounded to it
        grain = np.ldexp(1.0, e - low - 4 - 20)
        a = np.where(a < np.ldexp(1.0, e - low - 1), np.rint(a / grain) * grain, a)
        y = np.floor(a / q + (r.astype(np.float64) * 16 + 8) / 2 ** 20) * q
        if second:
            y = np.where((y == 0) & (b > 0), np.ldexp(1.0, e - low - 4), y)
        out.append((np.sign(b) * y).astype(np.float32))
    return np.concatenate(out) if out else x


def to_bf16(x, bits):
    """Stochastic rounding to bfloat16 (as float32); bits: the element's 32 random bits."""
    u = x.view(np.uint32)
    r = ((bits * np.uint64(0x9E3779B1)) & M32) >> np.uint64(16)
    finite = (u & 0x7F800000) != 0x7F800000
    y = np.where(finite, (u.astype(np.uint64) + r) & np.uint64(0xFFFF0000), (u & 0xFFFF0000).astype(np.uint64) | np.where(u & 0xFFFF, 0x400000, 0).astype(np.uint64))
    return y.astype(np.uint32).view(np.float32)


class Tensors:
    """A list of tensors under AdamW with one set of hyper-parameters, on float32 arrays; bits 32 or 8, bf16 or float32 parameters."""

    def __init__(self, params, hp, bits=32, bf16=False, seed=0, index=0):
        self.hp, self.bits, self.bf16, self.seed = hp, bits, bf16, seed
        self.p = [x.copy() for x in params]
        self.m = [np.zeros_like(x) for x in params]
        self.v = [np.zeros_like(x) for x in params]
        self.ema = [x.copy() for x in params]
        self.t = [0] * len(params)
        self.index, at = [], index
        for x in params:
            self.index.append(at)
            at += len(x)

    def step(self, grads, max_norm=None):
        factor = 1.0
        if max_norm is not None:
            norm = float(np.sqrt(sum(float(np.sum(g.astype(np.float64) ** 2)) for g in grads if g is not None)))
            f = max_norm / (norm + 1e-6)
            factor = 1.0 if f >= 1 else np.float32(f)
        s = scalars(self.hp, 1)
        for i, g in enumerate(grads):
            if g is None:
                self.ema[i] = self.ema[i] * s['d'] + self.p[i] * s['cd']
                continue
            self.t[i] += 1
            p, m, v, e = step32(self.p[i], g, self.m[i], self.v[i], self.hp, self.t[i], factor, self.ema[i])
            h = random_bits(self.index[i], len(p), self.seed, self.t[i])
            if self.bits == 8:
                m, v = to_8_bits(m, h & np.uint64(0xFFFF), False), to_8_bits(v, h >> np.uint64(16), True)
            self.p[i] = to_bf16(p, h) if self.bf16 else p
            self.m[i], self.v[i], self.ema[i] = m, v, e

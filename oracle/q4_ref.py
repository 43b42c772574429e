"""Float64 restatement of the 4-bit KV cache: row format, rotary positions with three
axes, attention over held rows, accumulated weights and eviction.

Written from the definitions in include/dz_attn.h, one sequence and one head at a
time; the norm, the rotation's '+' sign and the gate are the reference's
(Daiza-engine/src/math/rmsnorm.rs:152-178, math/rope.rs:187-231,
model/attention.rs:90-203)."""
import numpy as np

HD, GRP, PAIRS, GROUP = 256, 6, 32, 32
SCALE_MAX = 896.0
EPS = float(np.float32(1e-6))


def scale(amax):
    """max|x| / 7 to 4 significant bits (nearest even; grid 2^-17 below 2^-14), at most 896."""
    t = np.minimum(np.asarray(amax, np.float64) / 7, SCALE_MAX)
    _, e = np.frexp(t)
    step = np.ldexp(1.0, np.maximum(e, -13) - 4)
    return np.minimum(np.rint(t / step) * step, SCALE_MAX)


def codes(x):
    """Codes [..., 256] and scales [..., 8] of rows x [..., 256]."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), 0.0, x)
    g = x.reshape(*x.shape[:-1], HD // GROUP, GROUP)
    s = scale(np.abs(g).max(-1))
    safe = np.where(s > 0, s, 1.0)[..., None]
    c = np.clip(np.rint(np.clip(g / safe, -9, 9)), -7, 7)
    return np.where(s[..., None] > 0, c, 0.0).reshape(x.shape), s


def hold(x):
    """The values that a cache holds for rows x."""
    c, s = codes(x)
    return c * np.repeat(s, GROUP, -1)


def axes(sections=(11, 11, 10), interleaved=False):
    if interleaved:
        return np.array([1 if i % 3 == 1 and i < 3 * sections[1] else 2 if i % 3 == 2 and i < 3 * sections[2] else 0
                         for i in range(PAIRS)])
    return np.repeat([0, 1, 2], sections)


def turn(x, norm, pos, axis=None, base=1.0e7, eps=EPS):
    """RMS norm and rotation of x [tokens][heads][256] at pos [tokens][3]."""
    axis = axes() if axis is None else axis
    x = np.asarray(x, np.float64)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(norm, np.float64)
    theta = np.asarray(pos, np.float64)[:, axis] * base ** (-2.0 * np.arange(PAIRS) / 64)
    c, s = np.cos(theta)[:, None], np.sin(theta)[:, None]
    a, b = x[..., :PAIRS], x[..., PAIRS:2 * PAIRS]
    return np.concatenate([a * c + b * s, b * c + a * s, x[..., 2 * PAIRS:]], -1)


class Cache:
    """K and V of one layer and sequence as held, [length][kv heads][256], and the accumulated weights."""

    def __init__(self, kvc, k=None, v=None):
        self.k = np.zeros((0, kvc, HD)) if k is None else hold(k)
        self.v = np.zeros((0, kvc, HD)) if v is None else hold(v)
        self.w = np.zeros((kvc, len(self.k)))

    def extend(self, q_gate, k, v, q_norm, k_norm, pos=None, axis=None):
        """T tokens in order: append, attend, gate.  q_gate [T][6 kvc][512], k and v [T][kvc][256];
        returns [T][6 kvc][256].  The weights grow as in a decode call per token."""
        n, T, kvc = len(self.k), len(k), self.k.shape[1]
        pos = np.repeat(np.arange(n, n + T)[:, None], 3, 1) if pos is None else np.asarray(pos)
        q_gate = np.asarray(q_gate, np.float64)
        q = turn(q_gate[..., :HD], q_norm, pos, axis) / 16
        self.k = np.concatenate([self.k, hold(turn(k, k_norm, pos, axis))])
        self.v = np.concatenate([self.v, hold(v)])
        self.w = np.concatenate([self.w, np.zeros((kvc, T))], 1)
        out = np.empty((T, GRP * kvc, HD))
        for t in range(T):
            m = n + t + 1
            for i in range(GRP * kvc):
                s = self.k[:m, i // GRP] @ q[t, i]
                p = np.exp(s - s.max())
                p /= p.sum()
                out[t, i] = p @ self.v[:m, i // GRP]
                self.w[i // GRP, :m] += p
        with np.errstate(over="ignore"):
            return out / (1 + np.exp(-q_gate[..., HD:]))

    def evict(self, keep, recent):
        """The last `recent` entries and the heaviest others, `keep` in all; the kept indices [kvc][keep]."""
        n = len(self.k)
        if n <= keep:
            return np.repeat(np.arange(n)[None], len(self.w), 0)
        recent = min(recent, keep)
        old = n - recent
        idx = np.stack([np.concatenate([np.sort(np.lexsort((np.arange(old), -w[:old]))[:keep - recent]),
                                        np.arange(old, n)]) for w in self.w])
        h = np.arange(len(self.w))
        self.k, self.v = self.k[idx.T, h], self.v[idx.T, h]
        self.w = np.take_along_axis(self.w, idx, 1)
        return idx

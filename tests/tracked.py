"""Values in float64 together with a bound on how far an f32 evaluation may be off them, and the plain forms of the
adapter, control and clipping operators in that arithmetic.

Every f32 operation adds at most half a step of its result, U = 2^-24 relative (torch.finfo(float32).eps / 2); a sum of K
products in any order adds at most (K + 1) U times the sum of the products' magnitudes.  Bounds propagate to first
order with the magnitudes enlarged by their own bounds, so nothing here is fitted to an observed error."""
import numpy as np

U = 2.0 ** -24


class T:
    """v: exact values, e: bound on |f32 value - v|"""

    def __init__(self, v, e=0.0):
        self.v = np.asarray(v, np.float64)
        self.e = np.broadcast_to(np.asarray(e, np.float64), self.v.shape)

    @property
    def mag(self):
        return np.abs(self.v) + self.e

    def __getitem__(self, i):
        return T(self.v[i], self.e[i])

    @property
    def T(self):
        return T(self.v.T, self.e.T)


def add(a, b):
    v = a.v + b.v
    return T(v, a.e + b.e + U * (np.abs(v) + a.e + b.e))


def mul(a, b):
    return T(a.v * b.v, a.mag * b.e + a.e * b.mag + U * a.mag * b.mag)


def dot(a, b, extra=0):
    """a @ b, summed in f32 in any order (also together with `extra` more terms of other sums)"""
    k = a.v.shape[-1]
    return T(a.v @ b.v, a.mag @ b.e + a.e @ b.mag + (k + 1 + extra) * U * (a.mag @ b.mag))


def relu(a):
    return T(np.maximum(a.v, 0.0), a.e)


def tanh(a):
    # the slope is at most 1; the evaluation is 1 - 2 / (e^2x + 1) with an exponential and a reciprocal of at most
    # 2 ulp each (4 U relative) and three more roundings, on quantities of at most 2: 2 (4 U + 4 U) + 4 U
    return T(np.tanh(a.v), a.e + 20 * U)


def split(flat, shapes):
    out, at = [], 0
    for s in shapes:
        n = int(np.prod(s))
        out.append(flat[at:at + n].reshape(s))
        at += n
    return out


def adapter_shapes(dims, rank):
    _, h1, h2, out = dims
    return [(h1, rank), (rank, h2), (h2, rank), (rank, out)]


def layers(params, bank, slots, scale, x, rank, dims):
    """h1, u2, h2, u3, logits of every row"""
    w1, b1, w2, b2, w3, b3 = [T(p) for p in params]
    h1 = relu(add(dot(T(x), w1, 1), b1))
    n, S = len(x), len(bank)

    def low(h, j):
        u = T(np.zeros((n, rank)))
        up = T(np.zeros((n, adapter_shapes(dims, rank)[j + 1][1])))
        u.e, up.e = u.e.copy(), up.e.copy()
        for s in range(S):
            rows = np.flatnonzero(slots == s)
            if not len(rows):
                continue
            f = split(bank[s], adapter_shapes(dims, rank))
            part = mul(dot(h[rows], T(f[j])), T(np.float64(np.float32(scale))))
            u.v[rows], u.e[rows] = part.v, part.e
            q = dot(part, T(f[j + 1]))
            up.v[rows], up.e[rows] = q.v, q.e
        return u, up

    u2, up2 = low(h1, 0)
    h2 = tanh(add(add(dot(h1, w2, rank + 1), up2), b2))
    u3, up3 = low(h2, 2)
    return h1, u2, h2, u3, add(add(dot(h2, w3, rank + 1), up3), b3)


def control(logits, c, classes):
    """(z, p): controlled logits and probabilities; c: None or a dict of host arrays (sets, set_of_row and any table)"""
    z, e = logits.v.copy(), logits.e.copy()
    for i in range(len(z)):
        k = -1 if c is None else int(c["set_of_row"][i]) if c.get("set_of_row") is not None else 0
        if c is None or k < 0 or k >= c["sets"]:
            continue
        if c.get("counts") is not None:
            n = c["counts"][k].astype(np.float64)
            rep = np.float64(c["repetition"][k]) if c.get("repetition") is not None else 1.0
            pre = np.float64(c["presence"][k]) if c.get("presence") is not None else 0.0
            freq = np.float64(c["frequency"][k]) if c.get("frequency") is not None else 0.0
            seen = n > 0
            grow = np.where(seen, max(rep, 1.0 / rep), 1.0)
            z[i] = np.where(seen, np.where(z[i] > 0, z[i] / rep, z[i] * rep) - pre, z[i]) - freq * n
            e[i] = e[i] * grow + 4 * U * (np.abs(z[i]) + np.abs(logits.v[i]) * grow + abs(pre) + 2 * abs(freq) * n)
        if c.get("bias") is not None:
            z[i] += c["bias"][k]
            e[i] = e[i] + U * np.abs(z[i])
        if c.get("allow") is not None:
            bit = (c["allow"][k][np.arange(classes) // 32] >> (np.arange(classes) % 32).astype(np.uint32)) & 1
            z[i][bit == 0] = -np.inf
            e[i][bit == 0] = 0.0
    top = z.max(axis=1, keepdims=True, initial=-np.inf)
    shift = np.where(np.isinf(top), 0.0, top)
    ex = np.exp(z - shift)
    total = ex.sum(axis=1, keepdims=True)
    p = np.where(total > 0, ex / np.where(total > 0, total, 1.0), 0.0)
    # relative: twice the largest error of an exponent (its own rounding of |z - max| U with it), the exponential's 2 ulp
    # in numerator and sum, the sum of `classes` terms and the division
    far = np.where(ex > 1e-45, np.abs(z - shift), 0.0)
    d = 2 * (np.where(np.isfinite(z), e, 0.0).max(axis=1, keepdims=True) + U * far.max(axis=1, keepdims=True))
    rel = np.expm1(d) + (classes + 12) * U
    return T(z, np.where(np.isfinite(z), e, 0.0)), T(p, p * rel + 1e-37)


def train(params, bank, slots, scale, x, labels, rank, dims, c=None):
    """grad [slots][param_count], loss and live rows of each slot"""
    _, n1, n2, out = dims
    h1, u2, h2, u3, logits = layers(params, bank, slots, scale, x, rank, dims)
    _, p = control(logits, c, out)
    S = len(bank)
    live = (x != 0).any(axis=1) & (slots >= 0) & (slots < S) & (labels >= 0) & (labels < out)
    row = np.arange(len(x))
    lab = np.where((labels >= 0) & (labels < out), labels, 0)
    if c is not None:
        z, _ = control(T(np.zeros((len(x), out))), c, out)
        live &= np.isfinite(z.v[row, lab])
    t = np.zeros((len(x), out))
    t[row, lab] = 1.0
    d3 = T(np.where(live[:, None], p.v - t, 0.0), np.where(live[:, None], p.e + U * np.abs(p.v - t), 0.0))
    loss = np.where(live, -np.log(np.maximum(p.v[row, lab], 1e-12)), 0.0)
    loss_e = np.where(live, p.e[row, lab] / np.maximum(p.v[row, lab] - p.e[row, lab], 1e-12) + 4 * U * np.abs(loss), 0.0)
    w3 = T(params[4])
    grads, stats, stats_e = [], [], []
    for s in range(S):
        rows = np.flatnonzero(slots == s)
        a2, b2, a3, b3 = [T(f) for f in split(bank[s], adapter_shapes(dims, rank))]
        sc = T(np.float64(np.float32(scale)))
        D3, H1, H2 = d3[rows], h1[rows], h2[rows]
        g3 = mul(dot(D3, b3.T), sc)
        one = T(1.0 - H2.v * H2.v, 2 * H2.mag * H2.e + 3 * U)
        d2 = mul(add(dot(D3, w3.T, rank), dot(g3, a3.T)), one)
        g2 = mul(dot(d2, b2.T), sc)
        parts = [dot(H1.T, g2, 4), dot(u2[rows].T, d2, 4), dot(H2.T, g3, 4), dot(u3[rows].T, D3, 4)]
        grads.append(T(np.concatenate([q.v.ravel() for q in parts]), np.concatenate([q.e.ravel() for q in parts])))
        stats.append([loss[rows].sum(), live[rows].sum()])
        stats_e.append([loss_e[rows].sum() + U * loss[rows].sum(), 0.0])
    return (T(np.stack([g.v for g in grads]), np.stack([g.e for g in grads])), T(np.array(stats), np.array(stats_e)))


def check(got, want, what=""):
    """Every value within its bound (non-finite ones equal)"""
    got = np.asarray(got, np.float64)
    assert got.shape == want.v.shape, (what, got.shape, want.v.shape)
    same = (got == want.v) | (np.isnan(got) & np.isnan(want.v))
    off = np.where(same, 0.0, np.abs(got - want.v))
    bad = ~(off <= want.e) & ~same
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(np.isnan(off), np.inf, off - want.e)), off.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} values out of bounds, worst at {i}: got {got[i]}, want {want.v[i]} +- {want.e[i]}")

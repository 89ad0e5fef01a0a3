"""The operators of linear-attention layers in 64 bits, for the tests: the causal convolution, the gated delta
rule token by token with a bound on what fp32 may be off, and choosing a token by its definition."""

import numpy as np
import torch

EPS = 2.0 ** -24            # a rounding to fp32 is off by at most this, relative to the value


def half_step(dtype, x):
    """What a rounding to dtype is off by at most: half a step, that of the smallest numbers below them."""
    return torch.finfo(dtype).eps / 2 * np.abs(x) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


class Sequences:
    """lens: (rows, tokens with them) of each sequence. slots are dealt out shuffled over n_slots."""

    def __init__(self, lens, spare=2, seed=0):
        self.lens, self.B = lens, len(lens)
        self.cu = np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.int32)
        self.kv = np.array([kv for _, kv in lens], np.int32)
        self.n_slots = self.B + spare
        self.slots = np.random.default_rng(seed).permutation(self.n_slots)[:self.B].astype(np.int32)
        self.T, self.max_q = int(self.cu[-1]), max([0] + [n for n, _ in lens])

    def dev(self, device):
        return [torch.from_numpy(x.copy()).to(device) for x in (self.cu, self.kv, self.slots)]

    def has_state(self, b):
        return 0 <= self.slots[b] < self.n_slots


def sigmoid(x):
    t = np.exp(-np.abs(x))
    return np.where(x >= 0, 1.0, t) / (1 + t)


def conv(x, w, bias, silu, before):
    """Rows [n][C] behind the inputs `before` [taps-1][C] -> rows and the sizes their sums go by."""
    taps = w.shape[1]
    u = np.concatenate([before, x])
    y = sum(u[j:j + len(x)] * w[:, j] for j in range(taps)) + (0 if bias is None else bias)
    size = sum(np.abs(u[j:j + len(x)] * w[:, j]) for j in range(taps)) + (0 if bias is None else np.abs(bias))
    return (y * sigmoid(y) if silu else y), size


def delta(q, k, v, a, b, a_log, dt_bias, S, scale, eps=1e-6, z=None, norm=None, norm_eps=1e-6, keep=None):
    """One sequence: q, k [n][Hk][Dk], v [n][Hv][Dv], a, b [n][Hv], S [Hv][Dk][Dv] -> rows, the state
    after `keep` rows (all), and bounds of both.

    The bounds: with keys of length 1 and beta in [0, 1] neither a fade nor a correction lengthens a
    column's error, so what a token adds stays, faded. A token adds at most 64 roundings of
    |v| + |column of S|: the sums over 128 products (19 in a row at most), the length of k (13), beta,
    the fade and its logarithm (8), the correction and its place in the state (24 left)."""
    n, Hk, Dk = q.shape
    Hv, Dv = v.shape[1:]
    q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + eps) for x in (q, k))
    q, k = (np.repeat(x, Hv // Hk, 1) for x in (q * scale, k))
    g = np.exp(-np.exp(a_log) * (np.maximum(a + dt_bias, 0) + np.log1p(np.exp(-np.abs(a + dt_bias)))))
    beta = sigmoid(b)
    S = S.copy()
    off = np.zeros((Hv, Dv))
    out, tol = np.zeros((n, Hv, Dv)), np.zeros((n, Hv, Dv))
    keep = n if keep is None else max(0, min(keep, n))
    kept = (S.copy(), off.copy())
    for t in range(n):
        before = np.sqrt((S * S).sum(1))
        S = S * g[t][:, None, None]
        d = beta[t][:, None] * (v[t] - (S * k[t][:, :, None]).sum(1))
        S = S + k[t][:, :, None] * d[:, None, :]
        length = before + np.abs(v[t]) + np.sqrt((S * S).sum(1))
        off = g[t][:, None] * off + 64 * EPS * length
        out[t] = (S * q[t][:, :, None]).sum(1)
        tol[t] = np.sqrt((q[t] ** 2).sum(-1))[:, None] * (off + 64 * EPS * length)
        if t + 1 == keep:
            kept = (S.copy(), off.copy())
    if z is not None:
        r = 1 / np.sqrt((out * out).mean(-1, keepdims=True) + norm_eps)
        gate = norm * z * sigmoid(z)
        tol = np.abs(gate) * r * (tol + np.abs(out) * r * np.sqrt((tol * tol).mean(-1, keepdims=True)))
        out = out * r * gate
        tol = tol + 16 * EPS * np.abs(out)
    return out, kept[0], tol, kept[1]


def choose(x, u, T=1.0, k=0, p=1.0, m=0.0):
    """A row's token by the definition, in 64 bits, its share, and how near u came to a border."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if not (x > -np.inf).any():
        return -1, 0.0, 1.0
    order = np.lexsort((np.arange(len(x)), -x))
    if not T > 0:
        return int(order[0]), 1.0, 1.0
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.where(np.isneginf(x) | np.isposinf(top), 0.0, np.exp((x - top) / T)))
    if k > 0:
        order = order[:k]
    total = w[order].sum()
    upto = np.cumsum(w[order])
    near = 1.0
    if p < 1:
        before = upto - w[order]
        n = max(1, int((before < p * total).sum()))
        near = min(near, np.abs(upto[:n + 1] / total - p).min())
        order = order[:n]
    if m > 0:
        order = order[w[order] >= min(m, 1.0)]
    ids = np.sort(order)
    share = np.cumsum(w[ids]) / w[ids].sum()
    at = min(int((share <= u).sum()), len(ids) - 1)
    while w[ids[at]] == 0:
        at -= 1
    near = min(near, np.abs(share - u).min() if u > 0 else 1.0)
    return int(ids[at]), w[ids[at]] / w[ids].sum(), near

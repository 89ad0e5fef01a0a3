"""Sequences over a paged key/value cache for the tests: page tables, the cache's element order
(restated from include/rlq.h with numpy), and attention in 64 bits."""

import numpy as np
import torch


def pack_keys(x):
    """[..., positions, D] -> the cache's order, same shape."""
    *lead, P, D = x.shape
    x = x.reshape(*lead, P // 32, 32, D // 16, 2, 8)
    n = len(lead)
    return x.transpose(*range(n), n, n + 2, n + 3, n + 1, n + 4).reshape(*lead, P, D)


def unpack_keys(x):
    *lead, P, D = x.shape
    x = x.reshape(*lead, P // 32, D // 16, 2, 32, 8)
    n = len(lead)
    return x.transpose(*range(n), n, n + 3, n + 1, n + 2, n + 4).reshape(*lead, P, D)


def pack_values(x):
    *lead, P, D = x.shape
    x = x.reshape(*lead, P // 32, 2, 2, 2, 4, D // 32, 32)          # block, t, a, h, b, u, d
    n = len(lead)
    return x.transpose(*range(n), n, n + 5, n + 1, n + 3, n + 6, n + 2, n + 4).reshape(*lead, P, D)


def unpack_values(x):
    *lead, P, D = x.shape
    x = x.reshape(*lead, P // 32, D // 32, 2, 2, 32, 2, 4)          # block, u, t, h, d, a, b
    n = len(lead)
    return x.transpose(*range(n), n, n + 2, n + 5, n + 3, n + 6, n + 1, n + 4).reshape(*lead, P, D)


class Sequences:
    """lens: (new tokens, tokens with them) per sequence; pages are dealt out shuffled."""

    def __init__(self, lens, page, seed=0, spare=1):
        rng = np.random.default_rng(seed)
        self.lens, self.page = lens, page
        need = [-(-kv // page) for _, kv in lens]
        self.n_pages = max(1, sum(need)) + spare
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), max([1] + need)), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.cu = np.concatenate([[0], np.cumsum([q for q, _ in lens])]).astype(np.int32)
        self.kv = np.array([kv for _, kv in lens], np.int32)
        self.T = int(self.cu[-1])
        self.max_q, self.max_kv = max(q for q, _ in lens), max(kv for _, kv in lens)

    def dev(self, device):
        return [torch.from_numpy(x.copy()).to(device) for x in (self.cu, self.kv, self.table)]


def attend(q, keys, values, kv, scale, window=0, cap=0.0, hidden=()):
    """Rows q [n][H][D], the last of a sequence of `kv` tokens, over keys and values [kv][KV][D], in
    64 bits. Returns the rows and, for tolerances, sum_j w_j |v_j| of each. hidden: positions no row
    sees."""
    n, H, D = q.shape
    G = H // keys.shape[1]
    out, size = np.zeros((n, H, D)), np.zeros((n, H, D))
    for i in range(n):
        pos = kv - n + i
        at = np.arange(kv)
        seen = at <= pos
        if window:
            seen &= at > pos - window
        seen[list(hidden)] = False
        if not seen.any():
            continue
        k, v = keys[seen].astype(np.float64), values[seen].astype(np.float64)
        for h in range(H):
            s = k[:, h // G] @ q[i, h].astype(np.float64) * scale
            if cap:
                s = cap * np.tanh(s / cap)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h], size[i, h] = w @ v[:, h // G], w @ np.abs(v[:, h // G])
    return out, size


HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}      # half a step among fp16's smallest numbers


def attention_tolerance(ref, size, q, keys, kv, scale, cap, dtype, out_dtype):
    """Per element. Rounding of the row: half a step. A weight: half a step of the cache's type (two
    terms of bf16 where fp16 rows leave: 2^-16), and what its score is off: the product of D terms in
    fp32, each addition half a step (2^-24) of at most sum |q_i k_i| scale, four more operations, a cap's
    tanh 2^-21 cap; exp2 2^-22. The sums over the keys: half a step of their size an addition."""
    D = q.shape[-1]
    qk = float(np.abs(q).max(initial=0)) * float(np.abs(keys).astype(np.float64).sum(-1).max(initial=0)) * scale
    weight = 2.0 ** -16 if dtype == torch.bfloat16 and out_dtype == torch.float16 else HALF_STEP[dtype]
    off = (D + 4) * 2.0 ** -24 * qk + 2.0 ** -21 * cap + 2.0 ** -22
    return HALF_STEP[out_dtype] * np.abs(ref) + (weight + 2 * off + 2 * kv * 2.0 ** -24) * size + TINY[out_dtype]

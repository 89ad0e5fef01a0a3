"""The recurrent layers of a decoding step, and the choice of a token, as cases.

Three operators of raceline_amd.ops, each next to what the library already runs:

  causal_conv  the stacked in projection's rows -> the short causal convolution of every channel with
               its SiLU, and the sequences' last inputs
  gated_delta  the convolved rows -> the gated delta rule over a state per sequence and value head
               (single tokens, drafts, prompts), its rows normalised and gated for the out projection
  sample       rows of adjusted logits and a random number each -> tokens, by temperature, top-k, top-p
               and min-p

Heads of the linear layers are those of raceline_amd.synth's model configuration (16 key and 32 value
heads of 128, 4 taps) and generic ones; the vocabulary has 248,320 rows.

`own` chooses who computes: the plain form below (elementary torch operations in 32 bits, in 64 for
sums of logarithms and for the weights of tokens), or the library's kernels.
"""

from __future__ import annotations

import math
import random

import torch

own = False

VOCAB = 248320
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HEADS = {"9b": (16, 32, 128, 128), "shared": (4, 12, 128, 64), "h64": (8, 8, 64, 64), "wide": (2, 8, 64, 128)}


def listed():
    return [
        # one token of a 9B layer: launches and latency
        dict(name="conv_9b_token", op="conv", heads="9b", B=1, q=1, ragged=False, fresh=False, taps=4, dtype="f16",
             bias=False),
        # 24 sequences verifying a draft of four beside their last token
        dict(name="conv_drafts", op="conv", heads="9b", B=24, q=5, ragged=False, fresh=False, taps=4, dtype="bf16",
             bias=False),
        # a prompt's chunk of a 9B layer: the stream of rows
        dict(name="conv_9b_chunk", op="conv", heads="9b", B=1, q=2048, ragged=False, fresh=False, taps=4, dtype="f16",
             bias=False),
        # one token of one sequence
        dict(name="delta_9b_token", op="delta", heads="9b", B=1, q=1, ragged=False, fresh=False, dtype="f16", gate=True),
        # nine sequences verifying drafts, bf16 rows
        dict(name="delta_drafts", op="delta", heads="shared", B=9, q=5, ragged=False, fresh=False, dtype="bf16",
             gate=True),
        # 48 users decoding together: the stream of states
        dict(name="delta_9b_users", op="delta", heads="9b", B=48, q=1, ragged=False, fresh=False, dtype="f16", gate=True),
        # a chunk of a 9B layer's prompt, on the state that the chunks before it left
        dict(name="delta_9b_chunk", op="delta", heads="9b", B=1, q=2048, ragged=False, fresh=False, dtype="f16",
             gate=True),
        # six whole prompts of different lengths in small heads, rows not gated
        dict(name="delta_prompts", op="delta", heads="h64", B=6, q=1537, ragged=True, fresh=True, dtype="bf16",
             gate=False),
        # a long prompt in one call: the most arithmetic, and the longest chain
        dict(name="delta_9b_long", op="delta", heads="9b", B=1, q=8192, ragged=False, fresh=True, dtype="bf16", gate=True),
        # one sequence's next token, the usual filters
        dict(name="sample_one", op="sample", rows=1, vocab=VOCAB, k=40, p=0.95, m=0.0, t=0.7),
        # sixteen sequences by the nucleus alone: its border is looked for among all tokens
        dict(name="sample_nucleus", op="sample", rows=16, vocab=VOCAB, k=0, p=0.9, m=0.0, t=1.0),
        # every row of a draft batch, hot, cut by min-p
        dict(name="sample_min_p", op="sample", rows=45, vocab=VOCAB, k=0, p=1.0, m=0.02, t=1.5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["conv", "delta", "delta", "delta", "sample"])
    if op == "sample":
        return dict(op=op, rows=_log_int(rng, 1, 40), vocab=VOCAB - rng.randint(0, 240000), k=rng.choice([0, 0, 1, 20, 500]),
                    p=rng.choice([1.0, 0.5, 0.8, 0.99]), m=rng.choice([0.0, 0.0, 0.05, 0.3]),
                    t=round(rng.uniform(0.2, 2.0), 3))
    heads, dtype = rng.choice(sorted(HEADS)), rng.choice(["f16", "bf16"])
    form = rng.choice(["token", "draft", "chunk", "prompts"])
    if form in ("token", "draft"):
        B, q = _log_int(rng, 1, 40), 1 if form == "token" else rng.randint(2, 8)
    elif form == "chunk":
        B, q = rng.randint(1, 2), _log_int(rng, 9, 1000)
    else:
        B, q = rng.randint(2, 7), _log_int(rng, 17, 400)
    case = dict(op=op, heads=heads, B=B, q=q, ragged=rng.random() < 0.7, fresh=rng.random() < 0.4, dtype=dtype)
    if op == "conv":
        return dict(case, taps=rng.choice([2, 3, 4, 4]), bias=rng.random() < 0.3)
    return dict(case, gate=rng.random() < 0.7)


# ------------------------------------------------------------------ what a case holds

def _lengths(case):
    """New tokens of each sequence: the case's own, or spread below them."""
    B, q = case["B"], case["q"]
    if not case["ragged"]:
        return [q] * B
    r = random.Random("%d %d" % (B, q))
    return [q] + [r.randint(1, q) for _ in range(B - 1)]


def _gen(seed, stream):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 64 + stream)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _sequences(case):
    """Row starts, lengths with the tokens before the call (none for some where the case says so) and
    states, shuffled, two more than the sequences use."""
    n = _lengths(case)
    order = list(range(case["B"] + 2))
    random.Random(len(n)).shuffle(order)
    cu = [0]
    for a in n:
        cu.append(cu[-1] + a)
    kv = [a + (0 if case["fresh"] and i % 2 == 0 else 100) for i, a in enumerate(n)]
    ints = dict(dtype=torch.int32, device="cuda")
    return dict(case=case, cu=torch.tensor(cu, **ints), kv=torch.tensor(kv, **ints), T=cu[-1], max_q=max(n),
                slots=torch.tensor(order[:case["B"]], **ints), states=case["B"] + 2)


def prepare(case, seed):
    return _PREPARE[case["op"]](case, seed)


def _prepare_conv(case, seed):
    Hk, Hv, Dk, Dv = HEADS[case["heads"]]
    C, K, g, s = 2 * Hk * Dk + Hv * Dv, case["taps"], _gen(seed, 1), _sequences(case)
    # the rows that the stacked in projection gives: the convolution's channels, then the gate z
    s["rows"] = _normal(g, s["T"], C + Hv * Dv) * 1.5
    s["C"], s["w"] = C, _normal(g, C, K) / math.sqrt(K)
    s["bias"] = _normal(g, C) * 0.2 if case["bias"] else None
    s["state"] = _normal(g, s["states"], K - 1, C) * 1.5
    return s


def _prepare_delta(case, seed):
    Hk, Hv, Dk, Dv = HEADS[case["heads"]]
    g, s = _gen(seed, 2), _sequences(case)
    T, C = s["T"], 2 * Hk * Dk + Hv * Dv
    # what the convolution and its SiLU give; keys of a head have much in common
    x = _normal(g, T, C) + 0.7 * _normal(g, C)
    s["x"] = (x * torch.sigmoid(x)).to(DTYPES[case["dtype"]])
    s["ba"] = _normal(g, T, 2 * Hv)
    # decays from nearly none to a few tokens: rates of 1 to 16, steps of 0.001 to 0.1
    s["a_log"] = torch.log(1 + 15 * torch.rand(Hv, generator=g, device="cuda"))
    step = torch.exp(torch.rand(Hv, generator=g, device="cuda") * math.log(100.0)) * 0.001
    s["dt"] = torch.log(torch.expm1(step))
    s["state"] = _normal(g, s["states"], Hv, Dk, Dv) * 0.2
    if case["gate"]:
        s["z"] = _normal(g, T, Hv * Dv) * 1.5
        s["norm"] = 1 + 0.2 * _normal(g, Dv)
    return s


def _prepare_sample(case, seed):
    g, rows, V = _gen(seed, 3), case["rows"], case["vocab"]
    # a few tokens stand out of the rest
    lift = torch.rand((rows, V), generator=g, device="cuda").pow(2000) * 14
    s = dict(case=case, logits=_normal(g, rows, V) * 2 + lift)
    s["u"] = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
    spread = torch.rand((4, rows), generator=g, device="cuda")
    s["t"] = case["t"] * (0.8 + 0.4 * spread[0])
    s["k"] = (case["k"] * (0.5 + spread[1])).ceil().to(torch.int32)          # 0: all
    s["p"] = 1 - (1 - case["p"]) * (0.5 + spread[2])
    s["m"] = case["m"] * (0.5 + spread[3])
    s["probs"] = torch.empty(rows, device="cuda")
    return s


_PREPARE = {"conv": _prepare_conv, "delta": _prepare_delta, "sample": _prepare_sample}


def _split(s, x):
    """q, k and v of the convolved rows."""
    Hk, Hv, Dk, Dv = HEADS[s["case"]["heads"]]
    return x[:, :Hk * Dk], x[:, Hk * Dk:2 * Hk * Dk], x[:, 2 * Hk * Dk:]


# ------------------------------------------------------------------ the framework's calls

def run(s):
    op = s["case"]["op"]
    if own:
        return _OWN[op](s)
    return _PLAIN[op](s)


def _own_conv(s):
    from raceline_amd import ops

    y = ops.causal_conv(s["rows"][:, :s["C"]], s["w"], s["state"], s["cu"], s["kv"], s["slots"], bias=s["bias"],
                        out_dtype=DTYPES[s["case"]["dtype"]])
    return y, s["state"]


def _own_delta(s):
    from raceline_amd import ops

    Hv = s["a_log"].numel()
    q, k, v = _split(s, s["x"])
    o = ops.gated_delta(q, k, v, s["ba"][:, Hv:], s["ba"][:, :Hv], s["a_log"], s["dt"], s["state"], s["cu"], s["kv"],
                        s["slots"], max_q=s["max_q"], z=s.get("z"), norm=s.get("norm"),
                        out_dtype=DTYPES[s["case"]["dtype"]])
    return o, s["state"]


def _own_sample(s):
    from raceline_amd import ops

    tokens = ops.sample(s["logits"], s["u"], temperature=s["t"], top_k=s["k"], top_p=s["p"], min_p=s["m"],
                        probs=s["probs"])
    return tokens, s["probs"]


_OWN = {"conv": _own_conv, "delta": _own_delta, "sample": _own_sample}


# ------------------------------------------------------------------ the plain forms

def _silu(x):
    return x / (1 + torch.exp(-x))


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _inputs_at(s, row0, at, slot, fresh):
    """Input rows `at` tokens behind the sequences' first rows, from the state where that is negative."""
    x, state = s["rows"][:, :s["C"]], s["state"]
    old = state[slot, (at + state.shape[1]).clamp(0, state.shape[1] - 1)]
    old = torch.where(fresh[..., None], 0.0, old)
    return torch.where((at >= 0)[..., None], x[row0 + at.clamp(min=0)], old)


def _plain_conv(s):
    K, cu, slots = s["case"]["taps"], s["cu"].long(), s["slots"].long()
    row = torch.arange(s["T"], device="cuda")
    seq = torch.searchsorted(cu, row, right=True) - 1
    n = cu[1:] - cu[:-1]
    fresh = s["kv"] <= n
    y = sum(_inputs_at(s, cu[seq], row - cu[seq] - (K - 1 - j), slots[seq], fresh[seq]) * s["w"][:, j] for j in range(K))
    if s["bias"] is not None:
        y = y + s["bias"]
    y = _silu(y).to(DTYPES[s["case"]["dtype"]])
    back = torch.arange(-(K - 1), 0, device="cuda")
    s["state"][slots] = _inputs_at(s, cu[:-1, None], n[:, None] + back, slots[:, None], fresh[:, None])
    return y, s["state"]


def _inverse(L):
    """(I + L)^-1 of strictly lower triangular L, whose size is a power of two: the inverses of the blocks
    on the diagonal, joined in pairs."""
    n = L.shape[-1]
    T = torch.eye(n, device="cuda").expand(L.shape).contiguous()
    for k in range(n.bit_length() - 1):
        w = 1 << k
        at = torch.arange(n, device="cuda")
        pair, low = at // (2 * w), at // w % 2
        part = (pair[:, None] == pair) & (low[:, None] > low)
        T = T - torch.matmul(torch.matmul(T, torch.where(part, L, 0.0)), T)
    return T


def _plain_delta(s):
    # the rule's chunked form: within a chunk the tokens' corrections solve a triangular system, all chunks
    # at once; the state goes through the chunks one after the other, which is the loop at the end
    c, (Hk, Hv, Dk, Dv) = s["case"], HEADS[s["case"]["heads"]]
    B, cu, slots, G = c["B"], s["cu"].long(), s["slots"].long(), Hv // Hk
    C = min(64, 1 << (s["max_q"] - 1).bit_length())
    N = -(-s["max_q"] // C)
    i = torch.arange(N * C, device="cuda")
    here = i < (cu[1:] - cu[:-1])[:, None]
    row = (cu[:-1, None] + i).clamp(max=s["T"] - 1)

    def heads(x, H):                                              # [T][H * D] -> [B][H][N][C][D], zeros behind the rows
        x = torch.where(here[..., None], x[row].float(), 0.0)
        return x.view(B, N, C, H, -1).permute(0, 3, 1, 2, 4)

    q, k, v = _split(s, s["x"])
    q, k = (x * torch.rsqrt(x.square().sum(-1, keepdim=True) + 1e-6) for x in (heads(q, Hk), heads(k, Hk)))
    q, k = (x.repeat_interleave(G, 1) for x in (q / math.sqrt(Dk), k))
    v = heads(v, Hv)
    beta = heads(1 / (1 + torch.exp(-s["ba"][:, :Hv])), Hv)
    rate = heads(-torch.exp(s["a_log"]) * _softplus(s["ba"][:, Hv:] + s["dt"]), Hv)[..., 0]
    total = torch.cumsum(rate.double(), -1)
    lower = torch.ones((C, C), dtype=torch.bool, device="cuda").tril()
    fade = torch.exp(torch.where(lower, total[..., :, None] - total[..., None, :], -math.inf)).float()
    grow, left = torch.exp(total).float()[..., None], torch.exp(total[..., -1:] - total).float()[..., None]
    kt = k.transpose(-1, -2).contiguous()
    T = _inverse(torch.where(lower.tril(-1), beta * fade * torch.matmul(k, kt), 0.0))
    U, W = torch.matmul(T, beta * v), torch.matmul(T, beta * grow * k)
    A, q, kt = fade * torch.matmul(q, kt), q * grow, (k * left).transpose(-1, -2).contiguous()
    S = torch.where((s["kv"] <= cu[1:] - cu[:-1])[:, None, None, None], 0.0, s["state"][slots])
    out = torch.empty_like(U)
    for n in range(N):
        u = U[:, :, n] - torch.matmul(W[:, :, n], S)
        out[:, :, n] = torch.matmul(q[:, :, n], S) + torch.matmul(A[:, :, n], u)
        S = grow[:, :, n, -1:] * S + torch.matmul(kt[:, :, n], u)
    s["state"][slots] = S
    o = out.permute(0, 2, 3, 1, 4).reshape(B, N * C, Hv, Dv)[here]
    if c["gate"]:
        o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + 1e-6) * s["norm"] * _silu(s["z"].view(-1, Hv, Dv))
    return o.reshape(-1, Hv * Dv).to(DTYPES[c["dtype"]]), s["state"]


def _plain_sample(s):
    x = s["logits"].double()
    V = x.shape[1]
    top, order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp((top - top[:, :1]) / s["t"].double()[:, None])
    k = torch.where(s["k"] > 0, s["k"], V)[:, None]
    w = torch.where(torch.arange(V, device="cuda") < k, w, 0.0)
    upto = torch.cumsum(w, -1)
    kept = (upto - w < s["p"].double()[:, None] * upto[:, -1:]) & (w >= s["m"].double()[:, None])
    w = torch.zeros_like(w).scatter_(1, order, torch.where(kept, w, 0.0))
    upto = torch.cumsum(w, -1)
    total = upto[:, -1:]
    token = (upto <= s["u"][:, None] * total).sum(-1)
    s["probs"].copy_((w.gather(1, token[:, None]) / total)[:, 0])
    return token.to(torch.int32), s["probs"]


_PLAIN = {"conv": _plain_conv, "delta": _plain_delta, "sample": _plain_sample}


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 32 * case["rows"], "flops": 10 * n}
    Hk, Hv, Dk, Dv = HEADS[case["heads"]]
    T, C = sum(_lengths(case)), 2 * Hk * Dk + Hv * Dv
    old = sum(1 for i in range(case["B"]) if not (case["fresh"] and i % 2 == 0))     # states that are read
    if case["op"] == "conv":
        K = case["taps"]
        return {"bytes": 6 * T * C + 4 * (K - 1) * C * (case["B"] + old) + 4 * K * C, "flops": (2 * K + 4) * T * C}
    gate = 4 * Hv * Dv if case["gate"] else 0
    return {"bytes": T * (2 * C + 8 * Hv + 2 * Hv * Dv + gate) + 4 * Hv * Dk * Dv * (case["B"] + old),
            "flops": 7 * T * Hv * Dk * Dv}


# ------------------------------------------------------------------ the same in 64 bits, apart from the above

def exact(case, seed):
    return _EXACT[case["op"]](case, prepare(case, seed))


def _exact_conv(case, s):
    K, C, state, out, at = case["taps"], s["C"], s["state"].double(), [], 0
    for b, n in enumerate(_lengths(case)):
        slot = int(s["slots"][b])
        before = torch.zeros_like(state[slot]) if int(s["kv"][b]) <= n else state[slot]
        x = torch.cat([before, s["rows"][at:at + n, :C].double()])
        y = torch.stack([x[j:j + n] for j in range(K)], -1).mul(s["w"].double()).sum(-1)
        y = y if s["bias"] is None else y + s["bias"].double()
        out.append(y * torch.sigmoid(y))
        state[slot] = x[n:]
        at += n
    return torch.cat(out), state


def _exact_delta(case, s):
    Hk, Hv, Dk, Dv = HEADS[case["heads"]]
    T, state = s["T"], s["state"].double()
    q, k, v = (x.double() for x in _split(s, s["x"]))
    q, k = (x.reshape(T, Hk, 1, Dk) for x in (q, k))
    q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6) for x in (q, k))
    q, k = (x.expand(T, Hk, Hv // Hk, Dk).reshape(T, Hv, Dk, 1) for x in (q * Dk ** -0.5, k))
    v = v.reshape(T, Hv, 1, Dv)
    b, a = s["ba"].double()[:, :Hv], s["ba"].double()[:, Hv:]
    beta = torch.sigmoid(b).view(T, Hv, 1, 1)
    gamma = torch.exp(-s["a_log"].double().exp() * torch.nn.functional.softplus(a + s["dt"].double(), threshold=700))
    gamma = gamma.view(T, Hv, 1, 1)
    o = torch.empty((T, Hv, Dv), dtype=torch.float64, device="cuda")
    at = 0
    for i, n in enumerate(_lengths(case)):
        slot = int(s["slots"][i])
        S = torch.zeros_like(state[slot]) if int(s["kv"][i]) <= n else state[slot].clone()
        for t in range(at, at + n):                               # the rule as it is defined, token by token
            S = S * gamma[t]
            S = S + k[t] * (beta[t] * (v[t] - (S * k[t]).sum(1, keepdim=True)))
            o[t] = (S * q[t]).sum(1)
        state[slot] = S
        at += n
    if case["gate"]:
        z = s["z"].double().view(T, Hv, Dv)
        o = o / torch.sqrt((o * o).sum(-1, keepdim=True) / Dv + 1e-6) * s["norm"].double() * z * torch.sigmoid(z)
    return o.reshape(T, Hv * Dv), state


def _exact_sample(case, s):
    tokens, probs = [], []
    for r in range(case["rows"]):
        x = s["logits"][r].double() / s["t"][r].double()
        p = torch.softmax(x, -1)
        ids = torch.argsort(s["logits"][r], descending=True, stable=True)
        if int(s["k"][r]):
            ids = ids[:int(s["k"][r])]
        share = p[ids] / p[ids].sum()
        ids = ids[(torch.cumsum(share, 0) - share < s["p"][r].double()) & (p[ids] >= s["m"][r].double() * p.max())]
        ids = torch.sort(ids).values
        share = p[ids] / p[ids].sum()
        at = int((torch.cumsum(share, 0) <= s["u"][r]).sum().clamp(max=len(ids) - 1))
        tokens.append(ids[at])
        probs.append(share[at])
    return torch.stack(tokens).to(torch.int32), torch.stack(probs)


_EXACT = {"conv": _exact_conv, "delta": _exact_delta, "sample": _exact_sample}

"""The attention half of a decoding step, and the logits before a token is chosen, as cases.

Three operators of raceline_amd.ops, each next to what the library already runs:

  rope_append    the stacked qkv linear's rows -> rotated queries, and keys and values in a
                 paged cache (optionally with the per-head RMS norm of q and k)
  attention      a chunk of new tokens (one, a draft's few, a prompt's many) of each sequence
                 over its pages; the rows go into the o linear
  adjust_logits  penalties for repeated tokens, biases and a grammar's mask on the head's
                 logits, before the top-k

Head counts and sizes are those of the 9B and 27B layers of raceline_amd.configs (16 or 20 query
heads and 4 key/value heads of 256 with 64 rotary dimensions, as raceline_amd.synth writes
them) and generic ones (heads of 64 and 128); the vocabulary has 248,320 rows.

`own` chooses who computes: the plain form below (elementary torch operations in 32 bits, in 64
for the angles), or the library's kernels.
"""

from __future__ import annotations

import math
import random

import torch

own = False

VOCAB = 248320
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HEADS = {"9b": (16, 4, 256), "27b": (20, 4, 256), "h128": (32, 8, 128), "h64": (12, 12, 64)}


def listed():
    return [
        # one token and its four drafts of a 9B model, with the norms of q and k: launches and latency
        dict(name="rope_9b_draft", op="rope", heads="9b", B=1, q=5, ctx=4000, ragged=False, page=64, dtype="f16",
             rot=64, layout="half", scaling="plain", norm=True),
        # a 27B model's prompt chunk, the third of its prompt
        dict(name="rope_27b_chunk", op="rope", heads="27b", B=1, q=2048, ctx=4096, ragged=False, page=256, dtype="f16",
             rot=64, layout="half", scaling="plain", norm=False),
        # 37 sequences with chunks of all lengths far into a stretched context, whole head rotated
        dict(name="rope_ragged_far", op="rope", heads="h128", B=37, q=300, ctx=120000, ragged=True, page=64,
             dtype="bf16", rot=128, layout="interleaved", scaling="parts", norm=False),
        # one token of one sequence: the smallest call
        dict(name="attn_9b_token", op="attn", heads="9b", B=1, q=1, kv=1900, ragged=False, page=64, dtype="f16",
             out="f16", window=0, cap=0.0),
        # 32 users decoding together, contexts of all lengths: the largest stream of bytes
        dict(name="attn_27b_users", op="attn", heads="27b", B=32, q=1, kv=16384, ragged=True, page=256, dtype="f16",
             out="f16", window=0, cap=0.0),
        # nine sequences verifying drafts inside a sliding window, cache in bf16
        dict(name="attn_draft_window", op="attn", heads="h128", B=9, q=5, kv=6001, ragged=True, page=64, dtype="bf16",
             out="f16", window=4096, cap=0.0),
        # the last chunk of an 8192-token prompt: the most arithmetic
        dict(name="attn_27b_chunk", op="attn", heads="27b", B=1, q=2048, kv=8192, ragged=False, page=256, dtype="f16",
             out="f16", window=0, cap=0.0),
        # six whole prompts of different lengths in one call, capped scores
        dict(name="attn_prompts_cap", op="attn", heads="h128", B=6, q=1537, kv=1537, ragged=True, page=64,
             dtype="bf16", out="bf16", window=0, cap=30.0),
        # small heads without sharing, a short chunk at the end of a long context
        dict(name="attn_small_heads", op="attn", heads="h64", B=1, q=333, kv=20011, ragged=False, page=64,
             dtype="f16", out="f16", window=0, cap=0.0),
        # one sequence's logits after a short conversation
        dict(name="logits_one", op="logits", rows=1, vocab=VOCAB, tokens=901, prompt=0.8, biases=0, mask=False),
        # sixteen sequences with long histories, biases and a grammar: the largest call of the head
        dict(name="logits_sixteen", op="logits", rows=16, vocab=VOCAB, tokens=8000, prompt=0.7, biases=200, mask=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "attn", "attn", "attn", "logits"])
    dtype = rng.choice(["f16", "bf16"])
    heads = rng.choice(sorted(HEADS))
    page = rng.choice([32, 64, 96, 256])
    if op == "rope":
        D = HEADS[heads][2]
        return dict(op=op, heads=heads, B=_log_int(rng, 1, 40), q=_log_int(rng, 1, 400), ctx=_log_int(rng, 1, 130000),
                    ragged=rng.random() < 0.7, page=page, dtype=dtype, rot=rng.choice([D, D // 2, D // 4, 20]),
                    layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["plain", "linear", "parts"]),
                    norm=rng.random() < 0.5)
    if op == "logits":
        return dict(op=op, rows=rng.randint(1, 16), vocab=VOCAB - rng.randint(0, 216000), tokens=_log_int(rng, 1, 8000),
                    prompt=rng.choice([0.0, 0.5, 0.9]), biases=rng.choice([0, 3, 300]), mask=rng.random() < 0.5)
    form = rng.choice(["token", "draft", "chunk", "prompt"])
    kv = _log_int(rng, 17, 16000)
    if form in ("token", "draft"):
        B, q = _log_int(rng, 1, 24), 1 if form == "token" else rng.randint(2, 8)
    elif form == "chunk":
        B, q = rng.randint(1, 2), _log_int(rng, 9, 800)
    else:
        kv = _log_int(rng, 17, 1500)
        B, q = rng.randint(1, 6), kv
    return dict(op=op, heads=heads, B=B, q=min(q, kv), kv=kv, ragged=rng.random() < 0.7, page=page, dtype=dtype,
                out=rng.choice([dtype, "f16"]), window=rng.choice([0, 0, 1 + kv // 3]), cap=rng.choice([0.0, 0.0, 30.0]))


# ------------------------------------------------------------------ what a case holds

def _lengths(case):
    """(new tokens, tokens in the cache with them) of each sequence: the case's own, or spread
    below them."""
    B, q, kv = case["B"], case["q"], case.get("kv", case["q"] + case.get("ctx", 0))
    if not case["ragged"]:
        return [q] * B, [kv] * B
    r = random.Random("%d %d %d" % (B, q, kv))
    qs, kvs = [], []
    for b in range(B):
        n = q if b == 0 or q <= 8 else r.randint(1, q)
        base = kv - q if "ctx" in case else r.randint(0, kv - q) if kv - q > 8 else kv - q
        qs.append(n)
        kvs.append(kv if b == 0 else base + n)
    return qs, kvs


def _gen(seed, stream):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 64 + stream)
    return g


def _sequences(case):
    """Row starts, lengths and a page table with shuffled pages. A rope case's table holds only
    the pages that the call writes (-1: pages not there, as behind a sliding window)."""
    qs, kvs = _lengths(case)
    page = case["page"]
    width = -(-max(kvs) // page)
    rows, n = [], 0
    for a, b in zip(qs, kvs):
        first = (b - a) // page if case["op"] == "rope" else 0
        last = -(-b // page)
        rows.append([-1] * first + list(range(n, n + last - first)) + [-1] * (width - last))
        n += last - first
    order = list(range(n + 1))                       # one page more than the sequences use
    random.Random(n).shuffle(order)
    rows = [[order[p] if p >= 0 else -1 for p in r] for r in rows]
    cu = [0]
    for a in qs:
        cu.append(cu[-1] + a)
    ints = dict(dtype=torch.int32, device="cuda")
    return dict(cu=torch.tensor(cu, **ints), kv=torch.tensor(kvs, **ints), table=torch.tensor(rows, **ints),
                pages=n + 1, T=cu[-1], max_q=max(qs), max_kv=max(kvs))


def _frequencies(case):
    """Radians per token of each rotated pair, 64 bits."""
    rot, base = case["rot"], 1e6
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if case["scaling"] == "linear":
        f = f / 4
    if case["scaling"] == "parts":                   # by turns over the original context: stretch slow pairs only
        turns = 32768 * f / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        f = (1 - keep) * f / 4 + keep * f
    return f.cuda()


def prepare(case, seed):
    if case["op"] == "logits":
        return _prepare_logits(case, seed)
    H, KV, D = HEADS[case["heads"]]
    s = _sequences(case)
    s.update(case=case, H=H, KV=KV, D=D)
    g, dt = _gen(seed, 1), DTYPES[case["dtype"]]
    shape = (s["pages"], KV, case["page"], D)
    s["k"] = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt)
    s["v"] = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt)
    if case["op"] == "rope":
        s["qkv"] = torch.randn((s["T"], (H + 2 * KV) * D), generator=g, device="cuda") * 1.5
        s["freq"] = _frequencies(case)
        s["m"] = 0.1 * math.log(4) + 1 if case["scaling"] == "parts" else 1.0
        if case["norm"]:
            s["qn"] = 1 + 0.2 * torch.randn(D, generator=g, device="cuda")
            s["kn"] = 1 + 0.2 * torch.randn(D, generator=g, device="cuda")
    else:
        # scores with a standard deviation of 1.5: some keys stand out
        s["q"] = (torch.randn((s["T"], H * D), generator=g, device="cuda") * 1.5).to(dt)
        s["scale"] = 1 / math.sqrt(D)
    return s


def _prepare_logits(case, seed):
    g = _gen(seed, 2)
    rows, V, n = case["rows"], case["vocab"], case["tokens"]
    s = dict(case=case, logits=torch.randn((rows, V), generator=g, device="cuda") * 3)
    # words repeat: ids fall off like a text's
    u = torch.rand((rows, n), generator=g, device="cuda")
    s["tokens"] = (u.pow(6) * V).to(torch.int32).clamp_(0, V - 1)
    s["n"] = (n - torch.arange(rows, device="cuda") * (n // 40)).to(torch.int32)
    s["prompt"] = (s["n"] * case["prompt"]).to(torch.int32)
    s["rep"] = 1 + 0.3 * torch.rand(rows, generator=g, device="cuda")
    s["pres"] = torch.rand(rows, generator=g, device="cuda")
    s["freq"] = torch.rand(rows, generator=g, device="cuda") * 0.5
    if case["biases"]:
        s["ids"] = (torch.rand((rows, case["biases"]), generator=g, device="cuda").pow(3) * V).to(torch.int32).clamp_(0, V - 1)
        s["bias"] = torch.randn((rows, case["biases"]), generator=g, device="cuda") * 4
    if case["mask"]:                                 # bit v % 32 of word v / 32: token v is allowed
        s["allowed"] = torch.randint(-2**31, 2**31, (rows, -(-V // 32)), generator=g, device="cuda").to(torch.int32)
    return s


# ------------------------------------------------------------------ the framework's calls

def run(s):
    op = s["case"]["op"]
    if own:
        return _OWN[op](s)
    return _PLAIN[op](s)


def _own_rope(s):
    from raceline_amd import ops

    c, H, KV, D = s["case"], s["H"], s["KV"], s["D"]
    qkv = s["qkv"]
    q = ops.rope_append(qkv[:, :H * D], qkv[:, H * D:(H + KV) * D], qkv[:, (H + KV) * D:], s["k"], s["v"], s["cu"],
                        s["kv"], s["table"], s["freq"], interleaved=c["layout"] == "interleaved", mscale=s["m"],
                        q_norm=s.get("qn"), k_norm=s.get("kn"), eps=1e-6)
    return q, s["k"], s["v"]


def _own_attn(s):
    from raceline_amd import ops

    c = s["case"]
    return ops.attention(s["q"], s["k"], s["v"], s["cu"], s["kv"], s["table"], max_q=s["max_q"], max_kv=s["max_kv"],
                         scale=s["scale"], window=c["window"], softcap=c["cap"], out_dtype=DTYPES[c["out"]])


def _own_logits(s):
    from raceline_amd import ops

    return ops.adjust_logits(s["logits"], tokens=s["tokens"], n_tokens=s["n"], n_prompt=s["prompt"],
                             repetition=s["rep"], presence=s["pres"], frequency=s["freq"], bias_ids=s.get("ids"),
                             bias=s.get("bias"), allowed=s.get("allowed"))


_OWN = {"rope": _own_rope, "attn": _own_attn, "logits": _own_logits}


# ------------------------------------------------------------------ the plain forms

# The cache holds blocks of 32 positions of one key/value head: keys as [D/16][2][32][8] (step of
# 16 dimensions, half of it, key, dimension), values as [D/32][2][2][32][2][4] (tile of 32
# dimensions, t, h, dimension, a, b: key 16 t + 8 a + 4 h + b).

def _key_offset(p, d):
    return (d // 16) * 512 + (d % 16 // 8) * 256 + p % 32 * 8 + d % 8


def _value_offset(p, d):
    t, a, h, b = p % 32 // 16, p % 16 // 8, p % 8 // 4, p % 4
    return (d // 32) * 1024 + t * 512 + h * 256 + d % 32 * 8 + a * 4 + b


def _rows(s):
    """Sequence and position of each row."""
    cu, kv = s["cu"].long(), s["kv"].long()
    row = torch.arange(s["T"], device="cuda")
    seq = torch.searchsorted(cu, row, right=True) - 1
    return seq, kv[seq] - (cu[seq + 1] - row)


def _plain_rope(s):
    c, H, KV, D = s["case"], s["H"], s["KV"], s["D"]
    T, rot, page, dt = s["T"], c["rot"], c["page"], s["k"].dtype
    seq, pos = _rows(s)
    x = s["qkv"].view(T, H + 2 * KV, D)
    q, k, v = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * s["qn"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * s["kn"]
    angle = pos.double()[:, None] * s["freq"]
    cos, sin = ((t * s["m"]).float()[:, None] for t in (angle.cos(), angle.sin()))
    x = torch.cat([q, k], 1)
    head, rest = x[..., :rot], x[..., rot:]
    if c["layout"] == "half":
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        head = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    x = torch.cat([head, rest], -1)
    q, k = x[:, :H], x[:, H:]
    block = s["table"].long()[seq, pos // page][:, None] * KV + torch.arange(KV, device="cuda")
    at = (block * page + (pos % page // 32 * 32)[:, None]) * D
    d = torch.arange(D, device="cuda")
    s["k"].view(-1)[at[..., None] + _key_offset(pos[:, None, None], d)] = k.to(dt)
    s["v"].view(-1)[at[..., None] + _value_offset(pos[:, None, None], d)] = v.to(dt)
    return q.to(dt).reshape(T, H * D), s["k"], s["v"]


def _unpack(k, v):
    """Pages in the cache's order -> [page][head][position][dimension]."""
    P, KV, page, D = k.shape
    k = k.view(P, KV, page // 32, D // 16, 2, 32, 8).permute(0, 1, 2, 5, 3, 4, 6).reshape(P, KV, page, D)
    v = v.view(P, KV, page // 32, D // 32, 2, 2, 32, 2, 4).permute(0, 1, 2, 4, 7, 5, 8, 3, 6).reshape(P, KV, page, D)
    return k, v


def _plain_attn(s):
    c, H, KV, D = s["case"], s["H"], s["KV"], s["D"]
    B, T, page, G = len(s["kv"]), s["T"], c["page"], H // KV
    cu, kv, table = s["cu"].long(), s["kv"].long(), s["table"].long().clamp(min=0)
    S, n = table.shape[1] * page, s["max_q"]
    k, v = (x[table].transpose(1, 2).reshape(B, KV, S, D).float() for x in _unpack(s["k"], s["v"]))
    at = torch.arange(S, device="cuda")
    v = torch.where((at < kv[:, None])[:, None, :, None], v, 0.0)
    i = torch.arange(n, device="cuda")
    row = (cu[:-1, None] + i).clamp(max=T - 1)
    here = i < (cu[1:] - cu[:-1])[:, None]
    pos = kv[:, None] - (cu[1:] - cu[:-1])[:, None] + i
    q = s["q"].float().view(T, KV, G, D)[row].permute(0, 2, 3, 1, 4).reshape(B, KV, G * n, D)
    x = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    seen = at <= pos[..., None]
    if c["window"]:
        seen = seen & (at > pos[..., None] - c["window"])
    x = x.view(B, KV, G, n, S).masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, KV, G * n, S), v).view(B, KV, G, n, D) / torch.where(total == 0, 1.0, total)
    out = torch.empty((T, H * D), dtype=DTYPES[c["out"]], device="cuda")
    out[row[here]] = o.permute(0, 3, 1, 2, 4)[here].reshape(-1, H * D).to(out.dtype)
    return out


def _plain_logits(s):
    x, V = s["logits"], s["case"]["vocab"]
    rows, n = s["tokens"].shape
    j = torch.arange(n, device="cuda")
    said, made = j < s["n"][:, None], (j >= s["prompt"][:, None]) & (j < s["n"][:, None])
    ids = s["tokens"].long()
    any_ = torch.zeros((rows, V), device="cuda").scatter_add_(1, ids, said.float()) > 0
    count = torch.zeros((rows, V), device="cuda").scatter_add_(1, ids, made.float())
    rep = s["rep"][:, None]
    x = torch.where(any_, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["freq"][:, None] * count - s["pres"][:, None] * (count > 0)
    if "ids" in s:
        x = x + torch.zeros_like(x, dtype=torch.float64).scatter_add_(1, s["ids"].long(), s["bias"].double()).float()
    if "allowed" in s:
        bits = s["allowed"].repeat_interleave(32, 1)[:, :V] >> (torch.arange(V, device="cuda") % 32)
        x = torch.where(bits & 1 == 1, x, -math.inf)
    return x


_PLAIN = {"rope": _plain_rope, "attn": _plain_attn, "logits": _plain_logits}


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    if case["op"] == "logits":
        n = case["rows"] * case["vocab"]
        read = case["rows"] * (4 * case["tokens"] + 8 * case["biases"]) + (n // 8 if case["mask"] else 0)
        return {"bytes": 8 * n + read, "flops": 6 * n}
    H, KV, D = HEADS[case["heads"]]
    qs, kvs = _lengths(case)
    if case["op"] == "rope":
        n = sum(qs) * (H + 2 * KV) * D
        return {"bytes": 6 * n, "flops": 6 * n}
    W, bytes_, pairs = case["window"], 0, 0
    for q, kv in zip(qs, kvs):
        first = max(0, kv - q + 1 - W) if W else 0
        bytes_ += 4 * q * H * D + 4 * (kv - first) * KV * D
        pairs += sum(min(p + 1, W) if W else p + 1 for p in range(kv - q, kv))
    return {"bytes": bytes_, "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------ the same in 64 bits, apart from the above

def exact(case, seed):
    return _EXACT[case["op"]](case, prepare(case, seed))


def _exact_rope(case, s):
    H, KV, D, rot, page = s["H"], s["KV"], s["D"], case["rot"], case["page"]
    qs, kvs = _lengths(case)
    x = s["qkv"].double().view(-1, H + 2 * KV, D)
    if case["norm"]:
        w = torch.cat([s["qn"].double().expand(H, D), s["kn"].double().expand(KV, D), torch.ones((KV, D), device="cuda").double()])
        r = 1 / torch.sqrt((x * x).sum(-1, keepdim=True) / D + 1e-6)
        r[:, H + KV:] = 1
        x = x * r * w
    pos = torch.cat([torch.arange(b - a, b) for a, b in zip(qs, kvs)]).cuda()
    turn = torch.polar(torch.full((len(pos), rot // 2), float(s["m"]), device="cuda").double(), pos[:, None] * s["freq"])
    head = x[:, :H + KV, :rot].unflatten(-1, (2, rot // 2) if case["layout"] == "half" else (rot // 2, 2))
    head = head.transpose(-1, -2) if case["layout"] == "half" else head
    y = torch.view_as_real(torch.view_as_complex(head.contiguous()) * turn[:, None])
    y = (y.transpose(-1, -2) if case["layout"] == "half" else y).flatten(-2)
    x = torch.cat([torch.cat([y, x[:, :H + KV, rot:]], -1), x[:, H + KV:]], 1)
    k, v = s["k"].double(), s["v"].double()
    # blocks in plain order, written by position, and back into the cache's order
    kk, vv = _unpack(k, v)
    seq = torch.cat([torch.full((a,), i) for i, a in enumerate(qs)]).cuda()
    kk[s["table"][seq, pos // page].long(), :, pos % page] = x[:, H:H + KV]
    vv[s["table"][seq, pos // page].long(), :, pos % page] = x[:, H + KV:]
    P = k.shape[0]
    k = kk.view(P, KV, page // 32, 32, D // 16, 2, 8).permute(0, 1, 2, 4, 5, 3, 6).reshape(k.shape)
    v = vv.view(P, KV, page // 32, 2, 2, 2, 4, D // 32, 32).permute(0, 1, 2, 7, 3, 5, 8, 4, 6).reshape(v.shape)
    return x[:, :H].reshape(-1, H * D), k, v


def _exact_attn(case, s):
    H, KV, D, page = s["H"], s["KV"], s["D"], case["page"]
    G, out, at = H // KV, [], 0
    d = torch.arange(D, device="cuda")
    for b, (n, kv) in enumerate(zip(*_lengths(case))):
        p = torch.arange(kv, device="cuda")
        base = (s["table"][b].long()[p // page] * KV * page + p % page // 32 * 32)[:, None] * D
        pos = torch.arange(kv - n, kv, device="cuda")
        heads = []
        for h in range(KV):
            o = base + h * page * D
            K = s["k"].view(-1)[o + _key_offset(p[:, None], d)].double()
            V = s["v"].view(-1)[o + _value_offset(p[:, None], d)].double()
            for j in range(G):
                c = (h * G + j) * D
                x = s["q"][at:at + n, c:c + D].double() @ K.T * s["scale"]
                if case["cap"]:
                    x = torch.tanh(x / case["cap"]) * case["cap"]
                far = pos[:, None] - p
                x[(far < 0) | (far >= case["window"] if case["window"] else far < 0)] = -math.inf
                heads.append(torch.softmax(x, -1) @ V)
        out.append(torch.cat(heads, -1))
        at += n
    return torch.cat(out)


def _exact_logits(case, s):
    x, V = s["logits"].double(), case["vocab"]
    out = []
    for r in range(case["rows"]):
        n, first = int(s["n"][r]), int(s["prompt"][r])
        t = s["tokens"][r].long()
        all_, made = (torch.bincount(v, minlength=V) for v in (t[:n], t[first:n]))
        y = x[r].clone()
        rep = s["rep"][r].double()
        y = torch.where((all_ > 0) & (y > 0), y / rep, torch.where(all_ > 0, y * rep, y))
        y = y - made * s["freq"][r].double() - (made > 0) * s["pres"][r].double()
        if case["biases"]:
            y.index_add_(0, s["ids"][r].long(), s["bias"][r].double())
        if case["mask"]:
            v = torch.arange(V, device="cuda")
            y[((s["allowed"][r].long()[v // 32] >> (v % 32)) & 1) == 0] = -math.inf
        out.append(y)
    return torch.stack(out)


_EXACT = {"rope": _exact_rope, "attn": _exact_attn, "logits": _exact_logits}

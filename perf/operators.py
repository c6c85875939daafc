"""What the operators of log probabilities and of the small-batch MoE layer are measured on.

Three operators, in the order in which one decode step uses them:

* ``moe``: a whole mixture-of-experts feed-forward layer (router, top-k softmax, SwiGLU experts, weighted
  sum) for 1 to 16 rows;
* ``linear``: log probability of a given token and entropy of the next-token distribution of every row,
  from the hidden states and the LM head, with no logits in memory (scoring a prompt);
* ``token``: log probability and rank of given tokens, entropy and top alternatives from logits that are
  there already (a decode step that reports log probabilities).

With ``own`` false, ``run`` computes them from elementary torch operations in 32 bits.
"""

import math

import torch

own = False

NAN, INF = float("nan"), float("inf")


def listed():
    return [
        # ---- token: the logits of a decode step
        # one chat that asks for 20 alternatives a token: the smallest call, latency counts
        dict(name="token_b1_top20", op="token", rows=1, vocab=151936, dtype="fp32", top=20, masked=0.0),
        # the default decode batch with a few alternatives
        dict(name="token_b32_top5", op="token", rows=32, vocab=151936, dtype="fp32", top=5, masked=0.0),
        # the widest decode step over the largest vocabulary
        dict(name="token_b256_top20", op="token", rows=256, vocab=248320, dtype="fp32", top=20, masked=0.0),
        # odd sizes, 16-bit logits (many equal values), most of the vocabulary masked as by a grammar
        dict(name="token_b7_bf16_masked", op="token", rows=7, vocab=32003, dtype="bf16", top=9, masked=0.97),
        # ---- linear: scoring
        # one row: a candidate answer's next token; the LM head is read once
        dict(name="linear_t1", op="linear", rows=1, vocab=151936, hidden=4096, packed=True, softcap=0.0),
        # a prompt chunk: perplexity of a document
        dict(name="linear_t2048", op="linear", rows=2048, vocab=151936, hidden=4096, packed=True, softcap=0.0),
        # a tiny model's head, a few rows: launch latency
        dict(name="linear_tiny", op="linear", rows=37, vocab=32000, hidden=256, packed=True, softcap=0.0),
        # odd sizes, a plain weight and capped logits
        dict(name="linear_odd_capped", op="linear", rows=777, vocab=50257, hidden=1608, packed=False, softcap=30.0),
        # ---- moe: one layer's feed-forward for the rows of a decode step
        # a single chat: eight experts of 128 are read
        dict(name="moe_t1", op="moe", rows=1, hidden=2048, experts=128, top=8, inner=768, renorm=True, first=0,
             local=128),
        # sixteen chats: most experts are read
        dict(name="moe_t16", op="moe", rows=16, hidden=2048, experts=128, top=8, inner=768, renorm=True, first=0,
             local=128),
        # few wide experts, odd inner size, half of them on this rank (rows may have no expert here)
        dict(name="moe_t5_wide_half", op="moe", rows=5, hidden=4096, experts=8, top=2, inner=1423, renorm=True,
             first=4, local=4),
        # a tiny model: launch latency
        dict(name="moe_tiny", op="moe", rows=3, hidden=256, experts=16, top=4, inner=128, renorm=False, first=0,
             local=16),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["token", "linear", "moe"])
    if op == "token":
        vocab = _log_int(rng, 1000, 262144)
        rows = _log_int(rng, 1, min(256, 256 * 248320 // vocab))
        return dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["fp32", "bf16"]), top=rng.randint(0, 20),
                    masked=rng.choice([0.0, 0.0, 0.5, 0.99]))
    if op == "linear":
        vocab, hidden = _log_int(rng, 1000, 152000), 8 * _log_int(rng, 8, 512)
        rows = _log_int(rng, 1, min(4096, 2048 * 151936 * 4096 // (vocab * hidden), 2048 * 151936 // vocab))
        return dict(op=op, rows=rows, vocab=vocab, hidden=hidden, packed=rng.random() < 0.5,
                    softcap=rng.choice([0.0, 0.0, 30.0]))
    hidden, inner = 8 * _log_int(rng, 8, 512), _log_int(rng, 24, 1536)
    experts = _log_int(rng, 2, max(2, min(128, 128 * 768 * 2048 // (hidden * inner))))
    top = rng.randint(1, min(8, experts))
    rows = rng.randint(1, max(1, min(16, 16 * 8 * 768 * 2048 // (top * hidden * inner))))
    local = experts if rng.random() < 0.6 else max(1, experts // 2)
    return dict(op=op, rows=rows, hidden=hidden, experts=experts, top=top, inner=inner, renorm=rng.random() < 0.7,
                first=experts - local, local=local)


# ------------------------------------------------------------------ inputs
def _randn(g, *shape, scale=1.0, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0.0, scale, generator=g)


def _tiles(w):
    """[..., N, K] -> the tile-contiguous layout the framework keeps GEMM weights in: tiles of 128 rows x 64
    columns, each one contiguous piece, N and K zero-padded; experts (a leading dim) back to back. [*, 64]."""
    n, k = w.shape[-2:]
    w = torch.nn.functional.pad(w, (0, -k % 64, 0, -n % 128))
    w = w.view(-1, w.shape[-2] // 128, 128, w.shape[-1] // 64, 64)
    return w.permute(0, 1, 3, 2, 4).contiguous().view(-1, 64)


def _token_state(case, g):
    B, V = case["rows"], case["vocab"]
    logits = _randn(g, B, V, scale=2.5)
    # rows from unsure to almost certain: one token of each row stands out by 0 to 20
    peak = torch.randint(0, V, (B, 1), device="cuda", generator=g)
    lift = torch.rand(B, 1, device="cuda", generator=g) * 20.0
    logits.scatter_add_(1, peak, lift)
    if case["masked"]:
        drop = torch.rand(B, V, device="cuda", generator=g) < case["masked"]
        drop.scatter_(1, peak, False)
        logits.masked_fill_(drop, -INF)
    # half of the rows ask for the token that stands out, half for any one
    tokens = torch.where(torch.rand(B, device="cuda", generator=g) < 0.5, peak[:, 0],
                         torch.randint(0, V, (B,), device="cuda", generator=g))
    return dict(logits=logits.bfloat16() if case["dtype"] == "bf16" else logits, tokens=tokens)


def _linear_state(case, g):
    T, V, H = case["rows"], case["vocab"], case["hidden"]
    w = _randn(g, V, H, scale=1.3 / math.sqrt(H), dtype=torch.bfloat16)
    tokens = torch.randint(0, V, (T,), device="cuda", generator=g)
    # hidden states that lean towards their token: its logit is lifted by 0 to 15
    lift = torch.rand(T, 1, device="cuda", generator=g) * 15.0 / 1.69
    x = (_randn(g, T, H) + lift * w[tokens].float()).bfloat16()
    return dict(x=x, w=w, tokens=tokens, tiles=_tiles(w) if case["packed"] else None)


def _moe_state(case, g):
    T, H, E, I, L = case["rows"], case["hidden"], case["experts"], case["inner"], case["local"]
    bf = torch.bfloat16
    x = _randn(g, T, H, dtype=bf)
    router = _randn(g, E, H, scale=1.4 / math.sqrt(H), dtype=bf)
    gate, up = (_randn(g, L, I, H, scale=1.0 / math.sqrt(H), dtype=bf) for _ in range(2))
    down = _randn(g, L, H, I, scale=1.0 / math.sqrt(I), dtype=bf)
    # the framework's expert layout: gate and up interleaved by 64 rows, the inner size padded to 64
    pad = -I % 64
    both = torch.stack([torch.nn.functional.pad(m, (0, 0, 0, pad)).view(L, -1, 64, H) for m in (gate, up)], 2)
    n_gate_up = 2 * (I + pad)
    return dict(x=x, router=router, gate=gate, up=up, down=down, n_gate_up=n_gate_up,
                gate_up_tiles=_tiles(both.view(L, n_gate_up, H)),
                down_tiles=_tiles(torch.nn.functional.pad(down, (0, pad))))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"token": _token_state, "linear": _linear_state, "moe": _moe_state}[case["op"]](case, g)
    return dict(state, case=case)


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    return {"token": _plain_token, "linear": _plain_linear, "moe": _plain_moe}[case["op"]](case, state)


def _own(case, s):
    from b200serve import ops
    if case["op"] == "token":
        return ops.token_logprobs(s["logits"], s["tokens"], top=case["top"])._asdict()
    if case["op"] == "linear":
        w = s["w"]
        if case["packed"]:
            w = ops.PackedWeight.from_packed(s["tiles"], case["vocab"], case["hidden"])
        logprob, entropy = ops.linear_logprobs(s["x"], w, s["tokens"], softcap=case["softcap"])
        return dict(logprob=logprob, entropy=entropy)
    return ops.moe_layer(s["x"], s["router"], s["gate_up_tiles"], s["n_gate_up"], s["down_tiles"], case["hidden"],
                         case["top"], renormalize=case["renorm"], first_expert=case["first"])


def _stats(logits, tokens):
    """Log probability of ``tokens`` and entropy of the rows of fp32 ``logits`` (-inf: masked)."""
    d = logits - logits.amax(-1, keepdim=True)
    p = d.exp()
    s = p.sum(-1)
    log_s = s.log()
    logprob = d.gather(1, tokens[:, None])[:, 0] - log_s
    entropy = log_s - (p * d.clamp_min(-1e30)).sum(-1) / s        # a masked entry adds 0 * -1e30
    return logprob, entropy, log_s, d


def _plain_token(case, s):
    logits, tokens, k = s["logits"].float(), s["tokens"], case["top"]
    logprob, entropy, log_s, d = _stats(logits, tokens)
    at = logits.gather(1, tokens[:, None])
    ids = torch.arange(logits.shape[1], device=logits.device)
    rank = (logits > at).sum(-1) + ((logits == at) & (ids < tokens[:, None])).sum(-1)
    best = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :k]     # ties: lowest id first
    top = d.gather(1, best) - log_s[:, None]
    best = torch.where(top == -INF, -1, best)
    return dict(logprob=logprob, rank=rank.int(), entropy=entropy, top_ids=best.int(), top_logprobs=top)


def _plain_linear(case, s):
    logits = s["x"].float() @ s["w"].float().t()
    if case["softcap"]:
        logits = case["softcap"] * torch.tanh(logits / case["softcap"])
    logprob, entropy, _, _ = _stats(logits, s["tokens"])
    return dict(logprob=logprob, entropy=entropy)


def _plain_moe(case, s):
    x, L = s["x"].float(), case["local"]
    p = torch.softmax(x @ s["router"].float().t(), -1)
    wts, ids = torch.topk(p, case["top"], -1)
    if case["renorm"]:
        wts = wts / wts.sum(-1, keepdim=True)
    here = ids - case["first"]
    wts = torch.where((here >= 0) & (here < L), wts, 0.0)            # another rank adds the other experts
    here = here.clamp(0, L - 1)
    g = torch.einsum("th,tkih->tki", x, s["gate"][here].float())
    u = torch.einsum("th,tkih->tki", x, s["up"][here].float())
    act = g * torch.sigmoid(g) * u * wts[..., None]
    return torch.einsum("tki,tkhi->th", act, s["down"][here].float()).to(s["x"].dtype)


# ------------------------------------------------------------------ work and the 64-bit answer
def work(case):
    if case["op"] == "token":
        B, V = case["rows"], case["vocab"]
        size = 2 if case["dtype"] == "bf16" else 4
        return dict(bytes=B * V * size + B * (8 + 12 + 8 * case["top"]), flops=5 * B * V)
    if case["op"] == "linear":
        T, V, H = case["rows"], case["vocab"], case["hidden"]
        return dict(bytes=2 * (T * H + V * H) + T * 16, flops=2 * T * V * H)
    T, H, E, k, I, L = (case[n] for n in ("rows", "hidden", "experts", "top", "inner", "local"))
    read = L * (1.0 - (1.0 - k / E) ** T)              # experts of this rank that some row takes, on average
    return dict(bytes=2 * (E * H + read * 3 * I * H + 2 * T * H), flops=2 * T * E * H + 6 * T * k * L / E * I * H)


def _exact_rows(logits, tokens, k):
    """(logprob, entropy, k largest log probabilities) of 64-bit logits, one row at a time."""
    lp, ent, top = [], [], []
    for row, t in zip(logits, tokens.tolist()):
        lse = torch.logsumexp(row, 0)
        logp = row - lse
        kept = logp[logp > -INF]
        ent.append(-(kept.exp() * kept).sum())
        lp.append(logp[t])
        best = torch.topk(logp, min(k, logp.numel())).values
        top.append(torch.nn.functional.pad(best, (0, k - best.numel()), value=-INF))
    return torch.stack(lp), torch.stack(ent), torch.stack(top)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "token":
        lp, ent, top = _exact_rows(s["logits"].double(), s["tokens"], case["top"])
        return dict(logprob=lp, rank=None, entropy=ent, top_ids=None, top_logprobs=top)
    if case["op"] == "linear":
        lps, ents = [], []
        for t0 in range(0, case["rows"], 512):
            x, cols = s["x"][t0:t0 + 512].double(), []
            for v0 in range(0, case["vocab"], 16384):
                cols.append(x @ s["w"][v0:v0 + 16384].double().t())
            logits = torch.cat(cols, 1)
            if case["softcap"]:
                logits = torch.tanh(logits / case["softcap"]) * case["softcap"]
            lp, ent, _ = _exact_rows(logits, s["tokens"][t0:t0 + 512], 0)
            lps.append(lp)
            ents.append(ent)
        return dict(logprob=torch.cat(lps), entropy=torch.cat(ents))
    out = []
    for x in s["x"].double():
        z = s["router"].double() @ x
        chosen = torch.topk(z, case["top"]).indices.tolist()
        p = torch.exp(z - torch.logsumexp(z, 0))
        share = p[chosen].sum() if case["renorm"] else 1.0
        y = torch.zeros_like(x)
        for e in chosen:
            i = e - case["first"]
            if 0 <= i < case["local"]:
                g, u = s["gate"][i].double() @ x, s["up"][i].double() @ x
                y = y + p[e] / share * (s["down"][i].double() @ (g / (1.0 + torch.exp(-g)) * u))
        out.append(y)
    return torch.stack(out)

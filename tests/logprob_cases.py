"""64-bit references and error bounds shared by the log-probability and MoE-layer tests."""

import math

import torch

NAN, INF = float("nan"), float("inf")


def reference_row(row: torch.Tensor, token: int, top: int):
    """(logprob, rank, entropy, top ids, top logprobs) of one row of logits, in 64 bits, by definition."""
    x = row.double().cpu()
    V = x.numel()
    if bool(x.isnan().any()) or float(x.max()) in (INF, -INF):
        return NAN, -1, NAN, [-1] * top, [NAN] * top
    m = x.max()
    logp = (x - m) - torch.log(torch.exp(x - m).sum())      # m + log s would lose log s beside a large m
    kept = logp[logp > -INF]
    entropy = float(-(kept.exp() * kept).sum())
    lp, rank = NAN, -1
    if 0 <= token < V:
        lp = float(logp[token])
        rank = int((x > x[token]).sum()) + int((x[:token] == x[token]).sum())
    order = torch.sort(x, descending=True, stable=True).indices[:top].tolist()
    ids = [i if float(x[i]) > -INF else -1 for i in order] + [-1] * (top - len(order))
    return lp, rank, entropy, ids, [float(logp[i]) if i >= 0 else -INF for i in ids]


# fp32 statistics of V logits: a term e^d carries ex2's 2^-22 and the rounding of d and of
# d log2(e), 2^-23 |d| each, where the terms that matter have |d| <= ln V; a sum of partial sums of
# at most 64 terms each, joined in trees, adds 80 * 2^-24
def log_s_bound(V: int) -> float:
    return (1 + math.log(max(V, 2))) * 2.0 ** -22 + 80 * 2.0 ** -24


def logprob_bound(V: int, value, logit_err: float = 0.0) -> float:
    """log p = (x - m) - log s: the bound of log s, two roundings, and twice an error of the logits."""
    v = abs(value) if math.isfinite(value) else 0.0
    return 2 * logit_err + log_s_bound(V) + v * 2.0 ** -22


def entropy_bound(V: int, logit_err: float = 0.0) -> float:
    """H = log s - t / s: t's terms carry the relative error of s's twice over (e^d and d), |t| / s <= ln V;
    |dH| <= sum p |log p + H| |dx| <= 2 ln V |dx|."""
    return log_s_bound(V) * (1 + 4 * math.log(max(V, 2))) + 2 * math.log(max(V, 2)) * logit_err


def check_token_logprobs(got, logits, tokens, top):
    V = logits.shape[1]
    assert got.logprob.dtype == got.entropy.dtype == got.top_logprobs.dtype == torch.float32
    assert got.rank.dtype == got.top_ids.dtype == torch.int32
    assert got.top_ids.shape == got.top_logprobs.shape == (logits.shape[0], top)
    for b in range(logits.shape[0]):
        lp, rank, ent, ids, lps = reference_row(logits[b], int(tokens[b]), top)
        assert got.rank[b].item() == rank, (b, got.rank[b].item(), rank)
        assert got.top_ids[b].tolist() == ids, b
        _close(got.logprob[b].item(), lp, logprob_bound(V, lp), (b, "logprob"))
        _close(got.entropy[b].item(), ent, entropy_bound(V), (b, "entropy"))
        for j, v in enumerate(lps):
            _close(got.top_logprobs[b, j].item(), v, logprob_bound(V, v), (b, "top", j))


def _close(a, ref, tol, where):
    if math.isnan(ref):
        assert math.isnan(a), (where, a)
    elif math.isinf(ref):
        assert a == ref, (where, a, ref)
    else:
        assert abs(a - ref) <= tol, (where, a, ref, tol)


def check_linear_logprobs(got, x, w, tokens, softcap):
    """w [V, H] plain. The logits' own error: a product of 16 elements at a time is added to the fp32 sum, and each
    addition may cut one unit in the last place of the largest partial sum (bounded by sum |x| |w|), once for the
    sum and once for the alignment of the products."""
    V, H = w.shape
    lp, ent = got
    xd, wd = x.double().cpu(), w.double().cpu()
    logits = xd @ wd.t()
    spread = (xd.abs() @ wd.abs().t()).amax(-1)
    if softcap:
        logits = softcap * torch.tanh(logits / softcap)
    for t in range(x.shape[0]):
        a, _, e, _, _ = reference_row(logits[t], int(tokens[t]), 0)
        err = (math.ceil(H / 16) * 2.0 ** -22) * float(spread[t]) + (softcap or 0.0) * 2.0 ** -21
        if math.isnan(a) and 0 <= int(tokens[t]) < V:
            assert math.isnan(lp[t].item()) and math.isnan(ent[t].item()), t
            continue
        _close(lp[t].item(), a, logprob_bound(V, a, err), (t, "logprob"))
        _close(ent[t].item(), e, entropy_bound(V, err), (t, "entropy"))


# ------------------------------------------------------------------ MoE layer
def pack(stacked: torch.Tensor) -> torch.Tensor:
    """[E, N, K] -> tiles of 128 x 64 (zero-padded), experts back to back, [*, 64]."""
    E, N, K = stacked.shape
    w = torch.nn.functional.pad(stacked, (0, -K % 64, 0, -N % 128))
    return w.view(E, w.shape[1] // 128, 128, w.shape[2] // 64, 64).permute(0, 1, 3, 2, 4).reshape(-1, 64).contiguous()


class MoECase:
    """Random layer of E experts of which [first, first + local) are here. Rows whose k-th and next router logit
    are closer than 1e-3 are drawn again, so that no rounding can change the choice."""

    def __init__(self, T, H, E, k, inner, first=0, local=None, renorm=True, seed=0):
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g)
        self.T, self.H, self.E, self.k, self.inner = T, H, E, k, inner
        self.first, self.local, self.renorm = first, E if local is None else local, renorm
        self.router = (rnd(E, H) * 1.4 / math.sqrt(H)).bfloat16()
        rows = []
        while len(rows) < T:
            r = rnd(H).bfloat16()
            z = (self.router.double() @ r.double()).sort(descending=True).values
            if k == E or float(z[k - 1] - z[k]) > 1e-3:
                rows.append(r)
        self.x = torch.stack(rows) if T else torch.empty(0, H, dtype=torch.bfloat16)
        L = self.local
        self.gate, self.up = ((rnd(L, inner, H) / math.sqrt(H)).bfloat16() for _ in range(2))
        self.down = (rnd(L, H, inner) / math.sqrt(inner)).bfloat16()
        pad = -inner % 64
        both = torch.stack([torch.nn.functional.pad(m, (0, 0, 0, pad)).view(L, -1, 64, H)
                            for m in (self.gate, self.up)], 2)
        self.n_gate_up = 2 * (inner + pad)
        self.gate_up_tiles = pack(both.view(L, self.n_gate_up, H))
        self.down_tiles = pack(torch.nn.functional.pad(self.down, (0, pad)))

    def args(self, device="cpu"):
        to = lambda t: t.to(device)
        return (to(self.x), to(self.router), to(self.gate_up_tiles), self.n_gate_up, to(self.down_tiles), self.H,
                self.k, self.renorm, self.first)

    def reference(self, x=None):
        """(out [T, H] in 64 bits, bound [T, H] of a kernel's error)."""
        x = (self.x if x is None else x).double()
        out, bound = torch.zeros(x.shape[0], self.H).double(), torch.zeros(x.shape[0], self.H).double()
        step = math.ceil(self.H / 16) * 2.0 ** -22
        step2 = math.ceil((self.inner + 64) * self.k / 16) * 2.0 ** -22
        for t in range(x.shape[0]):
            z = self.router.double() @ x[t]
            p = torch.softmax(z, -1)
            ids = torch.sort(p, descending=True, stable=True).indices[:self.k].tolist()
            share = float(p[ids].sum()) if self.renorm else 1.0
            dz = step * float((self.router.double().abs() @ x[t].abs()).max())
            for e in ids:
                i = e - self.first
                if not 0 <= i < self.local:
                    continue
                G, U, D = self.gate[i].double(), self.up[i].double(), self.down[i].double()
                g, u, w = G @ x[t], U @ x[t], float(p[e]) / share
                dg, du = step * (G.abs() @ x[t].abs()), step * (U.abs() @ x[t].abs())
                s = g * torch.sigmoid(g)
                act = w * s * u
                # |d silu| <= 1.1; the activation is kept as two bf16, each off by at most half a step; the
                # router's error moves a weight by at most 2 dz of itself, e^. and sigmoid add 2^-20
                dact = w * (1.1 * u.abs() * dg + s.abs() * du) + act.abs() * (2.0 ** -16 + 2 * dz + 2.0 ** -20)
                out[t] += D @ act
                bound[t] += D.abs() @ dact + step2 * (D.abs() @ act.abs())
        return out, bound + (out.abs() + bound) * 2.0 ** -8

"""The 8-bit key/value cache's definition in 64 bits, token by token lists instead of a layout (test infrastructure)."""
import math

import torch

BLOCK = 64


def e4m3_grid(y):
    """Round-half-even to e4m3's values, saturating; float64."""
    y = y.clamp(-448.0, 448.0)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return (y / step).round() * step


def block_scale(x, kind):
    """Scale (a float that fp32 holds) of one block of float64 values."""
    fin = x[torch.isfinite(x)].abs()
    top = fin.max().item() if fin.numel() else 0.0
    if top == 0.0:
        return 1.0
    if kind == torch.int8:
        return max((torch.tensor(top, dtype=torch.float32) / 127).item(), 2.0 ** -100)
    p = math.floor(math.log2(top / 448)) - 1
    while 448 * 2.0 ** p < top:
        p += 1
    return 2.0 ** max(p, -100)


def block_codes(x, scale, kind):
    """Codes as float64 numbers (e4m3 may hold NaN)."""
    if kind == torch.int8:
        q = (x.float() / torch.tensor(scale, dtype=torch.float32)).double().round()     # the definition divides in fp32
        return torch.where(q.isnan(), 0.0, q.clamp(-127, 127))
    return e4m3_grid(x / scale)


class RefCache:
    """Values, scales and codes of every sequence and head as lists; ``x[b][h]`` are float64 ``[n, 128]``."""

    def __init__(self, batch, heads, kind):
        self.batch, self.heads, self.kind = batch, heads, kind
        z = lambda: [[torch.zeros(0, 128, dtype=torch.float64) for _ in range(heads)] for _ in range(batch)]
        self.raw = {"k": z(), "v": z()}             # bf16 values as they came, or the cached values after an eviction

    def append(self, key, value, counts=None):
        for name, x in (("k", key), ("v", value)):
            x = x.detach().cpu().double()
            for b in range(self.batch):
                n = x.shape[2] if counts is None else int(counts[b])
                for h in range(self.heads):
                    self.raw[name][b][h] = torch.cat((self.raw[name][b][h], x[b, h, :n]))

    def length(self, b):
        return self.raw["k"][b][0].shape[0]

    def values(self, name, b, h):
        """(values [n, 128], codes [n, 128], scale per token [n]); the tail has scale 1 and its values as codes."""
        x = self.raw[name][b][h]
        n, full = x.shape[0], x.shape[0] // BLOCK * BLOCK
        codes, scale = x.clone(), torch.ones(n, dtype=torch.float64)
        for i in range(0, full, BLOCK):
            s = block_scale(x[i:i + BLOCK], self.kind)
            codes[i:i + BLOCK] = block_codes(x[i:i + BLOCK], s, self.kind)
            scale[i:i + BLOCK] = s
        return codes * scale[:, None], codes, scale

    def evict(self, weights, budget, recent, sink):
        """kept[b][h] (list of int); the cache then holds the kept tokens' values (fp32 products; the tail rounds to bf16)."""
        kept = []
        for b in range(self.batch):
            n = self.length(b)
            kept.append([])
            for h in range(self.heads):
                idx = choose(weights[b, h, :n], budget, recent, sink)
                kept[b].append(idx)
                for name in ("k", "v"):
                    val, codes, scale = self.values(name, b, h)
                    x = (codes.float() * scale.float()[:, None])[idx]
                    full = len(idx) // BLOCK * BLOCK
                    x[full:] = x[full:].to(torch.bfloat16).float()
                    self.raw[name][b][h] = x.double()
        return kept


def choose(w, budget, recent, sink):
    n = w.numel()
    if n <= budget:
        return list(range(n))
    lo, hi = sink, n - recent
    rank = sorted(range(lo, hi), key=lambda t: (0 if math.isnan(w[t]) else 1, -float(w[t]) if not math.isnan(w[t]) else 0.0, t))
    return sorted(list(range(lo)) + rank[: budget - recent - sink] + list(range(hi, n)))


def attend(ref, query, b, h, sm_scale=None):
    """Attention of one query head ``query [S, 128]`` over (b, h): (out, tolerance of out, lse, tolerance of lse, p, relative
    tolerance of p), float64.  Rows that see nothing: zeros, -inf, p = 0.

    Tolerances count the roundings of a kernel that multiplies codes in f16 with fp32 accumulation:
      logits: 128 products summed in fp32, each step at most 2^-23 of the running magnitude (a tensor core may truncate):
              dl <= 128 * 2^-23 * A, A = sm_scale log2(e) sum |q k| -- and three fp32 roundings of the result;
      p:      relative ln2 * dl from its own logit and as much from the log-sum-exp, 2^-20 for exp2, log2 and the sums;
      out:    p rounded to f16 (2^-11) or, below 2^-14 of the largest numerator, to a grid of 2^-24 (half a step 2^-25 of
              the largest p s_v, for each code), fp32 sums 2^-20, and one rounding to bf16 (2^-8)."""
    k, _, _ = ref.values("k", b, h)
    v, codes, sv = ref.values("v", b, h)
    q = query.detach().cpu().double()
    S, n = q.shape[0], k.shape[0]
    f = (128 ** -0.5 if sm_scale is None else sm_scale) * math.log2(math.e)
    seen = torch.arange(n)[None, :] < (n - S + 1 + torch.arange(S))[:, None]
    logit = torch.where(seen, q @ k.T * f, -math.inf)
    mag = torch.where(seen, (q.abs() @ k.abs().T) * abs(f), 0.0).amax(-1) if n else torch.zeros(S, dtype=torch.float64)
    top = logit.amax(-1) if n else torch.full((S,), -math.inf, dtype=torch.float64)
    safe = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp2(logit - safe[:, None])
    total = e.sum(-1)
    lse = torch.where(total > 0, safe + torch.log2(total.clamp_min(1e-300)), -math.inf)
    p = e / total.clamp_min(1e-300)[:, None]
    vis = lambda x: torch.where(seen[:, :, None], x[None], 0.0)
    out = (p[:, :, None] * vis(v)).sum(1)
    dl = 128 * 2.0 ** -23 * mag + 3 * 2.0 ** -24 * torch.where(top == -math.inf, 0.0, top.abs()) + 2.0 ** -22
    rel = 2 * math.log(2) * dl + 2.0 ** -20
    spread = (p[:, :, None] * vis(v.abs())).sum(1)
    small = 2.0 ** -25 * (p * sv).amax(-1)[:, None] * vis(codes.abs()).sum(1) if n else torch.zeros_like(out)
    tol = 2.0 ** -8 * out.abs() + (2.0 ** -11 + rel[:, None]) * spread + small + 1e-30
    return out, tol, lse, dl + 2.0 ** -21 + 2.0 ** -22 * torch.where(lse == -math.inf, 0.0, lse.abs()), p, rel

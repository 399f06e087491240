"""Cases of the 8-bit key/value cache operators: storing tokens, attention over the cache, eviction by attention weight.

The cache of one layer holds keys and values in 8 bits, ``[B, Hkv, capacity, 128]`` codes (e4m3 or int8) with one fp32
scale for every block of 64 tokens of a head; the tokens behind the last complete block stay in bf16
(``[B, Hkv, 64, 128]``, token t in row t % 64).  Shapes are those of the layers this repository benchmarks: 32 query
heads over 8 key/value heads and 28 over 4, head size 128.  ``own`` selects the framework's kernels; otherwise every
operator is computed with elementary torch operations.
"""
import math

import torch

own = False

BLOCK, D = 64, 128
LOG2E = math.log2(math.e)


def listed():
    heads, few = {"hq": 32, "hkv": 8}, {"hq": 28, "hkv": 4}
    return [
        # one decoding step of a chat of a few thousand tokens: latency counts
        {"name": "attend_4k", "op": "attend", "batch": 1, **heads, "length": 4133, "queries": 1, "type": "e4m3", "weights": False},
        # one decoding step after a 131072-token prompt, the length of the benchmark's layer
        {"name": "attend_128k", "op": "attend", "batch": 1, **heads, "length": 131072, "queries": 1, "type": "e4m3", "weights": False},
        # the same for 28 / 4 heads at 262144 tokens, with the attention weights that eviction goes by
        {"name": "attend_256k_weights", "op": "attend", "batch": 1, **few, "length": 262144, "queries": 1, "type": "int8", "weights": True},
        # a million tokens
        {"name": "attend_1m", "op": "attend", "batch": 1, **heads, "length": 1048576, "queries": 1, "type": "e4m3", "weights": False},
        # a served batch of sequences of different lengths
        {"name": "attend_batch_ragged", "op": "attend", "batch": 16, **heads, "length": 32768, "queries": 1, "type": "e4m3", "weights": True},
        # five proposed tokens checked at once
        {"name": "attend_5_tokens", "op": "attend", "batch": 2, **heads, "length": 50001, "queries": 5, "type": "int8", "weights": False},
        # a follow-up question of 256 tokens
        {"name": "attend_256_tokens", "op": "attend", "batch": 1, **heads, "length": 16384, "queries": 256, "type": "e4m3", "weights": False},
        # one new token for each sequence of a served batch
        {"name": "store_token", "op": "store", "batch": 32, **heads, "length": 8192, "tokens": 1, "type": "e4m3"},
        # a whole prompt
        {"name": "store_128k", "op": "store", "batch": 1, **heads, "length": 0, "tokens": 131072, "type": "e4m3"},
        # a padded batch of follow-up prompts of odd lengths
        {"name": "store_chunk_ragged", "op": "store", "batch": 3, **heads, "length": 3001, "tokens": 1777, "type": "int8"},
        # a 131072-token prompt cut down to 4096 tokens before decoding
        {"name": "evict_128k", "op": "evict", "batch": 1, **heads, "length": 131072, "budget": 4096, "type": "e4m3"},
        # a served batch cut down to an odd budget
        {"name": "evict_batch_ragged", "op": "evict", "batch": 8, **few, "length": 9000, "budget": 1001, "type": "int8"},
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], evenly spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, hkv = rng.choice([(32, 8), (28, 4), (8, 8), (16, 2), (6, 2), (4, 1)])
    case = {"op": rng.choice(["attend", "attend", "store", "evict"]), "batch": rng.choice([1, 1, 2, 3, 7, 16]), "hq": hq, "hkv": hkv,
            "type": rng.choice(["e4m3", "int8"])}
    room = 4 * 1048576 // (case["batch"] * hkv)                  # tokens of a sequence: half the largest listed cache in all
    if case["op"] == "attend":
        case["queries"] = rng.choice([1, 1, 1, 2, 3, 8, 17, 64, 200])
        if case["queries"] > 8:
            room = min(room, 131072 * 8 // (case["batch"] * hq * case["queries"] // 8))
        case["length"] = _spread(rng, max(case["queries"], 40), max(room, 2 * case["queries"], 100))
        case["weights"] = rng.random() < 0.4
    elif case["op"] == "store":
        case["length"] = rng.choice([0, _spread(rng, 1, 8192)])
        case["tokens"] = _spread(rng, 1, min(room // 2, 131072))
    else:
        case["length"] = _spread(rng, 600, min(room, 524288))
        case["budget"] = _spread(rng, 90, min(case["length"], 16384))
    return case


def _lengths(case, gen):
    """Tokens held by each sequence: the first the longest, the others down to a third of it."""
    n = case["length"]
    low = max(case.get("queries", 1), n // 3)
    r = torch.randint(low, n + 1, (case["batch"],), generator=gen, device="cuda", dtype=torch.int32)
    r[0] = n
    return r


def _scale_of(x, kind):
    """fp32 scale of each block of ``x [..., tokens, 128]``: of its largest finite magnitude."""
    top = torch.where(x.isfinite(), x.abs(), 0.0).amax((-1, -2))
    if kind == "int8":
        s = (top / 127).clamp_min(2.0 ** -100)
    else:                                   # the smallest power of two that brings the block within e4m3's 448
        m, e = torch.frexp(top)
        s = torch.ldexp(torch.ones_like(top), (e - 8 - (m <= 0.875).to(e.dtype)).clamp_min(-100))
    return torch.where(top > 0, s, 1.0)


def _codes_of(x, scale, kind):
    y = x / scale[..., None, None]
    if kind == "int8":
        return y.round().clamp(-127, 127).nan_to_num(0.0).to(torch.int8)
    return y.clamp(-448, 448).to(torch.float8_e4m3fn)


def _kind(case):
    return torch.int8 if case["type"] == "int8" else torch.float8_e4m3fn


def _held(case, capacity, gen):
    """A cache that holds tokens: keys with a few strong channels and strong first tokens, values of about one.  Every
    block is filled; what lies behind a sequence's length is left from an earlier use."""
    b, h = case["batch"], case["hkv"]
    chan = 1.0 + 2.0 * (torch.rand(h, 1, D, generator=gen, device="cuda") > 0.95)
    state = {"k_tail": torch.randn(b, h, BLOCK, D, generator=gen, device="cuda") * chan, "v_tail": torch.randn(b, h, BLOCK, D, generator=gen, device="cuda")}
    state = {n: t.to(torch.bfloat16) for n, t in state.items()}
    for n in ("k", "v"):
        codes = torch.empty(b, h, capacity, D, dtype=_kind(case), device="cuda")
        scale = torch.empty(b, h, capacity // BLOCK, device="cuda")
        for i in range(b):
            for j in range(h):
                x = torch.randn(capacity, D, generator=gen, device="cuda")
                if n == "k":
                    x = x * chan[j]
                    x[:4] *= 2.0
                x = x.to(torch.bfloat16).float().view(-1, BLOCK, D)
                scale[i, j] = _scale_of(x, case["type"])
                codes[i, j] = _codes_of(x, scale[i, j], case["type"]).view(capacity, D)
        state[n], state[n + "_scale"] = codes, scale
    return state


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    b, h = case["batch"], case["hkv"]
    if case["op"] == "store":
        n = case["tokens"]
        start = _lengths(case, gen) if case["length"] else torch.zeros(b, dtype=torch.int32, device="cuda")
        counts = torch.randint(max(1, n // 2), n + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
        counts[0] = n
        window = (n + 2 * BLOCK - 2) // BLOCK * BLOCK                      # from the block the first new token lies in
        capacity = (case["length"] + n + BLOCK - 1) // BLOCK * BLOCK
        shape = (b, n, h, D)                                                # as a projection leaves them: heads inside
        state = {"start": start, "counts": counts, "first": start // BLOCK * BLOCK, "lengths": start + counts, "window": window,
                 "key": torch.randn(shape, generator=gen, device="cuda").to(torch.bfloat16).transpose(1, 2),
                 "value": torch.randn(shape, generator=gen, device="cuda").to(torch.bfloat16).transpose(1, 2)}
        for t in ("k", "v"):
            state[t] = torch.zeros(b, h, capacity, D, device="cuda").to(_kind(case))
            state[t + "_scale"] = torch.ones(b, h, capacity // BLOCK, device="cuda")
            state[t + "_tail"] = torch.randn(b, h, BLOCK, D, generator=gen, device="cuda").to(torch.bfloat16)
    else:
        capacity = (case["length"] + BLOCK - 1) // BLOCK * BLOCK
        state = _held(case, capacity, gen)
        state["lengths"] = _lengths(case, gen)
        if case["op"] == "attend":
            state["query"] = torch.randn(b, case["queries"], case["hq"], D, generator=gen, device="cuda").to(torch.bfloat16).transpose(1, 2)
        if case["op"] == "evict" or case["weights"]:
            # weights accumulated so far: few tokens hold most of them, and some were never looked at
            w = torch.exp(2.0 * torch.randn(b, h, capacity, generator=gen, device="cuda"))
            state["sums"] = torch.where(torch.rand(b, h, capacity, generator=gen, device="cuda") < 0.1, 0.0, w)
            state["sums_out"] = torch.zeros_like(state["sums"])
    if case["op"] == "evict":
        state["budget"], state["recent"], state["sink"] = case["budget"], case["budget"] // 4, 4
    state["op"], state["kind"], state["longest"] = case["op"], case["type"], case["length"]
    if own:
        from minference_b200 import KV8Cache

        tails = state["k_tail"], state["v_tail"]
        if case["op"] == "store" and case["length"] and case["tokens"] > 1:
            # these tokens replace the tail they complete: the next pass on this state needs it as it was
            state["cache_tails"] = tails
            tails = tails[0].clone(), tails[1].clone()
        state["cache"] = KV8Cache(state["k"], state["v"], state["k_scale"], state["v_scale"], *tails)
    return state


def run(state):
    if own:
        return _run_own(state)
    return {"store": _store, "attend": _attend, "evict": _evict}[state["op"]](state)


def _run_own(state):
    from minference_b200 import kv8_attention, kv8_evict, kv8_load, kv8_store

    cache = state["cache"]
    if state["op"] == "store":
        if "cache_tails" in state:
            cache.k_tail.copy_(state["cache_tails"][0])
            cache.v_tail.copy_(state["cache_tails"][1])
        kv8_store(cache, state["key"], state["value"], state["start"], counts=state["counts"])
        k, v = kv8_load(cache, state["lengths"], first=state["first"], count=state["window"])
        return {"k": k, "v": v}
    if state["op"] == "attend":
        if "sums" in state:
            out = kv8_attention(state["query"], cache, state["lengths"], max_length=state["longest"], weights=state["sums_out"], add_to=state["sums"])
            return {"out": out, "sums": state["sums_out"]}
        out, lse = kv8_attention(state["query"], cache, state["lengths"], max_length=state["longest"], return_lse=True)
        return {"out": out, "lse": lse}
    small, lengths, sums, kept = kv8_evict(cache, state["lengths"], state["sums"], state["budget"], recent=state["recent"], sink=state["sink"],
                                           max_length=state["longest"])
    k, v = kv8_load(small, lengths, count=state["budget"])
    return {"k": k, "v": v, "lengths": lengths, "sums": sums[..., : state["budget"]], "kept": kept}


# ---- the plain forms -------------------------------------------------------------------------------------------------


def _as_stored(x, first, end, kind):
    """Values that the cache gives back for tokens ``x [B, H, n, 128]`` from position ``first [B]`` (a block's start) on,
    when the sequences end at ``end [B]``: complete blocks through 8 bits, the others as they are, zeros behind the end."""
    b, h, n, _ = x.shape
    x = x.float()
    at = first[:, None].long() + torch.arange(n, device=x.device)
    live = at < end[:, None]
    blocks = x.view(b, h, n // BLOCK, BLOCK, D)
    scale = _scale_of(blocks, kind)
    through = (_codes_of(blocks, scale, kind).float() * scale[..., None, None]).view(b, h, n, D)
    whole = (at // BLOCK + 1) * BLOCK <= end[:, None]
    x = torch.where(whole[:, None, :, None], through, x)
    return torch.where(live[:, None, :, None], x, 0.0).to(torch.bfloat16)


def _store(state):
    start, counts, first, n = state["start"].long(), state["counts"].long(), state["first"].long(), state["window"]
    at = first[:, None] + torch.arange(n, device=start.device)
    old = at < start[:, None]
    out = {}
    for name, new in (("k", state["key"]), ("v", state["value"])):
        held = state[name + "_tail"].index_select(2, torch.arange(n, device=start.device) % BLOCK)
        i = (at - start[:, None]).clamp(0, new.shape[2] - 1)[:, None, :, None].expand(-1, new.shape[1], -1, D)
        x = torch.where(old[:, None, :, None], held, new.gather(2, i))
        out[name] = _as_stored(x, first, start + counts, state["kind"])
    return out


def _values(state, name):
    """The cache's tokens in fp32, ``[B, H, capacity, 128]``: the last incomplete block of each sequence from bf16."""
    codes, scale, tail, n = state[name], state[name + "_scale"], state[name + "_tail"], state["lengths"].long()
    b, h, cap, _ = codes.shape
    x = (codes.view(b, h, cap // BLOCK, BLOCK, D).float() * scale[..., None, None]).view(b, h, cap, D)
    at = (n // BLOCK * BLOCK)[:, None] + torch.arange(BLOCK, device=n.device)
    put = at < n[:, None]
    at = at.clamp_max(cap - 1)[:, None, :, None].expand(-1, h, -1, D)
    return x.scatter(2, at, torch.where(put[:, None, :, None], tail.float(), x.gather(2, at)))


def _attend(state):
    q, n = state["query"].float(), state["lengths"].long()
    k, v = _values(state, "k"), _values(state, "v")
    b, hq, s, _ = q.shape
    hkv, cap = k.shape[1], k.shape[2]
    q = q.reshape(b, hkv, hq // hkv * s, D)
    at = torch.arange(cap, device=q.device)
    end = n[:, None] - s + 1 + torch.arange(s, device=q.device)                      # query i sees the tokens before end[:, i]
    seen = (at < end[..., None])[:, None].repeat(1, 1, hq // hkv, 1)                 # [B, 1, G*S, capacity]
    logits = torch.where(seen, (q @ k.transpose(2, 3)) * (D ** -0.5 * LOG2E), -math.inf)
    top = logits.amax(-1, keepdim=True).clamp_min(-1e30)
    p = torch.exp2(logits - top)
    total = p.sum(-1, keepdim=True)
    p = p / total.clamp_min(1e-30)
    v = torch.where((at < n[:, None])[:, None, :, None], v, 0.0)
    out = (p @ v).view(b, hq, s, D).to(torch.bfloat16)
    if "sums" in state:
        live = (at < n[:, None])[:, None]
        return {"out": out, "sums": torch.where(live, state["sums"] + p.sum(2), state["sums_out"])}
    return {"out": out, "lse": (top + torch.log2(total)).view(b, hq, s)}


def _evict(state):
    n, budget, recent, sink, w = state["lengths"].long(), state["budget"], state["recent"], state["sink"], state["sums"]
    b, h, cap = w.shape
    at = torch.arange(cap, device=w.device)
    end = n[:, None, None]
    rank = torch.where((at < sink) | (at >= end - recent), math.inf, w)               # kept whatever their weight
    rank = torch.where(at < end, rank, -math.inf).expand(b, h, cap)
    order = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]     # equal weights: the earlier token
    held = n.clamp_max(budget)
    slot = torch.arange(budget, device=w.device)
    order = torch.where(slot < held[:, None, None], order, cap).sort(-1).values
    live = order < cap
    take = order.clamp_max(cap - 1)
    pad = (budget + BLOCK - 1) // BLOCK * BLOCK - budget
    out = {}
    for name in ("k", "v"):
        x = _values(state, name).gather(2, take[..., None].expand(-1, -1, -1, D))
        x = torch.where(live[..., None], x, 0.0)
        x = torch.cat((x, x.new_zeros(b, h, pad, D)), 2)
        out[name] = _as_stored(x, torch.zeros_like(n), held, state["kind"])[:, :, :budget]
    return {**out, "lengths": held.to(torch.int32), "sums": torch.where(live, w.gather(2, take), 0.0),
            "kept": torch.where(live, order, -1).to(torch.int32)}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------


def work(case):
    b, hq, h, n = case["batch"], case["hq"], case["hkv"], case["length"]
    tokens = n + (b - 1) * (n + max(case.get("queries", 1), n // 3)) / 2          # expected over the lengths prepare() makes
    if case["op"] == "store":
        new = case["tokens"] * (1 + (b - 1) * 0.75) * h * D
        return {"bytes": 2 * new * 2 + 2 * b * h * D * ((case["tokens"] + 2 * BLOCK - 2) // BLOCK * BLOCK) * 2, "flops": 2 * new}
    if case["op"] == "attend":
        rows = b * hq * case["queries"]
        read = tokens * h * 2 * D + tokens * h / BLOCK * 8 + 2 * rows * D * 2
        if case["weights"]:
            read += 2 * 4 * tokens * h
        pairs = tokens - b * (case["queries"] - 1) / 2
        return {"bytes": read, "flops": 4.0 * D * hq * case["queries"] * pairs}
    kept = case["budget"] * b * h
    return {"bytes": 4 * tokens * h + kept * (2 * D + 2 * D * 2 + 8), "flops": tokens * h}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------


def _exact_block(x, kind):
    """One block ``[64, 128]`` (float64) through 8 bits and back."""
    top = x.abs().max().item()
    if top == 0:
        return x
    if kind == "int8":
        s = torch.tensor(top, dtype=torch.float64).div(127).to(torch.float32).double().item()
        return (x / s).round() * s
    p = math.floor(math.log2(top / 448))
    while 448 * 2.0 ** p < top:
        p += 1
    y = x * 2.0 ** -p
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return (y / step).round() * step * 2.0 ** p


def _exact_blocks(x, kind):
    return torch.stack([_exact_block(blk, kind) for blk in x.split(BLOCK)]).view_as(x) if x.numel() else x


def _exact_tokens(state, name, i, j):
    """Tokens of sequence i, head j, in float64."""
    n = int(state["lengths"][i])
    full = n // BLOCK
    x = state[name][i, j, : full * BLOCK].double().view(full, BLOCK, D) * state[name + "_scale"][i, j, :full].double()[:, None, None]
    return torch.cat((x.reshape(-1, D), state[name + "_tail"][i, j, : n - full * BLOCK].double()))


def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    b, h = case["batch"], case["hkv"]
    if case["op"] == "store":
        if case["tokens"] * b * h > 8 * 131072:
            return None                                     # block by block it would take too long
        out = {t: torch.zeros(b, h, state["window"], D, dtype=torch.float64, device="cuda") for t in ("k", "v")}
        for t, new in (("k", state["key"]), ("v", state["value"])):
            for i in range(b):
                old, n = int(state["start"][i]) % BLOCK, int(state["counts"][i])
                for j in range(h):
                    x = torch.cat((state[t + "_tail"][i, j, :old], new[i, j, :n])).double()
                    whole = (old + n) // BLOCK * BLOCK
                    out[t][i, j, : old + n] = torch.cat((_exact_blocks(x[:whole], case["type"]), x[whole:]))
        return out
    if case["op"] == "attend":
        s, group = case["queries"], case["hq"] // h
        out = torch.zeros(b, case["hq"], s, D, dtype=torch.float64, device="cuda")
        lse = torch.zeros(b, case["hq"], s, dtype=torch.float64, device="cuda")
        sums = state["sums_out"].double() if case["weights"] else None
        for i in range(b):
            n = int(state["lengths"][i])
            hidden = torch.arange(n, device="cuda")[None, :] > torch.arange(n - s, n, device="cuda")[:, None]
            for j in range(h):
                k, v = _exact_tokens(state, "k", i, j), _exact_tokens(state, "v", i, j)
                if case["weights"]:
                    sums[i, j, :n] = state["sums"][i, j, :n].double()
                for g in range(j * group, (j + 1) * group):
                    a = (state["query"][i, g].double() @ k.T / math.sqrt(D)).masked_fill_(hidden, -math.inf)
                    lse[i, g] = torch.logsumexp(a, -1) / math.log(2)
                    a = torch.softmax(a, -1)
                    out[i, g] = a @ v
                    if case["weights"]:
                        sums[i, j, :n] += a.sum(0)
        return {"out": out, "sums": sums} if case["weights"] else {"out": out, "lse": lse}
    budget = case["budget"]
    if budget * b * h > 4 * 131072:
        return None
    out = {t: torch.zeros(b, h, budget, D, dtype=torch.float64, device="cuda") for t in ("k", "v")}
    sums = torch.zeros(b, h, budget, dtype=torch.float64, device="cuda")
    for i in range(b):
        n = int(state["lengths"][i])
        m = min(n, budget)
        for j in range(h):
            w = state["sums"][i, j, :n].double()
            forced = torch.zeros(n, dtype=torch.bool, device="cuda")
            forced[: state["sink"]] = True
            forced[max(0, n - state["recent"]):] = True
            rest = torch.nonzero(~forced).flatten()
            best = rest[torch.argsort(-w[rest], stable=True)[: m - int(forced.sum())]] if m < n else rest
            idx = torch.cat((torch.nonzero(forced).flatten(), best)).sort().values
            sums[i, j, :m] = w[idx]
            for t in ("k", "v"):
                x = _exact_tokens(state, t, i, j)[idx]
                whole = m // BLOCK * BLOCK
                out[t][i, j, :m] = torch.cat((_exact_blocks(x[:whole], case["type"]), x[whole:]))
    return {**out, "lengths": None, "sums": sums, "kept": None}

"""The paged latent cache of the MLA layers, as a serving program uses it around the decode step: new tokens are
appended, attended, their attention weight per cached position is accumulated, and sequences are cut down to the
positions that carry it. One case is one call of one operator.

Notation: T new tokens of B sequences (sequence b has the rows cu_new[b] .. cu_new[b + 1]), H heads, a cached
position is 512 latent values and 64 rope values, found through block_table[b][position // page_size]. Token i of
a sequence with n new tokens and L positions sees the first L - n + i + 1 of them.
"""

import math

import torch

own = False

LATENT, ROPE = 512, 64
DIMS = LATENT + ROPE
SCALE = 192 ** -0.5          # the model's (qk_nope_dim + qk_rope_dim) ** -0.5
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


# --- the cases -----------------------------------------------------------------------------------------------

def listed():
    return [
        # one decode step's new entries of a small batch: a launch and little else
        {"name": "append-step", "op": "append", "batch": 8, "new": 1, "length": 8192, "ragged": True, "page": 64},
        # a prompt chunk's entries of several sequences
        {"name": "append-chunk", "op": "append", "batch": 5, "new": 4096, "length": 4096, "ragged": True, "page": 16},
        # one token of one short sequence on one rank of eight: latency alone
        {"name": "attend-token", "op": "attend", "batch": 1, "new": 1, "heads": 12, "length": 517, "ragged": False, "page": 16},
        # one token each of a full batch on one rank of eight: the cache is read once
        {"name": "attend-batch", "op": "attend", "batch": 64, "new": 1, "heads": 12, "length": 8192, "ragged": False, "page": 64},
        # one token each on an unsharded model: 96 rows share each cached position
        {"name": "attend-heads", "op": "attend", "batch": 8, "new": 1, "heads": 96, "length": 8192, "ragged": True, "page": 64},
        # drafted tokens checked against caches of different lengths
        {"name": "attend-draft", "op": "attend", "batch": 8, "new": 5, "heads": 12, "length": 8000, "ragged": True, "page": 48},
        # a chunk of a long prompt on one rank of eight: bound by the products
        {"name": "attend-chunk", "op": "attend", "batch": 2, "new": 1024, "heads": 12, "length": 8192, "ragged": True, "page": 64},
        # whole prompts from empty caches: half of the scores are masked
        {"name": "attend-prompt", "op": "attend", "batch": 3, "new": 900, "heads": 24, "length": 900, "ragged": True, "page": 32},
        # the weight that one decode step's tokens put on each position
        {"name": "mass-step", "op": "mass", "batch": 16, "new": 1, "heads": 12, "length": 8192, "ragged": True, "page": 64},
        # the weight of a prompt's last tokens, the window that an eviction after the prompt looks at
        {"name": "mass-window", "op": "mass", "batch": 4, "new": 32, "heads": 96, "length": 8192, "ragged": True, "page": 64},
        # a short sequence cut down to a quarter
        {"name": "evict-short", "op": "evict", "batch": 1, "length": 1000, "budget": 250, "ragged": False, "page": 16},
        # a full batch's caches cut down to half, into pages of their own
        {"name": "evict-batch", "op": "evict", "batch": 16, "length": 8192, "budget": 4096, "ragged": True, "page": 64},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "mass", "evict"))
    page = rng.choice((8, 16, 32, 48, 64, 128, 10))
    while True:
        batch, length = _spread(rng, 1, 64), _spread(rng, 1, 16384)
        case = {"op": op, "batch": batch, "length": length, "ragged": rng.random() < 0.7, "page": page}
        if op == "evict":
            case["budget"] = max(1, min(length, int(length * rng.uniform(0.1, 1.1))))
        else:
            case["new"] = min(length, _spread(rng, 1, 2048) if rng.random() < 0.6 else rng.randint(1, 6))
        if op in ("attend", "mass"):
            case["heads"] = rng.choice((1, 6, 12, 12, 16, 24, 31, 48, 96))
        # the working set of the plain form stays small, and no case costs more than the largest listed ones
        w = work(case)
        padded = batch * length * (DIMS + case.get("new", 0) * case.get("heads", 0))
        if w["flops"] <= 3.2e11 and w["bytes"] <= 6.0e8 and padded <= 6.0e8:
            return case


# --- inputs --------------------------------------------------------------------------------------------------

def _lengths(case):
    """Host lists: new tokens and cached positions (the new ones included) of each sequence."""
    B, L = case["batch"], case["length"]
    n = case.get("new", 1)
    new, length = [], []
    for b in range(B):
        f = 1.0 if not case["ragged"] or b == 0 else 0.35 + 0.65 * ((b * 7919) % 97) / 97.0
        length.append(max(1, int(L * f)))
        new.append(max(1, min(length[-1], int(n * f) if n > 8 else n)))
    return new, length


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=gen, device="cuda") * std + mean).to(BF16)

    B, page = case["batch"], case["page"]
    new, length = _lengths(case)
    pages = [-(-x // page) for x in length]
    columns = max(pages)
    extra = 0
    if case["op"] == "evict":
        extra = B * -(-min(case["budget"], max(length)) // page)
    total = sum(pages) + extra
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((B, columns), dtype=torch.int32, device="cuda")
    at = 0
    for b in range(B):
        table[b, :pages[b]] = order[at:at + pages[b]]
        at += pages[b]
    s = {"op": case["op"], "page": page, "table": table, "columns": columns, "max_length": max(length),
         "kv": normal(total, page, LATENT), "pe": normal(total, page, ROPE),
         "lengths": torch.tensor(length, dtype=torch.int64, device="cuda")}
    if case["op"] == "evict":
        per = extra // B
        s["dst"] = order[at:].view(B, per).contiguous()
        s["budget"], s["sinks"] = case["budget"], min(4, case["budget"])
        s["recent"] = min(64, case["budget"] // 4)
        # a few heavy positions and a long tail, as attention leaves it; some exact ties
        weight = torch.randn((B, columns * page), generator=gen, device="cuda").mul(1.5).exp()
        s["mass"] = torch.where(torch.rand(weight.shape, generator=gen, device="cuda") < 0.1,
                                (weight * 4).round() / 4, weight)
        return s
    T = sum(new)
    starts = [0]
    for x in new:
        starts.append(starts[-1] + x)
    s["cu_new"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["tokens"], s["max_new"] = T, max(new)
    if case["op"] == "append":
        s["raw"] = normal(T, DIMS)
        s["norm"] = normal(LATENT, std=0.1, mean=1.0)
        s["before"] = s["lengths"] - (s["cu_new"][1:] - s["cu_new"][:-1])
        return s
    H = case["heads"]
    s["heads"] = H
    # absorbed queries: the product of a unit query's 128 values with kb's rows (std 512 ** -0.5)
    s["q_latent"], s["q_pe"] = normal(T, H, LATENT, std=0.5), normal(T, H, ROPE)
    if case["op"] == "mass":
        s["lse"] = _attend(s)[1]
        s["mass"] = torch.rand((B, columns * page), generator=gen, device="cuda")
    return s


# --- the plain forms -----------------------------------------------------------------------------------------

def _rows(s):
    """For each new token its sequence, its number within it, and the positions it sees."""
    cu = s["cu_new"].long()
    n = cu[1:] - cu[:-1]
    seq = torch.repeat_interleave(torch.arange(n.numel(), device=cu.device), n, output_size=s["tokens"])
    i = torch.arange(s["tokens"], device=cu.device) - cu[seq]
    return seq, i, s["lengths"][seq] - n[seq] + i + 1


def _scores(s):
    """Masked scores [B, max_new, H, positions], and the cached latents [B, positions, 512], both in 32 bits."""
    seq, i, sees = _rows(s)
    B, P = s["table"].shape[0], s["max_length"]
    at = torch.arange(P, device="cuda")
    slot = s["table"].long()[:, at // s["page"]] * s["page"] + at % s["page"]
    live = at < s["lengths"][:, None]
    kv = s["kv"].view(-1, LATENT)[slot].to(F32).masked_fill(~live[..., None], 0)
    pe = s["pe"].view(-1, ROPE)[slot].to(F32).masked_fill(~live[..., None], 0)
    q = torch.zeros((B, s["max_new"], s["heads"], DIMS), device="cuda")
    q[seq, i] = torch.cat((s["q_latent"], s["q_pe"]), -1).to(F32)
    limit = torch.zeros((B, s["max_new"]), dtype=torch.int64, device="cuda")
    limit[seq, i] = sees
    scores = q.flatten(1, 2) @ torch.cat((kv, pe), -1).transpose(1, 2) * SCALE
    scores = scores.view(B, s["max_new"], s["heads"], P)
    return scores.masked_fill_((at >= limit[..., None])[:, :, None], -math.inf), kv, seq, i


def _attend(s):
    scores, kv, seq, i = _scores(s)
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    p = (scores - top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(1, 2) @ kv).view(*p.shape[:3], LATENT) / total.clamp_min(1e-30)
    lse = (top + total.log())[..., 0]
    return out[seq, i].to(BF16), lse[seq, i]


def _mass(s):
    scores, _, seq, i = _scores(s)
    lse = torch.zeros(scores.shape[:3], device="cuda")
    lse[seq, i] = s["lse"]
    weight = (scores - lse[..., None]).exp_().sum((1, 2))
    out = s["mass"].clone()
    out[:, :s["max_length"]] += weight
    return out


def _append(s):
    seq, i, _ = _rows(s)
    x = s["raw"].to(F32)
    latent = x[:, :LATENT]
    latent = latent * torch.rsqrt(latent.square().mean(-1, keepdim=True) + 1e-6) * s["norm"].to(F32)
    at = s["before"][seq] + i
    slot = s["table"].long()[seq, at // s["page"]] * s["page"] + at % s["page"]
    s["kv"].view(-1, LATENT)[slot] = latent.to(BF16)
    s["pe"].view(-1, ROPE)[slot] = s["raw"][:, LATENT:]
    return s["before"] + (s["cu_new"][1:] - s["cu_new"][:-1])


def _evict(s):
    length, budget = s["lengths"][:, None], s["budget"]
    at = torch.arange(s["mass"].shape[1], device="cuda")
    key = s["mass"].masked_fill((at < s["sinks"]) | (at >= length - s["recent"]), math.inf)
    key = key.masked_fill(at >= length, -math.inf)
    first = key.sort(dim=1, descending=True, stable=True).indices[:, :budget]
    count = length.clamp_max(budget)
    rank = torch.arange(first.shape[1], device="cuda")
    kept = first.masked_fill(rank >= count, 1 << 40).sort(1).values
    live = rank < count
    seq, j = live.nonzero(as_tuple=True)
    src = kept[seq, j]
    table, dst, page = s["table"].long(), s["dst"].long(), s["page"]
    a, b = table[seq, src // page] * page + src % page, dst[seq, j // page] * page + j % page
    kv, pe = s["kv"].view(-1, LATENT), s["pe"].view(-1, ROPE)
    kv[b], pe[b] = kv[a], pe[a]
    mass = torch.zeros_like(s["mass"])
    mass[seq, j] = s["mass"][seq, src]
    out = torch.full((table.shape[0], budget), -1, dtype=torch.int32, device="cuda")
    out[seq, j] = src.to(torch.int32)
    return count[:, 0], mass, out


def run(s):
    """One call of one operator. What is cut down or appended goes to the state's pages, which are returned."""
    op = s["op"]
    if own:
        from kimi_k3_goalbox_b200 import latent_cache as lc
        cache = (s["kv"], s["pe"], s["table"])
        if op == "append":
            return {"lengths": lc.append(s["raw"], s["norm"], *cache, s["before"], s["cu_new"]), "kv": s["kv"], "pe": s["pe"]}
        if op == "attend":
            out, lse = lc.attend(s["q_latent"], s["q_pe"], *cache, s["lengths"], s["cu_new"])
            return {"out": out, "lse": lse}
        if op == "mass":
            return {"mass": lc.attention_mass(s["q_latent"], s["q_pe"], s["lse"], *cache, s["lengths"], s["cu_new"],
                                              mass=s["mass"])}
        lengths, mass, kept = lc.evict(*cache, s["lengths"], s["mass"], s["budget"], sinks=s["sinks"],
                                       recent=s["recent"], dst_table=s["dst"])
        return {"lengths": lengths, "mass": mass, "kept": kept, "kv": s["kv"], "pe": s["pe"]}
    if op == "append":
        return {"lengths": _append(s), "kv": s["kv"], "pe": s["pe"]}
    if op == "attend":
        out, lse = _attend(s)
        return {"out": out, "lse": lse}
    if op == "mass":
        return {"mass": _mass(s)}
    lengths, mass, kept = _evict(s)
    return {"lengths": lengths, "mass": mass, "kept": kept, "kv": s["kv"], "pe": s["pe"]}


# --- what the path cannot do without --------------------------------------------------------------------------

def work(case):
    new, length = _lengths(case)
    B, T, entry = case["batch"], sum(new), 2 * DIMS
    if case["op"] == "append":      # the rows in, the entries out, the norm's weight
        return {"bytes": 2 * T * entry + 2 * LATENT, "flops": 4 * T * LATENT}
    if case["op"] == "evict":       # each position's weight once, each kept entry in and out, and its new weight and number
        kept = sum(min(x, case["budget"]) for x in length)
        return {"bytes": 4 * sum(length) + kept * (2 * entry + 8), "flops": sum(length)}
    H = case["heads"]
    # token i sees length - new + i + 1 positions
    pairs = sum(n * (x - n) + n * (n + 1) // 2 for n, x in zip(new, length))
    if case["op"] == "mass":        # the queries and the cache in, the accumulated weights in and out
        return {"bytes": T * H * (entry + 4) + sum(length) * (entry + 8), "flops": 2 * pairs * H * DIMS}
    return {"bytes": T * H * (entry + 2 * LATENT + 4) + sum(length) * entry, "flops": 2 * pairs * H * (DIMS + LATENT)}


# --- the definition in 64 bits -------------------------------------------------------------------------------

def _entries(s, b, count):
    """The first `count` cached positions of sequence b, in 64 bits."""
    page = s["page"]
    ids = s["table"][b, :-(-count // page)].long()
    kv = s["kv"][ids].reshape(-1, LATENT)[:count].to(F64)
    return kv, s["pe"][ids].reshape(-1, ROPE)[:count].to(F64)


def exact(case, seed):
    s = prepare(case, seed)
    B = case["batch"]
    lengths = s["lengths"].tolist()
    if case["op"] == "evict":
        page, budget = s["page"], s["budget"]
        kv, pe = s["kv"].clone(), s["pe"].clone()
        mass, kept = torch.zeros_like(s["mass"], dtype=F64), torch.full((B, budget), -1, dtype=torch.int32)
        weights, table, dst = s["mass"].tolist(), s["table"].tolist(), s["dst"].tolist()
        for b in range(B):
            n = lengths[b]
            must = [p for p in range(n) if p < s["sinks"] or p >= n - s["recent"]]
            free = sorted((p for p in range(s["sinks"], n - s["recent"])), key=lambda p: (-weights[b][p], p))
            if n <= budget:
                chosen = list(range(n))
            else:
                chosen = sorted(must + free[:budget - len(must)])
            src = torch.tensor([table[b][p // page] * page + p % page for p in chosen], device="cuda")
            to = torch.tensor([dst[b][j // page] * page + j % page for j in range(len(chosen))], device="cuda")
            kv.view(-1, LATENT)[to] = s["kv"].view(-1, LATENT)[src]
            pe.view(-1, ROPE)[to] = s["pe"].view(-1, ROPE)[src]
            mass[b, :len(chosen)] = s["mass"][b].double()[torch.tensor(chosen, device="cuda")]
            kept[b, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
        return {"lengths": torch.tensor([min(n, budget) for n in lengths]), "mass": mass, "kept": kept.cuda(),
                "kv": kv.to(F64), "pe": pe.to(F64)}
    starts = s["cu_new"].tolist()
    if case["op"] == "append":
        kv, pe, page = s["kv"].to(F64), s["pe"].to(F64), s["page"]
        for b in range(B):
            x = s["raw"][starts[b]:starts[b + 1]].to(F64)
            norm = (x[:, :LATENT].pow(2).sum(1, keepdim=True) / LATENT + 1e-6).sqrt()
            first = lengths[b] - len(x)
            slots = torch.arange(first, lengths[b], device="cuda")
            slots = s["table"][b].long()[slots.div(page, rounding_mode="floor")] * page + slots.remainder(page)
            kv.view(-1, LATENT)[slots] = x[:, :LATENT] / norm * s["norm"].to(F64)
            pe.view(-1, ROPE)[slots] = x[:, LATENT:]
        return {"lengths": s["lengths"], "kv": kv, "pe": pe}
    out, lses = [], []
    mass = s["mass"].to(F64) if case["op"] == "mass" else None
    for b in range(B):
        n = starts[b + 1] - starts[b]
        kv, pe = _entries(s, b, lengths[b])
        rows = slice(starts[b], starts[b + 1])
        step = max(1, int(4e7 // (case["heads"] * lengths[b])))   # tokens at a time
        for t in range(0, n, step):
            some = slice(rows.start + t, min(rows.start + t + step, rows.stop))
            score = (torch.einsum("thd,pd->thp", s["q_latent"][some].to(F64), kv)
                     + torch.einsum("thd,pd->thp", s["q_pe"][some].to(F64), pe)) * SCALE
            sees = lengths[b] - n + 1 + torch.arange(t, t + score.shape[0], device="cuda")
            hidden = torch.arange(lengths[b], device="cuda")[None] >= sees[:, None]
            score = torch.where(hidden[:, None], torch.full((), -math.inf, dtype=F64, device="cuda"), score)
            if mass is not None:
                mass[b, :lengths[b]] += torch.exp(score - s["lse"][some].to(F64)[..., None]).sum((0, 1))
            else:
                lse = torch.logsumexp(score, -1)
                out.append(torch.einsum("thp,pd->thd", torch.exp(score - lse[..., None]), kv))
                lses.append(lse)
    return {"mass": mass} if mass is not None else {"out": torch.cat(out), "lse": torch.cat(lses)}

"""What one step of many requests at once needs beside its products, as cases that can be timed and compared.

  attend  the new tokens of several sequences are written into a paged cache held in 4 bits, then attend over it
  sample  one token per row of logits, by temperature, top-k, top-p and min-p, from given uniform numbers
  adapt   every row's own low-rank adapter, added to the rows that a shared projection gave

Each has a plain form (elementary torch operations) and the calls that a user makes of this library.
"""
import math

import torch

own = False

GPU = torch.device("cuda")
F4, F8 = torch.float32, torch.float64
GROUP = 64      # values of a cached row that share a scale and a least value
PAGE = 16       # tokens of a page
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one request of the small dense decoder: the smallest call, where latency counts
        {"name": "attend_one", "kind": "attend", "type": "f32", "heads": 16, "kv": 8, "dim": 128, "seqs": 1, "context": 512, "count": 1, "prompt": 0},
        # a step of sixteen requests of the mixture-of-experts decoder, of all lengths
        {"name": "attend_streams", "kind": "attend", "type": "f32", "heads": 32, "kv": 4, "dim": 128, "seqs": 16, "context": 2300, "count": 1, "prompt": 0},
        # many requests with long caches: what four bits are for
        {"name": "attend_long", "kind": "attend", "type": "bf16", "heads": 32, "kv": 4, "dim": 128, "seqs": 48, "context": 32000, "count": 1, "prompt": 0},
        # four drafted tokens and the last one of four requests, heads of 64
        {"name": "attend_verify", "kind": "attend", "type": "f32", "heads": 24, "kv": 4, "dim": 64, "seqs": 4, "context": 1531, "count": 5, "prompt": 0},
        # a whole prompt whose length is no multiple of anything
        {"name": "attend_prompt", "kind": "attend", "type": "bf16", "heads": 32, "kv": 4, "dim": 128, "seqs": 1, "context": 0, "count": 1, "prompt": 2011},
        # a later chunk of a long prompt beside three requests that decode
        {"name": "attend_chunk", "kind": "attend", "type": "bf16", "heads": 16, "kv": 8, "dim": 128, "seqs": 4, "context": 6001, "count": 1, "prompt": 512},
        # the end of a step of one request, with the settings that servers have by default
        {"name": "sample_one", "kind": "sample", "type": "f32", "rows": 1, "vocab": 151936, "filter": "k50p95", "dist": False},
        # sixteen requests, each with settings of its own
        {"name": "sample_mixed", "kind": "sample", "type": "f32", "rows": 16, "vocab": 151936, "filter": "mixed", "dist": False},
        # the largest batch, nucleus sampling alone; the distributions are kept for a later verification
        {"name": "sample_many", "kind": "sample", "type": "bf16", "rows": 256, "vocab": 151936, "filter": "p90", "dist": True},
        # one request with an adapter on the fused query, key and value projection
        {"name": "adapt_one", "kind": "adapt", "type": "bf16", "rows": 1, "K": 2048, "N": 5120, "adapters": 8, "rank": 16},
        # a step of many requests, each with its own of many adapters
        {"name": "adapt_many", "kind": "adapt", "type": "bf16", "rows": 64, "K": 2048, "N": 4096, "adapters": 48, "rank": 32},
        # prompts of a few adapters
        {"name": "adapt_prompts", "kind": "adapt", "type": "f16", "rows": 2011, "K": 2048, "N": 6144, "adapters": 4, "rank": 64},
    ]


def spread(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "sample", "sample", "adapt", "adapt"])
    if kind == "sample":
        case = {"kind": kind, "type": rng.choice(["f32", "f32", "bf16"]), "rows": spread(rng, 1, 256), "vocab": spread(rng, 90, 262144),
                "filter": rng.choice(["mixed", "mixed", "k50p95", "p90", "all"]), "dist": rng.random() < 0.3}
        return case
    if kind == "adapt":
        rank = spread(rng, 1, 128)
        return {"kind": kind, "type": rng.choice(["bf16", "f16"]), "rows": spread(rng, 1, 2048), "K": 8 * spread(rng, 8, 1024), "N": spread(rng, 60, 8192),
                "adapters": spread(rng, 1, max(1, min(64, 2048 // rank))), "rank": rank}
    kv = rng.choice([1, 2, 4, 8])
    case = {"kind": kind, "type": rng.choice(["f32", "bf16"]), "heads": kv * rng.choice([1, 2, 3, 4, 6, 8, 8, 12, 16] if kv < 8 else [1, 2, 4]), "kv": kv,
            "dim": rng.choice([64, 128, 128]), "seqs": 1, "context": 0, "count": 1, "prompt": 0}
    how = rng.choice(["decode", "decode", "verify", "prompt"])
    if how == "prompt":
        case["prompt"] = spread(rng, 9, 2048)
        case["context"] = rng.choice([0, spread(rng, 1, 6000)])
        case["seqs"] = rng.choice([1, 1, 2, 4])
    else:
        case["count"] = 1 if how == "decode" else rng.randint(2, 8)
        case["seqs"] = spread(rng, 1, 48)
        case["context"] = spread(rng, 1, min(32000, 1500000 // case["seqs"] // case["count"]))
    return case


# -------------------------------------------------------------------------------------------- seeded values
class Values:
    """Random values on the GPU; every name has a stream of its own."""

    def __init__(self, seed):
        self.seed = seed

    def of(self, name):
        h = 2166136261
        for b in ("%d/%s" % (self.seed, name)).encode():
            h = (h ^ b) * 16777619 % (1 << 32)
        return torch.Generator(GPU).manual_seed(h)

    def normal(self, name, *shape):
        return torch.randn(*shape, generator=self.of(name), device=GPU)

    def uniform(self, name, *shape):
        return torch.rand(*shape, generator=self.of(name), device=GPU)

    def below(self, name, hi, *shape):
        return torch.randint(0, hi, shape, generator=self.of(name), device=GPU)


# ---------------------------------------------------------------------------- attention over a cache in 4 bits
# A cached row of a key head (or value head) is held in groups of 64 values.  A group has
#   m = fp16(least value)     d = fp16((largest - least) * fp32(1 / 15))
#   codes q_i = rint((x_i - m) / d) within 0..15, in fp32 (0 where d is 0)
# and stands for fp32(d q_i + m).  Token at position p of a sequence sees the cached rows 0..p of it, its own among them.
def lengths(case):
    """(tokens before the step, new tokens) of every sequence."""
    before = [case["context"]] + [max(0, round(case["context"] * (0.2 + 0.8 * math.modf(0.618034 * e)[0]))) for e in range(1, case["seqs"])]
    new = [case["prompt"] or case["count"]] + [case["count"]] * (case["seqs"] - 1)
    return before, new


def pack(x):
    """x [..., dim] -> codes [..., dim / 2] (two of neighbouring values to a byte), scales and least values [..., dim / 64]."""
    g = x.float().unflatten(-1, (-1, GROUP))
    least, most = g.amin(-1), g.amax(-1)
    m, d = least.half(), ((most - least) * torch.tensor(1.0 / 15.0, device=GPU)).half()
    step = d.float()[..., None]
    q = torch.where(step > 0, torch.round((g - m.float()[..., None]) / step), 0.0).clamp(0, 15).to(torch.uint8).flatten(-2)
    return q[..., 0::2] | (q[..., 1::2] << 4), d, m


def unpack(codes, d, m):
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, GROUP))
    # d q is exact in 32 bits (11 and 4 bits), so that the sum is rounded once
    return (q.float() * d.float()[..., None] + m.float()[..., None]).flatten(-2)


def attend_inputs(case, seed):
    """New rows, the rows that the caches hold (one sequence's after the other's) and the softmax' scale."""
    v, t = Values(seed), TYPES[case["type"]]
    before, new = lengths(case)
    T, kv, dim = sum(new), case["kv"], case["dim"]
    # keys have a few dimensions that are larger and off zero, as rotary keys have; scores spread over a few units
    shape = 0.4 + 0.2 * v.normal("shape", kv, dim).abs() + 2.0 * (v.uniform("big", kv, dim) < 0.03)
    shift = 1.5 * v.normal("shift", kv, dim) * (v.uniform("off", kv, dim) < 0.05)
    def keys(name, n):
        return (v.normal(name, n, kv, dim).mul_(shape).add_(shift)).to(t)
    return {"q": (2.0 * v.normal("q", T, case["heads"], dim)).to(t), "k": keys("k", T), "v": (0.7 * v.normal("v", T, kv, dim)).to(t),
            "old_k": keys("old_k", sum(before)), "old_v": (0.7 * v.normal("old_v", sum(before), kv, dim)).to(t), "scale": dim ** -0.5}


def places(before, new):
    """Sequence and position of every token that `before` .. `before + new` names, and of every page its sequence needs."""
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))
    first = torch.cumsum(torch.tensor([0] + new), 0)[:-1]
    pos = torch.arange(sum(new)) - first[seq] + torch.tensor(before)[seq]
    return seq.to(GPU), pos.to(GPU)


class Cache:
    """The plain form's cache: pages of 16 tokens in any order and a table of them for each sequence."""

    def __init__(self, case, seed):
        before, new = lengths(case)
        need = [-(-(a + b) // PAGE) for a, b in zip(before, new)]
        ids = torch.randperm(sum(need), generator=torch.Generator().manual_seed(seed % (1 << 31)))
        self.table = torch.zeros(len(need), max(need), dtype=torch.long)
        self.table[torch.arange(max(need))[None] < torch.tensor(need)[:, None]] = ids
        self.table = self.table.to(GPU)
        shape = (sum(need), PAGE, case["kv"])
        self.k, self.v = ([torch.zeros(*shape, n, dtype=t, device=GPU) for n, t in ((case["dim"] // 2, torch.uint8), (case["dim"] // GROUP, torch.half), (case["dim"] // GROUP, torch.half))] for _ in "kv")
        self.case = case

    def write(self, seq, pos, k, v):
        page, slot = self.table[seq, pos // PAGE], pos % PAGE
        for to, x in ((self.k, k), (self.v, v)):
            for part, y in zip(to, pack(x)):
                part[page, slot] = y

    def rows(self, seq, pos):
        page, slot = self.table[seq, pos // PAGE], pos % PAGE
        return [unpack(*(part[page, slot] for part in held)) for held in (self.k, self.v)]

    def sequences(self):
        """Keys and values of all sequences, [sequence, position, head, dim], to the length of the longest."""
        return [unpack(*(part[self.table].flatten(1, 2) for part in held)) for held in (self.k, self.v)]


def attend_plain(s):
    case, cache, seq, pos = s["case"], s["cache"], s["seq"], s["pos"]
    cache.write(seq, pos, s["k"], s["v"])
    K, V = cache.sequences()
    # queries [sequence, place, head, dim], padded to the largest number of new tokens
    most, place = s["most"], s["place"]
    q = torch.zeros(case["seqs"], most, case["kv"], case["heads"] // case["kv"], case["dim"], device=GPU)
    q[seq, place] = s["q"].float().unflatten(1, (case["kv"], -1))
    last = torch.full((case["seqs"], most), -1, device=GPU)
    last[seq, place] = pos
    z = torch.einsum("scigd,spid->scigp", q, K) * s["scale"]
    z = z.masked_fill(torch.arange(K.shape[1], device=GPU) > last[:, :, None, None, None], -math.inf)
    w = torch.exp(z - z.amax(-1, keepdim=True).clamp(min=-3e38))
    y = torch.einsum("scigp,spid->scigd", w, V) / w.sum(-1)[..., None]
    held = cache.rows(seq, pos)
    return {"out": y[seq, place].flatten(1, 2).to(TYPES[case["type"]]), "k": held[0], "v": held[1]}


def attend_exact(case, seed):
    """Sequence by sequence and some heads at a time, in 64 bits; the codes by the definition's steps."""
    x = attend_inputs(case, seed)
    before, new = lengths(case)
    if sum(n * (b + n) for b, n in zip(before, new)) * case["heads"] * case["dim"] > 2e11:
        return None
    def held(rows):
        out = torch.empty(rows.shape, dtype=F8, device=GPU)
        for c in range(0, rows.shape[-1], GROUP):
            g = rows[..., c:c + GROUP].to(F4)
            lo, hi = g.min(-1, keepdim=True)[0], g.max(-1, keepdim=True)[0]
            m, d = lo.to(torch.float16).to(F4), ((hi - lo) * (torch.ones_like(lo) / 15)).to(torch.float16).to(F4)
            codes = torch.where(d > 0, (g - m) / d, torch.zeros_like(g)).round().clamp(0.0, 15.0)
            out[..., c:c + GROUP] = codes.to(F8) * d.to(F8) + m.to(F8)
        return out
    y, at, old = torch.empty(x["q"].shape, dtype=F8, device=GPU), 0, 0
    nk, nv, G = held(x["k"]), held(x["v"]), case["heads"] // case["kv"]
    for b, n in zip(before, new):
        for i in range(case["kv"]):
            K = torch.cat([held(x["old_k"][old:old + b, i]), nk[at:at + n, i]])
            V = torch.cat([held(x["old_v"][old:old + b, i]), nv[at:at + n, i]])
            for h in range(i * G, i * G + G):
                z = x["q"][at:at + n, h].to(F8) @ K.T * x["scale"]
                z = z.masked_fill(torch.ones(n, b + n, dtype=torch.bool, device=GPU).triu(b + 1), -math.inf)
                y[at:at + n, h] = torch.softmax(z, -1) @ V
        at, old = at + n, old + b
    return {"out": y, "k": nk, "v": nv}


def attend_work(case):
    before, new = lengths(case)
    T, total = sum(new), sum(before) + sum(new)
    size = TYPES[case["type"]].itemsize
    row = case["dim"] / 2 + 4 * (case["dim"] // GROUP)      # bytes of a cached key or value
    seen = sum(n * b + n * (n + 1) // 2 for b, n in zip(before, new))
    io = T * case["dim"] * (2 * case["heads"] + 2 * case["kv"]) * size + 2 * T * case["kv"] * case["dim"] * 4
    return {"bytes": 2 * case["kv"] * row * (total + T) + io, "flops": 4 * seen * case["heads"] * case["dim"]}


# --------------------------------------------------------------------------------------------------- sampling
# The order of a row's tokens is by falling logit, equal ones by rising index.  Kept is a beginning of that order: at
# most top_k (0: any number); of these the shortest beginning that holds a share top_p of their weights
# exp((logit - largest) / temperature); of these the ones with weights of min_p at least; the first one always.  The draw is the
# first kept token, by index, up to which the kept weights' sum is above uniform times their whole sum.  Temperature
# 0 takes the first of the order.  -inf and NaN have no weight; a row without any weight gives -1.
def sample_inputs(case, seed):
    v, rows, V = Values(seed), case["rows"], case["vocab"]
    # probabilities fall with a power of the rank, differently steep by row, in another order each; some rows have a grammar's mask
    order = v.uniform("order", rows, V).argsort(-1)
    steep = 1.0 + 1.2 * v.uniform("steep", rows, 1)
    x = 9.0 - steep * torch.log(torch.arange(1, V + 1, device=GPU).float())[None] + 0.4 * v.normal("noise", rows, V)
    x = torch.empty_like(x).scatter_(1, order, x)
    barred = (v.uniform("barred", rows, V) < 0.6) & (v.uniform("rule", rows, 1) < 0.25)
    x = x.masked_fill(barred, -math.inf).to(TYPES[case["type"]])
    def pick(name, *of):
        return torch.tensor(of, device=GPU)[v.below(name, len(of), rows)]
    one = torch.ones(rows, device=GPU)
    how = {"mixed": lambda: (pick("t", 0.7, 0.7, 1.0, 1.3, 0.0), pick("k", 0, 20, 50, 400), pick("p", 1.0, 0.9, 0.95, 0.5), pick("m", 0.0, 0.0, 0.05, 0.1)),
           "k50p95": lambda: (0.8 * one, (50 * one).long(), 0.95 * one, 0 * one), "p90": lambda: (one, (0 * one).long(), 0.9 * one, 0 * one),
           "all": lambda: (one, (0 * one).long(), one, 0 * one)}[case["filter"]]()
    return {"logits": x, "temperature": how[0].float(), "top_k": how[1].int(), "top_p": how[2].float(), "min_p": how[3].float(), "u": v.uniform("u", rows)}


def sample_plain(s):
    # in 64 bits throughout: a uniform number next to a border of two tokens decides between them
    x = s["logits"].double()
    x = torch.where(x.isnan(), -math.inf, x)
    V, greedy = x.shape[1], s["temperature"] == 0
    far = x - x.amax(-1, keepdim=True).clamp(min=-1e300)
    w = torch.exp(far / torch.where(greedy, 1.0, s["temperature"].double())[:, None])
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1]
    place = torch.arange(V, device=GPU)[None]
    k = torch.where(greedy, 1, torch.where(s["top_k"] > 0, s["top_k"], V))[:, None]
    ranked = w.gather(1, order) * (place < k)
    ahead = torch.cumsum(ranked, 1) - ranked
    inside = (ahead < s["top_p"].double()[:, None] * ranked.sum(1, keepdim=True)) | (s["top_p"][:, None] >= 1)
    kept = (place == 0) | ((place < k) & inside & (ranked >= s["min_p"].double()[:, None]))
    kept = torch.zeros_like(kept).scatter_(1, order, kept)
    w = w * kept
    upto, whole = torch.cumsum(w, 1), w.sum(1, keepdim=True)
    token = (upto <= s["u"].double()[:, None] * whole).sum(1).clamp(max=V - 1)
    p = w / whole
    some = whole[:, 0] > 0
    out = {"token": torch.where(some, token, -1).int(), "p": torch.where(some, p.gather(1, token[:, None])[:, 0], 0.0).float()}
    if s["case"]["dist"]:
        out["dist"] = torch.where(some[:, None], p, 0.0).float()
    return out


def sample_exact(case, seed):
    """Row by row."""
    s = sample_inputs(case, seed)
    share, dist = [], torch.zeros(case["rows"], case["vocab"], dtype=F8, device=GPU)
    for r in range(case["rows"]):
        x, T = s["logits"][r].to(F8), float(s["temperature"][r])
        value, index = x.sort(descending=True, stable=True)
        n = 1 if T == 0 else int(s["top_k"][r]) or case["vocab"]
        weight = ((value[:n] - value[0]) / (T or 1.0)).exp()
        if float(s["top_p"][r]) < 1:
            reached = (weight.cumsum(0) >= float(s["top_p"][r]) * weight.sum()).nonzero()
            weight = weight[:int(reached[0]) + 1]
        weight = weight[:max(1, int((weight >= float(s["min_p"][r])).sum()))]
        index, by_index = index[:len(weight)].sort()
        weight = weight[by_index] / weight.sum()
        at = int((weight.cumsum(0) <= float(s["u"][r])).sum())
        share.append(float(weight[min(at, len(weight) - 1)]))
        dist[r, index] = weight
    out = {"token": None, "p": torch.tensor(share, dtype=F8)}
    if case["dist"]:
        out["dist"] = dist
    return out


# --------------------------------------------------------------------------------------------------- adapters
# y[t] = base[t] + s_a (x[t] A_a^T) B_a^T with a = ids[t]; A_a [rank_a, K], B_a [N, rank_a]; ids of -1: y[t] = base[t].
def adapt_inputs(case, seed):
    v, t, n, r = Values(seed), TYPES[case["type"]], case["adapters"], case["rank"]
    ranks = [max(1, r // (1 + e % 3)) for e in range(n)]     # not all adapters are of the largest rank
    within = torch.arange(r, device=GPU)[None] < torch.tensor(ranks, device=GPU)[:, None]
    A = (v.normal("A", n, r, case["K"]) * case["K"] ** -0.5 * within[:, :, None]).to(t)
    B = (0.05 * v.normal("B", n, case["N"], r) * within[:, None, :]).to(t)
    ids = v.below("ids", n + 1, case["rows"]) - 1            # a row in n + 1 has none
    if case["rows"] > 256:                                   # prompts: rows of one request follow one another
        ids = ids[torch.arange(case["rows"], device=GPU) // 173 * 173]
    return {"x": v.normal("x", case["rows"], case["K"]), "base": v.normal("base", case["rows"], case["N"]), "ids": ids.int(), "A": A, "B": B, "ranks": ranks,
            "scales": [2.0 / (1 + e % 4) for e in range(n)]}


def adapt_plain(s):
    n, r = s["A"].shape[:2]
    # all adapters at once; a row keeps what its own gave
    mine = s["ids"][:, None] == torch.arange(n, device=GPU)
    h = (s["x"] @ s["A"].float().flatten(0, 1).T).unflatten(1, (n, r)) * (mine * s["factors"])[:, :, None]
    return s["base"] + h.flatten(1) @ s["B"].float().transpose(0, 1).flatten(1).T


def adapt_exact(case, seed):
    s = adapt_inputs(case, seed)
    y = s["base"].to(F8)
    for a in range(case["adapters"]):
        t = (s["ids"] == a).nonzero()[:, 0]
        y[t] += s["scales"][a] * (s["x"][t].to(F8) @ s["A"][a].to(F8).T @ s["B"][a].to(F8).T)
    return y


def adapt_work(case):
    n, r = case["adapters"], case["rank"]
    ranks = [max(1, r // (1 + e % 3)) for e in range(n)]
    used = n * (1 - (1 - 1 / (n + 1)) ** (case["rows"] if case["rows"] <= 256 else -(-case["rows"] // 173)))      # adapters that some row names, on average
    mean, rows = sum(ranks) / n, case["rows"]
    return {"bytes": used * mean * (case["K"] + case["N"]) * 2 + rows * (case["K"] + 2 * case["N"]) * 4, "flops": 2 * rows * n / (n + 1) * mean * (case["K"] + case["N"])}


# ------------------------------------------------------------------------------------------ this library's calls
_ctx = None


def context():
    """One context for all, as a program has."""
    global _ctx
    if _ctx is None:
        import densecore_b200 as dc
        _ctx = dc.Context(0)
    return _ctx


def own_cache(s):
    """The library's cache with the tokens before the step, and the step's batch."""
    case, ctx = s["case"], context()
    before, new = lengths(case)
    pages = [-(-(a + b) // PAGE) for a, b in zip(before, new)]
    kv = ctx.kv_cache_q4(1, case["heads"], case["kv"], case["dim"], sum(pages), case["seqs"], max(pages), dtype=case["type"])
    seqs = [kv.seq_alloc() for _ in before]
    torch.cuda.synchronize()
    if sum(before):
        kv.batch(seqs, [0] * len(seqs), before)
        kv.write_dev(0, s["old_k"].data_ptr(), s["old_v"].data_ptr())
    kv.batch(seqs, before, new)
    ctx.synchronize()
    s["kv"] = kv
    s["held"] = [torch.empty(sum(new), case["kv"], case["dim"], device=GPU) for _ in "kv"]
    s["out"] = torch.empty_like(s["q"])


def attend_own(s):
    k, v = s["held"]
    s["kv"].attend_dev(0, s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["scale"], s["out"].data_ptr(), k_held=k.data_ptr(), v_held=v.data_ptr())
    return {"out": s["out"], "k": k, "v": v}


def sample_own(s):
    case = s["case"]
    context().sample_rows_dev(s["logits"].data_ptr(), case["rows"], case["vocab"], s["temperature"].data_ptr(), s["top_k"].data_ptr(), s["top_p"].data_ptr(), s["min_p"].data_ptr(),
                              s["u"].data_ptr(), s["token"].data_ptr(), p=s["p"].data_ptr(), dist=s["dist"].data_ptr() if case["dist"] else 0, dtype=case["type"])
    return {"token": s["token"], "p": s["p"], **({"dist": s["dist"]} if case["dist"] else {})}


def own_adapters(s):
    case = s["case"]
    s["set"] = context().lora(case["K"], case["N"], case["adapters"], case["rank"], dtype=case["type"])
    for a, rank in enumerate(s["ranks"]):
        A, B = s["A"][a, :rank].contiguous(), s["B"][a, :, :rank].contiguous()
        torch.cuda.synchronize()
        s["set"].set_dev(a, rank, A.data_ptr(), B.data_ptr(), s["scales"][a])
        context().synchronize()
    s["y"] = torch.empty_like(s["base"])


def adapt_own(s):
    context().lora_add_dev(s["set"], s["x"].data_ptr(), s["case"]["rows"], s["ids"].data_ptr(), s["y"].data_ptr(), base_dev=s["base"].data_ptr())
    return s["y"]


# ------------------------------------------------------------------------------------------------ what is asked
def prepare(case, seed):
    kind = case["kind"]
    if kind == "attend":
        s = attend_inputs(case, seed)
        before, new = lengths(case)
        s["seq"], s["pos"] = places(before, new)
        s["most"], s["place"] = max(new), s["pos"] - torch.tensor(before, device=GPU)[s["seq"]]
    elif kind == "sample":
        s = sample_inputs(case, seed)
    else:
        s = adapt_inputs(case, seed)
        s["factors"] = torch.tensor(s["scales"], device=GPU)
    s["case"] = case
    # what a program keeps between calls, on either side: the cache that holds the earlier tokens, the adapters' handle, results' buffers
    if kind == "attend":
        if own:
            own_cache(s)
        else:
            s["cache"] = Cache(case, seed)
            s["cache"].write(*places([0] * case["seqs"], before), s["old_k"], s["old_v"])
        del s["old_k"], s["old_v"]
    elif own and kind == "sample":
        rows = case["rows"]
        s["token"], s["p"] = torch.empty(rows, dtype=torch.int32, device=GPU), torch.empty(rows, device=GPU)
        s["dist"] = torch.empty(rows, case["vocab"], device=GPU) if case["dist"] else None
    elif own:
        own_adapters(s)
    torch.cuda.synchronize()
    return s


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attend": attend_own, "sample": sample_own, "adapt": adapt_own}[kind](state)
    return {"attend": attend_plain, "sample": sample_plain, "adapt": adapt_plain}[kind](state)


def exact(case, seed):
    return {"attend": attend_exact, "sample": sample_exact, "adapt": adapt_exact}[case["kind"]](case, seed)


def work(case):
    if case["kind"] == "attend":
        return attend_work(case)
    if case["kind"] == "adapt":
        return adapt_work(case)
    size = TYPES[case["type"]].itemsize
    return {"bytes": case["rows"] * case["vocab"] * (size + (4 if case["dist"] else 0)) + 28 * case["rows"], "flops": 4 * case["rows"] * case["vocab"]}

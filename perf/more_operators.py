"""What steps of many requests need that follow one another on the GPU without the host, as cases that can be timed and compared.

  pages   block tables, slots and positions of a step's new tokens from the requests' lengths: drafted tokens that were rejected go, new ones get places
  attend  the new tokens of several sequences are written into a paged cache of 16-bit rows, then attend over it, wholly or over a window and the first tokens
  verify  the drafted tokens of many requests against the target's probabilities, and each request's next token, from given uniform numbers

Each has a plain form (elementary torch operations) and the calls that a user makes of this library.
"""
import math

import torch

own = False

GPU = torch.device("cuda")
F4, F8 = torch.float32, torch.float64
PAGE = 16       # tokens of a page
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ALL = 2**31 - 1


# ------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # sixteen requests with four drafts each, whose rejected tokens then go: the smallest call, where latency counts
        {"name": "pages_verify", "kind": "pages", "slots": 16, "longest": 2300, "count": 5, "admit": False},
        # all of many slots are given to new requests at once, with prompts of all lengths
        {"name": "pages_admit", "kind": "pages", "slots": 512, "longest": 8192, "count": 0, "admit": True},
        # one request of the small dense decoder
        {"name": "attend_one", "kind": "attend", "type": "f32", "heads": 16, "kv": 8, "dim": 128, "seqs": 1, "context": 512, "count": 1, "prompt": 0, "window": 0, "keep": 0},
        # a step of sixteen requests of the mixture-of-experts decoder, of all lengths
        {"name": "attend_streams", "kind": "attend", "type": "f32", "heads": 32, "kv": 4, "dim": 128, "seqs": 16, "context": 2300, "count": 1, "prompt": 0, "window": 0, "keep": 0},
        # many requests with long caches
        {"name": "attend_long", "kind": "attend", "type": "bf16", "heads": 32, "kv": 4, "dim": 128, "seqs": 48, "context": 32000, "count": 1, "prompt": 0, "window": 0, "keep": 0},
        # a layer with a window of as many requests: what lies behind the window is not read, but for the first tokens
        {"name": "attend_window", "kind": "attend", "type": "bf16", "heads": 16, "kv": 4, "dim": 128, "seqs": 64, "context": 20000, "count": 1, "prompt": 0, "window": 1024, "keep": 4},
        # four drafted tokens and the last one of many requests, heads of 64
        {"name": "attend_verify", "kind": "attend", "type": "f16", "heads": 24, "kv": 4, "dim": 64, "seqs": 32, "context": 6001, "count": 5, "prompt": 0, "window": 0, "keep": 0},
        # a whole prompt whose length is no multiple of anything
        {"name": "attend_prompt", "kind": "attend", "type": "bf16", "heads": 32, "kv": 4, "dim": 128, "seqs": 1, "context": 0, "count": 1, "prompt": 2011, "window": 0, "keep": 0},
        # a later chunk of a long prompt beside three requests that decode, in a layer with a window
        {"name": "attend_chunk", "kind": "attend", "type": "bf16", "heads": 16, "kv": 8, "dim": 128, "seqs": 4, "context": 6001, "count": 1, "prompt": 512, "window": 2048, "keep": 16},
        # the end of a speculative step of one request
        {"name": "verify_one", "kind": "verify", "type": "f32", "form": "logits", "requests": 1, "drafts": 4, "vocab": 151936},
        # ... of many, with as many drafts as each had time for
        {"name": "verify_many", "kind": "verify", "type": "bf16", "form": "logits", "requests": 128, "drafts": 4, "vocab": 151936},
        # ... whose target probabilities have gone through filters already
        {"name": "verify_filtered", "kind": "verify", "type": "f32", "form": "probs", "requests": 64, "drafts": 3, "vocab": 151936},
    ]


def spread(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["pages", "attend", "attend", "attend", "verify", "verify"])
    if kind == "pages":
        admit = rng.random() < 0.5
        slots = spread(rng, 1, 1024)
        return {"kind": kind, "slots": slots, "longest": spread(rng, 1, min(32000, 4000000 // slots)), "count": 0 if admit else rng.randint(1, 9), "admit": admit}
    if kind == "verify":
        requests = spread(rng, 1, 128)
        form = rng.choice(["logits", "logits", "probs"])
        return {"kind": kind, "type": rng.choice(["f32", "bf16"]) if form == "logits" else "f32", "form": form, "requests": requests, "drafts": rng.randint(1, 8 if requests < 64 else 4),
                "vocab": spread(rng, 90, 160000)}
    kv = rng.choice([1, 2, 4, 8])
    case = {"kind": kind, "type": rng.choice(["f32", "bf16", "f16"]), "heads": kv * rng.choice([1, 2, 3, 4, 6, 8, 8, 12, 16] if kv < 8 else [1, 2, 4]), "kv": kv,
            "dim": rng.choice([64, 128, 128]), "seqs": 1, "context": 0, "count": 1, "prompt": 0, "window": rng.choice([0, 0, spread(rng, 1, 4096)]), "keep": 0}
    if case["window"]:
        case["keep"] = rng.choice([0, 4, rng.randint(1, 64)])
    how = rng.choice(["decode", "decode", "verify", "prompt"])
    if how == "prompt":
        case["prompt"] = spread(rng, 9, 2048)
        case["context"] = rng.choice([0, spread(rng, 1, 6000)])
        case["seqs"] = rng.choice([1, 1, 2, 4]) if case["heads"] <= 32 else 1
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


# ------------------------------------------------------------------------------------- pages, slots, positions
# A step: every slot's sequence loses its last `drop` tokens (all, where it has fewer) and gets `count` new ones.  need = pages for what it then has; it frees what it holds
# beyond that, or asks for what is missing.  It is granted if it asks for none or the sum of what is asked up to it is there, freed pages included, and the sum of counts up to
# it is within the step's limit; refused ones lose their count.  The j-th page asked for, in the order of slots and places, is the j-th one freed, and behind those the newest of the pool's stack,
# onto which freed pages that nobody takes go in falling order.
# A pass is two steps, of which the second takes the first back: drafts come and all of them are rejected; or all slots go to other requests, and then again.
def pages_inputs(case, seed):
    v, n, longest = Values(seed), case["slots"], case["longest"]
    before = v.below("before", longest, n) + 1
    if case["admit"]:
        after = v.below("after", longest, n) + 1
        steps = [(torch.full((n,), ALL, device=GPU), after), (torch.full((n,), ALL, device=GPU), before)]
    else:
        count = v.below("count", case["count"], n) + 1
        steps = [(torch.zeros(n, device=GPU), count), (count, torch.zeros(n, device=GPU))]
    return {"before": before.int(), "steps": [(d.int(), c.int()) for d, c in steps]}


def pages_sizes(case):
    """Pages a slot's table holds, pages of the pool, new tokens of a step at most, largest count."""
    a_slot = -(-(case["longest"] + case["count"]) // PAGE)
    return a_slot, a_slot * case["slots"], case["slots"] * max(case["longest"], case["count"]), max(case["longest"], case["count"])


class Pool:
    """The plain form's state."""

    def __init__(self, slots, a_slot, pages, most):
        self.a_slot, self.most = a_slot, most
        self.lens, self.held = torch.zeros(slots, dtype=torch.long, device=GPU), torch.zeros(slots, dtype=torch.long, device=GPU)
        self.tables = torch.zeros(slots, a_slot, dtype=torch.long, device=GPU)
        self.stack, self.free = torch.arange(pages - 1, -1, -1, device=GPU), torch.tensor(pages, device=GPU)
        self.maps = torch.zeros(3, most, dtype=torch.long, device=GPU)      # slot in the cache, position, sequence of every new token

    def step(self, drop, count, max_count):
        drop, count = drop.long(), count.long()
        keep = self.lens - drop.clamp(min=0).minimum(self.lens)
        count = torch.where((count >= 0) & (count <= max_count) & (keep + count <= self.a_slot * PAGE), count, 0)
        need = (keep + count + PAGE - 1) // PAGE
        frees, asks = (self.held - need).clamp(min=0), (need - self.held).clamp(min=0)
        granted = ((asks == 0) | (asks.cumsum(0) <= self.free + frees.sum())) & (count.cumsum(0) <= self.most)
        asks, count = torch.where(granted, asks, 0), torch.where(granted, count, 0)
        place = torch.arange(self.a_slot, device=GPU)[None]
        # the stack with what is freed on top, the first of it topmost
        n_freed, freed = frees.sum(), (place >= need[:, None]) & (place < self.held[:, None])
        order = self.free + n_freed - 1 - (freed.flatten().cumsum(0) - 1).view_as(freed)
        self.stack = torch.cat([self.stack, self.stack[:1]])       # (one more place for what is not stored)
        self.stack[torch.where(freed, order, len(self.stack) - 1)] = self.tables
        top = self.free + n_freed
        taken = (place >= self.held[:, None]) & (place < (self.held + asks)[:, None])
        at = top - 1 - (taken.flatten().cumsum(0) - 1).view_as(taken)
        self.tables = torch.where(taken, self.stack[at.clamp(min=0)], self.tables)
        self.stack = self.stack[:-1]
        self.free = top - asks.sum()
        self.held, self.lens = torch.where(frees > 0, need, self.held + asks), keep + count
        ends = count.cumsum(0)
        t = torch.arange(self.most, device=GPU)
        seq = torch.searchsorted(ends, t, right=True).clamp(max=len(ends) - 1)
        starts = ends - count
        pos = keep[seq] + t - starts[seq]
        slot = self.tables[seq, (pos // PAGE).clamp(0, self.a_slot - 1)] * PAGE + pos % PAGE
        self.maps = torch.where(t < ends[-1], torch.stack([slot, pos, seq]), self.maps)
        self.counts, self.starts = count, torch.cat([starts, ends[-1:]])

    def outputs(self):
        return {"lens": self.lens.int(), "counts": self.counts.int(), "starts": self.starts.int(), "tables": self.tables.int(), "slots": self.maps[0].int(), "positions": self.maps[1].int(),
                "seqs": self.maps[2].int(), "free": self.free.int().view(1)}


def pages_plain(s):
    for drop, count in s["steps"]:
        s["pool"].step(drop, count, s["max_count"])
    return s["pool"].outputs()


def pages_work(case):
    # on average: a slot's numbers in and out, three numbers a new token, the pages that change hands read and written
    n, mean = case["slots"], (case["longest"] + 1) / 2
    tokens = n * 2 * mean if case["admit"] else n * (case["count"] + 1) / 2
    moved = 2 * n * case["longest"] / 3 / PAGE if case["admit"] else 2 * tokens / PAGE
    return {"bytes": 2 * n * 4 * 8 + 12 * tokens + 8 * moved, "flops": 2 * (20 * n + 8 * tokens)}


# ------------------------------------------------------------------------- attention over a paged 16-bit cache
# The token at position p of a sequence sees the cached rows k <= p, its own among them; where there is a window, the ones with k > p - window or k < keep.
# Rows of f32 are held as fp16, the others as they are.
def lengths(case):
    """(tokens before the step, new tokens) of every sequence."""
    before = [case["context"]] + [max(0, round(case["context"] * (0.2 + 0.8 * math.modf(0.618034 * e)[0]))) for e in range(1, case["seqs"])]
    new = [case["prompt"] or case["count"]] + [case["count"]] * (case["seqs"] - 1)
    return before, new


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
    """Sequence and position of every token that `before` .. `before + new` names."""
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
        t = TYPES["f16" if case["type"] == "f32" else case["type"]]
        self.k, self.v = (torch.zeros(sum(need), PAGE, case["kv"], case["dim"], dtype=t, device=GPU) for _ in "kv")

    def write(self, seq, pos, k, v):
        page, slot = self.table[seq, pos // PAGE], pos % PAGE
        self.k[page, slot], self.v[page, slot] = k.to(self.k.dtype), v.to(self.v.dtype)

    def rows(self, seq, pos):
        page, slot = self.table[seq, pos // PAGE], pos % PAGE
        return self.k[page, slot].float(), self.v[page, slot].float()


def seen(case, device="cpu"):
    """Positions of the keys that some new token of a sequence sees, [sequence, place]; places behind a sequence's end have positions behind it."""
    before, new = lengths(case)
    window, first = case["window"], torch.tensor(before, device=device)
    if not window:
        return torch.arange(max(b + n for b, n in zip(before, new)), device=device)[None].expand(len(new), -1)
    keep = min(case["keep"], max(before) + max(new))
    low = (first - window + 1).clamp(min=keep)      # the window of the first new token, kept ones listed apart
    span = min(window - 1 + max(new), max(max(0, b + n - keep) for b, n in zip(before, new)))
    return torch.cat([torch.arange(keep, device=device)[None].expand(len(new), -1), low[:, None] + torch.arange(span, device=device)[None]], 1)


def attend_plain(s):
    case, cache, seq, pos = s["case"], s["cache"], s["seq"], s["pos"]
    cache.write(seq, pos, s["k"], s["v"])
    most, place, key = s["most"], s["place"], s["seen"]
    inside = key.clamp(max=cache.table.shape[1] * PAGE - 1)
    K, V = cache.rows(torch.arange(case["seqs"], device=GPU)[:, None], inside)
    # queries [sequence, place, head, dim], padded to the largest number of new tokens
    q = torch.zeros(case["seqs"], most, case["kv"], case["heads"] // case["kv"], case["dim"], device=GPU)
    q[seq, place] = s["q"].float().unflatten(1, (case["kv"], -1))
    last = torch.full((case["seqs"], most), -1, device=GPU)
    last[seq, place] = pos
    z = torch.einsum("scigd,spid->scigp", q, K) * s["scale"]
    hidden = key[:, None] > last[:, :, None]
    if case["window"]:
        hidden |= (key[:, None] <= last[:, :, None] - case["window"]) & (key[:, None] >= case["keep"])
    z = z.masked_fill(hidden[:, :, None, None], -math.inf)
    w = torch.exp(z - z.amax(-1, keepdim=True).clamp(min=-3e38))
    y = torch.einsum("scigp,spid->scigd", w, V) / w.sum(-1)[..., None]
    return y[seq, place].flatten(1, 2).to(TYPES[case["type"]])


def attend_exact(case, seed):
    """Sequence by sequence, head by head, in 64 bits; windows as a mask over all keys."""
    x = attend_inputs(case, seed)
    before, new = lengths(case)
    if sum(n * (b + n) for b, n in zip(before, new)) * case["heads"] * case["dim"] > 2e11:
        return None
    if case["type"] == "f32":
        for name in ("k", "v", "old_k", "old_v"):
            x[name] = x[name].to(torch.float16)
    y, at, old = torch.empty(x["q"].shape, dtype=F8, device=GPU), 0, 0
    G = case["heads"] // case["kv"]
    for b, n in zip(before, new):
        row, col = torch.arange(b, b + n, device=GPU)[:, None], torch.arange(b + n, device=GPU)[None]
        sees = col <= row
        if case["window"]:
            sees = sees & ((row - col < case["window"]) | (col < case["keep"]))
        for h in range(case["heads"]):
            i = h // G
            K = torch.cat([x["old_k"][old:old + b, i], x["k"][at:at + n, i]]).to(F8)
            V = torch.cat([x["old_v"][old:old + b, i], x["v"][at:at + n, i]]).to(F8)
            z = (x["q"][at:at + n, h].to(F8) @ K.T * x["scale"]).where(sees, -math.inf)
            y[at:at + n, h] = torch.softmax(z, -1) @ V
        at, old = at + n, old + b
    return y


def attend_work(case):
    before, new = lengths(case)
    size, held = TYPES[case["type"]].itemsize, 2
    rows = pairs = 0
    for b, n in zip(before, new):
        first = max(0, b - case["window"] + 1) if case["window"] else 0
        rows += b + n - first + min(case["keep"], first)
        if not case["window"]:
            pairs += n * b + n * (n + 1) // 2
        else:
            pairs += sum(min(p + 1, case["window"]) + min(case["keep"], max(0, p + 1 - case["window"])) for p in range(b, b + n))
    T = sum(new)
    io = T * case["dim"] * (2 * case["heads"] + 2 * case["kv"]) * size + 2 * T * case["kv"] * case["dim"] * held
    return {"bytes": 2 * case["kv"] * case["dim"] * held * (rows - T) + io, "flops": 4 * pairs * case["heads"] * case["dim"]}


# ----------------------------------------------------------------------------- verification of drafted tokens
# p_i: the target's distribution behind a request's i-th token, softmax(logits / temperature) (temperature 0: one at the first largest), or given as it is.  q_i: the one that
# draft i was drawn from.  Draft i is accepted if u_i q_i(t_i) < p_i(t_i) and all before it are.  n: how many are.  The next token is drawn from max(0, p_n - q_n), where that is
# nothing or all drafts are accepted from p_n: the first, by index, up to which the sum is above the last uniform number times the whole.
def verify_inputs(case, seed):
    v, R, D, V = Values(seed), case["requests"], case["drafts"], case["vocab"]
    n = v.below("n", 2 * D, R).clamp(max=D) if R > 1 else torch.full((1,), D, device=GPU)       # half of the requests have all drafts
    starts = torch.cat([torch.zeros(1, dtype=torch.long, device=GPU), (n + 1).cumsum(0)])
    T = R * (D + 1)         # room for rows; the requests' rows follow one another without gaps
    # probabilities fall with a power of the rank, differently steep by row; the draft is near to the target
    steep = 1.0 + 1.2 * v.uniform("steep", T, 1)
    x = torch.empty(T, V, device=GPU)
    ranked = 9.0 - steep * torch.log(torch.arange(1, V + 1, device=GPU).float())[None]
    by = (torch.arange(V, device=GPU)[None] * 7919 + v.below("shift", V, T, 1)) % V if V % 7919 else torch.arange(V, device=GPU)[None].expand(T, V)
    x.scatter_(1, by, ranked).add_(v.normal("noise", T, V), alpha=0.3)
    del ranked, by
    T_of = torch.tensor([0.0, 0.7, 1.0, 1.0, 1.3], device=GPU)[v.below("t", 5, R)]
    if case["form"] == "probs":
        T_of = T_of.clamp(min=0.7)
    q = torch.empty(D, R, V, device=GPU)
    tokens = torch.empty(D, R, dtype=torch.int32, device=GPU)
    draws = v.uniform("draws", D, R)
    for i in range(D):
        y = x[(starts[:-1] + i).clamp(max=T - 1)] + 0.6 * v.normal("draft%d" % i, R, V)
        greedy = torch.zeros_like(y).scatter_(1, y.argmax(1, keepdim=True), 1.0)
        q[i] = torch.where(T_of[:, None] > 0, torch.softmax(y / T_of.clamp(min=0.1)[:, None], 1), greedy)
        tokens[i] = (q[i].double().cumsum(1) <= draws[i, :, None]).sum(1).clamp(max=V - 1).int()
    if case["form"] == "probs":     # of each row's likelier tokens alone
        x = torch.softmax(x, 1)
        x = x * (x >= 0.02 * x.amax(1, keepdim=True))
        x /= x.sum(1, keepdim=True)
    return {"target": x.to(TYPES[case["type"]]), "q": q, "tokens": tokens, "n": n.int(), "starts": starts.int(), "temperature": T_of, "u": v.uniform("u", R, D + 1)}


def verify_plain(s):
    # in 64 bits throughout: a uniform number next to a border of two tokens decides between them
    R, D = s["case"]["requests"], s["case"]["drafts"]
    n, request = s["n"].long(), torch.arange(R, device=GPU)
    def p_of(rows, request):
        x = s["target"][rows].double()
        if s["case"]["form"] == "probs":
            return x.clamp(min=0)
        T = s["temperature"][request, None].double()
        one = torch.zeros_like(x).scatter_(1, x.argmax(1, keepdim=True), 1.0)
        w = torch.exp((x - x.amax(1, keepdim=True)) / torch.where(T > 0, T, 1.0))
        return torch.where(T > 0, w / w.sum(1, keepdim=True), one)
    good = torch.ones(R, dtype=torch.bool, device=GPU)
    accepted = torch.zeros(R, dtype=torch.long, device=GPU)
    for i in range(D):
        t = s["tokens"][i].long()[:, None]
        rows = (s["starts"][:-1].long() + i).clamp(max=len(s["target"]) - 1)
        q, p = s["q"][i].gather(1, t)[:, 0].double(), p_of(rows, request).gather(1, t)[:, 0]
        good = good & (i < n) & (s["u"][:, i].double() * q < p)
        accepted += good
    p = p_of(s["starts"][:-1].long() + accepted, request)
    q = s["q"][accepted.clamp(max=D - 1), request].double() * (accepted < n)[:, None]
    w = (p - q).clamp(min=0)
    w = torch.where(w.sum(1, keepdim=True) > 0, w, p)
    upto = w.cumsum(1)
    token = (upto <= s["u"][:, D:].double() * upto[:, -1:]).sum(1).clamp(max=w.shape[1] - 1).int()
    place = torch.arange(D + 1, device=GPU)[None]
    drafted = torch.cat([s["tokens"].T, s["tokens"][:1].T], 1)
    tokens = torch.where(place < accepted[:, None], drafted, torch.where(place == accepted[:, None], token[:, None], -1))
    return {"tokens": tokens.int(), "accepted": accepted.int(), "rejected": (n - accepted).int()}


def verify_work(case):
    R, D, V = case["requests"], case["drafts"], case["vocab"]
    drafts = D if R == 1 else sum(min(k, D) for k in range(2 * D)) / (2 * D)
    if case["form"] == "probs":     # the row drawn from, and its draft's
        return {"bytes": R * V * 8 + R * drafts * 16, "flops": 4 * R * V}
    size = TYPES[case["type"]].itemsize
    return {"bytes": R * (drafts + 1) * V * size + R * V * 4, "flops": 4 * R * (drafts + 2) * V}


# ------------------------------------------------------------------------------------------ this library's calls
_ctx = None


def context():
    """One context for all, as a program has."""
    global _ctx
    if _ctx is None:
        import densecore_b200 as dc
        _ctx = dc.Context(0)
    return _ctx


class On:
    """An array of the library's as a tensor, which keeps its owner."""

    def __init__(self, owner, address, shape):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": shape, "typestr": "<i4", "data": (address, False), "version": 3}


def own_pool(s):
    case, ctx = s["case"], context()
    a_slot, pages, most, _ = pages_sizes(case)
    s["kv"] = kv = ctx.kv_cache_dev(1, 1, 1, 64, pages, case["slots"], a_slot, most, dtype="bf16")
    kv.step_dev(s["before"].data_ptr(), max_count=s["max_count"])
    ctx.synchronize()
    at, n = kv.arrays(), case["slots"]
    s["arrays"] = {k: torch.as_tensor(On(kv, at[k], shape), device=GPU) for k, shape in
                   {"lens": (n,), "counts": (n,), "starts": (n + 1,), "tables": (n, a_slot), "slots": (most,), "positions": (most,), "seqs": (most,), "free": (1,)}.items()}
    s["at"] = [(d.data_ptr(), c.data_ptr()) for d, c in s["steps"]]


def pages_own(s):
    for drop, count in s["at"]:
        s["kv"].step_dev(count, drop=drop, max_count=s["max_count"])
    return s["arrays"]


def own_cache(s):
    """The library's cache with the tokens before the step, and the step's places."""
    case, ctx = s["case"], context()
    before, new = lengths(case)
    need = [-(-(a + b) // PAGE) for a, b in zip(before, new)]
    kv = ctx.kv_cache_dev(1, case["heads"], case["kv"], case["dim"], sum(need), case["seqs"], max(need), max(sum(before), sum(new)), dtype=case["type"])
    counts = [torch.tensor(c, dtype=torch.int32, device=GPU) for c in (before, new)]
    torch.cuda.synchronize()
    if sum(before):
        kv.step_dev(counts[0].data_ptr(), max_count=max(before))
        kv.write_dev(0, s["old_k"].data_ptr(), s["old_v"].data_ptr())
    kv.step_dev(counts[1].data_ptr(), max_count=max(new))
    ctx.synchronize()
    s["kv"], s["out"] = kv, torch.empty_like(s["q"])
    s["at"] = [s[n].data_ptr() for n in ("q", "k", "v")]


def attend_own(s):
    q, k, v = s["at"]
    s["kv"].attend_dev(0, q, k, v, s["scale"], s["out"].data_ptr(), window=s["case"]["window"], keep_first=s["case"]["keep"])
    return s["out"]


def own_verify(s):
    R, D = s["case"]["requests"], s["case"]["drafts"]
    s["out"] = {"tokens": torch.empty(R, D + 1, dtype=torch.int32, device=GPU), "accepted": torch.empty(R, dtype=torch.int32, device=GPU),
                "rejected": torch.empty(R, dtype=torch.int32, device=GPU)}
    s["at"] = {k: s[k].data_ptr() for k in ("target", "q", "tokens", "n", "starts", "temperature", "u")}


def verify_own(s):
    case, at, out = s["case"], s["at"], s["out"]
    context().verify_rows_dev(at["target"], case["requests"], case["vocab"], case["drafts"], at["tokens"], at["q"], at["u"], out["tokens"].data_ptr(), out["accepted"].data_ptr(),
                              rejected=out["rejected"].data_ptr(), starts=at["starts"], n_drafts=at["n"], temperature=at["temperature"] if case["form"] == "logits" else 0,
                              dtype=case["type"], probs=case["form"] == "probs")
    return out


# ------------------------------------------------------------------------------------------------ what is asked
def prepare(case, seed):
    kind = case["kind"]
    s = {"pages": pages_inputs, "attend": attend_inputs, "verify": verify_inputs}[kind](case, seed)
    s["case"] = case
    # what a program keeps between calls, on either side: the pool, the cache that holds the earlier tokens, results' buffers
    if kind == "pages":
        a_slot, pages, most, s["max_count"] = pages_sizes(case)
        torch.cuda.synchronize()
        if own:
            own_pool(s)
        else:
            s["pool"] = Pool(case["slots"], a_slot, pages, most)
            s["pool"].step(torch.zeros_like(s["before"]), s["before"], s["max_count"])
    elif kind == "attend":
        before, new = lengths(case)
        if own:
            own_cache(s)
        else:
            s["seq"], s["pos"] = places(before, new)
            s["most"], s["place"] = max(new), s["pos"] - torch.tensor(before, device=GPU)[s["seq"]]
            s["seen"] = seen(case, GPU)
            s["cache"] = Cache(case, seed)
            s["cache"].write(*places([0] * case["seqs"], before), s["old_k"], s["old_v"])
        del s["old_k"], s["old_v"]
    elif own:
        own_verify(s)
    torch.cuda.synchronize()
    return s


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"pages": pages_own, "attend": attend_own, "verify": verify_own}[kind](state)
    return {"pages": pages_plain, "attend": attend_plain, "verify": verify_plain}[kind](state)


def exact(case, seed):
    return attend_exact(case, seed) if case["kind"] == "attend" else None       # (the others' outputs are whole numbers)


def work(case):
    return {"pages": pages_work, "attend": attend_work, "verify": verify_work}[case["kind"]](case)

"""Measured cases of the operators for serving over long and shared KV caches: rotary positions
(rope, rope_append), attention of a batch over a shared prefix (attention_prefix), attention
that accumulates each cache slot's weight (attention_scored) and eviction by that weight
(cache_evict).

`run` computes them in plain torch operations, or with `own` set by the library's calls.
Head layouts are those of the repository's decoder configurations (16/16 and 32/4 heads of
128) and of its tests (4/2 and 8/2 heads of 64)."""
import math

import torch

own = False

DEV = "cuda"


def listed():
    return [
        # one decode token of a 32/4-head layer: q and k heads side by side in a fused projection
        {"name": "rope-token", "op": "rope", "tokens": 1, "heads": 36, "dim": 128, "rotary": 128,
         "traditional": False, "scaling": "none", "far": 40000},
        # a long prompt of that layer, positions past the trained length (by-parts scaling)
        {"name": "rope-prompt-yarn", "op": "rope", "tokens": 16384, "heads": 36, "dim": 128, "rotary": 128,
         "traditional": False, "scaling": "yarn", "far": 120000},
        # interleaved pairs on half of a 64-wide head, an odd number of tokens
        {"name": "rope-partial", "op": "rope", "tokens": 4097, "heads": 8, "dim": 64, "rotary": 32,
         "traditional": True, "scaling": "linear", "far": 16000},
        # a decode step's q, k, v of 32 sequences at their own positions, k and v into the cache
        {"name": "append-step", "op": "append", "batch": 32, "new": 1, "heads": 16, "kv": 16, "dim": 128,
         "cap": 768, "traditional": False, "scaling": "none", "far": 700},
        # a few short requests behind a short common instruction
        {"name": "prefix-small", "op": "prefix", "batch": 3, "new": 1, "heads": 4, "kv": 2, "dim": 64,
         "prefix": 97, "cap": 64, "least": 1, "most": 41},
        # 32 conversations behind one 4096-token system prompt, a cache head per query head
        {"name": "prefix-batch", "op": "prefix", "batch": 32, "new": 1, "heads": 16, "kv": 16, "dim": 128,
         "prefix": 4096, "cap": 768, "least": 1, "most": 511},
        # 64 questions about one long document, grouped heads
        {"name": "prefix-document", "op": "prefix", "batch": 64, "new": 1, "heads": 32, "kv": 4, "dim": 128,
         "prefix": 32768, "cap": 1024, "least": 3, "most": 1000},
        # five draft tokens of each of 16 sequences checked at once
        {"name": "prefix-draft", "op": "prefix", "batch": 16, "new": 5, "heads": 32, "kv": 4, "dim": 128,
         "prefix": 8191, "cap": 512, "least": 5, "most": 333},
        # a decode step over ragged caches that keeps every slot's weight
        {"name": "scored-step", "op": "scored", "batch": 16, "new": 1, "heads": 32, "kv": 4, "dim": 128,
         "cap": 16384, "least": 100, "most": 16001},
        # a whole prompt, its slots' weights for the first eviction
        {"name": "scored-prompt", "op": "scored", "batch": 1, "new": 4096, "heads": 32, "kv": 4, "dim": 128,
         "cap": 4096, "least": 4096, "most": 4096},
        # one slot too many in each head's cache: the lightest goes
        {"name": "evict-step", "op": "evict", "batch": 32, "kv": 4, "dim": 128, "cap": 2112, "least": 2049,
         "most": 2049, "budget": 2048, "sinks": 4, "recent": 256, "inplace": True},
        # prompts' caches cut down into the smaller caches that decoding goes on with
        {"name": "evict-prompt", "op": "evict", "batch": 8, "kv": 4, "dim": 128, "cap": 16384, "least": 9000,
         "most": 16384, "budget": 2048, "sinks": 4, "recent": 512, "inplace": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "prefix", "scored", "prompt", "evict"])
    heads, kv, dim = rng.choice([(16, 16, 128), (32, 4, 128), (8, 2, 64), (4, 2, 64), (16, 16, 64), (6, 2, 128)])
    scaling = rng.choice(["none", "linear", "ntk", "yarn", "banded"])
    if op == "rope":
        t = _log(rng, 1, 16384)
        return {"op": "rope", "tokens": t, "heads": heads + (kv if dim == 128 else 0), "dim": dim,
                "rotary": rng.choice([dim, dim // 2, dim // 4]), "traditional": rng.random() < 0.5,
                "scaling": scaling, "far": _log(rng, 100, 1000000)}
    if op == "append":
        new = rng.choice([1, 1, 3, 17])
        cap = _log(rng, 64, 2048)
        return {"op": "append", "batch": _log(rng, 1, 64), "new": new, "heads": heads, "kv": kv, "dim": dim,
                "cap": cap, "traditional": rng.random() < 0.5, "scaling": scaling,
                "far": rng.randint(new, cap)}
    if op == "prefix":
        new = rng.choice([1, 1, 1, 2, 5, 8])
        b = _log(rng, 1, 64 // new if new > 1 else 64)
        most = _log(rng, new, 1000)
        return {"op": "prefix", "batch": b, "new": new, "heads": heads, "kv": kv, "dim": dim,
                "prefix": _log(rng, 1, 32768 if kv <= 4 else 8192), "cap": most + rng.randint(0, 24),
                "least": rng.randint(0, most), "most": most}
    if op == "scored":
        new = rng.choice([1, 1, 1, 2, 4])
        most = _log(rng, new, 16000 if kv <= 4 else 4000)
        return {"op": "scored", "batch": _log(rng, 1, 16 if kv <= 4 else 6), "new": new, "heads": heads, "kv": kv, "dim": dim,
                "cap": most + rng.randint(0, 300), "least": rng.randint(0, most), "most": most}
    if op == "prompt":
        new = _log(rng, 16, 4000)
        b = rng.randint(1, max(1, min(4, 4000 // new)))
        most = new + rng.choice([0, 0, rng.randint(0, 90)])
        return {"op": "scored", "batch": b, "new": new, "heads": heads, "kv": kv, "dim": dim,
                "cap": most + rng.randint(0, 9), "least": min(most, new), "most": most}
    most = _log(rng, 64, 16384 if kv <= 4 else 4096)
    budget = rng.randint(max(16, most // 16), most)
    sinks = rng.randint(0, 4)
    return {"op": "evict", "batch": _log(rng, 1, 8), "kv": kv, "dim": dim, "cap": most + rng.randint(0, 40),
            "least": rng.randint(most // 2, most), "most": most, "budget": budget, "sinks": sinks,
            "recent": rng.randint(0, budget - sinks), "inplace": rng.random() < 0.5}


# what the case's scaling means, for 4096-token training length
SCALING = {
    "none": None,
    "linear": {"type": "linear", "factor": 4.0},
    "ntk": {"type": "ntk", "factor": 4.0},
    "yarn": {"type": "yarn", "factor": 4.0, "original_len": 32768, "beta_fast": 32.0, "beta_slow": 1.0},
    "banded": {"type": "banded", "factor": 8.0, "original_len": 8192, "low_freq": 1.0, "high_freq": 4.0},
}
THETA = 1000000.0


def _lens(case):
    """Ragged lengths from `least` to `most`, in a mixed order (they belong to the case: its
    work follows from them)."""
    b = case["batch"]
    if b == 1:
        return [case["most"]]
    step = next(s for s in (7, 5, 3, 11, 13, 1) if math.gcd(s, b) == 1)
    return [case["least"] + (case["most"] - case["least"]) * ((i * step) % b) // (b - 1) for i in range(b)]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(torch.bfloat16)

    def ints(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device=DEV, dtype=torch.int32)

    s = dict(case)
    op, d = case["op"], case["dim"]
    if op == "rope":
        t = case["tokens"]
        start = ints(0, max(1, case["far"] - t), 1)
        s["x"] = normal(t, case["heads"], d)
        s["pos"] = start + torch.arange(t, dtype=torch.int32, device=DEV)
        return s
    b, kv = case["batch"], case["kv"]
    if op == "append":
        new, nh, cap = case["new"], case["heads"], case["cap"]
        qkv = normal(b * new, nh + 2 * kv, d)  # the fused projection's rows
        s["q"], s["k"], s["v"] = qkv[:, :nh], qkv[:, nh:nh + kv], qkv[:, nh + kv:]
        s["cache_k"], s["cache_v"] = normal(b, kv, cap, d), normal(b, kv, cap, d)
        end = ints(min(new, cap), min(case["far"], cap) + 1, b)
        s["slots"] = (end[:, None] - new + torch.arange(new, dtype=torch.int32, device=DEV)[None]).reshape(-1)
        s["pos"] = s["slots"].clone()
        return s
    lens = torch.tensor(_lens(case), dtype=torch.int32, device=DEV)
    cap = case["cap"]
    s["lens"] = lens
    s["cache_k"], s["cache_v"] = normal(b, kv, cap, d), normal(b, kv, cap, d)
    if op == "prefix":
        s["q"] = normal(b, case["new"], case["heads"], d)
        s["prefix_k"], s["prefix_v"] = normal(kv, case["prefix"], d), normal(kv, case["prefix"], d)
    elif op == "scored":
        s["q"] = normal(b, case["new"], case["heads"], d)
        s["acc"] = torch.zeros(b, kv, cap, device=DEV)
        if case["new"] < 16:  # a step: earlier steps have left weights
            s["acc"] += torch.rand(b, kv, cap, generator=g, device=DEV)
    else:
        # heavy slots and many light ones, as attention leaves them
        s["acc"] = torch.randn(b, kv, cap, generator=g, device=DEV).mul_(2.0).exp_()
        s["positions"] = torch.arange(cap, dtype=torch.int32, device=DEV).expand(b, kv, cap).contiguous()
        n = case["budget"]
        if case["inplace"]:
            s["to"] = (s["cache_k"], s["cache_v"], s["acc"], s["positions"])
        else:
            s["to"] = (torch.zeros(b, kv, n, d, dtype=torch.bfloat16, device=DEV),
                       torch.zeros(b, kv, n, d, dtype=torch.bfloat16, device=DEV),
                       torch.zeros(b, kv, n, device=DEV), torch.zeros(b, kv, n, dtype=torch.int32, device=DEV))
        s["lens_out"] = torch.zeros(b, dtype=torch.int32, device=DEV)
    return s


def run(s):
    return {"rope": _rope, "append": _append, "prefix": _prefix, "scored": _scored, "evict": _evict}[s["op"]](s)


# ------------------------------------------------------------------ rotary positions
def _inverse_frequencies(r, scaling):
    """fp64 [r/2] radians per position, and the factor on cos and sin."""
    i = torch.arange(0, r, 2, dtype=torch.float64, device=DEV)
    if scaling is None:
        return THETA ** (-i / r), 1.0
    f = scaling["factor"]
    if scaling["type"] == "linear":
        return THETA ** (-i / r) / f, 1.0
    if scaling["type"] == "ntk":
        return (THETA * f ** (r / (r - 2))) ** (-i / r), 1.0
    inv = THETA ** (-i / r)
    n = scaling["original_len"]
    if scaling["type"] == "banded":  # by rotations over the original length
        keep = ((n * inv / (2 * math.pi) - scaling["low_freq"]) / (scaling["high_freq"] - scaling["low_freq"])).clamp(0, 1)
        return inv * (keep + (1 - keep) / f), 1.0

    def dim_of(turns):  # the (fractional) pair that turns that often over the original length
        return r * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(THETA))

    lo = max(math.floor(dim_of(scaling["beta_fast"])), 0)
    hi = min(math.ceil(dim_of(scaling["beta_slow"])), r - 1)
    ramp = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return inv * ((1 - ramp) + ramp / f), 0.1 * math.log(f) + 1.0


def _rotate(x, pos, r, traditional, scaling):
    inv, factor = _inverse_frequencies(r, scaling)
    a = pos.double()[:, None] * inv[None]
    cos, sin = (a.cos() * factor).float()[:, None], (a.sin() * factor).float()[:, None]
    f = x[..., :r].float()
    if traditional:
        x1, x2 = f[..., 0::2], f[..., 1::2]
        y = torch.stack((x1 * cos - x2 * sin, x1 * sin + x2 * cos), dim=-1).flatten(-2)
    else:
        x1, x2 = f[..., : r // 2], f[..., r // 2:]
        y = torch.cat((x1 * cos - x2 * sin, x1 * sin + x2 * cos), dim=-1)
    return torch.cat((y.to(x.dtype), x[..., r:]), dim=-1)


def _rope(s):
    if own:
        from flashmlx_b200 import ops
        return ops.rope(s["x"], s["pos"], THETA, rotary_dim=s["rotary"], traditional=s["traditional"],
                        scaling=SCALING[s["scaling"]])
    return _rotate(s["x"], s["pos"], s["rotary"], s["traditional"], SCALING[s["scaling"]])


def _append(s):
    if own:
        from flashmlx_b200 import ops
        q = ops.rope_append(s["q"], s["k"], s["v"], s["pos"], s["slots"], s["cache_k"], s["cache_v"], THETA,
                            traditional=s["traditional"], scaling=SCALING[s["scaling"]])
        return {"q": q, "cache_k": s["cache_k"], "cache_v": s["cache_v"]}
    r, tr, sc = s["dim"], s["traditional"], SCALING[s["scaling"]]
    at = torch.arange(s["batch"], device=DEV).repeat_interleave(s["new"])
    slot = s["slots"].long()
    s["cache_k"][at, :, slot] = _rotate(s["k"], s["pos"], r, tr, sc)
    s["cache_v"][at, :, slot] = s["v"]
    return {"q": _rotate(s["q"], s["pos"], r, tr, sc), "cache_k": s["cache_k"], "cache_v": s["cache_v"]}


# ------------------------------------------------------------------ attention
def _rows(q, kv):
    """[B, L, nh, d] -> fp32 [B, kv, L * group, d]: a kv head's queries together."""
    b, n, nh, d = q.shape
    return q.float().reshape(b, n, kv, nh // kv, d).permute(0, 2, 1, 3, 4).reshape(b, kv, -1, d)


def _own_scores(s, rows):
    """Scores over the sequences' own caches, -inf where a query does not see the slot."""
    b, kv, _, d = rows.shape
    n, group = s["new"], s["heads"] // s["kv"]
    sc = rows @ s["cache_k"].float().transpose(-1, -2) * d ** -0.5
    j = torch.arange(s["cap"], device=DEV)
    end = s["lens"].long()[:, None] - n + torch.arange(n, device=DEV)[None]  # last visible slot
    seen = (j[None, None] <= end[..., None]).repeat_interleave(group, dim=1)
    return sc.masked_fill_(~seen[:, None], -math.inf)


def _softmax(sc):
    top = sc.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = sc.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(torch.where(total == 0, torch.ones_like(total), total))


def _back(o, n, nh):
    """[B, kv, L * group, d] -> [B, L, nh, d] bf16."""
    b, kv, _, d = o.shape
    return o.reshape(b, kv, n, nh // kv, d).permute(0, 2, 1, 3, 4).reshape(b, n, nh, d).to(torch.bfloat16)


def _prefix(s):
    if own:
        from flashmlx_b200 import ops
        return ops.attention_prefix(s["q"], s["prefix_k"], s["prefix_v"], s["cache_k"], s["cache_v"], s["lens"])
    b, n, nh, kv, d = s["batch"], s["new"], s["heads"], s["kv"], s["dim"]
    rows = _rows(s["q"], kv)
    shared = rows.transpose(0, 1).reshape(kv, -1, d)  # every sequence's queries of a kv head
    sp = (shared @ s["prefix_k"].float().transpose(-1, -2) * d ** -0.5).reshape(kv, b, -1, s["prefix"]).transpose(0, 1)
    p = _softmax(torch.cat((sp, _own_scores(s, rows)), dim=-1))
    pp = p[..., : s["prefix"]].transpose(0, 1).reshape(kv, -1, s["prefix"])
    o = (pp @ s["prefix_v"].float()).reshape(kv, b, -1, d).transpose(0, 1) + p[..., s["prefix"]:] @ s["cache_v"].float()
    return _back(o, n, nh)


def _scored(s):
    if own:
        from flashmlx_b200 import ops
        out = ops.attention_scored(s["q"], s["cache_k"], s["cache_v"], s["lens"], s["acc"])
        return {"out": out, "acc": s["acc"]}
    p = _softmax(_own_scores(s, _rows(s["q"], s["kv"])))
    s["acc"] += p.sum(dim=2)
    return {"out": _back(p @ s["cache_v"].float(), s["new"], s["heads"]), "acc": s["acc"]}


# ------------------------------------------------------------------ eviction
def _evict(s):
    k, v, acc, pos = s["cache_k"], s["cache_v"], s["acc"], s["positions"]
    if own:
        from flashmlx_b200 import ops
        to = None if s["inplace"] else s["to"]
        ops.cache_evict(k, v, acc, s["lens"], s["budget"], sinks=s["sinks"], recent=s["recent"], positions=pos, out=to,
                        lens_out=s["lens_out"])
        return {"k": s["to"][0], "v": s["to"][1], "acc": s["to"][2], "positions": s["to"][3], "lens": s["lens_out"]}
    cap, budget, d = s["cap"], s["budget"], s["dim"]
    lens = s["lens"].long()[:, None, None]
    keep_n = lens.clamp(max=budget)
    j = torch.arange(cap, device=DEV)[None, None]
    held = j < lens
    newest = torch.where(held, pos, torch.full_like(pos, -2 ** 31)).amax(-1, keepdim=True).long()
    safe = held & ((pos < s["sinks"]) | (pos.long() > newest - s["recent"]))
    key = acc.double().nan_to_num(nan=-1e300, posinf=1e300, neginf=-1e300)
    key = torch.where(safe, torch.full_like(key, 2e300), key)
    key = torch.where(held, key, torch.full_like(key, -math.inf))
    order = key.argsort(dim=-1, descending=True, stable=True)
    rank = torch.empty_like(order).scatter_(-1, order, j.expand_as(order).contiguous())
    kept = rank < keep_n
    # the k-th hole below keep_n takes the k-th kept slot from keep_n on
    holes = torch.where(~kept & (j < keep_n), j, cap).sort(dim=-1).values
    tails = torch.where(kept & (j >= keep_n), j, cap).sort(dim=-1).values
    source = torch.cat((j.expand_as(holes), torch.full_like(holes[..., :1], cap)), dim=-1)
    source = source.scatter(-1, holes, tails)[..., :min(cap, budget)]
    to_k, to_v, to_acc, to_pos = s["to"]
    m = source.shape[-1]
    fresh = j[..., :m] < keep_n
    source = torch.where(fresh, source, torch.zeros_like(source))
    wide = source[..., None].expand(-1, -1, -1, d)
    to_k[:, :, :m] = torch.where(fresh[..., None], k.gather(2, wide), to_k[:, :, :m])
    to_v[:, :, :m] = torch.where(fresh[..., None], v.gather(2, wide), to_v[:, :, :m])
    to_acc[:, :, :m] = torch.where(fresh, acc.gather(2, source), to_acc[:, :, :m])
    to_pos[:, :, :m] = torch.where(fresh, pos.gather(2, source), to_pos[:, :, :m])
    s["lens_out"].copy_(keep_n.reshape(-1))
    return {"k": to_k, "v": to_v, "acc": to_acc, "positions": to_pos, "lens": s["lens_out"]}


# ------------------------------------------------------------------ the work of a pass
def work(case):
    op, d = case["op"], case["dim"]
    if op == "rope":
        n = case["tokens"] * case["heads"] * d
        return {"bytes": 4 * n + 4 * case["tokens"], "flops": 3 * case["tokens"] * case["heads"] * case["rotary"]}
    if op == "append":
        t = case["batch"] * case["new"]
        n = t * (case["heads"] + 2 * case["kv"]) * d
        return {"bytes": 4 * n + 8 * t, "flops": 3 * t * (case["heads"] + case["kv"]) * d}
    lens, kv = _lens(case), case["kv"]
    if op == "evict":
        kept = [min(n, case["budget"]) for n in lens]
        # in place only the kept slots behind the budget move (their share if any slot may be kept)
        moved = [m * (n - m) / n if case["inplace"] and n else m for n, m in zip(lens, kept)]
        return {"bytes": kv * (8 * sum(lens) + sum(moved) * (8 * d + 16)), "flops": kv * sum(lens)}
    b, n, nh = case["batch"], case["new"], case["heads"]
    io = 4 * b * n * nh * d  # q and out
    pairs = sum(max(0, m - n + l + 1) for m in lens for l in range(n))
    if op == "prefix":
        return {"bytes": io + 4 * kv * d * (case["prefix"] + sum(lens)),
                "flops": 4 * nh * d * (pairs + b * n * case["prefix"])}
    return {"bytes": io + 4 * kv * d * sum(lens) + 8 * kv * sum(lens), "flops": 4 * nh * d * pairs}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op, d = case["op"], case["dim"]
    if op in ("rope", "append"):
        r = case["rotary"] if op == "rope" else d
        sc = SCALING[case["scaling"]]
        speeds, factor = [], 1.0
        for i in range(r // 2):
            base = THETA
            if sc and sc["type"] == "ntk":
                base = THETA * sc["factor"] ** (r / (r - 2))
            w = base ** (-2.0 * i / r)
            if sc and sc["type"] == "linear":
                w /= sc["factor"]
            if sc and sc["type"] == "banded":
                wave = 2 * math.pi / w
                if wave > sc["original_len"] / sc["low_freq"]:
                    w /= sc["factor"]
                elif wave > sc["original_len"] / sc["high_freq"]:
                    t = (sc["original_len"] / wave - sc["low_freq"]) / (sc["high_freq"] - sc["low_freq"])
                    w = (1 - t) * w / sc["factor"] + t * w
            if sc and sc["type"] == "yarn":
                first, last = (r / 2 * math.log(sc["original_len"] / (2 * math.pi * sc[b])) / math.log(THETA)
                               for b in ("beta_fast", "beta_slow"))
                first, last = max(math.floor(first), 0), min(math.ceil(last), r - 1)
                t = min(max((i - first) / max(last - first, 1e-3), 0.0), 1.0)
                w = w * (1 - t) + w / sc["factor"] * t
                factor = 1 + math.log(sc["factor"]) / 10
            speeds.append(w)
        turn = torch.polar(torch.tensor(factor, dtype=torch.float64, device=DEV),
                           s["pos"].double()[:, None] * torch.tensor(speeds, dtype=torch.float64, device=DEV))

        def rotated(x):
            x = x.double()
            part = x[..., :r].reshape(*x.shape[:-1], r // 2, 2) if case["traditional"] else \
                x[..., :r].reshape(*x.shape[:-1], 2, r // 2).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(part.contiguous()) * turn[:, None])
            z = z if case["traditional"] else z.transpose(-1, -2)
            return torch.cat((z.reshape(*x.shape[:-1], r), x[..., r:]), dim=-1)

        if op == "rope":
            return rotated(s["x"])
        k, ck, cv = rotated(s["k"]), s["cache_k"].double(), s["cache_v"].double()
        for t in range(case["batch"] * case["new"]):
            ck[t // case["new"], :, int(s["slots"][t])] = k[t]
            cv[t // case["new"], :, int(s["slots"][t])] = s["v"][t].double()
        return {"q": rotated(s["q"]), "cache_k": ck, "cache_v": cv}
    if op == "evict":
        return None  # moves: nothing is computed
    b, n, nh, kv = case["batch"], case["new"], case["heads"], case["kv"]
    group = nh // kv
    out = torch.zeros(b, n, nh, d, dtype=torch.float64, device=DEV)
    acc = s["acc"].double() if op == "scored" else None
    for i, m in enumerate(_lens(case)):
        for h in range(kv):
            k, v = s["cache_k"][i, h, :m].double(), s["cache_v"][i, h, :m].double()
            p0 = 0
            if op == "prefix":
                p0 = case["prefix"]
                k, v = torch.cat((s["prefix_k"][h].double(), k)), torch.cat((s["prefix_v"][h].double(), v))
            for lo in range(0, n, 512):
                hi = min(n, lo + 512)
                z = torch.einsum("lgd,jd->lgj", s["q"][i, lo:hi, h * group:(h + 1) * group].double(), k) / math.sqrt(d)
                hidden = torch.arange(p0 + m, device=DEV)[None] > torch.arange(lo, hi, device=DEV)[:, None] + (p0 + m - n)
                if p0:
                    hidden[:, :p0] = False
                z = z.masked_fill(hidden[:, None], -math.inf)
                p = torch.softmax(z, dim=-1).nan_to_num(nan=0.0) if z.shape[-1] else z
                out[i, lo:hi, h * group:(h + 1) * group] = torch.einsum("lgj,jd->lgd", p, v)
                if acc is not None:
                    acc[i, h, :m] += p.sum(dim=(0, 1))
    return out if op == "prefix" else {"out": out, "acc": acc}

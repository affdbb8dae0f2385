"""Plain 64-bit implementations of the serving operators (rotary positions, attention over a
shared prefix and ragged caches, slot weights, eviction) for their tests, with the error a
bf16 / fp32 kernel may make.  Written from the formulas, one sequence and head at a time.

Rounding to bf16 is off by at most U16 = 2^-8 of the value, an fp32 operation by U32 = 2^-24."""
from __future__ import annotations

import math

import torch

U16, U32 = 2.0 ** -8, 2.0 ** -24


def frequencies(r, theta, scaling):
    """[r / 2] radians per position and the factor on cos and sin, in Python floats."""
    kind = scaling["type"] if scaling else None
    f = scaling["factor"] if scaling else 1.0
    base = theta * f ** (r / (r - 2)) if kind == "ntk" else theta
    inv = [base ** (-2.0 * i / r) for i in range(r // 2)]
    m = 1.0
    if kind == "linear":
        inv = [w / f for w in inv]
    elif kind == "banded":
        n, lo, hi = scaling["original_len"], scaling["low_freq"], scaling["high_freq"]
        keep = [min(max((n * w / (2 * math.pi) - lo) / (hi - lo), 0.0), 1.0) for w in inv]
        inv = [w * k + w / f * (1 - k) for w, k in zip(inv, keep)]
    elif kind == "yarn":
        n = scaling["original_len"]
        index = lambda turns: r * math.log(n / (2 * math.pi * turns)) / (2 * math.log(theta))  # noqa: E731
        first, last = max(math.floor(index(scaling["beta_fast"])), 0), min(math.ceil(index(scaling["beta_slow"])), r - 1)
        keep = [1 - min(max((i - first) / max(last - first, 0.001), 0.0), 1.0) for i in range(r // 2)]
        inv = [w * k + w / f * (1 - k) for w, k in zip(inv, keep)]
        m = 0.1 * math.log(f) + 1
    if scaling and scaling.get("attn_factor"):
        m = scaling["attn_factor"]
    return inv, m


def rope(x, positions, theta, rotary=None, traditional=False, scaling=None):
    """x [T, heads, d], positions [T] -> (rotated fp64, allowed error)."""
    d = x.shape[-1]
    r = rotary or d
    inv, m = frequencies(r, theta, scaling)
    ang = positions.double().cpu()[:, None] * torch.tensor(inv, dtype=torch.float64)[None]
    cos, sin = ang.cos()[:, None] * m, ang.sin()[:, None] * m
    y = x.double().cpu().clone()
    i = torch.arange(r // 2)
    a, b = (2 * i, 2 * i + 1) if traditional else (i, i + r // 2)
    x1, x2 = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = x1 * cos - x2 * sin, x1 * sin + x2 * cos
    tol = torch.zeros_like(y)
    # the fp32 angle (one rounding of at most pi: pi 2^-24), sine and cosine (4 ulp), the two
    # products and their sum; fp64 positions * frequencies: |ang| 2^-51; then one bf16 rounding
    size = (x1.abs() + x2.abs()) * m * (16 * U32 + ang.abs()[:, None] * 2.0 ** -51)
    tol[..., a] = tol[..., b] = size
    tol[..., :r] += U16 * (y[..., :r].abs() + tol[..., :r])
    return y, tol


def attention(q, cache_k, cache_v, lens, prefix_k=None, prefix_v=None, acc=None, scale=None):
    """q [B, L, nh, d]; prefix [n_kv, P, d]; caches [B, n_kv, M, d].  Returns (out fp64, its
    allowed error, acc fp64 or None, its allowed error)."""
    B, L, nh, d = q.shape
    nkv = cache_k.shape[1] if cache_k is not None else prefix_k.shape[0]
    group = nh // nkv
    scale = scale or 1 / math.sqrt(d)
    q = q.double().cpu()
    out = torch.zeros(B, L, nh, d, dtype=torch.float64)
    tol = torch.zeros_like(out)
    acc64 = acc.double().cpu().clone() if acc is not None else None
    acc_tol = acc64.abs() * 2 * U32 if acc is not None else None
    for b in range(B):
        n = int(lens[b]) if lens is not None else 0
        for h in range(nkv):
            parts_k, parts_v = [], []
            if prefix_k is not None:
                parts_k.append(prefix_k[h].double().cpu()), parts_v.append(prefix_v[h].double().cpu())
            P = parts_k[0].shape[0] if parts_k else 0
            if n:
                parts_k.append(cache_k[b, h, :n].double().cpu()), parts_v.append(cache_v[b, h, :n].double().cpu())
            if not parts_k:
                continue
            k, v = torch.cat(parts_k), torch.cat(parts_v)
            heads = slice(h * group, (h + 1) * group)
            for l in range(L):
                seen = P + max(0, n - L + l + 1)
                if seen == 0:
                    continue
                rows = q[b, l, heads]
                z = rows @ k[:seen].T * scale
                p = torch.softmax(z, -1)
                o = p @ v[:seen]
                out[b, l, heads] = o
                # a score of d products and d sums in fp32 and its scaling; exp2 and its argument
                score = (rows.abs() @ k[:seen].abs().T * abs(scale)).amax(-1, keepdim=True)
                rel = 2 * ((d + 4) * U32 * score) + 16 * U32  # of a probability, numerator and sum
                mass = p @ v[:seen].abs()
                # probabilities rounded to bf16 for the product, its fp32 sums, one final rounding
                t = mass * (U16 + rel + (seen + 64) * U32)
                tol[b, l, heads] = t + U16 * (o.abs() + t)
                if acc is not None:
                    acc64[b, h, :seen] += p.sum(0)
                    acc_tol[b, h, :seen] += (p * (rel + (L * group + 64) * U32)).sum(0)
    return out, tol, acc64, acc_tol


def evict(cache_k, cache_v, acc, positions, lens, budget, sinks, recent, to):
    """The moves in plain Python: `to` = (k, v, acc, positions) CPU tensors that receive them
    (the inputs themselves when in place).  Returns the new lengths."""
    B, nkv, M, _ = cache_k.shape
    new = []
    for b in range(B):
        n_held = int(lens[b])
        n = min(n_held, budget)
        new.append(n)
        for h in range(nkv):
            w = acc[b, h].tolist()
            pos = positions[b, h].tolist() if positions is not None else list(range(M))
            newest = max(pos[:n_held], default=0)

            def rank(i):
                if pos[i] < sinks or pos[i] > newest - recent:
                    return (0, 0.0, i)
                return (1, math.inf if math.isnan(w[i]) else -w[i], i)

            kept = sorted(range(n_held), key=rank)[:n]
            stay = {i for i in kept if i < n}
            moves = list(zip([i for i in range(n) if i not in stay], sorted(i for i in kept if i >= n)))
            if to[0] is not cache_k:
                moves += [(i, i) for i in stay]
            for dst, src in moves:
                to[0][b, h, dst], to[1][b, h, dst] = cache_k[b, h, src], cache_v[b, h, src]
                to[2][b, h, dst] = w[src]
                if to[3] is not None:
                    to[3][b, h, dst] = pos[src]
    return new

"""The operators on the 8-bit key/value cache, restated from their definitions in 64 bits on the CPU.

A cache is two arrays of stored values (as the numbers they are, before the scale) and two of scales:
k, v [num_blocks, heads, block_size, head_dim] and k_scale, v_scale [num_blocks, heads], all float64.
"""
import math

import torch

TOP = {"int8": 127.0, "e4m3": 448.0}
TORCH = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def scale_for(amax: float, kind: str) -> float:
    """Least power of two s >= 2^-100 with amax <= top * s; NaN for what is not finite."""
    if not math.isfinite(amax):
        return math.nan
    s = 2.0 ** -100
    while amax > TOP[kind] * s:
        s *= 2
    return s


def to_stored(x: torch.Tensor, kind: str) -> torch.Tensor:
    """Nearest storable numbers, ties to even."""
    if kind == "int8":
        return x.round().clamp(-127, 127)
    step = torch.ldexp(torch.ones_like(x), (torch.frexp(x.abs().clamp_min(2.0 ** -6)).exponent - 4).to(torch.int32))
    return ((x / step).round() * step).clamp(-448, 448)


def append(cache, kind, table, lens, k, v, counts):
    """k, v: lists of [n_b, heads, d] float64.  Changes the cache in place."""
    bs = cache["k"].shape[2]
    for b, n in enumerate(counts):
        for name, x in (("k", k[b]), ("v", v[b])):
            for h in range(x.shape[1]):
                at = lens[b]
                while at < lens[b] + n:
                    j, first = at // bs, at % bs
                    end = min(bs, lens[b] + n - j * bs)
                    page = table[b][j]
                    new = x[at - lens[b]:at - lens[b] + end - first, h]
                    need = scale_for(new.abs().max().item(), kind)
                    old = cache[name + "_scale"][page, h].item()
                    after = need if first == 0 or math.isnan(need) or need > old else old
                    if first and not after == old:
                        cache[name][page, h, :first] = to_stored(cache[name][page, h, :first] * old / after, kind)
                    cache[name][page, h, first:end] = to_stored(new / after, kind)
                    cache[name + "_scale"][page, h] = after
                    at = j * bs + end


def rows(cache, name, table_row, n):
    """The first n tokens of a sequence [n, heads, d]."""
    bs = cache[name].shape[2]
    pages = [int(table_row[j]) for j in range((n + bs - 1) // bs)]
    if not pages:
        return torch.zeros(0, cache[name].shape[1], cache[name].shape[3], dtype=torch.float64)
    x = cache[name][pages] * cache[name + "_scale"][pages][:, :, None, None]
    return x.transpose(1, 2).flatten(0, 1)[:n]


def visible(p, n, window, sink):
    t = torch.arange(n)
    if window is None:
        return t <= p
    return (t <= p) & ((p - t <= window) | (t < sink))


def attn(cache, table, lens, q, window, sink, scale=None):
    """q [batch, queries, hq, d].  Returns out, lse, the weights [batch, heads, max len], sum of p|v| (for tolerances), and
    the largest sum of |q||k| * scale of a visible pair."""
    b, n, hq, d = q.shape
    hkv = cache["k"].shape[1]
    grp = hq // hkv
    scale = d ** -0.5 if scale is None else scale
    out, size = torch.zeros(b, n, hq, d, dtype=torch.float64), torch.zeros(b, n, hq, d, dtype=torch.float64)
    lse = torch.full((b, hq, n), -math.inf, dtype=torch.float64)
    w = torch.zeros(b, hkv, max([*lens, 1]), dtype=torch.float64)
    most = 0.0
    for i in range(b):
        k, v = rows(cache, "k", table[i], lens[i]), rows(cache, "v", table[i], lens[i])
        for j in range(n):
            p = lens[i] - n + j
            seen = visible(p, lens[i], window, sink)
            if not seen.any():
                continue
            qj = q[i, j].view(hkv, grp, d)
            s = torch.einsum("hgd,thd->hgt", qj, k[seen]) * scale
            most = max(most, (torch.einsum("hgd,thd->hgt", qj.abs(), k[seen].abs()) * scale).nan_to_num(0).max().item())
            lse[i, :, j] = torch.logsumexp(s, -1).flatten()
            pr = torch.softmax(s, -1)
            out[i, j] = torch.einsum("hgt,thd->hgd", pr, v[seen]).reshape(hq, d)
            size[i, j] = torch.einsum("hgt,thd->hgd", pr, v[seen].abs()).reshape(hq, d)
            w[i][:, :lens[i]][:, seen] += pr.sum(1)
    return out, lse, w, size, most


def weight_sums(q, k, lse, window, sink, scale, lens):
    """Packed: q [t, hq, d], k [t, hkv, d], lse [hq, t].  Returns sums [hkv, t], the largest sum of |q||k| * scale, the number of terms [t]."""
    t, hq, d = q.shape
    hkv = k.shape[1]
    grp = hq // hkv
    scale = d ** -0.5 if scale is None else scale
    out, terms, most, at = torch.zeros(hkv, t, dtype=torch.float64), torch.zeros(t), 0.0, 0
    for n in lens:
        seq = slice(at, at + n)
        i, j = torch.arange(n)[:, None], torch.arange(n)[None]
        seen = j <= i if window is None else (j <= i) & ((i - j <= window) | (j < sink))
        terms[seq] = seen.sum(0).float() * grp
        for h in range(hq):
            s = q[seq, h] @ k[seq, h // grp].T * scale
            most = max(most, (q[seq, h].abs() @ k[seq, h // grp].abs().T * scale).nan_to_num(0).max().item() if n else 0.0)
            w = (s - lse[h, seq].double()[:, None]).exp()
            w = torch.where(torch.isneginf(lse[h, seq])[:, None], torch.zeros_like(w), w)
            out[h // grp, seq] += torch.where(seen, w, torch.zeros_like(w)).sum(0)
        at += n
    return out, most, terms


def keep(w, n, budget, sink, recent):
    """The slots of one sequence and head that stay, in order: by sorting."""
    if n <= budget:
        return list(range(n))
    key = lambda t: -math.inf if math.isnan(w[t]) else -w[t]  # noqa: E731
    nan_first = sorted(range(sink, n - recent), key=lambda t: (not math.isnan(w[t]), key(t), t))
    return sorted([*range(sink), *nan_first[:budget - sink - recent], *range(n - recent, n)])


def evict(cache, kind, table, lens, weights, budget, new_table, sink, recent):
    """Changes the cache in place; returns new_lens, new weights as lists, kept as lists."""
    bs = cache["k"].shape[2]
    kept = [[keep(weights[b, h].tolist(), n, budget, sink, recent) for h in range(weights.shape[1])] for b, n in enumerate(lens)]
    for name in ("k", "v"):
        for b, n in enumerate(lens):
            x = rows(cache, name, table[b], n)
            for h, slots in enumerate(kept[b]):
                for at in range(0, len(slots), bs):
                    y = x[slots[at:at + bs], h]
                    page = int(new_table[b][at // bs])
                    s = scale_for(y.abs().max().item() if not torch.isnan(y).any() else math.nan, kind)
                    cache[name][page, h, :y.shape[0]] = to_stored(y / s, kind)
                    cache[name + "_scale"][page, h] = s
    return [min(n, budget) for n in lens], kept
